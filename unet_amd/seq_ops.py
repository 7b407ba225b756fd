"""torch.library registration of the sequence operators with the channels innermost (csrc/seq_conv.hip, csrc/ssm_scan.hip,
csrc/block_norm.hip): torch.ops.unetmi.seq_conv, .seq_conv_bwd, .seq_conv_step, .ssm_scan, .ssm_scan_bwd, .ssm_scan_step,
.block_norm and .block_norm_bwd.  ``unet_amd.ssm`` and ``unet_amd.norm`` are what user code calls: they add defaults and
autograd.

Outputs are dense; an output that a call does not have is an empty tensor.  Scratch memory is taken from torch's caching
allocator call by call (under graph capture: from the graph's own pool), never from a buffer that calls share.
"""

import torch

from . import _lib
from ._lib import PACK_NORM, PACK_SCAN, PACK_SEQ_CONV, check
from .ops import _LIBRARY, _ptr

_DTYPES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}
_FLOAT = torch.float32

_LIBRARY.define("seq_conv(Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu, bool want_state) "
                "-> (Tensor, Tensor)")
_LIBRARY.define("seq_conv_bwd(Tensor x, Tensor weight, Tensor? bias, Tensor? state, Tensor? lengths, bool silu, Tensor dy, "
                "Tensor? dstate_out) -> (Tensor, Tensor, Tensor, Tensor)")
_LIBRARY.define("seq_conv_step(Tensor x, Tensor weight, Tensor? bias, Tensor(a!) state, Tensor? slots, bool silu) -> Tensor")
_LIBRARY.define("ssm_scan(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, Tensor? state, "
                "Tensor? lengths, bool softplus, bool want_state, bool want_marks) -> (Tensor, Tensor, Tensor)")
_LIBRARY.define("ssm_scan_bwd(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, "
                "Tensor? lengths, bool softplus, Tensor marks, Tensor dy, Tensor? dstate_out, bool want_dstate) -> "
                "(Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor, Tensor)")
_LIBRARY.define("ssm_scan_step(Tensor x, Tensor dt, Tensor A, Tensor B, Tensor C, Tensor? D, Tensor? z, Tensor? dt_bias, "
                "Tensor(a!) state, Tensor? slots, bool softplus) -> Tensor")
_LIBRARY.define("block_norm(Tensor x, Tensor? gate, Tensor? post_weight, Tensor? residual, Tensor? scale, Tensor? pre_weight, "
                "float eps) -> (Tensor, Tensor)")
_LIBRARY.define("block_norm_bwd(Tensor x, Tensor? gate, Tensor? post_weight, Tensor? stream, Tensor? scale, Tensor? pre_weight, "
                "float eps, Tensor? d_out, Tensor? d_norm, bool has_residual, bool residual_f32) -> "
                "(Tensor, Tensor, Tensor, Tensor)")


MAX_STEP = 2 ** 25                # elements between two steps of an input (UNETMI_SEQ_MAX_STEP)

_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


def _refuse(op, name, t, dtype, shape, device):
    raise ValueError("unetmi::{}: {} must be a {} tensor of shape {} on device {}, got {} of shape {} on {}{}".format(
        op, name, dtype, tuple(shape), device, t.dtype, tuple(t.shape), t.device, "" if t.is_contiguous() else ", not contiguous"))


def _kind(x, op, dims):
    """(dtype code, device index) of a call's first activation."""
    if not x.is_cuda or x.dtype not in _DTYPES:
        raise ValueError("unetmi::{}: x must be a float32 or bfloat16 device tensor, got {} on {}".format(op, x.dtype, x.device))
    if x.dim() != dims:
        raise ValueError("unetmi::{}: x must have {} axes, got shape {}".format(op, dims, tuple(x.shape)))
    return _DTYPES[x.dtype], x.get_device()


def _same(t, name, op, dtype, dev, shape):
    """An activation of the call's type, device and shape."""
    if t.dtype is not dtype or t.get_device() != dev or t.shape != shape:
        _refuse(op, name, t, dtype, shape, dev)


def _dense(t, name, op, dtype, dev, shape):
    """A parameter, state or index tensor: contiguous too."""
    if t is not None and (t.dtype is not dtype or t.get_device() != dev or t.shape != shape or not t.is_contiguous()):
        _refuse(op, name, t, dtype, shape, dev)


def _rows(t):
    """(t, strides) with the last axis dense and steps not too far apart: a copy where they are not."""
    s = t.stride()
    if (s[-1] != 1 and t.shape[-1] > 1) or (len(s) > 2 and s[1] > MAX_STEP):
        t = t.contiguous()
        s = t.stride()
    return t, s


def _call(fn, what, dev, *args):
    """The entry point on the tensors' device and its current stream."""
    if dev == _current_device():
        code = fn(*args, _raw_stream(dev))
    else:
        with torch.cuda.device(dev):
            code = fn(*args, _raw_stream(dev))
    if code:
        check(code, what)


def _new(shape, dtype, like):
    return torch.empty(shape, dtype=dtype, device=like.device)


def _scratch(nbytes, like):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=like.device)


def plain(x):
    """An ordinary device tensor with no dispatch mode active: the public functions then call the implementations below
    themselves, which spares the dispatcher's part of a small call's time (5 of 20 us)."""
    return (x.is_cuda and (type(x) is torch.Tensor or type(x) is torch.nn.Parameter) and torch._C._len_torch_dispatch_stack() == 0
            and not torch.compiler.is_compiling())


# ---------------------------------------------------------------------------------------------------------------------
# the causal convolution
# ---------------------------------------------------------------------------------------------------------------------
def _conv_inputs(op, x, weight, bias, state, lengths):
    code, dev = _kind(x, op, 3)
    if weight.dim() != 2:
        raise ValueError("unetmi::{}: weight must be [channels, taps]".format(op))
    B, L, D = x.shape
    K = weight.shape[1]
    _dense(weight, "weight", op, _FLOAT, dev, (D, K))
    _dense(bias, "bias", op, _FLOAT, dev, (D,))
    _dense(state, "state", op, x.dtype, dev, (B, K - 1, D))
    _dense(lengths, "lengths", op, torch.int32, dev, (B,))
    return code, dev, B, L, D, K


def _seq_conv_cuda(x, weight, bias, state, lengths, silu, want_state):
    code, dev, B, L, D, K = _conv_inputs("seq_conv", x, weight, bias, state, lengths)
    x, s = _rows(x)
    y = _new((B, L, D), x.dtype, x)
    out = _new((B, K - 1, D) if want_state else (0,), x.dtype, x)
    d = PACK_SEQ_CONV.pack(B, L, D, K, _lib.ACT_SILU if silu else _lib.ACT_NONE, code, s[0], s[1], 0, 0)
    _call(_lib.lib.unetmi_seq_conv_fwd, "unetmi_seq_conv_fwd", dev, d, x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(state),
          _ptr(lengths), y.data_ptr(), out.data_ptr() if want_state else None)
    return y, out


def _seq_conv_bwd_cuda(x, weight, bias, state, lengths, silu, dy, dstate_out):
    """(dx, dweight [D, K], dbias [D], dstate or empty)"""
    op = "seq_conv_bwd"
    checked = _conv_inputs(op, x, weight, bias, state, lengths)
    _same(dy, "dy", op, x.dtype, checked[1], x.shape)
    _dense(dstate_out, "dstate_out", op, x.dtype, checked[1], (checked[2], checked[5] - 1, checked[4]))
    dx, dw, db, dstate = _conv_bwd(x, weight, bias, state, lengths, silu, dy, dstate_out, True, checked)
    return dx, dw, db, _new((0,), x.dtype, x) if dstate is None else dstate


def _conv_bwd(x, weight, bias, state, lengths, silu, dy, dstate_out, want_dstate, checked):
    """The launch, on inputs that were checked (by this call or by the forward call that saved them)."""
    code, dev, B, L, D, K = checked
    (x, s), (dy, g) = _rows(x), _rows(dy)
    dx, dw, db = _new((B, L, D), x.dtype, x), torch.empty_like(weight), _new((D,), _FLOAT, x)
    dstate = torch.empty_like(state) if want_dstate and state is not None else None
    if B == 0:
        return dx, dw.zero_(), db.zero_(), dstate
    d = PACK_SEQ_CONV.pack(B, L, D, K, _lib.ACT_SILU if silu else _lib.ACT_NONE, code, s[0], s[1], g[0], g[1])
    need = _lib.lib.unetmi_seq_conv_bwd_workspace_bytes(d)
    ws = _scratch(need, x)
    _call(_lib.lib.unetmi_seq_conv_bwd, "unetmi_seq_conv_bwd", dev, d, x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(state),
          _ptr(lengths), dy.data_ptr(), _ptr(dstate_out), dx.data_ptr(), dw.data_ptr(), db.data_ptr(),
          _ptr(dstate), ws.data_ptr(), ws.numel())
    return dx, dw, db, dstate


def _seq_conv_step_cuda(x, weight, bias, state, slots, silu):
    op = "seq_conv_step"
    code, dev = _kind(x, op, 2)
    if weight.dim() != 2 or state.dim() != 3:
        raise ValueError("unetmi::seq_conv_step: weight must be [channels, taps], state [slots, taps-1, channels]")
    B, D = x.shape
    K, n = weight.shape[1], state.shape[0]
    _dense(weight, "weight", op, _FLOAT, dev, (D, K))
    _dense(bias, "bias", op, _FLOAT, dev, (D,))
    _dense(state, "state", op, x.dtype, dev, (n, K - 1, D))
    _dense(slots, "slots", op, torch.int32, dev, (B,))
    x, s = _rows(x)
    y = _new((B, D), x.dtype, x)
    d = PACK_SEQ_CONV.pack(B, 1, D, K, _lib.ACT_SILU if silu else _lib.ACT_NONE, code, s[0], 0, 0, 0)
    _call(_lib.lib.unetmi_seq_conv_step, "unetmi_seq_conv_step", dev, d, x.data_ptr(), weight.data_ptr(), _ptr(bias), _ptr(slots), n,
          state.data_ptr(), y.data_ptr())
    return y


# ---------------------------------------------------------------------------------------------------------------------
# the scan
# ---------------------------------------------------------------------------------------------------------------------
def _scan_inputs(op, x, dt, A, B, C, D, z, dt_bias, dims):
    """Checks; B and C are [.., state] (one group) or [.., groups, state].  (code, dev, groups)"""
    code, dev = _kind(x, op, dims)
    shape, kind = x.shape, x.dtype
    _same(dt, "dt", op, kind, dev, shape)
    if z is not None:
        _same(z, "z", op, kind, dev, shape)
    if A.dim() != 2:
        raise ValueError("unetmi::{}: A must be [channels, state]".format(op))
    grouped = B.dim() == dims + 1
    groups = B.shape[-2] if grouped else 1
    N = A.shape[1]
    bc = shape[:-1] + ((groups, N) if grouped else (N,))
    _same(B, "B", op, kind, dev, bc)
    _same(C, "C", op, kind, dev, bc)
    channels = shape[-1]
    _dense(A, "A", op, _FLOAT, dev, (channels, N))
    _dense(D, "D", op, _FLOAT, dev, (channels,))
    _dense(dt_bias, "dt_bias", op, _FLOAT, dev, (channels,))
    return code, dev, groups, channels, N


def _scan_rows(x, dt, B, C, z, dy):
    """The inputs with rows that the kernels can walk, and the descriptor's strides."""
    x, xs = _rows(x)
    dt, ts = _rows(dt)
    B, bs = _rows(B)
    C, cs = _rows(C)
    z, zs = (None, (0, 0)) if z is None else _rows(z)
    dy, ys = (None, (0, 0)) if dy is None else _rows(dy)
    bg, cg = (bs[2], cs[2]) if len(bs) == 4 else (0, 0)
    return x, dt, B, C, z, dy, (xs[0], xs[1], ts[0], ts[1], zs[0], zs[1], ys[0], ys[1], bs[0], bs[1], bg, cs[0], cs[1], cg)


def _ssm_scan_cuda(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, want_marks):
    """(y, final state [B, channels, N] or empty, the states the backward call needs or empty)"""
    op, lib = "ssm_scan", _lib.lib
    code, dev, groups, channels, N = _scan_inputs(op, x, dt, A, B, C, D, z, dt_bias, 3)
    batch, length = x.shape[0], x.shape[1]
    _dense(state, "state", op, _FLOAT, dev, (batch, channels, N))
    _dense(lengths, "lengths", op, torch.int32, dev, (batch,))
    x, dt, B, C, z, _, strides = _scan_rows(x, dt, B, C, z, None)
    d = PACK_SCAN.pack(batch, length, channels, N, groups, code, softplus, 0, *strides)
    y = _new(x.shape, x.dtype, x)
    out = _new((batch, channels, N) if want_state else (0,), _FLOAT, x)
    marks = _new((lib.unetmi_ssm_scan_marks_bytes(d) // 4 if want_marks else 0,), _FLOAT, x)
    need = lib.unetmi_ssm_scan_fwd_workspace_bytes(d, lengths is not None)
    ws = _scratch(need, x) if need else None
    _call(lib.unetmi_ssm_scan_fwd, "unetmi_ssm_scan_fwd", dev, d, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(),
          _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(state), _ptr(lengths), y.data_ptr(), out.data_ptr() if want_state else None,
          marks.data_ptr() if want_marks else None, _ptr(ws), need)
    return y, out, marks


def _ssm_scan_bwd_cuda(x, dt, A, B, C, D, z, dt_bias, lengths, softplus, marks, dy, dstate_out, want_dstate):
    """(dx, ddt, dA, dB, dC, dD, dz or empty, ddt_bias, dstate or empty)"""
    op = "ssm_scan_bwd"
    checked = code, dev, groups, channels, N = _scan_inputs(op, x, dt, A, B, C, D, z, dt_bias, 3)
    batch, length = x.shape[0], x.shape[1]
    _same(dy, "dy", op, x.dtype, dev, x.shape)
    _dense(lengths, "lengths", op, torch.int32, dev, (batch,))
    _dense(dstate_out, "dstate_out", op, _FLOAT, dev, (batch, channels, N))
    size = PACK_SCAN.pack(batch, length, channels, N, groups, code, softplus, 0, *[0] * 14)
    _dense(marks, "marks", op, _FLOAT, dev, (_lib.lib.unetmi_ssm_scan_marks_bytes(size) // 4,))
    out = _scan_bwd(x, dt, A, B, C, D, z, dt_bias, lengths, softplus, marks, dy, dstate_out, want_dstate, checked)
    return tuple(_new((0,), _FLOAT if i == 8 else x.dtype, x) if t is None else t for i, t in enumerate(out))


def _scan_bwd(x, dt, A, B, C, D, z, dt_bias, lengths, softplus, marks, dy, dstate_out, want_dstate, checked):
    """The launch, on inputs that were checked (by this call or by the forward call that saved them)."""
    code, dev, groups, channels, N = checked
    lib = _lib.lib
    batch, length = x.shape[0], x.shape[1]
    x, dt, B, C, z, dy, strides = _scan_rows(x, dt, B, C, z, dy)
    d = PACK_SCAN.pack(batch, length, channels, N, groups, code, softplus, 0, *strides)
    kind = x.dtype
    dx, dB = _new(x.shape, kind, x), _new(B.shape, kind, x)
    ddt, dC, dz = torch.empty_like(dx), torch.empty_like(dB), None if z is None else torch.empty_like(dx)
    dA, dD = torch.empty_like(A), _new((channels,), _FLOAT, x)
    dbias = torch.empty_like(dD)
    dstate = _new((batch, channels, N), _FLOAT, x) if want_dstate else None
    if batch == 0:
        dA.zero_(), dD.zero_(), dbias.zero_()
    else:
        ws = _scratch(lib.unetmi_ssm_scan_bwd_workspace_bytes(d, lengths is not None), x)
        _call(lib.unetmi_ssm_scan_bwd, "unetmi_ssm_scan_bwd", dev, d, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(), C.data_ptr(),
              _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(lengths), marks.data_ptr(), dy.data_ptr(), _ptr(dstate_out), dx.data_ptr(),
              ddt.data_ptr(), dA.data_ptr(), dB.data_ptr(), dC.data_ptr(), dD.data_ptr(), dbias.data_ptr(),
              _ptr(dz), _ptr(dstate), ws.data_ptr(), ws.numel())
    return dx, ddt, dA, dB, dC, dD, dz, dbias, dstate


def _ssm_scan_step_cuda(x, dt, A, B, C, D, z, dt_bias, state, slots, softplus):
    op = "ssm_scan_step"
    code, dev, groups, channels, N = _scan_inputs(op, x, dt, A, B, C, D, z, dt_bias, 2)
    if state.dim() != 3:
        raise ValueError("unetmi::ssm_scan_step: state must be [slots, channels, state]")
    batch, n = x.shape[0], state.shape[0]
    _dense(state, "state", op, _FLOAT, dev, (n, channels, N))
    _dense(slots, "slots", op, torch.int32, dev, (batch,))
    x, xs = _rows(x)
    dt, ts = _rows(dt)
    B, bs = _rows(B)
    C, cs = _rows(C)
    z, zs = (None, (0,)) if z is None else _rows(z)
    bg, cg = (bs[1], cs[1]) if len(bs) == 3 else (0, 0)
    d = PACK_SCAN.pack(batch, 1, channels, N, groups, code, softplus, 0, xs[0], 0, ts[0], 0, zs[0], 0, 0, 0, bs[0], 0, bg, cs[0], 0, cg)
    y = _new(x.shape, x.dtype, x)
    _call(_lib.lib.unetmi_ssm_scan_step, "unetmi_ssm_scan_step", dev, d, x.data_ptr(), dt.data_ptr(), A.data_ptr(), B.data_ptr(),
          C.data_ptr(), _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(slots), n, state.data_ptr(), y.data_ptr())
    return y


# ---------------------------------------------------------------------------------------------------------------------
# the block norm
# ---------------------------------------------------------------------------------------------------------------------
def _norm_inputs(op, x, gate, post_weight, residual, scale, pre_weight, eps, residual_dtype):
    """(x, gate, residual, dev, descriptor) after the checks."""
    code, dev = _kind(x, op, 2)
    shape, kind = x.shape, x.dtype
    width = (shape[1],)
    _dense(post_weight, "post_weight", op, _FLOAT, dev, width)
    _dense(scale, "scale", op, _FLOAT, dev, width)
    _dense(pre_weight, "pre_weight", op, _FLOAT, dev, width)
    x, xs = _rows(x)
    gs = rs = (0,)
    if gate is not None:
        _same(gate, "gate", op, kind, dev, shape)
        gate, gs = _rows(gate)
    if residual is not None:
        residual_dtype = residual.dtype
        _same(residual, "residual", op, _FLOAT if residual_dtype is _FLOAT else kind, dev, shape)
        residual, rs = _rows(residual)
    return x, gate, residual, dev, PACK_NORM.pack(shape[0], shape[1], code, _DTYPES[residual_dtype], eps, xs[0], gs[0], rs[0])


def _block_norm_cuda(x, gate, post_weight, residual, scale, pre_weight, eps):
    """(r, n) with a residual (n empty without pre_weight), else (p, empty)"""
    x, gate, residual, dev, d = _norm_inputs("block_norm", x, gate, post_weight, residual, scale, pre_weight, eps, x.dtype)
    if residual is None and (scale is not None or pre_weight is not None):
        raise ValueError("unetmi::block_norm: scale and pre_weight belong to a residual stream")
    out = _new(x.shape, x.dtype if residual is None else residual.dtype, x)
    out_n = _new((0,) if pre_weight is None else x.shape, x.dtype, x)
    _call(_lib.lib.unetmi_block_norm_fwd, "unetmi_block_norm_fwd", dev, d, x.data_ptr(), _ptr(gate), _ptr(post_weight), _ptr(residual),
          _ptr(scale), _ptr(pre_weight), out.data_ptr(), None if pre_weight is None else out_n.data_ptr())
    return out, out_n


def _block_norm_bwd_cuda(x, gate, post_weight, stream, scale, pre_weight, eps, d_out, d_norm, has_residual, residual_f32):
    """(dx, dgate or empty, dresidual or empty, [dpost_weight, dscale, dpre_weight])"""
    op = "block_norm_bwd"
    rdtype = _FLOAT if residual_f32 else x.dtype
    x, gate, stream, dev, d = _norm_inputs(op, x, gate, post_weight, stream, scale, pre_weight, eps, rdtype)
    _dense(d_out, "d_out", op, rdtype if has_residual else x.dtype, dev, x.shape)
    _dense(d_norm, "d_norm", op, x.dtype, dev, x.shape)
    dx, dgate, dres, dweights = _norm_bwd(x, gate, post_weight, stream, scale, pre_weight, d_out, d_norm,
                                          rdtype if has_residual else None, (dev, d))
    return dx, _new((0,), x.dtype, x) if dgate is None else dgate, _new((0,), rdtype, x) if dres is None else dres, dweights


def _norm_bwd(x, gate, post_weight, stream, scale, pre_weight, d_out, d_norm, residual_dtype, checked):
    """The launch, on inputs that were checked."""
    dev, d = checked
    dx = _new(x.shape, x.dtype, x)
    dgate = None if gate is None else torch.empty_like(dx)
    dres = None if residual_dtype is None else _new(x.shape, residual_dtype, x)
    dweights = _new((3, x.shape[1]), _FLOAT, x)
    if x.shape[0] == 0:
        return dx, dgate, dres, dweights.zero_()
    ws = _scratch(_lib.lib.unetmi_block_norm_bwd_workspace_bytes(d), x)
    _call(_lib.lib.unetmi_block_norm_bwd, "unetmi_block_norm_bwd", dev, d, x.data_ptr(), _ptr(gate), _ptr(post_weight), _ptr(stream),
          _ptr(scale), _ptr(pre_weight), _ptr(d_out), _ptr(d_norm), dx.data_ptr(), _ptr(dgate),
          _ptr(dres), dweights.data_ptr(), ws.data_ptr(), ws.numel())
    return dx, dgate, dres, dweights


for _name, _fn in (("seq_conv", _seq_conv_cuda), ("seq_conv_bwd", _seq_conv_bwd_cuda), ("seq_conv_step", _seq_conv_step_cuda),
                   ("ssm_scan", _ssm_scan_cuda), ("ssm_scan_bwd", _ssm_scan_bwd_cuda), ("ssm_scan_step", _ssm_scan_step_cuda),
                   ("block_norm", _block_norm_cuda), ("block_norm_bwd", _block_norm_bwd_cuda)):
    _LIBRARY.impl(_name, _fn, "CUDA")


def _states_per_lane(n):
    return 1 if n <= 4 else 2 if n <= 8 else 4 if n <= 16 else 8 if n <= 32 else 16


@torch.library.register_fake("unetmi::seq_conv")
def _(x, weight, bias, state, lengths, silu, want_state):
    return x.new_empty(x.shape), x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2]) if want_state else (0,))


@torch.library.register_fake("unetmi::seq_conv_bwd")
def _(x, weight, bias, state, lengths, silu, dy, dstate_out):
    return (x.new_empty(x.shape), weight.new_empty(weight.shape), weight.new_empty((x.shape[2],)),
            x.new_empty((0,) if state is None else state.shape))


@torch.library.register_fake("unetmi::seq_conv_step")
def _(x, weight, bias, state, slots, silu):
    return x.new_empty(x.shape)


@torch.library.register_fake("unetmi::ssm_scan")
def _(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, want_marks):
    S = _states_per_lane(A.shape[1])
    steps = 16 if S <= 2 else 8 if S == 4 else 4
    marks = x.shape[0] * ((x.shape[1] + steps - 1) // steps) * x.shape[2] * 4 * S
    return (x.new_empty(x.shape), A.new_empty((x.shape[0],) + tuple(A.shape) if want_state else (0,)),
            A.new_empty((marks if want_marks else 0,)))


@torch.library.register_fake("unetmi::ssm_scan_bwd")
def _(x, dt, A, B, C, D, z, dt_bias, lengths, softplus, marks, dy, dstate_out, want_dstate):
    e = x.new_empty
    return (e(x.shape), e(x.shape), A.new_empty(A.shape), e(B.shape), e(B.shape), A.new_empty((A.shape[0],)),
            e((0,) if z is None else x.shape), A.new_empty((A.shape[0],)),
            A.new_empty((x.shape[0],) + tuple(A.shape) if want_dstate else (0,)))


@torch.library.register_fake("unetmi::ssm_scan_step")
def _(x, dt, A, B, C, D, z, dt_bias, state, slots, softplus):
    return x.new_empty(x.shape)


@torch.library.register_fake("unetmi::block_norm")
def _(x, gate, post_weight, residual, scale, pre_weight, eps):
    return (x.new_empty(x.shape, dtype=x.dtype if residual is None else residual.dtype),
            x.new_empty((0,) if pre_weight is None else x.shape))


@torch.library.register_fake("unetmi::block_norm_bwd")
def _(x, gate, post_weight, stream, scale, pre_weight, eps, d_out, d_norm, has_residual, residual_f32):
    return (x.new_empty(x.shape), x.new_empty((0,) if gate is None else x.shape),
            x.new_empty(x.shape if has_residual else (0,), dtype=_FLOAT if residual_f32 else x.dtype),
            x.new_empty((3, x.shape[1]), dtype=_FLOAT))


def _entry(name, impl):
    """The dispatcher's op, or its implementation itself where nothing else would look at the call."""
    op = getattr(torch.ops.unetmi, name).default

    def call(x, *args):
        return impl(x, *args) if plain(x) else op(x, *args)

    return call


seq_conv, seq_conv_bwd, seq_conv_step = (_entry("seq_conv", _seq_conv_cuda), _entry("seq_conv_bwd", _seq_conv_bwd_cuda),
                                         _entry("seq_conv_step", _seq_conv_step_cuda))
ssm_scan, ssm_scan_bwd, ssm_scan_step = (_entry("ssm_scan", _ssm_scan_cuda), _entry("ssm_scan_bwd", _ssm_scan_bwd_cuda),
                                         _entry("ssm_scan_step", _ssm_scan_step_cuda))
block_norm, block_norm_bwd = _entry("block_norm", _block_norm_cuda), _entry("block_norm_bwd", _block_norm_bwd_cuda)
