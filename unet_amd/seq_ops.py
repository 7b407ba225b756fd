"""torch.library registration of the sequence operators with the channels innermost (csrc/seq_conv.hip, csrc/ssm_scan.hip,
csrc/block_norm.hip): torch.ops.unetmi.seq_conv, .seq_conv_bwd, .seq_conv_step, .ssm_scan, .ssm_scan_bwd, .ssm_scan_step,
.block_norm and .block_norm_bwd.  ``unet_amd.ssm`` and ``unet_amd.norm`` are what user code calls: they add defaults and
autograd.

Outputs are dense; an output that a call does not have is an empty tensor.  Scratch memory is taken from torch's caching
allocator call by call (under graph capture: from the graph's own pool), never from a buffer that calls share.
"""

import ctypes

import torch

from . import _lib
from ._lib import NormDesc, ScanDesc, SeqConvDesc, check
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


def _act(t, name, op, like=None, shape=None):
    """An activation: fp32 or bfloat16 on the device of ``like``, of its type, with a dense last axis."""
    if not t.is_cuda or t.dtype not in _DTYPES:
        raise ValueError("unetmi::{}: {} must be a float32 or bfloat16 device tensor, got {} on {}".format(op, name, t.dtype, t.device))
    if like is not None and (t.dtype != like.dtype or t.device != like.device):
        raise ValueError("unetmi::{}: {} is {} on {}, expected {} on {}".format(op, name, t.dtype, t.device, like.dtype, like.device))
    if shape is not None and t.shape != shape:
        raise ValueError("unetmi::{}: {} has shape {}, expected {}".format(op, name, tuple(t.shape), tuple(shape)))
    if t.stride(-1) != 1 and t.shape[-1] > 1:
        raise ValueError("unetmi::{}: the last axis of {} must be dense".format(op, name))


def _dense(t, name, op, like, shape, dtype=_FLOAT):
    """A parameter, state or index tensor: dense, of one type and shape, on the device of ``like``."""
    if t is None:
        return
    if t.device != like.device or t.dtype != dtype or t.shape != shape or not t.is_contiguous():
        raise ValueError("unetmi::{}: {} must be a contiguous {} tensor of shape {} on {}, got {} of shape {} on {}".format(
            op, name, dtype, tuple(shape), like.device, t.dtype, tuple(t.shape), t.device))


class _On:
    """The device of a tensor made current (without a call where it is already), and its stream."""
    __slots__ = ("guard", "stream")

    def __init__(self, t):
        index = t.device.index
        self.guard = None if index == torch.cuda.current_device() else torch.cuda.device(index)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        self.stream = torch.cuda.current_stream().cuda_stream
        return self.stream

    def __exit__(self, *exc):
        if self.guard is not None:
            self.guard.__exit__(*exc)


def _scratch(nbytes, like):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=like.device)


# ---------------------------------------------------------------------------------------------------------------------
# the causal convolution
# ---------------------------------------------------------------------------------------------------------------------
def _conv_desc(op, x, weight, bias, silu):
    _act(x, "x", op)
    if x.dim() != 3 or weight.dim() != 2:
        raise ValueError("unetmi::{}: x must be [batch, length, channels] and weight [channels, taps]".format(op))
    B, L, D = x.shape
    K = weight.shape[1]
    _dense(weight, "weight", op, x, (D, K))
    _dense(bias, "bias", op, x, (D,))
    return SeqConvDesc(B, L, D, K, _lib.ACT_SILU if silu else _lib.ACT_NONE, _DTYPES[x.dtype], (x.stride(0), x.stride(1)), (0, 0))


def _seq_conv_cuda(x, weight, bias, state, lengths, silu, want_state):
    d = _conv_desc("seq_conv", x, weight, bias, silu)
    B, L, D = x.shape
    K = weight.shape[1]
    _dense(state, "state", "seq_conv", x, (B, K - 1, D), x.dtype)
    _dense(lengths, "lengths", "seq_conv", x, (B,), torch.int32)
    y = torch.empty((B, L, D), dtype=x.dtype, device=x.device)
    out = torch.empty((B, K - 1, D) if want_state else (0,), dtype=x.dtype, device=x.device)
    with _On(x) as stream:
        check(_lib.lib.unetmi_seq_conv_fwd(ctypes.byref(d), _ptr(x), _ptr(weight), _ptr(bias), _ptr(state), _ptr(lengths), _ptr(y),
                                           _ptr(out) if want_state else None, stream), "unetmi_seq_conv_fwd")
    return y, out


def _seq_conv_bwd_cuda(x, weight, bias, state, lengths, silu, dy, dstate_out):
    """(dx, dweight [D, K], dbias [D], dstate or empty)"""
    d = _conv_desc("seq_conv_bwd", x, weight, bias, silu)
    B, L, D = x.shape
    K = weight.shape[1]
    _dense(state, "state", "seq_conv_bwd", x, (B, K - 1, D), x.dtype)
    _dense(lengths, "lengths", "seq_conv_bwd", x, (B,), torch.int32)
    _dense(dstate_out, "dstate_out", "seq_conv_bwd", x, (B, K - 1, D), x.dtype)
    _act(dy, "dy", "seq_conv_bwd", x, x.shape)
    d.dy_stride[0], d.dy_stride[1] = dy.stride(0), dy.stride(1)
    dx = torch.empty((B, L, D), dtype=x.dtype, device=x.device)
    dw, db = torch.empty((D, K), dtype=_FLOAT, device=x.device), torch.empty((D,), dtype=_FLOAT, device=x.device)
    dstate = torch.empty((0,) if state is None else (B, K - 1, D), dtype=x.dtype, device=x.device)
    if B == 0:
        return dx, dw.zero_(), db.zero_(), dstate
    need = _lib.lib.unetmi_seq_conv_bwd_workspace_bytes(ctypes.byref(d))
    ws = _scratch(need, x)
    with _On(x) as stream:
        check(_lib.lib.unetmi_seq_conv_bwd(ctypes.byref(d), _ptr(x), _ptr(weight), _ptr(bias), _ptr(state), _ptr(lengths), _ptr(dy),
                                           _ptr(dstate_out), _ptr(dx), _ptr(dw), _ptr(db), None if state is None else _ptr(dstate),
                                           _ptr(ws), ws.numel(), stream), "unetmi_seq_conv_bwd")
    return dx, dw, db, dstate


def _seq_conv_step_cuda(x, weight, bias, state, slots, silu):
    op = "seq_conv_step"
    _act(x, "x", op)
    if x.dim() != 2 or weight.dim() != 2 or state.dim() != 3:
        raise ValueError("unetmi::seq_conv_step: x must be [rows, channels], weight [channels, taps], state [slots, taps-1, channels]")
    B, D = x.shape
    K = weight.shape[1]
    _dense(weight, "weight", op, x, (D, K))
    _dense(bias, "bias", op, x, (D,))
    _dense(state, "state", op, x, (state.shape[0], K - 1, D), x.dtype)
    _dense(slots, "slots", op, x, (B,), torch.int32)
    d = SeqConvDesc(B, 1, D, K, _lib.ACT_SILU if silu else _lib.ACT_NONE, _DTYPES[x.dtype], (x.stride(0), 0), (0, 0))
    y = torch.empty((B, D), dtype=x.dtype, device=x.device)
    with _On(x) as stream:
        check(_lib.lib.unetmi_seq_conv_step(ctypes.byref(d), _ptr(x), _ptr(weight), _ptr(bias), _ptr(slots), state.shape[0],
                                            _ptr(state), _ptr(y), stream), "unetmi_seq_conv_step")
    return y


# ---------------------------------------------------------------------------------------------------------------------
# the scan
# ---------------------------------------------------------------------------------------------------------------------
def _scan_desc(op, x, dt, A, B, C, D, z, dt_bias, softplus, step=False):
    _act(x, "x", op)
    lead = x.shape[:-1]
    if x.dim() != (2 if step else 3) or A.dim() != 2 or B.dim() != x.dim() + 1:
        raise ValueError("unetmi::{}: x must be [batch, {}channels], A [channels, state], B and C [batch, {}groups, state]".format(
            op, "" if step else "length, ", "" if step else "length, "))
    channels, (groups, state) = x.shape[-1], B.shape[-2:]
    _act(dt, "dt", op, x, x.shape)
    _act(B, "B", op, x, lead + (groups, A.shape[1]))
    _act(C, "C", op, x, B.shape)
    if z is not None:
        _act(z, "z", op, x, x.shape)
    _dense(A, "A", op, x, (channels, state))
    _dense(D, "D", op, x, (channels,))
    _dense(dt_bias, "dt_bias", op, x, (channels,))
    if step:
        return ScanDesc(x.shape[0], 1, channels, state, groups, _DTYPES[x.dtype], int(softplus), 0, (x.stride(0), 0), (dt.stride(0), 0),
                        (0 if z is None else z.stride(0), 0), (0, 0), (B.stride(0), 0, B.stride(1)), (C.stride(0), 0, C.stride(1)))
    return ScanDesc(x.shape[0], x.shape[1], channels, state, groups, _DTYPES[x.dtype], int(softplus), 0, x.stride()[:2], dt.stride()[:2],
                    (0, 0) if z is None else z.stride()[:2], (0, 0), B.stride()[:3], C.stride()[:3])


def _ssm_scan_cuda(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, want_marks):
    """(y, final state [B, channels, N] or empty, the states the backward call needs or empty)"""
    op = "ssm_scan"
    d = _scan_desc(op, x, dt, A, B, C, D, z, dt_bias, softplus)
    shape = (x.shape[0], x.shape[2], A.shape[1])
    _dense(state, "state", op, x, shape)
    _dense(lengths, "lengths", op, x, (x.shape[0],), torch.int32)
    ref, lib = ctypes.byref(d), _lib.lib
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    out = torch.empty(shape if want_state else (0,), dtype=_FLOAT, device=x.device)
    marks = torch.empty((lib.unetmi_ssm_scan_marks_bytes(ref) // 4 if want_marks else 0,), dtype=_FLOAT, device=x.device)
    need = lib.unetmi_ssm_scan_fwd_workspace_bytes(ref)
    ws = _scratch(need, x) if need else None
    with _On(x) as stream:
        check(lib.unetmi_ssm_scan_fwd(ref, _ptr(x), _ptr(dt), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z), _ptr(dt_bias), _ptr(state),
                                      _ptr(lengths), _ptr(y), _ptr(out) if want_state else None, _ptr(marks) if want_marks else None,
                                      _ptr(ws), need, stream), "unetmi_ssm_scan_fwd")
    return y, out, marks


def _ssm_scan_bwd_cuda(x, dt, A, B, C, D, z, dt_bias, lengths, softplus, marks, dy, dstate_out, want_dstate):
    """(dx, ddt, dA, dB, dC, dD, dz or empty, ddt_bias, dstate or empty)"""
    op = "ssm_scan_bwd"
    d = _scan_desc(op, x, dt, A, B, C, D, z, dt_bias, softplus)
    _act(dy, "dy", op, x, x.shape)
    d.dy_stride[0], d.dy_stride[1] = dy.stride(0), dy.stride(1)
    ref, lib = ctypes.byref(d), _lib.lib
    shape = (x.shape[0], x.shape[2], A.shape[1])
    _dense(lengths, "lengths", op, x, (x.shape[0],), torch.int32)
    _dense(dstate_out, "dstate_out", op, x, shape)
    _dense(marks, "marks", op, x, (lib.unetmi_ssm_scan_marks_bytes(ref) // 4,))

    def new(s, dtype=x.dtype):
        return torch.empty(s, dtype=dtype, device=x.device)

    dx, ddt, dB, dC = new(x.shape), new(x.shape), new(B.shape), new(B.shape)
    dz = new((0,) if z is None else x.shape)
    dA, dD, dbias = new(A.shape, _FLOAT), new(x.shape[2:], _FLOAT), new(x.shape[2:], _FLOAT)
    dstate = new(shape if want_dstate else (0,), _FLOAT)
    if x.shape[0] == 0:
        dA.zero_(), dD.zero_(), dbias.zero_()
    else:
        need = lib.unetmi_ssm_scan_bwd_workspace_bytes(ref)
        ws = _scratch(need, x)
        with _On(x) as stream:
            check(lib.unetmi_ssm_scan_bwd(ref, _ptr(x), _ptr(dt), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z), _ptr(dt_bias),
                                          _ptr(lengths), _ptr(marks), _ptr(dy), _ptr(dstate_out), _ptr(dx), _ptr(ddt), _ptr(dA),
                                          _ptr(dB), _ptr(dC), _ptr(dD), _ptr(dbias), None if z is None else _ptr(dz),
                                          _ptr(dstate) if want_dstate else None, _ptr(ws), ws.numel(), stream), "unetmi_ssm_scan_bwd")
    return dx, ddt, dA, dB, dC, dD, dz, dbias, dstate


def _ssm_scan_step_cuda(x, dt, A, B, C, D, z, dt_bias, state, slots, softplus):
    op = "ssm_scan_step"
    d = _scan_desc(op, x, dt, A, B, C, D, z, dt_bias, softplus, step=True)
    if state.dim() != 3:
        raise ValueError("unetmi::ssm_scan_step: state must be [slots, channels, state]")
    _dense(state, "state", op, x, (state.shape[0], x.shape[1], A.shape[1]))
    _dense(slots, "slots", op, x, (x.shape[0],), torch.int32)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    with _On(x) as stream:
        check(_lib.lib.unetmi_ssm_scan_step(ctypes.byref(d), _ptr(x), _ptr(dt), _ptr(A), _ptr(B), _ptr(C), _ptr(D), _ptr(z),
                                            _ptr(dt_bias), _ptr(slots), state.shape[0], _ptr(state), _ptr(y), stream),
              "unetmi_ssm_scan_step")
    return y


# ---------------------------------------------------------------------------------------------------------------------
# the block norm
# ---------------------------------------------------------------------------------------------------------------------
def _norm_desc(op, x, gate, post_weight, residual, scale, pre_weight, eps, residual_dtype):
    _act(x, "x", op)
    if x.dim() != 2:
        raise ValueError("unetmi::{}: x must be [rows, channels]".format(op))
    if gate is not None:
        _act(gate, "gate", op, x, x.shape)
    if residual is not None:
        _act(residual, "residual", op, None, x.shape)
        if residual.device != x.device or residual.dtype not in (x.dtype, _FLOAT):
            raise ValueError("unetmi::{}: residual must be float32 or of x's type, on x's device".format(op))
        residual_dtype = residual.dtype
    for t, name in ((post_weight, "post_weight"), (scale, "scale"), (pre_weight, "pre_weight")):
        _dense(t, name, op, x, (x.shape[1],))
    return NormDesc(x.shape[0], x.shape[1], _DTYPES[x.dtype], _DTYPES[residual_dtype], eps, x.stride(0),
                    0 if gate is None else gate.stride(0), 0 if residual is None else residual.stride(0))


def _block_norm_cuda(x, gate, post_weight, residual, scale, pre_weight, eps):
    """(r, n) with a residual (n empty without pre_weight), else (p, empty)"""
    d = _norm_desc("block_norm", x, gate, post_weight, residual, scale, pre_weight, eps, x.dtype)
    if residual is None and (scale is not None or pre_weight is not None):
        raise ValueError("unetmi::block_norm: scale and pre_weight belong to a residual stream")
    out = torch.empty(x.shape, dtype=x.dtype if residual is None else residual.dtype, device=x.device)
    out_n = torch.empty((0,) if pre_weight is None else x.shape, dtype=x.dtype, device=x.device)
    with _On(x) as stream:
        check(_lib.lib.unetmi_block_norm_fwd(ctypes.byref(d), _ptr(x), _ptr(gate), _ptr(post_weight), _ptr(residual), _ptr(scale),
                                             _ptr(pre_weight), _ptr(out), None if pre_weight is None else _ptr(out_n), stream),
              "unetmi_block_norm_fwd")
    return out, out_n


def _block_norm_bwd_cuda(x, gate, post_weight, stream, scale, pre_weight, eps, d_out, d_norm, has_residual, residual_f32):
    """(dx, dgate or empty, dresidual or empty, [dpost_weight, dscale, dpre_weight])"""
    op = "block_norm_bwd"
    rdtype = _FLOAT if residual_f32 else x.dtype
    d = _norm_desc(op, x, gate, post_weight, stream, scale, pre_weight, eps, rdtype)
    for t, name, dtype in ((d_out, "d_out", rdtype if has_residual else x.dtype), (d_norm, "d_norm", x.dtype)):
        _dense(t, name, op, x, x.shape, dtype)
    dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    dgate = torch.empty((0,) if gate is None else x.shape, dtype=x.dtype, device=x.device)
    dres = torch.empty(x.shape if has_residual else (0,), dtype=rdtype, device=x.device)
    dweights = torch.empty((3, x.shape[1]), dtype=_FLOAT, device=x.device)
    if x.shape[0] == 0:
        return dx, dgate, dres, dweights.zero_()
    ws = _scratch(_lib.lib.unetmi_block_norm_bwd_workspace_bytes(ctypes.byref(d)), x)
    with _On(x) as s:
        check(_lib.lib.unetmi_block_norm_bwd(ctypes.byref(d), _ptr(x), _ptr(gate), _ptr(post_weight), _ptr(stream), _ptr(scale),
                                             _ptr(pre_weight), _ptr(d_out), _ptr(d_norm), _ptr(dx), None if gate is None else _ptr(dgate),
                                             _ptr(dres) if has_residual else None, _ptr(dweights), _ptr(ws), ws.numel(), s),
              "unetmi_block_norm_bwd")
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
    steps = 16 if S <= 4 else 64 // S
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


seq_conv = torch.ops.unetmi.seq_conv.default
seq_conv_bwd = torch.ops.unetmi.seq_conv_bwd.default
seq_conv_step = torch.ops.unetmi.seq_conv_step.default
ssm_scan = torch.ops.unetmi.ssm_scan.default
ssm_scan_bwd = torch.ops.unetmi.ssm_scan_bwd.default
ssm_scan_step = torch.ops.unetmi.ssm_scan_step.default
block_norm = torch.ops.unetmi.block_norm.default
block_norm_bwd = torch.ops.unetmi.block_norm_bwd.default
