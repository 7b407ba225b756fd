"""Selective state space layers on the device: the short causal convolution and the scan, for whole sequences (with
gradients, initial and final states, padded batches) and for single tokens on a cache of streams.

A sequence layer next to the LSTM (unet_amd.lstm) and GRU (unet_amd.gru) recurrences, batch first like them.  Those carry a
matrix product from step to step and are latency-bound; here the state of every channel runs on its own,

    conv   y_t = silu(bias + sum_k weight_k x_{t-K+1+k})
    scan   dt = softplus(dt + dt_bias);  h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t;  y_t = (C_t . h_t + D x_t) silu(z_t)

so the time axis can be split over the chip.  Activations are fp32 or bfloat16 (all of one call alike), parameters fp32,
scan states fp32.  Inputs may be slices of wider tensors; only their last axis has to be dense (another is copied).
"""

import torch
from torch.autograd.function import once_differentiable

from . import seq_ops as _ops


def _index(t, low, high):
    """lengths / slots as the kernels take them: int32, other integer types held inside their useful range first."""
    if t is None or t.dtype == torch.int32:
        return t if t is None else t.contiguous()
    if t.dtype not in (torch.int64, torch.int16, torch.int8, torch.uint8):
        raise ValueError("unet_amd.ssm: lengths and slots are integer tensors, got {}".format(t.dtype))
    return t.clamp(low, high).to(torch.int32).contiguous()


def _needs_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _written(t):
    """The kernel wrote ``t`` through its pointer: what autograd saved of it is stale from here on."""
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


# ---------------------------------------------------------------------------------------------------------------------
# the causal convolution
# ---------------------------------------------------------------------------------------------------------------------
class _Conv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, lengths, silu, want_state):
        y, out = _ops.seq_conv(x, weight, bias, state, lengths, silu, want_state)
        ctx.save_for_backward(x, weight, bias, state, lengths)
        ctx.silu, ctx.checked = silu, (_ops._DTYPES[x.dtype], x.get_device(), *x.shape, weight.shape[1])
        ctx.set_materialize_grads(False)
        return y, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dout):
        x, weight, bias, state, lengths = ctx.saved_tensors
        if dy is None and dout is None:
            return (None,) * 7
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else dy
        if dout is not None:
            dout = dout.contiguous() if dout.numel() else None
        need = ctx.needs_input_grad
        if _ops.plain(dy):
            dx, dw, db, ds = _ops._conv_bwd(x, weight, bias, state, lengths, ctx.silu, dy, dout, need[3], ctx.checked)
        else:
            dx, dw, db, ds = _ops.seq_conv_bwd(x, weight, bias, state, lengths, ctx.silu, dy, dout)
        return (dx if need[0] else None, dw if need[1] else None, db if need[2] else None,
                ds if state is not None and need[3] else None, None, None, None)


def causal_conv(x, weight, bias=None, act=True, state=None, lengths=None, return_state=False):
    """x [batch, length, channels], weight [channels, taps] (2..4), bias [channels] -> y like x; SiLU unless ``act`` is False.

    state [batch, taps-1, channels]: the inputs before the first (zeros without).  lengths [batch]: where each sequence of a
    padded batch ends; y is zero from there on.  With return_state also the last taps-1 inputs of each sequence, the state
    that continues it (causal_conv again, or causal_conv_step).  Differentiable in x, weight, bias and state."""
    lengths = _index(lengths, 0, 2 ** 31 - 1)
    state = None if state is None else state.contiguous()
    if _needs_grad(x, weight, bias, state):
        y, out = _Conv.apply(x, weight.contiguous(), bias, state, lengths, bool(act), bool(return_state))
    else:
        y, out = _ops.seq_conv(x, weight, bias, state, lengths, bool(act), bool(return_state))
    return (y, out) if return_state else y


def causal_conv_step(x, state, weight, bias=None, act=True, slots=None):
    """One token of every row: x [rows, channels] -> y like x; inference only.

    state [num_slots, taps-1, channels] is a cache of streams, shifted in place; slots [rows] says which stream a row is
    (without: row i is stream i).  A negative slot is a padding row: zeros out, nothing touched.  A slot beyond the cache,
    or one that an earlier row of the call has, gives a row of NaN and touches nothing."""
    y = _ops.seq_conv_step(x, weight, bias, state, _index(slots, -1, 2 ** 31 - 1), bool(act))
    _written(state)
    return y


# ---------------------------------------------------------------------------------------------------------------------
# the scan
# ---------------------------------------------------------------------------------------------------------------------
class _Scan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state):
        y, out, marks = _ops.ssm_scan(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, True)
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, lengths, marks)
        ctx.softplus, ctx.has_state = softplus, state is not None
        ctx.checked = (_ops._DTYPES[x.dtype], x.get_device(), B.shape[-2] if B.dim() == 4 else 1, *A.shape)
        ctx.set_materialize_grads(False)
        return y, out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dout):
        x, dt, A, B, C, D, z, dt_bias, lengths, marks = ctx.saved_tensors
        if dy is None and dout is None:
            return (None,) * 12
        dy = torch.zeros(x.shape, dtype=x.dtype, device=x.device) if dy is None else dy
        if dout is not None:
            dout = dout.contiguous() if dout.numel() else None
        need = ctx.needs_input_grad
        args = (x, dt, A, B, C, D, z, dt_bias, lengths, ctx.softplus, marks, dy, dout, ctx.has_state and need[8])
        dx, ddt, dA, dB, dC, dD, dz, dbias, ds = _ops._scan_bwd(*args, ctx.checked) if _ops.plain(dy) else _ops.ssm_scan_bwd(*args)
        grads = (dx, ddt, dA, dB, dC, None if D is None else dD, None if z is None else dz, None if dt_bias is None else dbias,
                 ds if ctx.has_state else None)
        return tuple(g if n else None for g, n in zip(grads, need)) + (None, None, None)


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None, return_state=False):
    """x, dt, z [batch, length, channels], A [channels, N] (N <= 64; negative for a decaying state), B and C
    [batch, length, N] or [batch, length, groups, N], D and dt_bias [channels] -> y like x.

    softplus=False takes dt + dt_bias as the step sizes themselves.  state [batch, channels, N] fp32: where the recurrence
    starts (zeros without).  lengths [batch]: where each sequence of a padded batch ends; y is zero from there on.  With
    return_state also the state at each sequence's end.  Differentiable in every tensor but lengths."""
    lengths = _index(lengths, 0, 2 ** 31 - 1)
    A = A.contiguous()
    state = None if state is None else state.contiguous()
    if _needs_grad(x, dt, A, B, C, D, z, dt_bias, state):
        y, out = _Scan.apply(x, dt, A, B, C, D, z, dt_bias, state, lengths, bool(softplus), bool(return_state))
    else:
        y, out, _ = _ops.ssm_scan(x, dt, A, B, C, D, z, dt_bias, state, lengths, bool(softplus), bool(return_state), False)
    return (y, out) if return_state else y


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus=True, slots=None):
    """One token of every row: x, dt, z [rows, channels], B and C [rows, N] or [rows, groups, N] -> y like x; inference only.

    state [num_slots, channels, N] fp32 is a cache of streams, advanced in place; slots as in causal_conv_step."""
    y = _ops.ssm_scan_step(x, dt, A, B, C, D, z, dt_bias, state, _index(slots, -1, 2 ** 31 - 1), bool(softplus))
    _written(state)
    return y
