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

from . import seq_ops as _ops


def _index(t, low, high):
    """lengths / slots as the kernels take them: int32, 64-bit ones held inside their useful range first."""
    if t is None or (t.dtype is torch.int32 and t.is_contiguous()):
        return t
    if t.dtype is torch.int64:
        t = t.clamp(low, high)
    elif t.dtype not in (torch.int32, torch.int16, torch.int8, torch.uint8):
        raise ValueError("unet_amd.ssm: lengths and slots are integer tensors, got {}".format(t.dtype))
    return t.to(torch.int32).contiguous()


def _packed(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _flag(value, name):
    if value is not True and value is not False:
        raise ValueError("unet_amd.ssm: {} is True or False, got {!r}".format(name, value))
    return value


def causal_conv(x, weight, bias=None, act=True, state=None, lengths=None, return_state=False):
    """x [batch, length, channels], weight [channels, taps] (2..4), bias [channels] -> y like x; SiLU unless ``act`` is False.

    state [batch, taps-1, channels]: the inputs before the first (zeros without).  lengths [batch]: where each sequence of a
    padded batch ends; y is zero from there on.  With return_state also the last taps-1 inputs of each sequence, the state
    that continues it (causal_conv again, or causal_conv_step).  Differentiable (once) in x, weight, bias and state."""
    y, out = _ops.seq_conv(x, _packed(weight), bias, _packed(state), _index(lengths, 0, 2 ** 31 - 1), _flag(act, "act"),
                           bool(return_state))
    return (y, out) if return_state else y


def causal_conv_step(x, state, weight, bias=None, act=True, slots=None):
    """One token of every row: x [rows, channels] -> y like x; inference only (refused where autograd would record it).

    state [num_slots, taps-1, channels] is a cache of streams, shifted in place; slots [rows] says which stream a row is
    (without: row i is stream i).  A negative slot is a padding row: zeros out, nothing touched.  A slot beyond the cache,
    or one that an earlier row of the call has, gives a row of NaN and touches nothing."""
    return _ops.seq_conv_step(x, weight, bias, state, _index(slots, -1, 2 ** 31 - 1), _flag(act, "act"))


def selective_scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None, return_state=False):
    """x, dt, z [batch, length, channels], A [channels, N] (N <= 64; finite, negative for a decaying state), B and C
    [batch, length, N] or [batch, length, groups, N], D and dt_bias [channels] -> y like x.

    softplus=False takes dt + dt_bias as the step sizes themselves.  state [batch, channels, N] fp32: where the recurrence
    starts (zeros without).  lengths [batch]: where each sequence of a padded batch ends; y is zero from there on.  With
    return_state also the state at each sequence's end.  Differentiable (once) in every tensor but lengths."""
    y, out, _ = _ops.ssm_scan(x, dt, _packed(A), B, C, D, z, dt_bias, _packed(state), _index(lengths, 0, 2 ** 31 - 1),
                              _flag(softplus, "softplus"), bool(return_state), False)
    return (y, out) if return_state else y


def selective_scan_step(x, dt, A, B, C, state, D=None, z=None, dt_bias=None, softplus=True, slots=None):
    """One token of every row: x, dt, z [rows, channels], B and C [rows, N] or [rows, groups, N] -> y like x; inference only.

    state [num_slots, channels, N] fp32 is a cache of streams, advanced in place; slots and gradients as in causal_conv_step."""
    return _ops.ssm_scan_step(x, dt, A, B, C, D, z, dt_bias, state, _index(slots, -1, 2 ** 31 - 1), _flag(softplus, "softplus"))
