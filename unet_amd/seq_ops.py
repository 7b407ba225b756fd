"""The sequence operators with the channels innermost as dispatcher ops: torch.ops.unetmi.seq_conv, .seq_conv_bwd,
.seq_conv_step, .ssm_scan, .ssm_scan_bwd, .ssm_scan_step, .block_norm and .block_norm_bwd.

Their checks, launches and autograd nodes are C++ (csrc/torch_seq.cpp, libunetmi_torch.so) over the same C entry points as
the other ops'; this module loads it, ties it to the library that ``_lib`` has loaded, and gives the ops their shape
inference.  ``unet_amd.ssm`` and ``unet_amd.norm`` are what user code calls.
"""

import ctypes
import os
import re

import torch

from . import _lib

TORCH_LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libunetmi_torch.so")


def _load():
    """None, or why the library is not there."""
    again = "build it with `python -c 'import __graft_entry__ as g; g.build()'` or `make -C unet_amd/csrc`; there is no fallback path"
    if not os.path.exists(TORCH_LIB_PATH):
        return "{} is missing -- {}".format(TORCH_LIB_PATH, again)
    try:
        torch.ops.load_library(TORCH_LIB_PATH)
    except OSError as e:                                  # built against another torch, say
        return "{} does not load ({}) -- {}".format(TORCH_LIB_PATH, e.__cause__ or e, again)
    if ctypes.CDLL(TORCH_LIB_PATH).unetmi_torch_bind(os.fsencode(_lib.LIB_PATH)) != 0:
        raise ImportError("unet_amd: {} does not export the sequence operators".format(_lib.LIB_PATH))
    return None


# The rest of the package needs ctypes alone: without this library it still imports, and these operators raise when they are called.
unavailable = _load()


def _states_per_lane(n):
    return 1 if n <= 4 else 2 if n <= 8 else 4 if n <= 16 else 8 if n <= 32 else 16


def _fake(name):
    return torch.library.register_fake(name) if unavailable is None else lambda f: f


@_fake("unetmi::seq_conv")
def _(x, weight, bias, state, lengths, silu, want_state):
    return x.new_empty(x.shape), x.new_empty((x.shape[0], weight.shape[1] - 1, x.shape[2]) if want_state else (0,))


@_fake("unetmi::seq_conv_bwd")
def _(x, weight, bias, state, lengths, silu, dy, dstate_out):
    return (x.new_empty(x.shape), weight.new_empty(weight.shape), weight.new_empty((x.shape[2],)),
            x.new_empty((0,) if state is None else state.shape))


@_fake("unetmi::seq_conv_step")
def _(x, weight, bias, state, slots, silu):
    return x.new_empty(x.shape)


@_fake("unetmi::ssm_scan")
def _(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, want_marks):
    S = _states_per_lane(A.shape[1])
    steps = 16 if S <= 2 else 8 if S == 4 else 4
    marks = x.shape[0] * ((x.shape[1] + steps - 1) // steps) * x.shape[2] * 4 * S
    return (x.new_empty(x.shape), A.new_empty((x.shape[0],) + tuple(A.shape) if want_state else (0,)),
            A.new_empty((marks if want_marks else 0,)))


@_fake("unetmi::ssm_scan_bwd")
def _(x, dt, A, B, C, D, z, dt_bias, lengths, softplus, marks, dy, dstate_out, want_dstate):
    e = x.new_empty
    return (e(x.shape), e(x.shape), A.new_empty(A.shape), e(B.shape), e(B.shape), A.new_empty((A.shape[0],)),
            e((0,) if z is None else x.shape), A.new_empty((A.shape[0],)),
            A.new_empty((x.shape[0],) + tuple(A.shape) if want_dstate else (0,)))


@_fake("unetmi::ssm_scan_step")
def _(x, dt, A, B, C, D, z, dt_bias, state, slots, softplus):
    return x.new_empty(x.shape)


@_fake("unetmi::block_norm")
def _(x, gate, post_weight, residual, scale, pre_weight, eps, want_stats):
    return (x.new_empty(x.shape, dtype=x.dtype if residual is None else residual.dtype),
            x.new_empty((0,) if pre_weight is None else x.shape),
            x.new_empty((x.shape[0], 2) if want_stats else (0,), dtype=torch.float32))


@_fake("unetmi::block_norm_bwd")
def _(x, gate, post_weight, residual, scale, pre_weight, eps, stats, d_out, d_norm, has_residual, residual_f32):
    return (x.new_empty(x.shape), x.new_empty((0,) if gate is None else x.shape),
            x.new_empty(x.shape if has_residual else (0,), dtype=torch.float32 if residual_f32 else x.dtype),
            x.new_empty((3, x.shape[1]), dtype=torch.float32))


def _entry(name):
    """The op, with what an entry point of the library refuses raised as the package's UnetmiError."""
    if unavailable is not None:
        def missing(*args):
            raise ImportError("unet_amd: the sequence operators are not available: " + unavailable)

        return missing
    op = getattr(torch.ops.unetmi, name).default

    def call(*args):
        try:
            return op(*args)
        except RuntimeError as e:
            refused = re.match(r"unetmi_\w+ failed \((-?\d+)\): [^\n]*", str(e))
            if refused is None:
                raise
            raise _lib.UnetmiError(refused[0], int(refused[1])) from None

    return call


seq_conv, seq_conv_step, ssm_scan, ssm_scan_step, block_norm = (
    _entry(n) for n in ("seq_conv", "seq_conv_step", "ssm_scan", "ssm_scan_step", "block_norm"))
