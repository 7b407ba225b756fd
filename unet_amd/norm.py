"""The norms before and after a block of a residual stream, fused with the block's gate and the residual scale.

The networks of this package normalise per convolution channel (BatchNorm folded into the convolutions, layernorm_f,
layernorm_w_act); a block whose channels are innermost -- a state space layer, unet_amd.ssm -- norms over them instead:

    u = x silu(gate);  p = post_weight u / rms(u);  r = residual + scale p;  n = pre_weight r / rms(r)
"""

import torch
from torch.autograd.function import once_differentiable

from . import seq_ops as _ops


class _BlockNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, gate, post_weight, residual, scale, pre_weight, eps):
        out, out_n = _ops.block_norm(x, gate, post_weight, residual, scale, pre_weight, eps)
        ctx.save_for_backward(x, gate, post_weight, scale, pre_weight, out if pre_weight is not None else None)
        ctx.eps = eps
        ctx.residual = None if residual is None else residual.dtype
        ctx.set_materialize_grads(False)
        return out, out_n

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_norm):
        x, gate, post_weight, scale, pre_weight, stream = ctx.saved_tensors
        if pre_weight is None:
            d_norm = None
        if d_out is None and d_norm is None:
            return (None,) * 7
        d_out = None if d_out is None else d_out.contiguous()
        d_norm = None if d_norm is None else d_norm.contiguous()
        has = ctx.residual is not None
        dx, dgate, dres, dw = _ops.block_norm_bwd(x, gate, post_weight, stream, scale, pre_weight, ctx.eps, d_out, d_norm, has,
                                                  has and ctx.residual == torch.float32)
        d_post, d_scale, d_pre = dw.unbind()
        grads = (dx, None if gate is None else dgate, None if post_weight is None else d_post, dres if has else None,
                 None if scale is None else d_scale, None if pre_weight is None else d_pre)
        return tuple(g if n else None for g, n in zip(grads, ctx.needs_input_grad)) + (None,)


def block_norm(x, gate=None, post_weight=None, residual=None, scale=None, pre_weight=None, eps=1e-6):
    """x [..., channels] (channels <= 8192) -> p; with a residual -> r; with a residual and pre_weight -> (r, n).

    Every part is optional: without a gate u = x, without post_weight p = u, without a scale r = residual + p.  scale and the
    weights are fp32 [channels]; scale may also be a single value.  x and gate are fp32 or bfloat16; the residual stream is of
    their type or fp32, and r is what the stream becomes.  Differentiable in every tensor."""
    if residual is None and (scale is not None or pre_weight is not None):
        raise ValueError("unet_amd.norm: scale and pre_weight belong to a residual stream")
    shape = x.shape
    if scale is not None and scale.numel() == 1:
        scale = scale.reshape(1).expand(shape[-1])
    flat = [None if t is None else _flat(t, shape) for t in (x, gate, residual)]
    weights = [None if t is None else t.contiguous() for t in (post_weight, scale, pre_weight)]
    args = (flat[0], flat[1], weights[0], flat[2], weights[1], weights[2], float(eps))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:6]):
        out, out_n = _BlockNorm.apply(*args)
    else:
        out, out_n = _ops.block_norm(*args)
    return out.view(shape) if pre_weight is None else (out.view(shape), out_n.view(shape))


def _flat(t, shape):
    """[..., channels] as rows; a copy only where the rows are not evenly spaced."""
    if t.shape != shape:
        raise ValueError("unet_amd.norm: x, gate and residual have one shape, got {} and {}".format(tuple(shape), tuple(t.shape)))
    return t if t.dim() == 2 else t.reshape(-1, shape[-1])
