"""The norms before and after a block of a residual stream, fused with the block's gate and the residual scale.

The networks of this package normalise per convolution channel (BatchNorm folded into the convolutions, layernorm_f,
layernorm_w_act); a block whose channels are innermost -- a state space layer, unet_amd.ssm -- norms over them instead:

    u = x silu(gate);  p = post_weight u / rms(u);  r = residual + scale p;  n = pre_weight r / rms(r)
"""

from . import seq_ops as _ops


def _packed(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def block_norm(x, gate=None, post_weight=None, residual=None, scale=None, pre_weight=None, eps=1e-6):
    """x [..., channels] (channels <= 8192) -> p; with a residual -> r; with a residual and pre_weight -> (r, n).

    Every part is optional: without a gate u = x, without post_weight p = u, without a scale r = residual + p.  scale and the
    weights are fp32 [channels]; scale may also be a tensor of one value.  x and gate are fp32 or bfloat16; the residual stream is of
    their type or fp32, and r is what the stream becomes.  Differentiable (once) in every tensor."""
    if residual is None and (scale is not None or pre_weight is not None):
        raise ValueError("unet_amd.norm: scale and pre_weight belong to a residual stream")
    shape = x.shape
    rows = len(shape) == 2
    if not rows:                                          # [..., channels] as rows: a copy only where they are not evenly spaced
        for t in (gate, residual):
            if t is not None and t.shape != shape:
                raise ValueError("unet_amd.norm: x, gate and residual have one shape, got {} and {}".format(tuple(shape), tuple(t.shape)))
        x, gate, residual = (None if t is None else t.reshape(-1, shape[-1]) for t in (x, gate, residual))
    if scale is not None and scale.numel() == 1:
        scale = scale.reshape(1).expand(shape[-1])
    out, out_n, _ = _ops.block_norm(x, gate, _packed(post_weight), residual, _packed(scale), _packed(pre_weight), eps, False)
    if not rows:
        out, out_n = out.view(shape), out_n if pre_weight is None else out_n.view(shape)
    return out if pre_weight is None else (out, out_n)
