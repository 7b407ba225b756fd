"""64-bit restatements of the sequence operators (unet_amd.ssm, unet_amd.norm), one step of time after the other.

Every function takes ``magnitude``: with it, each product and sum is taken of absolute values, so that the result bounds,
element by element, the sum of the magnitudes of everything that was added up.  A computed value is then held to

    |got - want| <= roundings * 2^-24 * magnitude + half a step of the output's type

where ``roundings`` counts the fp32 roundings that the longest chain into one element can have.
"""

import torch


def sig(v):
    return torch.sigmoid(v)


def ends_of(lengths, batch, length):
    return torch.full((batch,), length) if lengths is None else lengths.cpu().long().clamp(0, length)


def f64(t):
    return None if t is None else t.detach().cpu().double()


def conv64(x, w, bias, state, lengths, silu, dy=None, dout=None, magnitude=False):
    """dict(y, state) and, with dy, dict(dx, dw, db, dstate)."""
    x, w, bias, state, dy, dout = (f64(t) for t in (x, w, bias, state, dy, dout))
    B, L, D = x.shape
    K = w.shape[1]
    bias = torch.zeros(D, dtype=torch.float64) if bias is None else bias
    state = torch.zeros(B, K - 1, D, dtype=torch.float64) if state is None else state
    mag = (lambda t: t.abs()) if magnitude else (lambda t: t)
    ends = ends_of(lengths, B, L)
    out = {"y": torch.zeros_like(x), "state": torch.zeros_like(state)}
    grads = {"dx": torch.zeros_like(x), "dw": torch.zeros_like(w), "db": torch.zeros_like(bias), "dstate": torch.zeros_like(state)}
    for b in range(B):
        n = int(ends[b])
        seen = torch.cat([state[b], x[b, :n]], 0)
        out["state"][b] = mag(seen[n:])
        d_seen = torch.zeros_like(seen)
        if dout is not None:
            d_seen[n:] += mag(dout[b])
        for t in range(n):
            terms = seen[t:t + K] * w.t()
            pre = terms.sum(0) + bias
            wide = terms.abs().sum(0) + bias.abs()
            slope = torch.ones_like(pre)
            if silu:
                out["y"][b, t] = wide * sig(pre) * (1 + wide) if magnitude else pre * sig(pre)
                slope = 1 + 2 * wide if magnitude else sig(pre) * (1 + pre * (1 - sig(pre)))
            else:
                out["y"][b, t] = wide if magnitude else pre
            if dy is not None:
                d = mag(dy[b, t]) * slope
                grads["db"] += d
                grads["dw"] += (mag(seen[t:t + K]) * d).t()
                d_seen[t:t + K] += mag(w.t()) * d
        grads["dx"][b, :n] = d_seen[K - 1:]
        grads["dstate"][b] = d_seen[:K - 1]
    if dy is not None or dout is not None:
        out.update(grads)
    return out


def scan64(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None, dy=None, dout=None, magnitude=False):
    """dict(y, state) and, with dy, the gradients dict(x, dt, A, B, C, D, z, dt_bias, state0)."""
    x, dt, A, B, C, D, z, dt_bias, state, dy, dout = (f64(t) for t in (x, dt, A, B, C, D, z, dt_bias, state, dy, dout))
    batch, L, ch = x.shape
    G, N = B.shape[-2:]
    group = torch.arange(ch) // (ch // G)
    zero = torch.zeros(ch, dtype=torch.float64)
    raw = dt + (zero if dt_bias is None else dt_bias)
    step = torch.nn.functional.softplus(raw, threshold=800) if softplus else raw
    skip = zero if D is None else D
    mag = (lambda t: t.abs()) if magnitude else (lambda t: t)
    x, B, C, skip = mag(x), mag(B)[:, :, group], mag(C)[:, :, group], mag(skip)
    size = mag(step)
    ends = ends_of(lengths, batch, L)
    h = torch.zeros(batch, ch, N, dtype=torch.float64) if state is None else mag(state)
    # fp32 has no normal number below 2^-126: a gate's sigmoid that small may come out as zero, off by up to 2^-126, which is
    # 2^-102 in units of 2^-24 (z below -87; the product of z, the sigmoid and y can still be a normal number)
    gate = torch.ones_like(x) if z is None else (mag(z) * (sig(z) + 2.0 ** -102) * (1 + mag(z)) if magnitude else z * sig(z))
    out = {"y": torch.zeros_like(x)}
    hs, bare = [h], torch.zeros_like(x)
    decay = lambda t: torch.exp(step[:, t, :, None] * A)  # noqa: E731
    for t in range(L):
        new = decay(t) * h + (size[:, t] * x[:, t])[..., None] * B[:, t]
        inside = (ends > t)[:, None]
        h = torch.where(inside[..., None], new, h)
        hs.append(h)
        bare[:, t] = torch.where(inside, (h * C[:, t]).sum(-1) + skip * x[:, t], zero)
        out["y"][:, t] = torch.where(inside, bare[:, t] * gate[:, t], zero)
    out["state"] = h
    if dy is None and dout is None:
        return out
    dy = torch.zeros_like(x) if dy is None else mag(dy)
    dy = torch.where((torch.arange(L)[None] < ends[:, None])[..., None], dy, zero)
    g = torch.zeros_like(h) if dout is None else mag(dout)
    d = {k: torch.zeros_like(x) for k in ("x", "dt", "z")}
    dB, dC = torch.zeros(batch, L, ch, N, dtype=torch.float64), torch.zeros(batch, L, ch, N, dtype=torch.float64)
    dA, dD = torch.zeros_like(A), torch.zeros_like(zero)
    if z is not None:
        s = sig(z)
        d["z"] = dy * bare * ((1 + 2 * z.abs()) if magnitude else s * (1 + z * (1 - s)))
    dyg = dy * gate
    for t in range(L - 1, -1, -1):
        inside = (ends > t)[:, None]
        keep = lambda v: torch.where(inside if v.dim() == 2 else inside[..., None], v, torch.zeros_like(v))  # noqa: E731
        ahead = g + dyg[:, t, :, None] * C[:, t]
        dC[:, t] = keep(dyg[:, t, :, None] * hs[t + 1])
        dB[:, t] = keep(ahead * (size[:, t] * x[:, t])[..., None])
        du = (ahead * B[:, t]).sum(-1)
        back = ahead * decay(t)
        w = back * hs[t]
        dstep = (w * mag(A)).sum(-1) + du * x[:, t]
        slope = sig(raw[:, t]) if softplus else torch.ones_like(dstep)
        d["dt"][:, t] = keep(dstep * slope * (1 + raw[:, t].abs() if magnitude and softplus else 1))
        d["x"][:, t] = keep(du * size[:, t] + dyg[:, t] * skip)
        dA += keep(w * size[:, t, :, None]).sum(0)
        dD += keep(dyg[:, t] * x[:, t]).sum(0)
        g = torch.where(inside[..., None], back, g)
    out.update(d_x=d["x"], d_dt=d["dt"], d_z=d["z"], d_A=dA, d_D=dD, d_dt_bias=d["dt"].sum((0, 1)), d_state=g,
               d_B=dB.unflatten(2, (G, ch // G)).sum(3), d_C=dC.unflatten(2, (G, ch // G)).sum(3))
    return out


def norm64(x, gate, post, residual, scale, pre, eps, d_out=None, d_norm=None, magnitude=False):
    """dict(p or r, n) and, with gradients given, dict(d_x, d_gate, d_post, d_residual, d_scale, d_pre)."""
    x, gate, post, residual, scale, pre, d_out, d_norm = (f64(t) for t in (x, gate, post, residual, scale, pre, d_out, d_norm))
    mag = (lambda t: t.abs()) if magnitude else (lambda t: t)
    u = mag(x)
    slope = None
    if gate is not None:
        s = sig(gate)
        u = u * mag(gate * s) * (1 + gate.abs() if magnitude else 1)
        slope = (1 + 2 * gate.abs()) if magnitude else s * (1 + gate * (1 - s))
        g_val = mag(gate * s) * (1 + gate.abs() if magnitude else 1)
    plain_u = x if gate is None else x * gate * sig(gate)
    inv_u = torch.rsqrt(plain_u.pow(2).mean(-1, keepdim=True) + eps)
    p = u if post is None else u * inv_u * mag(post)
    out = {}
    if residual is None:
        out["p"] = p
    else:
        plain_p = plain_u if post is None else plain_u * inv_u * post
        plain_r = residual + (plain_p if scale is None else scale * plain_p)
        r = mag(residual) + (p if scale is None else mag(scale) * p)
        inv_r = torch.rsqrt(plain_r.pow(2).mean(-1, keepdim=True) + eps)
        out["r"] = r
        if pre is not None:
            out["n"] = r * inv_r * mag(pre)
    if d_out is None and d_norm is None:
        return out
    d_p = torch.zeros_like(x) if d_out is None else mag(d_out)
    sign = 1 if magnitude else -1
    if residual is not None:
        d_r = d_p
        if pre is not None and d_norm is not None:
            inv, rr = inv_r, r
            g = mag(d_norm) * mag(pre)
            out["d_pre"] = (mag(d_norm) * rr * inv).sum(0)
            d_r = d_r + inv * (g + sign * rr * inv * inv * (g * rr).mean(-1, keepdim=True))
        out["d_residual"] = d_r
        out["d_scale"] = (d_r * p).sum(0)
        d_p = d_r if scale is None else d_r * mag(scale)
    d_u = d_p
    if post is not None:
        out["d_post"] = (d_p * u * inv_u).sum(0)
        g = d_p * mag(post)
        d_u = inv_u * (g + sign * u * inv_u * inv_u * (g * u).mean(-1, keepdim=True))
    if gate is not None:
        out["d_gate"] = d_u * mag(x) * slope
        d_u = d_u * g_val
    out["d_x"] = d_u
    return out


def held(got, want, magnitude, roundings, what):
    """|got - want| within the roundings of the computation and half a step of the result's type, element by element."""
    assert tuple(got.shape) == tuple(want.shape), "{}: {} against {}".format(what, tuple(got.shape), tuple(want.shape))
    if not want.numel():
        return
    half = torch.finfo(got.dtype).eps / 2
    g = got.detach().cpu().double()
    assert torch.isfinite(g).all(), what + ": not finite"
    computed = roundings * 2.0 ** -24 * magnitude
    room = computed + half * (want.abs() + computed) + 1e-37
    worst = ((g - want).abs() / room).max().item()
    print("{}: {:.3f} of the room".format(what, worst))
    assert worst <= 1.0, "{}: {:.2f} times the room that its roundings leave".format(what, worst)
