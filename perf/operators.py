"""The selective state space operators and the fused block norm: cases, their plain forms and their exact values.

Three operators, each with its serving and its training form:

conv   y_t = silu(bias + sum_k w_k x_{t-K+1+k}) along time for every channel (x [batch, length, channels]), over the
       inputs that came before the prompt, for prompts, for single tokens on a cache of slots, and with its gradients.
scan   h_t = exp(dt_t A) h_{t-1} + dt_t x_t B_t,   y_t = (C_t . h_t + D x_t) silu(z_t),   dt = softplus(raw + bias):
       A [channels, state], B and C [batch, length, groups, state] shared by the channels of a group.
norm   u = x silu(gate),  p = w_post u / rms(u),  r = residual + scale p,  n = w_pre r / rms(r): what stands between two
       blocks of a residual stream, any of its parts left out.

``run`` computes the plain form in 32 bits, or with ``own`` makes the calls of unet_amd.ssm / unet_amd.norm.
"""

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one stream of an enhancement service, one frame at a time: the latency of the smallest call
        dict(name="scan token 1 stream", op="scan", mode="token", dtype="bf16", batch=1, channels=1280, state=16, groups=1, slots=1),
        # a full server: 256 streams taken out of a cache of 320 slots
        dict(name="scan token 256 streams", op="scan", mode="token", dtype="bf16", batch=256, channels=2048, state=16, groups=1, slots=320),
        # one long recording on its own: few rows, a long time axis
        dict(name="scan prompt 1 x 8192", op="scan", mode="prompt", dtype="bf16", batch=1, length=8192, channels=2048, state=16, groups=1, ragged=False),
        # a padded batch of recordings of odd lengths, one of them empty
        dict(name="scan prompt ragged 8 x 2001", op="scan", mode="prompt", dtype="bf16", batch=8, length=2001, channels=1280, state=16, groups=2, ragged=True),
        # the bottleneck of a U-Net in training: 32 x 4 frequency rows of 501 frames, twice the 128 channels
        dict(name="scan train 128 x 501", op="scan", mode="train", dtype="fp32", batch=128, length=501, channels=256, state=16, groups=1),
        # the largest: a wide model's training step
        dict(name="scan train 4 x 4096", op="scan", mode="train", dtype="bf16", batch=4, length=4096, channels=2048, state=16, groups=1),
        # the convolution of the same server
        dict(name="conv token 256 streams", op="conv", mode="token", dtype="bf16", batch=256, channels=2048, taps=4, slots=320),
        # the convolution of a padded batch of prompts
        dict(name="conv prompt 8 x 4096", op="conv", mode="prompt", dtype="bf16", batch=8, length=4096, channels=2048, taps=4, ragged=True),
        # the recurrent bottleneck's width (2 x 384) in fp32 training at 501 frames
        dict(name="conv train 32 x 501", op="conv", mode="train", dtype="fp32", batch=32, length=501, channels=768, taps=4),
        # between two blocks while single frames are served
        dict(name="norm token 64 rows", op="norm", mode="infer", dtype="bf16", rows=64, channels=2048, form="full"),
        # between two blocks over a batch of prompts, an odd number of rows
        dict(name="norm prompt 16387 rows", op="norm", mode="infer", dtype="bf16", rows=16387, channels=2048, form="full"),
        # the gate and the norm inside a block in fp32 training, an odd width
        dict(name="norm train 16032 rows", op="norm", mode="train", dtype="fp32", rows=16032, channels=1285, form="full"),
    ]


def spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["conv", "scan", "scan", "norm"])
    dtype = rng.choice(["fp32", "bf16"])
    most = 4 * 4096 * 2048                              # elements of the largest listed case
    if op == "norm":
        channels = spread(rng, 64, 4096)
        rows = spread(rng, 1, min(20000, most // channels))
        return dict(op=op, mode=rng.choice(["infer", "train"]), dtype=dtype, rows=rows, channels=channels,
                    form=rng.choice(["gate", "residual", "post", "full"]))
    mode = rng.choice(["token", "prompt", "train"])
    groups = rng.choice([1, 1, 2])
    channels = groups * spread(rng, 32, 1024)
    if mode == "token":
        case = dict(op=op, mode=mode, dtype=dtype, batch=spread(rng, 1, 256), channels=channels)
        case["slots"] = case["batch"] + rng.randrange(64)
    else:
        case = dict(op=op, mode=mode, dtype=dtype, length=spread(rng, 1, 4096), channels=channels)
        case["batch"] = spread(rng, 1, max(1, min(128, most // 4 // (channels * case["length"]))))
        if mode == "prompt":
            case["ragged"] = rng.random() < 0.5
    if op == "conv":
        case["taps"] = rng.choice([2, 3, 4])
    else:
        case["state"] = rng.choice([4, 7, 8, 12, 16, 16, 16])
        case["groups"] = groups
    return case


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    gen = torch.Generator(device=dev).manual_seed(int(seed) * 7919 + 17)
    kind = DTYPES[case["dtype"]]

    def normal(*shape, dtype=torch.float32, scale=1.0, shift=0.0):
        return (torch.randn(shape, generator=gen, device=dev) * scale + shift).to(dtype)

    def uniform(low, high, *shape):
        return torch.rand(shape, generator=gen, device=dev) * (high - low) + low

    c = case["channels"]
    s = {"case": dict(case)}
    if case["op"] == "norm":
        rows, form = case["rows"], case["form"]
        s["x"] = normal(rows, c, dtype=kind)
        if form in ("gate", "full"):
            s["gate"] = normal(rows, c, dtype=kind)
        if form != "residual":
            s["post_weight"] = uniform(0.5, 1.5, c)
        if form in ("residual", "full"):
            s["residual"] = normal(rows, c, dtype=kind, scale=2.0)
            s["scale"] = uniform(0.1, 1.0, c)
            s["pre_weight"] = uniform(0.5, 1.5, c)
        if case["mode"] == "train":
            s["d_first"] = normal(rows, c, dtype=kind)
            if "residual" in s:
                s["d_second"] = normal(rows, c, dtype=kind)
        return s

    batch, mode = case["batch"], case["mode"]
    lead = (batch,) if mode == "token" else (batch, case["length"])
    if mode == "token":
        # the streams of this step, in no order, out of the cache's slots
        s["slots"] = torch.randperm(case["slots"], generator=gen, device=dev)[:batch].to(torch.int32)
    if mode == "prompt" and case["ragged"]:
        lengths = torch.randint(1, case["length"] + 1, (batch,), generator=gen, device=dev, dtype=torch.int32)
        lengths[0] = case["length"]
        if batch > 2:
            lengths[batch // 2] = 0
        s["lengths"] = lengths
    # x and z as the two halves of one projection, as a block has them
    xz = normal(*lead, 2 * c, dtype=kind)
    s["x"] = xz[..., :c]
    if case["op"] == "conv":
        k = case["taps"]
        s["weight"], s["bias"] = uniform(-0.5, 0.5, c, k), uniform(-0.5, 0.5, c)
        if mode != "train":
            s["state"] = normal(case["slots"] if mode == "token" else batch, k - 1, c, dtype=kind)
    else:
        n, g = case["state"], case["groups"]
        s["z"] = xz[..., c:]
        # the logarithm of the step sizes spread over 1e-3 .. 1e-1, where softplus is small
        step = torch.exp(uniform(math.log(1e-3), math.log(1e-1), c))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))
        s["dt"] = normal(*lead, c, dtype=kind, scale=0.7)
        bc = normal(*lead, 2 * g * n, dtype=kind)
        s["B"], s["C"] = (t.unflatten(-1, (g, n)) for t in (bc[..., :g * n], bc[..., g * n:]))
        s["A"] = -torch.arange(1, n + 1, device=dev, dtype=torch.float32) * uniform(0.8, 1.25, c, n)
        s["D"] = uniform(0.5, 1.5, c)
        if mode != "train":
            s["state"] = normal(case["slots"] if mode == "token" else batch, c, n)
    if mode == "train":
        s["d_y"] = normal(*lead, c, dtype=kind)
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------------------------------------------------
def silu(v):
    return v / (1.0 + torch.exp(-v))


def silu_slope(v):
    s = 1.0 / (1.0 + torch.exp(-v))
    return s * (1.0 + v * (1.0 - s))


def softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-torch.abs(v)))


def valid(lengths, length):
    return torch.arange(length, device=lengths.device)[None, :] < lengths[:, None]


def taps_of(padded, weight, length):
    """sum_k w_k x_{t+k} of the inputs with the ones before them in front."""
    return sum(weight[:, k] * padded[:, k:k + length] for k in range(weight.shape[1]))


def conv_infer(s):
    x, weight, state = s["x"].float(), s["weight"], s["state"]
    k = weight.shape[1]
    if "slots" in s:
        rows = s["slots"].long()
        window = torch.cat([state[rows].float(), x[:, None]], 1)
        y = silu((window * weight.t()).sum(1) + s["bias"])
        state[rows] = window[:, 1:].to(state.dtype)
        return {"y": y.to(s["x"].dtype), "state": state}
    length = x.shape[1]
    padded = torch.cat([state.float(), x], 1)
    y = silu(taps_of(padded, weight, length) + s["bias"])
    ends = torch.full((x.shape[0],), length, device=x.device)
    if "lengths" in s:
        ends = s["lengths"].long()
        y = torch.where(valid(ends, length)[..., None], y, torch.zeros_like(y))
    last = ends[:, None] + torch.arange(k - 1, device=x.device)
    after = padded.gather(1, last[..., None].expand(-1, -1, x.shape[2]))
    return {"y": y.to(s["x"].dtype), "state": after.to(state.dtype)}


def conv_train(s):
    x, weight, dy = s["x"].float(), s["weight"], s["d_y"].float()
    length, k, kind = x.shape[1], weight.shape[1], s["x"].dtype
    padded = torch.nn.functional.pad(x, (0, 0, k - 1, 0))
    pre = taps_of(padded, weight, length) + s["bias"]
    d_pre = dy * silu_slope(pre)
    d_x = taps_of(torch.nn.functional.pad(d_pre, (0, 0, 0, k - 1)), weight.flip(1), length)
    d_weight = torch.stack([(d_pre * padded[:, j:j + length]).sum((0, 1)) for j in range(k)], 1)
    return {"y": silu(pre).to(kind), "d_x": d_x.to(kind), "d_weight": d_weight, "d_bias": d_pre.sum((0, 1))}


def recurrence(a, b):
    """h_t = a_t h_{t-1} + b_t along axis 1 from zero: the steps are taken in pairs, the pairs' recurrence is half as long."""
    length = a.shape[1]
    if length == 1:
        return b
    half = length // 2
    odd = recurrence(a[:, 1::2] * a[:, 0:2 * half:2], a[:, 1::2] * b[:, 0:2 * half:2] + b[:, 1::2])
    h = torch.empty_like(b)
    h[:, 1::2] = odd
    h[:, 0] = b[:, 0]
    rest = (length - 1) // 2
    h[:, 2::2] = a[:, 2::2] * odd[:, :rest] + b[:, 2::2]
    return h


def per_channel(t, channels):
    """[..., groups, state] of a group for each of its channels: [..., channels, state]."""
    return t.float().repeat_interleave(channels // t.shape[-2], dim=-2)


def scan_infer(s):
    x, z, A, state = s["x"].float(), s["z"].float(), s["A"], s["state"]
    c, kind = x.shape[-1], s["x"].dtype
    dt = softplus(s["dt"].float() + s["dt_bias"])
    B, C = per_channel(s["B"], c), per_channel(s["C"], c)
    if "slots" in s:
        rows = s["slots"].long()
        h = torch.exp(dt[..., None] * A) * state[rows] + (dt * x)[..., None] * B
        y = ((h * C).sum(-1) + s["D"] * x) * silu(z)
        state[rows] = h
        return {"y": y.to(kind), "state": state}
    length = x.shape[1]
    keep = None
    if "lengths" in s:
        keep = valid(s["lengths"], length)[..., None]
        dt = torch.where(keep, dt, torch.zeros_like(dt))         # a step of size zero leaves the state as it is
    a = torch.exp(dt[..., None] * A)
    b = (dt * x)[..., None] * B
    b[:, 0] += a[:, 0] * state
    h = recurrence(a, b)
    y = ((h * C).sum(-1) + s["D"] * x) * silu(z)
    if keep is not None:
        y = torch.where(keep, y, torch.zeros_like(y))
    return {"y": y.to(kind), "state": h[:, -1].contiguous()}


def scan_train(s):
    x, z, A, D, dy = s["x"].float(), s["z"].float(), s["A"], s["D"], s["d_y"].float()
    c, kind, groups = x.shape[-1], s["x"].dtype, s["B"].shape[-2]
    raw = s["dt"].float() + s["dt_bias"]
    dt = softplus(raw)
    B, C = per_channel(s["B"], c), per_channel(s["C"], c)
    a = torch.exp(dt[..., None] * A)
    h = recurrence(a, (dt * x)[..., None] * B)
    y = (h * C).sum(-1) + D * x
    out = y * silu(z)
    d_y = dy * silu(z)
    d_z = dy * y * silu_slope(z)
    # the adjoint of the state runs the same recurrence from the last step to the first
    after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
    g = recurrence(after.flip(1), (d_y[..., None] * C).flip(1)).flip(1)
    of_group = lambda t: t.unflatten(2, (groups, c // groups)).sum(3)  # noqa: E731
    d_C = of_group(d_y[..., None] * h)
    d_B = of_group(g * (dt * x)[..., None])
    d_u = (g * B).sum(-1)
    before = torch.cat([torch.zeros_like(h[:, :1]), h[:, :-1]], 1)
    w = g * a * before
    d_dt = (w * A).sum(-1) + d_u * x
    d_raw = d_dt / (1.0 + torch.exp(-raw))
    return {"y": out.to(kind), "d_x": (d_u * dt + d_y * D).to(kind), "d_dt": d_raw.to(kind), "d_z": d_z.to(kind),
            "d_B": d_B.to(kind), "d_C": d_C.to(kind), "d_A": (w * dt[..., None]).sum((0, 1)), "d_D": (d_y * x).sum((0, 1)),
            "d_dt_bias": d_raw.sum((0, 1))}


def norm_plain(s):
    x, kind = s["x"].float(), s["x"].dtype
    u = x * silu(s["gate"].float()) if "gate" in s else x
    inv_u = torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
    p = u * inv_u * s["post_weight"] if "post_weight" in s else u
    out = {}
    if "residual" in s:
        r = s["residual"].float() + s["scale"] * p
        inv_r = torch.rsqrt((r * r).mean(-1, keepdim=True) + EPS)
        out["r"], out["n"] = r.to(kind), (r * inv_r * s["pre_weight"]).to(kind)
    else:
        out["p"] = p.to(kind)
    if "d_first" not in s:
        return out
    d_p = s["d_first"].float()
    if "residual" in s:
        d_n = s["d_second"].float()
        out["d_pre_weight"] = (d_n * r * inv_r).sum(0)
        g = d_n * s["pre_weight"]
        d_r = d_p + inv_r * (g - r * inv_r * inv_r * (g * r).mean(-1, keepdim=True))
        out["d_residual"] = d_r.to(kind)
        out["d_scale"] = (d_r * p).sum(0)
        d_p = d_r * s["scale"]
    d_u = d_p
    if "post_weight" in s:
        out["d_post_weight"] = (d_p * u * inv_u).sum(0)
        g = d_p * s["post_weight"]
        d_u = inv_u * (g - u * inv_u * inv_u * (g * u).mean(-1, keepdim=True))
    if "gate" in s:
        z = s["gate"].float()
        out["d_gate"] = (d_u * x * silu_slope(z)).to(kind)
        d_u = d_u * silu(z)
    out["d_x"] = d_u.to(kind)
    return out


# ---------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------------------------------------------------
def leaves_of(s, names):
    return {k: s[k].detach().requires_grad_() for k in names if k in s}


def own_conv(s):
    from unet_amd import ssm
    mode = s["case"]["mode"]
    if mode == "token":
        y = ssm.causal_conv_step(s["x"], s["state"], s["weight"], s["bias"], slots=s["slots"])
        return {"y": y, "state": s["state"]}
    if mode == "prompt":
        y, state = ssm.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s.get("lengths"), return_state=True)
        return {"y": y, "state": state}
    p = leaves_of(s, ("x", "weight", "bias"))
    y = ssm.causal_conv(p["x"], p["weight"], p["bias"])
    grads = torch.autograd.grad(y, list(p.values()), s["d_y"])
    return {"y": y, **{"d_" + k: g for k, g in zip(p, grads)}}


def own_scan(s):
    from unet_amd import ssm
    mode = s["case"]["mode"]
    if mode == "token":
        y = ssm.selective_scan_step(s["x"], s["dt"], s["A"], s["B"], s["C"], s["state"], D=s["D"], z=s["z"],
                                    dt_bias=s["dt_bias"], slots=s["slots"])
        return {"y": y, "state": s["state"]}
    if mode == "prompt":
        y, state = ssm.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["D"], z=s["z"], dt_bias=s["dt_bias"],
                                      state=s["state"], lengths=s.get("lengths"), return_state=True)
        return {"y": y, "state": state}
    p = leaves_of(s, ("x", "dt", "z", "B", "C", "A", "D", "dt_bias"))
    y = ssm.selective_scan(p["x"], p["dt"], p["A"], p["B"], p["C"], D=p["D"], z=p["z"], dt_bias=p["dt_bias"])
    grads = torch.autograd.grad(y, list(p.values()), s["d_y"])
    return {"y": y, **{"d_" + k: g for k, g in zip(p, grads)}}


def own_norm(s):
    from unet_amd import norm
    names = ("x", "gate", "post_weight", "residual", "scale", "pre_weight")
    if "d_first" not in s:
        out = norm.block_norm(**{k: s[k] for k in names if k in s}, eps=EPS)
        return {"r": out[0], "n": out[1]} if "residual" in s else {"p": out}
    p = leaves_of(s, names)
    out = norm.block_norm(**p, eps=EPS)
    if "residual" in s:
        grads = torch.autograd.grad(out, list(p.values()), (s["d_first"], s["d_second"]))
        out = {"r": out[0], "n": out[1]}
    else:
        grads = torch.autograd.grad(out, list(p.values()), s["d_first"])
        out = {"p": out}
    return {**out, **{"d_" + k: g for k, g in zip(p, grads)}}


def run(state):
    op = state["case"]["op"]
    if own:
        return {"conv": own_conv, "scan": own_scan, "norm": own_norm}[op](state)
    with torch.no_grad():
        if op == "norm":
            return norm_plain(state)
        if op == "conv":
            return conv_train(state) if state["case"]["mode"] == "train" else conv_infer(state)
        return scan_train(state) if state["case"]["mode"] == "train" else scan_infer(state)


# ---------------------------------------------------------------------------------------------------------------------
# the bytes and operations of one pass
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    e = DTYPES[case["dtype"]].itemsize
    c = case["channels"]
    if case["op"] == "norm":
        full, cells = case["form"] in ("residual", "full"), case["rows"] * c
        inputs = 1 + (case["form"] in ("gate", "full")) + full
        outputs = 2 if full else 1
        params = 4 * c * ((case["form"] != "residual") + 2 * full)
        passes = {"bytes": cells * e * (inputs + outputs) + params, "flops": cells * 16}
        if case["mode"] == "train":         # the inputs once, the outputs, their gradients in, the inputs' gradients out
            passes = {"bytes": cells * e * (2 * inputs + 2 * outputs) + 2 * params, "flops": cells * 60}
        return passes
    steps = case["batch"] * case.get("length", 1)
    cells = steps * c
    if case["op"] == "conv":
        k = case["taps"]
        states = 0 if case["mode"] == "train" else 2 * case["batch"] * (k - 1) * c * e
        if case["mode"] == "train":
            return {"bytes": cells * e * 4 + 8 * c * (k + 1), "flops": cells * (6 * k + 20)}
        return {"bytes": cells * e * 2 + states + 4 * c * (k + 1), "flops": cells * (2 * k + 6)}
    n, g = case["state"], case["groups"]
    params = 4 * c * (n + 2)
    shared = steps * 2 * g * n * e
    if case["mode"] == "train":             # x, dt, z, the gradient of y in; y and three gradients out
        return {"bytes": cells * e * 8 + 2 * shared + 2 * params, "flops": cells * (n * 24 + 40)}
    return {"bytes": cells * e * 4 + shared + params + 2 * case["batch"] * c * n * 4, "flops": cells * (n * 7 + 20)}


# ---------------------------------------------------------------------------------------------------------------------
# the exact values: 64 bits, one step of time after the other
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    wide = {k: v.double() if torch.is_tensor(v) and v.is_floating_point() else v for k, v in s.items()}
    return {"conv": exact_conv, "scan": exact_scan, "norm": exact_norm}[case["op"]](case, wide)


def exact_conv(case, s):
    w, bias, k = s["weight"], s["bias"], case["taps"]
    if case["mode"] == "token":
        rows = s["slots"].long()
        seen = torch.cat([s["state"][rows], s["x"].unsqueeze(1)], dim=1)
        pre = torch.einsum("bkc,ck->bc", seen, w) + bias
        state = s["state"].clone()
        state[rows] = seen[:, 1:]
        return {"y": pre * torch.sigmoid(pre), "state": state}
    x = s["x"]
    batch, length, c = x.shape
    if case["mode"] == "prompt":
        ends = s["lengths"].tolist() if "lengths" in s else [length] * batch
        y, state = torch.zeros_like(x), torch.empty_like(s["state"])
        for b in range(batch):
            seen = torch.cat([s["state"][b], x[b, :ends[b]]], dim=0)
            state[b] = seen[ends[b]:]
            if ends[b]:
                pre = torch.conv1d(seen.t()[None], w[:, None], bias, groups=c)[0].t()
                y[b, :ends[b]] = pre * torch.sigmoid(pre)
        return {"y": y, "state": state}
    zero = x.new_zeros(batch, c)
    window = [zero] * k
    d_w, d_b = torch.zeros_like(w), torch.zeros_like(bias)
    y, d_x = torch.empty_like(x), x.new_zeros(batch, length + k, c)
    for t in range(length):
        window = window[1:] + [x[:, t]]
        pre = bias.expand(batch, c)
        for j in range(k):
            pre = pre + window[j] * w[:, j]
        sig = torch.sigmoid(pre)
        y[:, t] = pre * sig
        d = s["d_y"][:, t] * (sig + pre * sig * (1 - sig))
        d_b += d.sum(0)
        for j in range(k):
            d_w[:, j] += (d * window[j]).sum(0)
            if t - (k - 1) + j >= 0:
                d_x[:, t - (k - 1) + j] += d * w[:, j]
    return {"y": y, "d_x": d_x[:, :length], "d_weight": d_w, "d_bias": d_b}


def exact_scan(case, s):
    A, D = s["A"], s["D"]
    c, n, g = case["channels"], case["state"], case["groups"]
    step = torch.nn.functional.softplus(s["dt"] + s["dt_bias"], threshold=700.0)
    gate = s["z"] * torch.sigmoid(s["z"])
    group_of = torch.arange(c, device=A.device) // (c // g)
    if case["mode"] == "token":
        rows = s["slots"].long()
        h = s["state"][rows]
        h = torch.exp(step[:, :, None] * A) * h + (step * s["x"])[:, :, None] * s["B"][:, group_of]
        y = torch.einsum("bcn,bcn->bc", h, s["C"][:, group_of]) + D * s["x"]
        state = s["state"].clone()
        state[rows] = h
        return {"y": y * gate, "state": state}
    batch, length = case["batch"], case["length"]
    x = s["x"]
    h = x.new_zeros(batch, c, n) if case["mode"] == "train" else s["state"].clone()
    bare = torch.empty(batch, length, c, dtype=torch.float64, device=x.device)
    keep = []
    ends = s["lengths"] if "lengths" in s else None
    for t in range(length):
        new = torch.exp(step[:, t, :, None] * A) * h + (step[:, t] * x[:, t])[:, :, None] * s["B"][:, t, group_of]
        if ends is not None:
            new = torch.where((ends > t)[:, None, None], new, h)
        h = new
        bare[:, t] = (h * s["C"][:, t, group_of]).sum(-1) + D * x[:, t]
        if case["mode"] == "train":
            keep.append(h)
    y = bare * gate
    if case["mode"] == "prompt":
        if ends is not None:
            y[torch.arange(length, device=x.device)[None] >= ends[:, None]] = 0
        return {"y": y, "state": h}
    sig = torch.sigmoid(s["z"])
    d_z = s["d_y"] * bare * sig * (1 + s["z"] * (1 - sig))
    d_bare = s["d_y"] * gate
    d_x, d_step = D * d_bare, torch.zeros_like(bare)
    d_B, d_C = torch.zeros_like(s["B"]), torch.zeros_like(s["C"])
    d_A = torch.zeros_like(A)
    adjoint = torch.zeros_like(h)
    for t in range(length - 1, -1, -1):
        adjoint = adjoint + d_bare[:, t, :, None] * s["C"][:, t, group_of]
        d_C[:, t] = (d_bare[:, t, :, None] * keep[t]).reshape(batch, g, c // g, n).sum(2)
        d_B[:, t] = (adjoint * (step[:, t] * x[:, t])[:, :, None]).reshape(batch, g, c // g, n).sum(2)
        d_u = (adjoint * s["B"][:, t, group_of]).sum(-1)
        decay = torch.exp(step[:, t, :, None] * A)
        flow = adjoint * decay * (keep[t - 1] if t else 0)
        d_step[:, t] = (flow * A).sum(-1) + d_u * x[:, t]
        d_x[:, t] += d_u * step[:, t]
        d_A += (flow * step[:, t, :, None]).sum(0)
        adjoint = adjoint * decay
    d_dt = d_step * torch.sigmoid(s["dt"] + s["dt_bias"])
    return {"y": y, "d_x": d_x, "d_dt": d_dt, "d_z": d_z, "d_B": d_B, "d_C": d_C, "d_A": d_A, "d_D": (d_bare * x).sum((0, 1)),
            "d_dt_bias": d_dt.sum((0, 1))}


def exact_norm(case, s):
    """The forward values as written, the gradients by automatic differentiation."""
    names = ("x", "gate", "post_weight", "residual", "scale", "pre_weight")
    p = {k: s[k].clone().requires_grad_() for k in names if k in s}

    def rms(v):
        return torch.sqrt(v.pow(2).sum(-1, keepdim=True) / v.shape[-1] + EPS)

    with torch.enable_grad():
        v = p["x"]
        if "gate" in p:
            v = v * (p["gate"] * torch.sigmoid(p["gate"]))
        if "post_weight" in p:
            v = v / rms(v) * p["post_weight"]
        if "residual" in p:
            r = p["residual"] + p["scale"] * v
            values = (r, r / rms(r) * p["pre_weight"])
        else:
            values = (v,)
        grads = ()
        if case["mode"] == "train":
            grads = torch.autograd.grad(values, list(p.values()), tuple(s[k] for k in ("d_first", "d_second") if k in s))
    out = {"r": values[0], "n": values[1]} if len(values) > 1 else {"p": values[0]}
    out.update({"d_" + k: t for k, t in zip(p, grads)})
    return {k: v.detach() for k, v in out.items()}
