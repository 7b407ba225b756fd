"""The sequence operators (unet_amd.ssm: causal convolution and selective scan; unet_amd.norm: block norm) against 64-bit
restatements (seq_oracle.py), element by element, within what the fp32 roundings of the computation and the output's type
leave.  Rounding counts: a state after m steps has taken two roundings a step and its decays' errors (each at most a few
2^-24 of values whose sum of exponents bounds them), a sum over n terms at most n; hardware exponentials, reciprocals and
the softplus series add a few tens."""

import gc

import pytest
import torch

from seq_oracle import conv64, held, norm64, scan64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def rnd(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def dev(t, device):
    return None if t is None else t.to(device)


def sliced(t, device, pad=8):
    """``t`` as a slice of a wider tensor whose other elements are NaN: rows are strided, reading past one shows."""
    wide = torch.full(t.shape[:-1] + (t.shape[-1] + pad,), float("nan"), dtype=t.dtype, device=device)
    wide[..., :t.shape[-1]] = t.to(device)
    return wide[..., :t.shape[-1]]


# ---------------------------------------------------------------------------------------------------------------------
# causal convolution
# ---------------------------------------------------------------------------------------------------------------------
CONV = [
    # batch, length, channels, taps, silu, bias, state, lengths
    (1, 1, 1, 2, True, True, False, None),
    (2, 1, 8, 4, True, True, True, None),
    (3, 2, 40, 4, True, False, True, [2, 0, 1]),
    (2, 37, 72, 3, False, True, False, None),
    (4, 129, 512, 4, True, True, True, [129, 1, 0, 67]),
    (2, 500, 37, 2, True, True, True, None),
    (1, 1030, 520, 4, True, True, False, None),
    (3, 5, 1288, 3, True, True, True, [5, 2, 9]),
]


def conv_inputs(B, L, D, K, bias, state, lengths, dtype):
    return (rnd((B, L, D), 1, dtype), rnd((D, K), 2), rnd((D,), 3) if bias else None, rnd((B, K - 1, D), 4, dtype) if state else None,
            None if lengths is None else torch.tensor(lengths, dtype=torch.int32), rnd((B, L, D), 5, dtype), rnd((B, K - 1, D), 6, dtype))


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,D,K,silu,bias,state,lengths", CONV)
def test_causal_conv(device, B, L, D, K, silu, bias, state, lengths, dtype):
    from unet_amd import ssm
    x, w, b, s, n, dy, ds = conv_inputs(B, L, D, K, bias, state, lengths, dtype)
    want = conv64(x, w, b, s, n, silu, dy, ds)
    room = conv64(x, w, b, s, n, silu, dy, ds, magnitude=True)
    for strided in (False, True):
        put = (lambda t: sliced(t, device)) if strided else (lambda t: t.to(device))
        leaves = [None if t is None else t.requires_grad_() for t in (put(x), dev(w, device), dev(b, device), dev(s, device))]
        y, out = ssm.causal_conv(leaves[0], leaves[1], leaves[2], act=silu, state=leaves[3], lengths=dev(n, device), return_state=True)
        held(y, want["y"], room["y"], 16, "y")
        assert torch.equal(out.cpu().double(), want["state"])
        given = [t for t in leaves if t is not None]
        grads = iter(torch.autograd.grad((y, out), given, (put(dy), dev(ds, device))))
        count = 24 + B * L
        held(next(grads), want["dx"], room["dx"], 24, "dx")
        held(next(grads), want["dw"], room["dw"], count, "dw")
        if bias:
            held(next(grads), want["db"], room["db"], count, "db")
        if state:
            held(next(grads), want["dstate"], room["dstate"], 24, "dstate")
        with torch.no_grad():
            assert torch.equal(ssm.causal_conv(put(x), dev(w, device), dev(b, device), act=silu, state=dev(s, device),
                                               lengths=dev(n, device)), y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,slots_n,D,K", [(1, 1, 8, 4), (5, 9, 37, 3), (300, 333, 264, 2), (4, 6, 2056, 4)])
def test_causal_conv_step_continues_a_prompt(device, rows, slots_n, D, K, dtype):
    """A prompt, then single tokens on its state: the same numbers as the whole sequence at once; padding rows, slots out of
    range and slots used twice touch nothing."""
    from unet_amd import ssm
    L, extra = 7, 3
    x = rnd((rows, L + extra, D), 1, dtype)
    w, b = rnd((D, K), 2), rnd((D,), 3)
    want = conv64(x, w, b, None, None, True)
    room = conv64(x, w, b, None, None, True, magnitude=True)
    xd, wd, bd = x.to(device), w.to(device), b.to(device)
    _, state = ssm.causal_conv(xd[:, :L], wd, bd, return_state=True)
    cache = rnd((slots_n, K - 1, D), 9, dtype).to(device)
    slots = torch.randperm(slots_n, generator=torch.Generator().manual_seed(3))[:rows].to(device)
    cache[slots] = state
    before = cache.clone()
    for t in range(L, L + extra):
        y = ssm.causal_conv_step(xd[:, t], cache, wd, bd, slots=slots if t % 2 else slots.int())
        held(y, want["y"][:, t], room["y"][:, t], 16, "token {}".format(t))
    others = [i for i in range(slots_n) if i not in slots.tolist()]
    assert torch.equal(cache[others], before[others])
    assert torch.equal(cache[slots], xd[:, L + extra - (K - 1):].contiguous() if K > 1 else cache[slots])
    if rows >= 4:
        odd = slots.clone()
        odd[0], odd[2], odd[3] = -1, slots[1], slots_n
        before = cache.clone()
        y = ssm.causal_conv_step(xd[:, 0], cache, wd, bd, slots=odd)
        assert (y[0] == 0).all() and y[2].isnan().all() and y[3].isnan().all() and y[1].isfinite().all()
        assert torch.equal(cache[slots[[0, 2, 3]]], before[slots[[0, 2, 3]]])
        assert not torch.equal(cache[slots[1]], before[slots[1]])


def test_causal_conv_ignores_what_lies_behind_the_end(device):
    """NaN and infinities behind the sequences' ends, in the inputs and in the output's gradient, reach nothing."""
    from unet_amd import ssm
    x, w, b, s, n, dy, ds = conv_inputs(4, 50, 72, 4, True, True, [50, 0, 2, 33], F32)
    want, room = conv64(x, w, b, s, n, True, dy, ds), conv64(x, w, b, s, n, True, dy, ds, magnitude=True)
    for i, k in enumerate(n.tolist()):
        x[i, k:], dy[i, k:] = float("nan"), float("inf")
    leaves = [t.to(device).requires_grad_() for t in (x, w, b, s)]
    for lengths in (n, n.long() + torch.tensor([2 ** 40, -(2 ** 40), 0, 0]), n.to(torch.int16)):
        y, out = ssm.causal_conv(leaves[0], leaves[1], leaves[2], state=leaves[3], lengths=lengths.to(device), return_state=True)
        grads = torch.autograd.grad((y, out), leaves, (dy.to(device), ds.to(device)))
        held(y, want["y"], room["y"], 16, "y")
        for g, k, count in zip(grads, ("dx", "dw", "db", "dstate"), (24, 224, 224, 24)):
            held(g, want[k], room[k], count, k)


# ---------------------------------------------------------------------------------------------------------------------
# selective scan
# ---------------------------------------------------------------------------------------------------------------------
SCAN = [
    # batch, length, channels, N, groups, D, z, bias, softplus, state, lengths
    (1, 1, 1, 1, 1, True, True, True, True, True, None),
    (2, 1, 64, 16, 1, True, True, True, True, False, None),
    (2, 3, 70, 4, 1, False, False, False, False, True, None),
    (3, 16, 64, 16, 1, True, True, True, True, True, [16, 0, 7]),
    (2, 17, 130, 7, 2, True, False, True, True, True, None),
    (2, 50, 96, 8, 3, False, True, False, True, False, [50, 33]),
    (1, 70, 200, 12, 1, True, True, True, False, True, None),
    (2, 129, 64, 16, 1, True, True, True, True, True, [129, 64]),
    (4, 100, 48, 24, 2, True, True, True, True, True, [1, 100, 15, 99]),
    (1, 65, 64, 64, 1, True, True, True, True, True, None),
    (2, 30, 40, 33, 1, True, True, True, True, False, [30, 29]),
    (1, 700, 64, 16, 1, True, True, True, True, True, [611]),
]


def scan_inputs(B, L, ch, N, G, D, z, bias, state, lengths, dtype, softplus):
    g = torch.Generator().manual_seed(77)
    x, dt = rnd((B, L, ch), 1, dtype), rnd((B, L, ch), 2, dtype, 0.7)
    if not softplus:
        dt = (dt.float().abs() * 0.3).to(dtype)
    p = dict(x=x, dt=dt, A=-torch.arange(1.0, N + 1) * (torch.rand((ch, N), generator=g) + 0.5),
             B=rnd((B, L, G, N), 3, dtype), C=rnd((B, L, G, N), 4, dtype),
             D=rnd((ch,), 5) if D else None, z=rnd((B, L, ch), 6, dtype) if z else None,
             dt_bias=(torch.rand((ch,), generator=g) * 4 - (5 if softplus else 0)).abs() * (-1 if softplus else 0.05) if bias else None,
             state=rnd((B, ch, N), 8) if state else None)
    n = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    return p, n, rnd((B, L, ch), 9, dtype), rnd((B, ch, N), 10)


def scan_case(device, dtype, B, L, ch, N, G, D, z, bias, softplus, state, lengths, strided):
    from unet_amd import ssm
    p, n, dy, ds = scan_inputs(B, L, ch, N, G, D, z, bias, state, lengths, dtype, softplus)
    want = scan64(**p, softplus=softplus, lengths=n, dy=dy, dout=ds)
    room = scan64(**p, softplus=softplus, lengths=n, dy=dy, dout=ds, magnitude=True)
    put = (lambda t: sliced(t, device)) if strided else (lambda t: t.to(device))
    leaves = {k: (put(t) if k in ("x", "dt", "z", "B", "C") else t.to(device)).requires_grad_() for k, t in p.items() if t is not None}
    nd = dev(n, device)
    if n is not None:                       # what lies behind a sequence's end is not used
        with torch.no_grad():
            for b in range(B):
                for k in ("x", "dt", "z", "B", "C"):
                    if k in leaves:
                        leaves[k][b, int(n[b]):] = float("nan")
    given = {"D": None, "z": None, "dt_bias": None, "state": None, **leaves}
    y, out = ssm.selective_scan(**given, softplus=softplus, lengths=nd, return_state=True)
    chain = 2 * L + N + 64
    held(y, want["y"], room["y"], chain, "y")
    held(out, want["state"], room["state"], chain, "state")
    grads = torch.autograd.grad((y, out), list(leaves.values()), (put(dy), dev(ds, device)))
    for k, g in zip(leaves, grads):
        steps = 4 * L + 2 * N + 96 + (ch if k in "BC" else 0) + (B * L if k in ("A", "D", "dt_bias") else 0)
        held(g, want["d_" + k], room["d_" + k], steps, "d " + k)
    with torch.no_grad():
        again = ssm.selective_scan(**given, softplus=softplus, lengths=nd)
        assert torch.equal(again, y)
    return grads


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("B,L,ch,N,G,D,z,bias,softplus,state,lengths", SCAN)
def test_selective_scan(device, B, L, ch, N, G, D, z, bias, softplus, state, lengths, dtype):
    for strided in (False, True):
        scan_case(device, dtype, B, L, ch, N, G, D, z, bias, softplus, state, lengths, strided)


def test_selective_scan_gradients_repeat_bit_for_bit(device):
    """No atomics: equal calls give equal bits, the sums over channels, steps and sequences among them."""
    a = scan_case(device, BF16, 3, 200, 192, 16, 1, True, True, True, True, True, [200, 77, 150], False)
    b = scan_case(device, BF16, 3, 200, 192, 16, 1, True, True, True, True, True, [200, 77, 150], False)
    assert all(torch.equal(u, v) for u, v in zip(a, b))


def test_selective_scan_gradient_is_the_slope_of_the_scan(device):
    """The device's gradients against central differences of the 64-bit scan along one direction in all inputs at once:
    the difference quotient of a smooth function is off by O(h^2) (h = 1e-4: 1e-8 of the third derivatives, which the unit
    inputs keep below 1e2), the device's gradients by their fp32 roundings, both far below 1e-3 of the slope's magnitude."""
    from unet_amd import ssm
    p, n, dy, ds = scan_inputs(2, 40, 64, 16, 1, True, True, True, True, [40, 23], F32, True)
    leaves = {k: t.to(device).requires_grad_() for k, t in p.items()}
    y, out = ssm.selective_scan(**leaves, lengths=n.to(device), return_state=True)
    grads = torch.autograd.grad((y, out), list(leaves.values()), (dy.to(device), ds.to(device)))
    way = {k: rnd(t.shape, 40 + i).double() for i, (k, t) in enumerate(p.items())}
    slope = sum((g.cpu().double() * way[k]).sum() for k, g in zip(leaves, grads))
    size = sum((g.cpu().double() * way[k]).pow(2).sum() for k, g in zip(leaves, grads)).sqrt()

    def value(h):
        r = scan64(**{k: t.double() + h * way[k] for k, t in p.items()}, lengths=n)
        return (r["y"] * dy.double()).sum() + (r["state"] * ds.double()).sum()

    quotient = (value(1e-4) - value(-1e-4)) / 2e-4
    assert abs(slope - quotient) <= 1e-3 * size, (slope, quotient, size)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,slots_n,ch,N,G,D,z,bias", [(1, 1, 64, 16, 1, True, True, True), (5, 7, 70, 5, 2, False, False, False),
                                                          (270, 300, 40, 16, 1, True, True, True), (4, 5, 1280, 64, 4, True, True, True)])
def test_selective_scan_step_continues_a_prompt(device, rows, slots_n, ch, N, G, D, z, bias, dtype):
    from unet_amd import ssm
    L, extra = 5, 3
    p, _, _, _ = scan_inputs(rows, L + extra, ch, N, G, D, z, bias, False, None, dtype, True)
    want, room = scan64(**p), scan64(**p, magnitude=True)
    q = {k: dev(t, device) for k, t in p.items() if k != "state"}
    seq = ("x", "dt", "B", "C", "z")
    part = lambda t0, t1: {k: (v[:, t0:t1] if k in seq and v is not None else v) for k, v in q.items()}  # noqa: E731
    y, state = ssm.selective_scan(**part(0, L), return_state=True)
    cache = rnd((slots_n, ch, N), 9).to(device)
    slots = torch.randperm(slots_n, generator=torch.Generator().manual_seed(3))[:rows].to(device)
    cache[slots] = state
    before = cache.clone()
    for t in range(L, L + extra):
        token = {k: (v[:, t] if k in seq and v is not None else v) for k, v in q.items()}
        y = ssm.selective_scan_step(**token, state=cache, slots=slots if t % 2 else slots.int())
        held(y, want["y"][:, t], room["y"][:, t], 2 * (L + extra) + N + 64, "token {}".format(t))
    held(cache[slots], want["state"], room["state"], 2 * (L + extra) + N + 64, "state")
    others = [i for i in range(slots_n) if i not in slots.tolist()]
    assert torch.equal(cache[others], before[others])
    if rows >= 4:
        odd = slots.clone()
        odd[0], odd[2], odd[3] = -7, slots[1], slots_n
        before = cache.clone()
        y = ssm.selective_scan_step(**token, state=cache, slots=odd)
        assert (y[0] == 0).all() and y[2].isnan().all() and y[3].isnan().all() and y[1].isfinite().all()
        assert torch.equal(cache[slots[[0, 2, 3]]], before[slots[[0, 2, 3]]])
        assert not torch.equal(cache[slots[1]], before[slots[1]])


def test_selective_scan_prompt_in_pieces(device):
    """A prompt taken in pieces of odd lengths, each from the state of the one before, is the prompt at once."""
    from unet_amd import ssm
    p, _, _, _ = scan_inputs(2, 300, 128, 16, 1, True, True, True, True, None, F32, True)
    q = {k: dev(t, device) for k, t in p.items()}
    whole, end = ssm.selective_scan(**q, return_state=True)
    room = scan64(**p, magnitude=True)
    state, at = q["state"], 0
    for n in (1, 97, 16, 186):
        piece = {k: (v[:, at:at + n] if k in ("x", "dt", "B", "C", "z") else v) for k, v in q.items() if k != "state"}
        y, state = ssm.selective_scan(**piece, state=state, return_state=True)
        held(y, whole[:, at:at + n].cpu().double(), room["y"][:, at:at + n], 2 * (2 * 300 + 80), "piece at {}".format(at))
        at += n
    held(state, end.cpu().double(), room["state"], 2 * (2 * 300 + 80), "state")


def test_selective_scan_at_the_ends_of_the_ranges(device):
    """Step sizes from e^-60 to 80 and gates far out on both sides: nothing overflows on the way to a finite value.  The
    softplus of v carries the rounding of v's own exponent, |v| 2^-24 of it, hence the count."""
    from unet_amd import ssm
    p, _, dy, _ = scan_inputs(1, 64, 64, 16, 1, True, True, False, False, None, F32, True)
    p["dt"] = torch.linspace(-60, 80, 64 * 64).view(1, 64, 64)
    p["z"] = torch.linspace(120, -120, 64 * 64).view(1, 64, 64)
    want, room = scan64(**p, dy=dy), scan64(**p, dy=dy, magnitude=True)
    leaves = {k: t.to(device).requires_grad_() for k, t in p.items() if t is not None}
    y = ssm.selective_scan(**leaves)
    held(y, want["y"], room["y"], 2 * 64 + 16 + 64 + 200, "y")
    for k, g in zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy.to(device))):
        held(g, want["d_" + k], room["d_" + k], 4 * 64 + 2 * 16 + 96 + 400 + 64, "d " + k)


@pytest.mark.parametrize("N", [3, 8, 16])
def test_selective_scan_of_a_growing_state_that_starts_late(device, N):
    """A > 0 over a split time axis: a state that is still zero stays zero where the decay of a whole chunk overflows."""
    from unet_amd import ssm
    L, ch = 512, 64
    x, dy = rnd((1, L, ch), 1), rnd((1, L, ch), 2)
    x[:, :-3] = 0
    dy[:, 3:] = 0
    p = dict(x=x, dt=torch.ones(1, L, ch), A=torch.full((ch, N), 2.0), B=rnd((1, L, 1, N), 3), C=rnd((1, L, 1, N), 4))
    q = {k: v.to(device).requires_grad_() for k, v in p.items()}
    y = ssm.selective_scan(**q, softplus=False)
    grads = torch.autograd.grad(y, list(q.values()), dy.to(device))
    want, room = (scan64(**p, softplus=False, dy=dy, magnitude=m) for m in (False, True))
    held(y, want["y"], room["y"], 2 * L + N + 64, "y")
    for k, g in zip(q, grads):
        held(g, want["d_" + k], room["d_" + k], 5 * L + 2 * N + 96 + ch, "d " + k)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("N,L,lengths", [(4, 330, [330, 0, 223]), (8, 289, None), (5, 1000, [1000, 511, 65])])
def test_selective_scan_of_few_states_in_chunks(device, N, L, lengths, dtype):
    scan_case(device, dtype, 3, L, 72, N, 1, True, True, True, True, True, lengths, False)


def test_more_than_two_to_the_31_elements(device):
    """Sequences, caches and rows whose last elements lie beyond 2^31: the same bits as the last part on its own."""
    from unet_amd import norm, ssm
    ch, L, tail = 131072, 16416, 32
    gen = torch.Generator(device=device).manual_seed(5)
    x = torch.randn((1, L, ch), generator=gen, device=device, dtype=BF16)
    w = torch.randn((ch, 4), generator=gen, device=device)
    y, end = ssm.causal_conv(x, w, return_state=True)
    _, before = ssm.causal_conv(x[:, :L - tail], w, return_state=True)
    y1, end1 = ssm.causal_conv(x[:, L - tail:], w, state=before, return_state=True)
    assert torch.equal(y[:, L - tail:], y1) and torch.equal(end, end1)
    del y, y1
    A = -torch.rand((ch, 4), generator=gen, device=device) - 0.5
    B, C = (torch.randn((1, L, 4), generator=gen, device=device, dtype=BF16) for _ in range(2))
    y, end = ssm.selective_scan(x, x, A, B, C, return_state=True)
    _, before = ssm.selective_scan(x[:, :L - tail], x[:, :L - tail], A, B[:, :L - tail], C[:, :L - tail], return_state=True)
    y1, end1 = ssm.selective_scan(x[:, L - tail:], x[:, L - tail:], A, B[:, L - tail:], C[:, L - tail:], state=before, return_state=True)
    assert torch.equal(y[:, L - tail:], y1) and torch.equal(end, end1)
    del y, y1
    rows = x.view(-1, 8192)
    pre = torch.rand((8192,), generator=gen, device=device)
    r, n = norm.block_norm(rows, residual=rows, pre_weight=pre)
    r1, n1 = norm.block_norm(rows[-7:], residual=rows[-7:], pre_weight=pre)
    assert torch.equal(r[-7:], r1) and torch.equal(n[-7:], n1)
    del r, n, rows
    cache = torch.zeros((4100, ch, 4), device=device)                  # 2.1e9 states
    slots = torch.tensor([4099, 0], device=device)
    token = x[0, :2]
    y = ssm.selective_scan_step(token, token, A, B[0, :2], C[0, :2], cache, slots=slots)
    small = torch.zeros((2, ch, 4), device=device)
    assert torch.equal(y, ssm.selective_scan_step(token, token, A, B[0, :2], C[0, :2], small))
    assert torch.equal(cache[4099], small[0]) and torch.equal(cache[0], small[1]) and not cache[1:4099].any()


def test_selective_scan_long_and_wide_offsets(device):
    """Element offsets beyond 2^31: a batch of expanded (stride 0) rows and a slice far into a large buffer."""
    from unet_amd import ssm
    ch, N, L = 64, 16, 24
    p, _, _, _ = scan_inputs(1, L, ch, N, 1, True, True, True, False, None, BF16, True)
    q = {k: dev(t, device) for k, t in p.items() if t is not None}
    want = ssm.selective_scan(**q)
    stride = (2 ** 31 + 4096) // (L - 1) // 8 * 8 + 8                    # the last step lies beyond 2^31 elements
    big = torch.empty((stride * (L - 1) + ch,), dtype=BF16, device=device)
    far = big.as_strided((1, L, ch), (0, stride, 1))
    far.copy_(q["x"])
    assert torch.equal(ssm.selective_scan(**{**q, "x": far}), want)
    assert torch.equal(ssm.causal_conv(far, q["A"][:, :4].contiguous()), ssm.causal_conv(q["x"], q["A"][:, :4].contiguous()))
    del big, far
    many = ssm.selective_scan(**{k: (t.expand(3, *t.shape[1:]) if k in ("x", "dt", "B", "C", "z") else t) for k, t in q.items()})
    assert all(torch.equal(many[i:i + 1], want) for i in range(3))


# ---------------------------------------------------------------------------------------------------------------------
# block norm
# ---------------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("xt,rt", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("gate,post,residual,scale,pre", [(1, 1, 0, 0, 0), (0, 1, 0, 0, 0), (1, 0, 0, 0, 0), (0, 0, 1, 0, 1), (0, 0, 1, 1, 1),
                                                          (1, 1, 1, 1, 1), (0, 1, 1, 0, 0), (1, 1, 1, 1, 0)])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 37), (5, 512), (9, 520), (2, 4096), (3, 8192), (700, 72), (2, 5001)])
def test_block_norm(device, rows, D, gate, post, residual, scale, pre, xt, rt):
    from unet_amd import norm
    eps = 1e-5
    t = [rnd((rows, D), 1, xt), rnd((rows, D), 2, xt) if gate else None, rnd((D,), 3) if post else None,
         rnd((rows, D), 4, rt) if residual else None, rnd((D,), 5) if scale else None, rnd((D,), 6) if pre else None]
    d_out, d_n = rnd((rows, D), 7, rt if residual else xt), rnd((rows, D), 8, xt) if pre else None
    names = ("x", "gate", "post_weight", "residual", "scale", "pre_weight")
    for strided in (False, True):
        put = (lambda v: sliced(v, device)) if strided else (lambda v: v.to(device))
        leaves = {k: (put(v) if v.dim() == 2 else v.to(device)).requires_grad_() for k, v in zip(names, t) if v is not None}
        out = norm.block_norm(**leaves, eps=eps)
        out = out if pre else (out,)
        want = norm64(*t, eps, d_out, d_n)
        room = norm64(*t, eps, d_out, d_n, magnitude=True)
        # a mean over a row: 8 terms a thread, 6 exchanges, 16 waves; its root halves the error, then a few products
        held(out[0], want["r" if residual else "p"], room["r" if residual else "p"], 64, "r")
        if pre:
            held(out[1], want["n"], room["n"], 128, "n")
        grads = torch.autograd.grad(out, list(leaves.values()), [put(d) if d.dim() == 2 else d for d in (d_out, d_n) if d is not None])
        for k, g in zip(leaves, grads):
            short = k.replace("_weight", "")
            held(g, want["d_" + short], room["d_" + short], 192 + (rows if g.dim() == 1 else 0), "d " + k)


@pytest.mark.parametrize("size,eps", [(1e14, 1e-6), (1e-14, 0.0)])
def test_block_norm_of_large_and_small_values(device, size, eps):
    """Rows whose squares are far from 1: every part scales with them or does not."""
    from unet_amd import norm
    names = ("x", "gate", "post_weight", "residual", "scale", "pre_weight")
    t = [rnd((6, 200), 1) * size, rnd((6, 200), 2), rnd((200,), 3) * size, rnd((6, 200), 4) * size, rnd((200,), 5), rnd((200,), 6)]
    d_out, d_n = rnd((6, 200), 7) / size, rnd((6, 200), 8)
    leaves = {k: v.to(device).requires_grad_() for k, v in zip(names, t)}
    grads = torch.autograd.grad(norm.block_norm(**leaves, eps=eps), list(leaves.values()), (d_out.to(device), d_n.to(device)))
    want, room = (norm64(*t, eps, d_out, d_n, magnitude=m) for m in (False, True))
    for k, g in zip(leaves, grads):
        short = k.replace("_weight", "")
        held(g, want["d_" + short], room["d_" + short], 192 + (6 if g.dim() == 1 else 0), "d " + k)


@pytest.mark.parametrize("xt,rt", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("rows,D", [(20000, 40), (9000, 520), (2000, 1100), (600, 5001), (520, 8192)])
def test_block_norm_of_many_rows(device, rows, D, xt, rt):
    """More rows than blocks: a block's threads go on to the next row, over one wave and over up to sixteen."""
    test_block_norm(device, rows, D, 1, 1, 1, 1, 1, xt, rt)


def test_block_norm_without_some_gradients_and_with_a_single_scale(device):
    """Only one of the two outputs used; the scale as one value (its gradient the sum over the channels)."""
    from unet_amd import norm
    x, res, w = (rnd((2, 5, 96), 1).to(device).requires_grad_(), rnd((2, 5, 96), 2).to(device).requires_grad_(),
                 rnd((96,), 3).to(device).requires_grad_())
    s = torch.tensor(0.5, device=device, requires_grad=True)
    r, n = norm.block_norm(x, residual=res, scale=s, pre_weight=w)
    assert r.shape == n.shape == x.shape
    gx, gs, gw = torch.autograd.grad(n.sum(), (x, s, w), retain_graph=True)
    full = norm64(x.reshape(-1, 96), None, None, res.reshape(-1, 96), s.expand(96), w, 1e-6, None, torch.ones(10, 96))
    room = norm64(x.reshape(-1, 96), None, None, res.reshape(-1, 96), s.expand(96), w, 1e-6, None, torch.ones(10, 96), magnitude=True)
    held(gx.reshape(-1, 96), full["d_x"], room["d_x"], 192, "d x")
    held(gw, full["d_pre"], room["d_pre"], 202, "d w")
    held(gs.reshape(1), full["d_scale"].sum().reshape(1), room["d_scale"].sum().reshape(1), 300, "d s")
    gr, gx = torch.autograd.grad(r.sum(), (res, x))
    assert torch.equal(gr, torch.ones_like(gr)) and torch.equal(gx, torch.full_like(gx, 0.5))


# ---------------------------------------------------------------------------------------------------------------------
# how programs call them
# ---------------------------------------------------------------------------------------------------------------------
def test_empty_calls(device):
    from unet_amd import norm, ssm
    e = lambda *s: torch.empty(s, device=device)  # noqa: E731
    state = rnd((2, 8, 4), 1).to(device)
    y, s = ssm.selective_scan(e(2, 0, 8), e(2, 0, 8), -torch.ones(8, 4, device=device), e(2, 0, 4), e(2, 0, 4), state=state, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(s, state)
    before = rnd((2, 2, 8), 2).to(device)
    y, s = ssm.causal_conv(e(2, 0, 8), torch.ones(8, 3, device=device), state=before, return_state=True)
    assert y.shape == (2, 0, 8) and torch.equal(s, before)
    assert ssm.selective_scan(e(0, 5, 8), e(0, 5, 8), -torch.ones(8, 4, device=device), e(0, 5, 4), e(0, 5, 4)).shape == (0, 5, 8)
    assert norm.block_norm(e(0, 8), post_weight=torch.ones(8, device=device)).shape == (0, 8)


def test_gradients_of_empty_calls(device):
    """No step or no sequence: parameters get zeros, a state's gradient goes straight through."""
    from unet_amd import norm, ssm
    for B, L in ((2, 0), (0, 5), (0, 0)):
        x = torch.zeros(B, L, 8, device=device, requires_grad=True)
        bc = torch.zeros(B, L, 4, device=device, requires_grad=True)
        A = -torch.ones(8, 4, device=device)
        A.requires_grad_()
        state, before = rnd((B, 8, 4), 1).to(device).requires_grad_(), rnd((B, 2, 8), 2).to(device).requires_grad_()
        w, b = rnd((8, 3), 3).to(device).requires_grad_(), rnd((8,), 4).to(device).requires_grad_()
        ds, dc = rnd((B, 8, 4), 5).to(device), rnd((B, 2, 8), 6).to(device)
        y, s = ssm.selective_scan(x, x, A, bc, bc, D=b, z=x, dt_bias=b, state=state, return_state=True)
        gx, gA, gb, gs = torch.autograd.grad((y, s), (x, A, b, state), (torch.zeros_like(y), ds))
        assert gx.shape == x.shape and torch.equal(gs, ds) and not gA.any() and not gb.any()
        y, s = ssm.causal_conv(x, w, b, state=before, return_state=True)
        gx, gw, gb, gs = torch.autograd.grad((y, s), (x, w, b, before), (torch.zeros_like(y), dc))
        assert gx.shape == x.shape and torch.equal(gs, dc) and not gw.any() and not gb.any()
    x = torch.zeros(0, 8, device=device, requires_grad=True)
    r, n = norm.block_norm(x, gate=x, post_weight=b, residual=x, scale=b, pre_weight=b)
    gx, gb = torch.autograd.grad((r, n), (x, b), (torch.zeros_like(r), torch.zeros_like(n)))
    assert gx.shape == x.shape and not gb.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_inputs_in_other_orders(device, dtype):
    """Channels-first tensors seen through a transpose, inputs broadcast over the batch or the groups, gradients that arrive
    expanded: what the same values give when dense, bit for bit, and a broadcast input's gradient is the sum over its copies."""
    from unet_amd import norm, ssm
    B, L, C, N, G = 3, 45, 48, 5, 4
    A = (-torch.rand((C, N), generator=torch.Generator().manual_seed(1)) - 0.1).to(device)
    w, one = rnd((C, 4), 2).to(device), rnd((C,), 3).to(device)
    x = rnd((B, C, L), 4, dtype).to(device).transpose(1, 2)
    dt = rnd((1, L, C), 5, dtype).to(device).expand(B, L, C)
    bm = rnd((B, L, 1, N), 6, dtype).to(device).expand(B, L, G, N)
    cm = rnd((B, N, L, G), 7, dtype).to(device).permute(0, 2, 3, 1)
    z = rnd((B, L, 1), 8, dtype).to(device).expand(B, L, C)
    dy = rnd((1, 1, C), 9, dtype).to(device).expand(B, L, C)

    def both(call, *tensors):
        out = []
        for dense in (False, True):
            leaves = [(t.contiguous() if dense else t.detach()).requires_grad_() for t in tensors]
            y = call(*leaves)
            out.append([y] + list(torch.autograd.grad(y, leaves, dy.reshape(y.shape) if not dense else dy.contiguous().reshape(y.shape))))
        assert all(torch.equal(a, b) for a, b in zip(*out))

    both(lambda x, dt, bm, cm, z: ssm.selective_scan(x, dt, A, bm, cm, D=one, z=z, dt_bias=one), x, dt, bm, cm, z)
    both(lambda x: ssm.causal_conv(x, w, one), x)
    both(lambda z: ssm.causal_conv(z, w, one), z)
    both(lambda x, z: norm.block_norm(x, gate=z, post_weight=one), x, z)
    both(lambda x, z: norm.block_norm(x, residual=z, pre_weight=one)[1], x, z)
    narrow = rnd((B, L, 1, N), 6, dtype).to(device).requires_grad_()
    wide = narrow.detach().expand(B, L, G, N).contiguous().requires_grad_()
    g, = torch.autograd.grad(ssm.selective_scan(x, dt, A, narrow.expand(B, L, G, N), cm), narrow, dy)
    h, = torch.autograd.grad(ssm.selective_scan(x, dt, A, wide, cm), wide, dy)
    assert torch.equal(g, h.sum(2, keepdim=True))
    # tokens
    state, cache = rnd((B, C, N), 10).to(device), rnd((B, 3, C), 11, dtype).to(device)
    for t in (0, L - 1):
        s, c = state.clone(), cache.clone()
        a = ssm.selective_scan_step(x[:, t], dt[:, t], A, bm[:, t], cm[:, t], state, z=z[:, t])
        b = ssm.selective_scan_step(*(v[:, t].contiguous() for v in (x, dt)), A, bm[:, t].contiguous(), cm[:, t].contiguous(), s, z=z[:, t].contiguous())
        assert torch.equal(a, b) and torch.equal(s, state)
        assert torch.equal(ssm.causal_conv_step(x[:, t], cache, w), ssm.causal_conv_step(x[:, t].contiguous(), c, w)) and torch.equal(c, cache)


def test_inference_mode(device):
    """Caches made inside and outside of inference mode."""
    from unet_amd import norm, ssm
    x = rnd((2, 6, 16), 1).to(device)
    w, A, bc = rnd((16, 4), 2).to(device), -torch.ones(16, 4, device=device), rnd((2, 6, 4), 3).to(device)
    want, state = ssm.selective_scan(x, x, A, bc, bc, return_state=True)
    u, before = ssm.causal_conv(x, w, return_state=True)
    outside = torch.zeros(2, 16, 4, device=device), torch.zeros(2, 3, 16, device=device)
    with torch.inference_mode():
        for s, c in (outside, (torch.zeros(2, 16, 4, device=device), torch.zeros(2, 3, 16, device=device))):
            for t in range(6):
                y = ssm.selective_scan_step(x[:, t], x[:, t], A, bc[:, t], bc[:, t], s)
                v = ssm.causal_conv_step(x[:, t], c, w)
            assert torch.allclose(y, want[:, -1], rtol=1e-4, atol=1e-5) and torch.allclose(s, state, rtol=1e-4, atol=1e-5)
            assert torch.equal(c, before) and torch.allclose(v, u[:, -1], rtol=1e-5, atol=1e-6)
        assert torch.equal(norm.block_norm(x, gate=x), norm.block_norm(x.clone(), gate=x.clone()))


def block(p, x):
    """A state space block as a program has it: norm, projections, conv, scan, gated norm, projection, residual."""
    from unet_amd import norm, ssm
    h = norm.block_norm(x, post_weight=p["norm"])
    xz = h @ p["in"]
    c = p["in"].shape[1] // 2
    u = ssm.causal_conv(xz[..., :c], p["conv_w"], p["conv_b"])
    dbc = u @ p["dbc"]
    n = p["A"].shape[1]
    y = ssm.selective_scan(u, dbc[..., :1] * p["dt_w"], p["A"], dbc[..., 1:1 + n], dbc[..., 1 + n:], D=p["D"], z=xz[..., c:], dt_bias=p["dt_b"])
    r, out = norm.block_norm(y @ p["out"], residual=x, scale=p["scale"], pre_weight=p["norm"])
    return r, out


def block_params(width, device):
    c, n = 2 * width, 16
    return {k: v.to(device).requires_grad_() for k, v in dict(
        norm=rnd((width,), 1) * 0.1 + 1, **{"in": rnd((width, 2 * c), 2, scale=width ** -0.5)}, conv_w=rnd((c, 4), 3, scale=0.5), conv_b=rnd((c,), 4),
        dbc=rnd((c, 1 + 2 * n), 5, scale=c ** -0.5), dt_w=rnd((c,), 6, scale=0.2), dt_b=rnd((c,), 7) - 3,
        A=-torch.arange(1.0, n + 1).expand(c, n).contiguous(), D=rnd((c,), 8), out=rnd((c, width), 9, scale=c ** -0.5), scale=rnd((width,), 10)).items()}


def test_block_gradients_in_a_graph(device):
    """A whole block forward and backward, captured and replayed several times with new inputs and eager work between the
    replays: every replay is the eager result, bit for bit."""
    p = block_params(64, device)
    keys = list(p)
    leaves = [p[k].detach().clone().requires_grad_() for k in keys]

    def step(x, ps):
        r, n = block(dict(zip(keys, ps)), x)
        return (r, n) + torch.autograd.grad((r, n), ps, (torch.ones_like(r), n.detach()))

    x = rnd((2, 150, 64), 20).to(device)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(x, leaves)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(x, leaves)
    for seed in (21, 22, 23):
        x.copy_(rnd((2, 150, 64), seed))
        graph.replay()
        torch.cuda.synchronize()
        kept = [t.clone() for t in got]
        eager = step(x, [p[k] for k in keys])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(kept, eager)), [i for i, (a, b) in enumerate(zip(kept, eager)) if not torch.equal(a, b)]


def test_a_captured_backward_beside_an_eager_graph(device):
    """While an eager graph of the same leaves lives, their gradients belong to the default stream, which a capture cannot
    wait for: the backward pass says so before it is tried.  Once that graph is gone the same capture works."""
    from unet_amd import norm, ssm
    w = rnd((64, 4), 1).to(device).requires_grad_()
    A = (-0.1 - torch.rand(64, 8, generator=torch.Generator().manual_seed(6))).to(device).requires_grad_()
    scale = rnd((64,), 2).to(device).requires_grad_()
    x, dy = rnd((2, 40, 64), 3).to(device), rnd((2, 40, 64), 4).to(device)
    bc = rnd((2, 40, 8), 5).to(device)
    calls = [("causal_conv", lambda: ssm.causal_conv(x, w), w), ("selective_scan", lambda: ssm.selective_scan(x, x, A, bc, bc), A),
             ("block_norm", lambda: norm.block_norm(x, residual=x, scale=scale), scale)]
    for name, call, leaf in calls:
        want, = torch.autograd.grad(call(), leaf, dy)
        alive = call()
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="eager graph on the default stream"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                torch.autograd.grad(call(), leaf, dy)
        torch.cuda.synchronize()
        del alive
        gc.collect()                                                   # the refused graph, which the exception's frames held
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got, = torch.autograd.grad(call(), leaf, dy)
        for _ in range(3):
            got.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want), name


def test_a_captured_backward_past_an_eager_input(device):
    """An input that an eager graph made does not stand in the way where its gradient is not asked for."""
    from unet_amd import ssm
    base = rnd((2, 40, 64), 1).to(device).requires_grad_()
    x = base * 2
    w = rnd((64, 4), 2).to(device).requires_grad_()
    dy = rnd((2, 40, 64), 3).to(device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, = torch.autograd.grad(ssm.causal_conv(x, w), w, dy)
    with pytest.raises(RuntimeError, match="eager graph on the default stream"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(ssm.causal_conv(x, w), x, dy)
    want, = torch.autograd.grad(ssm.causal_conv(x, w.detach().requires_grad_()), x, dy)
    assert torch.isfinite(want).all()
    leaf = w.detach().requires_grad_()
    want, = torch.autograd.grad(ssm.causal_conv(x, leaf), leaf, dy)
    for _ in range(3):
        got.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_tokens_in_a_graph(device):
    """A block's token step captured once and replayed over a growing stream, two graphs in turn on two caches, with eager
    work between: every token is the eager one, bit for bit."""
    from unet_amd import norm, ssm
    p = {k: v.detach() for k, v in block_params(64, device).items()}
    c, n = p["in"].shape[1] // 2, p["A"].shape[1]

    def token(x, conv, state, slots):
        xz = norm.block_norm(x, post_weight=p["norm"]) @ p["in"]
        u = ssm.causal_conv_step(xz[:, :c], conv, p["conv_w"], p["conv_b"], slots=slots)
        dbc = u @ p["dbc"]
        y = ssm.selective_scan_step(u, dbc[:, :1] * p["dt_w"], p["A"], dbc[:, 1:1 + n], dbc[:, 1 + n:], state, D=p["D"], z=xz[:, c:],
                                    dt_bias=p["dt_b"], slots=slots)
        return norm.block_norm(y @ p["out"], residual=x, scale=p["scale"], pre_weight=p["norm"])

    def cache(seed):
        return rnd((9, 3, c), seed).to(device), rnd((9, c, n), seed + 1).to(device)

    slots = torch.tensor([4, 0, -1, 8, 2], dtype=torch.int32, device=device)
    xs = [rnd((5, 64), 60 + i).to(device) for i in range(8)]
    caches, eager = [cache(50), cache(52)], [cache(50), cache(52)]
    x = xs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(x, *cache(54), slots)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for k in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(token(x, *caches[k], slots))
        graphs.append(g)
    for i, new in enumerate(xs):
        k = i % 2
        want = token(new, *eager[k], slots)
        x.copy_(new)
        graphs[k].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[k], want)), i
        assert all(torch.equal(a, b) for a, b in zip(caches[k], eager[k])), i


def test_two_streams_at_once(device):
    """Calls on two streams share nothing."""
    from unet_amd import ssm
    p, _, _, _ = scan_inputs(1, 900, 64, 16, 1, True, True, True, False, None, F32, True)
    q = {k: dev(t, device) for k, t in p.items() if t is not None}
    r = {k: (v * 0.5 if k in ("x", "z") else v) for k, v in q.items()}
    want = ssm.selective_scan(**q), ssm.selective_scan(**r)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(5):
        for s, a, g in zip(streams, (q, r), got):
            with torch.cuda.stream(s):
                g.append(ssm.selective_scan(**a))
    torch.cuda.synchronize()
    assert all(torch.equal(t, w) for g, w in zip(got, want) for t in g)


def test_saved_state_and_a_second_backward(device):
    """The backward pass changes nothing that it saved: the same graph can be run again; a cache written by a step is newer
    than what an earlier call saved of it."""
    from unet_amd import ssm
    p, _, dy, _ = scan_inputs(1, 40, 64, 16, 1, True, True, True, True, None, F32, True)
    q = {k: t.to(device).requires_grad_() for k, t in p.items()}
    y = ssm.selective_scan(**q)
    a = torch.autograd.grad(y, list(q.values()), dy.to(device), retain_graph=True)
    b = torch.autograd.grad(y, list(q.values()), dy.to(device))
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    w = rnd((64, 4), 1).to(device).requires_grad_()
    cache = rnd((1, 3, 64), 2).to(device)
    y = ssm.causal_conv(q["x"].detach(), w, state=cache)
    ssm.causal_conv_step(q["x"].detach()[:, 0], cache, w.detach())
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_gradients_under_create_graph(device):
    """create_graph gives the same gradients; asking for a second derivative says that there is none."""
    from unet_amd import norm, ssm
    x = rnd((1, 20, 64), 1).to(device).requires_grad_()
    w = rnd((64, 4), 2).to(device).requires_grad_()
    bc = rnd((1, 20, 4), 3).to(device)
    for name, call in (("causal_conv", lambda: ssm.causal_conv(x, w)),
                       ("selective_scan", lambda: ssm.selective_scan(x, x, -torch.ones(64, 4, device=device), bc, bc)),
                       ("block_norm", lambda: norm.block_norm(x, gate=x))):
        plain, = torch.autograd.grad(call().sum(), x)
        g, = torch.autograd.grad(call().sum(), x, create_graph=True)
        assert torch.equal(plain, g.detach()) and g.requires_grad
        with pytest.raises(RuntimeError, match=name + " can be differentiated once only"):
            g.sum().backward()


def test_ops_under_dispatcher_checks(device):
    """Schemas (what is written in place), autograd registration, shape inference, and the traced forward and backward with
    symbolic sizes."""
    import unet_amd  # noqa: F401
    B, L, C, N = 2, 40, 64, 8
    r = lambda *s: rnd(s, 1).to(device)  # noqa: E731
    g = lambda *s: r(*s).requires_grad_()  # noqa: E731
    A = -torch.arange(1.0, N + 1).expand(C, N).contiguous().to(device)
    for name, args in (
            ("seq_conv", (g(B, L, C), g(C, 4), g(C), g(B, 3, C), None, True, True)),
            ("seq_conv", (g(B, L, C), g(C, 4), None, None, None, False, False)),
            ("seq_conv_step", (r(B, C), r(C, 4), None, r(B, 3, C), None, True)),
            ("ssm_scan", (g(B, L, C), g(B, L, C), A.clone().requires_grad_(), g(B, L, N), g(B, L, N), g(C), g(B, L, C), g(C), g(B, C, N), None,
                          True, True, False)),
            ("ssm_scan", (g(B, L, C), g(B, L, C), A, g(B, L, 2, N), g(B, L, 2, N), None, None, None, None, None, True, False, False)),
            ("ssm_scan_step", (r(B, C), r(B, C), A, r(B, N), r(B, N), None, None, None, r(B, C, N), None, True)),
            ("block_norm", (g(5, C), g(5, C), g(C), g(5, C), g(C), g(C), 1e-6, False)),
            ("block_norm", (g(5, C), None, g(C), None, None, None, 1e-6, False))):
        torch.library.opcheck(getattr(torch.ops.unetmi, name).default, args)


def test_leaves_that_want_no_gradient(device):
    """Only some inputs want gradients, optional ones among them given and not: each gets its own."""
    from unet_amd import norm, ssm
    p, _, dy, _ = scan_inputs(1, 30, 64, 16, 1, True, True, True, True, None, F32, True)
    q = {k: t.to(device) for k, t in p.items()}
    every = {k: t.clone().requires_grad_() for k, t in q.items()}
    want = dict(zip(every, torch.autograd.grad(ssm.selective_scan(**every), list(every.values()), dy.to(device))))
    for some in (["state"], ["z", "A"], ["C"], ["dt_bias", "state"]):
        args = {k: (t.clone().requires_grad_() if k in some else t) for k, t in q.items()}
        got = torch.autograd.grad(ssm.selective_scan(**args), [args[k] for k in some], dy.to(device))
        assert all(torch.equal(g, want[k]) for k, g in zip(some, got))
    # without D the places of what follows it move up
    args = {k: (t.clone().requires_grad_() if k == "dt_bias" else t) for k, t in q.items() if k not in ("D", "z")}
    g, = torch.autograd.grad(ssm.selective_scan(**args), args["dt_bias"], dy.to(device))
    ref = scan64(**{k: t for k, t in p.items() if k not in ("D", "z")}, dy=dy)
    assert torch.allclose(g.cpu().double(), ref["d_dt_bias"], rtol=1e-3, atol=1e-4)
    s = rnd((1, 3, 64), 5).to(device).requires_grad_()
    w = rnd((64, 4), 2).to(device)
    a, = torch.autograd.grad(ssm.causal_conv(q["x"], w, state=s), s, dy.to(device))
    b = torch.autograd.grad(ssm.causal_conv(q["x"].requires_grad_(), w, torch.zeros(64, device=device).requires_grad_(), state=s), s, dy.to(device))[0]
    assert torch.equal(a, b)
    r = rnd((5, 64), 6).to(device).requires_grad_()
    pre = rnd((64,), 7).to(device).requires_grad_()
    x = rnd((5, 64), 8).to(device)
    gr, gp = torch.autograd.grad(norm.block_norm(x, residual=r, pre_weight=pre)[1].sum(), (r, pre))
    full = norm64(x, None, None, r, None, pre, 1e-6, None, torch.ones(5, 64))
    room = norm64(x, None, None, r, None, pre, 1e-6, None, torch.ones(5, 64), magnitude=True)
    held(gr, full["d_residual"], room["d_residual"], 192, "d residual")
    held(gp, full["d_pre"], room["d_pre"], 200, "d pre_weight")


def test_refusals_on_the_device(device):
    from unet_amd import norm, ssm
    from unet_amd._lib import UnetmiError
    x = torch.zeros(1, 4, 8, device=device)
    bc, A = torch.zeros(1, 4, 2, device=device), -torch.ones(8, 2, device=device)
    with pytest.raises(UnetmiError, match="taps"):
        ssm.causal_conv(x, torch.zeros(8, 5, device=device))
    with pytest.raises(ValueError, match="float32 or bfloat16"):
        ssm.causal_conv(x.half(), torch.zeros(8, 4, device=device))
    with pytest.raises(ValueError, match="weight"):
        ssm.causal_conv(x, torch.zeros(8, 4, device=device, dtype=BF16))
    with pytest.raises(ValueError, match="state"):
        ssm.causal_conv(x, torch.zeros(8, 4, device=device), state=torch.zeros(1, 2, 8, device=device))
    with pytest.raises(ValueError, match="dt must"):
        ssm.selective_scan(x, x.to(BF16), A, bc, bc)
    with pytest.raises(ValueError, match="shape"):
        ssm.selective_scan(x, x, A, bc, bc[..., :1])
    with pytest.raises(UnetmiError, match="64 states"):
        ssm.selective_scan(x, x, -torch.ones(8, 65, device=device), torch.zeros(1, 4, 65, device=device), torch.zeros(1, 4, 65, device=device))
    with pytest.raises(UnetmiError, match="groups"):
        ssm.selective_scan(x, x, A, torch.zeros(1, 4, 3, 2, device=device), torch.zeros(1, 4, 3, 2, device=device))
    with pytest.raises(ValueError, match="lengths"):
        ssm.selective_scan(x, x, A, bc, bc, lengths=torch.ones(2, dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="integer"):
        ssm.selective_scan(x, x, A, bc, bc, lengths=torch.ones(1, device=device))
    with pytest.raises(UnetmiError, match="fewer slots"):
        ssm.selective_scan_step(torch.zeros(3, 8, device=device), torch.zeros(3, 8, device=device), A, torch.zeros(3, 2, device=device),
                                torch.zeros(3, 2, device=device), torch.zeros(2, 8, 2, device=device))
    with pytest.raises(ValueError, match="act is True or False"):
        ssm.causal_conv(x, torch.zeros(8, 4, device=device), act="none")
    with pytest.raises(ValueError, match="contiguous"):
        ssm.causal_conv_step(x[0], torch.zeros(4, 8, 3, device=device).transpose(1, 2), torch.zeros(8, 4, device=device))
    with pytest.raises(ValueError, match="state must"):
        ssm.selective_scan_step(x[0], x[0], A, bc[0], bc[0], torch.zeros(4, 8, 2, device=device, dtype=BF16))
    with pytest.raises(ValueError, match="residual"):
        norm.block_norm(x, pre_weight=torch.ones(8, device=device))
    with pytest.raises(UnetmiError, match="8192"):
        norm.block_norm(torch.zeros(1, 8200, device=device), post_weight=torch.ones(8200, device=device))
    with pytest.raises(ValueError, match="one shape"):
        norm.block_norm(x, gate=x[:, :2])
    with pytest.raises(ValueError, match="too long"):                  # one element each: nothing is allocated
        ssm.causal_conv(x[:, :1, :1].expand(2 ** 32 + 1, 1, 1), torch.zeros(1, 4, device=device))
    long = x[:, :1, :1].expand(1, 2 ** 32 + 1, 1)
    with pytest.raises(ValueError, match="too long"):
        ssm.selective_scan(long, long, A[:1], bc[:, :1].expand(1, 2 ** 32 + 1, 2), bc[:, :1].expand(1, 2 ** 32 + 1, 2))
