"""Calls of the sequence operators that their own tests leave out: long time axes taken in one piece, strides of axes of one
element."""

import pytest
import torch

from seq_oracle import held, scan64

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def rnd(shape, seed, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def test_parameter_gradients_over_a_long_axis(device):
    """384 equal sequences of 65536 equal steps, enough blocks for the time axis to stay whole: what dA, dD and ddt_bias add up
    has one sign, so that a single running sum would be off by up to a rounding a step (thousands here, and to one side).
    Counted: 1024 terms between two partial sums in memory, 96 + 3 + 32 for the partial sums of 64 pieces of 384 sequences
    over 32 groups of rows in eights, and for a term 8 roundings each of a state and of an adjoint that forget half of
    themselves every step, 3 of a decay and a few products."""
    from unet_amd import ssm
    B, L = 384, 65536
    value = dict(x=1.1, dt=0.7, B=0.9, C=1.3, dy=0.7)
    value = {k: torch.tensor(v, dtype=F32).item() for k, v in value.items()}
    A, D, bias = -1.0, 0.5, 0.0
    decay = torch.exp(torch.tensor(value["dt"] * A, dtype=torch.float64)).item()
    state, states = 0.0, []
    for _ in range(L):
        states.append(state)
        state = decay * state + value["dt"] * value["x"] * value["B"]
    ahead, dA, dbias, wide = 0.0, 0.0, 0.0, 0.0
    for before in reversed(states):
        ahead += value["dy"] * value["C"]
        du, ahead = ahead * value["B"], ahead * decay
        w = ahead * before
        dA += w * value["dt"]
        dbias += w * A + du * value["x"]
        wide += abs(w * A) + du * value["x"]
    row = {k: torch.full((1, L, 1), v, device=device).expand(B, L, 1) for k, v in value.items()}
    leaves = [torch.full(s, v, device=device).requires_grad_() for s, v in (((1, 1), A), ((1,), D), ((1,), bias))]
    y = ssm.selective_scan(row["x"], row["dt"], leaves[0], row["B"], row["C"], D=leaves[1], dt_bias=leaves[2], softplus=False)
    got = torch.autograd.grad(y, leaves, row["dy"])
    dD = value["dy"] * value["x"] * L
    for name, g, want, size in zip(("dA", "dD", "ddt_bias"), got, (dA, dD, dbias), (dA, dD, wide)):
        held(g.reshape(1), torch.tensor([want * B], dtype=torch.float64), torch.tensor([size * B], dtype=torch.float64), 1024 + 131 + 45, name)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_parameter_gradients_of_sequences_that_end_in_different_pieces(device, dtype):
    """Lengths around the 1024 steps between two partial sums, on a time axis that is not split (384 blocks); what the scratch
    memory held before does not show."""
    from unet_amd import ssm
    B, L, ch, N = 6, 2500, 64, 3
    lengths = torch.tensor([0, 1, 1023, 1024, 1025, 2500], dtype=torch.int32)
    g = torch.Generator().manual_seed(3)
    p = dict(x=rnd((B, L, ch), 1, dtype), dt=rnd((B, L, ch), 2, dtype, 0.7), A=-torch.arange(1.0, N + 1) * (torch.rand((ch, N), generator=g) + 0.5),
             B=rnd((B, L, ch, N), 3, dtype), C=rnd((B, L, ch, N), 4, dtype), D=rnd((ch,), 5), z=rnd((B, L, ch), 6, dtype), dt_bias=rnd((ch,), 7) - 2)
    dy = rnd((B, L, ch), 9, dtype)
    want, room = (scan64(**p, lengths=lengths, dy=dy, magnitude=m) for m in (False, True))
    leaves = {k: t.to(device).requires_grad_() for k, t in p.items()}
    y = ssm.selective_scan(**leaves, lengths=lengths.to(device))
    torch.full((2 ** 26,), float("nan"), device=device)                 # freed at once: the scratch memory comes from here
    grads = torch.autograd.grad(y, list(leaves.values()), dy.to(device))
    for k, got in zip(leaves, grads):
        held(got, want["d_" + k], room["d_" + k], 4 * L + 2 * N + 96 + (B * L if k in ("A", "D", "dt_bias") else 0), "d " + k)


def test_norm_weight_gradients_over_many_rows(device):
    """2^26 equal rows: a weight's gradient adds up terms of one sign.  Counted: 1024 rows between two partial sums in memory,
    256 + 3 + 32 for the partial sums of 65536 threads' rows over 32 groups of rows in eights, 64 for a term (a mean over a row
    and a few products)."""
    from unet_amd import norm
    rows, D = 2 ** 26, 8
    x = torch.linspace(0.6, 1.7, D, dtype=F32)
    w, dy = torch.linspace(0.9, 1.3, D, dtype=F32), torch.linspace(0.7, 1.9, D, dtype=F32)
    leaf = w.to(device).requires_grad_()
    p = norm.block_norm(x.to(device).expand(rows, D), post_weight=leaf)
    got, = torch.autograd.grad(p, leaf, dy.to(device).expand(rows, D))
    v = x.double() * torch.rsqrt(x.double().pow(2).mean() + 1e-6)
    want = rows * dy.double() * v
    held(got, want, want.abs(), 1024 + 291 + 64, "d post_weight")


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_of_single_entries(device, dtype):
    """An axis of one element may have any stride (a prompt of one step out of a time-major buffer: the whole batch lies between
    two steps): the same as dense inputs, bit for bit."""
    from unet_amd import norm, ssm
    far = 2 ** 25

    def spread(t, axes):
        """The same values with the given strides on axes of one element."""
        strides = list(t.stride())
        for a in axes:
            assert t.shape[a] == 1
            strides[a] = far
        return t.as_strided(t.shape, strides)

    B, C, N = 3, 72, 5
    A = (-torch.rand((C, N), generator=torch.Generator().manual_seed(1)) - 0.1).to(device)
    w = rnd((C, 4), 2).to(device)
    x, dt, z, dy = (rnd((B, 1, C), 3 + i, dtype).to(device) for i in range(4))
    b, c = rnd((B, 1, N), 7, dtype).to(device), rnd((B, 1, 1, N), 8, dtype).to(device)
    grouped = b.view(B, 1, 1, N)

    def scan(move):
        leaves = [move(t, (1,)).detach().requires_grad_() for t in (x, dt, z)] + [move(grouped, (1, 2)).detach().requires_grad_(),
                                                                                 move(c, (1, 2)).detach().requires_grad_()]
        y = ssm.selective_scan(leaves[0], leaves[1], A, leaves[3], leaves[4], z=leaves[2])
        return (y,) + torch.autograd.grad(y, leaves, move(dy, (1,)))

    def conv(move):
        leaf = move(x, (1,)).detach().requires_grad_()
        y = ssm.causal_conv(leaf, w)
        return (y,) + torch.autograd.grad(y, leaf, move(dy, (1,)))

    def tokens(move):
        state, cache = torch.ones(1, C, N, device=device), torch.ones(1, 3, C, device=device, dtype=dtype)
        row = lambda t, axes: move(t[:1, 0], axes)  # noqa: E731
        return (ssm.selective_scan_step(row(x, (0,)), row(dt, (0,)), A, row(b, (0,)), row(b, (0,)), state, z=row(z, (0,))),
                ssm.causal_conv_step(row(x, (0,)), cache, w), state, cache,
                norm.block_norm(row(x, (0,)), gate=row(z, (0,)), residual=row(dy, (0,))))

    for call in (scan, conv, tokens):
        with torch.set_grad_enabled(call is not tokens):
            assert all(torch.equal(a, b) for a, b in zip(call(lambda t, axes: t), call(spread))), call.__name__
