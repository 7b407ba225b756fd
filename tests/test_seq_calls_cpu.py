"""How the sequence operators answer automatic differentiation's questions, without a GPU: plain torch stands in for the
kernels on CPU tensors, everything above them (checks, autograd nodes, refusals) is the package's own."""

import os
import subprocess
import sys

import pytest
import torch
from torch.autograd import forward_ad

F32 = torch.float32


def conv(x, weight, bias, state, lengths, silu, want_state):
    return x * weight[:, 0], x.new_zeros((x.shape[0], weight.shape[1] - 1, x.shape[2]) if want_state else (0,))


def conv_bwd(x, weight, bias, state, lengths, silu, dy, dstate_out):
    return dy * weight[:, 0], torch.zeros_like(weight), weight.new_zeros((x.shape[2],)), x.new_zeros((0,) if state is None else state.shape)


def conv_step(x, weight, bias, state, slots, silu):
    with torch.no_grad():
        state += 1
    return x * weight[:, 0]


def scan(x, dt, A, B, C, D, z, dt_bias, state, lengths, softplus, want_state, want_marks):
    return x * dt, A.new_zeros((x.shape[0],) + tuple(A.shape) if want_state else (0,)), A.new_zeros((0,))


def scan_bwd(x, dt, A, B, C, D, z, dt_bias, lengths, softplus, marks, dy, dstate_out, want_dstate):
    vector = A.new_zeros((A.shape[0],))
    return (dy * dt, dy * x, torch.zeros_like(A), torch.zeros_like(B), torch.zeros_like(C), vector, x.new_zeros((0,) if z is None else x.shape),
            vector.clone(), A.new_zeros((x.shape[0],) + tuple(A.shape) if want_dstate else (0,)))


def scan_step(x, dt, A, B, C, D, z, dt_bias, state, slots, softplus):
    with torch.no_grad():
        state += 1
    return x * dt


def block_norm(x, gate, post_weight, residual, scale, pre_weight, eps, want_stats):
    return x * 2, x.new_zeros((0,) if pre_weight is None else x.shape), x.new_zeros((x.shape[0], 2) if want_stats else (0,))


def block_norm_bwd(x, gate, post_weight, residual, scale, pre_weight, eps, stats, d_out, d_norm, has_residual, residual_f32):
    d_out = torch.zeros_like(x) if d_out is None else d_out
    return d_out * 2, x.new_zeros((0,) if gate is None else x.shape), x.new_zeros(x.shape if has_residual else (0,)), x.new_zeros((3, x.shape[1]))


@pytest.fixture
def ops():
    import unet_amd  # noqa: F401
    library = torch.library.Library("unetmi", "IMPL")
    for name, kernel in dict(seq_conv=conv, seq_conv_bwd=conv_bwd, seq_conv_step=conv_step, ssm_scan=scan, ssm_scan_bwd=scan_bwd,
                             ssm_scan_step=scan_step, block_norm=block_norm, block_norm_bwd=block_norm_bwd).items():
        library.impl(name, kernel, "CPU")
    yield torch.ops.unetmi
    library._destroy()


def rnd(*shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(sum(shape)), dtype=F32)


def sequence_calls():
    """(name, call, its floating tensors by name): every public call that autograd records."""
    from unet_amd import norm, ssm
    return [
        ("causal_conv", ssm.causal_conv, dict(x=rnd(2, 5, 8), weight=rnd(8, 4), bias=rnd(8), state=rnd(2, 3, 8))),
        ("selective_scan", ssm.selective_scan, dict(x=rnd(2, 5, 8), dt=rnd(2, 5, 8), A=-rnd(8, 4).abs(), B=rnd(2, 5, 4), C=rnd(2, 5, 4), D=rnd(8),
                                                    z=rnd(2, 5, 8), dt_bias=rnd(8), state=rnd(2, 8, 4))),
        ("block_norm", lambda **k: norm.block_norm(**k)[0], dict(x=rnd(5, 8), gate=rnd(5, 8), post_weight=rnd(8), residual=rnd(5, 8), scale=rnd(8),
                                                                 pre_weight=rnd(8))),
    ]


def token_calls():
    from unet_amd import ssm
    return [
        ("causal_conv_step", ssm.causal_conv_step, dict(x=rnd(2, 8), state=rnd(2, 3, 8), weight=rnd(8, 4), bias=rnd(8))),
        ("selective_scan_step", ssm.selective_scan_step, dict(x=rnd(2, 8), dt=rnd(2, 8), A=-rnd(8, 4).abs(), B=rnd(2, 4), C=rnd(2, 4),
                                                              state=rnd(2, 8, 4), D=rnd(8), z=rnd(2, 8), dt_bias=rnd(8))),
    ]


def test_forward_mode_derivatives_are_refused(ops):
    """A tangent on any input, with or without a gradient wanted of any, is refused and not dropped."""
    for name, call, given in sequence_calls() + token_calls():
        plain = call(**{k: t.clone() for k, t in given.items()})
        for k, t in given.items():
            with forward_ad.dual_level():
                dual = {**given, k: forward_ad.make_dual(t.clone(), torch.ones_like(t))}
                with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                    call(**dual)
                with torch.no_grad(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                    call(**dual)
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                torch.func.jvp(lambda v: call(**{**given, k: v}), (t,), (torch.ones_like(t),))
        with forward_ad.dual_level():                                  # a level without a tangent on these inputs
            assert torch.equal(call(**{k: t.clone() for k, t in given.items()}), plain), name
    for name, call, given in sequence_calls():
        with forward_ad.dual_level():
            leaves = {k: t.clone().requires_grad_() for k, t in given.items()}
            leaves["x"] = forward_ad.make_dual(leaves["x"], torch.ones_like(given["x"]))
            with pytest.raises(NotImplementedError, match="no forward-mode derivative"):
                call(**leaves)


def test_tangents_of_output_gradients_are_refused(ops):
    """Forward over reverse: the gradient of an output carries the tangent into the backward pass."""
    for name, call, given in sequence_calls():
        leaf = given["x"].clone().requires_grad_()
        y = call(**{**given, "x": leaf})
        plain, = torch.autograd.grad(y, leaf, torch.ones_like(y), retain_graph=True)
        assert plain.shape == leaf.shape
        with forward_ad.dual_level(), pytest.raises(NotImplementedError, match="no forward-mode derivative"):
            torch.autograd.grad(y, leaf, forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_vmap_takes_samples_one_by_one(ops):
    for name, call, given in sequence_calls():
        many = given["x"][None] * torch.arange(1.0, 4.0).reshape((3,) + (1,) * given["x"].dim())
        got = torch.func.vmap(lambda v: call(**{**given, "x": v}))(many)
        assert torch.equal(got, torch.stack([call(**{**given, "x": v}) for v in many])), name


def test_token_calls_refuse_to_be_recorded(ops):
    """Inference only: under grad mode an input, parameter or cache that requires a gradient is refused before the cache is
    touched; without grad mode, or detached, the same call runs."""
    for name, call, given in token_calls():
        for k in given:
            leaves = {n: t.clone().requires_grad_(n == k) for n, t in given.items()}
            with pytest.raises(RuntimeError, match=name + " is inference only"):
                call(**leaves)
            assert torch.equal(leaves["state"], given["state"])
            made = {**leaves, k: leaves[k] * 1}                          # no leaf, but part of a graph
            with pytest.raises(RuntimeError, match=name + " is inference only"):
                call(**made)
            with torch.no_grad():
                y = call(**leaves)
            assert not y.requires_grad and torch.equal(leaves["state"], given["state"] + 1)
            with torch.inference_mode():
                assert torch.equal(call(**leaves), y)
            assert torch.equal(call(**{n: t.detach() for n, t in leaves.items()}), y)


@pytest.mark.parametrize("library", ["missing", "broken"])
def test_the_package_imports_without_the_sequence_operators(tmp_path, library):
    """A library that is not there, or does not load, is the sequence operators' trouble alone: the networks import and are
    built, and the operators say what is missing when they are called."""
    import unet_amd
    here, there = os.path.dirname(os.path.abspath(unet_amd.__file__)), tmp_path / "unet_amd"
    there.mkdir()
    for name in os.listdir(here):
        if name.endswith(".py") or name == "libunetmi.so":
            os.symlink(os.path.join(here, name), there / name)
    if library == "broken":
        (there / "libunetmi_torch.so").write_bytes(b"no library")
    code = """
import torch, unet_amd
assert unet_amd.__file__.startswith({!r}), unet_amd.__file__
unet_amd.UNet(*unet_amd.default_unet_blocks(c_in=2, c_last=1, f_dim=8))
for call in (lambda: unet_amd.ssm.causal_conv(torch.zeros(1, 4, 8), torch.zeros(8, 4)),
             lambda: unet_amd.norm.block_norm(torch.zeros(4, 8))):
    try:
        call()
    except ImportError as e:
        assert "libunetmi_torch.so" in str(e) and "build it" in str(e) and {!r} in str(e), e
    else:
        raise AssertionError("no refusal")
print("told")
""".format(str(tmp_path), "missing" if library == "missing" else "file too short")
    done = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, capture_output=True, text=True, env={**os.environ, "PYTHONPATH": str(tmp_path)})
    assert done.returncode == 0 and "told" in done.stdout, done.stderr
