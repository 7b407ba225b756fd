"""The sequence operators' host side without a GPU: shape inference, refusals of the C entry points and of the Python ones,
and the 64-bit restatements the device is tested against (against automatic differentiation and central differences)."""

import ctypes

import pytest
import torch

from seq_oracle import conv64, norm64, scan64


def rnd(shape, seed):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def test_sequence_ops_infer_shapes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    import unet_amd  # noqa: F401  (registers the ops)
    ops = torch.ops.unetmi
    with FakeTensorMode():
        x, w, c = torch.empty(2, 37, 24, dtype=torch.bfloat16), torch.empty(24, 4), torch.empty(24)
        y, s = ops.seq_conv(x, w, c, None, None, True, True)
        assert y.shape == x.shape and y.dtype == x.dtype and s.shape == (2, 3, 24) and s.dtype == x.dtype
        dx, dw, db, ds = ops.seq_conv_bwd(x, w, c, s, None, True, x, None)
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == c.shape and ds.shape == s.shape and dw.dtype == torch.float32
        assert ops.seq_conv_step(x[:, 0], w, c, torch.empty(5, 3, 24, dtype=x.dtype), None, True).shape == (2, 24)
        A, B, h = torch.empty(24, 16), torch.empty(2, 37, 3, 16, dtype=x.dtype), torch.empty(2, 24, 16)
        y, s, marks = ops.ssm_scan(x, x, A, B, B, c, x, c, h, None, True, True, True)
        assert y.shape == x.shape and y.dtype == x.dtype and s.shape == h.shape and s.dtype == torch.float32
        assert marks.shape == (2 * 5 * 24 * 16,)
        out = ops.ssm_scan_bwd(x, x, A, B, B, c, x, c, None, True, marks, x, None, True)
        assert [tuple(t.shape) for t in out] == [tuple(t.shape) for t in (x, x, A, B, B, c, x, c, h)]
        assert [t.dtype for t in out] == [t.dtype for t in (x, x, A, B, B, c, x, c, h)]
        assert ops.ssm_scan_step(x[:, 0], x[:, 0], A, B[:, 0], B[:, 0], c, None, c, h, None, True).shape == (2, 24)
        rows, r = x.reshape(-1, 24), torch.empty(74, 24)
        out, n, stats = ops.block_norm(rows, rows, c, r, c, c, 1e-6, True)
        assert stats.shape == (rows.shape[0], 2) and stats.dtype == torch.float32
        assert out.shape == n.shape == rows.shape and out.dtype == torch.float32 and n.dtype == torch.bfloat16
        dx, dg, dr, dw = ops.block_norm_bwd(rows, rows, c, r, c, c, 1e-6, stats, r, rows, True, True)
        assert dx.shape == dg.shape == dr.shape == rows.shape and dr.dtype == torch.float32 and dw.shape == (3, 24)


def test_marks_match_between_host_and_shape_inference():
    """The saved states' size, as the library and as shape inference have it, over every lane layout."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from unet_amd import _lib
    for N in (1, 4, 5, 8, 9, 16, 17, 32, 33, 64):
        for L in (0, 1, 4, 15, 16, 17, 333):
            d = _lib.ScanDesc(3, L, 70, N, 1, 0, 1, 0)
            with FakeTensorMode():
                x, B = torch.empty(3, L, 70), torch.empty(3, L, 1, N)
                marks = torch.ops.unetmi.ssm_scan(x, x, torch.empty(70, N), B, B, None, None, None, None, None, True, False, True)[2]
            assert _lib.lib.unetmi_ssm_scan_marks_bytes(ctypes.byref(d)) == 4 * marks.numel(), (N, L)


def test_c_entry_points_refuse():
    """Bad descriptors and missing pointers come back as codes with a message; nothing touches a device."""
    from unet_amd import _lib
    lib = _lib.lib
    conv = lambda **k: _lib.SeqConvDesc(**{**dict(batch=1, length=4, channels=8, taps=4, act=0, dtype=0), **k})  # noqa: E731
    scan = lambda **k: _lib.ScanDesc(**{**dict(batch=1, length=4, channels=8, state=4, groups=1, dtype=0, softplus=1), **k})  # noqa: E731
    norm = lambda **k: _lib.NormDesc(**{**dict(rows=4, channels=8, dtype=0, residual_dtype=0, eps=1e-6), **k})  # noqa: E731
    ref = ctypes.byref

    def refused(rc, code, text):
        assert rc == code and text in _lib.last_error(), (rc, _lib.last_error())

    fwd = lambda d: lib.unetmi_seq_conv_fwd(ref(d), *[None] * 8)  # noqa: E731
    refused(fwd(conv()), _lib.E_BAD_ARG, "null")
    refused(fwd(conv(taps=1)), _lib.E_UNSUPPORTED, "taps")
    refused(fwd(conv(taps=5)), _lib.E_UNSUPPORTED, "taps")
    refused(fwd(conv(act=1)), _lib.E_UNSUPPORTED, "activation")
    refused(fwd(conv(dtype=2)), _lib.E_UNSUPPORTED, "bfloat16")
    refused(fwd(conv(batch=-1)), _lib.E_BAD_DESC, "sizes")
    refused(fwd(conv(batch=70000)), _lib.E_UNSUPPORTED, "65535")
    refused(fwd(conv(x_stride=(-1, 0))), _lib.E_BAD_DESC, "stride")
    refused(lib.unetmi_seq_conv_fwd(None, *[None] * 8), _lib.E_BAD_ARG, "null descriptor")
    assert fwd(conv(batch=0)) == 0
    refused(lib.unetmi_seq_conv_bwd(ref(conv()), *[None] * 12, 0, None), _lib.E_BAD_ARG, "null")
    refused(lib.unetmi_seq_conv_step(ref(conv()), *[None] * 4, 1, None, None, None), _lib.E_BAD_ARG, "null")
    assert lib.unetmi_seq_conv_bwd_workspace_bytes(ref(conv())) > 0 and lib.unetmi_seq_conv_bwd_workspace_bytes(ref(conv(taps=9))) == 0
    one = ctypes.c_char_p(b"x" * 64)                         # a pointer that nothing may follow
    p = ctypes.cast(one, ctypes.c_void_p)
    refused(lib.unetmi_seq_conv_bwd(ref(conv()), *[p] * 12, 0, None), _lib.E_BAD_ARG, "workspace")
    refused(lib.unetmi_seq_conv_step(ref(conv(batch=3)), p, p, None, None, 2, p, p, None), _lib.E_BAD_ARG, "slots")

    fwd = lambda d: lib.unetmi_ssm_scan_fwd(ref(d), *[None] * 14, 0, None)  # noqa: E731
    refused(fwd(scan()), _lib.E_BAD_ARG, "null")
    refused(fwd(scan(state=65)), _lib.E_UNSUPPORTED, "64 states")
    refused(fwd(scan(state=0)), _lib.E_BAD_DESC, "sizes")
    refused(fwd(scan(groups=3)), _lib.E_BAD_DESC, "groups")
    refused(fwd(scan(dtype=7)), _lib.E_UNSUPPORTED, "bfloat16")
    refused(fwd(scan(batch=65536)), _lib.E_UNSUPPORTED, "65535")
    refused(fwd(scan(c_stride=(0, 0, -1))), _lib.E_BAD_DESC, "stride")
    refused(fwd(scan(length=1 << 29)), _lib.E_UNSUPPORTED, "steps")
    long = scan(length=4096)
    assert lib.unetmi_ssm_scan_fwd_workspace_bytes(ref(long), 0) > 0
    refused(lib.unetmi_ssm_scan_fwd(ref(long), *[p] * 13, None, 0, None), _lib.E_BAD_ARG, "workspace")
    refused(lib.unetmi_ssm_scan_bwd(ref(scan()), *[None] * 22, 0, None), _lib.E_BAD_ARG, "null")
    refused(lib.unetmi_ssm_scan_bwd(ref(scan()), *[p] * 22, 0, None), _lib.E_BAD_ARG, "workspace")
    refused(lib.unetmi_ssm_scan_bwd(ref(scan(batch=0)), *[p] * 22, 0, None), _lib.E_BAD_DESC, "empty")
    refused(lib.unetmi_ssm_scan_step(ref(scan(batch=2)), *[p] * 8, None, 1, p, p, None), _lib.E_BAD_ARG, "slots")

    fwd = lambda d, *a: lib.unetmi_block_norm_fwd(ref(d), *(a or [None] * 9), None)  # noqa: E731
    refused(fwd(norm()), _lib.E_BAD_ARG, "null")
    refused(fwd(norm(channels=8193)), _lib.E_UNSUPPORTED, "8192")
    refused(fwd(norm(dtype=1, residual_dtype=2)), _lib.E_UNSUPPORTED, "residual")
    refused(fwd(norm(eps=-1.0)), _lib.E_BAD_DESC, "eps")
    refused(fwd(norm(eps=float("nan"))), _lib.E_BAD_DESC, "eps")
    refused(fwd(norm(), p, None, None, None, p, None, p, None, None), _lib.E_BAD_ARG, "residual")
    refused(lib.unetmi_block_norm_bwd(ref(norm()), *[p] * 14, 0, None), _lib.E_BAD_ARG, "workspace")
    refused(lib.unetmi_block_norm_bwd(ref(norm()), *[p] * 6, None, *[p] * 7, 1 << 30, None), _lib.E_BAD_ARG, "null")     # no stats
    refused(lib.unetmi_block_norm_bwd(ref(norm(rows=0)), *[p] * 14, 0, None), _lib.E_BAD_DESC, "rows")


def test_cpu_tensors_have_no_kernel():
    from unet_amd import norm, ssm
    x = torch.zeros(1, 4, 8)
    with pytest.raises(NotImplementedError):
        ssm.causal_conv(x, torch.zeros(8, 4))
    with pytest.raises(NotImplementedError):
        norm.block_norm(x, post_weight=torch.ones(8))
    with pytest.raises(ValueError, match="residual"):
        norm.block_norm(x, scale=torch.ones(8))


def check_slopes(value, inputs, grads):
    """Gradients against central differences of a 64-bit function along one direction in all its inputs."""
    way = {k: rnd(t.shape, 90 + i) for i, (k, t) in enumerate(inputs.items())}
    h = 1e-5
    quotient = (value({k: t + h * way[k] for k, t in inputs.items()}) - value({k: t - h * way[k] for k, t in inputs.items()})) / (2 * h)
    parts = [(grads[k] * way[k]).sum() for k in inputs]
    assert abs(sum(parts) - quotient) <= 1e-6 * sum(abs(p) for p in parts)


def test_restatements_against_differences():
    lengths = torch.tensor([11, 4], dtype=torch.int32)
    i = dict(x=rnd((2, 11, 6), 1), dt=rnd((2, 11, 6), 2), A=-rnd((6, 5), 3).abs(), B=rnd((2, 11, 2, 5), 4), C=rnd((2, 11, 2, 5), 5), D=rnd((6,), 6),
             z=rnd((2, 11, 6), 7), dt_bias=rnd((6,), 8), state=rnd((2, 6, 5), 9))
    dy, ds = rnd((2, 11, 6), 10), rnd((2, 6, 5), 11)
    got = scan64(**i, lengths=lengths, dy=dy, dout=ds)

    def scan_value(v):
        r = scan64(**v, lengths=lengths)
        return (r["y"] * dy).sum() + (r["state"] * ds).sum()

    check_slopes(scan_value, i, {k: got["d_" + k] for k in i})
    i = dict(x=rnd((2, 11, 6), 1), w=rnd((6, 4), 2), bias=rnd((6,), 3), state=rnd((2, 3, 6), 4))
    ds = rnd((2, 3, 6), 5)
    got = conv64(**i, lengths=lengths, silu=True, dy=dy, dout=ds)

    def conv_value(v):
        r = conv64(**v, lengths=lengths, silu=True)
        return (r["y"] * dy).sum() + (r["state"] * ds).sum()

    check_slopes(conv_value, i, dict(x=got["dx"], w=got["dw"], bias=got["db"], state=got["dstate"]))
    i = dict(x=rnd((5, 9), 1), gate=rnd((5, 9), 2), post=rnd((9,), 3), residual=rnd((5, 9), 4), scale=rnd((9,), 5), pre=rnd((9,), 6))
    d1, d2 = rnd((5, 9), 7), rnd((5, 9), 8)
    got = norm64(**i, eps=1e-3, d_out=d1, d_norm=d2)

    def norm_value(v):
        r = norm64(**v, eps=1e-3)
        return (r["r"] * d1).sum() + (r["n"] * d2).sum()

    check_slopes(norm_value, i, {k: got["d_" + k] for k in i})
