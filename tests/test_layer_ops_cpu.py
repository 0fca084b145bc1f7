"""Refusals of the layer operators' C entry points and of their Python functions, all before any launch: runs without a GPU."""
import ctypes as C

import pytest
import torch

BASE = 0x7f0000000000      # addresses that nothing reads: every call below is refused first


def at(i, off=0):
    return C.c_void_p(BASE + i * 0x1000000 + off)


def _sel(**kw):
    from trading_bot_0_b200 import _lib as L
    d = L.SsdSelDims()
    d.batch, d.seqlen, d.channels, d.dstate, d.ngroups, d.dtype, d.device = 2, 100, 48, 16, 1, L.SSD_BF16, -1
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def _err(lib):
    return lib.ssd_last_error().decode()


@pytest.mark.parametrize("kw,needle", [(dict(batch=0), "positive"), (dict(seqlen=0), "positive"), (dict(channels=-1), "positive"),
                                       (dict(dstate=65), "dstate"), (dict(ngroups=5), "multiple of ngroups"), (dict(dtype=7), "dtype"),
                                       (dict(x_stride_l=47), "strides"), (dict(b_stride_l=15), "strides"), (dict(y_stride_l=8), "strides")])
def test_selscan_dims(lib, kw, needle):
    d = _sel(**kw)
    assert lib.ssd_selscan_workspace_bytes(C.byref(d), 0) == 0 and needle in _err(lib)


def test_selscan_pointers_and_workspace(lib):
    from trading_bot_0_b200 import _lib as L
    d = _sel()
    fwd, bwd = (lib.ssd_selscan_workspace_bytes(C.byref(d), p) for p in (0, 1))
    assert 0 < fwd < bwd
    p = L.SsdSelFwdPtrs()
    assert lib.ssd_selscan_forward(None, C.byref(p), at(20), fwd, None) == -6
    assert lib.ssd_selscan_forward(C.byref(d), C.byref(p), at(20), fwd, None) == -6
    for n in ("x", "dt", "A", "Bm", "Cm", "y"):
        setattr(p, n, at(1))
    assert lib.ssd_selscan_forward(C.byref(d), C.byref(p), None, fwd, None) == -6
    assert lib.ssd_selscan_forward(C.byref(d), C.byref(p), at(20), fwd - 1, None) == -4 and str(fwd) in _err(lib)
    b = L.SsdSelBwdPtrs()
    assert lib.ssd_selscan_backward(C.byref(d), C.byref(b), at(20), bwd, None) == -6
    for n in ("x", "dt", "A", "Bm", "Cm", "dy", "dx", "ddt", "dA", "dB", "dC"):
        setattr(b, n, at(1))
    assert lib.ssd_selscan_backward(C.byref(d), C.byref(b), at(20), fwd, None) == -4
    for given in ("z", "D", "dt_bias"):       # a gradient that nothing would hold
        setattr(b, given, at(2))
        assert lib.ssd_selscan_backward(C.byref(d), C.byref(b), at(20), bwd, None) == -6 and "go with" in _err(lib)
        setattr(b, given, None)
    s, q = L.SsdSelStepDims(), L.SsdStepPtrs()
    assert lib.ssd_selscan_step(C.byref(s), C.byref(q), None) == -1
    s.streams, s.channels, s.dstate, s.ngroups, s.device = 4, 48, 16, 1, -1
    assert lib.ssd_selscan_step(C.byref(s), C.byref(q), None) == -6
    s.x_stride_s = 5
    for n in ("state", "x", "dt", "A", "Bm", "Cm", "y"):
        setattr(q, n, at(1))
    assert lib.ssd_selscan_step(C.byref(s), C.byref(q), None) == -1 and "strides" in _err(lib)


def test_carry_entry_points(lib):
    from trading_bot_0_b200 import _lib as L
    d = L.SsdConvDims()
    d.batch, d.seqlen, d.channels, d.width, d.dtype, d.device, d.activation = 2, 50, 64, 4, L.SSD_BF16, -1, 1
    d.in_stride_l = d.out_stride_l = 64
    d.in_stride_b = d.out_stride_b = 3200
    f = lambda *a: lib.ssd_conv1d_carry_forward(C.byref(d), *a, None)
    assert f(None, at(2), None, None, None, at(3), None) == -6
    assert f(at(1), None, None, None, None, at(3), None) == -6
    assert f(at(1, 8), at(2), None, None, None, at(3), None) == -2
    assert f(at(1), at(2), None, at(4, 4), None, at(3), None) == -2
    assert f(at(1), at(2), None, at(4), None, at(3), at(4, 256)) == -1 and "overlap" in _err(lib)
    need = lib.ssd_conv1d_carry_workspace_bytes(C.byref(d))
    assert need > 0
    b = lambda dout, sl, din, dw, n: lib.ssd_conv1d_carry_backward(C.byref(d), at(1), at(2), None, None, None, dout, 3200, sl, None, din, None, dw,
                                                                   None, at(9), n, None)
    assert b(None, 64, at(6), at(7), need) == -6 and b(at(5), 64, None, at(7), need) == -6 and b(at(5), 64, at(6), None, need) == -6
    assert b(at(5), 60, at(6), at(7), need) == -2 and b(at(5), 66, at(6), at(7), need) == -2
    assert b(at(5), 64, at(6), at(7), need - 4) == -4
    assert lib.ssd_conv1d_step(C.byref(d), at(1), at(2), None, at(3), at(4), None) == -1 and "seqlen" in _err(lib)
    d.seqlen = 1
    assert lib.ssd_conv1d_step(C.byref(d), at(1), at(2), None, None, at(4), None) == -6
    d.channels = 60
    assert lib.ssd_conv1d_carry_workspace_bytes(C.byref(d)) == 0 and "multiple of 8" in _err(lib)


def test_linear_entry_points(lib):
    from trading_bot_0_b200 import _lib as L
    d = L.SsdLinearDims()
    assert lib.ssd_linear_workspace_bytes(C.byref(d), 0) == 0 and "positive" in _err(lib)
    d.rows, d.in_features, d.out_features, d.dtype, d.device = 100, 64, 96, L.SSD_BF16, -1
    fwd, bwd = (lib.ssd_linear_workspace_bytes(C.byref(d), p) for p in (0, 1))
    assert fwd > 0 and bwd > 0
    f = lambda x, w, out, n: lib.ssd_linear_forward(C.byref(d), x, w, None, None, out, None, at(9), n, None)
    assert f(None, at(2), at(3), fwd) == -6 and f(at(1), None, at(3), fwd) == -6 and f(at(1), at(2), None, fwd) == -6
    assert f(at(1), at(2), at(3), fwd - 1) == -4
    b = lambda dout, s: lib.ssd_linear_backward(C.byref(d), at(1), at(2), None, dout, s, at(4), at(5), None, at(9), bwd, None)
    assert b(None, 0) == -6 and b(at(3), 95) == -1
    d.activation = 1
    assert b(at(3), 0) == -6 and "pre" in _err(lib)
    for k, v in (("activation", 4), ("dtype", 5), ("x_stride_row", 63), ("out_stride_row", 95), ("residual_stride_row", 1)):
        old = getattr(d, k)
        setattr(d, k, v)
        assert lib.ssd_linear_workspace_bytes(C.byref(d), 0) == 0, k
        setattr(d, k, old)


def test_struct_sizes(lib):
    from trading_bot_0_b200 import _lib as L
    assert C.sizeof(L.SsdSelDims) == 8 * 4 + 12 * 8 and C.sizeof(L.SsdSelFwdPtrs) == 12 * 8 and C.sizeof(L.SsdSelBwdPtrs) == 22 * 8
    assert C.sizeof(L.SsdSelStepDims) == 8 * 4 + 6 * 8 and C.sizeof(L.SsdLinearDims) == 8 + 6 * 4 + 3 * 8


def test_python_functions_refuse_cpu_tensors(lib):
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import linear, prepost, selective
    x = torch.zeros(1, 8, 16)
    bc, A = torch.zeros(1, 8, 4), -torch.ones(16, 4)
    with pytest.raises(ValueError, match="CUDA"):
        selective.selective_scan_forward(x, x, A, bc, bc)
    with pytest.raises(ValueError, match="CUDA"):
        selective.selective_scan(x.requires_grad_(), x, A, bc, bc)
    with pytest.raises(ValueError, match="CUDA"):
        selective.selective_step(torch.zeros(1, 16, 4), x[:, 0], x[:, 0], A, bc[:, 0], bc[:, 0])
    with pytest.raises(ValueError, match="CUDA"):
        prepost.conv1d_carry_forward(x.detach(), torch.zeros(16, 4))
    with pytest.raises(ValueError, match="CUDA"):
        prepost.conv1d_step(torch.zeros(1, 3, 16), x.detach()[:, 0], torch.zeros(16, 4))
    with pytest.raises(ValueError, match="CUDA"):
        T.linear_forward(x.detach(), torch.zeros(8, 16))
    with pytest.raises(ValueError, match="activation"):
        linear.linear(x.detach(), torch.zeros(8, 16), activation="tanh")
    with pytest.raises(ValueError, match="tensor"):
        T.selective_scan(None, x, A, bc, bc)


def test_oracle_gradients_are_autograds():
    """The restatement's reverse recurrence against autograd of its own forward recurrence."""
    from oracle import layer_oracle as O
    g = torch.Generator().manual_seed(0)
    n = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)
    B, L, D, N = 2, 9, 6, 3
    ls = dict(x=n(B, L, D), dt=n(B, L, D), A=-n(D, N).abs(), Bm=n(B, L, 2, N), C=n(B, L, 2, N), D=n(D), z=n(B, L, D), init=n(B, D, N), dt_bias=n(D))
    dy, df = n(B, L, D), n(B, D, N)
    lengths = torch.tensor([9, 5])
    r = O.selective_scan_ref(*(ls[k] for k in ("x", "dt", "A", "Bm", "C", "D", "z", "init")), dt_bias=ls["dt_bias"], dt_softplus=True,
                             lengths=lengths, dy=dy, dfinal=df)
    v = {k: t.clone().requires_grad_() for k, t in ls.items()}
    h, ys = v["init"], []
    for t in range(L):
        live = (t < lengths)[:, None]
        s = torch.where(live, O.softplus(v["dt"][:, t] + v["dt_bias"]), 0.0)
        Bt, Ct = v["Bm"][:, t].repeat_interleave(3, 1), v["C"][:, t].repeat_interleave(3, 1)
        h = torch.exp(s[..., None] * v["A"]) * h + (s * v["x"][:, t])[..., None] * Bt
        ys.append(torch.where(live, ((h * Ct).sum(-1) + v["D"] * v["x"][:, t]) * torch.nn.functional.silu(v["z"][:, t]), 0.0))
    got = torch.autograd.grad([torch.stack(ys, 1), h], list(v.values()), [dy, df])
    for k, a in zip(("dx", "ddt", "dA", "dB", "dC", "dD", "dz", "dinit", "ddt_bias"), got):
        assert torch.allclose(a, r[k].reshape(a.shape), rtol=1e-12, atol=1e-12), k
