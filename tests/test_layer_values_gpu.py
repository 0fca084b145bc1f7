"""Values of the layer operators at the ends of their range: infinities, NaN, a type's lowest value, the tails of the activations, bits
that have to stay as they are."""
import pytest
import torch

from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {"fp32": torch.float32, "bf16": torch.bfloat16}
dev = lambda v: None if v is None else v.to(DEV)


@pytest.mark.parametrize("C", [16, 128])                 # the register kernels and the staged ones
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_silu_of_the_convolution_keeps_its_tails(lib, dtype, C):
    """Weights that pick one row, so that the pre-activation is the input exactly and the output silu of it.  Relative bound: half a step
    of the storage type; exp of an argument a that was multiplied by log2 e and rounded, (2 + 1.5 |a|) 2^-23; sum, reciprocal and
    product, 4 2^-23.  An absolute error of 2^-12 of the sigmoid would be most of silu(-8)."""
    from trading_bot_0_b200 import prepost as P
    t, K = TD[dtype], 3
    a = torch.linspace(-40, 40, 641 * C).to(t)
    x = a.view(1, 641, C)
    w = torch.zeros(C, K)
    w[:, -1] = 1.0
    v = x.double()
    ref, half = v * torch.sigmoid(v), torch.finfo(t).eps / 2
    tol = ref.abs() * (half + (6 + 1.5 * v.abs()) * 2.0 ** -23 * (1 + half)) + 1e-37
    out, _ = P.conv1d_carry_forward(dev(x), dev(w))
    over = ((out.double().cpu() - ref).abs() - tol).max().item()
    assert over <= 0, f"forward: {over:.3e} over the bound"
    step = P.conv1d_step(torch.zeros(641, K - 1, C, dtype=t, device=DEV), dev(x[0]), dev(w))
    assert torch.equal(step, out[0])
    many = dev(x[0]).repeat(40, 1)                       # streams enough for a thread to take several, the last ones fewer
    some = P.conv1d_step(torch.zeros(len(many), K - 1, C, dtype=t, device=DEV), many, dev(w))
    assert torch.equal(some.view(40, 641, C), step.expand(40, 641, C))


def _scan(dtype, B=2, L=21, D=24, N=8, seed=7):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    t = TD[dtype]
    return dict(x=n(B, L, D).to(t), dt=(0.5 * n(B, L, D) - 2.0).to(t), A=-(0.2 + 4.0 * torch.rand(D, N, generator=g)), Bm=n(B, L, 1, N).to(t),
                Cm=n(B, L, 1, N).to(t), D=n(D), z=n(B, L, D).to(t), init_state=n(B, D, N)), n(B, L, D).to(t), n(B, D, N)


ORDER = ("x", "dt", "A", "Bm", "Cm", "D", "z", "init_state")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_steps_that_are_switched_off(lib, dtype):
    """A step size of -inf, or of the type's lowest value, is a softplus of 0: the token leaves the state as it is, bit for bit, and takes
    no gradient; so does a channel whose bias is -inf.  Against the 64-bit recurrence with the bound of its own test."""
    from tests.test_selective_gpu import assert_near, _tokens
    from trading_bot_0_b200 import selective as S
    o, dy, dfin = _scan(dtype)
    B, L, D = o["x"].shape
    N = o["A"].shape[1]
    low = torch.finfo(TD[dtype]).min
    o["dt"][:, 3] = -float("inf")
    o["dt"][0, 5:9, ::2] = low
    o["dt"][1, 10:18] = -2.4e38                           # (log2 e times this is past fp32)
    o["dt"][:, -1] = -float("inf")
    bias = torch.zeros(D)
    bias[4] = -float("inf")
    ref, mag = (O.selective_scan_ref(*(o[k] for k in ORDER), dt_bias=bias, dt_softplus=True, dy=dy, dfinal=dfin, magnitude=m) for m in (False, True))
    tok = _tokens(o, dict(dt_bias=bias, dt_softplus=True), L)
    a = [dev(o[k]) for k in ORDER]
    kd = dict(dt_bias=dev(bias), dt_softplus=True)
    y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
    assert_near("y", y, ref["y"], mag["y"], tok, N)
    assert_near("final_state", fin, ref["final_state"], mag["final_state"], tok, 0)
    assert torch.equal(fin[:, 4].cpu(), o["init_state"][:, 4])
    g = S.selective_scan_backward(dev(dy), *a, dev(dfin), workspace=ws, **kd)
    for k, terms in dict(dx=N, ddt=N, dz=N, dA=B * L, dD=B * L, ddt_bias=B * L + N, dB=D, dC=D, dinit=0).items():
        assert_near(k, g[k], ref[k], mag[k], tok, terms)
    assert (g["ddt"][:, 3] == 0).all() and (g["ddt"][..., 4] == 0).all()
    st = a[7].clone()
    ys = [S.selective_step(st, a[0][:, t], a[1][:, t], a[2], a[3][:, t], a[4][:, t], a[5], a[6][:, t], **kd) for t in range(L)]
    assert_near("steps", torch.stack(ys, 1), ref["y"], mag["y"], tok, N)
    before = st.clone()
    S.selective_step(st, a[0][:, 3], a[1][:, 3], a[2], a[3][:, 3], a[4][:, 3], a[5], a[6][:, 3], **kd)
    assert torch.equal(st, before)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_step_as_large_as_the_type(lib, dtype):
    """softplus of the largest values is the value: with x = 0 there, everything is forgotten and nothing added."""
    from trading_bot_0_b200 import selective as S
    o, _, _ = _scan(dtype)
    o["dt"][:, 6] = torch.finfo(TD[dtype]).max
    o["x"][:, 6] = 0
    a = [dev(o[k]) for k in ORDER]
    y, _, _ = S.selective_scan_forward(*a, dt_softplus=True)
    assert (y[:, 6] == 0).all() and torch.isfinite(y).all()
    cut, _, _ = S.selective_scan_forward(*(v[:, 7:] if v.dim() > 2 and v.shape[1] == 21 else v for v in a[:7]), torch.zeros_like(a[7]), dt_softplus=True)
    half = torch.finfo(TD[dtype]).eps
    assert ((y[:, 7:] - cut).float().abs() <= half * cut.float().abs() + 2.0 ** -18).all()     # (tiles of 16 tokens start elsewhere)


ENDS = [float("inf"), -float("inf"), float("nan"), 3.3e38, -3.3e38, 2.4e38, -2.4e38, 0.0]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,K", [(3, 64), (40, 64), (300, 64), (50, 33), (64, 1536)])    # few rows, tensor cores or CUDA cores, splits
def test_softplus_of_the_projection_at_its_ends(lib, dtype, M, K):
    """The pre-activation is the bias (x is zero): inf, 0, NaN, the value itself; slopes 1, 0, NaN."""
    from trading_bot_0_b200 import linear as LN
    N = 48
    x, w = torch.zeros(M, K, dtype=TD[dtype]), torch.ones(N, K, dtype=TD[dtype])
    b = torch.tensor(ENDS).repeat(N // len(ENDS)).to(TD[dtype])
    want = torch.where(b < -1e30, 0.0, torch.where(b == 0, torch.log(torch.tensor(2.0)), b.float())).to(TD[dtype]).expand(M, N)
    out, pre = LN.linear_forward(dev(x), dev(w), dev(b), activation="softplus", for_backward=True)
    eps = torch.finfo(TD[dtype]).eps
    assert torch.allclose(out.cpu().float(), want.float(), rtol=eps, atol=0, equal_nan=True)
    _, _, db = LN.linear_backward(torch.ones(M, N, dtype=TD[dtype], device=DEV), dev(x), dev(w), pre, activation="softplus", want_dx=False,
                                  want_dweight=False)
    slope = torch.where(b.isnan(), b.float(), torch.sigmoid(b.float())) * M
    assert torch.allclose(db.cpu().float(), slope, rtol=eps, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("act", ["none", "silu", "softplus", "relu2"])
@pytest.mark.parametrize("M,K,N", [(3, 64, 48), (3, 64, 8200), (40, 64, 48), (64, 1536, 128), (300, 64, 520), (50, 33, 40), (64, 1540, 40), (2100, 40, 1300)])
def test_nan_goes_through_every_activation(lib, dtype, act, M, K, N):
    """A NaN in one row of x or in one bias makes that row and that column NaN, in the output and in the gradients that meet it, and
    nothing else; on the kernels of few rows, of the tensor cores (with and without splits) and of the CUDA cores."""
    from trading_bot_0_b200 import linear as LN
    g = torch.Generator().manual_seed(M + K)
    n = lambda *s: torch.randn(*s, generator=g).to(TD[dtype])
    x, w, b, r, dout = n(M, K), (n(N, K).float() / K ** 0.5).to(TD[dtype]), n(N), n(M, N), n(M, N)
    x[1, 5], b[7] = float("nan"), float("nan")
    bad = torch.zeros(M, N, dtype=torch.bool)
    bad[1], bad[:, 7] = True, True
    out, pre = LN.linear_forward(dev(x), dev(w), dev(b), dev(r), activation=act, for_backward=True)
    assert torch.equal(out.isnan().cpu(), bad)
    if act == "none":
        return
    dx, dw, db = LN.linear_backward(dev(dout), dev(x), dev(w), pre, activation=act)
    assert db.isnan().all()                               # (every column has the bad row in its sum)
    assert dx.isnan().all()                               # (every row has the bad column)
    finite = x.clone()
    finite[1, 5] = 0.5
    _, pre = LN.linear_forward(dev(finite), dev(w), dev(b), dev(r), activation=act, for_backward=True)
    dx, dw, db = LN.linear_backward(dev(dout), dev(finite), dev(w), pre, activation=act)
    col = torch.arange(N) == 7
    assert torch.equal(db.isnan().cpu(), col) and torch.equal(dw.isnan().any(1).cpu(), col) and dw[7].isnan().all()


def test_a_single_steps_decay_is_unbiased(lib):
    """50 steps without input: the states decay by exp(50 s A).  A decay's error per step scatters by 4e-8 over the 4096 pairs of channel
    and state, its mean by 6e-10; the offset that the scan's exponential is corrected for is 2e-8, met to 0.6e-8 in every interval of the
    argument.  Bound on the mean error per step: 0.6e-8 + 3 * 6e-10 + 1e-9 for the state's own roundings (2^-24 / sqrt(3) / sqrt(50 * 4096)
    three times, and the first)."""
    from trading_bot_0_b200 import selective as S
    g = torch.Generator().manual_seed(11)
    D, N, steps = 256, 16, 50
    A = -torch.exp(torch.rand(D, N, generator=g) * 2.0 - 2.0)
    s = 0.02 + 0.48 * torch.rand(1, D, generator=g)
    h0 = 1.0 + torch.rand(1, D, N, generator=g)
    st, z, bc = dev(h0).clone(), torch.zeros(1, D, device=DEV), torch.zeros(1, N, device=DEV)
    for _ in range(steps):
        S.selective_step(st, z, dev(s), dev(A), bc, bc)
    ref = h0.double() * torch.exp(steps * s.double()[..., None] * A.double())
    off = ((st.double().cpu() - ref) / ref).mean().item() / steps
    assert abs(off) <= 0.6e-8 + 3 * 6e-10 + 1e-9, off


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("N", [4, 16, 40])
def test_rows_end_inside_a_tile(lib, dtype, N):
    """A length inside a tile: state, outputs and gradients are, bit for bit, those of the same row cut there.  (Exact: past the length
    the decay is exp(0) and the input 0, so nothing is rounded again.)"""
    from trading_bot_0_b200 import selective as S
    L, D, lens = 40, 24, [1, 3, 5, 8, 9, 15, 17, 23, 31, 33, 39]
    g = torch.Generator().manual_seed(N)
    n = lambda *s: torch.randn(*s, generator=g)
    t, B = TD[dtype], len(lens)
    a = [dev(v) for v in (n(B, L, D).to(t), (0.5 * n(B, L, D) - 2).to(t), -(0.2 + 4 * torch.rand(D, N, generator=g)), n(B, L, N).to(t), n(B, L, N).to(t),
                          n(D), n(B, L, D).to(t), n(B, D, N))]
    dy, dfin = dev(n(B, L, D).to(t)), dev(n(B, D, N))
    y, fin, ws = S.selective_scan_forward(*a, dt_softplus=True, lengths=torch.tensor(lens, dtype=torch.int32, device=DEV), for_backward=True)
    gr = S.selective_scan_backward(dy, *a, dfin, dt_softplus=True, lengths=torch.tensor(lens, dtype=torch.int32, device=DEV), workspace=ws)
    for i, m in enumerate(lens):
        row = [v[i:i + 1, :m] if v.dim() == 3 and v.shape[:2] == (B, L) else v for v in a[:7]] + [a[7][i:i + 1]]
        y1, f1, w1 = S.selective_scan_forward(*row, dt_softplus=True, for_backward=True)
        assert torch.equal(f1[0], fin[i]) and torch.equal(y1[0], y[i, :m]), m
        g1 = S.selective_scan_backward(dy[i:i + 1, :m], *row, dfin[i:i + 1], dt_softplus=True, workspace=w1)
        for k in ("dx", "ddt", "dz", "dB", "dC"):
            assert torch.equal(g1[k][0], gr[k][i, :m]), (k, m)
        assert torch.equal(g1["dinit"][0], gr["dinit"][i]), m


@pytest.mark.parametrize("D,N,L", [(256, 16, 50), (512, 8, 50), (64, 64, 50), (256, 16, 200)])    # the last one in parts
def test_a_scans_decays_are_unbiased(lib, D, N, L):
    """The same over a sequence, forward (the final state) and backward (the gradient of the initial one); steps that vary from token to
    token, and a decay of at least exp(-50) over all.  Bound as above, the state's roundings 2^-24 / sqrt(3) / sqrt(L D N) each."""
    from trading_bot_0_b200 import selective as S
    g = torch.Generator().manual_seed(D + N + L)
    A = -torch.exp(torch.rand(D, N, generator=g) * 2.0 - 2.0)
    s = (0.02 + 0.48 * torch.rand(1, L, D, generator=g)) * 50 / max(L, 50)
    h0 = 1.0 + torch.rand(1, D, N, generator=g)
    z, bc = torch.zeros(1, L, D, device=DEV), torch.zeros(1, L, N, device=DEV)
    _, fin, _ = S.selective_scan_forward(z, dev(s), dev(A), bc, bc, init_state=dev(h0))
    dinit = S.selective_scan_backward(z, z, dev(s), dev(A), bc, bc, init_state=dev(h0), dfinal_state=dev(h0))["dinit"]
    ref = h0.double() * torch.exp(s.double().sum(1)[..., None] * A.double())
    for name, got in (("final state", fin), ("gradient of the initial state", dinit)):
        off = ((got.double().cpu() - ref) / ref).mean().item() / L
        assert abs(off) <= 0.6e-8 + 3 * 6e-10 + 1e-9, (name, off)
