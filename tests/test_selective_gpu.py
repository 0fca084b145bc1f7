"""The selective scan (a decay per channel and state), its gradients and its single step against the recurrence in 64 bits.

Tolerances.  An output is off by at most: half a step of its storage type; and the fp32 arithmetic, relative to the sum of the
magnitudes of its terms (the recurrence evaluated on magnitudes).  Per token that a term came through: 2^-22 for the exponential, 2^-22
for the roundings of product and sum, and for its argument s A, whose error relative to the argument is 2^-21 for the softplus and 2^-22
for two roundings, at most 3 |s A| 2^-22.  Then 16 2^-22 for the step size, the gate's sigmoid and the outer products, and 2^-24 per
term of a sum in order.  So (2 tokens + 16) 2^-22 + terms 2^-24 with tokens = L (1 + 1.5 max |s A|): the worst case of every
rounding."""
import pytest
import torch

from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {"fp32": torch.float32, "bf16": torch.bfloat16}


def _operands(B, L, D, N, G, dtype, *, gate, bias, skip, init, seed=5, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    t = TD[dtype]
    n = lambda *s: torch.randn(*s, generator=g)
    o = dict(x=n(B, L, D).to(t), dt=(0.5 * n(B, L, D)).to(t), A=-(0.2 + 4.0 * torch.rand(D, N, generator=g)), Bm=n(B, L, G, N).to(t),
             Cm=n(B, L, G, N).to(t), D=n(D) if skip else None, z=n(B, L, D).to(t) if gate else None,
             init_state=n(B, D, N) if init else None)
    kw = dict(dt_bias=0.5 * n(D) - 2.5, dt_softplus=True) if bias else dict(dt_softplus=False)
    if not bias:
        o["dt"] = o["dt"].abs() * 0.2
    return o, kw, n(B, L, D).to(t), n(B, D, N)


def _ref(o, kw, lengths=None, dy=None, dfinal=None, magnitude=False):
    return O.selective_scan_ref(o["x"], o["dt"], o["A"], o["Bm"], o["Cm"], o["D"], o["z"], o["init_state"], lengths=lengths, dy=dy,
                                dfinal=dfinal, magnitude=magnitude, **kw)


def _tokens(o, kw, L):
    s = o["dt"].float() + (kw["dt_bias"] if "dt_bias" in kw else 0.0)
    s = torch.nn.functional.softplus(s) if kw["dt_softplus"] else s
    return L * (1 + 1.5 * (s.abs().amax((0, 1)) * o["A"].abs().amax(1)).max().item())


def assert_near(name, got, ref, mag, tokens, terms):
    half = torch.finfo(got.dtype).eps / 2
    g = got.detach().double().cpu().reshape(ref.shape)
    assert torch.isfinite(g).all(), f"{name}: not finite"
    tol = half * ref.abs() + ((2 * tokens + 16) * 2.0 ** -22 + terms * 2.0 ** -24) * mag * (1 + half) + 1e-37
    over = ((g - ref).abs() - tol).max().item()
    assert over <= 0, f"{name}: {over:.3e} over the bound, largest error {(g - ref).abs().max().item():.3e}"


SHAPES = [   # B, L, D, N, G
    (1, 1, 1, 1, 1), (2, 1, 40, 16, 1), (1, 15, 33, 16, 1), (2, 16, 64, 16, 2), (3, 17, 100, 12, 2), (1, 130, 96, 4, 3), (2, 65, 31, 8, 1),
    (1, 200, 48, 32, 2), (2, 37, 40, 64, 1), (1, 300, 8, 16, 1), (40, 33, 256, 16, 1), (1, 67, 70, 23, 1), (2, 50, 34, 3, 2), (1, 31, 17, 61, 1)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,L,D,N,G", SHAPES)
def test_scan_and_gradients(lib, dtype, B, L, D, N, G):
    from trading_bot_0_b200 import selective as S
    full = (L + D) % 2 == 0
    o, kw, dy, dfin = _operands(B, L, D, N, G, dtype, gate=full, bias=full or N == 16, skip=D != 33, init=L != 16)
    T_ = _tokens(o, kw, L)
    ref, mag = (_ref(o, kw, dy=dy, dfinal=dfin, magnitude=m) for m in (False, True))
    dev = {k: None if v is None else v.to(DEV) for k, v in o.items()}
    kd = {k: v.to(DEV) if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    a = (dev["x"], dev["dt"], dev["A"], dev["Bm"], dev["Cm"], dev["D"], dev["z"], dev["init_state"])
    y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
    assert_near("y", y, ref["y"], mag["y"], T_, N)
    assert_near("final_state", fin, ref["final_state"], mag["final_state"], T_, 0)
    terms = dict(dx=N, ddt=N, dz=N, dA=B * L, dD=B * L, ddt_bias=B * L + N, dB=D, dC=D, dinit=0)
    g = S.selective_scan_backward(dy.to(DEV), *a, dfin.to(DEV), workspace=ws, **kd)
    again = S.selective_scan_backward(dy.to(DEV), *a, dfin.to(DEV), **kd)     # the states computed again
    want = {"dx", "ddt", "dA", "dB", "dC"} | ({"dz"} if o["z"] is not None else set()) | ({"dD"} if o["D"] is not None else set()) | \
        ({"dinit"} if o["init_state"] is not None else set()) | ({"ddt_bias"} if "dt_bias" in kw else set())
    assert set(g) == set(again) == want
    for k in sorted(want):
        assert_near(k, g[k], ref[k], mag[k], T_, terms[k])
        assert torch.equal(g[k], again[k]), k


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,L,D,N", [(6, 50, 40, 16), (6, 300, 24, 8), (6, 16, 64, 32)])
def test_lengths(lib, dtype, B, L, D, N):
    """Rows of length 0, 1, on and off tile borders, full and past the end (taken as full); NaN and infinities behind them."""
    from trading_bot_0_b200 import selective as S
    o, kw, dy, dfin = _operands(B, L, D, N, 1, dtype, gate=True, bias=True, skip=True, init=True)
    T_ = _tokens(o, kw, L)
    lengths = torch.tensor([0, 1, 16, min(33, L), L, L + 7], dtype=torch.int32)
    ref, mag = (_ref(o, kw, lengths, dy, dfin, m) for m in (False, True))
    dead = torch.arange(L)[None, :] >= lengths[:, None]
    bad = {k: o[k].clone() for k in ("x", "dt", "Bm", "Cm", "z")}
    bad["dy"] = dy.clone()
    for i, t in enumerate(bad.values()):
        t[dead] = [float("nan"), float("inf"), -float("inf")][i % 3]
    dev = {k: (bad.get(k, v)).to(DEV) for k, v in o.items()}
    kd = dict(dt_bias=kw["dt_bias"].to(DEV), dt_softplus=True, lengths=lengths.to(DEV))
    a = (dev["x"], dev["dt"], dev["A"], dev["Bm"], dev["Cm"], dev["D"], dev["z"], dev["init_state"])
    y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
    assert_near("y", y, ref["y"], mag["y"], T_, N)
    assert_near("final_state", fin, ref["final_state"], mag["final_state"], T_, 0)
    assert torch.equal(fin[0].cpu(), o["init_state"][0])
    g = S.selective_scan_backward(bad["dy"].to(DEV), *a, dfin.to(DEV), workspace=ws, **kd)
    terms = dict(dx=N, ddt=N, dz=N, dA=B * L, dD=B * L, ddt_bias=B * L + N, dB=D, dC=D, dinit=0)
    for k in g:
        assert_near(k, g[k], ref[k], mag[k], T_, terms[k])
    for k in ("dx", "ddt", "dz", "dB", "dC"):
        assert (g[k][dead.to(DEV)] == 0).all(), k


def test_strided_operands(lib):
    """x, z from one projection's halves, dt, B and C from another's odd columns, dy a slice; rows of other batch strides."""
    from trading_bot_0_b200 import selective as S
    B, L, D, N = 3, 45, 37, 7
    g = torch.Generator().manual_seed(9)
    xz = torch.randn(B, L, 2 * D + 5, generator=g).bfloat16()
    dbc = torch.randn(B + 1, L + 2, D + 2 * N + 3, generator=g).bfloat16()[:B, 1:L + 1]
    big = torch.randn(B, 2 * L, D, generator=g).bfloat16()
    o = dict(x=xz[..., 1:D + 1], z=xz[..., D + 3:2 * D + 3], dt=dbc[..., :D], Bm=dbc[..., D + 1:D + 1 + N], Cm=dbc[..., D + N + 2:D + 2 * N + 2],
             A=-torch.rand(D, N, generator=g) - 0.1, D=torch.randn(D, generator=g), init_state=None)
    dy, kw = big[:, ::2], dict(dt_bias=0.5 * torch.randn(D, generator=g) - 2.5, dt_softplus=True)
    T_ = _tokens(o, kw, L)
    ref, mag = (_ref(o, kw, dy=dy, magnitude=m) for m in (False, True))
    xzd, dbcd, bigd = xz.to(DEV), torch.cat([dbc, dbc[:1]]).to(DEV), big.to(DEV)
    dbcd = torch.nn.functional.pad(dbcd, (0, 4))[:B]
    dev = dict(x=xzd[..., 1:D + 1], z=xzd[..., D + 3:2 * D + 3], dt=dbcd[..., :D], Bm=dbcd[..., D + 1:D + 1 + N], Cm=dbcd[..., D + N + 2:D + 2 * N + 2])
    a = (dev["x"], dev["dt"], o["A"].to(DEV), dev["Bm"], dev["Cm"], o["D"].to(DEV), dev["z"], None)
    kd = dict(dt_bias=kw["dt_bias"].to(DEV), dt_softplus=True)
    y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
    assert_near("y", y, ref["y"], mag["y"], T_, N)
    grads = S.selective_scan_backward(bigd[:, ::2], *a, workspace=ws, **kd)
    for k, terms in dict(dx=N, ddt=N, dz=N, dA=B * L, dD=B * L, ddt_bias=B * L + N, dB=D, dC=D).items():
        assert_near(k, grads[k], ref[k].reshape(grads[k].shape), mag[k].reshape(grads[k].shape), T_, terms)


def test_gradients_against_differences(lib):
    """Directional derivatives against central differences of the forward.  The bound: the fp32 error of the two losses over the step
    (2^-22 (2 tokens + 16) of the sum of magnitudes, twice, over 2 eps) and the difference formula's own error, taken from the 64-bit
    recurrence along the same direction."""
    from trading_bot_0_b200 import selective as S
    B, L, D, N = 2, 37, 40, 16
    o, kw, dy, dfin = _operands(B, L, D, N, 2, "fp32", gate=True, bias=True, skip=True, init=True)
    T_ = _tokens(o, kw, L)
    leaves = ["x", "dt", "A", "Bm", "Cm", "D", "z", "init_state"]
    gen = torch.Generator().manual_seed(1)
    dev = {k: o[k].to(DEV).requires_grad_() for k in leaves}
    bias = kw["dt_bias"].to(DEV).requires_grad_()
    y, fin = S.selective_scan(*(dev[k] for k in leaves), dt_bias=bias, dt_softplus=True)
    grads = torch.autograd.grad([y, fin], [dev[k] for k in leaves] + [bias], [dy.to(DEV), dfin.to(DEV)])

    def loss64(vals, b):
        r = O.selective_scan_ref(*(vals[k] for k in leaves), dt_bias=b, dt_softplus=True)
        return (r["y"] * dy).sum() + (r["final_state"] * dfin).sum()
    mag = _ref(o, kw, magnitude=True)
    size = ((mag["y"] * dy.abs()).sum() + (mag["final_state"] * dfin.abs()).sum()).item()
    exact = _ref(o, kw, dy=dy, dfinal=dfin)
    names = dict(x="dx", dt="ddt", A="dA", Bm="dB", Cm="dC", D="dD", z="dz", init_state="dinit")
    eps = 2.0 ** -7
    for i, k in enumerate(leaves + ["dt_bias"]):
        e = exact[names.get(k, "ddt_bias")].reshape((o[k] if k in o else kw["dt_bias"]).shape)
        v = torch.rand(e.shape, generator=gen) * torch.sign(e).float() * (0.05 if k == "A" else 1.0)   # uphill: the terms do not cancel
        ends, ends64 = [], []
        for sgn in (1, -1):
            vals = dict(o)
            b = kw["dt_bias"]
            if k == "dt_bias":
                b = b + sgn * eps * v
            else:
                vals[k] = o[k] + sgn * eps * v
            yy, ff, _ = S.selective_scan_forward(*(vals[n].to(DEV) for n in leaves), dt_bias=b.to(DEV), dt_softplus=True)
            ends.append(((yy.double().cpu() * dy).sum() + (ff.double().cpu() * dfin).sum()).item())
            ends64.append(loss64(vals, b).item())
        num = (ends[0] - ends[1]) / (2 * eps)
        ana = (grads[i].double().cpu() * v).sum().item()
        formula = abs((ends64[0] - ends64[1]) / (2 * eps) - (e * v).sum().item())
        tol = 2 * (2 * T_ + 16) * 2.0 ** -22 * size / (2 * eps) * 1.5 + formula
        assert abs(num - ana) <= tol, f"{k}: {num} against {ana}, bound {tol}"


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("S_,D,N,G", [(1, 1, 1, 1), (3, 40, 16, 1), (5, 33, 12, 3), (2, 64, 64, 1), (300, 17, 4, 1), (4, 24, 32, 2), (7, 10, 50, 1)])
def test_step_is_a_scan_of_one_token(lib, dtype, S_, D, N, G):
    from trading_bot_0_b200 import selective as S
    o, kw, _, _ = _operands(S_, 1, D, N, G, dtype, gate=D != 33, bias=True, skip=D != 64, init=True)
    T_ = _tokens(o, kw, 1)
    ref, mag = (_ref(o, kw, magnitude=m) for m in (False, True))
    dev = {k: None if v is None else v.to(DEV) for k, v in o.items()}
    st = dev["init_state"].clone()
    one = lambda k: None if dev[k] is None else dev[k][:, 0]
    y = S.selective_step(st, one("x"), one("dt"), dev["A"], one("Bm"), one("Cm"), dev["D"], one("z"), dt_bias=kw["dt_bias"].to(DEV), dt_softplus=True)
    assert_near("y", y, ref["y"][:, 0], mag["y"][:, 0], T_, N)
    assert_near("state", st, ref["final_state"], mag["final_state"], T_, 0)
    # into the caller's rows, others left alone; the state one value off a 16-byte boundary
    room = torch.full((S_, D + 3), 7.0, dtype=TD[dtype], device=DEV)
    flat = torch.zeros(st.numel() + 1, device=DEV)
    odd = flat[1:].view(st.shape)
    odd.copy_(dev["init_state"])
    S.selective_step(odd, one("x"), one("dt"), dev["A"], one("Bm"), one("Cm"), dev["D"], one("z"), y=room[:, :D], dt_bias=kw["dt_bias"].to(DEV),
                     dt_softplus=True)
    assert torch.equal(room[:, :D], y) and (room[:, D:] == 7).all() and torch.equal(odd, st)


def test_prompt_then_tokens(lib):
    """A prompt's final state goes on token by token to what the whole sequence gives; a scan cut in two likewise."""
    from trading_bot_0_b200 import selective as S
    B, L, D, N, cut = 2, 90, 64, 16, 71
    o, kw, _, _ = _operands(B, L, D, N, 1, "fp32", gate=True, bias=True, skip=True, init=False)
    T_ = _tokens(o, kw, L)
    d = {k: None if v is None else v.to(DEV) for k, v in o.items()}
    kd = dict(dt_bias=kw["dt_bias"].to(DEV), dt_softplus=True)
    part = lambda a, b: (d["x"][:, a:b], d["dt"][:, a:b], d["A"], d["Bm"][:, a:b], d["Cm"][:, a:b], d["D"], d["z"][:, a:b])
    mag = _ref(o, kw, magnitude=True)
    ref = _ref(o, kw)
    y1, st, _ = S.selective_scan_forward(*part(0, cut), **kd)
    y2, fin, _ = S.selective_scan_forward(*part(cut, L), st, **kd)
    assert_near("y", torch.cat([y1, y2], 1), ref["y"], mag["y"], T_, N)
    assert_near("final", fin, ref["final_state"], mag["final_state"], T_, 0)
    for t in range(cut, L):
        y = S.selective_step(st, d["x"][:, t], d["dt"][:, t], d["A"], d["Bm"][:, t], d["Cm"][:, t], d["D"], d["z"][:, t], **kd)
        assert_near(f"y[{t}]", y, ref["y"][:, t], mag["y"][:, t], T_, N)
    assert_near("final", st, ref["final_state"], mag["final_state"], T_, 0)


def test_parts_and_streams_and_graph(lib):
    """One long sequence (cut into parts over the SMs): twice the same bits, on a side stream and from a graph replayed on new inputs."""
    from trading_bot_0_b200 import selective as S
    B, L, D, N = 1, 1500, 64, 16
    o, kw, dy, dfin = _operands(B, L, D, N, 1, "bf16", gate=True, bias=True, skip=True, init=True)
    T_ = _tokens(o, kw, L)
    d = {k: v.to(DEV) for k, v in o.items()}
    kd = dict(dt_bias=kw["dt_bias"].to(DEV), dt_softplus=True)
    a = (d["x"], d["dt"], d["A"], d["Bm"], d["Cm"], d["D"], d["z"], d["init_state"])
    dyd, dfd = dy.to(DEV), dfin.to(DEV)

    def both():
        y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
        g = S.selective_scan_backward(dyd, *a, dfd, workspace=ws, **kd)
        return [y, fin] + [g[k] for k in sorted(g)]
    want = both()
    ref, mag = (_ref(o, kw, dy=dy, dfinal=dfin, magnitude=m) for m in (False, True))
    assert_near("y", want[0], ref["y"], mag["y"], T_, N)
    g = dict(zip(sorted(["dx", "ddt", "dA", "dB", "dC", "dD", "dz", "dinit", "ddt_bias"]), want[2:]))
    for k, terms in dict(dx=N, ddt=N, dz=N, dA=B * L, dD=B * L, ddt_bias=B * L + N, dB=D, dC=D, dinit=0).items():
        assert_near(k, g[k], ref[k], mag[k], T_, terms)
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        there = both()
    torch.cuda.current_stream(DEV).wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(want, there))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = both()
    d["x"].copy_(d["x"].flip(1))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(both(), held))
    assert not torch.equal(held[0], want[0])


def test_extreme_values(lib):
    """Step sizes of 0 and of thousands (states kept, states forgotten), decays of zero, a bias far on either side."""
    from trading_bot_0_b200 import selective as S
    B, L, D, N = 1, 20, 32, 16
    o, kw, dy, dfin = _operands(B, L, D, N, 1, "fp32", gate=True, bias=True, skip=True, init=True)
    o["A"][:8] = 0.0
    kw["dt_bias"][8:16] = -110.0     # softplus underflows: nothing is added, nothing forgotten
    kw["dt_bias"][16:24] = 20.0      # everything is forgotten in one token
    o["z"][:, ::3] = -200.0
    o["z"][:, 1::3] = 200.0
    T_ = _tokens(o, kw, L)
    ref, mag = (_ref(o, kw, dy=dy, dfinal=dfin, magnitude=m) for m in (False, True))
    d = {k: v.to(DEV) for k, v in o.items()}
    a = (d["x"], d["dt"], d["A"], d["Bm"], d["Cm"], d["D"], d["z"], d["init_state"])
    kd = dict(dt_bias=kw["dt_bias"].to(DEV), dt_softplus=True)
    y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
    assert_near("y", y, ref["y"], mag["y"], T_, N)
    assert_near("final", fin, ref["final_state"], mag["final_state"], T_, 0)
    g = S.selective_scan_backward(dy.to(DEV), *a, dfin.to(DEV), workspace=ws, **kd)
    for k, terms in dict(dx=N, ddt=N, dz=N, dA=B * L, dD=B * L, ddt_bias=B * L + N, dB=D, dC=D, dinit=0).items():
        assert_near(k, g[k], ref[k], mag[k], T_, terms)


def test_operands_that_do_not_fit_are_refused(lib):
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import selective as S
    B, L, D, N = 2, 8, 16, 8
    o, kw, dy, _ = _operands(B, L, D, N, 1, "bf16", gate=True, bias=True, skip=True, init=True)
    d = {k: v.to(DEV) for k, v in o.items()}
    bias = kw["dt_bias"].to(DEV)
    base = dict(x=d["x"], dt=d["dt"], A=d["A"], Bm=d["Bm"], Cm=d["Cm"], D=d["D"], z=d["z"], init_state=d["init_state"], dt_bias=bias,
                dt_softplus=True)
    lens = torch.full((B,), L, dtype=torch.int32, device=DEV)
    for kwargs in (dict(x=d["x"].cpu()), dict(x=d["x"].half()), dict(x=d["x"][0]), dict(dt=d["dt"][:, :-1]), dict(dt=d["dt"].float()),
                   dict(A=d["A"].double()), dict(A=d["A"][:-1]), dict(A=d["A"].t().contiguous().t()), dict(Bm=d["Bm"][..., :-1]),
                   dict(Bm=d["Bm"].expand(B, L, 1, N)[:, :1].expand(B, L, 1, N)), dict(Cm=d["Cm"][:, :, 0]), dict(D=d["D"].bfloat16()),
                   dict(z=d["z"].transpose(1, 2).contiguous().transpose(1, 2)), dict(init_state=d["init_state"][:1]), dict(dt_bias=bias[:-1]),
                   dict(lengths=lens.long()), dict(lengths=lens.cpu()), dict(lengths=lens[:1]),
                   dict(Bm=torch.zeros(B, L, 3, N, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(ValueError):
            S.selective_scan_forward(**{**base, **kwargs})
    with pytest.raises(T._lib.SsdError, match="dstate"):
        S.selective_scan_forward(**{**base, "A": torch.zeros(D, 65, device=DEV), "Bm": torch.zeros(B, L, 65, dtype=torch.bfloat16, device=DEV),
                                    "Cm": torch.zeros(B, L, 65, dtype=torch.bfloat16, device=DEV), "init_state": None})
    with pytest.raises(T._lib.SsdError, match="positive"):
        S.selective_scan_forward(**{**base, **{k: base[k][:, :0] for k in ("x", "dt", "Bm", "Cm", "z")}})
    y, fin, ws = S.selective_scan_forward(**base)
    with pytest.raises(T._lib.SsdError, match="too small"):      # a forward-sized workspace keeps nothing for a backward
        S.selective_scan_backward(dy.to(DEV), **base, workspace=ws)
    with pytest.raises(ValueError, match="state"):
        S.selective_step(d["init_state"].bfloat16(), d["x"][:, 0], d["dt"][:, 0], d["A"], d["Bm"][:, 0], d["Cm"][:, 0])
    with pytest.raises(ValueError, match="y"):
        S.selective_step(d["init_state"], d["x"][:, 0], d["dt"][:, 0], d["A"], d["Bm"][:, 0], d["Cm"][:, 0], y=torch.empty(B, D, device=DEV))
