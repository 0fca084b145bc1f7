"""The causal convolution that carries its history, its gradients and its single step against the 64-bit restatement.

Tolerances: half a step of the storage type, and relative to the sum of the magnitudes of an output's terms 2^-24 per term; the silu's
sigmoid is within 2^-11 where the output is bf16 (of a value of at most the magnitude), and 2^-21 elsewhere and in the backward."""
import pytest
import torch

from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {"fp32": torch.float32, "bf16": torch.bfloat16}


def assert_near(name, got, ref, mag, terms, sig=2.0 ** -21):
    half = torch.finfo(got.dtype).eps / 2
    g = got.detach().double().cpu()
    assert torch.isfinite(g).all(), f"{name}: not finite"
    over = ((g - ref).abs() - (half * ref.abs() + (terms * 2.0 ** -24 + sig) * mag * (1 + half) + 1e-37)).max().item()
    assert over <= 0, f"{name}: {over:.3e} over the bound"


def _operands(B, L, C, K, dtype, bias=True, history=True):
    g = torch.Generator().manual_seed(B + 3 * L + 7 * C)
    n = lambda *s: torch.randn(*s, generator=g)
    t = TD[dtype]
    return (n(B, L, C).to(t), n(C, K) / K ** 0.5, 0.3 * n(C) if bias else None, n(B, K - 1, C).to(t) if history else None, n(B, L, C).to(t),
            n(B, K - 1, C).to(t))


dev = lambda v: None if v is None else v.to(DEV)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,L,C,K", [(1, 1, 8, 4), (2, 2, 24, 4), (3, 3, 40, 3), (2, 31, 136, 4), (2, 32, 128, 2), (2, 33, 264, 4), (1, 200, 384, 3),
                                     (5, 64, 520, 4), (3, 130, 64, 2), (1, 1100, 16, 4), (40, 67, 72, 4)])
def test_forward_and_backward(lib, dtype, B, L, C, K):
    from trading_bot_0_b200 import prepost as P
    activation, bias, history = C != 40, C != 136, L != 200
    x, w, b, h, dout, dnew = _operands(B, L, C, K, dtype, bias, history)
    ref, mag = (O.conv_carry_ref(x, w, b, h, activation=activation, dout=dout, dnew=dnew, magnitude=m) for m in (False, True))
    out, new = P.conv1d_carry_forward(dev(x), dev(w), dev(b), dev(h), activation=activation)
    fast = 2.0 ** -11 if dtype == "bf16" else 2.0 ** -21
    assert_near("out", out, ref["out"], mag["out"], K + 4, fast)
    assert torch.equal(new.double().cpu(), ref["history"])
    din, dw, db, dh = P.conv1d_carry_backward(dev(x), dev(w), dev(b), dev(h), dev(dout), dev(dnew), activation=activation)
    assert_near("din", din, ref["din"], mag["din"], 4 * K)
    assert_near("dweight", dw, ref["dweight"], mag["dweight"], B * L + 2 * K)
    assert (db is None) == (b is None) and (dh is None) == (h is None)
    if b is not None:
        assert_near("dbias", db, ref["dbias"], mag["dbias"], B * L + 2 * K)
    if h is not None:
        assert_near("dhistory", dh, ref["dhistory"], mag["dhistory"], 4 * K)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("L,C,K", [(40, 64, 4), (150, 200, 3), (2, 8, 4)])
def test_lengths(lib, dtype, L, C, K):
    """Lengths below the window (the new history then still holds rows of the old one), zero, on tile borders and past the end; NaN
    behind them."""
    from trading_bot_0_b200 import prepost as P
    lengths = torch.tensor([0, 1, 2, min(32, L), L - 1, L, L + 3], dtype=torch.int32)
    B = len(lengths)
    x, w, b, h, dout, dnew = _operands(B, L, C, K, dtype)
    dead = torch.arange(L)[None, :] >= lengths[:, None]
    x[dead], dout[dead] = float("nan"), float("inf")
    ref, mag = (O.conv_carry_ref(x, w, b, h, lengths=lengths, dout=dout, dnew=dnew, magnitude=m) for m in (False, True))
    out, new = P.conv1d_carry_forward(dev(x), dev(w), dev(b), dev(h), lengths=dev(lengths))
    assert_near("out", out, ref["out"], mag["out"], K + 4, 2.0 ** -11 if dtype == "bf16" else 2.0 ** -21)
    assert torch.equal(new.double().cpu(), ref["history"])
    assert torch.equal(new[0].cpu(), h[0]) and (out.cpu()[dead] == 0).all()
    din, dw, db, dh = P.conv1d_carry_backward(dev(x), dev(w), dev(b), dev(h), dev(dout), dev(dnew), lengths=dev(lengths))
    assert (din.cpu()[dead] == 0).all()
    for name, got, terms in (("din", din, 4 * K), ("dhistory", dh, 4 * K), ("dweight", dw, B * L + 2 * K), ("dbias", db, B * L + 2 * K)):
        assert_near(name, got, ref[name], mag[name], terms)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_strided_rows(lib, dtype):
    """Input and gradient as channel ranges of wider rows."""
    from trading_bot_0_b200 import prepost as P
    B, L, C, K = 2, 50, 48, 4
    x, w, b, h, dout, dnew = _operands(B, L, C, K, dtype)
    wide, wide_g = (torch.zeros(B, L, C + 32, dtype=TD[dtype], device=DEV) for _ in range(2))
    wide[..., 16:16 + C], wide_g[..., 8:8 + C] = dev(x), dev(dout)
    a = P.conv1d_carry_forward(dev(x), dev(w), dev(b), dev(h))
    c = P.conv1d_carry_forward(wide[..., 16:16 + C], dev(w), dev(b), dev(h))
    assert all(torch.equal(p, q) for p, q in zip(a, c))
    a = P.conv1d_carry_backward(dev(x), dev(w), dev(b), dev(h), dev(dout), dev(dnew))
    c = P.conv1d_carry_backward(wide[..., 16:16 + C], dev(w), dev(b), dev(h), wide_g[..., 8:8 + C], dev(dnew))
    assert all(torch.equal(p, q) for p, q in zip(a, c))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("K", [2, 3, 4])
def test_pieces_and_steps_are_one_sequence(lib, dtype, K):
    """A sequence in pieces (one of them shorter than the window) and token by token gives the bits of the whole; a step leaves rows
    that are not its own alone."""
    from trading_bot_0_b200 import prepost as P
    B, L, C = 3, 41, 80
    x, w, b, h, _, _ = _operands(B, L, C, K, dtype)
    x, w, b, h = dev(x), dev(w), dev(b), dev(h)
    whole, last = P.conv1d_carry_forward(x, w, b, h)
    outs, cur = [], h
    for lo, hi in ((0, 1), (1, 3), (3, 36), (36, 41)):
        o, cur = P.conv1d_carry_forward(x[:, lo:hi], w, b, cur)
        outs.append(o)
    assert torch.equal(torch.cat(outs, 1), whole) and torch.equal(cur, last)
    st = h.clone()
    for t in range(L):
        room = torch.full((B, C + 8), 5.0, dtype=TD[dtype], device=DEV)
        o = P.conv1d_step(st, x[:, t], w, b, out=room[:, :C])
        assert torch.equal(o, whole[:, t]) and (room[:, C:] == 5).all()
    assert torch.equal(st, last)
    zero, _ = P.conv1d_carry_forward(x, w, b)
    assert torch.equal(zero, P.conv1d_carry_forward(x, w, b, torch.zeros_like(h))[0])


def test_autograd_and_differences(lib):
    """The node's gradients are those of the explicit call; directional derivatives agree with central differences of the forward (bound:
    rounding of the two sums, 2^-20 of the sum of magnitudes over the step, and the formula's own error in 64 bits)."""
    from trading_bot_0_b200 import prepost as P
    B, L, C, K = 2, 19, 24, 4
    vals = list(_operands(B, L, C, K, "fp32"))
    dout, dnew = vals[4:]
    leaves = [dev(v).requires_grad_() for v in vals[:4]]
    out, new = P.causal_conv1d_carry(*leaves)
    grads = torch.autograd.grad([out, new], leaves, [dev(dout), dev(dnew)], retain_graph=True)
    din, dw, db, dh = P.conv1d_carry_backward(*leaves, dev(dout), dev(dnew))
    assert all(torch.equal(a, b) for a, b in zip(grads, (din, dw, db, dh)))
    only = torch.autograd.grad(new, leaves[0], dev(dnew))[0]
    assert torch.equal(only[:, -(K - 1):], dev(dnew)) and (only[:, :-(K - 1)] == 0).all()
    f64 = lambda v: (lambda r: (r["out"] * dout).sum() + (r["history"] * dnew).sum())(O.conv_carry_ref(*v))
    m = O.conv_carry_ref(*vals[:4], magnitude=True)
    size = ((m["out"] * dout.abs()).sum() + (m["history"] * dnew.abs()).sum()).item()
    g = torch.Generator().manual_seed(2)
    for i in range(4):
        v, ends, ends64, eps = torch.randn(vals[i].shape, generator=g), [], [], 2.0 ** -6
        for s in (1, -1):
            q = list(vals[:4])
            q[i] = q[i] + s * eps * v
            o, h = P.conv1d_carry_forward(*(dev(t) for t in q))
            ends.append(((o.double().cpu() * dout).sum() + (h.double().cpu() * dnew).sum()).item())
            ends64.append(f64(q).item())
        num, ana = (ends[0] - ends[1]) / (2 * eps), (grads[i].double().cpu() * v).sum().item()
        ref = O.conv_carry_ref(*vals[:4], dout=dout, dnew=dnew)[("din", "dweight", "dbias", "dhistory")[i]]
        tol = 2.0 ** -20 * size / eps + abs((ends64[0] - ends64[1]) / (2 * eps) - (ref * v).sum().item())
        assert abs(num - ana) <= tol, (i, num, ana, tol)


def test_graph_on_a_side_stream(lib):
    from trading_bot_0_b200 import prepost as P
    x, w, b, h, _, _ = (dev(v) for v in _operands(2, 40, 64, 4, "bf16"))
    st = h.clone()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out, new = P.conv1d_carry_forward(x, w, b, h)
        y = P.conv1d_step(st, x[:, 0], w, b)
    x.neg_()
    st.copy_(h)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, P.conv1d_carry_forward(x, w, b, h)[0]) and torch.equal(y, out[:, 0])


def test_operands_that_do_not_fit_are_refused(lib):
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import prepost as P
    x, w, b, h, dout, dnew = (dev(v) for v in _operands(2, 20, 32, 4, "bf16"))
    lens = torch.full((2,), 20, dtype=torch.int32, device=DEV)
    for args, kw in (((x.cpu(), w, b, h), {}), ((x, w.bfloat16(), b, h), {}), ((x, w[:-8], b, h), {}), ((x, w, b[:-1], h), {}),
                     ((x, w, b, h[:, :-1]), {}), ((x, w, b, h.float()), {}), ((x, w, b, h.cpu()), {}), ((x, w, b, h[:1]), {}),
                     ((x[:, :1].expand(2, 20, 32), w, b, h), {}), ((x, w, b, h), dict(lengths=lens.long())), ((x, w, b, h), dict(lengths=lens[:1]))):
        with pytest.raises(ValueError):
            P.conv1d_carry_forward(*args, **kw)
        if args[0] is x:
            with pytest.raises(ValueError):
                P.conv1d_carry_backward(*args, dout, dnew, **kw)
    with pytest.raises(ValueError):
        P.conv1d_carry_backward(x, w, b, h, dout[:, :-1], dnew)
    with pytest.raises(ValueError):
        P.conv1d_carry_backward(x, w, b, h, dout, dnew.float())
    with pytest.raises(T._lib.SsdError, match="multiple of 8"):
        P.conv1d_carry_forward(x[..., :28].contiguous(), w[:28].contiguous(), b[:28].contiguous(), h[..., :28].contiguous())
    with pytest.raises(T._lib.SsdError, match="16"):
        P.conv1d_carry_forward(torch.zeros(2, 20, 40, dtype=torch.bfloat16, device=DEV)[..., 4:36], w, b, h)
    with pytest.raises(ValueError):
        P.conv1d_step(h[:, :-1], x[:, 0], w, b)
    with pytest.raises(ValueError):
        P.conv1d_step(h, x[:, :1], w, b)
    with pytest.raises(ValueError):
        P.conv1d_step(h, x[:, 0], w, b, out=torch.empty(2, 32, device=DEV))
