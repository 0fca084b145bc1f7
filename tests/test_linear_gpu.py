"""The projection with its epilogue and its gradients against 64 bits.

Tolerances: half a step of the storage type on the result, and fp32 rounding of the sums: 2^-23 per term (product and addition, the
tensor cores may cut instead of round) relative to the sum of the terms' magnitudes, taken through the activation with its largest slope
around the value; 2^-20 for the activation's own functions.  The backward of an activation reads `pre`, off by its sum's rounding, through
act' (so by at most the largest |act''| times that), and writes dpre in the storage type, half a step off; both go into the gradients'
sums with the magnitudes of the other factor."""
import pytest
import torch

from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {"fp32": torch.float32, "bf16": torch.bfloat16}
dev = lambda v: None if v is None else v.to(DEV)

SHAPES = [   # M, K, N
    (1, 1, 1), (1, 64, 64), (2, 8, 24), (3, 100, 131), (4, 768, 320), (7, 264, 72), (8, 512, 136), (9, 64, 40), (16, 1536, 128), (33, 72, 264), (64, 256, 520),
    (65, 136, 100), (127, 40, 257), (128, 64, 256), (129, 128, 8), (200, 200, 200), (300, 1000, 96), (513, 320, 776), (1000, 24, 136), (1, 2048, 2056)]


def operands(M, K, N, dtype, bias, residual, seed=3):
    g = torch.Generator().manual_seed(seed + M + 5 * K + 11 * N)
    n = lambda *s: torch.randn(*s, generator=g).to(TD[dtype])
    return n(M, K), (n(N, K).float() / K ** 0.5).to(TD[dtype]), n(N) if bias else None, n(M, N) if residual else None, n(M, N)


def check_forward(out, pre, r, K, act):
    half = torch.finfo(out.dtype).eps / 2
    off = K * 2.0 ** -23 * r["pre_mag"]
    near = lambda s: O.dact_ref(r["pre"] + s * off, act).abs()
    slope = torch.maximum(near(1.0), near(-1.0)) + (2 * off if act == "relu2" else off)
    tol = half * r["out"].abs() + (off * slope + 2.0 ** -20 * (r["out"].abs() + r["out_mag"])) * (1 + half) + 1e-37
    err = (out.double().cpu().reshape(r["out"].shape) - r["out"]).abs()
    assert torch.isfinite(out).all() and (err <= tol).all(), f"out: {(err - tol).max().item():.3e} over the bound"
    if pre is not None:
        err, tol = (pre.double().cpu().reshape(r["pre"].shape) - r["pre"]).abs(), 2.0 ** -24 * r["pre"].abs() + off
        assert (err <= tol).all(), f"pre: {(err - tol).max().item():.3e} over the bound"


def check_backward(got, r, x, w, act, dtype):
    half = torch.finfo(TD[dtype]).eps / 2
    x, w = x.double().reshape(-1, x.shape[-1]), w.double()
    M, N = r["g"].shape
    curve = {"none": 0.0, "silu": 0.5, "softplus": 0.25, "relu2": 2.0}[act]      # largest |act''|
    pre_off = (x.shape[1] + 2) * 2.0 ** -23 * r["pre_mag"]
    doff = r["g"].abs() * (curve * pre_off * (1 + half) + 2.0 ** -20) + (half * r["dpre"].abs() if act != "none" else 0)
    gm = r["dpre"].abs() + doff
    for name, ref, off, terms, mag in (("dx", r["dx"], doff @ w.abs(), N, gm @ w.abs()), ("dweight", r["dweight"], doff.t() @ x.abs(), M, gm.t() @ x.abs()),
                                       ("dbias", r["dbias"], doff.sum(0), M, gm.sum(0))):
        if got.get(name) is None:
            continue
        g = got[name].double().cpu().reshape(ref.shape)
        tol = half * ref.abs() + (off + terms * 2.0 ** -23 * mag) * (1 + half) + 1e-37
        assert torch.isfinite(g).all() and ((g - ref).abs() <= tol).all(), f"{name}: {((g - ref).abs() - tol).max().item():.3e} over the bound"


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("i", range(len(SHAPES)), ids=["x".join(map(str, s)) for s in SHAPES])
def test_forward_and_backward(lib, dtype, i):
    from trading_bot_0_b200 import linear as LN
    M, K, N = SHAPES[i]
    act, bias, res = ("none", "silu", "softplus", "relu2")[i % 4], i % 3 != 0, i % 5 < 3
    x, w, b, r, dout = operands(M, K, N, dtype, bias, res)
    ref = O.linear_ref(x, w, b, r, act=act, dout=dout)
    out, pre = LN.linear_forward(dev(x), dev(w), dev(b), dev(r), activation=act, for_backward=True)
    check_forward(out, pre, ref, K, act)
    assert torch.equal(LN.linear_forward(dev(x), dev(w), dev(b), dev(r), activation=act)[0], out)
    dx, dw, db = LN.linear_backward(dev(dout), dev(x), dev(w), pre, activation=act, bias=bias)
    check_backward(dict(dx=dx, dweight=dw, dbias=db), ref, x, w, act, dtype)
    again = LN.linear_backward(dev(dout), dev(x), dev(w), pre, activation=act, bias=bias)
    assert all(p is q or torch.equal(p, q) for p, q in zip((dx, dw, db), again))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("act", ["none", "silu", "softplus", "relu2"])
@pytest.mark.parametrize("M,K,N", [(5, 64, 48), (150, 80, 264)])
def test_every_epilogue(lib, dtype, act, M, K, N):
    from trading_bot_0_b200 import linear as LN
    for bias in (False, True):
        for res in (False, True):
            x, w, b, r, dout = operands(M, K, N, dtype, bias, res)
            x = x * 4                                    # wide pre-activations: both ends of the functions
            ref = O.linear_ref(x, w, b, r, act=act, dout=dout)
            out, pre = LN.linear_forward(dev(x), dev(w), dev(b), dev(r), activation=act, for_backward=True)
            check_forward(out, pre, ref, K, act)
            dx, dw, db = LN.linear_backward(dev(dout), dev(x), dev(w), pre, activation=act, bias=bias)
            check_backward(dict(dx=dx, dweight=dw, dbias=db), ref, x, w, act, dtype)


@pytest.mark.parametrize("M", [3, 40, 200])
@pytest.mark.parametrize("shift", [0, 1, 8])
def test_strides_and_alignment(lib, M, shift):
    """Rows of x, residual and dout in wider ones, starting on 16 bytes and off them; a leading batch dim; the caller's out."""
    from trading_bot_0_b200 import linear as LN
    K, N = 72, 136
    x, w, b, r, dout = operands(M, K, N, "bf16", True, True)
    def wide(t):
        o = torch.full((M, t.shape[1] + 24), 9.0, dtype=t.dtype, device=DEV)[:, shift:shift + t.shape[1]]
        return o.copy_(dev(t))
    ref = O.linear_ref(x, w, b, r, act="silu", dout=dout)
    out, pre = LN.linear_forward(wide(x), dev(w), dev(b), wide(r), activation="silu", for_backward=True)
    check_forward(out, pre, ref, K, "silu")
    dx, dw, db = LN.linear_backward(wide(dout), wide(x), dev(w), pre, activation="silu")
    check_backward(dict(dx=dx, dweight=dw, dbias=db), ref, x, w, "silu", "bf16")
    three = dev(x).view(1, M, K)
    mine = torch.empty(1, M, N, dtype=torch.bfloat16, device=DEV)
    o3, _ = LN.linear_forward(three, dev(w), dev(b), dev(r).view(1, M, N), activation="silu", out=mine)
    assert o3 is mine or o3.data_ptr() == mine.data_ptr()
    check_forward(o3, None, ref, K, "silu")
    weight_off = torch.empty(N * K + 1, dtype=torch.bfloat16, device=DEV)[1:].view(N, K).copy_(dev(w))
    check_forward(LN.linear_forward(dev(x), weight_off, dev(b), dev(r), activation="silu")[0], None, ref, K, "silu")


def test_autograd_takes_what_is_needed(lib):
    from trading_bot_0_b200 import linear as LN
    x, w, b, r, dout = (dev(v) for v in operands(50, 64, 96, "bf16", True, True))
    ls = [v.clone().requires_grad_() for v in (x, w, b, r)]
    out = LN.linear(*ls, activation="relu2")
    g = torch.autograd.grad(out, ls, dout)
    _, pre = LN.linear_forward(x, w, b, r, activation="relu2", for_backward=True)
    want = LN.linear_backward(dout, x, w, pre, activation="relu2")
    assert all(torch.equal(p, q) for p, q in zip(g, (*want, dout)))
    frozen = LN.linear(x, w, ls[2], r, activation="relu2")
    assert torch.equal(torch.autograd.grad(frozen, ls[2], dout)[0], want[2])
    total = LN.linear(ls[0], w).sum()                   # an expanded gradient
    ones = LN.linear_backward(torch.ones_like(dout), x, w, bias=False, want_dweight=False)[0]
    assert torch.equal(torch.autograd.grad(total, ls[0])[0], ones)
    assert not LN.linear(x, w).requires_grad


def test_gradients_against_differences(lib):
    """fp32: central differences along random directions; bound as in the forward's test (rounding over the step) plus the formula's own
    error from 64 bits."""
    from trading_bot_0_b200 import linear as LN
    M, K, N, eps = 40, 33, 50, 2.0 ** -7
    x, w, b, r, dout = operands(M, K, N, "fp32", True, True)
    for act in ("silu", "softplus", "relu2"):
        ref = O.linear_ref(x, w, b, r, act=act, dout=dout)
        _, pre = LN.linear_forward(dev(x), dev(w), dev(b), dev(r), activation=act, for_backward=True)
        grads = LN.linear_backward(dev(dout), dev(x), dev(w), pre, activation=act)
        slope = 1.1 if act != "relu2" else 2.0 * ref["pre_mag"].max().item()
        size = ((K * 2.0 ** -23 * slope * ref["pre_mag"] + 2.0 ** -20 * (ref["out"].abs() + ref["out_mag"])) * dout.abs()).sum().item()
        g = torch.Generator().manual_seed(4)
        for i, name in enumerate(("dx", "dweight", "dbias")):
            v, ends, ends64 = torch.randn((x, w, b)[i].shape, generator=g), [], []
            for s in (1, -1):
                q = [x, w, b]
                q[i] = q[i] + s * eps * v
                ends.append((LN.linear_forward(*(dev(t) for t in q), dev(r), activation=act)[0].double().cpu() * dout).sum().item())
                ends64.append((O.linear_ref(*q, r, act=act)["out"] * dout).sum().item())
            num, ana = (ends[0] - ends[1]) / (2 * eps), (grads[i].double().cpu() * v).sum().item()
            tol = 1.5 * size / eps + abs((ends64[0] - ends64[1]) / (2 * eps) - (ref[name] * v).sum().item())
            assert abs(num - ana) <= tol, (act, name, num, ana, tol)


@pytest.mark.parametrize("M", [5, 100, 700])
def test_residual_in_place(lib, M):
    """The residual's own memory as the output, for the kernels of few, some and many rows."""
    from trading_bot_0_b200 import linear as LN
    x, w, b, r, _ = (dev(v) for v in operands(M, 192, 520, "bf16", True, True))
    want = LN.linear_forward(x, w, b, r, activation="silu")[0]
    mine = r.clone()
    assert torch.equal(LN.linear_forward(x, w, b, mine, activation="silu", out=mine)[0], want)


@pytest.mark.parametrize("M", [2, 24, 300])
def test_graph_and_stream(lib, M):
    from trading_bot_0_b200 import linear as LN
    x, w, b, r, dout = (dev(v) for v in operands(M, 128, 200, "bf16", True, True))

    def both():
        out, pre = LN.linear_forward(x, w, b, r, activation="silu", for_backward=True)
        return [out, *LN.linear_backward(dout, x, w, pre, activation="silu")]
    both()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = both()
    with torch.cuda.graph(other := torch.cuda.CUDAGraph(), stream=side):
        held2 = both()
    x.mul_(-0.5)
    graph.replay()
    other.replay()
    torch.cuda.synchronize()
    want = both()
    assert all(torch.equal(p, q) for p, q in zip(held, want)) and all(torch.equal(p, q) for p, q in zip(held2, want))


def test_operands_that_do_not_fit_are_refused(lib):
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import linear as LN
    x, w, b, r, dout = (dev(v) for v in operands(6, 32, 40, "bf16", True, True))
    for args, kw in (((x.cpu(), w), {}), ((x.half(), w), {}), ((x, w.float()), {}), ((x, w.cpu()), {}), ((x, w.t()), {}), ((x[:, :-1], w), {}),
                     ((x, w, b[:-1]), {}), ((x, w, b.float()), {}), ((x, w, b, r[:-1]), {}), ((x, w, b, r.float()), {}), ((x, w, b, r[:1]), {}),
                     ((x, w), dict(activation="tanh")), ((x, w), dict(out=torch.empty(5, 40, dtype=torch.bfloat16, device=DEV))),
                     ((x, w), dict(out=torch.empty(6, 40, device=DEV)))):
        with pytest.raises(ValueError):
            LN.linear_forward(*args, **kw)
    with pytest.raises(ValueError, match="overlaps"):
        LN.linear_forward(x, torch.zeros(32, 32, dtype=torch.bfloat16, device=DEV), out=x)
    inplace = r.clone()                                  # (the residual may be the output)
    assert torch.equal(LN.linear_forward(x, w, b, inplace, out=inplace)[0], LN.linear_forward(x, w, b, r)[0])
    with pytest.raises(ValueError, match="pre"):
        LN.linear_backward(dout, x, w, activation="silu")
    with pytest.raises(ValueError):
        LN.linear_backward(dout[:, :-1], x, w)
    with pytest.raises(T._lib.SsdError, match="positive"):
        LN.linear_forward(x[:0], w)


def test_output_that_overlaps_a_part_of_the_residual_is_refused(lib):
    """Blocks would read values of the residual that others have written; refused before any launch."""
    from trading_bot_0_b200 import linear as LN
    x, w, b, _, _ = (dev(v) for v in operands(6, 32, 40, "bf16", True, True))
    buf = torch.zeros(13 * 40, dtype=torch.bfloat16, device=DEV)
    out = buf[:240].view(6, 40)
    for r in (buf[40:280].view(6, 40), buf[8:248].view(6, 40), buf[:480].view(6, 80)[:, :40]):   # rows later, values later, rows further apart
        with pytest.raises(ValueError, match="residual"):
            LN.linear_forward(x, w, b, r, out=out)
    with pytest.raises(ValueError, match="bias"):
        LN.linear_forward(x, w, buf[200:240], out=out)
    apart = buf[240:480].view(6, 40)                      # directly behind it: nothing shared
    assert torch.equal(LN.linear_forward(x, w, b, apart, out=out)[0], LN.linear_forward(x, w, b, apart.clone())[0])
