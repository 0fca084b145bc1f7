"""The layer operators' kernels for large and for odd sizes: pairs of CTAs that walk several tiles, tile rows past the first eight, big tiles
on the CUDA cores, several output features or streams to a thread, with remainders everywhere.  Against 64 bits, with the bounds of the
operators' own tests."""
import pytest
import torch

from oracle import layer_oracle as O
from tests import test_carry_gpu as TC
from tests import test_linear_gpu as TL
from tests import test_selective_gpu as TS

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {"fp32": torch.float32, "bf16": torch.bfloat16}
dev = lambda v: None if v is None else v.to(DEV)

# M, K, N, dtype, activation.  74 pairs of CTAs share the tiles of a bf16 product; the forward's:
LARGE = [
    (5000, 136, 1544, "bf16", "silu"),       # 140 tiles of 256 x 224: two to a pair, 20 tile rows; dx and dW in 3 and 10 splits
    (9000, 72, 1544, "bf16", "softplus"),    # 252 tiles: four to a pair, both accumulators and their phases go round twice; 36 tile rows
    (4104, 64, 4112, "bf16", "relu2"),       # 289 tiles of 256 x 256, all remainders; dx and dW in 4 splits
    (19000, 24, 1032, "bf16", "none"),       # 75 tile rows: the last group of eight is three
    (600, 40, 20008, "bf16", "silu"),        # few tile rows, many columns
    (2100, 40, 1300, "fp32", "silu"),        # 187 tiles of 128 x 128 on the CUDA cores
    (2600, 1288, 130, "fp32", "softplus"),   # dx on tiles of 128 x 128
    (2100, 41, 1300, "bf16", "relu2"),       # the same for bf16 rows that no tensor map takes
    (200, 2048, 131, "bf16", "silu"),        # splits whose sums no tensor map takes
    (90, 1544, 133, "bf16", "softplus"),     # the same with the weights as the tiles' rows
    (3, 64, 8200, "bf16", "silu"),           # few rows: two features to a warp, the last warps with one and none
    (8, 72, 8193, "fp32", "softplus"),
    (1, 40, 9001, "bf16", "none"),
]


@pytest.mark.parametrize("M,K,N,dtype,act", LARGE, ids=["x".join(map(str, s)) for s in LARGE])
def test_projection(lib, M, K, N, dtype, act):
    from trading_bot_0_b200 import linear as LN
    x, w, b, r, dout = TL.operands(M, K, N, dtype, True, True)
    ref = O.linear_ref(x, w, b, r, act=act, dout=dout)
    out, pre = LN.linear_forward(dev(x), dev(w), dev(b), dev(r), activation=act, for_backward=True)
    TL.check_forward(out, pre, ref, K, act)
    bare = O.linear_ref(x, w, act=act)
    TL.check_forward(LN.linear_forward(dev(x), dev(w), activation=act)[0], None, bare, K, act)     # (two boxes in turn: no pre, no residual)
    mine = dev(r).clone()
    assert torch.equal(LN.linear_forward(dev(x), dev(w), dev(b), mine, activation=act, out=mine)[0], out)
    grads = LN.linear_backward(dev(dout), dev(x), dev(w), pre, activation=act)
    TL.check_backward(dict(zip(("dx", "dweight", "dbias"), grads)), ref, x, w, act, dtype)
    again = LN.linear_backward(dev(dout), dev(x), dev(w), pre, activation=act)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("S_,D,N,G", [(4739, 20, 4, 1), (4741, 30, 8, 3), (4737, 24, 16, 1), (4738, 33, 13, 1), (4743, 18, 32, 2), (4737, 17, 23, 1), (2501, 20, 64, 1),
                                      (2503, 20, 50, 2), (1187, 256, 16, 1)])
def test_steps_of_many_streams(lib, dtype, S_, D, N, G):
    """Four streams to a thread (4736 blocks and more in one), a number that four does not divide; every number of lanes to a channel, states
    in vectors and one by one.  The same streams 37 at a time, one to a thread, give the same bits."""
    from trading_bot_0_b200 import selective as S
    o, kw, _, _ = TS._operands(S_, 1, D, N, G, dtype, gate=D != 33, bias=True, skip=D != 24, init=True)
    T_ = TS._tokens(o, kw, 1)
    ref, mag = (TS._ref(o, kw, magnitude=m) for m in (False, True))
    d = {k: dev(v) for k, v in o.items()}
    st, bias = d["init_state"].clone(), dev(kw["dt_bias"])
    one = lambda k, a, b: None if d[k] is None else d[k][a:b, 0]

    def step(state, a, b):
        return S.selective_step(state, one("x", a, b), one("dt", a, b), d["A"], one("Bm", a, b), one("Cm", a, b), d["D"], one("z", a, b), dt_bias=bias,
                                dt_softplus=True)
    y = step(st, 0, S_)
    TS.assert_near("y", y, ref["y"][:, 0], mag["y"][:, 0], T_, N)
    TS.assert_near("state", st, ref["final_state"], mag["final_state"], T_, 0)
    for a in (0, 37, S_ // 2, S_ - 37):
        few = d["init_state"][a:a + 37].clone()
        assert torch.equal(step(few, a, a + 37), y[a:a + 37]) and torch.equal(few, st[a:a + 37])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("K", [2, 3, 4])
def test_convolution_steps_of_many_streams(lib, dtype, K):
    """Four streams to a thread, a number that four does not divide."""
    from trading_bot_0_b200 import prepost as P
    C = 512
    S_ = 4 * 148 * 512 // (C * (2 if dtype == "bf16" else 4) // 16) + 3
    x, w, b, h, _, _ = TC._operands(S_, 1, C, K, dtype)
    ref, mag = (O.conv_carry_ref(x, w, b, h, magnitude=m) for m in (False, True))
    st = dev(h).clone()
    out = P.conv1d_step(st, dev(x)[:, 0], dev(w), dev(b))
    TC.assert_near("out", out, ref["out"][:, 0], mag["out"][:, 0], K + 4, 2.0 ** -21)
    assert torch.equal(st.double().cpu(), ref["history"])
    odd = torch.empty(C * K + 1, device=DEV)[1:].view(C, K).copy_(dev(w))      # weights off 16 bytes
    st2 = dev(h).clone()
    assert torch.equal(P.conv1d_step(st2, dev(x)[:, 0], odd, dev(b)), out) and torch.equal(st2, st)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("B,L,D,N,G", [(5, 260, 36, 64, 2), (5, 260, 34, 40, 1), (5, 260, 70, 16, 2), (5, 260, 66, 3, 1), (5, 260, 48, 25, 3), (300, 33, 70, 16, 1)])
def test_scans_cut_into_parts_with_lengths(lib, dtype, B, L, D, N, G):
    """Every block shape over several parts of the sequence (the last size: so many blocks that there is one), rows that end in the first
    part, on borders, in the last, and nowhere; groups whose channels end inside a block."""
    from trading_bot_0_b200 import selective as S
    o, kw, dy, dfin = TS._operands(B, L, D, N, G, dtype, gate=D != 66, bias=True, skip=D != 48, init=D != 34)
    T_ = TS._tokens(o, kw, L)
    lengths = torch.tensor([0, 7, L - 1, L, L // 2 + 3] * (B // 5), dtype=torch.int32)
    ref, mag = (TS._ref(o, kw, lengths, dy, dfin, m) for m in (False, True))
    if o["z"] is not None:
        # dz = dy y0 s (1 + z (1 - s)): the magnitude has |s (1 + z (1 - s))| as one factor, which is 0 at z = -1.278, but the two terms of the
        # slope are each rounded and carry the sigmoid's error, so its own magnitude is s (1 + |z| (1 - s))
        z = o["z"].double()
        one = 1 - torch.sigmoid(z)
        mag["dz"] = mag["dz"] * ((1 + z.abs() * one) / (1 + z * one).abs())
    d = {k: dev(v) for k, v in o.items()}
    kd = dict(dt_bias=dev(kw["dt_bias"]), dt_softplus=True, lengths=dev(lengths))
    a = (d["x"], d["dt"], d["A"], d["Bm"], d["Cm"], d["D"], d["z"], d["init_state"])
    y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
    TS.assert_near("y", y, ref["y"], mag["y"], T_, N)
    TS.assert_near("final_state", fin, ref["final_state"], mag["final_state"], T_, 0)
    g = S.selective_scan_backward(dev(dy), *a, dev(dfin), workspace=ws, **kd)
    terms = dict(dx=N, ddt=N, dz=N, dA=B * L, dD=B * L, ddt_bias=B * L + N, dB=D, dC=D, dinit=0)
    for k in g:
        TS.assert_near(k, g[k], ref[k], mag[k], T_, terms[k])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_time_major_operands(lib, dtype):
    """Operands laid out [tokens, batch, channels]: batch rows nearer than tokens.  The bits of dense ones."""
    from trading_bot_0_b200 import linear as LN, prepost as P, selective as S
    B, L, D, N = 3, 75, 136, 16
    o, kw, dy, _ = TS._operands(B, L, D, N, 1, dtype, gate=True, bias=True, skip=True, init=True)
    d = {k: dev(v) for k, v in o.items()}
    turn = lambda v: v.transpose(0, 1).contiguous().transpose(0, 1)
    kd = dict(dt_bias=dev(kw["dt_bias"]), dt_softplus=True, lengths=torch.tensor([75, 20, 64], dtype=torch.int32, device=DEV))

    def scan(f):
        a = (f(d["x"]), f(d["dt"]), d["A"], f(d["Bm"]), f(d["Cm"]), d["D"], f(d["z"]), d["init_state"])
        y, fin, ws = S.selective_scan_forward(*a, for_backward=True, **kd)
        g = S.selective_scan_backward(f(dev(dy)), *a, workspace=ws, **kd)
        return [y, fin] + [g[k] for k in sorted(g)]
    assert all(torch.equal(p, q) for p, q in zip(scan(turn), scan(lambda v: v)))
    w = torch.randn(D, 4, device=DEV)

    def conv(f):
        return [*P.conv1d_carry_forward(f(d["x"]), w, lengths=kd["lengths"]),
                *P.conv1d_carry_backward(f(d["x"]), w, None, None, f(dev(dy)), lengths=kd["lengths"])[:2]]
    assert all(torch.equal(p, q) for p, q in zip(conv(turn), conv(lambda v: v)))
    W = torch.randn(24, D, device=DEV).to(TD[dtype])
    assert torch.equal(LN.linear(turn(d["x"]), W), LN.linear(d["x"], W))


def test_layers_side_by_side_on_two_streams(lib):
    """Training steps of both mixers at the same time on two streams, several times over: the bits of one after the other.  (Tensor memory,
    shared memory and the SMs are shared; workspaces are not.)"""
    import trading_bot_0_b200 as T
    from tests.test_mixer_gpu import _mamba2, _selective
    u, p, dout = _selective("bf16", B=4, L=512, d_model=256, D=512, rank=16)
    q, kw = _mamba2("bf16", d_model=256, H=16)
    u, dout = dev(u), dev(dout)
    lp, lq = [dev(v).requires_grad_() for v in p.values()], [dev(v).requires_grad_() for v in q.values()]

    def one():
        out, _, _ = T.selective_mixer(u, **dict(zip(p, lp)), residual=u)
        return [out, *torch.autograd.grad(out, lp, dout)]

    def two():
        out, _ = T.mamba2_mixer(u, **dict(zip(q, lq)), **kw, residual=u)
        return [out, *torch.autograd.grad(out, lq, dout)]
    want = one(), two()
    torch.cuda.synchronize()
    streams = torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)
    got = [], []
    for _ in range(8):
        for s, f, keep in zip(streams, (one, two), got):
            with torch.cuda.stream(s):
                keep.append(f())
    torch.cuda.synchronize()
    for keep, ref in zip(got, want):
        for run in keep:
            assert all(torch.equal(a, b) for a, b in zip(run, ref))
