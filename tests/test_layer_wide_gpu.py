"""The layer operators where offsets pass 32 bits: tensors of more than 2^31 elements against the same rows, streams or channels alone."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
rand = lambda *s, dtype=BF: torch.randn(*s, device=DEV, dtype=dtype)


@pytest.fixture(autouse=True)
def give_back():
    yield
    torch.cuda.empty_cache()                              # tens of GB


def close(name, a, b):
    """Two ways to the same bf16 values, sums in another order: a step of the type apart at most, beside 2^-16 of the largest."""
    a, b = a.float(), b.float()
    over = ((a - b).abs() - 2.0 ** -7 * b.abs() - 2.0 ** -16 * b.abs().max()).max().item()
    assert torch.isfinite(a).all() and over <= 0, f"{name}: {over:.3e}"


def test_steps(lib):
    from trading_bot_0_b200 import prepost as P, selective as S
    n, D, N = 131080, 1024, 16
    st = rand(n, D, N, dtype=F32)
    assert st.numel() > 2 ** 31
    x, dt, B, A = rand(n, D), rand(n, D), rand(n, N), -rand(D, N, dtype=F32).abs()
    ends = [slice(0, 40), slice(n - 40, n)]
    own = [st[e].clone() for e in ends]
    y = S.selective_step(st, x, dt, A, B, B, dt_softplus=True)
    for e, s in zip(ends, own):
        assert torch.equal(S.selective_step(s, x[e], dt[e], A, B[e], B[e], dt_softplus=True), y[e]) and torch.equal(s, st[e])
    del st, x, dt, B, y, own
    n, C = 400000, 1792
    h, x, w = rand(n, 3, C), rand(n, C), rand(C, 4, dtype=F32)
    assert h.numel() > 2 ** 31
    ends = [slice(0, 40), slice(n - 40, n)]
    own = [h[e].clone() for e in ends]
    out = P.conv1d_step(h, x, w)
    for e, s in zip(ends, own):
        assert torch.equal(P.conv1d_step(s, x[e], w), out[e]) and torch.equal(s, h[e])


def test_projection(lib):
    from trading_bot_0_b200 import linear as LN
    M, K, N = 2100003, 64, 1032
    x, w, b = rand(M, K), rand(N, K) / 8, rand(N)
    out, pre = LN.linear_forward(x, w, b, activation="silu", for_backward=True)
    assert out.numel() > 2 ** 31
    ends = torch.cat([torch.arange(300), torch.arange(M - 300, M)]).to(DEV)
    some, some_pre = LN.linear_forward(x[ends], w, b, activation="silu", for_backward=True)
    assert torch.equal(out[ends], some) and torch.equal(pre[ends], some_pre)
    del out
    dout = torch.zeros(M, N, dtype=BF, device=DEV)        # the rows between have no gradient
    dout[ends] = rand(600, N)
    dx, dw, db = LN.linear_backward(dout, x, w, pre, activation="silu")
    for name, a, c in zip(("dx", "dweight", "dbias"), (dx[ends], dw, db), LN.linear_backward(dout[ends], x[ends], w, some_pre, activation="silu")):
        close(name, a, c)
    assert (dx[300:M - 300] == 0).all()


def test_scan_and_convolution(lib):
    from trading_bot_0_b200 import prepost as P, selective as S
    L, D, N = 16400, 131072, 4
    x, dt, bc, A = rand(1, L, D), rand(1, L, D), rand(1, L, N), -rand(D, N, dtype=F32).abs() - 0.1
    assert x.numel() > 2 ** 31
    dy = rand(1, L, D)
    y, fin, ws = S.selective_scan_forward(x, dt, A, bc, bc, dt_softplus=True, for_backward=True)
    g = S.selective_scan_backward(dy, x, dt, A, bc, bc, dt_softplus=True, workspace=ws)
    for e in (slice(0, 64), slice(D - 64, D)):
        y1, f1, w1 = S.selective_scan_forward(x[..., e], dt[..., e], A[e], bc, bc, dt_softplus=True, for_backward=True)
        g1 = S.selective_scan_backward(dy[..., e], x[..., e], dt[..., e], A[e], bc, bc, dt_softplus=True, workspace=w1)
        close("y", y[..., e], y1)
        close("state", fin[:, e], f1)
        for k in ("dx", "ddt"):
            close(k, g[k][..., e], g1[k])
    del y, ws, g, dt, dy
    w = rand(D, 4, dtype=F32)
    out, new = P.conv1d_carry_forward(x, w)
    din, dw, _, _ = P.conv1d_carry_backward(x, w, None, None, out)
    for e in (slice(0, 64), slice(D - 64, D)):
        o1, n1 = P.conv1d_carry_forward(x[..., e], w[e].contiguous())
        assert torch.equal(o1, out[..., e]) and torch.equal(n1, new[..., e])
        d1, dw1, _, _ = P.conv1d_carry_backward(x[..., e], w[e].contiguous(), None, None, out[..., e])
        assert torch.equal(d1, din[..., e])
        assert ((dw1 - dw[e]).abs() <= L * 2.0 ** -20 * dw1.abs().max()).all()
