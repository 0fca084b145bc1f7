"""mamba2_mixer continued: a prompt, then tokens; a sequence in pieces; gradients through the history and the state."""
import pytest
import torch

from tests._util import assert_close
from tests.test_mixer_gpu import DEV, TD, _mamba2

pytestmark = pytest.mark.gpu


def _layer(dtype, L, **size):
    p, kw = _mamba2(dtype, **size)
    g = torch.Generator().manual_seed(2)
    u = torch.randn(3, L, 64, generator=g).to(TD[dtype]).to(DEV)
    return u, {k: v.to(DEV) for k, v in p.items()}, kw


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H,P,N", [(8, 32, 64), (3, 8, 16)])     # rows of the projection on 16 bytes, and off them
@pytest.mark.parametrize("cut", [1, 2, 3, 25])                   # prompts shorter than the window, as long, longer
def test_a_prompt_then_tokens(lib, dtype, H, P, N, cut):
    """The prompt's history and state, stepped on in place, give what the whole sequence gives."""
    import trading_bot_0_b200 as T
    L = 33
    u, p, kw = _layer(dtype, L, H=H, P=P, N=N)
    more = dict(algo="fp32_cores")
    whole, final = T.mamba2_mixer(u, **p, **kw, residual=u, **more)
    out, history, state = T.mamba2_mixer(u[:, :cut], **p, **kw, residual=u[:, :cut], return_history=True, **more)
    assert_close("prompt", out, whole[:, :cut], dtype)
    ys = [T.mamba2_mixer_step(u[:, t], history, state, **p, **kw, residual=u[:, t]) for t in range(cut, L)]
    assert_close("tokens", torch.stack(ys, 1), whole[:, cut:], dtype)
    assert_close("state", state, final, dtype)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_a_sequence_in_pieces(lib, dtype):
    import trading_bot_0_b200 as T
    u, p, kw = _layer(dtype, 70)
    whole, hist, final = T.mamba2_mixer(u, **p, **kw, return_history=True, chunk=64)
    outs, history, state = [], None, None
    for lo, hi in ((0, 2), (2, 3), (3, 40), (40, 70)):
        out, history, state = T.mamba2_mixer(u[:, lo:hi], **p, **kw, history=history, state=state, return_history=True, chunk=64)
        outs.append(out)
    assert_close("out", torch.cat(outs, 1), whole, dtype)
    assert torch.equal(history, hist)
    assert_close("state", state, final, dtype)
    two = T.mamba2_mixer(u[:, 40:], **p, **kw, history=torch.zeros_like(hist), state=torch.zeros_like(final), chunk=64)
    assert len(two) == 2 and len(T.mamba2_mixer(u, **p, **kw)) == 2
    fresh, _ = T.mamba2_mixer(u[:, 40:], **p, **kw, chunk=64)
    assert_close("a history and a state of zeros", two[0], fresh, dtype)


def test_gradients_through_the_pieces(lib):
    """fp32: the gradients of a loss over the pieces are those of the same loss over the whole, for the input and every parameter."""
    import trading_bot_0_b200 as T
    u, p, kw = _layer("fp32", 37)
    g = torch.Generator().manual_seed(3)
    dout, dfin = torch.randn(3, 37, 64, generator=g).to(DEV), torch.randn(3, kw["nheads"], kw["headdim"], kw["dstate"], generator=g).to(DEV)
    leaves = [u.requires_grad_(), *(v.requires_grad_() for v in p.values())]
    out, hist, fin = T.mamba2_mixer(u, **p, **kw, residual=u, return_history=True)
    dh = torch.randn(hist.shape, generator=g).to(DEV)
    want = torch.autograd.grad([out, hist, fin], leaves, [dout, dh, dfin])
    outs, history, state = [], None, None
    for lo, hi in ((0, 2), (2, 20), (20, 37)):
        o, history, state = T.mamba2_mixer(u[:, lo:hi], **p, **kw, residual=u[:, lo:hi], history=history, state=state, return_history=True)
        outs.append(o)
    got = torch.autograd.grad([torch.cat(outs, 1), history, state], leaves, [dout, dh, dfin])
    for k, a, b in zip(["u", *p], got, want):
        assert_close(k, a, b, "fp32")


def test_a_piece_and_a_step_in_captured_graphs(lib):
    import trading_bot_0_b200 as T
    u, p, kw = _layer("bf16", 20)
    _, history, state = T.mamba2_mixer(u[:, :9], **p, **kw, return_history=True)
    h, s, x, tok = history.clone(), state.clone(), u[:, 9:19].clone(), u[:, 19].clone()

    def on():
        out, h2, s2 = T.mamba2_mixer(x, **p, **kw, history=h, state=s, return_history=True)
        return [out, T.mamba2_mixer_step(tok, h2, s2, **p, **kw), h2, s2]
    on()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = on()
    x.copy_(x.flip(1))
    h.neg_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, on()))


def test_histories_and_states_that_do_not_fit_are_refused(lib):
    import trading_bot_0_b200 as T
    u, p, kw = _layer("bf16", 8)
    _, h, s = T.mamba2_mixer(u, **p, **kw, return_history=True)
    for bad in (dict(history=h[:, 1:]), dict(history=h.float()), dict(history=h[:2]), dict(state=s[:2]), dict(state=s.bfloat16()),
                dict(history=h, state=s[:, 1:])):
        with pytest.raises(ValueError):
            T.mamba2_mixer(u, **p, **kw, **bad)


@pytest.mark.parametrize("B,L,H,P", [(1, 9, 8, 32), (1, 9, 3, 8), (2, 3, 3, 8), (1, 1, 8, 32)])
@pytest.mark.parametrize("K", [2, 4])
def test_the_history_is_memory_of_its_own(lib, B, L, H, P, K):
    """Stepping on with a prompt's history leaves the prompt's graph as it was, whatever the rows' layout, and holds nothing of the
    projection's output."""
    import trading_bot_0_b200 as T
    p, kw = _mamba2("fp32", H=H, P=P, N=16)
    p["conv_weight"] = p["conv_weight"][:, :K].contiguous()
    p = {k: v.to(DEV) for k, v in p.items()}
    u = torch.randn(B, L, 64, generator=torch.Generator().manual_seed(6)).to(DEV)
    leaf = p["in_proj"].requires_grad_()
    out, history, state = T.mamba2_mixer(u, **p, **kw, return_history=True)
    want = torch.autograd.grad(out.sum(), leaf, retain_graph=True)[0]
    h = history.detach()
    assert h.untyped_storage().nbytes() == h.numel() * 4
    T.mamba2_mixer_step(u[:, 0], h, state.detach().clone(), **p, **kw)
    assert torch.equal(torch.autograd.grad(out.sum(), leaf)[0], want)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("H,P", [(3, 8), (5, 8), (8, 32)])
def test_one_row_whose_stride_is_off_16_bytes(lib, dtype, H, P):
    """A prompt of one token of one sequence: its row has no neighbour, whatever the strides say.  As in a batch of two."""
    import trading_bot_0_b200 as T
    u, p, kw = _layer(dtype, 1, H=H, P=P, N=16)
    both, hists, finals = T.mamba2_mixer(u[:2], **p, **kw, return_history=True)
    for i in range(2):
        out, history, final = T.mamba2_mixer(u[i:i + 1], **p, **kw, return_history=True)
        assert torch.equal(out[0], both[i]) and torch.equal(history[0], hists[i]) and torch.equal(final[0], finals[i])
        again, h2, f2 = T.mamba2_mixer(u[i:i + 1], **p, **kw, history=torch.zeros_like(history), state=torch.zeros_like(final), return_history=True)
        assert torch.equal(h2, history)
        assert_close("with a history of zeros", again, out, dtype)
        step = T.mamba2_mixer_step(u[i], torch.zeros_like(history), torch.zeros_like(final), **p, **kw)
        assert_close("as a step", step, out[:, 0], dtype)


@pytest.mark.parametrize("B,L", [(1, 1), (2, 1), (1, 2), (1, 5), (4, 3)])
@pytest.mark.parametrize("odd", [False, True])
def test_the_smallest_batches_train(lib, B, L, odd):
    """Both mixers with a handful of tokens, columns on 16 bytes and off them, against 64 bits; with and without the pieces' operands."""
    import trading_bot_0_b200 as T
    from tests.test_mixer_gpu import _mamba2_ref, _selective, _selective_ref
    size = dict(D=40, N=12, rank=3) if odd else {}
    u, p, dout = _selective("fp32", B=B, L=L, **size)
    leaves = [u.double().requires_grad_(), *(v.double().requires_grad_() for v in p.values())]
    ref, _ = _selective_ref(leaves[0], dict(zip(p, leaves[1:])), leaves[0])
    want = torch.autograd.grad(ref, leaves, dout.double())
    mine = [u.to(DEV).requires_grad_(), *(v.to(DEV).requires_grad_() for v in p.values())]
    D, N = p["A"].shape
    for extra in ({}, dict(history=torch.zeros(B, 3, D, device=DEV), state=torch.zeros(B, D, N, device=DEV))):
        out, _, _ = T.selective_mixer(mine[0], **dict(zip(p, mine[1:])), residual=mine[0], **extra)
        assert_close("out", out.detach(), ref.detach(), "fp32")
        for k, a, b in zip(["u", *p], torch.autograd.grad(out, mine, dout.to(DEV)), want):
            assert_close(k, a, b, "fp32")
    H, P, N = (3, 8, 16) if odd else (8, 32, 64)
    p, kw = _mamba2("fp32", H=H, P=P, N=N)
    g = torch.Generator().manual_seed(1)
    u, dout = torch.randn(B, L, 64, generator=g), torch.randn(B, L, 64, generator=g)
    leaves = [u.double().requires_grad_(), *(v.double().requires_grad_() for v in p.values())]
    ref, _ = _mamba2_ref(leaves[0], dict(zip(p, leaves[1:])), H, P, N, 1, leaves[0])
    want = torch.autograd.grad(ref, leaves, dout.double())
    mine = [u.to(DEV).requires_grad_(), *(v.to(DEV).requires_grad_() for v in p.values())]
    for extra in ({}, dict(history=torch.zeros(B, 3, p["conv_weight"].shape[0], device=DEV), state=torch.zeros(B, H, P, N, device=DEV))):
        out, _ = T.mamba2_mixer(mine[0], **dict(zip(p, mine[1:])), **kw, residual=mine[0], **extra)
        assert_close("out", out.detach(), ref.detach(), "fp32")
        grads = dict(zip(["u", *p], torch.autograd.grad(out, mine, dout.to(DEV))))
        if L == 1:      # the decay meets a state of zeros: dA is 0, the difference of sums whose size is that of dD's; no size of its own to go by
            assert grads.pop("A").abs().max() <= 1e-4 * grads["D"].abs().max()
        for k, b in zip(["u", *p], want):
            if k in grads:
                assert_close(k, grads[k], b, "fp32")
