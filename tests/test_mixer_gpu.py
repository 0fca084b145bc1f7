"""Whole mixers over the library's operators, run as a layer is: training with gradients, prompts (padded, in pieces), then tokens.
Against 64-bit restatements at the parity gates of the workload definition (tests/_util.py); pieces and tokens against the whole."""
import pytest
import torch

from oracle import layer_oracle as LO
from oracle import ssd_oracle as O
from tests._util import assert_close

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {"fp32": torch.float32, "bf16": torch.bfloat16}
F = torch.nn.functional


def _selective(dtype, B=2, L=50, d_model=48, D=64, N=16, rank=8, seed=3):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    t = TD[dtype]
    p = dict(in_proj=(n(2 * D, d_model) / d_model ** 0.5).to(t), conv_weight=n(D, 4) / 2, conv_bias=0.1 * n(D),
             x_proj=(n(rank + 2 * N, D) / D ** 0.5).to(t), dt_proj=(n(D, rank) / rank ** 0.5).to(t), dt_bias=0.5 * n(D) - 2.5,
             A=-(0.5 + 3 * torch.rand(D, N, generator=g)), D=n(D), out_proj=(n(d_model, D) / D ** 0.5).to(t))
    return n(B, L, d_model).to(t), p, n(B, L, d_model).to(t)


def _selective_ref(u, p, residual=None):
    """64 bits, differentiable, token by token."""
    D, N = p["A"].shape
    x, z = (u @ p["in_proj"].t()).split(D, -1)
    x = F.silu(F.conv1d(F.pad(x.transpose(1, 2), (3, 0)), p["conv_weight"][:, None], p["conv_bias"], groups=D).transpose(1, 2))
    dl, Bm, Cm = (x @ p["x_proj"].t()).split([p["dt_proj"].shape[1], N, N], -1)
    s = LO.softplus(dl @ p["dt_proj"].t() + p["dt_bias"])
    h, ys = torch.zeros(u.shape[0], D, N, dtype=u.dtype), []
    for t in range(u.shape[1]):
        h = torch.exp(s[:, t, :, None] * p["A"]) * h + (s[:, t] * x[:, t])[..., None] * Bm[:, t, None]
        ys.append((h * Cm[:, t, None]).sum(-1) + p["D"] * x[:, t])
    out = (torch.stack(ys, 1) * F.silu(z)) @ p["out_proj"].t()
    return (out if residual is None else out + residual), h


@pytest.mark.parametrize("D,rank,N", [(64, 8, 16), (40, 3, 12)])
def test_selective_mixer_trains(lib, D, rank, N):
    import trading_bot_0_b200 as T
    u, p, dout = _selective("fp32", D=D, rank=rank, N=N)
    u64, p64 = u.double().requires_grad_(), {k: v.double().requires_grad_() for k, v in p.items()}
    ref, fin = _selective_ref(u64, p64, u64)
    want = torch.autograd.grad(ref, [u64, *p64.values()], dout.double())
    ud, pd = u.to(DEV).requires_grad_(), {k: v.to(DEV).requires_grad_() for k, v in p.items()}
    out, hist, state = T.selective_mixer(ud, **pd, residual=ud)
    assert_close("out", out.detach(), ref.detach(), "fp32")
    assert_close("state", state.detach(), fin.detach(), "fp32")
    got = torch.autograd.grad(out, [ud, *pd.values()], dout.to(DEV))
    for k, a, b in zip(["u", *p], got, want):
        assert_close(k, a, b, "fp32")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_selective_mixer_prompt_pieces_and_tokens(lib, dtype):
    """A padded prompt; the same in pieces; then tokens; all against the whole sequence."""
    import trading_bot_0_b200 as T
    u, p, _ = _selective(dtype, B=3, L=41)
    u, p = u.to(DEV), {k: v.to(DEV) for k, v in p.items()}
    whole, hist, state = T.selective_mixer(u, **p)
    a, h1, s1 = T.selective_mixer(u[:, :17], **p)
    b, h2, s2 = T.selective_mixer(u[:, 17:], **p, history=h1, state=s1)
    assert_close("pieces", torch.cat([a, b], 1), whole, dtype)
    assert torch.equal(h2, hist)
    assert_close("state", s2, state, "fp32" if dtype == "fp32" else "bf16")
    lengths = torch.tensor([30, 0, 41], dtype=torch.int32, device=DEV)
    padded, hp, sp = T.selective_mixer(u, **p, lengths=lengths)
    assert (padded[0, 30:] == 0).all() and (padded[1] == 0).all()
    assert_close("padded", padded[0, :30], whole[0, :30], dtype)
    assert (sp[1] == 0).all() and (hp[1] == 0).all()
    for t in range(30, 41):      # row 0 goes on token by token
        y = T.selective_mixer_step(u[:1, t], hp[:1], sp[:1], **p)
        assert_close(f"token {t}", y[0], whole[0, t], dtype)
    assert_close("state", sp[0], state[0], "fp32" if dtype == "fp32" else "bf16")


def _mamba2(dtype, d_model=64, H=8, P=32, N=64, G=1, seed=5):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)
    t, hp, ch = TD[dtype], H * P, H * P + 2 * G * N
    return dict(in_proj=(n(hp + ch + H, d_model) / d_model ** 0.5).to(t), conv_weight=n(ch, 4) / 2, conv_bias=0.1 * n(ch), dt_bias=n(H) - 3.0,
                A=-torch.exp(torch.rand(H, generator=g) * 2.0), D=torch.ones(H), norm_weight=1 + 0.1 * n(hp),
                out_proj=(n(d_model, hp) / hp ** 0.5).to(t)), dict(nheads=H, headdim=P, dstate=N, ngroups=G)


def _mamba2_ref(u, p, H, P, N, G, residual):
    hp, gn = H * P, G * N
    zx = u @ p["in_proj"].t()
    z, xBC, dt = zx[..., :hp], zx[..., hp:2 * hp + 2 * gn], zx[..., 2 * hp + 2 * gn:]
    y, fin = O.mamba2_mixer_core_ref(xBC, dt, z.unflatten(-1, (H, P)), p["conv_weight"], p["conv_bias"], p["dt_bias"], p["A"], p["D"],
                                     p["norm_weight"], nheads=H, headdim=P, dstate=N, ngroups=G)
    return y.flatten(2) @ p["out_proj"].t() + residual, fin


@pytest.mark.parametrize("H,P,N", [(8, 32, 64), (3, 8, 16)])     # rows of the projection on 16 bytes, and off them
def test_mamba2_mixer_trains(lib, H, P, N):
    import trading_bot_0_b200 as T
    p, kw = _mamba2("fp32", H=H, P=P, N=N)
    g = torch.Generator().manual_seed(1)
    u, dout = torch.randn(2, 70, 64, generator=g), torch.randn(2, 70, 64, generator=g)
    u64, p64 = u.double().requires_grad_(), {k: v.double().requires_grad_() for k, v in p.items()}
    ref, _ = _mamba2_ref(u64, p64, H, P, N, 1, u64)
    want = torch.autograd.grad(ref, [u64, *p64.values()], dout.double())
    ud, pd = u.to(DEV).requires_grad_(), {k: v.to(DEV).requires_grad_() for k, v in p.items()}
    out, _ = T.mamba2_mixer(ud, **pd, **kw, residual=ud, chunk=64)
    assert_close("out", out.detach(), ref.detach(), "fp32")
    for k, a, b in zip(["u", *p], torch.autograd.grad(out, [ud, *pd.values()], dout.to(DEV)), want):
        assert_close(k, a, b, "fp32")


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_mamba2_mixer_tokens_are_the_prompt(lib, dtype):
    """Token by token from an empty state gives what the prompt gave, and its state."""
    import trading_bot_0_b200 as T
    p, kw = _mamba2(dtype)
    g = torch.Generator().manual_seed(2)
    u = torch.randn(3, 40, 64, generator=g).to(TD[dtype]).to(DEV)
    p = {k: v.to(DEV) for k, v in p.items()}
    out, fin = T.mamba2_mixer(u, **p, **kw, residual=u, algo="fp32_cores")
    hist = torch.zeros(3, 3, p["conv_weight"].shape[0], dtype=TD[dtype], device=DEV)
    state = torch.zeros(3, kw["nheads"], kw["headdim"], kw["dstate"], device=DEV)
    ys = [T.mamba2_mixer_step(u[:, t], hist, state, **p, **kw, residual=u[:, t]) for t in range(40)]
    assert_close("out", torch.stack(ys, 1), out, dtype)
    assert_close("state", state, fin, dtype)


def test_layers_in_a_captured_training_step(lib):
    """Two mixers one after the other, forward and backward captured on a side stream and replayed on new inputs: the bits of an eager
    step.  (No eager graph of the leaves may be alive during the capture: autograd would wait on the stream of its accumulation nodes.)"""
    import trading_bot_0_b200 as T
    u, p, dout = _selective("bf16", B=2, L=64)
    q, kw = _mamba2("bf16", d_model=48)
    u, dout = u.to(DEV), dout.to(DEV)
    leaves = [v.to(DEV).requires_grad_() for v in (*p.values(), *q.values())]
    pn, qn = dict(zip(p, leaves)), dict(zip(q, leaves[len(p):]))

    def step():
        h, _, _ = T.selective_mixer(u, **pn, residual=u)
        out, _ = T.mamba2_mixer(h, **qn, **kw, residual=h)
        return [out, *torch.autograd.grad(out, leaves, dout)]
    step()
    side = torch.cuda.Stream(DEV)
    side.wait_stream(torch.cuda.current_stream(DEV))
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream(DEV).wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        held = step()
    u.copy_(u.flip(1))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, step()))
