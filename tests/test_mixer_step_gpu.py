"""The mixers' single steps are no part of an autograd graph, whatever their parameters ask for."""
import pytest
import torch

from tests.test_mixer_gpu import DEV, _mamba2, _selective

pytestmark = pytest.mark.gpu


def test_steps_leave_no_graph(lib):
    """Their convolution and scan work in place and have no gradient; a graph of the projections alone would give part of one."""
    import trading_bot_0_b200 as T
    u, p, _ = _selective("bf16")
    u = u[:, 0].to(DEV)
    q = {k: v.to(DEV) for k, v in p.items()}
    D, N = p["A"].shape
    state = lambda: (torch.zeros(len(u), 3, D, dtype=u.dtype, device=DEV), torch.zeros(len(u), D, N, device=DEV))
    want = T.selective_mixer_step(u, *state(), **q, residual=u)
    asks = {k: v.clone().requires_grad_() for k, v in q.items()}
    out = T.selective_mixer_step(u.clone().requires_grad_(), *state(), **asks, residual=u.clone().requires_grad_())
    assert not out.requires_grad and torch.equal(out, want)
    p, kw = _mamba2("bf16", d_model=u.shape[1])
    q = {k: v.to(DEV) for k, v in p.items()}
    state = lambda: (torch.zeros(len(u), 3, p["conv_weight"].shape[0], dtype=u.dtype, device=DEV),
                     torch.zeros(len(u), kw["nheads"], kw["headdim"], kw["dstate"], device=DEV))
    want = T.mamba2_mixer_step(u, *state(), **q, **kw, residual=u)
    asks = {k: v.clone().requires_grad_() for k, v in q.items()}
    out = T.mamba2_mixer_step(u, *state(), **asks, **kw, residual=u)
    assert not out.requires_grad and torch.equal(out, want)
