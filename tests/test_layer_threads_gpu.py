"""Every entry point as the first CUDA work of a host thread: autograd's own threads, and a caller's."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
rand = lambda *s, dtype=BF: torch.randn(*s, device=DEV, dtype=dtype)


def _on_a_new_thread(f):
    got = []

    def run():
        try:
            got.append(f())
        except BaseException as e:    # noqa: BLE001 (handed to the caller)
            got.append(e)
    t = threading.Thread(target=run)
    t.start()
    t.join()
    if isinstance(got[0], BaseException):
        raise got[0]
    return got[0]


def _calls():
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import linear as LN, prepost as P, selective as S
    torch.manual_seed(0)
    x, W, dout, pre = rand(300, 64), rand(136, 64), rand(300, 136), rand(300, 136, dtype=F32)
    yield "projection", lambda: LN.linear_forward(x, W)[0]
    yield "projection in splits", lambda a=rand(64, 1536), b=rand(128, 1536): LN.linear_forward(a, b)[0]
    yield "projection, few rows", lambda: LN.linear_forward(x[:4], W)[0]
    yield "projection backward", lambda: LN.linear_backward(dout, x, W, bias=False)[:2]
    yield "projection backward, activation", lambda: LN.linear_backward(dout, x, W, pre, activation="silu")
    B, L, D, N = 2, 40, 64, 16
    u, A, bc, w = rand(B, L, D), -torch.rand(D, N, device=DEV), rand(B, L, N), rand(D, 4, dtype=F32)
    yield "scan", lambda: S.selective_scan_forward(u, u, A, bc, bc, dt_softplus=True)[:2]
    yield "scan backward", lambda: list(S.selective_scan_backward(u, u, u, A, bc, bc, dt_softplus=True).values())
    yield "convolution", lambda: P.conv1d_carry_forward(u, w)
    yield "convolution backward", lambda: P.conv1d_carry_backward(u, w, None, None, u)[:2]
    s4 = dict(x=rand(2, 256, 8, 64), dt=rand(2, 256, 8).abs() * 0.1, A=-torch.ones(8, device=DEV), Bm=rand(2, 256, 1, 128), Cm=rand(2, 256, 1, 128))
    yield "SSD scan", lambda: T.forward(**s4, chunk=128)[:2]
    _, _, ws = T.forward(**s4, chunk=128, for_backward=True)
    dy = rand(2, 256, 8, 64)
    yield "SSD backward", lambda: [v for k, v in T.backward(dy, **s4, chunk=128).items() if k in ("dx", "dB", "dC", "ddt")]
    yield "SSD backward from what the forward kept", lambda: [v for k, v in T.backward(dy, **s4, chunk=128, workspace=ws, fwd_saved=True).items() if k in ("dx", "dB", "dC", "ddt")]


def test_first_work_of_a_thread(lib):
    flat = lambda v: [v] if isinstance(v, torch.Tensor) else [t for t in v if t is not None]
    bad = []
    for name, f in _calls():
        want = flat(f())
        torch.cuda.synchronize()
        try:
            got = flat(_on_a_new_thread(f))
            torch.cuda.synchronize()
            if not all(torch.equal(a, b) for a, b in zip(want, got)):
                bad.append((name, "other values"))
        except Exception as e:    # noqa: BLE001
            bad.append((name, str(e)))
    assert not bad, bad


def test_first_work_of_autograds_thread(lib):
    """A backward that begins with a projection, in a process where autograd's thread has done nothing yet."""
    import os
    import subprocess
    import sys
    code = """
import torch
from trading_bot_0_b200 import linear as LN
x, w, g = (torch.randn(*s, device="cuda:0").bfloat16() for s in ((300, 64), (136, 64), (300, 136)))
x.requires_grad_(); w.requires_grad_()
a = torch.autograd.grad(LN.linear(x, w), [x, w], g)
b = LN.linear_backward(g, x.detach(), w.detach(), bias=False)
assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
"""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
