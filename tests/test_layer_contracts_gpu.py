"""What the layer operators refuse, and what they owe to autograd: sizes of zero, outputs that share memory with inputs, tensors that are
changed in place while a node holds them, derivatives that the nodes do not have."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16
rand = lambda *s, dtype=BF: torch.randn(*s, device=DEV).to(dtype)


@pytest.mark.parametrize("lead", [(4,), (2, 3), (2, 1, 3), ()])
def test_projections_without_features_are_refused(lib, lead):
    """No input or no output features, in any number of dims: the library's error (not a division by zero on the host)."""
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import linear as LN
    E = T._lib.SsdError
    with pytest.raises(E, match="positive"):
        LN.linear_forward(rand(*lead, 0), rand(8, 0))
    with pytest.raises(E, match="positive"):
        LN.linear_forward(rand(*lead, 16), rand(0, 16), None, rand(*lead, 0))
    with pytest.raises(E, match="positive"):
        LN.linear_backward(rand(*lead, 0), rand(*lead, 16), rand(0, 16))
    with pytest.raises(E, match="positive"):
        LN.linear_backward(rand(*lead, 8), rand(*lead, 0), rand(8, 0))
    with pytest.raises(E, match="positive"):
        LN.linear(rand(*lead, 0).requires_grad_(), rand(8, 0))
    if lead:
        with pytest.raises(E, match="positive"):
            LN.linear_forward(rand(*lead, 16)[:0], rand(8, 16))


def test_a_mixer_without_a_rank_is_refused(lib):
    import trading_bot_0_b200 as T
    D, N = 16, 8
    p = dict(in_proj=rand(2 * D, 24), conv_weight=rand(D, 4, dtype=torch.float32), conv_bias=None, x_proj=rand(2 * N, D), dt_proj=rand(D, 0),
             dt_bias=rand(D, dtype=torch.float32), A=-torch.ones(D, N, device=DEV), D=None, out_proj=rand(24, D))
    with pytest.raises(T._lib.SsdError, match="positive"):
        T.selective_mixer(rand(2, 5, 24), **p)
    with pytest.raises(T._lib.SsdError, match="positive"):
        T.selective_mixer_step(rand(2, 24), rand(2, 3, D), torch.zeros(2, D, N, device=DEV), **p)


def test_a_node_notices_that_its_tensor_was_stepped(lib):
    """A step, or an output over a tensor that a node has saved: backward raises, as after torch's own in-place calls."""
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import linear as LN, prepost as P, selective as S
    f = torch.float32
    raises = lambda: pytest.raises(RuntimeError, match="modified by an inplace operation")
    B, L, D, N = 2, 6, 16, 8
    x, w, hist = rand(B, L, D).requires_grad_(), rand(D, 4, dtype=f), rand(B, 3, D)
    out, _ = P.causal_conv1d_carry(x, w, None, hist)
    P.conv1d_step(hist, rand(B, D), w)
    with raises():
        out.sum().backward()
    out, _ = P.causal_conv1d_carry(x, w, None, rand(B, 3, D))
    P.conv1d_step(rand(B, 3, D), rand(B, D), w, out=x.detach()[:, 0])
    with raises():
        out.sum().backward()
    A, bc, st = -torch.ones(D, N, device=DEV), rand(B, L, N), rand(B, D, N, dtype=f)
    y, _ = S.selective_scan(x, x, A, bc, bc, init_state=st)
    S.selective_step(st, rand(B, D), rand(B, D), A, rand(B, N), rand(B, N))
    with raises():
        y.sum().backward()
    z = rand(B, L, D)
    y, _ = S.selective_scan(x, x, A, bc, bc, z=z)
    S.selective_step(st, rand(B, D), rand(B, D), A, rand(B, N), rand(B, N), y=z[:, 2])
    with raises():
        y.sum().backward()
    W = rand(D, D).requires_grad_()
    u = rand(B, D)
    o = LN.linear(u, W)
    LN.linear_forward(rand(B, D), rand(D, D), out=u)
    with raises():
        o.sum().backward()
    H, Pd = 2, 8
    xs, dt, st4 = rand(B, L, H, Pd, dtype=f).requires_grad_(), rand(B, L, H, dtype=f).abs(), rand(B, H, Pd, N, dtype=f)
    a, b4 = -torch.ones(H, device=DEV), rand(B, L, 1, N, dtype=f)
    y, _ = T.ssd_scan(xs, dt, a, b4, b4, init_state=st4)
    T.state_update(st4, xs.detach()[:, 0], dt[:, 0], a, b4[:, 0], b4[:, 0])
    with raises():
        y.sum().backward()


def test_steps_count_as_one_change_each(lib):
    from trading_bot_0_b200 import linear as LN, prepost as P, selective as S
    f = torch.float32
    B, D, N = 3, 16, 8
    hist, st, y, o, W = rand(B, 3, D), rand(B, D, N, dtype=f), rand(B, D), rand(B, D), rand(D, D)
    args = (rand(B, D), rand(D, 4, dtype=f)), (rand(B, D), rand(B, D), -torch.ones(D, N, device=DEV), rand(B, N), rand(B, N))
    for i in range(1, 4):
        P.conv1d_step(hist, *args[0], out=o)
        S.selective_step(st, *args[1], y=y)
        assert hist._version == st._version == y._version == o._version == i
    LN.linear_forward(y, W, out=o)
    assert o._version == 4 and y._version == 3
    v = o._version
    with pytest.raises(ValueError):
        LN.linear_forward(y, W, rand(D + 1), out=o)
    assert o._version == v
    with torch.inference_mode():                          # tensors that keep no count, inside the mode and after it
        h2, s2 = rand(B, 3, D), rand(B, D, N, dtype=f)
        P.conv1d_step(h2, *args[0])
        S.selective_step(s2, *args[1])
    P.conv1d_step(h2, *args[0])
    S.selective_step(s2, *args[1])


@pytest.mark.parametrize("S_,D,N", [(5, 24, 8), (1, 40, 16), (300, 264, 16), (1201, 256, 64)])
def test_steps_write_over_their_own_operands_or_between_them(lib, S_, D, N):
    """The output over x, dt, z or the convolution's input themselves, and in rows between the input's: the same bits as apart."""
    from trading_bot_0_b200 import prepost as P, selective as S
    f = torch.float32
    x, dt, z, B, C, A, w, st, h = (rand(S_, D), rand(S_, D), rand(S_, D), rand(S_, N), rand(S_, N), -rand(D, N, dtype=f).abs(), rand(D, 4, dtype=f),
                                   rand(S_, D, N, dtype=f), rand(S_, 3, D))

    def scan(x, dt, z, y=None):
        s = st.clone()
        return S.selective_step(s, x, dt, A, B, C, None, z, y=y, dt_softplus=True), s
    want, state = scan(x, dt, z)
    for i in range(3):
        own = [x.clone(), dt.clone(), z.clone()]
        y, s = scan(*own, y=own[i])
        assert torch.equal(y, want) and torch.equal(s, state) and y.data_ptr() == own[i].data_ptr()
    wide = torch.zeros(S_, 2 * D + 8, dtype=BF, device=DEV)
    wide[:, :D] = x
    y, s = scan(wide[:, :D], dt, z, y=wide[:, D:2 * D])
    assert torch.equal(y, want) and torch.equal(s, state) and torch.equal(wide[:, :D], x)
    out = P.conv1d_step(hist := h.clone(), x, w)
    own = x.clone()
    assert torch.equal(P.conv1d_step(h2 := h.clone(), own, w, out=own), out) and torch.equal(h2, hist)
    assert torch.equal(P.conv1d_step(h3 := h.clone(), wide[:, :D], w, out=wide[:, D:2 * D]), out) and torch.equal(h3, hist)


def test_step_outputs_that_share_memory_are_refused(lib):
    import trading_bot_0_b200 as T
    from trading_bot_0_b200 import prepost as P, selective as S
    f, S_, D, N = torch.float32, 4, 16, 16
    buf = torch.zeros(S_ * 2, D, dtype=BF, device=DEV)
    x, B, C, A, w = buf[:S_], rand(S_, N), rand(S_, N), -torch.ones(D, N, device=DEV), rand(D, 4, dtype=f)
    st, h = rand(S_, D, N, dtype=f), rand(S_, 3, D)
    for y in (B, C, buf[1:S_ + 1], st.view(BF).view(-1)[:S_ * D].view(S_, D)):
        with pytest.raises(T._lib.SsdError, match="share"):
            S.selective_step(st, x, x, A, B, C, y=y)
    for out in (buf[1:S_ + 1], h.view(-1)[:S_ * D].view(S_, D)):
        with pytest.raises(T._lib.SsdError, match="share"):
            P.conv1d_step(h, x, w, out=out)
    with pytest.raises(T._lib.SsdError, match="share"):
        P.conv1d_step(h, h[:, 2], w)


@pytest.mark.parametrize("off", [0, 4])
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("M,K,N", [(3, 64, 48), (40, 64, 48), (64, 1536, 128), (300, 64, 520), (50, 33, 40), (64, 1540, 40), (33, 64, 41)])
def test_status_word_of_the_projection(lib, dtype, M, K, N, off):
    """The first word of a workspace that held something else is 0 after each call, on every path (few rows, tensor cores with and without
    splits, CUDA cores), also where the workspace starts off 256 bytes and where no gradient is wanted."""
    import ctypes as C
    import trading_bot_0_b200 as T
    from trading_bot_0_b200.ssd import workspace_status
    L = T._lib
    t = torch.float32 if dtype == "fp32" else BF
    x, w, out, dout, pre, dx, dw, db = (rand(M, K, dtype=t), rand(N, K, dtype=t), rand(M, N, dtype=t), rand(M, N, dtype=t), rand(M, N, dtype=torch.float32),
                                        rand(M, K, dtype=t), rand(N, K, dtype=t), rand(N, dtype=t))
    p = lambda v: C.c_void_p(v.data_ptr())
    s = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    d = L.SsdLinearDims()
    d.rows, d.in_features, d.out_features, d.dtype, d.device = M, K, N, L.SSD_BF16 if t == BF else L.SSD_F32, 0
    for act in (0, 1):
        d.activation = act
        n = [lib.ssd_linear_workspace_bytes(C.byref(d), k) for k in (0, 1)]
        ws = torch.empty(max(n) + 8, dtype=torch.uint8, device=DEV)[off:]

        def check(rc):
            assert rc == 0 and int(ws[:4].view(torch.int32)) == 0 and workspace_status(ws) == 0
            ws.fill_(0x5a)
        ws.fill_(0x5a)
        check(lib.ssd_linear_forward(C.byref(d), p(x), p(w), None, None, p(out), p(pre), p(ws), n[0], s))
        for want in ((dx, dw, db), (dx, dw, None), (dx, None, None), (None, dw, None), (None, None, db), (None, None, None)):
            check(lib.ssd_linear_backward(C.byref(d), p(x), p(w), p(pre), p(dout), 0, *(None if v is None else p(v) for v in want), p(ws), n[1], s))


def test_gradients_of_a_history_need_no_alignment(lib):
    """The gradient of the new history as a view that starts off 16 bytes (states of several layers flattened into one vector)."""
    from trading_bot_0_b200 import prepost as P
    B, L, C, K = 2, 9, 24, 4
    x, w, b, h = rand(B, L, C).requires_grad_(), rand(C, K, dtype=torch.float32).requires_grad_(), rand(C, dtype=torch.float32), rand(B, K - 1, C).requires_grad_()
    dout, dnew = rand(B, L, C), rand(B, K - 1, C)
    out, new = P.causal_conv1d_carry(x, w, b, h)
    off = torch.cat([rand(1), dnew.flatten()])[1:].view(B, K - 1, C)
    assert off.data_ptr() % 16 and off.is_contiguous()
    want = torch.autograd.grad([out, new], [x, w, h], [dout, dnew], retain_graph=True)
    got = torch.autograd.grad([out, new], [x, w, h], [dout, off], retain_graph=True)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    flat = torch.cat([rand(3), new.flatten()])            # and as autograd itself makes one
    g = torch.cat([rand(3), dnew.flatten()])
    got = torch.autograd.grad([out, flat], [x, w, h], [dout, g])
    assert all(torch.equal(p, q) for p, q in zip(got, want))


def _calls():
    """The differentiable calls: a function of its first tensor, and that tensor."""
    from trading_bot_0_b200 import linear as LN, prepost as P, selective as S
    f, B, L, D, N = torch.float32, 2, 6, 16, 4
    g = torch.Generator(device=DEV).manual_seed(1)
    n = lambda *s: torch.randn(*s, device=DEV, generator=g)
    w, A, bc, W, st = n(D, 4), -n(D, N).abs(), n(B, L, N), n(12, D), n(B, D, N)
    return {"linear": (lambda x: LN.linear(x, W, activation="silu"), n(B, L, D)),
            "conv": (lambda x: P.causal_conv1d_carry(x, w)[0], n(B, L, D)),
            "scan": (lambda x: S.selective_scan(x, x, A, bc, bc, dt_softplus=True)[0], n(B, L, D)),
            "scan state": (lambda h: S.selective_scan(n(B, L, D), n(B, L, D), A, bc, bc, init_state=h, dt_softplus=True)[1], st)}


@pytest.mark.parametrize("which", ["linear", "conv", "scan", "scan state"])
def test_a_second_derivative_is_refused(lib, which):
    """The nodes have one derivative.  Its values come with create_graph too; differentiating them again raises (it used to go on as if
    they were constants)."""
    f, x = _calls()[which]
    x = x.requires_grad_()
    torch.manual_seed(0)
    y = f(x)
    want = torch.autograd.grad(y.square().sum(), x, retain_graph=True)[0]
    g = torch.autograd.grad(y.square().sum(), x, create_graph=True)[0]
    assert torch.equal(g, want) and g.requires_grad
    with pytest.raises(RuntimeError, match="differentiable once"):
        torch.autograd.grad((g * x).sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        (g * x).sum().backward()


def test_the_residuals_gradient_is_as_often_differentiable_as_its_source(lib):
    from trading_bot_0_b200 import linear as LN
    x, W, r = rand(3, 16), rand(8, 16), rand(3, 8, dtype=BF).requires_grad_()
    g = torch.autograd.grad(LN.linear(x, W, None, r).pow(2).sum(), r, create_graph=True)[0]
    assert torch.equal(torch.autograd.grad(g.sum(), r)[0], torch.full_like(r, 2.0))


@pytest.mark.parametrize("which", ["linear", "conv", "scan", "scan state"])
def test_a_forward_mode_derivative_is_refused(lib, which):
    """With and without requires_grad: a tangent would be dropped."""
    import torch.autograd.forward_ad as fwAD
    f, x = _calls()[which]
    with fwAD.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            f(fwAD.make_dual(x, torch.ones_like(x)))
        with pytest.raises(ValueError, match="forward-mode"):
            f(fwAD.make_dual(x.clone().requires_grad_(), torch.ones_like(x)))
        f(x)
