"""The operators of a selective state space layer as they are measured: the scan with a decay per channel and state, the causal
convolution that carries its history, and the projection with bias, activation and residual in its epilogue; for training, for prompts
and for single tokens.

With `own` false `run` computes the plain form in 32 bits and rounds once; with `own` true it makes the framework's calls."""
import math

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp32": torch.float32}
ES = {"bf16": 2, "fp32": 4}


def listed():
    return [
        # one step of a handful of live streams at the policy's width: latency
        dict(name="scan_step_few", op="scan_step", S=4, D=256, N=16, G=1, dtype="bf16", gate=True),
        # one step of a rollout over thousands of environments
        dict(name="scan_step_rollout", op="scan_step", S=8192, D=256, N=16, G=1, dtype="bf16", gate=False),
        # one long prompt through a layer of 1536 channels
        dict(name="scan_prompt_layer", op="scan_prompt", B=1, L=4096, D=1536, N=16, G=1, dtype="bf16", gate=True, ragged=False),
        # training step of that layer
        dict(name="scan_train_layer", op="scan_train", B=4, L=2048, D=1536, N=16, G=1, dtype="bf16", gate=True, ragged=False),
        # fp32 training of a narrow policy over padded episodes of odd lengths, some of them empty
        dict(name="scan_train_policy", op="scan_train", B=32, L=333, D=200, N=12, G=2, dtype="fp32", gate=False, ragged=True),
        # prompts of a layer continued in pieces: history in, history out
        dict(name="conv_prompt_layer", op="conv_prompt", B=16, L=4096, C=1792, K=4, dtype="bf16", ragged=False),
        # fp32 training over padded episodes
        dict(name="conv_train_policy", op="conv_train", B=64, L=1000, C=384, K=4, dtype="fp32", ragged=True),
        # one step of a rollout
        dict(name="conv_step_rollout", op="conv_step", S=8192, C=384, K=4, dtype="bf16"),
        # input projection of a layer of 768 features over 4 x 4096 tokens: 2*1536 + 2*128 + 24 outputs
        dict(name="linear_in_layer", op="linear", M=16384, K=768, N=3352, dtype="bf16", act="none", bias=False, residual=False),
        # output projection with the residual stream, training
        dict(name="linear_train_layer", op="linear_train", M=16384, K=1536, N=768, dtype="bf16", act="silu", bias=True, residual=True),
        # output projection of a few live streams: latency and one reading of the weights
        dict(name="linear_step_few", op="linear", M=4, K=1536, N=768, dtype="bf16", act="none", bias=True, residual=True),
        # fp32 training of a small policy, odd sizes
        dict(name="linear_train_policy", op="linear_train", M=2000, K=100, N=131, dtype="fp32", act="softplus", bias=True, residual=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["scan_step", "scan_prompt", "scan_train", "conv_prompt", "conv_train", "conv_step", "linear", "linear_train"])
    dtype = rng.choice(["bf16", "bf16", "fp32"])
    if op.startswith("scan"):
        N, G = rng.choice([4, 8, 12, 16, 16, 16, 24, 32, 64]), rng.choice([1, 1, 1, 2])
        D = G * _log(rng, 24, 1536 // G)
        if op == "scan_step":
            S = max(1, min(_log(rng, 1, 8192), 8192 * 256 * 16 // (D * N)))
            return dict(op=op, S=S, D=D, N=N, G=G, dtype=dtype, gate=rng.random() < 0.5)
        B, L = _log(rng, 1, 32), _log(rng, 1, 4096)
        most = 4096 * 1536 * 16 if op == "scan_prompt" else 4 * 2048 * 1536 * 16
        B = max(1, min(B, most // (L * D * N)))
        L = max(1, min(L, most // (B * D * N)))
        return dict(op=op, B=B, L=L, D=D, N=N, G=G, dtype=dtype, gate=rng.random() < 0.5, ragged=rng.random() < 0.5)
    if op.startswith("conv"):
        C, K = 8 * _log(rng, 3, 224), rng.choice([2, 3, 4, 4])
        if op == "conv_step":
            return dict(op=op, S=_log(rng, 1, 8192), C=C, K=K, dtype=dtype)
        B, L = _log(rng, 1, 64), _log(rng, 1, 4096)
        B = max(1, min(B, 64 * 1000 * 384 // (L * C)))
        return dict(op=op, B=B, L=L, C=C, K=K, dtype=dtype, ragged=rng.random() < 0.5)
    most = 16384 * 1536 * 768
    if dtype == "bf16":
        K, N, M = 8 * _log(rng, 8, 256), 8 * _log(rng, 4, 420), _log(rng, 1, 16384)
    else:
        K, N, M = _log(rng, 24, 512), _log(rng, 16, 512), _log(rng, 1, 4096)
    M = max(1, min(M, most // (K * N)))
    return dict(op=op, M=M, K=K, N=N, dtype=dtype, act=rng.choice(["none", "silu", "softplus", "relu2"]), bias=rng.random() < 0.6,
                residual=rng.random() < 0.5)


# ---- inputs --------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = DT[case["dtype"]]

    def n(*s):
        return torch.randn(*s, generator=g, device="cuda")

    def u(*s):
        return torch.rand(*s, generator=g, device="cuda")

    def lengths():   # padded episodes: most of some length, some full, some empty
        if not case["ragged"]:
            return None
        r = u(case["B"])
        return torch.where(r < 0.1, 0, torch.where(r > 0.8, case["L"], (r * (case["L"] + 1)).long())).clamp(max=case["L"]).int()

    s = dict(op=case["op"], case=dict(case))
    if case["op"].startswith("scan"):
        D, N, G = case["D"], case["N"], case["G"]
        lead = (case["S"],) if case["op"] == "scan_step" else (case["B"], case["L"])
        s.update(x=n(*lead, D).to(t), dt=(0.5 * n(*lead, D)).to(t), Bm=n(*lead, G, N).to(t), C=(n(*lead, G, N) / N ** 0.5).to(t),
                 z=n(*lead, D).to(t) if case["gate"] else None, D=1.0 + 0.1 * n(D))
        s["A"] = -torch.arange(1, N + 1, device="cuda").float() * (1.0 + 0.1 * u(D, N))
        dt0 = torch.exp(math.log(1e-3) + u(D) * math.log(100.0))         # step sizes of 1e-3 to 1e-1
        s["dt_bias"] = dt0 + torch.log(-torch.expm1(-dt0))
        s["state"] = 0.1 * n(lead[0], D, N)
        if case["op"] != "scan_step":
            s["lengths"] = lengths()
        if case["op"] == "scan_train":
            s.update(dy=n(*lead, D).to(t), dfinal=0.1 * n(lead[0], D, N))
    elif case["op"].startswith("conv"):
        C, K = case["C"], case["K"]
        lead = (case["S"],) if case["op"] == "conv_step" else (case["B"], case["L"])
        s.update(x=n(*lead, C).to(t), w=n(C, K) / K ** 0.5, b=0.3 * n(C), history=n(lead[0], K - 1, C).to(t))
        if case["op"] != "conv_step":
            s["lengths"] = lengths()
        if case["op"] == "conv_train":
            s.update(dout=n(*lead, C).to(t), dnew=n(lead[0], K - 1, C).to(t))
    else:
        M, K, N = case["M"], case["K"], case["N"]
        s.update(x=n(M, K).to(t), w=(n(N, K) / K ** 0.5).to(t), b=(0.3 * n(N)).to(t) if case["bias"] else None,
                 r=n(M, N).to(t) if case["residual"] else None, act=case["act"])
        if case["op"] == "linear_train":
            s["dout"] = n(M, N).to(t)
    return s


def work(case):
    e, op = ES[case["dtype"]], case["op"]
    if op.startswith("scan"):
        D, N, G = case["D"], case["N"], case["G"]
        tok = case["S"] if op == "scan_step" else case["B"] * case["L"]
        rows = case["S"] if op == "scan_step" else case["B"]
        gate = 1 if case["gate"] else 0
        fwd = tok * ((3 + gate) * D + 2 * G * N) * e + 2 * rows * D * N * 4 + D * N * 4 + 2 * D * 4
        if op != "scan_train":
            return dict(bytes=fwd, flops=7 * tok * D * N)
        bwd = tok * ((5 + 2 * gate) * D + 4 * G * N) * e + 3 * rows * D * N * 4 + 2 * D * N * 4 + 4 * D * 4
        return dict(bytes=fwd + bwd, flops=(7 + 25) * tok * D * N)
    if op.startswith("conv"):
        C, K = case["C"], case["K"]
        tok, rows = (case["S"], case["S"]) if op == "conv_step" else (case["B"] * case["L"], case["B"])
        fwd = 2 * tok * C * e + 2 * rows * (K - 1) * C * e + (K + 1) * C * 4
        if op != "conv_train":
            return dict(bytes=fwd, flops=(2 * K + 5) * tok * C)
        return dict(bytes=fwd + 3 * tok * C * e + 3 * rows * (K - 1) * C * e + 2 * (K + 1) * C * 4, flops=(8 * K + 15) * tok * C)
    M, K, N = case["M"], case["K"], case["N"]
    fwd = (M * K + N * K + M * N * (2 if case["residual"] else 1) + N) * e
    if op == "linear":
        return dict(bytes=fwd, flops=2 * M * N * K)
    return dict(bytes=fwd + (M * N + 2 * M * K + 2 * N * K + N) * e, flops=6 * M * N * K)


# ---- plain forms ---------------------------------------------------------------------------------------------------------
def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _softplus(v):
    return torch.clamp(v, min=0.0) + torch.log1p(torch.exp(-v.abs()))


def _act(v, act):
    if act == "silu":
        return v * _sigmoid(v)
    if act == "softplus":
        return _softplus(v)
    return torch.clamp(v, min=0.0).square() if act == "relu2" else v


def _dact(v, act):
    if act == "silu":
        s = _sigmoid(v)
        return s * (1.0 + v * (1.0 - s))
    if act == "softplus":
        return _sigmoid(v)
    return 2.0 * torch.clamp(v, min=0.0) if act == "relu2" else torch.ones_like(v)


def _recur(a, b):
    """h_t = a_t h_{t-1} + b_t along dim 1, by doubling of the stride (no step of it depends on the tokens' number but in the log)."""
    a, s = a.clone(), 1
    while s < a.shape[1]:
        b[:, s:] += a[:, s:] * b[:, :-s]
        if 2 * s < a.shape[1]:
            a[:, s:] = a[:, s:] * a[:, :-s]
        s *= 2
    return b


def _per_channel(v, D):      # [.., G, N] -> [.., D, N]
    return v.float().repeat_interleave(D // v.shape[-2], dim=-2)


def _scan_plain(s, train):
    x, t = s["x"].float(), s["x"].dtype
    B, L, D = x.shape
    A, Dv = s["A"], s["D"]
    G, N = s["Bm"].shape[2:]
    valid = None if s["lengths"] is None else (torch.arange(L, device=x.device)[None, :] < s["lengths"][:, None])[..., None]
    pre = s["dt"].float() + s["dt_bias"]
    step = _softplus(pre)
    if valid is not None:
        step = step * valid
    Bf, Cf = _per_channel(s["Bm"], D), _per_channel(s["C"], D)
    a = torch.exp(step[..., None] * A)
    b = (step * x)[..., None] * Bf
    b[:, 0] += a[:, 0] * s["state"]
    h = _recur(a, b)
    y0 = (h * Cf).sum(-1) + Dv * x
    z = None if s["z"] is None else s["z"].float()
    gate = 1.0 if z is None else z * _sigmoid(z)
    y = y0 * gate
    if valid is not None:
        y = y * valid
    out = dict(y=y.to(t), final_state=h[:, -1].clone())
    if not train:
        return out
    dy = s["dy"].float()
    if valid is not None:
        dy = dy * valid
    if z is not None:
        out["dz"] = (dy * y0 * _dact(z, "silu")).to(t)
    dy0 = dy * gate
    # gradients of the states, from the last token to the first
    g = dy0[..., None] * Cf
    g[:, -1] += s["dfinal"]
    nxt = torch.cat([a[:, 1:], torch.ones_like(a[:, :1])], 1)
    g = _recur(nxt.flip(1), g.flip(1)).flip(1)
    prev = torch.cat([s["state"][:, None], h[:, :-1]], 1)
    dC = (dy0[..., None] * h).view(B, L, G, D // G, N).sum(3)
    dB = (g * (step * x)[..., None]).view(B, L, G, D // G, N).sum(3)
    gB = (g * Bf).sum(-1)
    q = g * a * prev
    dstep = x * gB + (q * A).sum(-1)
    ddt = dstep * _sigmoid(pre)
    if valid is not None:
        ddt = ddt * valid
    out.update(dx=(step * gB + Dv * dy0).to(t), ddt=ddt.to(t), dA=(q * step[..., None]).sum((0, 1)), dB=dB.to(t), dC=dC.to(t),
               dD=(dy0 * x).sum((0, 1)), ddt_bias=ddt.sum((0, 1)), dinit=a[:, 0] * g[:, 0])
    return out


def _scan_step_plain(s):
    x, D = s["x"].float(), s["x"].shape[1]
    step = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(step[..., None] * s["A"]) * s["state"] + (step * x)[..., None] * _per_channel(s["Bm"], D)
    y = (h * _per_channel(s["C"], D)).sum(-1) + s["D"] * x
    if s["z"] is not None:
        y = y * _act(s["z"].float(), "silu")
    s["state"].copy_(h)
    return dict(y=y.to(s["x"].dtype), state=s["state"])


def _conv_plain(s, train):
    t = s["x"].dtype
    K = s["w"].shape[1]
    ext = torch.cat([s["history"], s["x"]], 1).float()
    B, L = s["x"].shape[:2]
    pre = s["b"] + sum(s["w"][:, k] * ext[:, k:k + L] for k in range(K))
    out = _act(pre, "silu")
    length = torch.full((B,), L, device=ext.device) if s["lengths"] is None else s["lengths"].long()
    rows = length[:, None] + torch.arange(K - 1, device=ext.device)
    new = ext[torch.arange(B, device=ext.device)[:, None], rows]
    valid = (torch.arange(L, device=ext.device)[None, :] < length[:, None])[..., None]
    if s["lengths"] is not None:
        out = out * valid
    got = dict(out=out.to(t), history=new.to(t))
    if not train:
        return got
    dpre = s["dout"].float() * _dact(pre, "silu")
    if s["lengths"] is not None:
        dpre = dpre * valid
    dext = torch.zeros_like(ext)
    dext.index_put_((torch.arange(B, device=ext.device)[:, None], rows), s["dnew"].float(), accumulate=False)
    for k in range(K):
        dext[:, k:k + L] += s["w"][:, k] * dpre
    got.update(din=dext[:, K - 1:].to(t), dhistory=dext[:, :K - 1].to(t), dbias=dpre.sum((0, 1)),
               dweight=torch.stack([(dpre * ext[:, k:k + L]).sum((0, 1)) for k in range(K)], 1))
    return got


def _conv_step_plain(s):
    ext = torch.cat([s["history"], s["x"][:, None]], 1)
    out = _act(s["b"] + (ext.float() * s["w"].t()).sum(1), "silu")
    s["history"].copy_(ext[:, 1:])
    return dict(out=out.to(s["x"].dtype), history=s["history"])


def _linear_plain(s, train):
    t = s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    pre = x @ w.t()
    if s["b"] is not None:
        pre = pre + s["b"].float()
    out = _act(pre, s["act"])
    if s["r"] is not None:
        out = out + s["r"].float()
    if not train:
        return dict(out=out.to(t))
    dpre = s["dout"].float() * _dact(pre, s["act"])
    got = dict(out=out.to(t), dx=(dpre @ w).to(t), dweight=(dpre.t() @ x).to(t))
    if s["b"] is not None:
        got["dbias"] = dpre.sum(0).to(t)
    return got


def run(s):
    op = s["op"]
    if not own:
        if op == "scan_step":
            return _scan_step_plain(s)
        if op.startswith("scan"):
            return _scan_plain(s, op == "scan_train")
        if op == "conv_step":
            return _conv_step_plain(s)
        if op.startswith("conv"):
            return _conv_plain(s, op == "conv_train")
        return _linear_plain(s, op == "linear_train")
    from trading_bot_0_b200 import linear, prepost, selective
    if op == "scan_step":
        y = selective.selective_step(s["state"], s["x"], s["dt"], s["A"], s["Bm"], s["C"], s["D"], s["z"], dt_bias=s["dt_bias"],
                                     dt_softplus=True)
        return dict(y=y, state=s["state"])
    if op.startswith("scan"):
        a = (s["x"], s["dt"], s["A"], s["Bm"], s["C"], s["D"], s["z"], s["state"])
        kw = dict(dt_bias=s["dt_bias"], dt_softplus=True, lengths=s["lengths"])
        y, fin, saved = selective.selective_scan_forward(*a, for_backward=op == "scan_train", **kw)
        out = dict(y=y, final_state=fin)
        if op == "scan_train":
            g = selective.selective_scan_backward(s["dy"], *a, s["dfinal"], workspace=saved, **kw)
            out.update({k: g[k] for k in ("dx", "ddt", "dA", "dB", "dC", "dD", "ddt_bias", "dinit")})
            if s["z"] is not None:
                out["dz"] = g["dz"]
        return out
    if op == "conv_step":
        return dict(out=prepost.conv1d_step(s["history"], s["x"], s["w"], s["b"]), history=s["history"])
    if op.startswith("conv"):
        out, new = prepost.conv1d_carry_forward(s["x"], s["w"], s["b"], s["history"], lengths=s["lengths"])
        got = dict(out=out, history=new)
        if op == "conv_train":
            got["din"], got["dweight"], got["dbias"], got["dhistory"] = prepost.conv1d_carry_backward(
                s["x"], s["w"], s["b"], s["history"], s["dout"], s["dnew"], lengths=s["lengths"])
        return got
    out, pre = linear.linear_forward(s["x"], s["w"], s["b"], s["r"], activation=s["act"], for_backward=op == "linear_train")
    got = dict(out=out)
    if op == "linear_train":
        got["dx"], got["dweight"], db = linear.linear_backward(s["dout"], s["x"], s["w"], pre, activation=s["act"], bias=s["b"] is not None)
        if s["b"] is not None:
            got["dbias"] = db
    return got


# ---- the definition in 64 bits -------------------------------------------------------------------------------------------
def exact(case, seed):
    """Token by token (scan, convolution) with autograd's gradients, in 64 bits."""
    s = prepare(case, seed)
    op = case["op"]
    train = op.endswith("train")
    d = {k: v.double().requires_grad_(train and k not in ("dy", "dfinal", "dout", "dnew")) for k, v in s.items()
         if isinstance(v, torch.Tensor) and v.is_floating_point()}
    F = torch.nn.functional
    if op.startswith("scan"):
        if op == "scan_step":
            x, dt, Bm, C, z = (None if s[k] is None else d[k][:, None] for k in ("x", "dt", "Bm", "C", "z"))
        else:
            x, dt, Bm, C, z = (d.get(k) for k in ("x", "dt", "Bm", "C", "z"))
        rep = x.shape[2] // Bm.shape[2]
        h, ys = d["state"], []
        for t in range(x.shape[1]):
            st = F.softplus(dt[:, t] + d["dt_bias"], threshold=200.0)
            Bt, Ct = Bm[:, t].repeat_interleave(rep, 1), C[:, t].repeat_interleave(rep, 1)
            new = torch.exp(st[..., None] * d["A"]) * h + (st * x[:, t])[..., None] * Bt
            y = torch.einsum("bdn,bdn->bd", new, Ct) + d["D"] * x[:, t]
            if z is not None:
                y = y * F.silu(z[:, t])
            if s.get("lengths") is not None:
                live = (t < s["lengths"])[:, None]
                y, new = torch.where(live, y, 0.0), torch.where(live[..., None], new, h)
            h = new
            ys.append(y)
        y = torch.stack(ys, 1)
        if op == "scan_step":
            return dict(y=y[:, 0], state=h)
        out = dict(y=y, final_state=h)
        if train:
            names = ["x", "dt", "A", "Bm", "C", "D", "dt_bias", "state"] + (["z"] if z is not None else [])
            gs = torch.autograd.grad([y, h], [d[k] for k in names], [d["dy"], d["dfinal"]])
            out.update(zip(["dx", "ddt", "dA", "dB", "dC", "dD", "ddt_bias", "dinit"] + (["dz"] if z is not None else []), gs))
        return {k: v.detach() for k, v in out.items()}
    if op.startswith("conv"):
        x = d["x"][:, None] if op == "conv_step" else d["x"]
        Bn, L, _ = x.shape
        K = d["w"].shape[1]
        ext = torch.cat([d["history"], x], 1)
        out = F.silu(F.conv1d(ext.transpose(1, 2), d["w"][:, None], d["b"], groups=ext.shape[2]).transpose(1, 2))
        if op == "conv_step":
            return dict(out=out[:, 0], history=ext[:, 1:])
        n = [L] * Bn if s["lengths"] is None else s["lengths"].tolist()
        new = torch.stack([ext[i, m:m + K - 1] for i, m in enumerate(n)])
        out = torch.stack([torch.cat([out[i, :m], torch.zeros_like(out[i, m:])]) for i, m in enumerate(n)])
        got = dict(out=out, history=new)
        if train:
            gs = torch.autograd.grad([out, new], [d[k] for k in ("x", "w", "b", "history")], [d["dout"], d["dnew"]])
            got.update(zip(("din", "dweight", "dbias", "dhistory"), gs))
        return {k: v.detach() for k, v in got.items()}
    pre = F.linear(d["x"], d["w"], d.get("b"))
    out = {"none": lambda v: v, "silu": F.silu, "softplus": lambda v: F.softplus(v, threshold=200.0),
           "relu2": lambda v: F.relu(v) ** 2}[case["act"]](pre)
    if s["r"] is not None:
        out = out + d["r"]
    got = dict(out=out)
    if train:
        names = ["x", "w"] + (["b"] if s["b"] is not None else [])
        got.update(zip(["dx", "dweight", "dbias"], torch.autograd.grad(out, [d[k] for k in names], d["dout"])))
    return {k: v.detach() for k, v in got.items()}
