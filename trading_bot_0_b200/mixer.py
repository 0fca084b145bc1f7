"""Whole mixers of state space layers, from the layer's input to its output, over this library's operators: for training and prompts
(differentiable), and for one token per stream with the layer's state updated in place.

    mamba2_mixer / mamba2_mixer_step          projection -> conv + silu -> SSD scan (one decay per head), gated -> RMS norm -> projection
    selective_mixer / selective_mixer_step    projection -> conv + silu -> projections of step size, B and C -> selective scan (a decay per
                                              channel and state), gated -> projection

u [batch, seqlen, features] ([streams, features] for a step) in bf16 or fp32; projection weights in u's type, conv and norm weights, A, D
and dt_bias fp32, as the operators take them.  `residual` (u's shape) is added in the output projection's epilogue.

A training step may be captured into a CUDA graph, backward included, as long as no eager autograd graph of the same leaves is alive
during the capture: autograd then waits on the stream of that graph's accumulation nodes, which ends the capture.
"""
from __future__ import annotations

import torch

from .linear import linear, linear_forward
from .prepost import causal_conv1d_carry, conv1d_step, mamba2_mixer_core, rmsnorm, rmsnorm_forward
from .selective import selective_scan, selective_step
from .ssd import ssd_scan, state_update


def _project(x, weight, bias=None, residual=None):
    """linear outside of autograd: a step's convolution and scan have no gradient, and a graph of its projections alone would give
    part of one."""
    return linear_forward(x, weight, bias, residual)[0]


def _aligned(t):
    """`t` itself where its rows start on 16 bytes (what the conv and the tensor-core scan take), else a copy; a single row too has a
    stride that they look at."""
    e = t.element_size()
    ok = t.data_ptr() % 16 == 0 and all(t.stride(i) * e % 16 == 0 for i in range(t.dim() - 1))
    return t if ok else t.clone(memory_format=torch.contiguous_format)


def _mamba2_parts(zxbcdt, hp, gn):
    z, xBC, dt = zxbcdt[..., :hp], zxbcdt[..., hp:2 * hp + 2 * gn], zxbcdt[..., 2 * hp + 2 * gn:]
    return _aligned(z), _aligned(xBC), dt


def _last_rows(t, n):
    """The last n rows of t [batch, rows, channels], zeros before its first: the history that a convolution leaves."""
    rows = t.shape[1]
    last = t[:, rows - n:] if rows >= n else torch.nn.functional.pad(t, (0, 0, n - rows, 0))
    return last.clone(memory_format=torch.contiguous_format)     # (some rows of one sequence are contiguous where they are)


def mamba2_mixer(u, in_proj, conv_weight, conv_bias, dt_bias, A, D, norm_weight, out_proj, *, nheads, headdim, dstate, ngroups, residual=None,
                 in_bias=None, out_bias=None, chunk=128, eps=1e-5, algo="auto", history=None, state=None, return_history=False):
    """Differentiable.  in_proj gives the columns z (nheads*headdim) | x, B, C (nheads*headdim + 2*ngroups*dstate) | dt (nheads).
    `history` [batch, width-1, conv channels] and `state` [batch, nheads, headdim, dstate] continue an earlier call.  Returns out
    [batch, seqlen, out features] and the scan's final state; with `return_history` out, the new history and the state, which are what
    mamba2_mixer_step goes on with.  All rows of a batch are of one length (the scan takes no lengths)."""
    hp, gn, heads = nheads * headdim, ngroups * dstate, (nheads, headdim)
    z, xBC, dt = _mamba2_parts(linear(u, in_proj, in_bias), hp, gn)
    if history is None:
        y, final = mamba2_mixer_core(xBC, dt, z.unflatten(-1, heads), conv_weight, conv_bias, dt_bias, A, D, norm_weight, nheads=nheads,
                                     headdim=headdim, dstate=dstate, ngroups=ngroups, chunk=chunk, eps=eps, algo=algo, init_state=state)
        if return_history:
            history = _last_rows(xBC, conv_weight.shape[1] - 1)
    else:
        c, history = causal_conv1d_carry(xBC, conv_weight, conv_bias, history)
        x, Bm, Cm = c.split([hp, gn, gn], -1)
        y, final = ssd_scan(x.unflatten(-1, heads), dt, A, Bm.unflatten(-1, (ngroups, dstate)), Cm.unflatten(-1, (ngroups, dstate)), D,
                            z.unflatten(-1, heads), state, chunk=chunk, algo=algo, dt_bias=dt_bias, dt_softplus=True)
        y = rmsnorm(y.flatten(2), norm_weight, eps=eps)
    out = linear(y, out_proj, out_bias, residual)
    return (out, history, final) if return_history else (out, final)


def mamba2_mixer_step(u, history, state, in_proj, conv_weight, conv_bias, dt_bias, A, D, norm_weight, out_proj, *, nheads, headdim, dstate,
                      ngroups, residual=None, in_bias=None, out_bias=None, eps=1e-5):
    """One token per stream, IN PLACE on `history` [streams, width-1, conv channels] and `state` [streams, nheads, headdim, dstate].  No
    part of an autograd graph."""
    hp, gn = nheads * headdim, ngroups * dstate
    z, xBC, dt = _mamba2_parts(_project(u, in_proj, in_bias), hp, gn)
    c = conv1d_step(history, xBC, conv_weight, conv_bias)
    y = state_update(state, c[:, :hp].unflatten(1, (nheads, headdim)), dt, A, c[:, hp:hp + gn].unflatten(1, (ngroups, dstate)),
                     c[:, hp + gn:].unflatten(1, (ngroups, dstate)), D, z.unflatten(1, (nheads, headdim)), dt_bias=dt_bias, dt_softplus=True)
    y, _ = rmsnorm_forward(y.view(-1, hp), norm_weight, eps=eps)
    return _project(y, out_proj, out_bias, residual)


def _selective_parts(x, x_proj, dt_proj, dstate, project):
    dbc = project(x, x_proj)
    rank = dbc.shape[-1] - 2 * dstate
    return project(dbc[..., :rank], dt_proj), dbc[..., rank:rank + dstate], dbc[..., rank + dstate:]


def selective_mixer(u, in_proj, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, D, out_proj, *, residual=None, history=None, state=None,
                    lengths=None):
    """Differentiable.  in_proj gives the columns x | z (channels each), x_proj dt's factor (rank) | B | C (dstate each), dt_proj the
    channels' step sizes.  `history` [batch, width-1, channels] and `state` [batch, channels, dstate] continue an earlier call; `lengths`
    (int32 [batch] on the device) ends rows early: out is the residual there, or zero, and gradients are zeros; u has to be finite there all
    the same, since its rows take part in the projections' products.  Returns out, the new history and the new state."""
    D_, N = A.shape
    xz = linear(u, in_proj)
    x, history = causal_conv1d_carry(_aligned(xz[..., :D_]), conv_weight, conv_bias, history, lengths=lengths)
    dt, Bm, Cm = _selective_parts(x, x_proj, dt_proj, N, linear)
    y, state = selective_scan(x, dt, A, Bm, Cm, D, xz[..., D_:], state, dt_bias=dt_bias, dt_softplus=True, lengths=lengths)
    return linear(y, out_proj, None, residual), history, state


def selective_mixer_step(u, history, state, in_proj, conv_weight, conv_bias, x_proj, dt_proj, dt_bias, A, D, out_proj, *, residual=None):
    """One token per stream, IN PLACE on `history` [streams, width-1, channels] and `state` [streams, channels, dstate].  No part of an
    autograd graph."""
    D_, N = A.shape
    xz = _project(u, in_proj)
    x = conv1d_step(history, _aligned(xz[:, :D_]), conv_weight, conv_bias)
    dt, Bm, Cm = _selective_parts(x, x_proj, dt_proj, N, _project)
    y = selective_step(state, x, dt, A, Bm, Cm, D, xz[:, D_:], dt_bias=dt_bias, dt_softplus=True)
    return _project(y, out_proj, None, residual)
