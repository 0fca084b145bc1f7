"""Selective scan with a decay per channel and state, the Mamba-1 form of the recurrence that ssd.py evaluates with one decay per
head.  Per batch row and channel d (group g), with state h [dstate]:

    s = act(dt + dt_bias);   h_t[n] = exp(s A[d, n]) h_{t-1}[n] + s x B_t[g, n];   y_t = (sum_n C_t[g, n] h_t[n] + D x) silu(z_t)

x, dt, z, y [batch, seqlen, channels] and B, C [batch, seqlen, ngroups, dstate] (or [batch, seqlen, dstate] for one group) in bf16
or fp32 with rows that may lie apart; A [channels, dstate], D, dt_bias, states and their gradients fp32; dstate at most 64.  All
arithmetic is fp32.  `lengths` (int32 [batch] on the device): tokens at or past a row's length are not read, leave its state as it
is, and get zeros as output and as gradient.  The calls only enqueue work on the current stream and may be captured into a graph.
"""
from __future__ import annotations

from . import _lib as L


def selective_scan_forward(x, dt, A, Bm, Cm, D=None, z=None, init_state=None, *, dt_bias=None, dt_softplus=False, lengths=None,
                           for_backward=False, workspace=None):
    """y, final_state [batch, channels, dstate], workspace.  With `for_backward` the workspace has room for the states that the
    backward starts from; a `workspace` handed in has to have that size for it too (see SsdSelBwdPtrs.fwd_saved)."""
    return L.host().selscan_forward(x, dt, A, Bm, Cm, D, z, init_state, dt_bias, dt_softplus, lengths, for_backward, workspace)


def selective_scan_backward(dy, x, dt, A, Bm, Cm, D=None, z=None, init_state=None, dfinal_state=None, *, dt_bias=None,
                            dt_softplus=False, lengths=None, workspace=None):
    """Gradients as a dict: dx, ddt, dB, dC, dz in the storage type, dA, dD, dinit, ddt_bias fp32 (those whose operand was given).
    `workspace`: what the forward with for_backward=True returned for these inputs; without it the states are computed again."""
    return L.host().selscan_backward(dy, x, dt, A, Bm, Cm, D, z, init_state, dfinal_state, dt_bias, dt_softplus, lengths, workspace)


def selective_scan(x, dt, A, Bm, Cm, D=None, z=None, init_state=None, *, dt_bias=None, dt_softplus=False, lengths=None):
    """Differentiable, once: returns (y, final_state)."""
    return L.host().selscan(x, dt, A, Bm, Cm, D, z, init_state, dt_bias, dt_softplus, lengths)


def selective_step(state, x, dt, A, Bm, Cm, D=None, z=None, *, y=None, dt_bias=None, dt_softplus=False):
    """One token per stream, IN PLACE on `state` [streams, channels, dstate] fp32; x, dt, z [streams, channels], B, C
    [streams, ngroups, dstate] or [streams, dstate].  Returns y; a `y` given may be x, dt or z itself, and shares no memory with an operand
    or the state otherwise."""
    return L.host().selscan_step(state, x, dt, A, Bm, Cm, D, z, y, dt_bias, dt_softplus)
