"""A layer's projection with its epilogue: out = act(x W^T + bias) + residual, and its gradients.

x [.., in_features], weight [out_features, in_features], bias, residual and out in one storage type (bf16 or fp32); products are
added in fp32 and the result is rounded once.  bf16 rows that start on 16 bytes run on the tensor cores, other sizes and strides and
fp32 on the CUDA cores.  `activation` is "none", "silu", "softplus" or "relu2" (max(v, 0) squared).

Every wait inside the tensor-core kernel is bounded.  When one runs out the outputs are NaN; these calls own their workspaces, so that is
the only sign of it here (a caller of the C entry points reads the workspace's status word).
"""
from __future__ import annotations

from . import _lib as L

ACTIVATIONS = {"none": 0, "silu": 1, "softplus": 2, "relu2": 3}


def _act(name):
    if name not in ACTIVATIONS:
        raise ValueError(f"linear: unknown activation {name!r}; one of {', '.join(ACTIVATIONS)}")
    return ACTIVATIONS[name]


def linear_forward(x, weight, bias=None, residual=None, *, activation="none", for_backward=False, out=None):
    """out, pre.  `pre` = x W^T + bias in fp32, kept for the backward of an activation (else None): in bf16 its rounding would go
    through the activation's slope into every gradient, beside that of dpre, which the products read in the storage type."""
    return L.host().linear_forward(x, weight, bias, residual, _act(activation), for_backward, out)


def linear_backward(dout, x, weight, pre=None, *, activation="none", bias=True, want_dx=True, want_dweight=True):
    """dx, dweight, dbias (None where not wanted); the gradient of the residual is dout.  In bf16 with an activation dout act'(pre) is rounded
    to bf16 as the products' operand, which adds as much to the error of dx and dweight as rounding them does (0.0023 of their size in all
    where the latter alone gives 0.0017); dbias is summed before that."""
    return L.host().linear_backward(dout, x, weight, pre, _act(activation), want_dx, want_dweight, bias)


def linear(x, weight, bias=None, residual=None, *, activation="none"):
    """Differentiable, once."""
    return L.host().linear(x, weight, bias, residual, _act(activation))
