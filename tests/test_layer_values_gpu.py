"""Values of the layer operators at the ends of their range: infinities, NaN, a type's lowest value, the tails of the activations, bits
that have to stay as they are."""
import pytest
import torch

from oracle import layer_oracle as O

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TD = {"fp32": torch.float32, "bf16": torch.bfloat16}
dev = lambda v: None if v is None else v.to(DEV)


@pytest.mark.parametrize("C", [16, 128])                 # the register kernels and the staged ones
@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_silu_of_the_convolution_keeps_its_tails(lib, dtype, C):
    """Weights that pick one row, so that the pre-activation is the input exactly and the output silu of it.  Relative bound: half a step
    of the storage type; exp of an argument a that was multiplied by log2 e and rounded, (2 + 1.5 |a|) 2^-23; sum, reciprocal and
    product, 4 2^-23.  An absolute error of 2^-12 of the sigmoid would be most of silu(-8)."""
    from trading_bot_0_b200 import prepost as P
    t, K = TD[dtype], 3
    a = torch.linspace(-40, 40, 641 * C).to(t)
    x = a.view(1, 641, C)
    w = torch.zeros(C, K)
    w[:, -1] = 1.0
    v = x.double()
    ref, half = v * torch.sigmoid(v), torch.finfo(t).eps / 2
    tol = ref.abs() * (half + (6 + 1.5 * v.abs()) * 2.0 ** -23 * (1 + half)) + 1e-37
    out, _ = P.conv1d_carry_forward(dev(x), dev(w))
    over = ((out.double().cpu() - ref).abs() - tol).max().item()
    assert over <= 0, f"forward: {over:.3e} over the bound"
    step = P.conv1d_step(torch.zeros(641, K - 1, C, dtype=t, device=DEV), dev(x[0]), dev(w))
    assert torch.equal(step, out[0])
    many = dev(x[0]).repeat(40, 1)                       # streams enough for a thread to take several, the last ones fewer
    some = P.conv1d_step(torch.zeros(len(many), K - 1, C, dtype=t, device=DEV), many, dev(w))
    assert torch.equal(some.view(40, 641, C), step.expand(40, 641, C))
