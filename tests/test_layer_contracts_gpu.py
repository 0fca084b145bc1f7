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
