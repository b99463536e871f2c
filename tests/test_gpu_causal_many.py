"""The causal mixer's operators on many sequences."""
import pytest
import torch

import causal_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,C", [(65536, 3), (70001, 8)])
def test_conv_step_of_more_sequences_than_a_grid_s_second_dimension(gpu, B, C, dtype):
    """Against 64 bits: a chain of K products behind a bias, off by half a step of its partial sums each."""
    import m2_amd
    K = 3
    g = torch.Generator(device=gpu).manual_seed(C)
    x, state = (torch.randn(*s, generator=g, device=gpu).to(dtype) for s in ((B, C), (B, K - 1, C)))
    w, bias = torch.randn(C, K, generator=g, device=gpu), torch.randn(C, generator=g, device=gpu)
    rows = torch.cat([state, x.unsqueeze(1)], 1)
    y = m2_amd.causal_conv_step(x, state, w, bias)
    assert torch.equal(state, rows[:, 1:])
    products = rows.double() * w.double().t()
    R.within("y", y, products.sum(1) + bias.double(), K * R.U * (products.abs().sum(1) + bias.double().abs()))
