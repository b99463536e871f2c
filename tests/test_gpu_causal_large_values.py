"""The causal mixer's operators on values near the end of fp32's range whose results are well within it."""
import pytest
import torch

import causal_reference as R
import test_gpu_group_norm as norm

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("shape,groups,dtype", [((5, 64), 4, F32), ((3, 200, 64), 4, F32), ((2, 3000, 48), 3, F32), ((2, 1, 9, 6), 2, F32), ((5, 64), 4, BF16), ((3, 200, 64), 16, BF16), ((2, 300, 48), 24, BF16),
                                                ((2, 1, 9, 6), 2, BF16)])
def test_norm_of_large_means(gpu, shape, groups, dtype):
    """Means of 1.5 2^64, whose squares pass fp32's range, with spreads whose squares do not: up to 3 times 2^57 (bf16; a sum of 800 squares of 2^58 on average is 2^125.6) or 2^52 (fp32; 48000: 2^121.6)."""
    import m2_amd
    g = torch.Generator(device=gpu).manual_seed(3)
    steps = torch.randint(-3, 4, shape, generator=g, device=gpu).double()
    x = (2.0 ** 64 * (1.5 + steps * 2.0 ** (-7 if dtype == BF16 else -12))).to(dtype)
    y = m2_amd.group_norm(x, groups)
    xh, off, _ = norm._xh_error(x.double(), groups, 1e-5)
    R.within("y", y, xh, off)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_silu_of_large_values(gpu, dtype):
    """x sigmoid(x) is x, or nothing (below 2^-100), far from 0; its slope 1 or nothing."""
    import m2_amd
    x = torch.tensor([-3e38, -1e38, -1e36, -1e30, -1e20, -1000.0, -200.0, -100.0, 100.0, 1000.0, 1e20, 1e38, 3e38], device=gpu).to(dtype)
    one = torch.ones(1, 1, device=gpu)
    leaf = x.view(1, -1, 1).clone().requires_grad_()
    y = m2_amd.causal_conv(leaf, one, activation="silu")
    want = torch.where(x > 0, x, torch.zeros_like(x))
    assert ((y.flatten().double() - want.double()).abs() <= 2.0 ** -100 + R.half_step(dtype) * want.double()).all(), y
    slope, = torch.autograd.grad(y, leaf, torch.ones_like(y))
    assert ((slope.flatten().double() - (x > 0).double()).abs() <= 2.0 ** -20).all(), slope
    assert torch.equal(m2_amd.causal_conv_step(x.view(-1, 1), torch.empty(x.numel(), 0, 1, device=gpu, dtype=dtype), one, activation="silu").flatten(), y.flatten())
    z = x.view(1, -1, 1)
    ones = torch.ones_like(z)
    gated = m2_amd.selective_scan(ones, ones, -one, torch.zeros_like(z), torch.zeros_like(z), D=one[0], z=z)
    assert ((gated.flatten().double() - want.double()).abs() <= 2.0 ** -100 + 2 * R.half_step(dtype) * want.double()).all(), gated
