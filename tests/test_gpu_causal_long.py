"""causal_conv and group_norm at sizes whose threads go through their loops more than once (runs of 16 and 32 positions, several rows a wave, several blocks a thread, more than 128 partial results), and
group_norm on strided inputs, against 64 bits with the bounds of test_gpu_causal_conv and test_gpu_group_norm."""
import pytest
import torch

import test_gpu_causal_conv as conv
import test_gpu_group_norm as norm

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# a thread takes 32 positions where 512 threads a compute unit are left, else 16 or 8: 16, 32, 32 (one channel a thread), 32
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,L,C,K", [(8, 1025, 1536, 4), (8, 2049, 1536, 3), (6, 2050, 1001, 8), (65, 300, 1000, 1)])
def test_conv(gpu, B, L, C, K, dtype):
    for act in (None, "silu"):
        conv.test_forward(gpu, B, L, C, K, act, dtype)
    conv.test_gradient(gpu, B, L, C, K, "silu", dtype)


# tokens: two and more rows a wave, in pairs and one by one (1024 fp32 values in four vectors of a lane); sequences: 16 and more positions a thread in blocks of four, 256 partial results and more
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("shape,groups", [((20001, 64), 2), ((20001, 96), 32), ((20001, 1024), 1), ((17003, 127), 1), ((8, 2048, 1536), 32), ((3, 4001, 960), 20), ((64, 700, 250), 5)])
def test_norm(gpu, shape, groups, dtype):
    for act in (None, "gelu"):
        norm.test_forward(gpu, shape, groups, act, dtype)
    norm.test_gradient(gpu, shape, groups, "silu", dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("view", [lambda t: t[:, :, :7, :24], lambda t: t[::2, 3:4], lambda t: t[:, 0], lambda t: t.transpose(1, 2), lambda t: t[..., 5:29], lambda t: t[:, :, :, ::2],
                                  lambda t: t[0:1].expand(6, 10, 14, 48), lambda t: t[:, :, 0, 1:33], lambda t: t[:, 0, 0], lambda t: t[:, 3, 1, 8:40], lambda t: t[:, 3, 1, 7:31], lambda t: t[:3].permute(1, 0, 2, 3)])
def test_norm_of_strided_inputs(gpu, view, dtype, monkeypatch):
    made = norm._inputs

    def strided(gpu, shape, dtype, seed=0):
        base = torch.randn(6, 10, 14, 48, generator=torch.Generator(device=gpu).manual_seed(seed), device=gpu).to(dtype)
        return dict(made(gpu, shape, dtype, seed), x=view(base))

    monkeypatch.setattr(norm, "_inputs", strided)
    shape = tuple(view(torch.empty(6, 10, 14, 48)).shape)
    for act in (None, "silu", "gelu"):
        norm.test_forward(gpu, shape, 4, act, dtype)
        norm.test_gradient(gpu, shape, 4, act, dtype)
