"""What Int4Linear may lose: nothing of a row beside values that meet codes of zero, and no more than a sum in fp32 does.

`kernel` of a size is what m2_int4_linear_fwd runs it on: few rows, more rows, or many rows in half precision (which take a workspace)."""
import math

import pytest
import torch

U = 2.0 ** -24                                  # half a step of fp32
SUMMED = [(1, 700, 768), (1, 8000, 1536), (3, 30522, 768), (4, 6200, 1000), (20, 4000, 768), (7, 30522, 520), (40, 2000, 768), (16, 960, 960), (16, 30522, 768), (48, 30522, 400), (64, 12000, 768), (64, 1100, 300)]


def weights(gpu, N, K, group, seed=0):
    g = torch.Generator().manual_seed(seed + N + 3 * K + group)
    codes = torch.randint(0, 16, (N, K), generator=g)
    scales = (torch.rand(N, -(-K // group), generator=g) * 0.02 + 0.001).to(torch.bfloat16)
    return codes, scales


def make(gpu, codes, scales, group):
    import m2_amd
    K = codes.shape[1]
    even = torch.nn.functional.pad(codes, (0, K % 2), value=8)
    packed = (even[:, 0::2] | even[:, 1::2] << 4).to(torch.uint8)
    w = (codes - 8).double() * scales.double().repeat_interleave(group, 1)[:, :K]
    return m2_amd.Int4Linear.from_packed(packed.to(gpu), scales.to(gpu), K, group), w.to(gpu)


def rows(gpu, M, K, dtype=torch.float32, seed=0):
    return torch.randn(M, K, generator=torch.Generator().manual_seed(seed + M + K)).to(gpu).to(dtype)


def many(M, N, K, dtype):
    from m2_amd._lib import lib
    return lib.m2_int4_workspace_bytes(M, N, K, 0 if dtype == torch.float32 else 1) > 0


def of_sums(K, group, many):
    """n products added one after the other, partial sums growing as a walk, are off by U sqrt(n / 6) of their result in the root mean square (roundings of
    U / sqrt(3) of partial sums sqrt(j)); the groups' sums are added in the same way, and the result is rounded once.  A quarter is left for seeds.  In half
    precision n is K, and a row's values, cut to two halves, are off by 2 U at most, in the root mean square below U."""
    n = K if many else min(group, K)
    return 1.25 * U * (math.sqrt(n / 6) + math.sqrt(math.ceil(K / group) / 6) + 1 + many)


def test_the_bound_notices_lost_bits():
    """Rows cut to 18 bits are outside of it, also where it is widest."""
    codes, scales = weights(None, 400, 1024, 64)
    w = (codes - 8).double() * scales.double().repeat_interleave(64, 1)
    x = torch.randn(20, 1024, generator=torch.Generator().manual_seed(3))
    cut = x.view(torch.int32).bitwise_and(-64).view(torch.float32)
    y = x.double() @ w.t()
    assert (cut.double() @ w.t() - y).pow(2).mean().sqrt() / y.pow(2).mean().sqrt() > of_sums(1024, 64, True)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype,M,N,K", [(t, *size) for t in (torch.float32, torch.bfloat16) for size in SUMMED if t == torch.bfloat16 or size not in ((48, 30522, 400), (64, 12000, 768))])
def test_large_values_on_codes_of_zero(gpu, dtype, group, M, N, K):
    """Such a product is exactly 0 and a sum with it what it was: not a bit of the result changes (where rows are not taken in half precision)."""
    assert not many(M, N, K, dtype)
    codes, scales = weights(gpu, N, K, group)
    places = [0, 37, K // 2, K - 1]
    codes[:, places] = 8
    lin, w = make(gpu, codes, scales, group)
    x = rows(gpu, M, K, dtype)
    x[:, places] = 0
    want = lin(x)
    for power in (4, 12, 20, 26, 60):
        for p, place in enumerate(places):
            x[:, place] = 2.0 ** power * (1 + p / 8)
        assert torch.equal(lin(x), want), power


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", SUMMED + [(40, 30522, 768), (200, 30522, 768), (20, 40000, 512), (64, 1792, 5000), (128, 1792, 1792), (512, 3000, 1000)])
@pytest.mark.parametrize("kind", ["normal", "one sign", "mean"])
def test_errors_are_those_of_sums(gpu, group, M, N, K, kind):
    codes, scales = weights(gpu, N, K, group)
    lin, w = make(gpu, codes, scales, group)
    x = rows(gpu, M, K)
    x = x.abs() if kind == "one sign" else x + 8 if kind == "mean" else x
    y = x.double() @ w.t()
    err = (lin(x).double() - y).pow(2).mean().sqrt() / y.pow(2).mean().sqrt()
    assert err <= of_sums(K, group, many(M, N, K, torch.float32)), err


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(3, 2000, 512), (20, 40000, 512), (200, 40000, 512), (64, 16000, 1500), (512, 3000, 1000)])
def test_scales_far_below_their_rows_largest(gpu, dtype, group, M, N, K):
    """Rows that have nothing where scales are large get what the small scales give, to the errors of their sums and the result's rounding.  bf16 scales of 8 bits have
    them all in half precision down to 2^-27 of the largest (half a unit of its last place is 2^-25 where that is 2^10, and their last bit 2^-8 of them).
    Where rows are few a result is 16 times a sum that is kept in steps of 2^-149: each of the additions of groups and parts is off by up to 2^-150 more, times 16 2^-146.  That shows below 2^-122."""
    for power, offset in ((20, 0), (26, 0), (26, 100), (22, -110), (20, 125)):
        codes, scales = weights(gpu, N, K, group)
        s = scales.float() / 0.021 * 2.0 ** offset
        s[:, 0] = 2.0 ** offset
        s[:, 1:] = s[:, 1:] * 2.0 ** (1 - power) + 2.0 ** (offset - power)
        scales = s.to(torch.bfloat16)
        lin, w = make(gpu, codes, scales, group)
        x = rows(gpu, M, K, dtype)
        x[:, :group] = 0
        y = x.double() @ w.t()
        err = (lin(x).double() - y).pow(2).mean().sqrt() / y.pow(2).mean().sqrt()
        tol = of_sums(K, group, many(M, N, K, dtype)) + (torch.finfo(dtype).eps / 2 if dtype == torch.bfloat16 else 0)
        tol += 2.0 ** -146 * (math.ceil(K / group) + 8) / y.pow(2).mean().sqrt()
        assert err <= tol, (power, offset, err)


@pytest.mark.gpu
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(3, 2000, 512), (20, 40000, 512), (200, 40000, 512), (64, 16000, 1500), (512, 3000, 1000), (130, 30522, 640), (256, 8192, 1024), (512, 8192, 700), (512, 30522, 400)])
def test_fp32_values_far_below_their_rows_largest(gpu, group, M, N, K):
    """A few large values on codes of zero.  In half precision the others are off by 2 U of themselves where they are 2^-27 of the largest or more (the root mean square of that is
    the 1 that is added), smaller ones by 2^-50 of it: 2^-26 at most here, beside rows of size 1."""
    for power in (12, 18, 22, 24):
        codes, scales = weights(gpu, N, K, group)
        codes[:, [0, K // 2, K - 1]] = 8
        lin, w = make(gpu, codes, scales, group)
        x = rows(gpu, M, K)
        x[:, [0, K // 2, K - 1]] = 2.0 ** power
        y = x.double() @ w.t()
        err = (lin(x).double() - y).pow(2).mean().sqrt() / y.pow(2).mean().sqrt()
        assert err <= of_sums(K, group, many(M, N, K, torch.float32)), (power, err)
