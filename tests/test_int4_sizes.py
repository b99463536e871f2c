"""Sizes at which a product's offsets would pass 32 bits are refused before anything is launched."""
import ctypes

import pytest


def test_sizes_behind_2_30_are_refused():
    from m2_amd._lib import lib
    p = ctypes.c_void_p(4096)

    def linear(N, K, dtype):
        return lib.m2_int4_linear_fwd(p, 0, p, None, p, p, 1, N, K, 64, 0, dtype, None)

    for dtype in (0, 1):
        for N, K in ((2 ** 30 + 1, 64), (2 ** 31 - 1, 64), (16, 2 ** 30 + 1), (16, 2 ** 31 - 127), (16, 2 ** 31 - 1)):
            assert linear(N, K, dtype) == -2 and b"2^30" in lib.m2_last_error()


def test_modules_of_such_sizes_are_refused():
    import m2_amd
    for k, n in ((2 ** 30 + 1, 4), (4, 2 ** 30 + 1)):
        with pytest.raises(ValueError, match="2\\^30"):
            m2_amd.Int4Linear(k, n, device="meta")


@pytest.mark.gpu
def test_rows_of_such_sizes_are_refused(gpu):
    import torch
    from m2_amd import ops
    one = torch.zeros(1, device=gpu, dtype=torch.bfloat16)
    weight = torch.zeros(16, dtype=torch.uint8, device=gpu)
    with pytest.raises(ValueError, match="2\\^30"):
        ops.int4_linear(one.expand(1, 2 ** 30 + 1), weight, 16, 64)
    with pytest.raises(ValueError, match="2\\^30"):
        ops.int4_linear(one.expand(1, 64), weight, 2 ** 30 + 1, 64)
