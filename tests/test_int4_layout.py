"""The order of 4-bit weights in memory, and what the entry points refuse before anything is launched."""
import ctypes

import pytest
import torch


def _code_at(weight, N, K, group, n, k):
    """The code of W[n, k] by the words of the header."""
    kt = (K + 127) // 128
    tile = (n // 16 * kt + k // 128) * (1024 + 16 * (128 // group) * 2)
    kk = k % 128
    lane, j = 16 * (kk // 8 % 4) + n % 16, kk % 8
    word = int.from_bytes(bytes(weight[tile + lane * 16 + kk // 32 * 4:][:4].tolist()), "little")
    scale = tile + 1024 + (n % 16 * (128 // group) + kk // group) * 2
    return word >> (16 * (j % 2) + 4 * (j // 2)) & 15, int.from_bytes(bytes(weight[scale:scale + 2].tolist()), "little")


@pytest.mark.parametrize("N,K,group", [(1, 1, 32), (17, 129, 64), (40, 300, 128), (16, 128, 32)])
def test_codes_and_scales_lie_where_the_header_says(N, K, group):
    import m2_amd
    from m2_amd import ops
    g = torch.Generator().manual_seed(N + 1)
    codes = torch.randint(0, 16, (N, K + K % 2), generator=g)
    scales = torch.rand(N, -(-K // group), generator=g).to(torch.bfloat16)
    lin = m2_amd.Int4Linear.from_packed((codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8), scales, K, group)
    assert lin.weight.numel() == ops.int4_weight_bytes(N, K, group)
    bits = scales.view(torch.int16).to(torch.int32) & 0xFFFF
    for n in range(N):
        for k in range(0, K, 7):
            assert _code_at(lin.weight, N, K, group, n, k) == (codes[n, k].item(), bits[n, k // group].item())
    factor = lin.weight[-(-N // 16) * 16 * -4:].view(torch.float32)
    most = scales.float().amax(1) * factor[:N]
    assert (torch.frexp(factor).mantissa == 0.5).all() and ((most >= 0.5) & (most < 1) | (scales == 0).all(1)).all()
    last = (-(-N // 16) * 16 - 1, -(-K // 128) * 128 - 1)
    if N % 16 and K % 128:
        assert _code_at(lin.weight, N, K, group, *last) == (8, 0)
    back, s = lin.packed()
    assert torch.equal(s, scales) and torch.equal(back & 15, codes[:, 0::2].to(torch.uint8))
    assert torch.equal((back >> 4)[:, :K // 2], codes[:, 1::2].to(torch.uint8)[:, :K // 2])


def test_quantized_values():
    import m2_amd
    w = torch.tensor([[7.0, -7.0, 3.4, -3.6, 0.0, 0.5, 1.5, -8.0 / 7 * 7]] + [[0.0] * 8] + [[1e-40] * 8])
    codes, scales = m2_amd.quantize_int4(w[:, :7], 32)
    assert scales.shape == (3, 1) and scales[0] == 1.0 and scales[1] == 0
    assert [(codes[0, i // 2] >> 4 * (i % 2) & 15).item() - 8 for i in range(7)] == [7, -7, 3, -4, 0, 0, 2]
    assert (codes[1] == 0x88).all()
    for bad in (torch.zeros(3), torch.zeros(0, 4), torch.zeros(2, 2, 2)):
        with pytest.raises(ValueError):
            m2_amd.quantize_int4(bad)
    with pytest.raises(ValueError):
        m2_amd.quantize_int4(w, 48)
    w[0, 0] = float("nan")                        # shows in every product with that group
    codes, scales = m2_amd.quantize_int4(w, 32)
    assert torch.isnan(scales[0]).all() and (codes[0] == 0x88).all()


def test_modules_refuse_what_does_not_fit():
    import m2_amd
    make = m2_amd.Int4Linear.from_packed
    codes, scales = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.bfloat16)
    make(codes, scales, 64, 64)
    make(codes, scales, 63, 64)
    for args in ((codes, scales, 65, 64), (codes, scales, 64, 32), (codes.int(), scales, 64, 64), (codes, scales.float(), 64, 64), (codes, scales[:3], 64, 64),
                 (codes, scales, 64, 16), (codes, scales, 64, 64, torch.zeros(5))):
        with pytest.raises(ValueError):
            make(*args)
    with pytest.raises(ValueError):
        m2_amd.Int4Linear(0, 4)
    with pytest.raises(RuntimeError, match="GPU"):
        m2_amd.Int4Linear(64, 4)(torch.zeros(1, 64))
    with pytest.raises(RuntimeError, match="GPU"):
        m2_amd.token_logprobs(torch.zeros(1, 64), torch.zeros(1, dtype=torch.int64))


def test_entry_points_refuse_before_a_launch():
    from m2_amd._lib import lib
    p, off = ctypes.c_void_p(4096), ctypes.c_void_p(4104)
    assert lib.m2_int4_weight_bytes(16, 128, 128) == 1024 + 32 + 64 and lib.m2_int4_weight_bytes(17, 129, 32) == 4 * (1024 + 128) + 128
    assert lib.m2_int4_weight_bytes(0, 128, 128) == 0 and lib.m2_int4_weight_bytes(4, 0, 32) == 0 and lib.m2_int4_weight_bytes(4, 4, 16) == 0
    assert lib.m2_int4_weight_bytes(2 ** 31 - 1, 2 ** 31 - 1, 128) == 2 ** 27 * (2 ** 24 * 1056 + 64)

    def linear(x=p, x_row=64, w=p, bias=None, out=p, M=1, N=16, K=64, group=64, gelu=0, dtype=1, workspace=None):
        return lib.m2_int4_linear_fwd(x, x_row, w, bias, out, workspace, M, N, K, group, gelu, dtype, None)

    need = lib.m2_int4_workspace_bytes
    assert need(1, 30522, 64, 1) == need(0, 64, 64, 1) == need(4096, 64, 0, 1) == need(4096, 64, 64, 1) == 0
    assert need(4097, 30522, 129, 1) == 257 * (2 * 4096 + 64) and need(4097, 30522, 129, 0) == 257 * (2 * 8192 + 64)
    assert linear(M=4096, N=30522) == -1 and b"workspace" in lib.m2_last_error() and linear(M=4096, N=30522, workspace=off) == -2

    assert linear(x=None) == linear(w=None) == linear(out=None) == -1 and b"null" in lib.m2_last_error()
    assert linear(M=0) == linear(N=-1) == linear(K=0) == linear(x_row=-1) == linear(dtype=2) == linear(gelu=2) == -1
    assert linear(group=16) == linear(w=off) == -2 and b"aligned" in lib.m2_last_error()
    assert linear(x=ctypes.c_void_p(4097)) == linear(out=ctypes.c_void_p(4097)) == linear(x=ctypes.c_void_p(4098), dtype=0) == -2
    assert linear(bias=ctypes.c_void_p(4098)) == -2

    def fwd(x=p, inner=1, outer=0, row=0, tokens=None, allowed=None, a_row=0, lp=None, h=p, stats=p, ids=None, top=None, rows=1, V=8, k=0, dtype=1):
        return lib.m2_token_scores_fwd(x, inner, outer, row, tokens, -100, allowed, a_row, lp, h, stats, ids, top, None, rows, V, k, dtype, None)

    assert fwd(x=None) == fwd(h=None) == fwd(stats=None) == fwd(tokens=p) == fwd(k=1) == fwd(k=1, ids=p) == -1
    assert fwd(rows=0) == fwd(V=0) == fwd(inner=0) == fwd(outer=-1) == fwd(row=-1) == fwd(dtype=2) == fwd(allowed=p, a_row=7) == -1
    assert fwd(k=9, ids=p, top=p) == fwd(V=100, k=33, ids=p, top=p) == fwd(k=-1) == fwd(x=ctypes.c_void_p(4097)) == fwd(V=2 ** 30 + 1) == -2

    def bwd(x=p, tokens=p, allowed=None, a_row=0, h=p, stats=p, ids=None, g=(None, None, None), grad=p, grad_row=8, rows=1, V=8, k=0, dtype=1, strides=(1, 1)):
        return lib.m2_token_scores_bwd(x, 1, 0, 0, tokens, -100, allowed, a_row, h, stats, ids, g[0], strides[0], g[1], strides[1], g[2], grad, grad_row, rows, V, k, dtype, None)

    assert bwd(x=None) == bwd(h=None) == bwd(stats=None) == bwd(grad=None) == bwd(grad_row=7) == bwd(rows=0) == -1
    assert bwd(g=(p, None, None), tokens=None) == bwd(g=(None, None, p)) == bwd(g=(None, None, p), k=2) == bwd(g=(p, p, None), strides=(-1, 1)) == -1
    assert bwd(grad=ctypes.c_void_p(4097)) == bwd(k=33, V=40, grad_row=40) == -2
