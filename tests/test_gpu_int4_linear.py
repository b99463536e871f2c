"""Products with 4-bit weights against fp64, from codes and scales of the test's own."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                                  # half a step of fp32


def weights(gpu, N, K, group, seed=0):
    """(codes (N, K) 0 .. 15, scales bf16, what from_packed takes of the codes, W in fp64)"""
    g = torch.Generator().manual_seed(seed + N + 3 * K + group)
    codes = torch.randint(0, 16, (N, K), generator=g)
    codes[0, :] = torch.arange(K) % 16
    scales = (torch.rand(N, -(-K // group), generator=g) * 0.02 + 0.001).to(torch.bfloat16)
    even = torch.nn.functional.pad(codes, (0, K % 2), value=5)              # what stands behind the last column is not read
    packed = (even[:, 0::2] | even[:, 1::2] << 4).to(torch.uint8)
    w = (codes - 8).double() * scales.double().repeat_interleave(group, 1)[:, :K]
    return codes, scales.to(gpu), packed.to(gpu), w.to(gpu)


def gelu(v):
    return torch.special.ndtr(v) * v


def check(got, x, w, scales, group, bias=None, act=None):
    """Sums of K products of random signs: every one of the up to 2 K additions rounds a partial sum of a group, of values up to 16 + 15 and 24 times a
    row's largest, in the root mean square sqrt(group) of them, by less than U; eight standard deviations of the walk.  Then the sums of groups (no larger),
    the bias, GELU (slope below 1.13, erf to 4 ulp of values up to 1) and the result's own rounding."""
    K = x.shape[-1]
    x2 = x.double().reshape(-1, K)
    y = x2 @ w.t() + (0 if bias is None else bias.double())
    size = x2.abs().amax(1, keepdim=True) * scales.double().amax(1)
    tol = 8 * U * 55 * math.sqrt(min(group, K)) * math.sqrt(2 * K + 64) * size + 4 * U * (0 if bias is None else bias.double().abs())
    if act == "gelu":
        tol = 1.13 * tol + 8 * U * y.abs()
        y = gelu(y)
    tol = tol + torch.finfo(x.dtype).eps / 2 * y.abs() + 1e-40
    assert got.dtype == x.dtype and got.shape == (*x.shape[:-1], w.shape[0])
    err = (got.double().reshape(y.shape) - y).abs()
    assert (err <= tol).all(), (err / tol).max()


def rows(gpu, *shape, seed=0, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed + sum(shape))).to(gpu).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 128), (2, 17, 129), (3, 15, 31), (4, 64, 96), (5, 100, 960), (8, 33, 257), (15, 48, 768), (16, 250, 1000), (17, 31, 640),
                                   (33, 257, 768), (64, 130, 320), (65, 96, 1792), (130, 259, 200), (1, 30522, 768), (7, 1000, 4097), (1, 300, 8192), (300, 513, 384), (600, 1100, 768), (1030, 70, 136), (150, 30522, 768), (1030, 1793, 1792), (18, 30522, 776)])
def test_against_fp64(gpu, dtype, group, M, N, K):
    import m2_amd
    codes, scales, packed, w = weights(gpu, N, K, group)
    x, bias = rows(gpu, M, K, dtype=dtype), rows(gpu, N, dtype=torch.float32)
    lin = m2_amd.Int4Linear.from_packed(packed, scales, K, group, bias)
    check(lin(x), x, w, scales, group, bias)
    check(lin(x, activation="gelu"), x, w, scales, group, bias, "gelu")
    check(m2_amd.Int4Linear.from_packed(packed, scales, K, group)(x), x, w, scales, group)


@pytest.mark.parametrize("M,N", [(20, 1200), (64, 1200), (120, 1200), (256, 1200), (512, 1200), (300, 1800), (100, 10_000), (50, 6000), (50, 20_000), (130, 30_522)])
@pytest.mark.parametrize("K", [5, 100, 300, 520, 1000, 1403])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts_of_long_rows(gpu, dtype, M, N, K):
    """Sizes that are shared out differently, over rows, columns and parts of K, parts with no tile among them."""
    import m2_amd
    _, scales, packed, w = weights(gpu, N, K, 64)
    x = rows(gpu, M, K, dtype=dtype)
    check(m2_amd.Int4Linear.from_packed(packed, scales, K, 64)(x), x, w, scales, 64)


@pytest.mark.parametrize("M,N,K", [(100, 1200, 3403), (512, 1200, 5003), (256, 4000, 3003), (512, 4096, 1792), (300, 30_522, 400), (64, 8192, 4096), (40, 30_522, 500), (64, 30_522, 300), (90, 16_000, 800), (128, 16_000, 400), (128, 30_522, 400)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_parts_of_large_products(gpu, dtype, M, N, K):
    import m2_amd
    for group in (32, 128):
        _, scales, packed, w = weights(gpu, N, K, group)
        x, bias = rows(gpu, M, K, dtype=dtype), rows(gpu, N, dtype=torch.float32)
        check(m2_amd.Int4Linear.from_packed(packed, scales, K, group, bias)(x, activation="gelu"), x, w, scales, group, bias, "gelu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N", [(1, 70), (6, 70), (40, 70), (200, 70), (300, 51001)])
def test_rows_any_distance_apart(gpu, dtype, M, N):
    import m2_amd
    K, group = 200, 64
    _, scales, packed, w = weights(gpu, N, K, group)
    lin = m2_amd.Int4Linear.from_packed(packed, scales, K, group)
    room = rows(gpu, M + 2, K + 9, dtype=dtype)
    for x in (room[:M, :K], room[:M, 1:K + 1], room[1:M + 1, 8:K + 8], room[:1, 3:K + 3].expand(M, K), room.flatten()[5:5 + M * K].view(M, K),
              room[:M, :K].t().contiguous().t(), room[:M, :K].unflatten(0, (1, M)), room[:2 * (M // 2), :K].unflatten(0, (-1, 2))[:, 1:] if M > 1 else room[:1, :K]):
        check(lin(x), x, w, scales, group)
        assert torch.equal(lin(x), lin(x.contiguous().clone()))
    both = rows(gpu, 3, M, 2 * K, dtype=dtype)[:, : max(1, M - 1), K // 2:K // 2 + K]      # rows at two distances
    check(lin(both), both, w, scales, group)
    again = room[:M, :K].expand(3, M, K)          # the same rows three times over
    check(lin(again), again, w, scales, group)
    v = rows(gpu, K, dtype=dtype)
    check(lin(v), v, w, scales, group)
    assert lin(room[:0, :K]).shape == (0, N)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N", [(1, 48), (5, 48), (20, 48), (100, 48), (300, 33500)])
def test_each_code_in_each_place(gpu, dtype, M, N):
    """Unit rows: column k of W comes back exactly, whatever the order of the codes."""
    import m2_amd
    K, group = 300, 32
    codes, scales, packed, w = weights(gpu, N, K, group)
    lin = m2_amd.Int4Linear.from_packed(packed, scales, K, group)
    assert torch.equal(lin.dequantized().double(), w)
    x = torch.eye(K, device=gpu).to(dtype)
    for k in range(0, K, M):
        got, want = lin(x[k:k + M]), w[:, k:k + M].t()
        if dtype == torch.float32:
            assert torch.equal(got.double(), want)
        else:
            assert torch.equal(got, want.float().to(dtype))      # the value rounded once
    # constant rows: sums of up to 16 + 15 and 24 each, every addition off by U of at most 55 K
    for v in (1.0, -3.0):
        c = torch.full((M, K), v, device=gpu, dtype=dtype)
        y = v * w.sum(1)
        tol = U * 2 * group * 55 * abs(v) * scales.double().sum(1) * group + torch.finfo(dtype).eps / 2 * y.abs()
        assert ((lin(c).double() - y).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M,N", [(1, 100), (4, 100), (5, 100), (30, 100), (90, 100), (300, 100), (16, 17000), (30, 17000), (300, 17000)])
def test_rows_are_their_own(gpu, dtype, M, N):
    """A row's bits do not depend on the rows beside it; NaN and infinities stay in their row."""
    import m2_amd
    K, group = 768, 64
    _, scales, packed, w = weights(gpu, N, K, group)
    lin = m2_amd.Int4Linear.from_packed(packed, scales, K, group)
    x = rows(gpu, M + 2, K, dtype=dtype)
    clean = lin(x)
    x[M, 5] = float("nan")
    x[M + 1, 700] = float("inf")
    dirty = lin(x)
    assert torch.equal(dirty[:M], clean[:M]) and torch.isnan(dirty[M]).all() and not torch.isfinite(dirty[M + 1]).any()
    zero = torch.zeros(M, K, device=gpu, dtype=dtype)
    assert (lin(zero) == 0).all()


@pytest.mark.parametrize("M,N", [(6, 40), (30, 40), (300, 2700)])
def test_bits_of_fp32_rows(gpu, M, N):
    """The low bits of a row take part: rows that differ from bf16 ones by parts of 2^-9 and 2^-17."""
    import m2_amd
    K, group = 512, 128
    _, scales, packed, w = weights(gpu, N, K, group)
    lin = m2_amd.Int4Linear.from_packed(packed, scales, K, group)
    g = torch.Generator().manual_seed(2)
    x = (torch.randint(-2 ** 23, 2 ** 23, (M, K), generator=g).double() * 2.0 ** -20).float().to(gpu)
    check(lin(x), x, w, scales, group)
    for scale in (2.0 ** 100, 2.0 ** -100):
        check(lin(x * scale), x * scale, w, scales, group)
    one = torch.zeros(M, K, device=gpu)
    one[0, 77] = 1 + 2.0 ** -23
    got, want = lin(one)[0].double(), one[0, 77].double() * w[:, 77]
    if M < 300:
        assert torch.equal(got, want.float().double())
    else:      # two exact products in one sum of the matrix unit, which is off by less than its last bit whatever way it rounds
        assert ((got - want).abs() < 2.0 ** -23 * want.abs() + 1e-40).all()


def test_offsets_beyond_32_bits(gpu):
    """Rows of x 2^30 + 40 values apart, and a weight of more than 2^31 bytes, of which the last rows are looked at."""
    import m2_amd
    from m2_amd import ops
    N, K, group = 33, 96, 32
    _, scales, packed, w = weights(gpu, N, K, group)
    lin = m2_amd.Int4Linear.from_packed(packed, scales, K, group)
    room = torch.empty(2 * (2 ** 30 + 40) + K, dtype=torch.bfloat16, device=gpu)
    x = room.as_strided((3, K), (2 ** 30 + 40, 1))
    x.copy_(rows(gpu, 3, K))
    check(lin(x), x, w, scales, group)
    del room, x
    N, K, group = 64 * 1024, 65536, 128
    _, scales, packed, w = weights(gpu, 16, K, group)
    last = m2_amd.Int4Linear.from_packed(packed, scales, K, group)
    big = torch.zeros(ops.int4_weight_bytes(N, K, group), dtype=torch.uint8, device=gpu)
    assert big.numel() > 2 ** 31
    tiles = 16 * 4                                # bytes of the rows' factors, behind all tiles
    big[-N * 4:].view(torch.float32).fill_(1.0)
    big[-tiles:] = last.weight[-tiles:]
    big[-(N // 16 - 1) * tiles - last.weight.numel():-(N // 16) * tiles] = last.weight[:-tiles]
    for M in (1, 20, 200):
        x = rows(gpu, M, K)
        got = ops.int4_linear(x, big, N, group)
        check(got[:, -16:], x, w, scales, group)
        assert (got[:, :-16] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N", [40, 40_000])
def test_ranges_of_rows_and_scales(gpu, dtype, N):
    """Rows and scales of any size, and rows and groups of sizes far apart: errors stay relative to the largest of each."""
    import m2_amd
    K, group = 512, 64
    codes, scales, packed, w = weights(gpu, N, K, group)
    powers = torch.tensor([2.0 ** (5 * (i % 40 - 20)) for i in range(N)], device=gpu)[:, None]       # 2^-100 .. 2^95, row by row
    wide = (scales.float() * powers * torch.tensor([1, 2.0 ** -4, 2.0 ** -12, 1, 2.0 ** -30, 1, 0, 1], device=gpu)).to(torch.bfloat16)
    w = (codes.to(gpu) - 8).double() * wide.double().repeat_interleave(group, 1)
    lin = m2_amd.Int4Linear.from_packed(packed, wide, K, group)
    for M in (3, 20, 200):
        x = rows(gpu, M, K, dtype=dtype)
        x[:, ::3] *= 2.0 ** -9
        x = x * torch.tensor([2.0 ** (i % 9 - 4) for i in range(M)], device=gpu, dtype=dtype)[:, None]
        y = x.double() @ w.t()
        size = x.double().abs().amax(1, keepdim=True) * wide.double().amax(1)
        tol = 8 * U * 55 * math.sqrt(group) * math.sqrt(2 * K + 64) * size + torch.finfo(dtype).eps / 2 * y.abs() + 1e-37
        assert ((lin(x).double() - y).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_powers_that_cancel(gpu, dtype):
    """Rows whose largest value, 2^115, meets codes that stand for zero, times scales of 2^38; rows of 2^-140 times scales of 2^60: what comes out is in range."""
    import m2_amd
    M, N, K, group = 200, 40_000, 512, 64
    codes, scales, packed, w = weights(gpu, N, K, group)
    codes[:, 0] = 8
    packed = (codes[:, 0::2] | codes[:, 1::2] << 4).to(torch.uint8).to(gpu)
    for big, small, power in ((2.0 ** 115, 2.0 ** 80, 38), (2.0 ** -140, 2.0 ** -140, 60)):
        s = (scales.float() * 2.0 ** power).to(torch.bfloat16)
        lin = m2_amd.Int4Linear.from_packed(packed, s, K, group)
        x = (rows(gpu, M, K, dtype=torch.float32) * small).to(dtype)
        x[:, 0] = big
        y = x.double() @ ((codes.to(gpu) - 8).double() * s.double().repeat_interleave(group, 1)).t()
        most = s.double().abs().amax(1)
        size = x[:, 1:].double().abs().amax(1, keepdim=True) * most
        # a row's values become multiples of 2^-24 where its largest is 2^14 or more: each is off by 2^-39 of the largest at most, and is taken 8 times a scale
        largest = x.double().abs().amax(1, keepdim=True)
        tol = 8 * U * 55 * math.sqrt(group) * math.sqrt(2 * K + 64) * size + K * 8 * 2.0 ** -39 * largest * most + torch.finfo(dtype).eps / 2 * y.abs()
        got = lin(x).double()
        assert torch.isfinite(got).all() and ((got - y).abs() <= tol).all()


def test_factors_are_powers_of_two(gpu):
    """Weights laid out on the GPU hold the same bytes as on the CPU, scales of all sizes."""
    import m2_amd
    exponents = torch.arange(-126, 128)
    scales = torch.ldexp(torch.full((254,), 1.25), exponents).to(torch.bfloat16)[:, None]
    codes = torch.randint(0, 256, (254, 16), dtype=torch.uint8, generator=torch.Generator().manual_seed(0))
    a, b = (m2_amd.Int4Linear.from_packed(codes.to(d), scales.to(d), 32, 32).weight.cpu() for d in ("cpu", gpu))
    assert torch.equal(a, b)
    factor = b[-256 * 4:].view(torch.float32)
    assert (torch.frexp(factor).mantissa == 0.5).all() and torch.equal(torch.frexp(factor[:254]).exponent, 1 - (exponents + 1).clamp(-120, 120).to(torch.int32))


def test_views_of_negatives(gpu):
    """Rows whose memory holds the negatives of their values, as imaginary parts of conjugates do."""
    import m2_amd
    for M, K in ((3, 200), (20, 200), (2, 1)):
        _, scales, packed, w = weights(gpu, 50, K, 32)
        lin = m2_amd.Int4Linear.from_packed(packed, scales, K, 32)
        x = rows(gpu, M, K, dtype=torch.float32)
        for v in (torch._neg_view(-x), torch.complex(x, -x).conj().imag):
            assert v.is_neg() and torch.equal(lin(v), lin(x))


def test_what_is_around_stays(gpu):
    import m2_amd
    from m2_amd import ops
    from m2_amd._lib import check as ok, lib
    for M, N, K, dtype in ((1, 17, 70, torch.bfloat16), (3, 50, 768, torch.float32), (37, 30, 129, torch.bfloat16), (100, 77, 96, torch.float32), (513, 70, 200, torch.bfloat16), (200, 130, 160, torch.float32), (200, 30522, 520, torch.bfloat16),
                           (40, 30522, 408, torch.float32)):
        _, scales, packed, w = weights(gpu, N, K, 32)
        lin = m2_amd.Int4Linear.from_packed(packed, scales, K, 32)
        x = rows(gpu, M, K, dtype=dtype)
        room = torch.full((M * N + 64,), 7.0, device=gpu, dtype=dtype)
        workspace = torch.empty(lib.m2_int4_workspace_bytes(M, N, K, 1 if dtype == torch.bfloat16 else 0) + 16, dtype=torch.uint8, device=gpu)
        ok(lib.m2_int4_linear_fwd(x.data_ptr(), K, lin.weight.data_ptr(), None, room.data_ptr() + 32 * room.element_size(), workspace.data_ptr(), M, N, K, 32, 0,
                                  1 if dtype == torch.bfloat16 else 0, ops._stream()))
        assert (room[:32] == 7).all() and (room[-32:] == 7).all()
        check(room[32:-32].view(M, N), x, w, scales, 32)


def test_from_weights(gpu):
    """Quantized weights are half a step of their group's scale off (a step and a half where the scale's rounding pushes a code out); the module keeps them."""
    import m2_amd
    g = torch.Generator().manual_seed(1)
    linear = torch.nn.Linear(330, 70)
    with torch.no_grad():
        linear.weight[3] = 0                      # groups of zeros
        linear.weight[4, 64:] = 0
    lin = m2_amd.Int4Linear.from_linear(linear.to(gpu), 64)
    w = lin.dequantized()
    padded = torch.nn.functional.pad(linear.weight.detach(), (0, -330 % 64)).view(70, -1, 64)
    step = (padded.abs().amax(-1, keepdim=True) / 7 * (1 + 2.0 ** -8)).expand_as(padded).reshape(70, -1)[:, :330]
    assert ((w - linear.weight.detach()).abs() <= step * (0.5 + 7 * 2.0 ** -7)).all()
    assert (w[3] == 0).all()
    x = torch.randn(5, 330, generator=g).to(gpu)
    with torch.no_grad():
        y = lin(x)
        ref = x.double() @ w.double().t() + linear.bias.double()
    assert (y.double() - ref).abs().max() < 1e-4
    other = m2_amd.Int4Linear(330, 70, group_size=64, device=gpu)
    other.load_state_dict(lin.state_dict())
    assert torch.equal(other(x), y)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        assert torch.equal(lin(x), lin(x.to(torch.bfloat16)))
    moved = m2_amd.Int4Linear.from_linear(linear.cpu(), 64).to(gpu).to(torch.bfloat16)      # only the bias changes its type
    assert torch.equal(moved.weight, lin.weight) and moved(x).dtype == torch.float32


def test_captured_beside_eager_calls_and_streams(gpu):
    import m2_amd
    for M, N, K in ((1, 96, 1536), (6, 500, 768), (50, 300, 256), (400, 12000, 768)):
        _, scales, packed, w = weights(gpu, N, K, 64)
        lin = m2_amd.Int4Linear.from_packed(packed, scales, K, 64)
        xs = [rows(gpu, M, K, seed=s) for s in range(3)]
        want = [lin(x) for x in xs]
        a = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            lin(a)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = lin(a)
        for turn in range(4):
            a.copy_(xs[turn % 3])
            torch.cuda.synchronize()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                graph.replay()
            eager = lin(xs[1])
            torch.cuda.synchronize()
            assert torch.equal(out, want[turn % 3]) and torch.equal(eager, want[1])


def test_refusals(gpu):
    import m2_amd
    from m2_amd import ops
    lin = m2_amd.Int4Linear(64, 10, device=gpu)
    x = torch.randn(2, 64, device=gpu)
    for bad, error in ((x.cpu(), RuntimeError), (x.half(), TypeError), (x[:, :63], ValueError), (x[0, 0], ValueError), (x[:, :0], ValueError)):
        with pytest.raises(error):
            lin(bad)
    with pytest.raises(ValueError):
        lin(x, activation="relu")
    with pytest.raises(RuntimeError, match="no gradient"):
        lin(x.clone().requires_grad_())
    with pytest.raises(RuntimeError):
        m2_amd.Int4Linear(64, 10)(x)                                       # its weight on the CPU
    with pytest.raises(RuntimeError):
        torch.func.vmap(lin)(x)
    with pytest.raises(ValueError):
        ops.int4_linear(x, lin.weight[:-1], 10, 64)
    with pytest.raises(ValueError):
        ops.int4_linear(x, lin.weight, 10, 48)
    one = m2_amd.Int4Linear(1, 1, device=gpu)
    with pytest.raises(RuntimeError, match="more workgroups than a launch holds"):
        one(torch.zeros(1, 1, device=gpu, dtype=torch.bfloat16).expand(2 ** 30, 1))
