"""group_norm against the same in 64 bits.

A mean of n values is off by at most (log2 n + 24) U of the largest, d = x - mean by that and U of itself; rstd by 4 U and half the relative error of the variance (2 (log2 n + 24) U, sums of
squares of one sign, and what the mean is off by against sqrt(var)).  So with T = (log2 n + 24) U: xh is off by T (2 |xh| + largest / std) + 6 U |xh|."""
import math

import pytest
import torch

import causal_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32

SIZES = [((1, 1), 1), ((3, 5), 1), ((5, 24), 3), ((7, 48), 48), ((33, 1536), 24), ((9, 1002), 2), ((100, 61), 1), ((2, 4096), 1), ((3, 9000), 2), ((65, 768), 768 // 24), ((4, 3584), 1),
         ((1, 2, 8), 2), ((2, 1, 40), 4), ((3, 7, 30), 5), ((2, 100, 96), 8), ((1, 1000, 61), 1), ((4, 33, 1536), 32), ((2, 5, 6, 64), 4), ((2, 3000, 16), 2), ((1, 300, 1002), 6)]


def _inputs(gpu, shape, dtype, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed + sum(shape))
    C = shape[-1]
    x = torch.randn(*shape, generator=g, device=gpu) * (0.5 + torch.rand(C, generator=g, device=gpu)) + torch.randn(C, generator=g, device=gpu)
    return {"x": x.to(dtype), "weight": torch.randn(C, generator=g, device=gpu), "bias": torch.randn(C, generator=g, device=gpu)}


def _xh_error(x, groups, eps):
    """(xh, what it may be off by, rstd), of x in 64 bits"""
    N, C = x.shape[0], x.shape[-1]
    v = x.reshape(N, -1, groups, C // groups)
    n = v.shape[1] * v.shape[3]
    T = (math.log2(n) + 24) * R.U
    c = v - v.mean((1, 3), keepdim=True)
    r = 1 / torch.sqrt((c * c).mean((1, 3), keepdim=True) + eps)
    xh = c * r
    off = T * (2 * xh.abs() + v.abs().amax((1, 3), keepdim=True) * r) + 6 * R.U * xh.abs()
    return xh.reshape(x.shape), off.reshape(x.shape), r.expand_as(v).reshape(x.shape)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape,groups", SIZES)
def test_forward(gpu, shape, groups, act, dtype):
    import m2_amd
    for affine, eps in ((True, 1e-5), (False, 1e-3)):
        ins = _inputs(gpu, shape, dtype)
        w, b = (ins["weight"], ins["bias"]) if affine else (None, None)
        y = m2_amd.group_norm(ins["x"], groups, w, b, eps=eps, activation=act)
        d = R.doubles(ins, False)
        want = R.norm(d["x"], groups, d["weight"] if affine else None, d["bias"] if affine else None, eps, act)
        xh, off, _ = _xh_error(d["x"], groups, eps)
        wd, bd = (d["weight"].abs(), d["bias"].abs()) if affine else (1.0, 0.0)
        pre = wd * off + 2 * R.U * (wd * xh.abs() + bd)
        # slopes are at most 1.13; SiLU's and erf's own arithmetic is off by 7 U of the value, erf's tail by 4 U of pre; SiLU's exponential, for bf16, by 2 |pre| U more
        most = wd * xh.abs() + bd
        R.within("y", y, want, 1.13 * pre + ((11 + (2 * most if dtype == BF16 else 0)) * R.U * most if act else 0))
        assert y.dtype == dtype and y.is_contiguous()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", [None, "silu", "gelu"])
@pytest.mark.parametrize("shape,groups", SIZES)
def test_gradient(gpu, shape, groups, act, dtype):
    """g = gy act'(pre): |act''| <= 0.8, its own arithmetic 12 U (1 + |pre|), for bf16 2 |pre| U more of that.  gw, gb: sums of N S terms, off by (log2 of them + 64) U of their magnitudes (a thread adds up to 64 in a row) and by their
    terms' errors.  gx = r (t - mean t - xh mean(t xh)): the same with n terms of a group, and the errors of r, xh and t in each place."""
    import m2_amd
    ins = _inputs(gpu, shape, dtype, seed=3)
    gy = torch.randn(*shape, generator=torch.Generator(device=gpu).manual_seed(9), device=gpu).to(dtype)
    d = R.doubles(ins)
    want = R.norm(d["x"], groups, d["weight"], d["bias"], 1e-5, act)
    wx, ww, wb = torch.autograd.grad(want, [d["x"], d["weight"], d["bias"]], gy.double())
    mine = {k: t.detach().requires_grad_() for k, t in ins.items()}
    gx, gw, gb = torch.autograd.grad(m2_amd.group_norm(mine["x"], groups, mine["weight"], mine["bias"], activation=act), list(mine.values()), gy)
    x, w, b = (t.detach() for t in d.values())
    xh, off, r = _xh_error(x, groups, 1e-5)
    pre = (w * xh).abs() + b.abs()
    g = gy.double().abs() * 1.13
    g_off = gy.double().abs() * (0.8 * (w.abs() * off + 2 * R.U * pre) + (12 + (2 * pre if dtype == BF16 else 0)) * R.U * (1 + pre)) if act else torch.zeros_like(g)
    lead = tuple(range(x.dim() - 1))
    count = x.numel() // x.shape[-1]
    T = (math.log2(count) + 64) * R.U
    R.within("weight", gw, ww, (g * off + g_off * xh.abs() + T * g * xh.abs()).sum(lead))
    R.within("bias", gb, wb, (g_off + T * g).sum(lead))
    N, C = x.shape[0], x.shape[-1]
    t, t_off = g * w.abs(), g_off * w.abs() + R.U * g * w.abs()

    def mean(v):
        m = v.reshape(N, -1, groups, C // groups)
        return m.mean((1, 3), keepdim=True).expand_as(m).reshape(v.shape)

    n = x[0].numel() // groups
    Tn = (math.log2(n) + 64) * R.U
    m1, m2 = mean(t), mean(t * xh.abs())
    m1_off, m2_off = mean(t_off) + Tn * m1, mean(t_off * xh.abs() + t * off) + Tn * m2
    size = t + m1 + xh.abs() * m2
    # r itself is off by (4 U + the variance's part), which is off / |xh| at most where xh is its group's largest: T' = (log2 n + 24) U (2 + largest / std)
    r_off = (4 * R.U + (math.log2(n) + 24) * R.U * (2 + mean((x.abs().reshape(N, -1, groups, C // groups).amax((1, 3), keepdim=True)).expand(N, x[0].numel() // C, groups, C // groups).reshape(x.shape)) * r))
    R.within("x", gx, wx, r * (t_off + m1_off + xh.abs() * m2_off + off * m2 + (r_off + 4 * R.U) * size))


def test_large_mean(gpu):
    """Values 1000 with a spread of 1: the mean's own rounding is 2^-24 of 1000, no square of it cancels."""
    import m2_amd
    for shape, groups in (((64, 256), 4), ((2, 500, 64), 4)):
        x = torch.randn(*shape, device=gpu, generator=torch.Generator(device=gpu).manual_seed(2)) + 1000
        y = m2_amd.group_norm(x, groups)
        _, off, _ = _xh_error(x.double(), groups, 1e-5)
        R.within("y", y, R.norm(x.double(), groups), off)
        assert off.max() < 0.01


def test_strides(gpu):
    import m2_amd
    base = torch.randn(6, 10, 14, 48, device=gpu)
    for x in (base[:, :, :7, :24], base[::2, 3:4], base[:, 0], base.transpose(1, 2), base[..., 5:29], base[:, :, :, ::2], base[0:1].expand(6, 10, 14, 48), base[:, :, 0, 1:33]):
        for dtype in (F32, BF16):
            v = x.to(dtype) if dtype == BF16 else x
            a, b = v.detach().requires_grad_(), v.detach().clone(memory_format=torch.contiguous_format).requires_grad_()
            p, q = m2_amd.group_norm(a, 4, activation="silu"), m2_amd.group_norm(b, 4, activation="silu")
            g = torch.randn_like(q)
            R.within("y", p.detach(), q.detach().double(), 2 * R.half_step(dtype) * q.detach().double().abs() + 60 * R.U * (1 + q.detach().double().abs()) * (1 + v.double().abs().max()))
            R.within("gx", torch.autograd.grad(p, a, g)[0], torch.autograd.grad(q, b, g)[0].double(), (2 * R.half_step(dtype) + 200 * R.U) * 20)


def test_not_finite_stays_in_its_group(gpu):
    import m2_amd
    for shape in ((5, 64), (5, 30, 64)):
        x = torch.randn(*shape, device=gpu)
        clean = m2_amd.group_norm(x, 4)
        x[2, ..., 20] = float("nan")
        y = m2_amd.group_norm(x, 4)
        hit = torch.zeros_like(x, dtype=torch.bool)
        hit[2, ..., 16:32] = True
        assert torch.isnan(y[hit]).all() and torch.equal(y[~hit], clean[~hit])


def test_nothing(gpu):
    import m2_amd
    x = torch.empty(0, 7, 16, device=gpu, requires_grad=True)
    w = torch.ones(16, device=gpu, requires_grad=True)
    y = m2_amd.group_norm(x, 4, w)
    gx, gw = torch.autograd.grad(y.sum(), [x, w])
    assert y.shape == x.shape and gx.shape == x.shape and not gw.any()
