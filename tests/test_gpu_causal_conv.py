"""causal_conv and causal_conv_step against the same in 64 bits.

An output is a chain of K fused products behind a bias: each of K roundings is half a step of a partial sum, which is at most S = |bias| + sum |w x|, so `pre` is off by
K U S.  SiLU's slope is at most 1.1; its own arithmetic (an exponential whose argument has been rounded and corrected, a sum, a reciprocal, a product: 1.5, 0.5, 1 and
0.5 steps of 2 U) is off by 7 U |y|.  For bf16 results the argument, x log2 e, is not corrected: rounded twice (log2 e, the product) it is off by |x| log2 e 2 U at most, the exponential by
|x| 2 U of itself, and y by that: (7 + 2 |pre|) U |y|."""
import pytest
import torch

import causal_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _inputs(gpu, B, L, C, K, dtype, bias=True, state=False, ragged=False, seed=0, pad=0):
    g = torch.Generator(device=gpu).manual_seed(seed * 101 + B + L + C + K)

    def randn(*s):
        return torch.randn(*s, generator=g, device=gpu)

    x = randn(B, L, C + pad).to(dtype)[..., pad:]
    lengths = None
    if ragged:
        lengths = torch.randint(0, L + 1, (B,), generator=g, device=gpu)
        lengths[0] = L
        if B > 1:
            lengths[1] = 0
        if B > 2:
            lengths[2] = min(1, L)
    return {"x": x, "weight": randn(C, K), "bias": randn(C) if bias else None, "state": randn(B, K - 1, C).to(dtype) if state else None}, lengths


def _bounds(ins, lengths, act, y):
    a = {k: None if t is None else t.detach().double().abs() for k, t in ins.items()}
    S, _ = R.conv(a["x"], a["weight"], a["bias"], None, a["state"], lengths)
    K = ins["weight"].shape[1]
    return 1.1 * K * R.U * S + ((7 + (2 * S if ins["x"].dtype == BF16 else 0)) * R.U * y.abs() if act else 0)


SIZES = [(1, 1, 1, 1), (1, 1, 64, 4), (2, 3, 7, 4), (3, 31, 24, 2), (4, 33, 100, 3), (2, 257, 1002, 4), (5, 100, 768, 5), (1, 300, 129, 6), (2, 65, 66, 7), (3, 40, 1536, 8),
         (1, 5000, 16, 4), (2, 1025, 8, 1)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("B,L,C,K", SIZES)
def test_forward(gpu, B, L, C, K, act, dtype):
    import m2_amd
    for bias, state, ragged, pad in ((True, False, False, 0), (False, True, True, 0), (True, True, True, 3), (True, True, False, 8)):
        ins, lengths = _inputs(gpu, B, L, C, K, dtype, bias, state, ragged, pad=pad)
        y, last = m2_amd.causal_conv(ins["x"], ins["weight"], ins["bias"], act, ins["state"], lengths, return_state=True)
        d = R.doubles(ins, False)
        want, end = R.conv(d["x"], d["weight"], d["bias"], act, d["state"], lengths)
        R.within("y", y, want, _bounds(ins, lengths, act, want))
        assert y.dtype == dtype and torch.equal(last.double(), end)
        assert torch.equal(m2_amd.causal_conv(ins["x"], ins["weight"], ins["bias"], act, ins["state"], lengths), y)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("act", [None, "silu"])
@pytest.mark.parametrize("B,L,C,K", SIZES)
def test_gradient(gpu, B, L, C, K, act, dtype):
    """Each gradient is a sum of products g w or g x, g = gy act'(pre).  g is off by 8 U of itself (the slope's arithmetic; for bf16 2 |pre| U more) and by half of gy for each unit that pre is
    off (|act''| <= 0.5); a sum of n terms of magnitudes M by n U M at most (n: K taps and the state's gradient, or all B L positions, of which one thread adds up to 32, then
    a tree of less)."""
    import m2_amd
    for bias, state, ragged, pad in ((True, True, True, 0), (False, False, False, 8), (True, True, False, 3)):
        ins, lengths = _inputs(gpu, B, L, C, K, dtype, bias, state, ragged, pad=pad, seed=1)
        g = torch.Generator(device=gpu).manual_seed(5)
        gy = torch.randn(B, L, C + pad, generator=g, device=gpu).to(dtype)[..., pad:]
        gl = torch.randn(B, K - 1, C, generator=g, device=gpu).to(dtype)
        names = [k for k, t in ins.items() if t is not None and t.numel()]
        d = R.doubles(ins)
        want = R.conv(d["x"], d["weight"], d["bias"], act, d["state"], lengths)
        outs, given = (list(want), [gy.double(), gl.double()]) if K > 1 else ([want[0]], [gy.double()])
        wants = dict(zip(names, torch.autograd.grad(outs, [d[k] for k in names], given)))
        mine = {k: None if t is None else t.detach().requires_grad_() for k, t in ins.items()}
        y, last = m2_amd.causal_conv(mine["x"], mine["weight"], mine["bias"], act, mine["state"], lengths, return_state=True)
        outs, given = ([y, last], [gy, gl]) if K > 1 else ([y], [gy])
        gots = dict(zip(names, torch.autograd.grad(outs, [mine[k] for k in names], given)))
        # magnitudes: |g| with what pre may be off by, through the same sums of absolute values
        a = {k: None if t is None else t.detach().double().abs().requires_grad_() for k, t in ins.items()}
        S, end = R.conv(a["x"], a["weight"], a["bias"], None, a["state"], lengths)
        G = gy.double().abs() * 1.1
        E = ((8 + (2 * S.detach() if dtype == BF16 else 0)) * R.U * G + 0.5 * gy.double().abs() * K * R.U * S.detach()) if act else torch.zeros_like(G)
        for name in names:
            n = K + 1 if name in ("x", "state") else min(B * L, 32) + B * L // 32
            total, = torch.autograd.grad([S, end] if K > 1 else [S], [a[name]], [G * n * R.U + E, gl.double().abs() * n * R.U] if K > 1 else [G * n * R.U + E], retain_graph=True)
            R.within(name, gots[name], wants[name], total)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,C,K", [(1, 1, 1), (1, 1536, 4), (3, 77, 2), (130, 1002, 3), (7, 64, 8), (0, 5, 4)])
def test_step(gpu, B, C, K, dtype):
    """Steps give what the whole gives, bit for bit where nothing rounds differently: the chain of products is the same."""
    import m2_amd
    ins, _ = _inputs(gpu, B, 6, C, K, dtype, state=True, pad=2)
    for act in (None, "silu"):
        whole, last = m2_amd.causal_conv(ins["x"], ins["weight"], ins["bias"], act, ins["state"], return_state=True)
        state = ins["state"].clone()
        for t in range(6):
            kept, other = state.clone(), torch.empty_like(state)
            apart = m2_amd.causal_conv_step(ins["x"][:, t], state, ins["weight"], ins["bias"], act, out_state=other)
            assert torch.equal(state, kept)
            y = m2_amd.causal_conv_step(ins["x"][:, t], state, ins["weight"], ins["bias"], act)
            assert torch.equal(y, apart) and torch.equal(state, other) and torch.equal(y, whole[:, t])
        assert torch.equal(state, last)


def test_parts_give_the_whole(gpu):
    import m2_amd
    ins, _ = _inputs(gpu, 2, 100, 96, 4, BF16)
    whole, last = m2_amd.causal_conv(ins["x"], ins["weight"], ins["bias"], "silu", return_state=True)
    state, parts = None, []
    for a, b in ((0, 1), (1, 3), (3, 64), (64, 100)):
        y, state = m2_amd.causal_conv(ins["x"][:, a:b], ins["weight"], ins["bias"], "silu", state, return_state=True)
        parts.append(y)
    assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(state, last)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_lies_behind_the_end_is_not_read(gpu, bad):
    import m2_amd
    ins, _ = _inputs(gpu, 4, 50, 40, 4, F32, state=True)
    lengths = torch.tensor([0, 1, 33, 50], device=gpu)
    ok = R.inside(lengths, 4, 50, gpu)
    gy = torch.randn(4, 50, 40, device=gpu)
    results = []
    for fill in (0.0, bad):
        mine = {k: t.detach().requires_grad_() for k, t in dict(ins, x=torch.where(ok, ins["x"], torch.full_like(ins["x"], fill))).items()}
        y, last = m2_amd.causal_conv(mine["x"], mine["weight"], mine["bias"], "silu", mine["state"], lengths, return_state=True)
        grads = torch.autograd.grad([y, last], list(mine.values()), [torch.where(ok, gy, torch.full_like(gy, fill)), torch.ones_like(last)])
        results.append([y.detach(), last.detach(), *grads])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    assert not results[0][0].masked_select(~ok).any() and not results[0][2].masked_select(~ok).any()


def test_a_value_that_is_not_finite_stays_with_its_taps(gpu):
    import m2_amd
    for K in range(1, 9):
        x = torch.randn(1, 40, 16, device=gpu)
        w = torch.randn(16, K, device=gpu)
        clean = m2_amd.causal_conv(x, w)
        x[0, 17, 3] = float("inf")
        y = m2_amd.causal_conv(x, w)
        hit = torch.zeros(1, 40, 16, dtype=torch.bool, device=gpu)
        hit[0, 17:17 + K, 3] = True
        assert not torch.isfinite(y[hit]).any() and torch.equal(y[~hit], clean[~hit])


def test_lengths_outside_count_as_the_nearest(gpu):
    import m2_amd
    ins, _ = _inputs(gpu, 3, 9, 8, 4, F32)
    a = m2_amd.causal_conv(ins["x"], ins["weight"], lengths=torch.tensor([-5, 10 ** 12, 4], device=gpu), return_state=True)
    b = m2_amd.causal_conv(ins["x"], ins["weight"], lengths=torch.tensor([0, 9, 4], device=gpu), return_state=True)
    assert all(torch.equal(p, q) for p, q in zip(a, b))
