"""Log probabilities of given tokens, entropies and alternatives, and their gradient, against the definition in fp64."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24                                  # half a step of fp32
INF = float("inf")
BLOCK = 256                                     # threads that share a row: V / BLOCK values are summed one after the other


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def definition(logits, tokens, top_k, allowed, ignore=-100, grads=None):
    """Row by row in fp64 on the CPU: (lp, H, ids, top, gradient)."""
    V = logits.shape[-1]
    x = logits.detach().double().cpu().reshape(-1, V)
    t = None if tokens is None else tokens.cpu().reshape(-1)
    a = None if allowed is None else allowed.cpu().expand(logits.shape).reshape(-1, V)
    lps, hs, idss, tops, gr = [], [], [], [], []
    for r in range(x.shape[0]):
        z = x[r].clone()
        if a is not None:
            z[~a[r]] = -INF
        real = z != -INF                          # NaN is among them
        broken = bool(torch.isnan(z).any() or (z == INF).any())
        if broken:
            logp = torch.full_like(z, math.nan)
            h = torch.tensor(math.nan, dtype=torch.float64)
        elif not real.any():
            logp = torch.full_like(z, -INF)
            h = torch.tensor(0.0, dtype=torch.float64)
        else:
            logp = z - z[real].max()              # first: log V is lost beside values of 1e38
            logp = logp - torch.logsumexp(logp, 0)
            h = -(logp[real].exp() * logp[real]).sum()
        hs.append(h)
        order = [] if broken else torch.sort(torch.where(real, z, torch.tensor(-INF, dtype=z.dtype)), descending=True, stable=True).indices[:top_k].tolist()
        ids = [-1] * top_k if broken else [i if real[i] else -1 for i in order]
        idss.append(ids)
        tops.append([math.nan if broken else -INF if i < 0 else logp[i].item() for i in ids])
        bad = False
        if t is not None:
            ti = t[r].item()
            if ti == ignore:
                lps.append(0.0)
            elif not 0 <= ti < V:
                lps.append(math.nan)
                bad = True
            else:
                lps.append(logp[ti].item())
        if grads is not None:
            g_lp, g_h, g_top = [None if g is None else g.detach().double().cpu().reshape(x.shape[0], -1)[r] for g in grads]
            d = torch.zeros_like(z)
            if broken:
                d[real] = math.nan
            elif real.any():
                p = logp.exp()
                own = torch.zeros_like(z)
                if g_lp is not None and t[r].item() != ignore:
                    if bad:
                        own[:] = math.nan
                    else:
                        own[t[r]] += g_lp[0]
                total = own.sum()
                if g_top is not None:
                    for i, g in zip(ids, g_top):
                        if i >= 0:
                            own[i] += g
                            total = total + g
                gh = 0.0 if g_h is None else g_h[0]
                d = torch.where(real, own - p * total - gh * p * torch.where(real, logp + h, torch.zeros_like(z)), d)
            gr.append(d)
    lead = logits.shape[:-1]
    shape = lambda v, *more: torch.tensor(v, dtype=torch.float64).reshape((*lead, *more))      # noqa: E731
    return (None if t is None else shape(lps), torch.stack(hs).reshape(lead) if hs else shape([]), torch.tensor(idss, dtype=torch.int64).reshape((*lead, top_k)),
            shape(tops, top_k), torch.stack(gr).reshape(logits.shape) if gr else None)


def close(got, want, tol):
    got, want = got.detach().double().cpu(), want.float().double()      # (below the lowest fp32 value: -inf)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(got[inf], want[inf]) and not torch.isinf(got[~inf]).any()
    fine = ~inf & ~torch.isnan(want)
    err, tol = (got - want).abs()[fine], tol.expand(want.shape)[fine]
    assert (err <= tol).all(), (err / tol).max()


def compare(logits, tokens, top_k=0, allowed=None, grads=None, ignore=-100):
    import m2_amd
    x = logits.detach()
    if grads is not None:
        x = x.requires_grad_()
    r = m2_amd.token_logprobs(x, tokens, top_k, allowed, ignore)
    lp, h, ids, top, grad = definition(logits, tokens, top_k, allowed, ignore, grads)
    V = logits.shape[-1]
    # A log probability: the difference to the maximum and the product with log2 e round by |lp| or less, log and its sum by a few units; every exp of
    # the sum is off by its argument's rounding (weighted with the exp itself: below one unit of the sum) and one ulp; the sum's own roundings are
    # a random walk over V / BLOCK + 20 additions.  The entropy adds the same for sum e d, whose value is below log V + 1 times the sum.
    units = 16 + 4 * math.sqrt(V / BLOCK + 20)
    if lp is not None:
        close(r.logprobs, lp, U * (units + 4 * torch.nan_to_num(lp, posinf=0, neginf=0).abs()))
    close(r.entropy, h, U * units * 2 * torch.tensor(math.log(V) + 2, dtype=torch.float64))
    if top_k:
        assert torch.equal(r.top_ids.cpu(), ids)
        close(r.top_logprobs, top, U * (units + 4 * torch.nan_to_num(top, posinf=0, neginf=0).abs()))
    else:
        assert r.top_ids is None and r.top_logprobs is None
    assert tokens is not None or r.logprobs is None
    if grads is not None:
        outs = [(o, g) for o, g in zip((r.logprobs, r.entropy, r.top_logprobs), grads) if g is not None]
        got, = torch.autograd.grad([o for o, _ in outs], [x], [g for _, g in outs])
        assert got.shape == logits.shape and got.dtype == logits.dtype
        # p carries the log probability's error and its own; what it is multiplied with is at most the sum of the outputs' gradients, each with |lp| + H
        size = sum(g.detach().double().cpu().abs().reshape(*logits.shape[:-1], -1).sum(-1, keepdim=True) for g in grads if g is not None)
        z = logits.detach().double().cpu()
        logp = (z - torch.nan_to_num(z, nan=-INF, posinf=-INF).amax(-1, keepdim=True)).nan_to_num(0, 0, 0).abs() + math.log(V)
        p = torch.minimum(torch.ones_like(z), torch.exp(2 * math.log(V) - logp)) if allowed is None else torch.ones_like(z)
        tol = U * size * (8 + (units + 6 * logp) * (2 + logp + math.log(V)) * p) + _half_step(logits.dtype) * torch.nan_to_num(grad).abs() + 1e-37
        close(got, grad, tol)
    return r


def _logits(gpu, shape, dtype, seed=0, scale=2.0):
    g = torch.Generator(device=gpu).manual_seed(seed + sum(shape))
    x = torch.randn(*shape, generator=g, device=gpu) * scale - 6
    x.scatter_add_(-1, torch.randint(0, shape[-1], (*shape[:-1], 4), generator=g, device=gpu), torch.full((*shape[:-1], 4), 9.0, device=gpu))
    return x.to(dtype)


def _tokens(gpu, lead, V, seed=0):
    return torch.randint(0, V, lead, generator=torch.Generator().manual_seed(seed + V)).to(gpu)


def _grads(gpu, lead, top_k, seed=0):
    g = torch.Generator(device=gpu).manual_seed(seed + 5)
    rn = lambda *s: torch.randn(s, generator=g, device=gpu)      # noqa: E731
    return [rn(*lead), rn(*lead), rn(*lead, top_k) if top_k else None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V,top_k", [(1, 1, 1), (3, 2, 2), (2, 7, 3), (5, 8, 8), (2, 9, 1), (3, 63, 32), (2, 257, 5), (4, 1023, 32), (3, 2048, 10), (2, 2049, 0),
                                          (7, 8191, 17), (3, 30522, 5), (2, 30528, 32), (300, 1000, 4), (1, 65537, 8), (2, 131073, 32), (1, 262147, 20)])
def test_against_fp64(gpu, dtype, rows, V, top_k):
    x = _logits(gpu, (rows, V), dtype)
    compare(x, _tokens(gpu, (rows,), V), top_k, grads=_grads(gpu, (rows,), top_k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [5, 300, 4097, 30522])
@pytest.mark.parametrize("per_row", [False, True])
def test_allowed_tokens(gpu, dtype, V, per_row):
    rows, k = 9, min(V, 12)
    x = _logits(gpu, (rows, V), dtype)
    a = torch.rand((rows, V) if per_row else (V,), generator=torch.Generator().manual_seed(V)).to(gpu) < 0.6
    if per_row:
        a[1] = False                              # nothing left
        a[2] = False
        a[2, V - 1] = True                        # one left
        a[3] = False
        a[3, :2] = True
    else:
        a[V // 2] = True
    x[0][~(a[0] if per_row else a)] = float("nan")      # masked places may hold anything
    x[4][~(a[4] if per_row else a)] = INF
    x[5][~(a[5] if per_row else a)] = -INF
    compare(x, _tokens(gpu, (rows,), V), k, a, _grads(gpu, (rows,), k))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [3, 700, 30522])
def test_values_at_the_ends(gpu, dtype, V):
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    x = _logits(gpu, (12, V), dtype)
    x[0] = -INF
    x[1] = low                                    # a mask of the type's lowest value over the whole row: uniform
    x[2, 1:] = low
    x[3, 1:] = -INF
    x[4, V - 1] = float("nan")
    x[5, 0] = INF
    x[6, : V // 2] = -INF
    x[7] = high
    x[8, 0], x[8, 1:] = high, low
    x[9] = 0.0
    x[9, ::2] = -0.0                              # equal to 0: ties go by id
    x[10, V - 1] = high
    tokens = _tokens(gpu, (12,), V)
    tokens[3] = V - 1                             # a token of probability zero
    compare(x, tokens, min(V, 6), grads=_grads(gpu, (12,), min(V, 6)))


@pytest.mark.parametrize("rows,V", [(3, 30522), (700, 4000), (1, 200_003)])
def test_one_token_has_nearly_all(gpu, rows, V):
    """What the other tokens add to 1 is all of log s and of the entropy.  Eight values of a vector are added to the 1 among them in three steps, half a unit of
    its last bit each, and all others apart from it; each of the others is off by its argument's rounding, 2 units for each e-fold, below 30 of them."""
    import m2_amd
    x = _logits(gpu, (rows, V), torch.float32, scale=1.0) - 6
    x[:, V // 3] = torch.linspace(4, 22, rows, device=gpu)
    r = m2_amd.token_logprobs(x, torch.full((rows,), V // 3, device=gpu), 1)
    lp, h, ids, top, _ = definition(x, torch.full((rows,), V // 3), 1, None)
    assert torch.equal(r.top_ids.cpu(), ids)
    close(r.logprobs, lp, U * (4 + 64 * lp.abs()))
    close(r.entropy, h, U * (4 + 128 * h))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,V", [(1, 30522), (30, 30522), (700, 4003), (3000, 900), (2, 262147), (5, 17)])
def test_entropy_where_one_token_has_nearly_all(gpu, dtype, rows, V):
    """To its own last bits.  Each e^d is off by the rounding of d log2 e below 2^5, 2^-20 ln 2, by that constant's, 2^-26 of it, and by an ulp: 20 U in all; three sums of positive numbers
    in five steps each, U each; what stands beside a 1 loses four times U of that 1 and is mended where the rest is below 1 / 16, so up to 64 U of it."""
    import m2_amd
    x = _logits(gpu, (rows, V), torch.float32, scale=1.0) - 6
    at = torch.randint(0, V, (rows,), generator=torch.Generator().manual_seed(V)).to(gpu)
    if rows > 4:
        at[:3] = torch.tensor([0, V - 1, V - 2])
    x = x.scatter(1, at[:, None], torch.linspace(6, 14, rows, device=gpu)[:, None]).to(dtype)
    _, h, _, _, _ = definition(x, at.cpu(), 1, None)
    for top in (0, 3):
        r = m2_amd.token_logprobs(x, at, top)
        close(r.entropy, h, U * (20 + 15 + 64) * h)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,levels", [(4096, 1), (4096, 2), (30522, 3), (30522, 40), (70001, 1)])
def test_ties_go_to_the_lowest_id(gpu, dtype, V, levels):
    g = torch.Generator().manual_seed(V + levels)
    x = torch.randint(0, levels, (6, V), generator=g).to(gpu).to(dtype)
    x[1] = 0
    x[1, -3:] = 1                                 # the only ones above a level that fills the row
    x[2] = 0
    x[2, 5:5 + 40] = 1
    x[3] = torch.arange(V, device=gpu).flip(0).float().div(V).to(dtype)
    x[4] = torch.arange(V, device=gpu).float().div(V).to(dtype)
    x[5] = -INF
    x[5, V - 2000:] = 1
    for k in (1, 7, 32):
        compare(x, None, k)


@pytest.mark.parametrize("V", [8192, 30522])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_the_largest_in_few_places(gpu, dtype, V):
    """All large values next to one another, a fixed distance apart, or where one thread or one group of them meets them."""
    for start, step, count in ((0, 1, 200), (V - 200, 1, 200), (3, 8, 500), (1, 64, 100), (5, 512, 15), (0, 2048, 4), (7, 256, 30), (16, 1024, 7)):
        x = torch.randn(2, V, generator=torch.Generator().manual_seed(step)).to(gpu)
        at = torch.arange(start, min(V, start + step * count), step)
        x[0, at] += 20
        x[1, at] = 30 + (at.float() * 37 % 11).to(gpu)
        compare(x.to(dtype), None, 32)
    each = torch.arange(V, device=gpu)
    for group in (each // 8 % 64 == 3, each // 4 % 64 == 60, each // 8 % 256 == 255, each % 512 < 30):      # hundreds in one of the places that share a maximum
        x = torch.randn(2, V, generator=torch.Generator().manual_seed(9)).to(gpu)
        x[0, group] += 20
        x[1, group] = 30 + (each[group].float() * 37 % 11)
        compare(x.to(dtype), None, 32)
        compare(x.to(dtype), None, 3)


def test_tokens_that_are_none(gpu):
    import m2_amd
    x = _logits(gpu, (6, 1000), torch.float32)
    t = torch.tensor([-100, -1, 1000, 2 ** 40, 3, -2 ** 62], device=gpu)
    r = compare(x, t, 3, grads=_grads(gpu, (6,), 3))
    assert r.logprobs[0] == 0 and torch.isnan(r.logprobs[[1, 2, 3, 5]]).all()
    r = compare(x, t, 3, grads=_grads(gpu, (6,), 3), ignore=1000)
    assert r.logprobs[2] == 0 and torch.isnan(r.logprobs[0])
    r = compare(x, t, 3, grads=_grads(gpu, (6,), 3), ignore=3)      # a token of the vocabulary may be the one to ignore
    assert r.logprobs[4] == 0
    assert m2_amd.token_logprobs(x).logprobs is None


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_any_distance_apart(gpu, dtype):
    import m2_amd
    full = _logits(gpu, (4, 6, 1003), dtype)
    cases = [full[:, :, :1000], full[:, :, 3:], full[:, 1:, 1:], full[::2, 1:4, :997], full[1], full[1, 2], full.transpose(0, 1), full[:, :, ::2], full[:, :, :1],
             full[:1].expand(3, 6, 1003), full[:, 2:3, 5:], full.view(2, 2, 6, 1003)[:, 1, 2:], full.view(2, 2, 2, 3, 1003)[:, :1, :, 1:], full[2, 3, 7:8]]
    for x in cases:
        k = min(4, x.shape[-1])
        t = _tokens(gpu, x.shape[:-1], x.shape[-1])
        compare(x, t, k, grads=_grads(gpu, x.shape[:-1], k))
        dense = m2_amd.token_logprobs(x.contiguous(), t, k)
        got = m2_amd.token_logprobs(x, t, k)
        assert all(torch.equal(a, b) for a, b in zip(got, dense))
    a = torch.rand(4, 6, 1003, generator=torch.Generator().manual_seed(1)).to(gpu) < 0.5
    x, t = full[:, 1:, 2:], _tokens(gpu, (4, 5), 1001)
    compare(x, t, 4, a[:, 1:, 2:], _grads(gpu, (4, 5), 4))
    compare(x, t, 4, a[:1, :1, 2:].expand(4, 5, 1001), _grads(gpu, (4, 5), 4))
    compare(x, t.t().contiguous().t(), 4, a[0, 0, ::1][2:], _grads(gpu, (4, 5), 4))
    for lead in ((0,), (2, 0)):
        e = torch.empty(*lead, 50, device=gpu, dtype=dtype).requires_grad_()
        r = m2_amd.token_logprobs(e, torch.empty(*lead, dtype=torch.int64, device=gpu), 3)
        assert r.logprobs.shape == lead and r.top_ids.shape == (*lead, 3)
        r.logprobs.sum().backward()
        assert e.grad.shape == e.shape


def test_offsets_beyond_32_bits(gpu):
    """Rows 2^30 + 24 values apart: the third begins more than 2^32 bytes behind the first."""
    V, row = 517, 2 ** 30 + 24
    room = torch.empty(2 * row + V, dtype=torch.bfloat16, device=gpu)
    x = room.as_strided((3, V), (row, 1))
    x.copy_(_logits(gpu, (3, V), torch.bfloat16))
    compare(x, _tokens(gpu, (3,), V), 5, grads=_grads(gpu, (3,), 5))


def test_many_rows_and_nothing_behind_them(gpu):
    """More rows than a launch has workgroups in a dimension; what lies around the results is left alone."""
    from m2_amd import ops
    from m2_amd._lib import check, lib
    rows, V, k = 66_000, 19, 3
    x = _logits(gpu, (rows, V), torch.bfloat16)
    t = _tokens(gpu, (rows,), V)
    room = [torch.full((rows + 2,), 7.0, device=gpu), torch.full((rows + 2,), 7.0, device=gpu), torch.full((2 * rows + 2,), 7.0, device=gpu),
            torch.full((rows * k + 2,), 7, dtype=torch.int64, device=gpu), torch.full((rows * k + 2,), 7.0, device=gpu)]
    check(lib.m2_token_scores_fwd(x.data_ptr(), rows, 0, V, t.data_ptr(), -100, None, 0, *[r.data_ptr() + r.element_size() for r in room], None, rows, V, k, 1, ops._stream()))
    grad = torch.full((rows * (V + 4) + 8,), 7.0, dtype=torch.bfloat16, device=gpu)
    g = [v.contiguous() for v in _grads(gpu, (rows,), k)]
    check(lib.m2_token_scores_bwd(x.data_ptr(), rows, 0, V, t.data_ptr(), -100, None, 0, room[1].data_ptr() + 4, room[2].data_ptr() + 4, room[3].data_ptr() + 8,
                                  g[0].data_ptr(), 1, g[1].data_ptr(), 1, g[2].data_ptr(), grad.data_ptr() + 8, V + 4, rows, V, k, 1, ops._stream()))
    for r in room:
        assert r[0] == 7 and r[-1] == 7
    logp = x.double().log_softmax(-1)
    assert (room[0][1:-1].double() - logp.gather(-1, t[:, None])[:, 0]).abs().max() < U * 200
    assert torch.equal(room[3][1:-1].view(rows, k).sort(-1).values[:, 0] >= 0, torch.ones(rows, dtype=torch.bool, device=gpu))
    assert (grad[:4] == 7).all() and (grad[4:-4].view(rows, V + 4)[:, V:] == 7).all() and (grad[-4:] == 7).all()
    p, h = logp.exp(), -(logp.exp() * logp).sum(-1, keepdim=True)
    want = -p * (g[0][:, None].double() + g[2].double().sum(-1, keepdim=True) + g[1][:, None].double() * (logp + h))
    want.scatter_add_(-1, t[:, None], g[0][:, None].double())
    want.scatter_add_(-1, room[3][1:-1].view(rows, k), g[2].double())
    assert ((grad[4:-4].view(rows, V + 4)[:, :V].double() - want).abs() <= 2.0 ** -8 * want.abs() + U * 2000).all()


def test_gradient_against_differences(gpu):
    """Central differences of the operator itself.  A step e of a logit: rounding of the outputs U |f| / e, third derivative e^2 / 6 below 1 each."""
    import m2_amd
    rows, V, k, e = 2, 11, 3, 2.0 ** -7
    x = torch.randn(rows, V, generator=torch.Generator().manual_seed(3)).to(gpu)
    t, g = _tokens(gpu, (rows,), V), _grads(gpu, (rows,), k)

    def f(v):
        r = m2_amd.token_logprobs(v, t, k)
        return sum((o.double() * w.double()).sum() for o, w in zip((r.logprobs, r.entropy, r.top_logprobs), g))

    v = x.clone().requires_grad_()
    r = m2_amd.token_logprobs(v, t, k)
    torch.autograd.backward([r.logprobs, r.entropy, r.top_logprobs], g)
    size = sum(w.abs().sum().item() for w in g)
    for i in range(rows):
        for j in range(V):
            up, down = x.clone(), x.clone()
            up[i, j] += e
            down[i, j] -= e
            step = (up[i, j] - down[i, j]).double()
            d = (f(up) - f(down)) / step
            assert abs(d.item() - v.grad[i, j].item()) < size * (e * e + 40 * U / e)


def test_what_is_asked_for_alone(gpu):
    """Gradients of some outputs, of one output's sum (an expanded gradient), none, and of a part of the rows."""
    import m2_amd
    x, t = _logits(gpu, (5, 300), torch.float32), _tokens(gpu, (5,), 300)
    g = _grads(gpu, (5,), 4)
    for keep in ((0,), (1,), (2,), (0, 2), (1, 2)):
        compare(x, t, 4, grads=[v if i in keep else None for i, v in enumerate(g)])
    one = torch.ones((), device=gpu)
    compare(x, t, 4, grads=[one.expand(5), None, None])
    compare(x, t, 4, grads=[None, one.expand(5), one.expand(5, 4)])
    compare(x, t, 4, grads=[g[0][::1].repeat_interleave(2)[::2], None, g[2].t().contiguous().t()])
    v = x.clone().requires_grad_()
    r = m2_amd.token_logprobs(v, t, 4)
    assert not r.top_ids.requires_grad and r.logprobs.requires_grad
    r.logprobs[1:3].sum().backward()
    assert (v.grad[[0, 3, 4]] == 0).all() and (v.grad[1:3] != 0).any()
    with pytest.raises(RuntimeError):
        a, = torch.autograd.grad(m2_amd.token_logprobs(v, t).logprobs.sum(), v, create_graph=True)
        a.sum().backward()
    r = m2_amd.token_logprobs(v, t, 4)
    v.data_ptr()
    with torch.no_grad():
        v.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        r.logprobs.sum().backward()


def test_same_bits_every_time(gpu):
    import m2_amd
    x, t = _logits(gpu, (40, 30522), torch.bfloat16), _tokens(gpu, (40,), 30522)
    g = _grads(gpu, (40,), 10)

    def once():
        v = x.detach().requires_grad_()
        r = m2_amd.token_logprobs(v, t, 10)
        return [*[o.detach() for o in r], *torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], [v], g)]

    first = once()
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, once()))


@pytest.mark.parametrize("rows,V", [(1, 30522), (3, 200001), (64, 1000)])
def test_captured_beside_eager_calls_and_streams(gpu, rows, V):
    """Two captured graphs and eager calls in turns, on two streams, each with inputs of its own."""
    import m2_amd
    xs = [_logits(gpu, (rows, V), torch.bfloat16, seed=s) for s in range(3)]
    t, g = _tokens(gpu, (rows,), V), _grads(gpu, (rows,), 6)

    def call(x):
        v = x.detach().requires_grad_()
        r = m2_amd.token_logprobs(v, t, 6)
        return [*[o.detach() for o in r], *torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], [v], g)]

    want = [call(x) for x in xs]
    side = torch.cuda.Stream()
    graphs, outs, ins = [], [], [x.clone() for x in xs[:2]]
    for i in range(2):
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call(ins[i])
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(call(ins[i]))
        graphs.append(graph)
    for turn in range(4):
        for i in range(2):
            ins[i].copy_(xs[(i + turn) % 3])
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()
        eager = call(xs[2])
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[(i + turn) % 3]))
        assert all(torch.equal(a, b) for a, b in zip(eager, want[2]))


def test_views_of_negatives(gpu):
    """Logits and gradients whose memory holds the negatives of their values, as imaginary parts of conjugates do."""
    import m2_amd

    def negative_view(t):
        v = torch.complex(t, -t).conj().imag
        assert v.is_neg() and torch.equal(v, t)
        return v

    for rows, V in ((5, 300), (1, 70), (4, 1)):
        x, t, (gl, gh, ga) = _logits(gpu, (rows, V), torch.float32, seed=5), _tokens(gpu, (rows,), V), _grads(gpu, (rows,), 1)
        a, b = x.clone().requires_grad_(), torch._neg_view(-x).requires_grad_()
        assert b.is_neg()
        one, other = m2_amd.token_logprobs(a, t, 1), m2_amd.token_logprobs(b, t, 1)
        assert all(torch.equal(p, q) for p, q in zip(one, other))
        assert torch.equal(m2_amd.token_logprobs(negative_view(x), t).logprobs, one.logprobs)
        ins = [torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], [v], g)[0]
               for r, v, g in ((one, a, (gl, gh, ga)), (other, b, tuple(negative_view(g) for g in (gl, gh, ga))))]
        assert torch.equal(ins[0], ins[1])


def test_graph_is_kept_and_let_go(gpu):
    """A second backward pass where the graph is kept is the first; where it is not, and where what is saved has changed, it is refused."""
    import m2_amd
    x, t = _logits(gpu, (4, 600), torch.float32), _tokens(gpu, (4,), 600)
    g = _grads(gpu, (4,), 3)

    def call():
        v = x.clone().requires_grad_()
        return v, m2_amd.token_logprobs(v, t, 3)

    v, r = call()
    outs = [r.logprobs, r.entropy, r.top_logprobs]
    assert not r.top_ids.requires_grad and all(o.requires_grad and not o.is_leaf for o in outs)
    first = torch.autograd.grad(outs, [v], g, retain_graph=True)[0]
    assert torch.equal(torch.autograd.grad(outs, [v], g)[0], first)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(outs, [v], g)
    for change in ("logits", "entropy", "ids", "tokens"):
        v, r = call()
        with torch.no_grad():
            {"logits": v, "entropy": r.entropy, "ids": r.top_ids, "tokens": t}[change].add_(0)
        with pytest.raises(RuntimeError):
            torch.autograd.grad([r.logprobs], [v], g[:1])
    seen = []
    v, r = call()
    r.entropy.register_hook(lambda h: seen.append(h) or 2 * h)
    r.logprobs.retain_grad()
    (r.entropy.sum() + (r.logprobs * g[0]).sum()).backward()
    a, b = call()
    assert len(seen) == 1 and torch.equal(r.logprobs.grad, g[0])
    assert torch.equal(v.grad, torch.autograd.grad([b.logprobs, b.entropy], [a], [g[0], torch.full((4,), 2.0, device=gpu)])[0])


def test_recomputed_in_the_backward_pass(gpu):
    """Under activation checkpointing, whose hooks hand the saved tensors out again."""
    import m2_amd
    from torch.utils.checkpoint import checkpoint
    h, w = torch.randn(6, 40, device=gpu), torch.randn(500, 40, device=gpu)
    t = _tokens(gpu, (6,), 500)
    grads = []
    for again in (False, True):
        v = w.clone().requires_grad_()
        f = lambda: m2_amd.token_logprobs(h @ v.t(), t, 3)
        r = checkpoint(f, use_reentrant=False) if again else f()
        grads.append(torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + r.top_logprobs.sum(), [v])[0])
    assert torch.equal(*grads)


def test_refusals(gpu):
    import m2_amd
    f = m2_amd.token_logprobs
    x, t = torch.randn(4, 50, device=gpu), torch.zeros(4, dtype=torch.int64, device=gpu)
    for bad, error in (((x.cpu(), t.cpu()), RuntimeError), ((x.half(), t), TypeError), ((x.double(), t), TypeError), ((x, t.int()), ValueError),
                       ((x, t[:3]), ValueError), ((x, t.cpu()), ValueError), ((x, t, 33), ValueError), ((x, t, -1), ValueError), ((x[:, :5], t, 6), ValueError),
                       ((x, t, 0, torch.ones(49, dtype=torch.bool, device=gpu)), ValueError), ((x, t, 0, torch.ones(50, device=gpu)), ValueError),
                       ((x, t, 0, torch.ones(50, dtype=torch.bool)), ValueError), ((x[:, :0], t), ValueError), ((x[0, 0], None), ValueError)):
        with pytest.raises(error):
            f(*bad)
    from torch.func import vmap
    with pytest.raises(RuntimeError):
        vmap(lambda v: f(v[None], t[:1]).entropy)(x)
    import torch.autograd.forward_ad as fw
    with fw.dual_level(), pytest.raises(RuntimeError):
        f(fw.make_dual(x, torch.ones_like(x)), t)
