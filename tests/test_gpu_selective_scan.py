"""selective_scan and selective_scan_step against the recurrence in 64 bits, position by position.

The bound runs beside the recurrence: M[t] = a M[t-1] + |b| bounds the states, E[t] what they are off by.  A decay exp(d A) is off, relative to itself, by 4 U (the exponential) and |d A| times
what its argument is off by: 4 U for the rounded log2 e, product and A log2 e, and 10 U for d itself (softplus: an exponential, a quotient, a series); an input by 14 U (d, two products, one sum).
The state's passage through shared memory multiplies once more for every 16 positions and each of the waves: counted as one more decay a position.  So
    E[t] = a (E[t-1] + U (10 + 28 |d A|) M[t-1]) + 16 U |b|,    y: sum |C| E + (N + 4) U (sum |C| M + |D x|), gate: slope 1.1, 8 U; for bf16 (8 + 2 |z|) U, its exponential's
argument being only rounded."""
import pytest
import torch

import causal_reference as R

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
ORDER = ("x", "dt", "A", "B", "C", "D", "z", "dt_bias", "state")


def _inputs(gpu, B, L, C, N, G, dtype, parts=("D", "z", "dt_bias", "state"), ragged=False, seed=0, pad=0):
    g = torch.Generator(device=gpu).manual_seed(seed * 77 + B + L + C + N)

    def randn(*s):
        return torch.randn(*s, generator=g, device=gpu)

    shared = (B, L, N) if G is None else (B, L, G, N)
    ins = {"x": randn(B, L, C + pad).to(dtype)[..., pad:], "dt": (randn(B, L, C) - 2).to(dtype), "A": -torch.exp(randn(C, N)), "B": randn(*shared[:-1], N + pad).to(dtype)[..., :N],
           "C": randn(*shared[:-1], N + pad).to(dtype)[..., pad:], "D": randn(C), "z": randn(B, L, C + pad).to(dtype)[..., :C], "dt_bias": 0.5 * randn(C), "state": randn(B, C, N)}
    for name in ("D", "z", "dt_bias", "state"):
        if name not in parts:
            ins[name] = None
    lengths = None
    if ragged:
        lengths = torch.randint(0, L + 1, (B,), generator=g, device=gpu)
        lengths[0] = L
        if B > 1:
            lengths[1] = 0
        if B > 2:
            lengths[2] = min(1, L)
    return ins, lengths


def _same(a, b):
    """Bit for bit (values beyond the type's range, from steps below 0, among them)."""
    kind = torch.int16 if a.dtype == BF16 else torch.int32
    return torch.equal(a.view(kind), b.view(kind))


def _call(ins, softplus, lengths=None):
    import m2_amd
    return m2_amd.selective_scan(*[ins[k] for k in ORDER[:5]], D=ins["D"], z=ins["z"], dt_bias=ins["dt_bias"], dt_softplus=softplus, state=ins["state"], lengths=lengths, return_state=True)


def _reference(d, softplus, lengths=None):
    return R.scan(*[d[k] for k in ORDER[:8]], softplus, d["state"], lengths)


def _bounds(d, softplus, lengths, dtype=F32):
    """What y and the last state may be off by."""
    x, Bm, Cm = d["x"].abs(), d["B"].abs(), d["C"].abs()
    B, L, C = x.shape
    if Bm.dim() == 3:
        Bm, Cm = Bm.unsqueeze(2), Cm.unsqueeze(2)
    each, N = C // Bm.shape[2], d["A"].shape[1]
    ok = R.inside(lengths, B, L, x.device)
    s = d["dt"] if d["dt_bias"] is None else d["dt"] + d["dt_bias"]
    if softplus:
        s = torch.logaddexp(s, torch.zeros_like(s))
    s, x = torch.where(ok, s, torch.zeros_like(s)), torch.where(ok, x, torch.zeros_like(x))
    M = torch.zeros(B, C, N, dtype=torch.float64, device=x.device) if d["state"] is None else d["state"].abs()
    E, ys = torch.zeros_like(M), []
    for t in range(L):
        b, c = (m[:, t].repeat_interleave(each, 1) for m in (Bm, Cm))
        arg = s[:, t, :, None] * d["A"]
        a, put = torch.exp(arg), (s[:, t] * x[:, t]).abs().unsqueeze(-1) * b
        E = a * (E + R.U * (10 + 28 * arg.abs()) * M) + 16 * R.U * put
        M = a * M + put
        skip = 0 if d["D"] is None else (d["D"] * x[:, t]).abs()
        off, size = (c * E).sum(-1) + (N + 4) * R.U * ((c * M).sum(-1) + skip), (c * M).sum(-1) + skip
        ys.append(off if d["z"] is None else R.silu(d["z"][:, t]).abs() * (off + (8 + (2 * d["z"][:, t].abs() if dtype == BF16 else 0)) * R.U * size))
    return torch.stack(ys, 1), E


SIZES = [(1, 1, 1, 1, None), (1, 1, 64, 16, None), (2, 2, 5, 3, None), (3, 17, 40, 16, 2), (2, 129, 100, 16, None), (1, 300, 33, 8, 1), (2, 150, 24, 61, 3), (4, 65, 130, 4, None), (1, 257, 70, 2, None),
         (2, 40, 12, 128, 2), (1, 70, 9, 200, None), (2, 33, 7, 256, None), (1, 1000, 20, 16, None), (40, 19, 256, 16, 4), (20, 140, 336, 24, None), (3, 128, 64, 64, None), (70, 50, 260, 32, 1),
         (17, 37, 1024, 1, 1), (65, 21, 130, 100, None), (140, 35, 8, 130, 2), (2, 50, 12, 16, 12), (1, 33, 6, 70, 6)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,L,C,N,G", SIZES)
def test_forward(gpu, B, L, C, N, G, dtype):
    import m2_amd
    for parts, softplus, ragged, pad in ((("D", "z", "dt_bias", "state"), True, False, 0), ((), True, True, 3), (("z", "state"), False, True, 8), (("D", "dt_bias"), True, False, 4)):
        ins, lengths = _inputs(gpu, B, L, C, N, G, dtype, parts, ragged, pad=pad)
        if not softplus:
            ins["dt"] = ins["dt"].abs()
        y, last = _call(ins, softplus, lengths)
        d = R.doubles(ins, False)
        want, end = _reference(d, softplus, lengths)
        y_off, end_off = _bounds(d, softplus, lengths, dtype)
        R.within("y", y, want, y_off)
        R.within("state", last, end, end_off)
        assert y.dtype == dtype and last.dtype == F32
        if ragged:
            assert not y.masked_select(~R.inside(lengths, B, L, gpu)).any()
        assert torch.equal(m2_amd.selective_scan(*[ins[k] for k in ORDER[:8]], softplus, ins["state"], lengths), y)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,L,C,N,G", SIZES)
def test_gradient(gpu, B, L, C, N, G, dtype):
    """Against autograd's of the recurrence in 64 bits.  Magnitudes come from the formula with absolute values: dh >= 0, every term of every sum >= 0."""
    for parts, softplus, ragged, pad in ((("D", "z", "dt_bias", "state"), True, True, 0), ((), True, False, 3), (("z", "state"), False, False, 8)):
        ins, lengths = _inputs(gpu, B, L, C, N, G, dtype, parts, ragged, pad=pad, seed=4)
        if not softplus:
            ins["dt"] = ins["dt"].abs()
        g = torch.Generator(device=gpu).manual_seed(6)
        gy, gl = torch.randn(B, L, C + pad, generator=g, device=gpu).to(dtype)[..., pad:], torch.randn(B, C, N, generator=g, device=gpu)
        names = [k for k in ORDER if ins[k] is not None]
        d = R.doubles(ins)
        wants = torch.autograd.grad(list(_reference(d, softplus, lengths)), [d[k] for k in names], [gy.double(), gl.double()])
        mine = {k: None if t is None else t.detach().requires_grad_() for k, t in ins.items()}
        gots = torch.autograd.grad(list(_call(mine, softplus, lengths)), [mine[k] for k in names], [gy, gl])
        sizes, count = _magnitudes(d, softplus, lengths, gy.double(), gl.double())
        for name, got, want in zip(names, gots, wants):
            R.within(name, got, want, R.U * count * sizes[name])


def _magnitudes(d, softplus, lengths, gy, gl):
    """{input: sum of the absolute values of what its gradient is made of}, and how many roundings, in U, a product has seen at most: L decays of U (10 + 28 |d A|), 40 elsewhere, 88 in sums."""
    v = {k: None if t is None else t.detach() for k, t in d.items()}
    x, Bm, Cm, A = v["x"].abs(), v["B"].abs(), v["C"].abs(), v["A"]
    flat = Bm.dim() == 3
    if flat:
        Bm, Cm = Bm.unsqueeze(2), Cm.unsqueeze(2)
    B, L, C = x.shape
    G, N = Bm.shape[2:]
    ok = R.inside(lengths, B, L, x.device)
    raw = v["dt"] if v["dt_bias"] is None else v["dt"] + v["dt_bias"]
    s = torch.logaddexp(raw, torch.zeros_like(raw)) if softplus else raw
    s, x, gy = (torch.where(ok, t, torch.zeros_like(t)) for t in (s, x, gy.abs()))
    Bw, Cw = (m.repeat_interleave(C // G, 2) for m in (Bm, Cm))
    a = torch.exp(s.unsqueeze(-1) * A)
    put = (s.abs() * x).unsqueeze(-1) * Bw
    h = [torch.zeros(B, C, N, dtype=x.dtype, device=x.device) if v["state"] is None else v["state"].abs()]
    for t in range(L):
        h.append(a[:, t] * h[-1] + put[:, t])
    before, after = torch.stack(h[:-1], 1), torch.stack(h[1:], 1)
    z = v["z"]
    u = gy if z is None else gy * R.silu(z).abs()
    D = torch.zeros(C, dtype=x.dtype, device=x.device) if v["D"] is None else v["D"].abs()
    dh, carry = [None] * L, gl.abs()
    for t in range(L - 1, -1, -1):
        dh[t] = Cw[:, t] * u[:, t].unsqueeze(-1) + carry
        carry = a[:, t] * dh[t]
    dh = torch.stack(dh, 1)
    keep = dh * a * before
    into = (dh * Bw).sum(-1)
    gd = (keep * A.abs()).sum(-1) + x * into
    if softplus:
        gd = gd * torch.sigmoid(raw)
    gd = torch.where(ok, gd, torch.zeros_like(gd))

    def shared(t):
        t = t.view(B, L, G, C // G, N).sum(3)
        return t.squeeze(2) if flat else t

    out = {"x": s.abs() * into + D * u, "dt": gd, "A": (keep * s.abs().unsqueeze(-1)).sum((0, 1)), "B": shared(dh * (s.abs() * x).unsqueeze(-1)), "C": shared(u.unsqueeze(-1) * after),
           "D": (u * x).sum((0, 1)), "dt_bias": gd.sum((0, 1)), "state": carry}
    if z is not None:
        # silu'(z) is within 1.1, and off by 8 U of 1 where it passes zero
        out["z"] = gy * 1.1 * ((after * Cw).sum(-1) + D * x)
    return out, L * (10 + 28 * (s.unsqueeze(-1) * A).abs().max().item()) + 40 + 88


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,C,N,G", [(1, 1, 1, None), (1, 1536, 16, None), (3, 66, 61, 3), (130, 20, 4, 1), (2, 9, 256, None), (5, 24, 7, 2), (0, 5, 4, None), (2, 33, 100, None)])
def test_step(gpu, B, C, N, G, dtype):
    import m2_amd
    L = 4
    for parts, softplus, pad in ((("D", "z", "dt_bias", "state"), True, 0), (("state",), False, 3)):
        ins, _ = _inputs(gpu, B, L, C, N, G, dtype, parts, pad=pad)
        d = R.doubles(ins, False)
        state, wants = ins["state"].clone(), []
        for t in range(L):
            at = {k: v[:, t] if k in ("x", "dt", "B", "C", "z") and v is not None else v for k, v in ins.items()}
            kept, other = state.clone(), torch.empty_like(state)
            apart = m2_amd.selective_scan_step(at["x"], at["dt"], state, at["A"], at["B"], at["C"], at["D"], at["z"], at["dt_bias"], softplus, out_state=other)
            assert _same(state, kept)
            y = m2_amd.selective_scan_step(at["x"], at["dt"], state, at["A"], at["B"], at["C"], at["D"], at["z"], at["dt_bias"], softplus)
            assert _same(y, apart) and _same(state, other) and y.dtype == dtype
            if B:
                part = {k: v[:, :t + 1] if k in ("x", "dt", "B", "C", "z") and v is not None else v for k, v in d.items()}
                want, end = _reference(part, softplus)
                y_off, end_off = _bounds(part, softplus, None, dtype)
                R.within("y", y, want[:, -1], y_off[:, -1])
                R.within("state", state, end, end_off)


@pytest.mark.parametrize("C,N", [(24, 16), (1600, 16), (8, 61), (40, 1)])
def test_parts_give_the_whole(gpu, C, N):
    """A sequence in parts, each going on from the last one's state, is the whole within the bounds of both."""
    import m2_amd
    ins, _ = _inputs(gpu, 2, 300, C, N, None, F32)
    whole, last = _call(ins, True)
    state, ys = ins["state"], []
    for a, b in ((0, 1), (1, 17), (17, 200), (200, 300)):
        part = {k: v[:, a:b] if k in ("x", "dt", "B", "C", "z") else v for k, v in ins.items()}
        y, state = _call(dict(part, state=state), True)
        ys.append(y)
    y_off, end_off = _bounds(R.doubles(ins, False), True, None)
    R.within("y", torch.cat(ys, 1), whole.double(), 2 * y_off)
    R.within("state", state, last.double(), 2 * end_off)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -3e38])
def test_what_lies_behind_the_end_is_not_read(gpu, bad):
    for N, C in ((16, 40), (61, 12)):
        ins, _ = _inputs(gpu, 4, 150, C, N, None, F32)
        lengths = torch.tensor([0, 1, 77, 150], device=gpu)
        ok = R.inside(lengths, 4, 150, gpu)
        gy = torch.randn(4, 150, C, device=gpu)
        results = []
        for fill in (0.0, bad):
            filled = {k: torch.where(ok, v, torch.full_like(v, fill)) if k in ("x", "dt", "B", "C", "z") else v for k, v in ins.items()}
            mine = {k: v.detach().requires_grad_() for k, v in filled.items()}
            y, last = _call(mine, True, lengths)
            grads = torch.autograd.grad([y, last], [mine[k] for k in ORDER], [torch.where(ok, gy, torch.full_like(gy, fill)), torch.ones_like(last)])
            results.append([y.detach(), last.detach(), *grads])
        assert all(torch.equal(a, b) for a, b in zip(*results))
        for t in (0, 2, 3, 5, 6, 8):      # y, and the gradients of x, dt, B, C, z
            assert not results[0][t].masked_select(~ok).any()
        assert torch.equal(results[0][1][0], ins["state"][0])


def test_gradient_against_differences(gpu):
    """The derivative along a direction, by central differences of the recurrence in 64 bits (step 1e-5: off by 1e-10 of the third derivative), against the gradients' product with it."""
    ins, lengths = _inputs(gpu, 2, 60, 10, 5, None, F32, seed=8)
    gen = torch.Generator(device=gpu).manual_seed(1)
    mine = {k: t.detach().requires_grad_() for k, t in ins.items()}
    y, last = _call(mine, True)
    gy, gl = torch.randn(y.shape, generator=gen, device=gpu), torch.randn(last.shape, generator=gen, device=gpu)
    grads = dict(zip(ORDER, torch.autograd.grad([y, last], [mine[k] for k in ORDER], [gy, gl])))
    sizes, count = _magnitudes(R.doubles(ins), True, None, gy.double(), gl.double())
    for name in ORDER:
        way = torch.randn(ins[name].shape, generator=gen, device=gpu).double()
        found = []
        for sign in (1, -1):
            d = R.doubles(ins, False)
            d[name] = d[name] + sign * 1e-5 * way
            a, b = _reference(d, True)
            found.append((a * gy.double()).sum() + (b * gl.double()).sum())
        slope = (found[0] - found[1]) / 2e-5
        got = (grads[name].double() * way).sum()
        room = R.U * count * (sizes[name] * way.abs()).sum() + 1e-6 * (sizes[name] * way.abs()).sum()
        assert abs(got - slope) <= room, (name, got.item(), slope.item(), room.item())


def test_long_offsets(gpu):
    """Positions whose place in memory passes 2^31 values: one channel block of a projection 300000 values wide, 8000 positions."""
    import m2_amd
    wide = torch.zeros(8000, 300000, dtype=BF16, device=gpu)
    part = torch.randn(8000, 40, device=gpu, generator=torch.Generator(device=gpu).manual_seed(3)).to(BF16)
    wide[:, 299960:] = part
    x = wide[:, 299960:].unsqueeze(0)
    ins, _ = _inputs(gpu, 1, 8000, 40, 16, None, BF16, ("D",))
    a, b = (m2_amd.selective_scan(v, *[ins[k] for k in ORDER[1:6]], dt_softplus=True) for v in (x, part.unsqueeze(0)))
    assert torch.equal(a, b)
    w = torch.randn(40, 4, device=gpu)
    assert torch.equal(m2_amd.causal_conv(x, w), m2_amd.causal_conv(part.unsqueeze(0), w))
    assert torch.equal(m2_amd.group_norm(x, 4), m2_amd.group_norm(part.unsqueeze(0), 4))


def test_rows_far_apart(gpu):
    """Rows 2^24 values apart: further than the kernels' 32-bit offsets go, they are copied."""
    import m2_amd
    wide = torch.randn(5, 2 ** 24, generator=torch.Generator(device=gpu).manual_seed(1), device=gpu)
    ins, _ = _inputs(gpu, 1, 5, 24, 16, None, F32, ("D", "z"))
    far = dict(ins, x=wide[:, :24].unsqueeze(0), B=wide[:, 100:116].unsqueeze(0), z=wide[:, 200:224].unsqueeze(0))
    near = {k: None if v is None else v.contiguous() for k, v in far.items()}
    gy = wide[:, 300:324].unsqueeze(0)
    results = []
    for which, g in ((far, gy), (near, gy.contiguous())):
        mine = {k: None if v is None else v.detach().requires_grad_() for k, v in which.items()}
        y, last = _call(mine, True)
        results.append([y.detach(), last.detach(), *torch.autograd.grad(y, [v for v in mine.values() if v is not None], g)])
    assert all(torch.equal(a, b) for a, b in zip(*results))
    # one position: its distance to a next one says nothing
    one = wide.as_strided((1, 1, 24), (2 ** 25, 2 ** 26, 1))
    a = m2_amd.selective_scan(one, ins["dt"][:, :1], ins["A"], ins["B"][:, :1], ins["C"][:, :1])
    assert torch.equal(a, m2_amd.selective_scan(one.contiguous(), ins["dt"][:, :1], ins["A"], ins["B"][:, :1], ins["C"][:, :1]))
