"""selective_scan and its gradient on every plan that a call may get (lanes, states a lane, waves, sets of channels a workgroup), against the recurrence in 64 bits.

The forward's bound is test_gpu_selective_scan's.  The gradient's runs beside the adjoint recurrence, as that one does beside the states: MD[t] = |C u| + a[t + 1] MD[t + 1] bounds dh, with the decays
that carry it, and ED[t] what it is off by; a decay adds U (10 + 28 |d A|) of what it carries, to dh as to a state.  With M and E the states' own:
    u = gy silu(z)                 (9, for bf16 2 |z| more) U |u|
    dh[t] = C u + a dh[t + 1]      ED = a (ED[t + 1] + U (10 + 28 |d A|) MD[t + 1]) + |C| (off u) + 4 U |C u|
    sum_n dh B                     sum ED |B| + (N + 4) U sum MD |B|
    dh a h[t - 1]                  a (ED M + MD E) + U (14 + 28 |d A|) a MD M
d is off by 10 U, softplus' slope by (12 + |its argument|) U, SiLU's by (10, for bf16 2 |z| more) U of its parts.  A sum over positions and sequences passes 16 positions of a lane, a step's sum for
each 64 or 32 positions, 16 of waves and lanes and a sequence's for each eight; one over channels 12 of lanes, the workgroup's sets, and each eighth workgroup: so many U of its terms."""
import ctypes

import pytest
import torch

import causal_reference as R
import test_gpu_selective_scan as scan

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def plan_of(B, L, C, N, G, backward):
    """-> (lanes a channel, states a lane, waves, workgroups, sets)"""
    from m2_amd._lib import check, lib
    found = (ctypes.c_int * 5)()
    check(lib.m2_selective_scan_plan(B, L, C, G or 1, N, backward, found))
    return tuple(found)


def gradient_bounds(d, softplus, lengths, gy, gl, dtype):
    """{input: what its gradient may be off by}"""
    U = R.U
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
    lanes, each, waves, workgroups, sets = plan_of(B, L, C, N, G, 1)
    over_positions = 16 + -(-L // (16 * waves)) + 16 + -(-B // 8)
    over_channels = 12 + sets + -(-(workgroups // (B * G)) // 8)
    arg = s.unsqueeze(-1) * A
    a, decay = torch.exp(arg), U * (10 + 28 * arg.abs())
    dx = s.abs() * x

    def wide(m, t):
        return m[:, t].repeat_interleave(C // G, 1)

    M = [torch.zeros(B, C, N, dtype=x.dtype, device=x.device) if v["state"] is None else v["state"].abs()]
    E = [torch.zeros_like(M[0])]
    for t in range(L):
        put = dx[:, t].unsqueeze(-1) * wide(Bm, t)
        E.append(a[:, t] * (E[-1] + decay[:, t] * M[-1]) + 16 * U * put)
        M.append(a[:, t] * M[-1] + put)
    z = v["z"]
    more = 2 * z.abs() if z is not None and dtype == BF16 else 0
    u = gy if z is None else gy * R.silu(z).abs()
    u_off = torch.zeros_like(u) if z is None else (9 + more) * U * u
    D = torch.zeros(C, dtype=x.dtype, device=x.device) if v["D"] is None else v["D"].abs()
    bound = {k: torch.zeros_like(t) for k, t in v.items() if t is not None}
    shared = {k: torch.zeros(B, L, G, N, dtype=x.dtype, device=x.device) for k in ("B", "C")}
    carry, off = gl.abs(), torch.zeros_like(gl)
    for t in range(L - 1, -1, -1):
        b, c, ut = wide(Bm, t), wide(Cm, t), u[:, t].unsqueeze(-1)
        MD, ED = c * ut + carry, off + c * u_off[:, t].unsqueeze(-1) + 4 * U * c * ut
        into, into_off = (MD * b).sum(-1), (ED * b).sum(-1) + (N + 4) * U * (MD * b).sum(-1)
        kept, kept_off = a[:, t] * MD * M[t], a[:, t] * (ED * M[t] + MD * E[t] + (4 * U + decay[:, t]) * MD * M[t])
        gd = (kept * A.abs()).sum(-1) + x[:, t] * into
        gd_off = (kept_off * A.abs()).sum(-1) + (N + 4) * U * (kept * A.abs()).sum(-1) + x[:, t] * into_off + 2 * U * gd
        if softplus:
            slope = torch.sigmoid(raw[:, t])
            gd, gd_off = slope * gd, slope * (gd_off + (12 + raw[:, t].abs()) * U * gd)
        gd, gd_off = (torch.where(ok[:, t], q, torch.zeros_like(q)) for q in (gd, gd_off))
        bound["dt"][:, t] = gd_off
        bound["x"][:, t] = torch.where(ok[:, t], s[:, t].abs() * (into_off + 14 * U * into) + D * (u_off[:, t] + 4 * U * u[:, t]), torch.zeros_like(into))
        bound["A"] += (s[:, t].abs().unsqueeze(-1) * (kept_off + (14 + over_positions) * U * kept)).sum(0)
        if "D" in bound:
            bound["D"] += ((u_off[:, t] + (4 + over_positions) * U * u[:, t]) * x[:, t]).sum(0)
        if "dt_bias" in bound:
            bound["dt_bias"] += (gd_off + over_positions * U * gd).sum(0)
        if z is not None:
            p, zt = torch.sigmoid(z[:, t]), z[:, t].abs()
            parts = p + zt * p * (1 - p)
            y, y_off = (c * M[t + 1]).sum(-1) + D * x[:, t], (c * E[t + 1]).sum(-1)
            bound["z"][:, t] = gy[:, t] * parts * (y_off + (N + 16 + (more[:, t] if dtype == BF16 else 0)) * U * y)
        for name, q in (("B", (ED + (14 + over_channels) * U * MD) * dx[:, t].unsqueeze(-1)), ("C", ut * (E[t + 1] + (4 + over_channels) * U * M[t + 1]) + u_off[:, t].unsqueeze(-1) * M[t + 1])):
            shared[name][:, t] = torch.where(ok[:, t].unsqueeze(-1), q.view(B, G, C // G, N).sum(2), torch.zeros_like(shared[name][:, t]))
        carry, off = a[:, t] * MD, a[:, t] * (ED + decay[:, t] * MD)
    for name in ("B", "C"):
        bound[name] = shared[name].squeeze(2) if flat else shared[name]
    if "state" in bound:
        bound["state"] = off
    return bound


def check_gradient(gpu, B, L, C, N, G, dtype, variants, seed=4):
    for parts, softplus, ragged, pad in variants:
        ins, lengths = scan._inputs(gpu, B, L, C, N, G, dtype, parts, ragged, pad=pad, seed=seed)
        if not softplus:
            ins["dt"] = ins["dt"].abs()
        g = torch.Generator(device=gpu).manual_seed(6)
        gy, gl = torch.randn(B, L, C + pad, generator=g, device=gpu).to(dtype)[..., pad:], torch.randn(B, C, N, generator=g, device=gpu)
        names = [k for k in scan.ORDER if ins[k] is not None]
        d = R.doubles(ins)
        wants = torch.autograd.grad(list(scan._reference(d, softplus, lengths)), [d[k] for k in names], [gy.double(), gl.double()])
        mine = {k: None if t is None else t.detach().requires_grad_() for k, t in ins.items()}
        gots = torch.autograd.grad(list(scan._call(mine, softplus, lengths)), [mine[k] for k in names], [gy, gl])
        bounds = gradient_bounds(d, softplus, lengths, gy.double(), gl.double(), dtype)
        for name, got, want in zip(names, gots, wants):
            R.within(name, got, want, bounds[name])
            # a bound that a wrong gradient could pass would say nothing (the two that add up terms of either sign over all positions are the widest)
            assert bounds[name].sum() <= (0.03 if name in ("A", "dt_bias") else 0.002) * want.abs().sum(), (name, bounds[name].sum().item(), want.abs().sum().item())


ALL = ("D", "z", "dt_bias", "state")
VARIANTS = ((ALL, True, True, 0), ((), True, False, 3), (("z", "state"), False, False, 8))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,L,C,N,G", scan.SIZES)
def test_gradient(gpu, B, L, C, N, G, dtype):
    check_gradient(gpu, B, L, C, N, G, dtype, VARIANTS)


# (sizes), (lanes a channel, states a lane, waves)
FORWARD = [((1, 250, 1536, 16, None), (8, 2, 12)), ((1, 90, 1536, 16, None), (8, 2, 6)), ((1, 40, 1536, 16, None), (8, 2, 3)), ((9, 400, 130, 16, None), (8, 2, 12)), ((3, 200, 700, 5, None), (4, 2, 12)),
           ((5, 250, 130, 24, 2), (16, 2, 12)), ((2, 300, 130, 61, None), (32, 2, 8)), ((66, 90, 130, 2, None), (1, 2, 8)), ((17, 150, 256, 3, None), (2, 2, 8)), ((66, 70, 130, 16, None), (8, 2, 2)),
           ((66, 70, 512, 2, None), (2, 1, 2)), ((9, 40, 1536, 5, None), (4, 2, 2)), ((9, 150, 130, 24, None), (8, 4, 8)), ((5, 100, 700, 16, None), (4, 4, 8)), ((1, 100, 1002, 100, None), (32, 4, 2)),
           ((2, 80, 130, 200, None), (64, 4, 2)), ((66, 40, 1002, 1, None), (1, 1, 2)), ((17, 70, 256, 24, None), (16, 2, 2))]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size,plan", FORWARD)
def test_forward_plans(gpu, size, plan, dtype):
    B, L, C, N, G = size
    if torch.cuda.get_device_properties(gpu).multi_processor_count == 256:
        assert plan_of(B, L, C, N, G, 0)[:3] == plan
    scan.test_forward(gpu, B, L, C, N, G, dtype)


# (sizes), (lanes a channel, states a lane, waves, sets): mostly, the last workgroup of a group has fewer sets and its last set fewer channels; from 64 states on sets are joined for memory's sake
BACKWARD = [((40, 150, 500, 16, None), (8, 2, 4, 2)), ((40, 150, 1000, 16, 2), (8, 2, 4, 2)), ((40, 130, 1530, 16, None), (8, 2, 4, 3)), ((17, 150, 1919, 5, None), (4, 2, 4, 2)), ((66, 100, 700, 3, None), (4, 1, 4, 3)),
            ((66, 130, 1910, 1, None), (2, 1, 4, 4)), ((17, 70, 1919, 3, None), (4, 1, 4, 2)), ((1, 700, 1535, 128, None), (64, 2, 2, 2)), ((3, 250, 701, 256, None), (64, 4, 2, 2)), ((40, 150, 701, 64, None), (32, 2, 4, 2))]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("size,plan", BACKWARD)
def test_gradient_plans(gpu, size, plan, dtype):
    B, L, C, N, G = size
    if torch.cuda.get_device_properties(gpu).multi_processor_count == 256:
        found = plan_of(B, L, C, N, G, 1)
        assert found[:3] + found[4:] == plan
    check_gradient(gpu, B, L, C, N, G, dtype, VARIANTS[:2] if B * L * C * N < 2 ** 27 else VARIANTS[:1])
