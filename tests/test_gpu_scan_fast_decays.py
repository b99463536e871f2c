"""selective_scan where A lies at the end of fp32's range: such a state forgets at once, and the positions behind a sequence's end, which have a step of 0, leave it as it is."""
import pytest
import torch

import causal_reference as R
import test_gpu_selective_scan as scan

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def _results(ins, lengths, gy, gl):
    mine = {k: v.detach().requires_grad_() for k, v in ins.items()}
    y, last = scan._call(mine, True, lengths)
    return dict(zip(("y", "last", *scan.ORDER), (y.detach(), last.detach(), *torch.autograd.grad([y, last], [mine[k] for k in scan.ORDER], [gy, gl]))))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,L,C,N,G", [(2, 37, 24, 16, None), (3, 200, 10, 5, 2), (1, 250, 1536, 16, None), (2, 70, 6, 61, None), (1, 40, 3, 200, None), (4, 33, 5, 1, None)])
def test_fast_decays(gpu, B, L, C, N, G, dtype):
    for ragged in (False, True):
        ins, lengths = scan._inputs(gpu, B, L, C, N, G, dtype, ragged=ragged, seed=2)
        fast = torch.rand(C, N, generator=torch.Generator(device=gpu).manual_seed(4), device=gpu) < 0.3
        fast[0, 0] = True
        ins["A"] = torch.where(fast, torch.full_like(ins["A"], -3e38), ins["A"])
        g = torch.Generator(device=gpu).manual_seed(5)
        gy, gl = torch.randn(B, L, C, generator=g, device=gpu).to(dtype), torch.randn(B, C, N, generator=g, device=gpu)
        found = _results(ins, lengths, gy, gl)
        d = R.doubles(ins, False)
        want, end = scan._reference(d, True, lengths)
        y_off, end_off = scan._bounds(d, True, lengths, dtype)
        R.within("y", found["y"], want, y_off)
        R.within("state", found["last"], end, end_off)
        d = R.doubles(ins)
        wants = dict(zip(scan.ORDER, torch.autograd.grad(list(scan._reference(d, True, lengths)), [d[k] for k in scan.ORDER], [gy.double(), gl.double()])))
        for name, w in wants.items():
            # (how near: the other tests; here 2^-7 of the largest, which a state that is not forgotten, or a value that is none, passes)
            assert torch.isfinite(found[name]).all() and (found[name].double() - w).abs().max() <= 2.0 ** -7 * w.abs().max(), name
        # beyond the range it is the same, but for what is multiplied by A
        beyond = _results(dict(ins, A=torch.where(fast, torch.full_like(ins["A"], -float("inf")), ins["A"])), lengths, gy, gl)
        for name in ("y", "last", "x", "B", "C", "D", "z", "state"):
            assert torch.equal(found[name], beyond[name]), name


@pytest.mark.parametrize("N", [1, 5, 16])
def test_fast_decays_of_a_step(gpu, N):
    """A step of 0 leaves a state as it is."""
    import m2_amd
    g = torch.Generator(device=gpu).manual_seed(N)
    x, B, C, state = (torch.randn(*s, generator=g, device=gpu) for s in ((3, 8), (3, N), (3, N), (3, 8, N)))
    A, dt = torch.full((8, N), -3e38, device=gpu), torch.zeros(3, 8, device=gpu)
    dt[1] = 0.5
    kept = state.clone()
    y = m2_amd.selective_scan_step(x, dt, state, A, B, C)
    assert torch.equal(state[0::2], kept[0::2]) and torch.isfinite(y).all()
    want = 0.5 * x[1].double().unsqueeze(1) * B[1].double()
    R.within("state", state[1], want, 2 * R.U * want.abs())
