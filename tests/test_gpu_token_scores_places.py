"""Every place of token_logprobs' gradient against its own size, and masks at each number of threads to a row."""
import math

import pytest
import torch

U = 2.0 ** -24                                  # half a step of fp32
SPAN = 256 * 4 * 8                              # values of a workgroup of the gradient, bf16 (fp32 half as many)


def definition(logits, tokens, top_k, allowed, grads):
    """In fp64: log probabilities of all places, entropy, ids, and the gradient with what its error may be at each place.

    The gradient is -p f away from tokens and alternatives, f = sum of the outputs' gradients g + g_H (log p + H).  p carries the log probability's error (`units` and a few of |log p|, as
    its argument is a difference and a product) and its own ulps; f the errors of a sum of up to 33 terms, of log p and of H.  Below 2^-126 exp gives 0.  At the outputs' own places the sum of
    their g comes on top, off by a few U.  The result is rounded to its type."""
    z = logits.detach().double()
    if allowed is not None:
        z = z.masked_fill(~allowed, -math.inf)
    V = z.shape[1]
    empty = torch.isneginf(z).all(1, keepdim=True)
    lp = z - torch.logsumexp(z, 1, keepdim=True).masked_fill(empty, 0)
    none = torch.isneginf(z)
    real = lp.masked_fill(none, 0)
    p = lp.exp()
    h = -(p * real).sum(1, keepdim=True)
    order = torch.sort(z, dim=1, descending=True, stable=True).indices[:, :top_k]
    ids = order.masked_fill(none.gather(1, order), -1)
    g_lp, g_h, g_top = (g.double() for g in grads)
    asked = (tokens != -100).unsqueeze(1)
    at = torch.where(asked, tokens.unsqueeze(1), torch.zeros_like(tokens.unsqueeze(1)))
    own = torch.zeros_like(z).scatter_add_(1, at, g_lp.unsqueeze(1) * asked).scatter_add_(1, order, g_top * (ids >= 0))
    total, size = own.sum(1, keepdim=True), (g_lp.unsqueeze(1) * asked).abs() + (g_top * (ids >= 0)).abs().sum(1, keepdim=True)
    g_h = g_h.unsqueeze(1)
    f = total + g_h * (real + h)
    units = 16 + 4 * math.sqrt(V / 128 + 20)
    off = U * ((units + 6 * real.abs()) * f.abs() + 40 * size + g_h.abs() * (units * 2 * (math.log(V) + 2) + 8 * real.abs() + 4 * h))
    grad = (own - p * f).masked_fill(none, 0)
    tol = p * off + 2.0 ** -125 * (f.abs() + 1) + torch.finfo(logits.dtype).eps / 2 * grad.abs() + (own != 0) * 8 * U * (size + f.abs() * p)
    return lp, h.squeeze(1), ids, grad, tol.masked_fill(none, 0), units


def check_gradient(got, grad, tol):
    err = (got.double() - grad).abs()
    assert (err <= tol).all(), (err / tol).nan_to_num().max()


def make(device, rows, V, top_k, dtype, mask):
    g = torch.Generator().manual_seed(rows + 3 * V + top_k)
    x = torch.randn(rows, V, generator=g) * 2 - 6
    x.scatter_add_(1, torch.randint(0, V, (rows, 4), generator=g), torch.full((rows, 4), 9.0))
    tokens = torch.randint(0, V, (rows,), generator=g)
    tokens[rows // 3] = -100
    allowed = None if mask is None else torch.rand(V, generator=g) < 0.6 if mask == "shared" else torch.rand(rows, V, generator=g) < 0.5
    if mask == "rows":
        allowed[rows // 2] = False
        if rows > 2:
            allowed[0] = False
            allowed[0, [V // 3, V - 1]] = True
    grads = [torch.randn(rows, generator=g), torch.randn(rows, generator=g), torch.randn(rows, top_k, generator=g)]
    return x.to(dtype).to(device), tokens.to(device), None if allowed is None else allowed.to(device), [t.to(device) for t in grads]


# one workgroup of 512, 256 and 128 threads a row, and several
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [None, "shared", "rows"])
@pytest.mark.parametrize("rows,V,top_k", [(2, 30528, 32), (3, 30522, 5), (2, 131073, 32), (1, 262147, 20), (7, 8191, 3), (300, 8195, 7), (400, 30522, 10), (1100, 3001, 32), (1300, 8200, 4), (2000, 70, 1)])
def test_every_place(gpu, dtype, mask, rows, V, top_k):
    import m2_amd
    x, tokens, allowed, grads = make(gpu, rows, V, top_k, dtype, mask)
    lp, h, ids, grad, tol, units = definition(x, tokens, top_k, allowed, grads)
    x.requires_grad_()
    r = m2_amd.token_logprobs(x, tokens, top_k, allowed)
    check_gradient(torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], x, grads)[0], grad, tol)
    assert torch.equal(r.top_ids, ids)
    for got, want in ((r.logprobs, lp.gather(1, tokens.clamp_min(0).unsqueeze(1)).squeeze(1).masked_fill(tokens == -100, 0)),
                      (r.top_logprobs, lp.gather(1, ids.clamp_min(0)).masked_fill(ids < 0, -math.inf))):
        inf = torch.isneginf(want)
        assert torch.equal(torch.isneginf(got), inf)
        assert ((got.double() - want).abs() <= U * (units + 4 * want.abs()))[~inf].all()
    assert ((r.entropy.double() - h).abs() <= U * units * 2 * (math.log(V) + 2)).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", [None, "rows"])
@pytest.mark.parametrize("V", [30522, 131073])
def test_the_check_notices(dtype, mask, V):
    """Mistakes planted in a gradient of the definition's: all of them are outside of what it allows, in each row that has a gradient."""
    x, tokens, allowed, grads = make("cpu", 3, V, 8, dtype, mask)
    _, _, ids, grad, tol, _ = definition(x, tokens, 8, allowed, grads)
    check_gradient(grad.to(dtype), grad, tol)
    span = SPAN // (2 if dtype == torch.float32 else 1)
    places = torch.arange(V)
    dense = torch.ones(3, V, dtype=torch.bool).scatter_(1, ids.clamp_min(0), False)
    dense.scatter_(1, tokens.clamp_min(0).unsqueeze(1), False)
    wrong = {
        "nothing behind the first span": torch.where(dense & (places >= span), torch.zeros_like(grad), grad),
        "nothing in the last vector": torch.where(dense & (places >= V - 8), torch.zeros_like(grad), grad),
        "a span's vectors in the next one's place": torch.where(dense & (places >= span), grad.roll(span, 1), grad),
        "cut to 12 bits": torch.where(dense, grad.float().view(torch.int32).bitwise_and(-4096 * (1 if dtype == torch.float32 else 256)).view(torch.float32).double(), grad),
    }
    for name, got in wrong.items():
        bad = ((got - grad).abs() > tol).any(1)
        has = (grad != 0).logical_and(dense & (places >= V - 8)).any(1)
        assert bad[has].all() and has.any(), name
        with pytest.raises(AssertionError):
            check_gradient(got, grad, tol)
