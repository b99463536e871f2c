"""Arguments of Int4Linear and token_logprobs beside the rows: what their memory holds is not always what they are."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 40])
def test_bias_and_tokens_of_negatives(gpu, dtype, M):
    """Views whose memory holds the negatives of their values."""
    import m2_amd
    from m2_amd import ops
    w, bias = torch.randn(70, 96, device=gpu), torch.randn(70, device=gpu)
    lin = m2_amd.Int4Linear.from_weight(w, bias, 32)
    x = torch.randn(M, 96, device=gpu).to(dtype)
    want = lin(x)
    for view in (torch._neg_view(-bias),):
        assert view.is_neg() and torch.equal(ops.int4_linear(x, lin.weight, 70, 32, view), want)
        assert torch.equal(m2_amd.Int4Linear.from_weight(w, view, 32)(x), want)
        lin.bias = view
        assert torch.equal(lin(x), want)
    tokens = torch.randint(0, 70, (M,), device=gpu)
    logits = x.repeat(1, 2)[:, :70].requires_grad_()
    a, b = (m2_amd.token_logprobs(logits, t) for t in (tokens, torch._neg_view(-tokens)))
    assert torch.equal(a.logprobs, b.logprobs)
    assert torch.equal(*(torch.autograd.grad(r.logprobs.sum(), logits)[0] for r in (a, b)))


def test_bias_that_asks_for_gradients_is_refused(gpu):
    """It would get none."""
    import m2_amd
    lin = m2_amd.Int4Linear.from_weight(torch.randn(70, 96, device=gpu), torch.randn(70, device=gpu), 32)
    x = torch.randn(3, 96, device=gpu)
    want = lin(x)
    lin.bias.requires_grad_()
    with pytest.raises(RuntimeError, match="bias: this operator has no gradient"):
        lin(x)
    with torch.no_grad():
        assert torch.equal(lin(x), want)
    bias = torch.nn.Parameter(lin.bias.detach().clone())
    del lin.bias
    lin.bias = bias
    with pytest.raises(RuntimeError, match="bias: this operator has no gradient"):
        lin(x)
    lin.bias.requires_grad_(False)
    assert torch.equal(lin(x), want)
