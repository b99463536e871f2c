"""The gradient of token_logprobs where hooks keep the saved tensors in another layout, or hand out others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def padded(t):
    """The same values, rows seven apart."""
    room = t.new_zeros(*t.shape[:-1], t.shape[-1] + 7)
    room[..., 3:3 + t.shape[-1]] = t
    return room[..., 3:3 + t.shape[-1]]


def apart(t):
    """The same values, none beside another."""
    return t.unsqueeze(-1).repeat(*[1] * t.dim(), 2)[..., 0]


HOOKS = {
    "clone": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(memory_format=torch.contiguous_format), lambda t: t),
    "save_on_cpu": torch.autograd.graph.save_on_cpu,
    "padded": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, padded),
    "apart": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t, apart),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [37, 4099])
@pytest.mark.parametrize("hooks", HOOKS)
def test_saved_in_another_layout(gpu, dtype, V, hooks):
    import m2_amd
    g = torch.Generator().manual_seed(V)
    B, L = 3, 5
    logits = torch.randn(B, L, V + 9, generator=g).to(gpu).to(dtype)[..., :V]
    tokens = torch.randint(0, V, (B, L, 2), generator=g).to(gpu)[..., 1]
    masks = (torch.rand(B, L, V + 13, generator=g).to(gpu) < 0.5)[..., 2:V + 2]
    masks[1, 2] = False
    for allowed in (None, masks, masks[0, 0].clone(), masks[0, 0].expand(B, L, V), masks[:, :1].expand(B, L, V), masks.transpose(0, 1).contiguous().transpose(0, 1)):
        def grads():
            x = logits.detach().requires_grad_()
            r = m2_amd.token_logprobs(x, tokens, 4, allowed)
            loss = r.logprobs.nan_to_num(neginf=0).sum() + 0.3 * r.entropy.sum() + (r.top_logprobs.nan_to_num(neginf=0) * torch.arange(1, 5, device=gpu)).sum()
            return loss, x
        loss, x = grads()
        want, = torch.autograd.grad(loss, x)
        with HOOKS[hooks]():
            loss, x = grads()
        got, = torch.autograd.grad(loss, x)
        assert torch.equal(got, want)


@pytest.mark.parametrize("other", [lambda t: t[..., :-1] if t.dim() else t, lambda t: t.to(torch.float16), lambda t: t.cpu(), lambda t: t.flatten()[:3]])
def test_other_tensors_are_refused(gpu, other):
    import m2_amd
    V = 64
    for which in range(6):      # logits, tokens, allowed tokens, entropies, sums, ids, as they are saved
        seen = []
        def unpack(i):
            return other(seen[i]) if i == which else seen[i]
        def pack(t):
            seen.append(t)
            return len(seen) - 1
        x = torch.randn(6, V, device=gpu).requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            r = m2_amd.token_logprobs(x, torch.zeros(6, dtype=torch.int64, device=gpu), 3, torch.ones(6, V, dtype=torch.bool, device=gpu))
            loss = r.logprobs.sum()
        assert len(seen) == 6
        with pytest.raises(RuntimeError, match="came back"):
            loss.backward()
