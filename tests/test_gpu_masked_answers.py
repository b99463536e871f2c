"""What a masked-LM head answers, end to end: hidden states of the encoder at a few places, the head's two products in 4 bits, and log probabilities of
given words with entropy and alternatives."""
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def _model(gpu):
    import m2_amd
    cfg = m2_amd.m2_bert_80m(128)
    cfg.num_hidden_layers = 2
    model = m2_amd.BertModel(cfg)
    model.load_state_dict(m2_amd.seeded_state_dict(cfg, 11))
    return cfg, model.to(gpu).eval()


def _head(cfg, model, gpu, group):
    import m2_amd
    g = torch.Generator().manual_seed(4)
    d = cfg.hidden_size
    dense = m2_amd.Int4Linear.from_weight(torch.randn(d, d, generator=g).to(gpu) / d ** 0.5, torch.randn(d, generator=g).to(gpu) * 0.1, group)
    words = model.embeddings.word_embeddings.weight.detach() * 20
    decoder = m2_amd.Int4Linear.from_weight(words, torch.randn(words.shape[0], generator=g).to(gpu) * 0.1, group)
    gamma, beta = (torch.rand(d, generator=g) + 0.5).to(gpu), (torch.randn(d, generator=g) * 0.1).to(gpu)

    def head(h):
        t = dense(h, activation="gelu")
        n32, n16, _ = m2_amd.ops.layernorm(t, gamma, beta, 1e-12, want_f32=h.dtype == torch.float32, want_bf16=h.dtype == torch.bfloat16)
        return decoder(n32 if h.dtype == torch.float32 else n16)

    def plain(h):
        t = h.double() @ dense.dequantized().double().t() + dense.bias.double()
        t = torch.special.ndtr(t) * t
        t = (t - t.mean(-1, keepdim=True)) / (t.var(-1, unbiased=False, keepdim=True) + 1e-12).sqrt() * gamma.double() + beta.double()
        return t @ decoder.dequantized().double().t() + decoder.bias.double()

    return head, plain


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("places", [1, 7, 60, 200])
def test_encoder_to_words(gpu, dtype, places):
    """How far a log probability may be off.  fp32: sums of 768 products with logits of some ten units, 1e-4.  bf16: a logit is rounded once, by 2^-8 of itself at most
    (a quarter at 64, which the logits here reach: words 20 times the initial ones); the two roundings before it (transform, LayerNorm) come into it as sums of 768 random ones,
    2^-9 of the logits' root mean square each, six deviations of which are below 2^-8 of the largest.  A log probability is the difference of two such."""
    import m2_amd
    cfg, model = _model(gpu)
    head, plain = _head(cfg, model, gpu, 64)
    g = torch.Generator().manual_seed(places)
    ids = torch.randint(0, cfg.vocab_size, (2, 128), generator=g).to(gpu)
    with torch.no_grad():
        hidden, _ = model(ids)
        at = torch.randperm(256, generator=g)[:places].to(gpu)
        rows = hidden.reshape(256, -1)[at].to(dtype)
        logits = head(rows)
        words = ids.reshape(-1)[at]
        r = m2_amd.token_logprobs(logits, words, top_k=5)
    ref = plain(rows)
    assert logits.shape == (places, cfg.vocab_size) and logits.dtype == dtype
    logp = ref.log_softmax(-1)
    tol = 1e-4 if dtype == torch.float32 else 4 * 2.0 ** -8 * ref.abs().max()
    assert (r.logprobs.double() - logp.gather(-1, words[:, None])[:, 0]).abs().max() < tol
    assert (r.entropy.double() + (logp.exp() * logp).sum(-1)).abs().max() < tol * 3
    # the alternatives are those of the logits as they are, and nearly the reference's
    assert torch.equal(r.top_ids, logits.float().sort(dim=-1, descending=True, stable=True).indices[:, :5])
    assert ((logp.gather(-1, r.top_ids) - logp.topk(5).values).abs() < 2 * tol).all()


def test_the_loss_of_a_head_in_training(gpu):
    """Gradients reach a head of plain parameters: the mean log probability of the asked words against torch's cross entropy in fp64."""
    import m2_amd
    cfg, model = _model(gpu)
    g = torch.Generator().manual_seed(0)
    ids = torch.randint(0, cfg.vocab_size, (2, 128), generator=g).to(gpu)
    with torch.no_grad():
        hidden, _ = model(ids)
    labels = torch.where(torch.rand(2, 128, generator=g).to(gpu) < 0.15, ids, torch.full_like(ids, -100))
    w = (model.embeddings.word_embeddings.weight.detach() * 3).requires_grad_()
    b = torch.zeros(cfg.vocab_size, device=gpu, requires_grad=True)
    logits = torch.nn.functional.linear(hidden, w, b)
    loss = -m2_amd.token_logprobs(logits, labels).logprobs.sum() / (labels != -100).sum()
    got = torch.autograd.grad(loss, [w, b])
    w64, b64 = w.detach().double().requires_grad_(), b.detach().double().requires_grad_()
    ref = torch.nn.functional.cross_entropy(torch.nn.functional.linear(hidden.double(), w64, b64).reshape(-1, cfg.vocab_size), labels.reshape(-1))
    want = torch.autograd.grad(ref, [w64, b64])
    assert abs(loss.item() - ref.item()) < 1e-5 * abs(ref.item())
    for a, c in zip(got, want):      # fp32 products of 768 and of 256 terms on the way
        assert (a.double() - c).norm() < 1e-5 * c.norm()


def test_threads_and_streams_at_once(gpu):
    """Four threads with a stream each, sharing the weights."""
    import m2_amd
    cfg, model = _model(gpu)
    head, _ = _head(cfg, model, gpu, 128)
    g = torch.Generator().manual_seed(1)
    rows = [torch.randn(n, cfg.hidden_size, generator=g).to(gpu).to(torch.bfloat16) for n in (1, 9, 33, 150)]

    def answer(h):
        logits = head(h).float().requires_grad_()
        r = m2_amd.token_logprobs(logits, torch.zeros(h.shape[0], dtype=torch.int64, device=gpu), 3)
        return [r.logprobs.detach(), r.entropy.detach(), r.top_ids, *torch.autograd.grad(r.logprobs.sum(), [logits])]

    want = [answer(h) for h in rows]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i] = answer(rows[i])
                torch.cuda.current_stream().synchronize()
        except Exception as e:      # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip(a, b))
