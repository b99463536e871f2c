"""The operators a masked-LM answer is made of, as cases that can be prepared, run and timed: products of few rows with 4-bit weights
(the head's two products), and log probabilities of given tokens with entropy and top alternatives, with and without their gradient.

`own` False: elementary torch operations in 32 bits, rounded once at the end.  `own` True: m2_amd's kernels, as a user calls them.

A case is a dict of plain values:

    kind     "linear"   y = act(x W^T + b), W in 4 bits with a bf16 scale for each group of K
             "scores"   log probability of a given token, entropy and the top alternatives of every row of logits
             "loss"     the same, with the gradient of the logits for given gradients of the outputs
    f32      True: fp32 rows or logits; False: bf16
    M, N, K, group, gelu          "linear": rows, output features, input features, values that share a scale, erf-GELU on the way out
    rows, V, top, pad, mask       "scores" and "loss": rows, vocabulary, alternatives asked for, columns behind the vocabulary that belong to
                                  the rows in memory, "" / "shared" / "rows": which tokens are allowed (nothing, one list, one per row)
    ignored                       share of the rows whose token is not asked for (-100)
"""
from __future__ import annotations

import math

import torch

own = False

IGNORED = -100


def _linear(name, M, N, K, group, f32=False, gelu=False):
    case = {"kind": "linear", "M": M, "N": N, "K": K, "group": group, "f32": f32, "gelu": gelu}
    return dict(case, name=name) if name else case


def _scores(name, kind, rows, V, top, f32=False, pad=0, mask="", ignored=0.0):
    case = {"kind": kind, "rows": rows, "V": V, "top": top, "f32": f32, "pad": pad, "mask": mask, "ignored": ignored}
    return dict(case, name=name) if name else case


def listed():
    return [
        # one masked place: hidden state to logits over the word embeddings, 768 wide
        _linear("linear_M1_768_words", 1, 30528, 768, 64),
        # the head's transform for three masked places, fp32 outside autocast, the 960-wide model
        _linear("linear_M3_960_gelu_f32", 3, 960, 960, 32, f32=True, gelu=True),
        # the masked places of a sentence, 1536 wide, a vocabulary that is not padded
        _linear("linear_M13_1536_words", 13, 30522, 1536, 128),
        # one row of a long product (the intermediate width of the 1792-wide model): nothing but weights
        _linear("linear_M1_7168_long", 1, 16384, 7168, 128),
        # every position of a text of 512 tokens: the compute-heavy end
        _linear("linear_M512_768_words", 512, 30528, 768, 64),
        # the masked places of a batch in fp32
        _linear("linear_M40_768_words_f32", 40, 30522, 768, 32, f32=True),
        # one masked place: the five most likely words
        _scores("scores_1x30522_top5", "scores", 1, 30522, 5),
        # 15 % of 4096 positions, the vocabulary's columns of a product padded to 30528
        _scores("scores_615x30522_top10_padded", "scores", 615, 30522, 10, pad=6),
        # every position of a batch of texts: likelihoods and entropies only
        _scores("scores_8192x30522", "scores", 8192, 30522, 0),
        # a long vocabulary of which each row may use a part of its own, one row nothing
        _scores("scores_24x131073_top32_masked_f32", "scores", 24, 131073, 32, f32=True, mask="rows"),
        # one sentence's loss with its gradient, fp32 logits, most positions not asked for
        _scores("loss_128x30522_f32", "loss", 128, 30522, 0, f32=True, ignored=0.85),
        # the masked places of a training batch: loss, entropy and alternatives with their gradient
        _scores("loss_4915x30528_top10", "loss", 4915, 30528, 10),
    ]


def _between(rng, low, high):
    """A whole number between two, spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "scores", "loss"])
    f32 = rng.random() < 0.4
    if kind == "linear":
        while True:
            M, N = _between(rng, 1, 512), _between(rng, 64, 40000)
            K = rng.choice([768, 960, 1536, 1792, _between(rng, 100, 8192)])
            if N * K <= 16384 * 7168 and M * N * K * (3 if f32 else 1) <= 512 * 30528 * 768:
                return _linear("", M, N, K, rng.choice([32, 64, 128]), f32, rng.random() < 0.3)
    while True:
        rows = _between(rng, 1, 8192)
        V = rng.choice([30522, 30528, _between(rng, 500, 131073)])
        if rows * V <= (8192 * 30522 if kind == "scores" else 4915 * 30528) // (2 if f32 else 1):
            mask = rng.choice(["", "", "", "shared", "rows"])
            return _scores("", kind, rows, V, rng.choice([0, 1, rng.randint(2, 32)]), f32, rng.choice([0, 0, rng.randint(1, 9)]), mask, rng.choice([0.0, 0.1, 0.85]))


def _scaled(w, group):
    """w (N, K) in 4 bits: codes 0 .. 15 as (N, ceil(K / 2)) bytes, even k in the low half, and a bf16 scale for each group of a row."""
    N, K = w.shape
    groups = -(-K // group)
    padded = torch.zeros(N, groups * group, device=w.device)
    padded[:, :K] = w
    padded = padded.view(N, groups, group)
    scales = (padded.abs().amax(-1) / 7).to(torch.bfloat16)
    codes = torch.round(padded / scales.float().clamp_min(1e-30).unsqueeze(-1)).clamp(-8, 7) + 8
    codes = codes.view(N, -1)[:, :K + K % 2].to(torch.uint8)
    if codes.shape[1] < K + K % 2:
        codes = torch.nn.functional.pad(codes, (0, 1), value=8)
    return codes[:, 0::2] | (codes[:, 1::2] << 4), scales


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed * 9973 + 17)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    dtype = torch.float32 if case["f32"] else torch.bfloat16
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        # weights as they come out of training (0.02 wide), rows as a LayerNorm leaves them
        packed, scales = _scaled(randn(N, K) * 0.02, case["group"])
        state = {"x": randn(M, K).to(dtype), "packed": packed, "scales": scales, "bias": randn(N) * 0.1}
        if own:
            import m2_amd
            # the weights in the kernels' order, made once, as a program that serves does
            state["linear"] = m2_amd.Int4Linear.from_packed(packed, scales, K, group_size=case["group"], bias=state["bias"])
        return {"case": case, **state}
    rows, V = case["rows"], case["V"]
    # logits as a masked-LM head gives them: low for nearly all words, a few stand out in every row
    logits = randn(rows, V + case["pad"]) * 2.0 - 6.0
    likely = torch.randint(0, V, (rows, 8), generator=gen, device=dev)
    logits.scatter_add_(1, likely, randn(rows, 8).abs() * 6.0)
    tokens = torch.where(torch.rand(rows, generator=gen, device=dev) < 0.6, likely[:, 0], torch.randint(0, V, (rows,), generator=gen, device=dev))
    tokens = torch.where(torch.rand(rows, generator=gen, device=dev) < case["ignored"], torch.full_like(tokens, IGNORED), tokens)
    allowed = None
    if case["mask"] == "shared":
        allowed = torch.rand(V, generator=gen, device=dev) < 0.7
    elif case["mask"] == "rows":
        allowed = torch.rand(rows, V, generator=gen, device=dev) < 0.5
        allowed[rows // 2] = False                    # a row that nothing is left of
        if rows > 2:
            allowed[0] = False
            allowed[0, V // 3] = allowed[0, V - 1] = True
    state = {"case": case, "logits": logits.to(dtype)[:, :V], "tokens": tokens, "allowed": allowed}
    if case["kind"] == "loss":
        state["grads"] = [randn(rows) / rows, randn(rows) * 0.1 / rows] + ([randn(rows, case["top"]) * 0.1 / rows] if case["top"] else [])
    return state


def _dequantized(state):
    case = state["case"]
    N, K, group = case["N"], case["K"], case["group"]
    codes = torch.stack((state["packed"] & 15, state["packed"] >> 4), -1).view(N, -1)[:, :K].float() - 8
    return codes * state["scales"].float().repeat_interleave(group, 1)[:, :K]


def _plain_linear(state):
    y = state["x"].float() @ _dequantized(state).t() + state["bias"]
    if state["case"]["gelu"]:
        y = 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    return y.to(state["x"].dtype)


def _first_keys(x, top):
    """Ids of the largest values of each row, ties to the lowest id: by keys that hold both and are all different."""
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits)
    keys = (bits << 32) + (0xFFFFFFFF - torch.arange(x.shape[1], device=x.device))
    return 0xFFFFFFFF - (keys.topk(top, -1).values & 0xFFFFFFFF)


def _plain_scores(state, with_grad):
    case, tokens = state["case"], state["tokens"]
    x = state["logits"].float()
    if state["allowed"] is not None:
        x = x.masked_fill(~state["allowed"], -math.inf)
    largest = x.amax(-1, keepdim=True)
    largest = torch.where(largest > -math.inf, largest, torch.zeros_like(largest))
    e = torch.exp(x - largest)
    s = e.sum(-1, keepdim=True).clamp_min(1e-30)      # at least 1, or the row is empty
    logp = x - largest - s.log()
    p = e / s
    entropy = -(p * logp.clamp_min(-1e30)).sum(-1)
    asked = tokens != IGNORED
    at = tokens.clamp_min(0).unsqueeze(-1)
    out = {"logprobs": torch.where(asked, logp.gather(-1, at).squeeze(-1), torch.zeros_like(entropy)), "entropy": entropy}
    ids = None
    if case["top"]:
        ids = _first_keys(x, case["top"])
        out["top_logprobs"] = logp.gather(-1, ids)
        out["top_ids"] = torch.where(out["top_logprobs"] > -math.inf, ids, torch.full_like(ids, -1))
    if with_grad:
        g_lp = torch.where(asked, state["grads"][0], torch.zeros_like(entropy)).unsqueeze(-1)
        g_h = state["grads"][1].unsqueeze(-1)
        total = g_lp
        if ids is not None:
            total = total + state["grads"][2].sum(-1, keepdim=True)
        grad = -p * (total + g_h * (logp.clamp_min(-1e30) + entropy.unsqueeze(-1)))
        grad.scatter_add_(-1, at, g_lp)
        if ids is not None:
            grad.scatter_add_(-1, ids, state["grads"][2])
        grad = grad.masked_fill(x == -math.inf, 0.0)
        out["grad"] = grad.to(state["logits"].dtype)
    return out


def _own_scores(state, with_grad):
    import m2_amd
    logits, top = state["logits"], state["case"]["top"]
    if with_grad:
        logits = logits.detach().requires_grad_()
    r = m2_amd.token_logprobs(logits, state["tokens"], top_k=top, allowed=state["allowed"], ignore_index=IGNORED)
    out = {"logprobs": r.logprobs, "entropy": r.entropy}
    if top:
        out["top_logprobs"], out["top_ids"] = r.top_logprobs, r.top_ids
    if with_grad:
        outputs = [r.logprobs, r.entropy] + ([r.top_logprobs] if top else [])
        out["grad"], = torch.autograd.grad(outputs, [logits], state["grads"])
    return out


def run(state):
    case = state["case"]
    if case["kind"] == "linear":
        if own:
            return state["linear"](state["x"], activation="gelu" if case["gelu"] else None)
        return _plain_linear(state)
    with_grad = case["kind"] == "loss"
    return _own_scores(state, with_grad) if own else _plain_scores(state, with_grad)


def work(case):
    size = 4 if case["f32"] else 2
    if case["kind"] == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // case["group"])
        return {"bytes": N * (-(-K // 2)) + 2 * N * groups + 4 * N + size * M * (K + N), "flops": 2 * M * N * K}
    rows, V = case["rows"], case["V"]
    mask = {"": 0, "shared": V, "rows": rows * V}[case["mask"]]
    passes, each = (3, 20) if case["kind"] == "loss" else (1, 10)
    return {"bytes": size * rows * V * passes + mask * (2 if passes == 3 else 1) + rows * (16 + 12 * case["top"]), "flops": each * rows * V}


def _exact_scores(state, with_grad):
    """From the definition: -sum p log p and so on, the gradient term by term."""
    x, tokens, top = state["logits"].double(), state["tokens"], state["case"]["top"]
    if state["allowed"] is not None:
        x = torch.where(state["allowed"], x, torch.tensor(-math.inf, dtype=torch.float64, device=x.device))
    empty = torch.isneginf(x).all(1)
    lse = torch.where(empty, torch.zeros_like(x[:, 0]), torch.logsumexp(x, 1))
    x -= lse[:, None]                                  # log probabilities from here on
    p = x.exp()
    entropy = torch.special.entr(p).sum(1)
    rows = torch.arange(len(tokens), device=x.device)
    asked = tokens != IGNORED
    out = {"logprobs": torch.where(asked, x[rows, tokens * asked], torch.zeros_like(lse)), "entropy": entropy}
    chosen = None
    if top:
        values, order = torch.sort(x, dim=1, descending=True, stable=True)
        out["top_logprobs"], chosen = values[:, :top].clone(), order[:, :top].clone()
        del values, order
        out["top_ids"] = chosen.masked_fill(torch.isneginf(out["top_logprobs"]), -1)
    if with_grad:
        masked = torch.isneginf(x)
        g = [t.double() for t in state["grads"]]
        x = x.masked_fill(masked, 0.0)                 # p is zero there
        grad = -g[1][:, None] * p * (x + entropy[:, None])
        grad -= (g[0] * asked)[:, None] * p
        grad[rows, tokens * asked] += g[0] * asked
        if chosen is not None:
            given = torch.zeros_like(p).scatter_(1, chosen, g[2])
            grad += given - given.sum(1, keepdim=True) * p
            del given
        out["grad"] = grad.masked_fill(masked, 0.0)
    return out


def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    if case["kind"] != "linear":
        return _exact_scores(state, case["kind"] == "loss")
    N, K, group = case["N"], case["K"], case["group"]
    byte = state["packed"].long()
    w = torch.empty(N, 2 * byte.shape[1], dtype=torch.float64, device=byte.device)
    w[:, 0::2], w[:, 1::2] = (byte % 16 - 8).double(), (byte // 16 - 8).double()
    w = w[:, :K]
    for g in range(state["scales"].shape[1]):
        w[:, g * group:(g + 1) * group] *= state["scales"][:, g:g + 1].double()
    y = torch.mm(state["x"].double(), w.t()) + state["bias"].double()
    return torch.special.ndtr(y) * y if case["gelu"] else y
