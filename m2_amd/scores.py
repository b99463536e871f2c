"""What masked-LM logits say about given tokens: log probability, entropy and the most likely alternatives, in one pass over the logits,
and their gradient.

The reference leaves this to torch (`CrossEntropyLoss` over the head's logits, bert/src/bert_layers.py:1027-1064,1070-1318); the pooler is the
other thing a forward is turned into (`BertModel`, `M2BertTextEncoder`).
"""
from __future__ import annotations

from typing import NamedTuple, Optional

import torch

from . import ops


class TokenLogprobs(NamedTuple):
    """fp32 / int64, each of the logits' shape without its last dimension (the alternatives: with `top_k` in its place)."""
    logprobs: Optional[torch.Tensor]          # of the given tokens; None where none were given
    entropy: torch.Tensor                     # of the row's distribution, in nats
    top_ids: Optional[torch.Tensor]           # the most likely tokens, most likely first, equal ones by id; None for top_k = 0
    top_logprobs: Optional[torch.Tensor]


def token_logprobs(logits: torch.Tensor, tokens: Optional[torch.Tensor] = None, top_k: int = 0, allowed: Optional[torch.Tensor] = None,
                   ignore_index: int = -100) -> TokenLogprobs:
    """Log softmax of `logits` (..., V), fp32 or bf16 on the GPU, at `tokens` (...) int64, its entropy, and its `top_k` (0 to 32) largest values.

    `allowed`: bool, (V) for all rows or of the logits' shape; other tokens have probability zero whatever their logits hold (NaN too), as have
    those whose logit is -inf.  They get no gradient and are no alternatives: where fewer than `top_k` are left, ids are -1 and log
    probabilities -inf.  A row that nothing is left of has log probability -inf, entropy 0 and no gradient.  A row with a NaN or +inf
    among its allowed values is NaN throughout, its ids -1.  A token equal to `ignore_index` gives 0 and no gradient; one outside the vocabulary NaN
    (nothing is read there), in the row's gradient too.

    Differentiable once with respect to `logits`: log probabilities, entropy and the alternatives' log probabilities (their ids are taken
    as given).  Arithmetic is fp32; rows may lie any distance apart."""
    return TokenLogprobs(*ops.token_logprobs(logits, tokens, top_k, allowed, ignore_index))
