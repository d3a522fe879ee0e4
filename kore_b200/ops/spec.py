"""Verification of drafted tokens (speculative decoding).

CUDA tensors run the native kernel; CPU tensors run the PyTorch definition below."""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import List, Optional, Sequence

import torch

from ._lib import native


@dataclass
class Verdict:
    accepted: torch.Tensor   # [B] int32: drafts accepted
    next: torch.Tensor       # [B] int64: the token after them
    logp: torch.Tensor       # [T] fp32: log-probs of the accepted drafts and of ``next``, row by row


class Lookup:
    """Drafts for a growing sequence by look-up in itself: what followed the last
    earlier place with the same ``ngram`` last tokens (fewer, down to one, where no
    place has them). A token costs ``ngram`` dictionary entries, a draft as many look-ups."""

    def __init__(self, tokens: Sequence[int] = (), ngram: int = 3):
        self.tokens: List[int] = []
        self.after = [{} for _ in range(ngram)]      # the last n tokens -> where what followed them begins
        self.extend(tokens)

    def extend(self, tokens: Sequence[int]) -> None:
        for t in tokens:
            j = len(self.tokens)
            for n in range(1, min(len(self.after), j) + 1):
                self.after[n - 1][tuple(self.tokens[j - n:])] = j
            self.tokens.append(t)

    def draft(self, k: int) -> List[int]:
        """Up to k tokens."""
        for n in range(min(len(self.after), len(self.tokens)), 0, -1):
            at = self.after[n - 1].get(tuple(self.tokens[-n:]))
            if at is not None:
                return self.tokens[at:at + max(k, 0)]
        return []


def verify(logits: torch.Tensor, tokens: torch.Tensor, q_start: torch.Tensor, u: torch.Tensor,
           temperature: float = 1.0, *, draft_probs: Optional[torch.Tensor] = None) -> Verdict:
    """Accept or reject each sequence's drafted tokens and draw the token after them.

    Sequence b was fed tokens[q_start[b] : q_start[b + 1]]: its last known token and
    the drafts after it. Row t of ``logits`` [T, V] (bf16 or fp32) is about the token
    after tokens[t], with p = softmax(logits[t] / temperature). ``draft_probs`` (fp32
    [T, V], rows aligned with ``logits``) is the distribution q that each draft was
    drawn from; without it a draft was certain (q is 1 at it). With the uniform
    numbers u [T, 2] in [0, 1):

    * the draft x after row t is accepted while u[t, 0] q(x) < p(x);
    * at the first rejected row r, ``next`` is the lowest v whose running sum of
      max(0, p - q) exceeds u[r, 1] of the total (of p where nothing is left);
      if all are accepted, r is the last row and ``next`` is drawn from p.

    The emitted tokens are distributed as if drawn from p one by one. Temperature
    0 is greedy: a draft is accepted while it is the (lowest) argmax, log-probs are
    those at temperature 1. ``logp`` is 0 in rows behind r, before the first sequence
    and behind the last one. Logits of -inf are masked tokens; at a row that has no distribution
    (all -inf, any NaN or +inf) nothing is accepted, ``next`` is -1 and its log-prob
    NaN. A draft outside the vocabulary is rejected. A sequence without rows gives
    0 and -1."""
    if not 0 <= temperature < math.inf:
        raise ValueError("verify: temperature must be finite and not negative")
    if logits.is_cuda:
        return Verdict(*native().spec_verify(logits, tokens, q_start, u, float(temperature), draft_probs))
    T, V = logits.shape
    starts = q_start.tolist()
    logp = torch.zeros(T, dtype=torch.float32)
    accepted, nxt = [], []
    for a, b in zip(starts[:-1], starts[1:]):
        t, y = a, -1
        while t < b:
            z = logits[t].double()
            lp = torch.log_softmax((z - z.max()) / (temperature if temperature > 0 else 1.0), -1)
            p = lp.exp()
            x = int(tokens[t + 1]) if t + 1 < b else -1
            if torch.isnan(p).any():
                logp[t] = math.nan
                break
            if 0 <= x < V:
                q = draft_probs[t].double() if draft_probs is not None else None
                if (x == int(z.argmax())) if temperature == 0 else float(u[t, 0]) * (1.0 if q is None else float(q[x])) < float(p[x]):
                    logp[t] = lp[x]
                    t += 1
                    continue
            if temperature == 0:
                y = int(z.argmax())
            else:
                w = p
                if t + 1 < b and draft_probs is not None:
                    w = (p - draft_probs[t].double()).clamp_min(0)
                elif 0 <= x < V:
                    w = p.clone()
                    w[x] = 0
                w = w if float(w.sum()) > 0 else p
                c = torch.cumsum(w, 0)
                y = min(int(torch.searchsorted(c, float(u[t, 1]) * c[-1:], right=True)), int(w.nonzero()[-1]))
            logp[t] = lp[y]
            break
        accepted.append(t - a)
        nxt.append(y)
    return Verdict(torch.tensor(accepted, dtype=torch.int32), torch.tensor(nxt, dtype=torch.long), logp)
