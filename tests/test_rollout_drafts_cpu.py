"""Sampling with drafts in the rollout engine: tokens emitted behind accepted and rejected drafts."""
import math

import pytest
import torch
from test_rollout_paged_cpu import _engine

from kore_b200.engine.rollout import GenRequest, _Seq
from kore_b200.ops import spec


def model_logprobs(eng, contexts, temperature):
    """log p of every next token of each context, from one packed forward [tokens, V] a context."""
    seqs = [_Seq(GenRequest(c, 1), eng.cache.alloc(-(-len(c) // eng.page_size)), 0, 0, list(c)) for c in contexts]
    logits, _, starts = eng._forward(seqs, fresh=True, all_rows=True)
    for s in seqs:
        eng.cache.release(s.pages)
    lp = torch.log_softmax(logits.double() / temperature, -1)
    return [lp[a:b] for a, b in zip(starts.tolist()[:-1], starts.tolist()[1:])]


def count_drafts(monkeypatch):
    """Counts of the drafts fed, accepted and rejected from here on, and at the rows that came to a decision
    how often the draft was emitted, in excess of the model's probabilities, with that sum's variance."""
    n, verify = dict(fed=0, accepted=0, rejected=0, excess=0.0, var=0.0), spec.verify

    def counted(logits, tokens, q_start, u, temperature=1.0, **kw):
        v = verify(logits, tokens, q_start, u, temperature, **kw)
        fed = (q_start[1:] - q_start[:-1] - 1).cpu()
        n["fed"] += int(fed.sum())
        n["accepted"] += int(v.accepted.sum())
        n["rejected"] += int((v.accepted.cpu() < fed).sum())
        if temperature > 0:
            for a, b, acc, y in zip(q_start.tolist()[:-1], q_start.tolist()[1:], v.accepted.tolist(), v.next.tolist()):
                for t in range(a, min(a + acc + 1, b - 1)):
                    x = int(tokens[t + 1])
                    p = float(torch.softmax(logits[t].double() / temperature, -1)[x])
                    n["excess"] += float(t < a + acc or y == x) - p          # a rejected draft is not drawn again
                    n["var"] += p * (1 - p)
        return v

    monkeypatch.setattr(spec, "verify", counted)
    return n


@pytest.mark.parametrize("shared", [False, True])
def test_tokens_behind_drafts_are_distributed_as_the_model(shared, monkeypatch):
    """Given the tokens before it, a token's log-prob has the model's mean and variance there, and it is the
    likeliest one, or the one that was drafted, as often as the model says: sums of such differences are within
    five standard deviations."""
    temperature, n = 0.03, count_drafts(monkeypatch)
    eng, plain = _engine(shared_attention=shared), _engine()
    prompt = [5, 6, 7, 5, 6, 7, 5, 6, 9, 9, 9, 9]
    diff, var, hits, hits_var = 0.0, 0.0, 0.0, 0.0
    for seed in range(30):
        outs = eng.generate([GenRequest(prompt, 16, rid=i, share_key="p") for i in range(8)], temperature=temperature, seed=seed, draft_tokens=4)
        for o, lp in zip(outs, model_logprobs(plain, [prompt + o.tokens[:-1] for o in outs], temperature)):
            lp = lp[len(prompt) - 1:]
            tokens = torch.tensor(o.tokens)
            got = lp[torch.arange(16), tokens]
            assert (got - torch.tensor(o.logps, dtype=torch.float64)).abs().max() < 1e-4       # the reported log-prob is its row's
            p, lp, got, tokens = lp[1:].exp(), lp[1:], got[1:], tokens[1:]                      # the first token is the prefill's
            mean = (p * lp).sum(-1)
            diff += float((got - mean).sum())
            var += float(((p * lp * lp).sum(-1) - mean * mean).sum())
            top = p.max(-1)
            hits += float(((tokens == top.indices).double() - top.values).sum())
            hits_var += float((top.values * (1 - top.values)).sum())
    assert n["fed"] > 1000 and n["accepted"] > 300 and n["rejected"] > 300, n
    assert abs(n["excess"]) < 5 * math.sqrt(n["var"]), n
    assert abs(diff) < 5 * math.sqrt(var) and abs(hits) < 5 * math.sqrt(hits_var), (diff, var, hits, hits_var)


@pytest.mark.parametrize("k", [1, 4, 9])
def test_accepted_drafts_save_their_steps(k, monkeypatch):
    """Greedy: the plain engine's tokens, one decode step less for each accepted draft that was kept."""
    n = count_drafts(monkeypatch)
    prompt = [3, 1, 4, 1, 5]
    want = _engine().generate([GenRequest(prompt, 60)], temperature=0.0)[0].tokens
    eng, steps = _engine(), []
    forward = eng._forward
    eng._forward = lambda *a, **b: steps.append(1) or forward(*a, **b)
    assert eng.generate([GenRequest(prompt, 60)], temperature=0.0, draft_tokens=k)[0].tokens == want
    assert n["accepted"] > 0 and len(steps) == 60 - n["accepted"], (n, len(steps))
