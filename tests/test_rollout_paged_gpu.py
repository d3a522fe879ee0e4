"""The rollout engines on the GPU with shared-prefix attention and drafted tokens:
transcripts' log-probs against the training engine's forward."""
import pytest
import torch

from kore_b200.engine.multiturn import MultiTurnRollout
from kore_b200.engine.qwen3_engine import Batch, Qwen3Engine
from kore_b200.engine.rollout import GenRequest, RolloutEngine
from kore_b200.engine.smoke import smoke_config
from kore_b200.models import Qwen3Weights
from kore_b200.ops import check_device_error

pytestmark = pytest.mark.gpu


def _weights():
    return Qwen3Weights(smoke_config(), device="cuda", dtype=torch.bfloat16, seed=0)


def _check(w, transcripts):
    """(context, tokens, logps) against the training engine at temperature 1, whose logits and
    whose own roundings are bf16 as the rollout's are (the bound of the plain rollout's test)."""
    tr = Qwen3Engine(w, allocate_grads=False)
    for context, tokens, logps in transcripts:
        m = torch.zeros(len(context) + len(tokens), dtype=torch.bool)
        m[len(context):] = True
        b = Batch.from_sequences([torch.tensor(context + tokens)], [m], device="cuda")
        lp, _ = tr.token_logprobs(b)
        assert (lp[b.targets >= 0].cpu() - torch.tensor(logps)).abs().mean() < 0.05
    assert check_device_error() == 0


@pytest.mark.parametrize("shared,k,page", [(True, 0, 64), (False, 5, 64), (True, 3, 16), (True, 7, 128)])
def test_generate(shared, k, page):
    w = _weights()
    eng = RolloutEngine(w, max_batch=8, page_size=page, num_pages=16384 // page, max_seq_len=2048, shared_attention=shared)
    g = torch.Generator().manual_seed(0)
    a, b = (torch.randint(0, w.cfg.vocab_size, (n,), generator=g).tolist() for n in (200, 77))
    a = a[:60] * 3 + a[180:]                         # repeats itself: there is something to look up
    reqs = [GenRequest(p, 40, rid=i, share_key=s) for i, (p, s) in enumerate([(a, 1), (a, 1), (a, 1), (b, 2), (b, 2), (b[:5], None)])]
    outs = eng.generate(reqs, temperature=1.0, seed=3, draft_tokens=k)
    assert all(len(o.tokens) == 40 for o in outs) and len({tuple(o.tokens) for o in outs}) == len(outs)
    _check(w, [(r.prompt, o.tokens, o.logps) for r, o in zip(reqs, outs)])
    assert len(eng.cache.free) == eng.cache.num_pages


def test_greedy_drafts_are_accepted():
    """A greedy random model runs into a loop: its continuation is found by look-up and accepted."""
    w = _weights()
    eng = RolloutEngine(w, max_batch=4, page_size=64, num_pages=64, max_seq_len=2048)
    steps = []
    forward = eng._forward
    eng._forward = lambda *a, **b: steps.append(1) or forward(*a, **b)
    out = eng.generate([GenRequest(list(range(20)), 200)], temperature=0.0, draft_tokens=7)[0]
    assert len(out.tokens) == 200 and len(steps) <= 200
    _check(w, [(list(range(20)), out.tokens, out.logps)])


@pytest.mark.parametrize("page", [16, 64])
def test_multiturn(page):
    w = _weights()
    eng = RolloutEngine(w, page_size=page, num_pages=16384 // page, max_seq_len=2048, shared_attention=True)
    g = torch.Generator().manual_seed(0)
    a, b = (torch.randint(0, w.cfg.vocab_size, (n,), generator=g).tolist() for n in (200, 77))
    prompts = [a, a, a, b, b]
    outs = MultiTurnRollout(eng, poll=16).run(prompts, num_turns=2, max_new=30, feedback=lambda t, i, gen: [1, 2, i],
                                              share_keys=[0, 0, 0, 1, 1], max_feedback=8, temperature=1.0, seed=5)
    assert len({tuple(o.gens[0]) for o in outs}) == len(outs)
    _check(w, [(o.contexts[t], o.gens[t], o.logps[t]) for o in outs for t in range(2)])
    assert len(eng.cache.free) == eng.cache.num_pages
