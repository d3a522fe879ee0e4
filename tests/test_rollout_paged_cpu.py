"""The rollout engines with shared-prefix attention and drafted tokens, on a tiny fp32 model."""
import pytest
import torch

from kore_b200.engine.multiturn import MultiTurnRollout
from kore_b200.engine.rollout import GenRequest, RolloutEngine
from kore_b200.models import PRESETS, Qwen3Weights
from kore_b200.ops import spec
from kore_b200.policy.configs import GRPOConfig


def _engine(**kw):
    torch.manual_seed(0)
    w = Qwen3Weights(PRESETS["qwen3-tiny"](200), device="cpu", dtype=torch.float32, seed=0)
    return RolloutEngine(w, max_batch=8, page_size=8, num_pages=200, max_seq_len=256, **kw)


def _requests(n=40):
    g = torch.Generator().manual_seed(1)
    a, b = (torch.randint(0, 200, (m,), generator=g).tolist() for m in (37, 20))
    return [GenRequest(p, n, rid=i, share_key=k) for i, (p, k) in enumerate([(a, "a"), (a, "a"), (a, "a"), (b, "b"), (b, "b"), (b[:9], None)])]


def _same(x, y):
    for a, b in zip(x, y):
        assert a.tokens == b.tokens and a.finish_reason == b.finish_reason
        assert torch.allclose(torch.tensor(a.logps), torch.tensor(b.logps), atol=1e-4)


def test_greedy_is_the_same_with_shared_attention_and_drafts():
    want = _engine().generate(_requests(), temperature=0.0)
    for kw, k in ((dict(shared_attention=True), 0), ({}, 4), (dict(shared_attention=True), 7)):
        eng = _engine(**kw)
        steps = []
        forward = eng._forward
        eng._forward = lambda *a, **b: steps.append(1) or forward(*a, **b)
        _same(eng.generate(_requests(), temperature=0.0, draft_tokens=k), want)
        assert len(eng.cache.free) == eng.cache.num_pages
        if k:       # a small random model repeats itself: drafts are accepted, steps are saved
            assert len(steps) < 41


def test_drafts_stop_at_eos_and_at_the_budget():
    want = _engine().generate(_requests(), temperature=0.0)
    eos = want[0].tokens[10]
    cut = _engine().generate(_requests(), temperature=0.0, eos_ids=[eos])
    _same(_engine().generate(_requests(), temperature=0.0, eos_ids=[eos], draft_tokens=5), cut)
    assert any(o.finish_reason == "stop" for o in cut)
    for n in (1, 2, 3):
        _same(_engine().generate(_requests(n), temperature=0.0, draft_tokens=5), _engine().generate(_requests(n), temperature=0.0))


def test_drafts_when_pages_run_out():
    """Drafts give way where the pool has no page for them; nothing is lost at the end."""
    eng = _engine()
    eng._num_pages = 14
    outs = eng.generate([GenRequest(list(range(30)), 60, rid=0), GenRequest(list(range(30)), 60, rid=1)], temperature=0.0, draft_tokens=7)
    assert all(o.finish_reason in ("kv_full", "length") for o in outs) and len(eng.cache.free) == 14


def test_drafted_samples_are_distributed_as_the_model():
    """First two sampled tokens of many samples of one prompt: with drafts as without, within five standard deviations."""
    eng = _engine()
    prompt, n = [5, 6, 7, 5, 6, 7, 5, 6], 400
    counts = []
    for k in (0, 3):
        outs = []
        for seed in range(n // 8):
            outs += eng.generate([GenRequest(prompt, 2, rid=i) for i in range(8)], temperature=0.05, seed=seed, draft_tokens=k)
        c = {}
        for o in outs:
            c[tuple(o.tokens)] = c.get(tuple(o.tokens), 0) + 1
        counts.append(c)
    for key in set(counts[0]) | set(counts[1]):
        a, b = counts[0].get(key, 0), counts[1].get(key, 0)
        assert abs(a - b) <= 5 * (max(a, b, 1) * 2) ** 0.5


def test_multiturn_is_the_same_with_shared_attention():
    outs = []
    for shared in (False, True):
        eng = _engine(shared_attention=shared)
        g = torch.Generator().manual_seed(3)
        p, q = (torch.randint(0, 200, (m,), generator=g).tolist() for m in (30, 19))
        outs.append(MultiTurnRollout(eng, poll=5).run([p, p, p, q, q], num_turns=3, max_new=9, feedback=lambda t, i, gen: [t + 1, i + 2],
                                                      share_keys=[0, 0, 0, 1, 1], max_feedback=4, temperature=0.0))
        assert len(eng.cache.free) == eng.cache.num_pages
    for a, b in zip(*outs):
        assert a.gens == b.gens and a.finish == b.finish and a.contexts == b.contexts
        for x, y in zip(a.logps, b.logps):
            assert torch.allclose(torch.tensor(x), torch.tensor(y), atol=1e-4)


def test_groups_of_a_batch():
    class S:
        def __init__(self, pages, shared):
            self.pages, self.shared_pages = pages, shared
    eng = _engine()
    a, b = [1, 2, 3, 4], [9, 8, 7]
    start, n = eng.prefix_groups([S(a, 0), S(a[:3] + [5], 3), S(a[:2] + [6], 2), S(b, 0), S([11], 0), S(b[:2] + [12], 2), S(b[:2] + [13], 2)], 8)
    assert start.tolist() == [0, 3, 4, 5, 7, 7, 7, 7, 7] and n.tolist() == [16, 0, 0, 16, 0, 0, 0, 0]


def test_lookup():
    draft = lambda tokens, k, n=3: spec.Lookup(tokens, n).draft(k)
    assert draft([1, 2, 3, 9, 1, 2, 3], 2) == [9, 1]
    assert draft([1, 2, 3, 8, 1, 2, 3, 9, 1, 2, 3], 5) == [9, 1, 2, 3]        # the last earlier place
    assert draft([4, 3, 7, 5, 3], 2) == [7, 5]                                # one token matches
    assert draft([1, 2, 3], 4) == [] and draft([], 3) == [] and draft([1, 1], 0) == [] and draft([1, 1], -2) == []
    assert draft([1, 1], 3) == [1]


@pytest.mark.parametrize("n", [1, 2, 3, 5])
def test_lookup_against_a_search(n):
    g = torch.Generator().manual_seed(n)
    tokens = torch.randint(0, 4, (120,), generator=g).tolist()
    look = spec.Lookup(tokens[:7], n)
    for end in range(7, len(tokens)):
        have, want = tokens[:end], []
        for m in range(min(n, end), 0, -1):
            places = [i for i in range(end - m) if have[i:i + m] == have[end - m:]]
            if places:
                want = have[places[-1] + m:places[-1] + m + 4]
                break
        assert look.draft(4) == want
        look.extend(tokens[end:end + 1])


def test_refusals():
    eng = _engine()
    for bad in (dict(draft_tokens=3, top_p=0.9), dict(draft_tokens=-1), dict(draft_tokens=2, draft_ngram=0)):
        with pytest.raises(ValueError):
            eng.generate(_requests(), temperature=1.0, **bad)
    w = eng.w
    with pytest.raises(ValueError):
        RolloutEngine(w, page_size=12, shared_attention=True)
    with pytest.raises(ValueError):
        RolloutEngine(w, max_batch=513, shared_attention=True)
    with pytest.raises(ValueError):
        RolloutEngine(w, max_batch=513, page_size=8, num_pages=9).generate(_requests(), draft_tokens=1)


def test_config_fields():
    c = GRPOConfig()
    assert c.rollout_shared_attention is False and c.rollout_draft_tokens == 0
