"""The rollout engines' page accounting: pages of ended sequences, errors, drafts. Tiny fp32 model."""
import pytest
import torch
from test_rollout_paged_cpu import _engine

from kore_b200.engine.multiturn import MultiTurnRollout
from kore_b200.engine.rollout import GenRequest, RolloutEngine, _Seq
from kore_b200.ops import spec


def _complete(eng):
    """Every page is free, once."""
    return sorted(eng.cache.free) == list(range(eng.cache.num_pages)) and not any(eng.cache.refcount) and not eng._prefix


def _prompt(n, seed=1):
    return torch.randint(0, 200, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


@pytest.mark.parametrize("max_batch", [1, 2, 3, 8])
@pytest.mark.parametrize("k", [0, 3])
def test_a_groups_first_sequence_ends_before_its_last_are_admitted(max_batch, k):
    """Its pages are free again: who comes later shares another's, or prefills its prompt itself."""
    budgets = [3, 9, 4, 8, 5, 7, 6, 12]
    p = _prompt(37)
    want = _engine().generate([GenRequest(p, n, rid=i) for i, n in enumerate(budgets)], temperature=0.0)
    eng = _engine()
    eng.max_batch = max_batch
    alloc = eng.cache.alloc

    def checked(n):
        assert not any(eng.cache.refcount[q] for q in eng.cache.free)       # no free page is in use
        return alloc(n)

    eng.cache.alloc = checked
    got = eng.generate([GenRequest(p, n, rid=i, share_key="a") for i, n in enumerate(budgets)], temperature=0.0, draft_tokens=k)
    assert [o.tokens for o in got] == [o.tokens for o in want] and _complete(eng)


@pytest.mark.parametrize("k", [0, 3])
@pytest.mark.parametrize("at", [0, 1, 2, 4])
def test_an_error_loses_no_page(k, at):
    """A forward that fails, and a row of logits without a distribution; then the same engine again."""
    reqs = lambda: [GenRequest(_prompt(37), 12, rid=i, share_key="a") for i in range(5)]
    want = _engine().generate(reqs(), temperature=0.0)
    eng = _engine()
    eng.max_batch = 3
    forward, calls = eng._forward, []

    def failing(*a, **kw):
        calls.append(1)
        if len(calls) == at + 1 and k == 0:
            raise KeyError("forward")
        out = forward(*a, **kw)
        if len(calls) >= at + 1 and kw.get("all_rows"):
            out[0].fill_(float("nan"))
        return out

    eng._forward = failing
    with pytest.raises(RuntimeError if k else KeyError):
        eng.generate(reqs(), temperature=0.0, draft_tokens=k)
    assert _complete(eng)
    eng._forward = forward
    assert [o.tokens for o in eng.generate(reqs(), temperature=0.0, draft_tokens=k)] == [o.tokens for o in want] and _complete(eng)


@pytest.mark.parametrize("k", [0, 3])
def test_results_are_in_the_requests_order_whatever_their_ids(k):
    """Requests of one rid (as the serving policy makes them), one of them twice."""
    prompts = [_prompt(n, n) for n in (5, 20, 11)]
    want = [_engine().generate([GenRequest(p, n)], temperature=0.0)[0].tokens for p, n in zip(prompts, (9, 4, 6))]
    reqs = [GenRequest(p, n) for p, n in zip(prompts, (9, 4, 6))]
    got = _engine().generate(reqs + reqs[1:2], temperature=0.0, draft_tokens=k)
    assert [o.tokens for o in got] == want + want[1:2] and all(o.rid == 0 for o in got)


def test_more_trajectories_than_shared_attention_takes_lose_no_page():
    eng = _engine()
    eng = RolloutEngine(eng.w, max_batch=8, page_size=8, num_pages=1200, max_seq_len=64, shared_attention=True)
    with pytest.raises(ValueError):
        MultiTurnRollout(eng).run([[1, 2, 3]] * 513, num_turns=1, max_new=2, feedback=lambda t, i, gen: [], max_feedback=1)
    assert _complete(eng)


@pytest.mark.parametrize("pool", [5, 6, 7, 12])
def test_rejected_drafts_keep_no_page(pool, monkeypatch):
    """Drafts that are all wrong change nothing: not which sequence the pool's last page goes to, nor who runs out."""
    reqs = lambda: [GenRequest(_prompt(20), 30, rid=0), GenRequest(_prompt(6), 4, rid=1), GenRequest(_prompt(9), 12, rid=2)][:2 + (pool > 6)]

    def outs(k):
        eng = _engine()
        eng._num_pages = pool
        got = eng.generate(reqs(), temperature=0.0, draft_tokens=k)
        assert _complete(eng)
        return [(o.tokens, o.finish_reason) for o in got]

    want = outs(0)
    used = {t for tokens, _ in want for t in tokens}
    wrong = next(t for t in range(200) if t not in used)
    monkeypatch.setattr(spec.Lookup, "draft", lambda self, k: [wrong] * max(k, 0))
    assert outs(7) == want


def test_a_sequence_without_room_is_an_error():
    """Pages that a sequence does not hold are another's: page 0 is not written in their place."""
    eng = _engine()
    for c in eng.cache.k + eng.cache.v:
        c.fill_(7.0)
    pages = eng.cache.alloc(2)
    s = _Seq(GenRequest([1] * 20, 1), pages, 0, 0, [1] * 20)
    with pytest.raises(RuntimeError, match="no room"):
        eng._forward([s], fresh=True)
    assert all((c == 7).all() for c in eng.cache.k + eng.cache.v) and s.length == 0 and len(s.pending) == 20
    eng.cache.release(pages)
    with pytest.raises(RuntimeError, match="no room"):              # 300 tokens with max_seq_len = 256
        eng.generate([GenRequest(_prompt(300), 1)], temperature=0.0)
    with pytest.raises(RuntimeError, match="no room"):
        eng.generate([GenRequest(_prompt(250), 20)], temperature=0.0, draft_tokens=3)
    assert _complete(eng)


@pytest.mark.parametrize("kw,tp,want", [(dict(rollout_draft_tokens=3), False, ["rollout_draft_tokens"]), (dict(rollout_shared_attention=True), False, []),
                                        (dict(rollout_draft_tokens=2, rollout_shared_attention=True), True, ["rollout_draft_tokens", "rollout_shared_attention"]),
                                        ({}, True, []), (dict(rollout_draft_tokens=3, batched_rollout=False), False, [])])
def test_grpo_names_options_that_its_rollout_does_not_use(kw, tp, want, monkeypatch):
    from kore_b200.env.base import SyntheticRewardEnv
    from kore_b200.policy import grpo
    from kore_b200.policy.configs import GRPOConfig
    eng = _engine()
    gc = GRPOConfig(num_trajectories=2, num_turns=1, tasks_per_step=1, max_response_length=4, max_prompt_length=64, temperature=1.0,
                    dynamic_sampling=False, starpo_s=False, bf16=False, total_steps=2, overlong_mask=False, top_p=1.0, **kw)
    tr = grpo.GRPOTrainer(gc, weights=eng.w, env=SyntheticRewardEnv(seed=0, prompt_len=16, feedback_len=4, vocab_size=eng.w.cfg.vocab_size),
                          rollout_kwargs=dict(num_pages=256, page_size=16, max_seq_len=512))
    said = []
    monkeypatch.setattr(grpo.log, "warning", lambda *a, **k: said.append(k["options"]))
    if tp:                              # the engine itself needs several GPUs
        monkeypatch.setattr(tr, "_use_tp", lambda: True)
        monkeypatch.setattr(tr, "_rollout_tp", lambda *a: [])
        tr.rollout_batch(["a"], [0, 1])
        tr.rollout_batch(["a"], [0, 1])
    else:
        tr.train_step(["a"])
        tr.train_step(["b"])
    assert said == ([want] if want else [])
