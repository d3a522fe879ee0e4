"""Drafts in the rollout engine on the GPU: accepted ones save steps, emitted ones are distributed as the model."""
import math

import pytest
import torch
from test_rollout_drafts_cpu import count_drafts

from kore_b200.engine.rollout import GenRequest, RolloutEngine
from kore_b200.engine.smoke import smoke_config
from kore_b200.models import Qwen3Weights
from kore_b200.ops import check_device_error, spec

pytestmark = pytest.mark.gpu


def _engine(**kw):
    return RolloutEngine(Qwen3Weights(smoke_config(), device="cuda", dtype=torch.bfloat16, seed=0), max_batch=32, page_size=64,
                         num_pages=256, max_seq_len=1024, **kw)


@pytest.mark.parametrize("shared", [False, True])
def test_accepted_drafts_save_their_steps(shared, monkeypatch):
    """Drafts that are the plain engine's own continuation: as many decode steps less as drafts were accepted.
    A step of several rows may round its logits otherwise than one of a single row and leave that
    continuation; the drafts after that are wrong, and cost nothing but their step."""
    eng = _engine(shared_attention=shared)
    prompt, n = list(range(20)), count_drafts(monkeypatch)
    want = prompt + eng.generate([GenRequest(prompt, 200)], temperature=0.0)[0].tokens
    monkeypatch.setattr(spec.Lookup, "draft", lambda self, k: want[len(self.tokens):len(self.tokens) + max(k, 0)] if self.tokens == want[:len(self.tokens)] else [])
    steps, forward = [], eng._forward
    eng._forward = lambda *a, **b: steps.append(1) or forward(*a, **b)
    out = eng.generate([GenRequest(prompt, 200)], temperature=0.0, draft_tokens=7)[0]
    assert len(out.tokens) == 200 and n["accepted"] >= 7 and len(steps) == 200 - n["accepted"], (n, len(steps))
    assert check_device_error() == 0 and len(eng.cache.free) == eng.cache.num_pages


def test_emitted_drafts_are_distributed_as_the_model(monkeypatch):
    """Over the rows that came to a decision, drafts are emitted as often as the model says, within five standard deviations."""
    eng, n = _engine(shared_attention=True), count_drafts(monkeypatch)
    g = torch.Generator().manual_seed(2)
    prompt = torch.randint(0, eng.w.cfg.vocab_size, (70,), generator=g).tolist()
    for seed in range(12):
        eng.generate([GenRequest(prompt, 40, rid=i, share_key="p") for i in range(32)], temperature=0.05, seed=seed, draft_tokens=4)
    assert n["fed"] > 3000 and n["accepted"] > 300 and n["rejected"] > 300, n
    assert abs(n["excess"]) < 5 * math.sqrt(n["var"]), n
