"""The rollout engines' page accounting: pages of ended sequences, errors, drafts. Tiny fp32 model."""
import pytest
import torch
from test_rollout_paged_cpu import _engine

from kore_b200.engine.rollout import GenRequest


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
