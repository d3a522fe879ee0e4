"""Edges of the step plan, shared-prefix attention and draft verification on CPU tensors."""
import math

import pytest
import torch
from paged_oracle import attention_oracle, build_cache

from test_paged_cpu import check_verify, verify_case

from kore_b200.ops import paged, spec


def _i(x):
    return torch.tensor(x, dtype=torch.int32)


@pytest.mark.parametrize("lead", [1, 5])
def test_rows_before_the_first_sequence(lead):
    a = build_cache([(5, [(9, 1), (30, 3)]), (0, [(7, 2)])], 8, 6, 2, dtype=torch.float32, D=16)
    want = attention_oracle(a)[0]
    q = torch.cat([torch.full((lead, 6, 16), math.nan), a["q"]])
    out = torch.full_like(q, 7.0)
    paged.prefix_attention(**{**a, "q": q, "q_start": a["q_start"] + lead}, max_q=3, out=out)
    assert (out[:lead] == 7).all() and torch.allclose(out[lead:].double(), want, atol=1e-5)


@pytest.mark.parametrize("tau", [0.8, 0.0])
def test_verify_rows_before_the_first_sequence(tau):
    z, tokens, qs, u, _ = verify_case(7, 100, [3, 4, 2])
    v = check_verify((z, tokens, qs[1:].contiguous(), u, None), tau)
    assert (v.logp[:3] == 0).all()


def check_extreme_temperatures(device):
    """From the smallest to the largest double: all weight on the largest logits, or the same on every token that is not masked."""
    z = torch.tensor([[0.0, 9.0, -math.inf, 9.0, 8.0, -math.inf, 3.0, 2.0]] * 2, device=device)
    u = torch.tensor([[0.5, 0.2], [0.5, 0.8]], device=device)
    tokens, qs = torch.zeros(2, dtype=torch.long, device=device), _i([0, 1, 2]).to(device)
    for tau, want, n in ((5e-324, [1, 3], 2), (1e-310, [1, 3], 2), (1e-200, [1, 3], 2), (1e-39, [1, 3], 2), (1e-30, [1, 3], 2),
                         (1e36, [1, 6], 6), (1e40, [1, 6], 6), (1e46, [1, 6], 6), (1e300, [1, 6], 6)):
        v = spec.verify(z, tokens, qs, u, tau)
        assert v.accepted.tolist() == [0, 0] and v.next.tolist() == want, tau
        assert (v.logp.cpu() + math.log(n)).abs().max() <= 2.0 ** -21, tau       # an fp32 result of up to 1.8 and sums of terms near 1
    for tau in (math.inf, math.nan, -1e-300):
        with pytest.raises(ValueError):
            spec.verify(z, tokens, qs, u, tau)


def test_verify_at_extreme_temperatures():
    check_extreme_temperatures("cpu")


def check_plan_with_an_empty_pool(device):
    """A stack without an entry is a pool: who lacks a page gets none, nor does who comes behind
    (the pages asked for up to there, 2, are more than the pool has)."""
    i = lambda x: _i(x).to(device)
    for free in (i([]), i([3, 4])[:0]):
        table = i([[5, 5], [6, 6], [7, 7]])
        p = paged.plan(i([0, 16, 15]), i([1, 1, 1]), table, 16, 3, free=free, free_count=i([0]))
        assert p.ok.tolist() == [False, False, False] and p.slots.tolist() == [-1, -1, -1]
        assert p.lens.tolist() == [0, 16, 15] and p.held.tolist() == [0, 1, 1] and p.free_count.tolist() == [0]
        assert table.tolist() == [[5, 5], [6, 6], [7, 7]]
        p = paged.plan(i([15, 16]), i([1, 1]), table[:2], 16, 2, free=free, free_count=i([0]))
        assert p.ok.tolist() == [True, False] and p.slots.tolist() == [5 * 16 + 15, -1] and p.lens.tolist() == [16, 16]


def test_plan_with_an_empty_pool():
    check_plan_with_an_empty_pool("cpu")


def check_plan_refuses_overlapping_rows(device):
    i = lambda x: _i(x).to(device)
    one, rows = i([1] * 5), i(list(range(20)))
    for table in (i([[0, 1, 2, 3]]).expand(5, 4), rows.as_strided((5, 4), (3, 1))):
        with pytest.raises((ValueError, RuntimeError)):
            paged.plan(i([0] * 5), one, table, 16, 5, free=i(list(range(9))), free_count=i([9]))
        p = paged.plan(i([0] * 5), one, table, 16, 5)              # without a pool a table is only read
        assert p.slots.tolist() == [16 * t for t in table[:, 0].tolist()]
    p = paged.plan(i([0]), i([40]), i([[7, 7, 7, 7]]).expand(1, 4).contiguous(), 16, 40, free=i([0, 1, 2]), free_count=i([3]))
    assert p.ok.tolist() == [True]


def test_plan_refuses_overlapping_rows():
    check_plan_refuses_overlapping_rows("cpu")


def test_attention_without_query_heads():
    a = build_cache([(20, [(25, 2), (21, 1)])], 16, 8, 2)
    out, lse = paged.prefix_attention(**{**a, "q": a["q"][:, :0]}, max_q=2, want_lse=True)
    assert out.shape == (3, 0, 128) and lse.shape == (3, 0)


def test_attention_refuses_starts_that_decrease():
    a = build_cache([(5, [(9, 2), (6, 1)]), (0, [(30, 3)])], 8, 6, 2, dtype=torch.float32, D=16)
    for bad in (dict(q_start=_i([0, 3, 2, 6])), dict(q_start=_i([4, 2, 3, 6])), dict(group_start=_i([2, 1, 3])), dict(group_start=_i([0, 3, 2]))):
        with pytest.raises(ValueError):
            paged.prefix_attention(**{**a, **bad}, max_q=3)
