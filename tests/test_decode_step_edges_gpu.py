"""Edges of the step plan, shared-prefix attention and draft verification on the GPU."""
import math

import pytest
import torch
from paged_oracle import build_cache, check_attention, plan_oracle
from test_decode_step_edges_cpu import check_extreme_temperatures, check_plan_refuses_overlapping_rows, check_plan_with_an_empty_pool
from test_paged_cpu import check_verify, verify_case

from kore_b200.ops import check_device_error, paged, spec

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("groups,hq,hkv,max_q", [
    ([(0, [(1000, 1), (1000, 1)])], 40, 8, 1),
    ([(0, [(4096, 1)])], 40, 8, 1),
    ([(300, [(301, 1), (900, 3), (20, 2)]), (0, [(0, 1), (65, 4)])], 16, 2, 4),
    ([(0, [(400, 300)]), (333, [(600, 130), (340, 5)])], 10, 2, 300),
])
@pytest.mark.parametrize("lead", [1, 5, 63])
def test_rows_before_the_first_sequence(groups, hq, hkv, max_q, lead):
    """A batch that begins behind other rows: those stay, the others are what the batch gives by itself."""
    a = build_cache(groups, 64, hq, hkv, device="cuda", seed=lead)
    want, wl = paged.prefix_attention(**a, max_q=max_q, want_lse=True)
    check_attention(want, wl, a)
    q = torch.cat([torch.full((lead, hq, 128), math.nan, dtype=torch.bfloat16, device="cuda"), a["q"]])
    out = torch.full_like(q, 7.0)
    got, lse = paged.prefix_attention(**{**a, "q": q, "q_start": a["q_start"] + lead}, max_q=max_q, want_lse=True, out=out)
    assert check_device_error() == 0
    assert (got[:lead] == 7).all() and torch.equal(got[lead:], want) and torch.equal(lse[lead:], wl)


@pytest.mark.parametrize("tau", [0.8, 0.0])
@pytest.mark.parametrize("lens", [[3, 4, 2], [700, 2], [5, 0, 0]])
def test_verify_rows_before_the_first_sequence(tau, lens):
    z, tokens, qs, u, _ = verify_case(7, 100, lens, device="cuda")
    for _ in range(4):
        junk = torch.full((len(z),), 5.0, device="cuda")          # the log-probs may get this memory
        del junk
        v = check_verify((z, tokens, qs[1:].contiguous(), u, None), tau)
        assert (v.logp[:lens[0]] == 0).all()


@pytest.mark.parametrize("B", [1024, 1025, 5000])
@pytest.mark.parametrize("pool", [False, True])
def test_plan_without_rows(B, pool):
    """Many sequences and no row to plan, whatever they ask for."""
    ctx, new, table = [b % 40 for b in range(B)], [b % 3 for b in range(B)], [[b, b + 1, b + 2] for b in range(B)]
    free = list(range(7)) if pool else None
    held = [0] * B if pool else None
    want = plan_oracle(ctx, new, table, 16, 0, held, free, 7)
    t = _i(table)
    p = paged.plan(_i(ctx), _i(new), t, 16, 0, held=_i(held) if pool else None, free=_i(free) if pool else None, free_count=_i([7]) if pool else None)
    for k in ("q_start", "lens", "pos", "slots", "held", "ok"):
        assert getattr(p, k).tolist() == want[k], k
    assert t.tolist() == want["table"] and (not pool or p.free_count.tolist() == [want["free_count"]])


@pytest.mark.parametrize("tau", [1e-10, 1e-13, 1e-18, 1e-30])
@pytest.mark.parametrize("probs", [False, True])
def test_verify_at_small_temperatures(tau, probs):
    """All weight is on the largest logit. Those of the definition's quotients that are not the
    maximum lie at least 2^-23 / tau below it: their weights are 0 whatever these are rounded to."""
    check_verify(verify_case(7, 5000, [3, 4, 2], probs=probs, device="cuda"), tau)


def test_draw_among_equal_logits_at_small_temperatures():
    V = 3001
    z = torch.randn(8, V, device="cuda")
    z[:, [0, 1500, 1501, 3000]] = 17.3
    u = torch.tensor([0.0, 0.25, 0.2499, 0.5, 0.7499, 0.75, 0.9999999, 0.5001], device="cuda")
    u = torch.stack([u.flip(0), u], 1)
    for tau in (1e-4, 1e-9, 1e-14, 1e-17, 1e-25):
        v = spec.verify(z, torch.zeros(8, dtype=torch.long, device="cuda"), _i(list(range(9))), u, tau)
        assert v.next.tolist() == [0, 1500, 0, 1501, 1501, 3000, 3000, 1501]
        assert (v.logp + math.log(4.0)).abs().max() <= 2.0 ** -22          # an fp32 result of 1.39


def test_verify_at_extreme_temperatures():
    check_extreme_temperatures("cuda")


def test_plan_with_an_empty_pool():
    check_plan_with_an_empty_pool("cuda")


def test_plan_refuses_overlapping_rows():
    check_plan_refuses_overlapping_rows("cuda")


def test_attention_without_query_heads():
    a = build_cache([(20, [(25, 2), (21, 1)])], 16, 8, 2, device="cuda")
    for q in (a["q"][:, :0], torch.empty(3, 0, 128, dtype=torch.bfloat16, device="cuda")):
        out, lse = paged.prefix_attention(**{**a, "q": q}, max_q=2, want_lse=True)
        assert out.shape == (3, 0, 128) and lse.shape == (3, 0)


@pytest.mark.parametrize("max_q", [1, 3, 9])
def test_starts_that_decrease_give_zeros_and_an_error(max_q):
    a = build_cache([(100, [(300, 2), (160, 1)]), (0, [(90, 3)])], 16, 10, 2, device="cuda")
    want, _ = paged.prefix_attention(**a, max_q=max_q)
    assert check_device_error() == 0
    for bad in (dict(q_start=_i([0, 3, 2, 6])), dict(q_start=_i([0, 6, 3, 6])), dict(group_start=_i([2, 1, 3])), dict(group_start=_i([0, 3, 2]))):
        out, lse = paged.prefix_attention(**{**a, **bad}, max_q=max_q, want_lse=True)
        assert check_device_error() == 3 and (out == 0).all() and lse.isneginf().all()
    got, _ = paged.prefix_attention(**a, max_q=max_q)
    assert check_device_error() == 0 and torch.equal(got, want)


def test_scales():
    """The smallest and large scales that fp32 holds; what it cannot hold is refused."""
    a = build_cache([(20, [(25, 2), (21, 1)]), (0, [(300, 5)])], 16, 8, 2, device="cuda")
    for scale in (1e-37, 1e-6, 3.0):
        out, lse = paged.prefix_attention(**a, max_q=5, scale=scale, want_lse=True)
        check_attention(out, lse, {**a, "scale": scale})
    for scale in (1e-39, 1e-50, 1e39, math.inf, math.nan):
        with pytest.raises(RuntimeError):
            paged.prefix_attention(**a, max_q=5, scale=scale)


def test_out_may_not_overlap_q():
    a = build_cache([(20, [(25, 2), (21, 1)])], 16, 8, 2, device="cuda")
    both = torch.empty(6, 8, 128, dtype=torch.bfloat16, device="cuda")
    q = both[:3].copy_(a["q"])
    for out in (q, both[2:5]):
        with pytest.raises(RuntimeError):
            paged.prefix_attention(**{**a, "q": q}, max_q=2, out=out)
    out, lse = paged.prefix_attention(**{**a, "q": q}, max_q=2, out=both[3:], want_lse=True)
    check_attention(out, lse, a)
    wide = torch.empty(4, 8 * 128 + 64, dtype=torch.bfloat16, device="cuda")
    q = wide[:3, 64:].copy_(a["q"].flatten(1)).unflatten(1, (8, 128))
    check_attention(*paged.prefix_attention(**{**a, "q": q}, max_q=2, want_lse=True), a)
