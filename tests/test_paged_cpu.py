"""The step plan, shared-prefix attention and draft verification on CPU tensors,
against 64-bit definitions, and their refusals."""
import math

import pytest
import torch
from paged_oracle import attention_oracle, build_cache, plan_oracle, verify_oracle

from kore_b200.ops import paged, spec


def _i(x):
    return torch.tensor(x, dtype=torch.int32)


PLANS = [
    dict(ctx=[0], new=[1], M=1, ps=16),
    dict(ctx=[5, 0, 31, 16], new=[1, 0, 2, 1], M=4, ps=16),
    dict(ctx=[5, 0, 31, 16], new=[40, 0, 2, 1], M=3, ps=16, pool=9, count=9),
    dict(ctx=[7, 7, 7, 7], new=[30, 30, 30, 30], M=5, ps=8, pool=9, count=9),       # runs short
    dict(ctx=[7, 7, 7], new=[99, 3, 1], M=4, ps=8, pool=9, count=9),                # the first does not fit its row
    dict(ctx=[8, 8], new=[1, 1], M=4, ps=8, pool=3, count=1, held=[3, 1]),          # pages held ahead
    dict(ctx=[-3, 4], new=[2, -1], M=2, ps=8, pool=3, count=7, rows=9),             # count past the stack, rows behind the last
    dict(ctx=[0, 0, 3], new=[4, 4, 4], M=2, ps=4, rows=6),                          # rows cut
    dict(ctx=[1, 2], new=[0, 0], M=1, ps=4, rows=3),
]


def plan_case(c):
    B, M = len(c["ctx"]), c["M"]
    table = [[100 + 10 * b + j for j in range(M)] for b in range(B)]
    rows = c.get("rows", sum(max(n, 0) for n in c["new"]))
    free = list(range(500, 500 + c["pool"])) if "pool" in c else None
    return table, rows, free


def check_plan(c, device):
    table, rows, free = plan_case(c)
    want = plan_oracle(c["ctx"], c["new"], table, c["ps"], rows, c.get("held"), free, c.get("count"))
    t = _i(table).reshape(len(table), c["M"]).to(device)
    put = lambda x: None if x is None else _i(x).to(device)
    stack = put(free)
    for again in range(2):                   # a step can be planned again
        got = paged.plan(put(c["ctx"]), put(c["new"]), t, c["ps"], rows, held=put(c.get("held")), free=stack,
                         free_count=None if free is None else put([c["count"]]))
        for k in ("q_start", "lens", "pos", "slots", "held"):
            assert getattr(got, k).dtype == torch.int32 and getattr(got, k).tolist() == want[k], k
        assert got.ok.tolist() == want["ok"] and t.tolist() == want["table"]
        assert (None if got.free_count is None else got.free_count.tolist()) == (None if free is None else [want["free_count"]])
    if stack is not None:
        assert stack.tolist() == free


@pytest.mark.parametrize("case", PLANS)
def test_plan(case):
    check_plan(case, "cpu")


def test_plan_refusals():
    t = _i([[0, 1]])
    with pytest.raises(ValueError):
        paged.plan(_i([0]), _i([1]), t, 16, 1, free=_i([3]))
    with pytest.raises(ValueError):
        paged.plan(_i([0]), _i([1]), t, 0, 1)
    with pytest.raises(ValueError):
        paged.plan(_i([0, 1]), _i([1, 1]), t, 16, 2)


GROUPS = [
    [(0, [(1, 1)])],
    [(5, [(9, 1), (6, 1), (30, 3)]), (16, [(40, 5)]), (0, [(3, 3), (0, 1), (7, 0)])],
    [(20, [(21, 1), (8, 2), (50, 2)])],       # a sequence shorter than its group's prefix
]


@pytest.mark.parametrize("groups", GROUPS)
@pytest.mark.parametrize("grouped", [True, False])
def test_prefix_attention(groups, grouped):
    a = build_cache(groups, 8, 6, 2, dtype=torch.float32, D=16)
    if not grouped:
        a.update(group_start=None, prefix_len=None)
    out, lse = paged.prefix_attention(**a, max_q=8, want_lse=True)
    want, wl, _, _ = attention_oracle(a)
    assert torch.allclose(out.double(), want, atol=1e-5) and torch.allclose(lse.double(), wl, atol=1e-5)


def test_prefix_attention_refusals():
    a = build_cache([(5, [(9, 1)])], 8, 6, 2, dtype=torch.float32, D=16)
    with pytest.raises(ValueError):
        paged.prefix_attention(**{**a, "prefix_len": None})
    with pytest.raises(ValueError):
        paged.prefix_attention(**{**a, "q": a["q"][:, :5]})


def verify_case(seed, V, lens, *, probs=False, dtype=torch.float32, device="cpu"):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    z = 2 * torch.randn(T, V, generator=g)
    top = torch.randint(0, V, (T,), generator=g)
    z[torch.arange(T), top] += 8 * torch.rand(T, generator=g)
    q = torch.softmax(z + 0.5 * torch.randn(T, V, generator=g), -1) if probs else None
    pick = torch.multinomial(q, 1, generator=g)[:, 0] if probs else torch.where(torch.rand(T, generator=g) < 0.7, top, torch.randint(0, V, (T,), generator=g))
    tokens = torch.cat([top[:1], pick[:-1]])
    q_start = [0]
    for n in lens:
        q_start.append(q_start[-1] + n)
    u = torch.rand(T, 2, generator=g)
    to = lambda x: None if x is None else x.to(device)
    return to(z.to(dtype)), to(tokens), to(_i(q_start)), to(u), to(q)


def V_chain(V):
    return 8 * (-(-V // (4096 * 8)))


def check_verify(case, tau):
    z, tokens, qs, u, q = case
    v = spec.verify(z, tokens, qs, u, tau, draft_probs=q)
    acc, nxt, logp = verify_oracle(z, tokens.tolist(), qs.tolist(), u.cpu(), tau, q)
    assert v.accepted.dtype == torch.int32 and v.accepted.tolist() == acc
    assert v.next.dtype == torch.long and v.next.tolist() == nxt
    n = qs.tolist()[-1]
    a, b = v.logp.double().cpu(), logp
    assert torch.equal(a.isnan(), b.isnan())
    # fp32 result (2^-24 of it); the sum behind its logarithm has terms that are off by up to 2^-21 and is taken in
    # fp32: a chain of V / 4096 vectors' elements a thread (8 each) and a tree over the threads
    tol = 2.0 ** -20 + (V_chain(z.shape[1]) + 24) * 2.0 ** -24 + 2.0 ** -24 * b.abs()
    fine = ~b.isnan()
    assert ((a - b).abs()[fine] <= tol[fine]).all(), float((a - b).abs()[fine].max())
    assert (a[n:] == 0).all()
    return v


@pytest.mark.parametrize("tau", [1.0, 0.6, 0.0])
@pytest.mark.parametrize("probs", [False, True])
def test_verify(tau, probs):
    check_verify(verify_case(1, 101, [4, 1, 0, 9, 2, 5], probs=probs), tau)


def test_verify_distribution():
    """The emitted token is distributed as the target's probabilities, drafts from another distribution or not."""
    V, n = 5, 20000
    g = torch.Generator().manual_seed(0)
    z, q = torch.randn(V, generator=g), torch.softmax(torch.randn(V, generator=g), -1)
    p = torch.softmax(z.double(), -1)
    for probs in (q.expand(2 * n, V), None):
        draft = torch.multinomial(q, n, replacement=True, generator=g) if probs is not None else torch.full((n,), 2)
        tokens = torch.stack([torch.zeros(n, dtype=torch.long), draft], 1).reshape(-1)
        v = spec.verify(z.expand(2 * n, V), tokens, _i(list(range(0, 2 * n + 1, 2))), torch.rand(2 * n, 2, generator=g), draft_probs=probs)
        first = torch.where(v.accepted > 0, draft, v.next)
        freq = torch.bincount(first, minlength=V).double() / n
        assert (freq - p).abs().max() < 5 * math.sqrt(0.25 / n)        # five standard deviations


def test_verify_refuses_negative_temperature():
    with pytest.raises(ValueError):
        spec.verify(torch.zeros(1, 4), torch.zeros(1, dtype=torch.long), _i([0, 1]), torch.zeros(1, 2), -1.0)
