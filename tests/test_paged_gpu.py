"""The step plan and shared-prefix attention on the GPU, against 64-bit definitions."""
import math

import pytest
import torch
from paged_oracle import attention_oracle, build_cache, check_attention, plan_oracle
from test_paged_cpu import PLANS, check_plan

from kore_b200.engine.rollout import paged_attention_reference
from kore_b200.ops import check_device_error, paged

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------------ plan
@pytest.mark.parametrize("case", PLANS)
def test_plan(case):
    check_plan(case, "cuda")


@pytest.mark.parametrize("B,new,ps,short", [(1, 5000, 64, False), (1023, 1, 16, True), (1025, 9, 8, False),
                                            (2500, 3, 16, True), (64, 700, 128, True), (31, 0, 16, False)])
def test_plan_sizes(B, new, ps, short):
    g = torch.Generator().manual_seed(B)
    ctx = torch.randint(0, 200, (B,), generator=g).tolist()
    n = torch.randint(0, new + 1, (B,), generator=g).tolist()
    M = (200 + new) // ps + 2
    table = torch.randint(0, 10 ** 4, (B, M), generator=g).tolist()
    held = [-(-c // ps) + int(k) for c, k in zip(ctx, torch.randint(0, 2, (B,), generator=g))]
    asked = sum(max(0, -(-(c + m) // ps) - h) for c, m, h in zip(ctx, n, held))
    pool = max(1, asked // 2) if short else asked + 3
    rows = sum(n) + 7
    free = torch.randperm(pool, generator=g).tolist()
    want = plan_oracle(ctx, n, table, ps, rows, held, free, pool)
    t = _i(table)
    got = paged.plan(_i(ctx), _i(n), t, ps, rows, held=_i(held), free=_i(free), free_count=_i([pool]))
    for k in ("q_start", "lens", "pos", "slots", "held", "ok"):
        assert getattr(got, k).tolist() == want[k], k
    assert t.tolist() == want["table"] and got.free_count.tolist() == [want["free_count"]]
    wide = torch.full((B, M + 3), -7, dtype=torch.int32, device="cuda")          # rows of a wider table
    wide[:, :M] = _i(table)
    paged.plan(_i(ctx), _i(n), wide[:, :M], ps, rows, held=_i(held), free=_i(free), free_count=_i([pool]))
    assert wide[:, :M].tolist() == want["table"] and (wide[:, M:] == -7).all()


def test_plan_without_sequences_and_with_wide_numbers():
    none = torch.empty(0, dtype=torch.int32, device="cuda")
    p = paged.plan(none, none, torch.empty(0, 4, dtype=torch.int32, device="cuda"), 16, 3)
    assert p.q_start.tolist() == [0] and p.pos.tolist() == [0] * 3 and p.slots.tolist() == [-1] * 3 and p.lens.numel() == 0
    big = 2 ** 31 - 1                                  # lengths that fit no table
    p = paged.plan(_i([big, 5, big]), _i([1, 1, big]), torch.zeros(3, 4, dtype=torch.int32, device="cuda"), 16, 4)
    assert p.ok.tolist() == [False, True, False] and p.lens.tolist() == [big, 6, big]
    assert p.q_start.tolist() == [0, 1, 2, 4] and p.slots.tolist() == [-1, 5, -1, -1]


def test_plan_captured():
    """Captured and replayed over its own results: each replay appends a token to every sequence."""
    ps, B, steps = 16, 5, 40
    ctx, held, count = _i([0, 15, 16, 3, 40]), _i([0, 1, 1, 1, 3]), _i([12])
    one, table, free = _i([1] * B), torch.full((B, 6), -1, dtype=torch.int32, device="cuda"), torch.arange(100, 112, dtype=torch.int32, device="cuda")
    table[:, :3] = torch.arange(3 * B, dtype=torch.int32, device="cuda").view(B, 3)
    c, h, t, n = ctx.tolist(), held.tolist(), table.tolist(), 12
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        paged.plan(ctx, one, table.clone(), ps, B, held=held, free=free, free_count=count)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        p = paged.plan(ctx, one, table, ps, B, held=held, free=free, free_count=count)
        ctx.copy_(p.lens)
        held.copy_(p.held)
        count.copy_(p.free_count)
    for _ in range(steps):
        w = plan_oracle(c, [1] * B, t, ps, B, h, free.tolist(), n)
        c, h, t, n = w["lens"], w["held"], w["table"], w["free_count"]
        graph.replay()
        assert p.slots.tolist() == w["slots"] and p.ok.tolist() == w["ok"]
        assert ctx.tolist() == c and held.tolist() == h and table.tolist() == t and count.tolist() == [n]


def test_plan_refusals():
    t, one = _i([[0, 1]]), _i([1])
    for bad in (dict(ctx=_i([0, 1])), dict(new=torch.tensor([1], device="cuda")), dict(new=torch.tensor([1], dtype=torch.int32)),
                dict(table=t.t()), dict(table=torch.stack([t, t], -1)[..., 0]), dict(page_size=0), dict(rows=-1),
                dict(held=_i([1, 2])), dict(free=_i([3])), dict(free=_i([3]), free_count=_i([1, 2]))):
        a = dict(ctx=_i([0]), new=one, table=t, page_size=16, rows=1)
        a.update(bad)
        with pytest.raises(RuntimeError):
            paged.plan(a.pop("ctx"), a.pop("new"), a.pop("table"), a.pop("page_size"), a.pop("rows"), **a)


# ------------------------------------------------------------------- attention
def run(a, **kw):
    out, lse = paged.prefix_attention(**a, want_lse=True, **kw)
    assert check_device_error() == 0
    return out, lse


CASES = [
    # one row, one key; lengths around the 64 keys of a tile
    ([(0, [(1, 1)])], 64, 4, 4),
    ([(0, [(63, 1), (64, 1), (65, 1), (128, 1), (1, 1)])], 64, 10, 2),
    # nothing cached, and sequences without rows
    ([(0, [(0, 0), (5, 1), (0, 0)]), (0, [(0, 1)]), (0, [(7, 0)])], 16, 8, 4),
    # groups: prefixes that end inside a page or a tile, ragged suffixes, one and several query tokens
    ([(100, [(101, 1), (164, 1), (700, 1)]), (64, [(65, 1)]), (1, [(2, 1), (300, 1)])], 32, 40, 8),
    ([(200, [(205, 5), (260, 1), (203, 3)]), (129, [(140, 8), (137, 8)])], 64, 32, 4),
    # a sequence shorter than its group's prefix, one without rows, and one that is empty
    ([(150, [(151, 1), (40, 2), (500, 3), (90, 0), (0, 0)]), (0, [(33, 1)])], 16, 6, 1),
    # pages of odd sizes (boxes of 8 rows), of more than a tile, of three halves
    ([(70, [(75, 1), (200, 2)])], 8, 5, 1),
    ([(70, [(75, 1), (200, 2)])], 24, 16, 2),
    ([(70, [(75, 1), (333, 2)]), (0, [(97, 97)])], 96, 8, 8),
    ([(300, [(301, 1), (700, 2)])], 256, 12, 4),
    # more rows than a tile of 128: many samples of a prompt, long extends, 128 heads to one
    ([(500, [(510 + i, 1) for i in range(60)])], 64, 10, 2),
    ([(0, [(400, 300)]), (333, [(600, 130), (340, 5)])], 64, 10, 2),
    ([(90, [(100, 3), (95, 2)])], 64, 128, 1),
    ([(90, [(100, 3), (95, 2)])], 64, 100, 1),
    # long histories, split over many blocks
    ([(4097, [(4098, 1), (9000, 1)])], 64, 40, 8),
    ([(0, [(20000, 4)])], 64, 8, 1),
    ([(9000, [(9001 + 37 * i, 1 + i % 3) for i in range(20)])], 32, 16, 2),
]


@pytest.mark.parametrize("groups,ps,hq,hkv", CASES)
def test_prefix_attention(groups, ps, hq, hkv):
    a = build_cache(groups, ps, hq, hkv, device="cuda", seed=len(groups))
    check_attention(*run(a, max_q=max(m for _, s in groups for _, m in s) or 1), a)


@pytest.mark.parametrize("groups,ps,hq,hkv", CASES)
def test_without_groups(groups, ps, hq, hkv):
    """Each sequence by itself, through its own table; the hint max_q is off."""
    groups = [(0, [x]) for _, s in groups for x in s]
    a = build_cache(groups, ps, hq, hkv, device="cuda", seed=1)
    a.update(group_start=None, prefix_len=None)
    check_attention(*run(a, max_q=2), a)


def test_many_sequences():
    """512 sequences in 300 groups, some groups empty of shared keys, some of sequences."""
    g = torch.Generator().manual_seed(5)
    cut = sorted(torch.randint(0, 513, (299,), generator=g).tolist())
    groups = []
    for a, b in zip([0] + cut, cut + [512]):
        P = int(torch.randint(0, 90, (1,), generator=g))
        groups.append((P, [(P + 1 + int(torch.randint(0, 60, (1,), generator=g)), 1) for _ in range(b - a)]))
    a = build_cache(groups, 16, 4, 2, device="cuda", seed=2)
    check_attention(*run(a), a)


@pytest.mark.parametrize("big", [True, False])
def test_large_scores(big):
    """Scores that reach thousands, and rows whose scores are all equal."""
    a = build_cache([(100, [(130, 2), (101, 1)]), (0, [(70, 1)])], 16, 10, 2, device="cuda")
    if big:
        a["q"] = (a["q"].float() * 100).bfloat16()
    else:
        a["q"] = torch.zeros_like(a["q"])
    check_attention(*run(a, max_q=2), a)


def test_layouts():
    """q inside a wider projection; K and V interleaved per slot, heads before slots, and at offsets."""
    groups = [(100, [(130, 3), (101, 1)]), (0, [(77, 1)])]
    a = build_cache(groups, 32, 10, 2, device="cuda", q_pad=40)
    assert a["q"].stride(0) == 1320
    k, v = a["k_cache"], a["v_cache"]
    want = run(a, max_q=3)
    check_attention(*want, a)
    both = torch.full((k.shape[0], 2, 3, 128), math.nan, dtype=torch.bfloat16, device="cuda")
    both[:, :, 0], both[:, :, 2] = k, v
    heads = torch.empty(2, 2, k.shape[0], 128, dtype=torch.bfloat16, device="cuda")
    heads[0], heads[1] = k.transpose(0, 1), v.transpose(0, 1)
    for kk, vv in ((both[:, :, 0], both[:, :, 2]), (heads[0].transpose(0, 1), heads[1].transpose(0, 1))):
        got = run({**a, "k_cache": kk, "v_cache": vv}, max_q=3)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rows_behind_the_last_are_left():
    a = build_cache([(20, [(25, 2), (21, 1)])], 16, 8, 2, device="cuda", pad_rows=5)
    a["q"][3:] = math.nan
    out = torch.full((8, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
    got, lse = run(a, max_q=2, out=out)
    assert got is out and (out[3:] == 7).all()
    check_attention(got, lse, a)


def test_scale_and_no_lse():
    a = build_cache([(20, [(25, 2), (21, 1)])], 16, 8, 2, device="cuda")
    out, lse = paged.prefix_attention(**a, max_q=2, scale=0.02)
    assert lse is None
    check_attention(out, None, {**a, "scale": 0.02})


def test_repeats_are_equal_and_streams_do_not_share():
    a = build_cache([(2000, [(2100 + 13 * i, 1) for i in range(30)])], 64, 40, 8, device="cuda")
    b = build_cache([(0, [(700, 4)] * 3)], 64, 40, 8, device="cuda", seed=3)
    torch.cuda.synchronize()
    first, other = run(a)[0], run(b, max_q=4)[0]
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for _ in range(20):
        with torch.cuda.stream(s1):
            outs.append((paged.prefix_attention(**a)[0], first))
        with torch.cuda.stream(s2):
            outs.append((paged.prefix_attention(**b, max_q=4)[0], other))
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in outs) and check_device_error() == 0


def test_captured_with_changing_lengths():
    """Two graphs of the same kind, replayed in turn; lengths and groups change on the device in between."""
    x = build_cache([(128, [(150, 1), (300, 1)]), (64, [(70, 1), (64 + 200, 1)])], 64, 10, 2, device="cuda")
    y = build_cache([(10, [(400, 2), (20, 1)])], 64, 10, 2, device="cuda", seed=9)
    run(x), run(y, max_q=2)
    graphs = []
    for a, m in ((x, 1), (y, 2)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = paged.prefix_attention(**a, max_q=m, want_lse=True)
        graphs.append((graph, got, a))
    for step in range(3):
        for graph, _, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, (out, lse), a in graphs:
            check_attention(out, lse, a)
        x["lens"] -= 3                               # shorter histories, and another split into groups
        x["prefix_len"].copy_(_i([100, 0] if step == 0 else [0, 60]))
        y["q"].mul_(-1)
    assert check_device_error() == 0


def test_on_a_side_stream():
    """The launch goes to the current stream."""
    a = build_cache([(40, [(45, 2), (41, 1)])], 16, 8, 2, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, lse = paged.prefix_attention(**a, max_q=2, want_lse=True)
    torch.cuda.current_stream().wait_stream(side)
    check_attention(out, lse, a)


def test_offsets_past_32_bits():
    """A cache of more than 2^31 elements whose pages lie at both of its ends."""
    hkv, ps = 8, 64
    slots = (2 ** 31 // (hkv * 128) // ps + 50) * ps
    kc, vc = (torch.empty(slots, hkv, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert kc.numel() > 2 ** 31
    n = 5
    pages = [slots // ps - 1 - i if i % 2 else i for i in range(n)]
    small = [torch.randn(n * ps, hkv, 128).bfloat16() for _ in range(2)]
    for c, s in ((kc, small[0]), (vc, small[1])):
        for i, p in enumerate(pages):
            c[p * ps:(p + 1) * ps] = s[i * ps:(i + 1) * ps].cuda()
    q = torch.randn(2, 16, 128).bfloat16()
    one = dict(q=q, lens=torch.tensor([n * ps, n * ps - 9], dtype=torch.int32), q_start=torch.tensor([0, 1, 2], dtype=torch.int32),
               page_size=ps, group_start=torch.tensor([0, 2], dtype=torch.int32), prefix_len=torch.tensor([130], dtype=torch.int32))
    far = {k: v.cuda() if torch.is_tensor(v) else v for k, v in one.items()}
    out, lse = run(dict(far, k_cache=kc, v_cache=vc, table=_i([pages, pages])))
    rows = torch.arange(n, dtype=torch.int32)[None].expand(2, n).contiguous()
    check_attention(out, lse, dict(one, k_cache=small[0], v_cache=small[1], table=rows))


def test_plan_append_attend_together():
    """Drafted steps as an engine runs them: plan with a pool, append, attend; lengths roll back in between."""
    from kore_b200.ops import native
    torch.manual_seed(0)
    ps, B, hq, hkv, P = 16, 6, 10, 2, 37
    slots = 200 * ps
    kc, vc = (torch.full((slots, hkv, 128), math.nan, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    table = torch.zeros(B, 30, dtype=torch.int32, device="cuda")
    free, count = torch.randperm(200, device="cuda").int(), _i([200])
    # the prompt once, then its whole pages in every table
    p = paged.plan(_i([0]), _i([P]), table[:1], ps, P, free=free, free_count=count)
    k, v = (torch.randn(P, hkv, 128, device="cuda").bfloat16() for _ in range(2))
    native().kv_append(k, v, p.slots, kc, vc)
    hist = [(k, v)] * B
    table[1:, :P // ps] = table[0, :P // ps]
    lens, held, count = _i([P] + [P // ps * ps] * (B - 1)), _i([-(-P // ps)] + [P // ps] * (B - 1)), p.free_count
    hist = [(k, v)] + [(k[:P // ps * ps], v[:P // ps * ps])] * (B - 1)
    shared = P // ps * ps
    for step in range(12):
        new = torch.randint(0, 6, (B,)).tolist()
        T = sum(new)
        if T == 0:
            continue
        p = paged.plan(lens, _i(new), table, ps, T + 2, held=held, free=free, free_count=count)
        assert p.ok.all()
        k, v = (torch.randn(T + 2, hkv, 128, device="cuda").bfloat16() for _ in range(2))
        native().kv_append(k, v, p.slots, kc, vc)            # rows behind the last sequence have slot -1
        q = torch.randn(T + 2, hq, 128, device="cuda").bfloat16()
        out, _ = paged.prefix_attention(q, kc, vc, table, p.lens, p.q_start, ps, max_q=5, group_start=_i([0, B]), prefix_len=_i([shared]))
        at = 0
        for b, n in enumerate(new):
            hist[b] = tuple(torch.cat([h, x[at:at + n]]) for h, x in zip(hist[b], (k, v)))
            at += n
        L = [h[0].shape[0] for h in hist]
        assert p.lens.tolist() == L
        dense_k, dense_v = (torch.cat([h[i] for h in hist]) for i in range(2))
        starts = [0]
        for n in L:
            starts.append(starts[-1] + n)
        flat = dict(q=q, k_cache=dense_k, v_cache=dense_v, lens=p.lens, q_start=p.q_start, page_size=1,
                    table=torch.stack([torch.arange(max(L), dtype=torch.int32) + s for s in starts[:-1]]))
        check_attention(out, None, flat)
        keep = [n - int(torch.randint(0, 3, (1,))) if n > 2 else n for n in new]         # rejected drafts: the length goes back
        hist = [tuple(h[:L[b] - new[b] + keep[b]] for h in hist[b]) for b in range(B)]
        lens, held, count = _i([h[0].shape[0] for h in hist]), p.held, p.free_count
    assert len(set(table[b, j].item() for b in range(B) for j in range(P // ps, held[b]))) == sum(held.tolist()) - B * (P // ps)


def test_attention_agrees_with_the_engines_reference():
    a = build_cache([(0, [(700, 1), (33, 1)])], 64, 40, 8, device="cuda", poison=False)
    out, _ = run({**a, "group_start": None, "prefix_len": None})
    want = paged_attention_reference(a["q"], a["k_cache"], a["v_cache"], a["table"], a["lens"], a["q_start"], 64, 1 / math.sqrt(128))
    # both round their result to bf16, and the kernel's probabilities are bf16 too
    assert ((out.float() - want.float()).norm() / want.float().norm()).item() < 3 * 2.0 ** -8


def test_refusals():
    a = build_cache([(20, [(25, 2), (21, 1)])], 16, 8, 2, device="cuda")
    bad = [dict(q=a["q"].float()), dict(q=a["q"][:, :7]), dict(q=a["q"][..., :64]), dict(q=a["q"].cpu().cuda()[:, ::2]),
           dict(k_cache=a["k_cache"][:, :1]), dict(v_cache=a["v_cache"].half()), dict(k_cache=a["k_cache"].cpu()),
           dict(table=a["table"].long()), dict(table=a["table"][:1]), dict(table=a["table"].t().contiguous().t()),
           dict(lens=a["lens"].long()), dict(q_start=a["q_start"][1:]), dict(page_size=12), dict(page_size=0), dict(max_q=0), dict(scale=0.0), dict(scale=-1.0),
           dict(group_start=None), dict(prefix_len=None), dict(prefix_len=_i([1, 2])),
           dict(group_start=_i([0, 1, 2, 3, 3]), prefix_len=_i([0] * 4)),
           dict(out=torch.empty(3, 8, 128, device="cuda")), dict(out=torch.empty(2, 8, 128, dtype=torch.bfloat16, device="cuda"))]
    for b in bad:
        with pytest.raises(RuntimeError):
            paged.prefix_attention(**{**dict(max_q=2), **a, **b})
    many = build_cache([(0, [(1, 1)] * 513)], 8, 1, 1, device="cuda")
    with pytest.raises(RuntimeError):
        paged.prefix_attention(**many)


def test_no_rows_and_no_sequences():
    a = build_cache([(0, [(9, 0), (0, 0)])], 16, 8, 2, device="cuda")
    assert run(a)[0].shape == (0, 8, 128)
    none = dict(a, table=a["table"][:0], lens=a["lens"][:0], q_start=a["q_start"][:1], group_start=None, prefix_len=None)
    assert run(none)[0].shape == (0, 8, 128)


def test_kv_append_skips_slots_outside_the_cache():
    from kore_b200.ops import native
    kc, vc = (torch.zeros(32, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    k, v = (torch.ones(4, 2, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    native().kv_append(k, v, _i([-1, 5, 32, 31]), kc, vc)
    for c in (kc, vc):
        assert (c[[5, 31]] == 1).all() and c.sum() == 2 * 2 * 128


def test_attention_oracle_and_cpu_definition_agree():
    a = build_cache([(20, [(25, 2), (21, 1)])], 16, 8, 2)
    out, lse = paged.prefix_attention(**a, max_q=2, want_lse=True)
    check_attention(out, lse, a)
    assert attention_oracle(a)[0].shape == out.shape
