"""The operators of a drafted decode step that this file times: the plan of a
step (block tables and slot maps from request lengths), attention for batches
whose sequences share a prefix, and the verification of drafted tokens.

``run`` computes them in plain form (torch operations, fp32; fp64 where a
rounding could move a token or a border) or, with ``own``, through
``kore_b200.ops``. ``exact`` gives the same outputs in 64 bits.
"""
import math
import random

import torch

own = False

DEV = "cuda"
D = 128              # head size of the models here


# --------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step of a 14B GRPO batch: one new token a sequence, every 64th of them needs a page
        dict(name="plan_decode", op="plan", B=64, new=1, ragged=False, ctx=7936, ps=64, spare=0, short=False),
        # a step of drafted tokens, one to eight a sequence, some pages held ahead
        dict(name="plan_drafts", op="plan", B=512, new=8, ragged=True, ctx=8192, ps=16, spare=2, short=False),
        # packed prefill of a whole rollout batch: ragged prompts, all pages new, the pool runs short for the last ones
        dict(name="plan_prefill", op="plan", B=256, new=4096, ragged=True, ctx=0, ps=64, spare=0, short=True),
        # a handful of samples of one short prompt: launch latency
        dict(name="share_small", op="share", groups=1, per=4, hq=40, hkv=8, P=200, S=60, k=0, ps=64),
        # the 14B GRPO decode step of one layer: 8 prompts x 8 samples, 1024-token prompts, transcripts of up to 7936 tokens
        dict(name="share_grpo_14b", op="share", groups=8, per=8, hq=40, hkv=8, P=1024, S=6912, k=0, ps=64),
        # samples of one long context (a repository in the prompt), heads of the MoE model
        dict(name="share_long_moe", op="share", groups=1, per=32, hq=32, hkv=4, P=32768, S=1500, k=0, ps=64),
        # drafted step: five query tokens a sequence, ragged prompts that end inside a page
        dict(name="share_draft", op="share", groups=5, per=13, hq=40, hkv=8, P=6011, S=2047, k=4, ps=32),
        # many samples of one prompt: the shared part is bound by its products
        dict(name="share_wide", op="share", groups=1, per=256, hq=40, hkv=8, P=16384, S=1024, k=0, ps=64),
        # one sequence's drafts on a small vocabulary: launch latency
        dict(name="verify_1", op="verify", B=1, k=3, V=32000, tau=1.0, probs=False, dtype="bf16"),
        # a drafted step of the 14B batch, drafts by look-up (no probabilities of their own), sampling temperature
        dict(name="verify_14b", op="verify", B=64, k=4, V=151936, tau=0.9, probs=False, dtype="bf16"),
        # the same with a draft model's probabilities
        dict(name="verify_probs", op="verify", B=48, k=7, V=151936, tau=1.0, probs=True, dtype="bf16"),
        # greedy decoding with one draft a sequence, fp32 logits, odd vocabulary
        dict(name="verify_greedy", op="verify", B=200, k=1, V=50257, tau=0.0, probs=False, dtype="fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["plan", "share", "share", "share", "verify", "verify"])
    if op == "plan":
        return dict(op=op, B=_log(rng, 1, 1024), new=_log(rng, 1, 1024), ragged=rng.random() < 0.7,
                    ctx=rng.choice([0, _log(rng, 1, 32768)]), ps=rng.choice([16, 32, 64, 128]),
                    spare=rng.choice([0, 0, 3]), short=rng.random() < 0.3)
    if op == "share":
        hq, hkv = rng.choice([(40, 8), (32, 4), (16, 8), (8, 8), (6, 2), (12, 1), (64, 4)])
        c = dict(op=op, groups=_log(rng, 1, 16), per=_log(rng, 1, 64), hq=hq, hkv=hkv, P=_log(rng, 1, 32768),
                 S=_log(rng, 8, 4096), k=rng.choice([0, 0, 0, 1, 3, 7]), ps=rng.choice([16, 32, 64, 128]))
        while c["groups"] * c["per"] > 256:
            c["groups"] = max(1, c["groups"] // 2)
        rows = c["groups"] * c["per"] * (c["k"] + 1)
        while rows * hq * (c["P"] + c["S"]) > 1.2e8 or (c["groups"] * c["P"] + rows * c["S"]) * hkv > 6e6:
            if c["P"] > c["S"]:
                c["P"] = max(1, c["P"] // 2)
            else:
                c["S"] = max(8, c["S"] // 2)
        return c
    V, k = _log(rng, 1000, 151936), rng.choice([0, 1, 2, 4, 7, 15])
    return dict(op=op, B=max(1, min(_log(rng, 1, 256), int(5e7 // (V * (k + 1))))), k=k, V=V, tau=rng.choice([1.0, 0.9, 0.6, 1.3, 0.0]),
                probs=rng.random() < 0.4, dtype=rng.choice(["bf16", "bf16", "fp32"]))


def _lengths(case):
    """The case's lengths, in the order that a seed then changes."""
    r = random.Random(repr(sorted((a, b) for a, b in case.items() if a != "name")))
    if case["op"] == "plan":
        B = case["B"]
        new = [r.randint(0 if case["ctx"] else 1, case["new"]) if case["ragged"] else case["new"] for _ in range(B)]
        return dict(new=new, ctx=[r.randint(max(1, case["ctx"] // 2), case["ctx"]) if case["ctx"] else 0 for _ in range(B)])
    if case["op"] == "share":
        G, B, n = case["groups"], case["groups"] * case["per"], case["k"] + 1
        return dict(P=[case["P"]] + [r.randint(max(1, case["P"] // 2), case["P"]) for _ in range(G - 1)],
                    S=[max(n, case["S"])] + [max(n, _log(r, max(1, case["S"] // 16), case["S"])) for _ in range(B - 1)],
                    n=[n] + [r.randint(1, n) for _ in range(B - 1)])
    return dict(n=[case["k"] + 1] + [r.randint(max(1, case["k"] - 2), case["k"] + 1) for _ in range(case["B"] - 1)])


# -------------------------------------------------------------------- inputs
def _int(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _starts(n):
    out = [0]
    for v in n:
        out.append(out[-1] + v)
    return out


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed) * 1013 + 11)
    r = random.Random(seed * 7 + 1)
    s, L = dict(case=dict(case)), _lengths(case)
    for v in L.values():
        r.shuffle(v)
    if case["op"] == "plan":
        B, ps = case["B"], case["ps"]
        M = -(-(case["ctx"] + case["new"]) // ps) + case["spare"] + 1
        held = [-(-c // ps) + r.randint(0, case["spare"]) for c in L["ctx"]]
        want = sum(max(0, -(-(c + n) // ps) - h) for c, n, h in zip(L["ctx"], L["new"], held))
        pool = max(1, want - want // 8) if case["short"] else want + 5
        pages = torch.randperm(B * M + pool, generator=g, device=DEV).int()
        s.update(ctx=_int(L["ctx"]), new=_int(L["new"]), held=_int(held), table=pages[:B * M].view(B, M).contiguous(),
                 free=pages[B * M:].contiguous(), count=_int([pool]), rows=sum(L["new"]))
        return s
    if case["op"] == "share":
        G, per, ps, hq, hkv = case["groups"], case["per"], case["ps"], case["hq"], case["hkv"]
        shared = [p // ps for p in L["P"]]                       # whole pages that a group's sequences share
        lens = [L["P"][b // per] + L["S"][b] for b in range(G * per)]
        M = max(-(-n // ps) for n in lens)
        total = sum(shared) + sum(-(-n // ps) - shared[b // per] for b, n in enumerate(lens))
        ids = list(range(total))
        r.shuffle(ids)
        table, tail, at = [], [], 0
        for b, n in enumerate(lens):
            grp = b // per
            if b % per == 0:
                common = ids[at:at + shared[grp]]
                at += shared[grp]
            mine = ids[at:at + -(-n // ps) - shared[grp]]
            at += len(mine)
            table.append(common + mine + [0] * (M - len(common) - len(mine)))
            if b % per and L["P"][grp] % ps:                     # the prompt's last, part-filled page is copied to each sample
                tail.append((table[b - b % per][shared[grp]], mine[0]))
        kc, vc = (torch.empty(total * ps, hkv, D, device=DEV, dtype=torch.bfloat16).normal_(0.0, 1.0, generator=g) for _ in range(2))
        if tail:
            a, b = torch.tensor(tail, device=DEV).T
            for c in (kc, vc):
                c.view(total, -1)[b] = c.view(total, -1)[a]
        q = torch.randn(sum(L["n"]), hq, D, generator=g, device=DEV) * 1.5
        s.update(q=q.bfloat16(), kc=kc, vc=vc, table=_int(table), lens=_int(lens), q_start=_int(_starts(L["n"])),
                 group_start=_int(list(range(0, G * per + 1, per))), prefix=_int(L["P"]),
                 longest=max(n - L["P"][b // per] for b, n in enumerate(lens)))
        return s
    V, T, q_start = case["V"], sum(L["n"]), _starts(L["n"])
    z = 2.0 * torch.randn(T, V, generator=g, device=DEV)
    top = torch.randint(0, V, (T, 1), generator=g, device=DEV)
    z.scatter_add_(1, top, 4.0 + 12.0 * torch.rand(T, 1, generator=g, device=DEV))       # from unsure to certain
    s.update(logits=z.to(torch.bfloat16 if case["dtype"] == "bf16" else torch.float32), q_start=_int(q_start),
             u=torch.rand(T, 2, generator=g, device=DEV), most=max(L["n"]))
    if case["probs"]:
        z = z.add_(torch.randn(T, V, generator=g, device=DEV), alpha=0.5)                # a draft model that mostly agrees
        s["probs"] = torch.softmax(z, -1)
        pick = torch.multinomial(s["probs"], 1, generator=g) if V < 1 << 24 else top
    else:
        pick = torch.where(torch.rand(T, 1, generator=g, device=DEV) < 0.85, top, torch.randint(0, V, (T, 1), generator=g, device=DEV))
    s["tokens"] = torch.cat([top[:1, 0], pick[:-1, 0]])          # row t's draft is fed in row t + 1
    return s


# ---------------------------------------------------------------- plain forms
def _plain_plan(s):
    ps, ctx, new, held, table = s["case"]["ps"], s["ctx"].long(), s["new"].long(), s["held"].long(), s["table"]
    B, M = table.shape
    end = torch.cumsum(new, 0)
    need = (ctx + new + ps - 1) // ps
    fits = need <= M
    take = torch.where(fits, (need - held).clamp_min(0), torch.zeros_like(need))
    C = torch.cumsum(take, 0)
    ok = fits & (C <= s["count"])
    col = torch.arange(M, device=DEV)[None]
    fresh = ok[:, None] & (col >= held[:, None]) & (col < need[:, None])
    at = s["count"] - 1 - (C - take)[:, None] - (col - held[:, None])
    table = torch.where(fresh, s["free"][at.clamp(0, s["free"].numel() - 1)], table)
    row = torch.arange(s["rows"], device=DEV)
    b = torch.searchsorted(end, row, right=True)
    pos = ctx[b] + row - (end - new)[b]
    page = table[b, (pos // ps).clamp_max(M - 1)].long()
    slots = torch.where(ok[b], page * ps + pos % ps, torch.full_like(pos, -1))
    got = torch.where(ok, take, torch.zeros_like(take))
    return dict(q_start=torch.cat([end.new_zeros(1), end]).int(), lens=torch.where(ok, ctx + new, ctx).int(), pos=pos.int(),
                slots=slots.int(), ok=ok, held=(held + got).int(), table=table, free_count=(s["count"] - got.sum()).int())


def _part(q, k, v, live):
    """Softmax attention over one part of the keys: q [n, r, hkv, g, D], k / v [n, p, hkv, D], live [n, r, p] -> max, sum, sum of p v."""
    z = torch.einsum("nrhgd,nphd->nrhgp", q, k) * (1.0 / math.sqrt(D))
    z = torch.where(live[:, :, None, None], z, torch.full_like(z, -math.inf))
    m = z.amax(-1)
    e = torch.exp(z - torch.where(m.isinf(), torch.zeros_like(m), m)[..., None])
    return m, e.sum(-1), torch.einsum("nrhgp,nphd->nrhgd", e, v)


def _plain_share(s):
    c, ps = s["case"], s["case"]["ps"]
    q, table, hkv, g = s["q"].float(), s["table"].long(), c["hkv"], c["hq"] // c["hkv"]
    T, starts, lens = q.shape[0], s["q_start"].long(), s["lens"].long()
    q = q.view(T, hkv, g, D)
    gs, P, n = s["group_start"].long(), s["prefix"].long(), starts[1:] - starts[:-1]
    row = torch.arange(T, device=DEV)
    seq = torch.searchsorted(starts[1:], row, right=True)
    grp_of = torch.searchsorted(gs[1:], torch.arange(lens.numel(), device=DEV), right=True)

    def keys(first, offset, count):                              # slots of `count` positions from `offset` of the sequences `first`
        at = offset[:, None] + torch.arange(count, device=DEV)[None]
        page = table[first[:, None], (at // ps).clamp_max(table.shape[1] - 1)]
        return at, (page * ps + at % ps)

    # the prefix: a group's rows against one copy of the keys
    g0, g1 = starts[gs[:-1]], starts[gs[1:]]
    R = c["per"] * (c["k"] + 1)
    rows = (g0[:, None] + torch.arange(R, device=DEV)[None])
    at, slots = keys(gs[:-1], torch.zeros_like(P), c["P"])
    live = (at < P[:, None])[:, None].expand(-1, R, -1)
    m1, l1, o1 = _part(q[rows.clamp_max(T - 1)], s["kc"][slots].float(), s["vc"][slots].float(), live)
    grp = grp_of[seq]
    back = row - g0[grp]
    m1, l1, o1 = m1[grp, back], l1[grp, back], o1[grp, back]
    # each sequence's own keys
    R = c["k"] + 1
    rows = starts[:-1, None] + torch.arange(R, device=DEV)[None]
    at, slots = keys(torch.arange(lens.numel(), device=DEV), P[grp_of], s["longest"])
    seen = (lens - n)[:, None] + torch.arange(R, device=DEV)[None]        # a row's own position
    live = (at[:, None] <= seen[:, :, None]) & (at < lens[:, None])[:, None]
    m2, l2, o2 = _part(q[rows.clamp_max(T - 1)], s["kc"][slots].float(), s["vc"][slots].float(), live)
    back = row - starts[seq]
    m2, l2, o2 = m2[seq, back], l2[seq, back], o2[seq, back]
    m = torch.maximum(m1, m2)
    a, b = torch.exp(m1 - m), torch.exp(m2 - m)
    total = l1 * a + l2 * b
    o = (o1 * a[..., None] + o2 * b[..., None]) / total[..., None]
    return dict(o=o.reshape(T, c["hq"], D).bfloat16(), lse=(m + torch.log(total)).reshape(T, c["hq"]))


def _plain_verify(s):
    c, tau, x = s["case"], s["case"]["tau"], s["tokens"]
    starts = s["q_start"].long()
    z = s["logits"].double()
    T, B, V = z.shape[0], starts.numel() - 1, z.shape[1]
    row = torch.arange(T, device=DEV)
    seq = torch.searchsorted(starts[1:], row, right=True)
    first, last = starts[:-1], starts[1:] - 1
    if tau > 0:
        z = z / tau
    e = torch.exp(z - z.amax(-1, keepdim=True))
    p = e / e.sum(-1, keepdim=True)
    draft = torch.cat([x[1:], x[:1]])                            # the token that row t's logits are about
    drafted = row < last[seq]
    if tau > 0:
        px = p.gather(1, draft[:, None])[:, 0]
        qx = s["probs"].gather(1, draft[:, None])[:, 0].double() if c["probs"] else torch.ones_like(px)
        good = drafted & (s["u"][:, 0].double() * qx < px)
    else:
        best = (z == z.amax(-1, keepdim=True)).int().argmax(-1)
        good = drafted & (draft == best)
    bad = torch.cumsum((~good).int(), 0)                         # accepted: no bad row from the sequence's first to this one
    upto = bad - torch.where(first > 0, bad[(first - 1).clamp_min(0)], torch.zeros_like(first))[seq]
    taken = good & (upto == 0)
    accepted = torch.zeros(B, dtype=torch.int64, device=DEV).scatter_add_(0, seq, taken.long())
    end = first + accepted                                       # the row that gives the next token
    if tau > 0:
        w = p[end]
        over = drafted[end][:, None]
        if c["probs"]:
            rest = (w - s["probs"][end].double()).clamp_min(0)
        else:
            rest = torch.where(torch.arange(V, device=DEV)[None] == draft[end][:, None], torch.zeros_like(w), w)
        w = torch.where(over & (rest.sum(-1, keepdim=True) > 0), rest, w)
        C = torch.cumsum(w, -1)
        nxt = (C > s["u"][end, 1:2].double() * C[:, -1:]).int().argmax(-1)
    else:
        nxt = best[end]
    logp = torch.log(p.gather(1, torch.where(taken, draft, torch.zeros_like(draft))[:, None])[:, 0])
    logp = torch.where(taken, logp, torch.zeros_like(logp))
    logp[end] = torch.log(p[end, nxt])
    return dict(accepted=accepted.int(), next=nxt, logp=logp.float())


# ------------------------------------------------------ through the framework
def _own(s):
    from kore_b200.ops import paged, spec
    c = s["case"]
    if c["op"] == "plan":
        p = paged.plan(s["ctx"], s["new"], s["table"], c["ps"], s["rows"], held=s["held"], free=s["free"], free_count=s["count"])
        return dict(q_start=p.q_start, lens=p.lens, pos=p.pos, slots=p.slots, ok=p.ok, held=p.held, table=s["table"],
                    free_count=p.free_count)
    if c["op"] == "share":
        o, lse = paged.prefix_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["q_start"], c["ps"], max_q=c["k"] + 1,
                                        group_start=s["group_start"], prefix_len=s["prefix"], want_lse=True)
        return dict(o=o, lse=lse)
    v = spec.verify(s["logits"], s["tokens"], s["q_start"], s["u"], c["tau"], draft_probs=s.get("probs"))
    return dict(accepted=v.accepted, next=v.next, logp=v.logp)


def run(state):
    with torch.no_grad():
        if own:
            return _own(state)
        return {"plan": _plain_plan, "share": _plain_share, "verify": _plain_verify}[state["case"]["op"]](state)


# ---------------------------------------------------------------------- work
def work(case):
    L = _lengths(case)
    if case["op"] == "plan":
        ps, B, T = case["ps"], case["B"], sum(L["new"])
        fresh = sum(max(0, -(-(c + n) // ps) - -(-c // ps)) for c, n in zip(L["ctx"], L["new"]))
        touched = sum(-(-(c + n) // ps) - c // ps for c, n in zip(L["ctx"], L["new"]) if n)
        # a row's position and slot out; lengths, new tokens and held pages in; starts, lengths, held and ok out; pages from the pool into the table, old ones read
        return dict(bytes=8 * T + 12 * B + 13 * B + 8 * fresh + 4 * (touched - fresh) + 8, flops=4 * T + 10 * B)
    if case["op"] == "share":
        per, hq, hkv, T = case["per"], case["hq"], case["hkv"], sum(L["n"])
        kv = sum(L["P"]) + sum(L["S"])
        pairs = sum(n * (L["P"][b // per] + S) - n * (n - 1) // 2 for b, (n, S) in enumerate(zip(L["n"], L["S"])))
        return dict(bytes=4 * D * hkv * kv + 4 * D * hq * T + 4 * hq * T, flops=4 * D * hq * pairs)
    T, V, B = sum(L["n"]), case["V"], case["B"]
    size = 2 if case["dtype"] == "bf16" else 4
    # every logit once, the draft's probabilities of the row that gives the next token
    return dict(bytes=T * V * size + (4 * B * V if case["probs"] and case["tau"] > 0 else 0) + 20 * T + 12 * B, flops=4 * T * V)


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """The outputs of ``run`` for these inputs from the definitions in 64 bits."""
    s, f8 = prepare(case, seed), torch.float64
    if case["op"] == "plan":
        ps, table, count, T = case["ps"], s["table"].tolist(), int(s["count"]), s["rows"]
        M, free, asked, got = len(table[0]), s["free"].tolist(), 0, 0
        out = dict(q_start=[0], lens=[], pos=[], slots=[], ok=[], held=[])
        for b, (c, n, h) in enumerate(zip(s["ctx"].tolist(), s["new"].tolist(), s["held"].tolist())):
            need = (c + n + ps - 1) // ps
            take = max(0, need - h) if need <= M else 0
            ok = need <= M and asked + take <= count
            for j in range(take if ok else 0):
                table[b][h + j] = free[count - 1 - asked - j]
            asked += take
            got += take if ok else 0
            out["q_start"].append(out["q_start"][-1] + n)
            out["lens"].append(c + n if ok else c)
            out["held"].append(h + take if ok else h)
            out["ok"].append(ok)
            out["pos"] += range(c, c + n)
            out["slots"] += [table[b][p // ps] * ps + p % ps if ok else -1 for p in range(c, c + n)]
        out = {k: torch.tensor(v, dtype=torch.bool if k == "ok" else torch.int32, device=DEV) for k, v in out.items()}
        return dict(out, table=_int(table), free_count=_int([count - got]))
    if case["op"] == "share":
        ps, rep = case["ps"], case["hq"] // case["hkv"]
        o, lse = [], []
        starts = s["q_start"].tolist()
        for b, n in enumerate(s["lens"].tolist()):
            at = torch.arange(n, device=DEV)
            slot = s["table"][b].long()[at // ps] * ps + at % ps
            k, v = (c[slot].to(f8).transpose(0, 1) for c in (s["kc"], s["vc"]))                  # [hkv, n, D]
            q = s["q"][starts[b]:starts[b + 1]].to(f8)
            m = q.shape[0]
            q = q.view(m, case["hkv"], rep, D).permute(1, 0, 2, 3).reshape(case["hkv"], m * rep, D)
            z = (q @ k.transpose(1, 2)).div_(math.sqrt(D)).view(case["hkv"], m, rep, n)
            hidden = at[None] > (n - m + torch.arange(m, device=DEV))[:, None]
            z.masked_fill_(hidden[None, :, None], -math.inf)
            lse.append(torch.logsumexp(z, -1).permute(1, 0, 2).reshape(m, -1))
            w = torch.softmax(z, -1).view(case["hkv"], m * rep, n) @ v
            o.append(w.view(case["hkv"], m, rep, D).permute(1, 0, 2, 3).reshape(m, -1, D))
        return dict(o=torch.cat(o), lse=torch.cat(lse))
    x, tau, V = s["tokens"].tolist(), case["tau"], case["V"]
    starts, u = s["q_start"].tolist(), s["u"].to(f8).tolist()
    logp = torch.zeros(s["logits"].shape[0], dtype=f8, device=DEV)
    accepted, nxt = [], []
    for a, b in zip(starts[:-1], starts[1:]):
        lp = torch.log_softmax(s["logits"][a:b].to(f8) / (tau if tau > 0 else 1.0), -1)
        t = a
        while t < b - 1:
            y, l = x[t + 1], lp[t - a]
            q = float(s["probs"][t, y]) if case["probs"] else 1.0
            if not (u[t][0] * q < math.exp(float(l[y])) if tau > 0 else y == int(s["logits"][t].argmax())):
                break
            logp[t] = l[y]
            t += 1
        w = lp[t - a].exp()
        if t < b - 1 and tau > 0:
            rest = (w - s["probs"][t].to(f8)).clamp_min(0) if case["probs"] else w.clone()
            if not case["probs"]:
                rest[x[t + 1]] = 0
            w = rest if float(rest.sum()) > 0 else w
        C = torch.cumsum(w, 0)
        y = int(torch.searchsorted(C, u[t][1] * C[-1:], right=True).clamp_max(V - 1)) if tau > 0 else int(s["logits"][t].argmax())
        accepted.append(t - a)
        nxt.append(y)
        logp[t] = lp[t - a, y]
    return dict(accepted=_int(accepted), next=torch.tensor(nxt, device=DEV), logp=logp)
