"""Inputs and 64-bit definitions for the tests of the paged plan, shared-prefix
attention and draft verification. Plain loops over sequences; nothing here uses the package."""
import math

import torch


def plan_oracle(ctx, new, table, ps, rows, held=None, free=None, count=None):
    table = [list(r) for r in table]
    M = len(table[0]) if table else 0
    count = min(max(count, 0), len(free)) if free is not None else 0
    out = dict(q_start=[0], lens=[], pos=[], slots=[], ok=[], held=[])
    asked = got = 0
    for b in range(len(table)):
        c, n = max(ctx[b], 0), max(new[b], 0)
        n = min(n, rows - out["q_start"][-1])
        need = (c + n + ps - 1) // ps
        h = (c + ps - 1) // ps if held is None else min(max(held[b], 0), M)
        take = max(0, need - h) if free is not None and need <= M else 0
        ok = need <= M and (free is None or asked + take <= count)
        if ok:
            for j in range(take):
                table[b][h + j] = free[count - 1 - asked - j]
            got += take
        asked += take
        out["q_start"].append(out["q_start"][-1] + n)
        out["lens"].append(c + n if ok else c)
        out["ok"].append(ok)
        out["held"].append(h + take if ok else h)
        out["pos"] += list(range(c, c + n))
        out["slots"] += [table[b][p // ps] * ps + p % ps if ok and table[b][p // ps] >= 0 else -1 for p in range(c, c + n)]
    pad = rows - out["q_start"][-1]
    out["pos"] += [0] * pad
    out["slots"] += [-1] * pad
    return dict(out, table=table, free_count=None if free is None else count - got)


def build_cache(groups, ps, hq, hkv, *, seed=0, device="cpu", poison=True, pad_rows=0, extra_cols=2, q_pad=0, D=128,
                dtype=torch.bfloat16):
    """``groups``: [(prefix, [(len, q_len), ...])]. Sequences of a group share the whole
    pages of the prefix and hold a copy of the part-filled one. With ``poison`` every
    slot that no sequence owns a token in is NaN, and unused table entries point nowhere."""
    g = torch.Generator().manual_seed(seed)
    seqs = [(gi, n, m) for gi, (_, s) in enumerate(groups) for n, m in s]
    need, tables = 0, []
    for prefix, s in groups:
        common = None
        for n, _ in s:
            pages = -(-max(n, prefix if common is None else 0) // ps)    # a group's first table covers the prefix
            keep = 0 if common is None else min(prefix // ps, pages)
            row = ([] if common is None else common[:keep]) + list(range(need, need + pages - keep))
            need += pages - keep
            if common is None:
                common = row
            tables.append(row)
    total = need + 1
    perm = torch.randperm(total, generator=g)
    M = max([len(t) for t in tables] + [1]) + extra_cols
    junk = 10 ** 6 if poison else 0
    table = torch.tensor([[int(perm[p]) for p in t] + [junk if i % 2 else (-1 if poison else 0) for i in range(M - len(t))]
                          for t in tables], dtype=torch.int32).reshape(len(tables), M)
    kc = torch.full((total * ps, hkv, D), math.nan if poison else 0.0, dtype=torch.float32)
    vc = kc.clone()

    def put(row, lo, hi, k, v):
        at = torch.arange(lo, hi)
        slot = table[row].long()[at // ps] * ps + at % ps
        kc[slot], vc[slot] = k, v

    b = 0
    for prefix, s in groups:
        pk, pv = (torch.randn(prefix, hkv, D, generator=g) for _ in range(2))
        for i, (n, _) in enumerate(s):
            own = max(0, n - prefix)
            hold = prefix if i == 0 else min(prefix, n)
            put(b, 0, hold, pk[:hold], pv[:hold])
            put(b, prefix, prefix + own, torch.randn(own, hkv, D, generator=g), torch.randn(own, hkv, D, generator=g))
            b += 1
    q_start = [0]
    for _, _, m in seqs:
        q_start.append(q_start[-1] + m)
    q = torch.randn(q_start[-1] + pad_rows, hq * D + q_pad, generator=g) * 1.5
    i32 = dict(dtype=torch.int32, device=device)
    starts = [0]
    for _, s in groups:
        starts.append(starts[-1] + len(s))
    q = q.to(dtype).to(device)
    return dict(q=q[:, :hq * D].unflatten(1, (hq, D)), k_cache=kc.to(dtype).to(device), v_cache=vc.to(dtype).to(device),
                table=table.to(device), lens=torch.tensor([n for _, n, _ in seqs], **i32),
                q_start=torch.tensor(q_start, **i32), page_size=ps,
                group_start=torch.tensor(starts, **i32), prefix_len=torch.tensor([p for p, _ in groups], **i32))


def attention_oracle(a):
    """(out, lse, tolerance of out, tolerance of lse) in 64 bits from the arguments of prefix_attention.

    Tolerances: an output is rounded to bf16 (at most 2^-8 of it), and so is each
    probability before its product (2^-8 of sum p |v|). A score is an fp32 sum of
    128 exact products: off by at most 128 * 2^-23 of the sum of their
    magnitudes, which moves probabilities by twice that (numerator and sum); 2^-18
    covers exp2, the running sums and the join of the parts."""
    ps, q = a["page_size"], a["q"].double().cpu()
    kc, vc = a["k_cache"].double().cpu(), a["v_cache"].double().cpu()
    table, lens, qs = a["table"].cpu().long(), a["lens"].tolist(), a["q_start"].tolist()
    hq, hkv, D = q.shape[1], kc.shape[1], q.shape[2]
    B = len(lens)
    lead, shared = list(range(B)), [0] * B
    if a.get("group_start") is not None:
        gs = a["group_start"].tolist()
        for g, n in enumerate(a["prefix_len"].tolist()):
            for b in range(gs[g], gs[g + 1]):
                lead[b], shared[b] = gs[g], n
    T = q.shape[0]
    out, lse = torch.zeros(T, hq, D, dtype=torch.float64), torch.full((T, hq), -math.inf, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    scale = a.get("scale") or 1.0 / math.sqrt(D)
    for b in range(B):
        m = qs[b + 1] - qs[b]
        for i in range(m):
            n = lens[b] - m + i + 1
            if n <= 0:
                continue
            at = torch.arange(n)
            page = torch.where(at < shared[b], table[lead[b]][at // ps], table[b][at // ps])
            slot = page * ps + at % ps
            k, v = (c[slot].repeat_interleave(hq // hkv, 1).transpose(0, 1) for c in (kc, vc))     # [hq, n, D]
            x = q[qs[b] + i]
            z = torch.einsum("hd,hnd->hn", x, k) * scale
            mag = (torch.einsum("hd,hnd->hn", x.abs(), k.abs()) * scale).amax(-1)
            t = qs[b] + i
            lse[t] = torch.logsumexp(z, -1)
            p = torch.softmax(z, -1)
            out[t] = torch.einsum("hn,hnd->hd", p, v)
            A = torch.einsum("hn,hnd->hd", p, v.abs())
            ds = 128 * 2.0 ** -23 * mag + 2.0 ** -18
            tol[t] = 2.0 ** -8 * (out[t].abs() + A) + 2 * ds[:, None] * A
            ltol[t] = ds + 2.0 ** -21 * lse[t].abs()
    return out, lse, tol, ltol


def check_attention(got, lse, a):
    want, wl, tol, ltol = attention_oracle(a)
    n = int(a["q_start"][-1])
    d = (got.double().cpu() - want).abs()[:n]
    assert torch.isfinite(got[:n]).all()
    assert (d <= tol[:n]).all(), float((d - tol[:n]).max())
    if lse is not None:
        lse = lse.double().cpu()[:n]
        empty = wl[:n].isneginf()
        assert (lse.isneginf() == empty).all()
        e = (lse - wl[:n]).abs()[~empty]
        assert (e <= ltol[:n][~empty]).all(), float((e - ltol[:n][~empty]).max())


def verify_oracle(logits, tokens, q_start, u, tau, probs=None):
    """(accepted, next, logp) from the definition in 64 bits, token by token."""
    z, T, V = logits.double().cpu(), logits.shape[0], logits.shape[1]
    logp = torch.zeros(T, dtype=torch.float64)
    acc, nxt = [], []
    for a, b in zip(q_start[:-1], q_start[1:]):
        t, y = a, -1
        while t < b:
            row = z[t] / (tau or 1.0)
            if torch.isnan(row).any() or row.max() == math.inf or row.max() == -math.inf:
                logp[t] = math.nan
                break
            e = torch.exp(row - row.max())
            p, total = e / e.sum(), e.sum()
            lp = row - row.max() - torch.log(total)
            drafted = t + 1 < b
            x = int(tokens[t + 1]) if drafted else -1
            if drafted and 0 <= x < V:
                good = x == int(row.argmax()) if tau == 0 else float(u[t, 0]) * (1.0 if probs is None else float(probs[t, x])) < float(p[x])
                if good:
                    logp[t] = lp[x]
                    t += 1
                    continue
            if tau == 0:
                y = int(row.argmax())
            else:
                w = p.clone()
                if drafted and probs is not None:
                    w = (p - probs[t].double().cpu()).clamp_min(0)
                elif 0 <= x < V:
                    w[x] = 0
                if float(w.sum()) <= 0:
                    w = p
                c = torch.cumsum(w, 0)
                past = (c > float(u[t, 1]) * c[-1]).nonzero()
                y = int(past[0]) if len(past) else int(w.nonzero()[-1])
            logp[t] = lp[y]
            break
        acc.append(t - a)
        nxt.append(y)
    return acc, nxt, logp
