"""The operators of a training step that this file times: the head's loss in
pieces of the vocabulary, the embedding with its sorted gradient, the router's
balance loss, and activation checkpoints in 8 bits.

``run`` computes them in plain form (fp32 torch operations) or, with ``own``,
through ``kore_b200.ops``. ``exact`` gives the same outputs in 64 bits.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 128          # columns that share one scale of an 8-bit checkpoint
TINY = 1e-30         # blocks whose largest magnitude is below this are held as zero


# --------------------------------------------------------------------- cases
def listed():
    return [
        # scoring one token with the tiny preset's head: launch latency
        dict(name="head_score_1", op="head", train=False, T=1, V=32000, H=256, tau=1.0),
        # log-probs, entropy and logsumexp of a packed rollout chunk, 14B head, ragged length, sampling temperature
        dict(name="head_score_14b", op="head", train=False, T=1003, V=151936, H=5120, tau=0.7),
        # a short micro-batch of the MoE model's head, forward and gradients
        dict(name="head_train_moe", op="head", train=True, T=1500, V=151936, H=2048, tau=1.0),
        # one 8192-token sequence of the 14B SFT step: forward and gradients
        dict(name="head_train_14b", op="head", train=True, T=8192, V=151936, H=5120, tau=1.0),
        # the tiny preset's embedding on a ragged batch, fp32 gradient buffer, scaled lookup, added to an existing gradient (tied head)
        dict(name="embed_tiny_tied", op="embed", T=129, V=32000, H=256, scale=16.0, grad="fp32", add=True),
        # a packed micro-batch of the 14B model: lookup and gradient of the whole table
        dict(name="embed_14b", op="embed", T=16384, V=151936, H=5120, scale=1.0, grad="bf16", add=False),
        # a decode-sized router batch with few experts
        dict(name="balance_small", op="balance", T=64, E=8, k=2, masked=0.0),
        # one layer's router over a packed 32k-token micro-batch, 128 experts, padding masked out
        dict(name="balance_moe", op="balance", T=32768, E=128, k=8, masked=0.125),
        # RMSNorm with the layer input kept in 8 bits: a handful of tokens
        dict(name="act8_norm_small", op="act8_norm", T=37, H=256, pad=0),
        # the same at a 14B layer over a packed micro-batch
        dict(name="act8_norm_14b", op="act8_norm", T=16384, H=5120, pad=0),
        # the 14B layer's gate|up kept in 8 bits: SwiGLU forward, and its backward from the 8-bit copy
        dict(name="act8_swiglu_14b", op="act8_swiglu", T=8192, H=17408, pad=0),
        # a strided block (the value columns' neighbours of a qkv buffer) held in 8 bits and read back, ragged length
        dict(name="act8_hold_qkv", op="act8_hold", T=5003, H=6144, pad=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["head", "head", "embed", "balance", "act8_norm", "act8_swiglu", "act8_hold"])
    if op == "head":
        T, V, H = _log(rng, 1, 8192), _log(rng, 1000, 151936), 8 * _log(rng, 8, 640)
        return dict(op=op, train=rng.random() < 0.6, T=T, V=V, H=H, tau=rng.choice([1.0, 0.7, 1.3]))
    if op == "embed":
        T, V, H = _log(rng, 1, 16384), _log(rng, 1000, 151936), 8 * _log(rng, 8, 640)
        return dict(op=op, T=T, V=V, H=H, scale=rng.choice([1.0, math.sqrt(H)]),
                    grad=rng.choice(["bf16", "fp32"]), add=rng.random() < 0.4)
    if op == "balance":
        E = rng.choice([8, 16, 60, 64, 127, 128, 256])
        return dict(op=op, T=_log(rng, 1, 32768), E=E, k=rng.choice([1, 2, 4, 8]), masked=rng.choice([0.0, 0.125, 0.5]))
    T = _log(rng, 1, 16384 if op != "act8_swiglu" else 8192)
    H = 8 * _log(rng, 8, 640 if op != "act8_swiglu" else 2176)
    return dict(op=op, T=T, H=H, pad=rng.choice([0, 0, 8, 512]) if op == "act8_hold" else 0)


# -------------------------------------------------------------------- inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 1009 + 7)


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _zipf(g, n, V):
    """Token ids with a natural-text frequency: P(rank r) ~ 1/r, ranks scattered over the ids."""
    u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
    r = torch.exp(u * math.log(V)).long().clamp_(1, V) - 1
    return (r * 7919 + 13) % V if math.gcd(7919, V) == 1 else r


def prepare(case, seed):
    g, op = _gen(seed), case["op"]
    s = dict(case=dict(case))
    if op == "head":
        T, V, H = case["T"], case["V"], case["H"]
        w = torch.empty(V, H, device=DEV, dtype=torch.bfloat16).normal_(0.0, 0.02, generator=g)
        y = _zipf(g, T, V)
        # hidden states lean towards their label's row, so that labels get anything from no to nearly all of the probability
        wy = w[y].float()
        lean = 14.0 * torch.rand(T, 1, generator=g, device=DEV)
        x = _randn(g, T, H) + lean * case["tau"] * wy / wy.square().sum(-1, keepdim=True).clamp_min(1e-6)
        skip = (torch.arange(T, device=DEV) % 16) == 15          # prompt and padding positions: no label
        y = torch.where(skip, torch.full_like(y, -1), y)
        coef = -(0.5 + torch.rand(T, generator=g, device=DEV)) / T
        s.update(x=x.bfloat16(), w=w, y=y, coef=torch.where(skip, torch.zeros_like(coef), coef))
        if case["train"]:
            s["dw"] = torch.empty(V, H, device=DEV, dtype=torch.bfloat16)     # the step's gradient buffer
    elif op == "embed":
        T, V, H = case["T"], case["V"], case["H"]
        dt = torch.float32 if case["grad"] == "fp32" else torch.bfloat16
        s.update(ids=_zipf(g, T, V), dy=(_randn(g, T, H) / math.sqrt(T)).bfloat16(),
                 table=torch.empty(V, H, device=DEV, dtype=torch.bfloat16).normal_(0.0, 0.02, generator=g),
                 dtable=torch.empty(V, H, device=DEV, dtype=dt))
        if case["add"]:
            s["before"] = torch.empty(V, H, device=DEV, dtype=dt).normal_(0.0, 0.01, generator=g)
    elif op == "balance":
        T, E, k = case["T"], case["E"], case["k"]
        # logits with a favourite expert or two, as an unbalanced router has
        p = torch.softmax(1.5 * _randn(g, T, E) + 1.0 * _randn(g, 1, E), -1)
        keep = torch.rand(T, generator=g, device=DEV) >= case["masked"] if case["masked"] else None
        s.update(probs=p, idx=p.topk(k, -1).indices.int(), keep=keep)
    else:
        T, H = case["T"], case["H"]
        wide = 2 * H if op == "act8_swiglu" else H
        # residual-stream-like columns: a few run much larger than the rest
        col = torch.exp(0.7 * _randn(g, 1, wide))
        x = (_randn(g, T, wide + case["pad"])[:, :wide] * col).bfloat16()
        buf = torch.empty(T, wide + case["pad"], device=DEV, dtype=torch.bfloat16)
        buf[:, :wide] = x
        s["x"] = buf[:, :wide]
        if op == "act8_norm":
            s["w"] = (1.0 + 0.1 * _randn(g, H)).bfloat16()
        if op == "act8_swiglu":
            s["dout"] = _randn(g, T, H).bfloat16()
    return s


# ---------------------------------------------------------------- plain forms
def _hold8(x):
    """x in 8 bits per 128 columns of a row, as the fp32 values that it stands for."""
    T, H = x.shape
    n = -(-H // BLOCK)
    b = torch.nn.functional.pad(x.float(), (0, n * BLOCK - H)).view(T, n, BLOCK)
    amax = b.abs().amax(-1, keepdim=True)
    live = amax >= TINY
    q = torch.round(b * torch.where(live, 127.0 / amax, torch.zeros_like(amax)))
    scale = torch.where(live, amax * (1.0 / 127.0), torch.zeros_like(amax))
    return (q * scale).view(T, n * BLOCK)[:, :H]


def _norm(x, w, eps=1e-6):
    r = torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    return (x * r * w.float()).bfloat16(), r[:, 0]


def _plain(s):
    c, op = s["case"], s["case"]["op"]
    if op == "head":
        x, w, y = s["x"].float(), s["w"].float(), s["y"]
        it = 1.0 / c["tau"]
        z = (x @ w.t()) * it
        top = z.amax(-1, keepdim=True)
        e = torch.exp(z - top)
        total = e.sum(-1, keepdim=True)
        lse = top + torch.log(total)
        ok = y >= 0
        at = y.clamp_min(0).unsqueeze(1)
        logp = torch.where(ok, (z.gather(1, at) - lse)[:, 0], torch.zeros_like(lse[:, 0]))
        p = e / total
        if not c["train"]:
            return dict(logp=logp, ent=lse[:, 0] - (p * z).sum(-1), lse=lse[:, 0])
        ct = (s["coef"] * it).unsqueeze(1)
        dz = p * -ct
        dz.scatter_add_(1, at, torch.where(ok.unsqueeze(1), ct, torch.zeros_like(ct)))
        s["dw"].copy_(dz.t() @ x)
        return dict(logp=logp, lse=lse[:, 0], dx=(dz @ w).bfloat16(), dw=s["dw"])
    if op == "embed":
        out = (s["table"][s["ids"]].float() * c["scale"]).bfloat16()
        g = s["before"].float() if c["add"] else torch.zeros(s["dtable"].shape, device=DEV)
        g = g.index_add(0, s["ids"], s["dy"].float() * c["scale"])
        s["dtable"].copy_(g)
        return dict(out=out, dtable=s["dtable"])
    if op == "balance":
        p, E = s["probs"], c["E"]
        m = torch.ones(c["T"], device=DEV) if s["keep"] is None else s["keep"].float()
        hit = (s["idx"].long().unsqueeze(-1) == torch.arange(E, device=DEV)).sum(1) * m.long().unsqueeze(-1)
        counts = hit.sum(0)
        n = m.sum().clamp_min(1.0)
        gain = 0.001 * E * counts.float() / (n * n)
        loss = (gain * (p * m.unsqueeze(-1)).sum(0)).sum()
        dl = m.unsqueeze(-1) * p * (gain - (gain * p).sum(-1, keepdim=True))
        return dict(loss=loss, counts=counts.int(), gain=gain, dlogits=dl)
    if op == "act8_hold":
        return dict(x8=_hold8(s["x"]).bfloat16())
    if op == "act8_norm":
        hn, rstd = _norm(s["x"].float(), s["w"])
        x8 = _hold8(s["x"])
        hn8, rstd8 = _norm(x8, s["w"])
        return dict(hn=hn, rstd=rstd, x8=x8.bfloat16(), hn8=hn8, rstd8=rstd8)
    F = c["H"]
    gate, up = s["x"][:, :F].float(), s["x"][:, F:].float()
    a = gate / (1 + torch.exp(-gate)) * up
    gu8, d = _hold8(s["x"]), s["dout"].float()
    gate, up = gu8[:, :F], gu8[:, F:]
    sg = 1 / (1 + torch.exp(-gate))
    act = gate * sg
    dgu = torch.cat([d * up * (sg + act * (1 - sg)), d * act], 1)
    return dict(a=a.bfloat16(), dgu=dgu.bfloat16(), a8=(act * up).bfloat16())


# ------------------------------------------------------ through the framework
def _own(s):
    from kore_b200.ops import act8, moe, vocab
    c, op = s["case"], s["case"]["op"]
    if op == "head":
        logp, ent, lse = vocab.head_fwd(s["x"], s["w"], s["y"], c["tau"], want_entropy=not c["train"])
        if not c["train"]:
            return dict(logp=logp, ent=ent, lse=lse)
        dx, dw = vocab.head_bwd(s["x"], s["w"], s["y"], lse, s["coef"], c["tau"], dw=s["dw"])
        return dict(logp=logp, lse=lse, dx=dx, dw=dw)
    if op == "embed":
        out = vocab.embed(s["ids"], s["table"], c["scale"])
        if c["add"]:
            s["dtable"].copy_(s["before"])
        vocab.embed_grad(s["ids"], s["dy"], s["dtable"], c["scale"], accumulate=c["add"])
        return dict(out=out, dtable=s["dtable"])
    if op == "balance":
        loss, counts, gain = moe.balance_loss(s["probs"], s["idx"], s["keep"], coef=0.001)
        return dict(loss=loss, counts=counts, gain=gain, dlogits=moe.balance_bwd(s["probs"], gain, s["keep"]))
    if op == "act8_hold":
        return dict(x8=act8.load(act8.save(s["x"])))
    if op == "act8_norm":
        hn, rstd, held = act8.rmsnorm_save(s["x"], s["w"], 1e-6)
        x8, hn8, rstd8 = act8.rmsnorm_load(held, s["w"], 1e-6)
        return dict(hn=hn, rstd=rstd, x8=x8, hn8=hn8, rstd8=rstd8)
    a, held = act8.swiglu_save(s["x"])
    dgu, a8 = act8.swiglu_bwd(s["dout"], held)
    return dict(a=a, dgu=dgu, a8=a8)


def run(state):
    with torch.no_grad():
        return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------- work
def work(case):
    op, T = case["op"], case["T"]
    if op == "head":
        V, H = case["V"], case["H"]
        b = 2 * (T + V) * H + 8 * T + 4 * T * (2 if case["train"] else 3)
        if not case["train"]:
            return dict(bytes=b, flops=2 * T * V * H)
        # three products; a 16th of the positions carries no label and needs no gradient
        return dict(bytes=b + 4 * T + 2 * (T + V) * H, flops=2 * T * V * H + 4 * (T - T // 16) * V * H)
    if op == "embed":
        V, H = case["V"], case["H"]
        pr = 1.0 / (torch.arange(1, V + 1, dtype=torch.float64) * math.log(V))
        rows = min(float(T), float((1 - torch.exp(-T * pr)).sum()))      # distinct ids expected
        size = 4 if case["grad"] == "fp32" else 2
        return dict(bytes=8 * T + 2 * H * (rows + 2 * T) + size * V * H * (2 if case["add"] else 1), flops=3 * T * H)
    if op == "balance":
        E, k = case["E"], case["k"]
        return dict(bytes=8 * T * E + 4 * T * k + (T if case["masked"] else 0) + 8 * E, flops=7 * T * E)
    H = case["H"]
    if op == "act8_hold":                       # x in, 8 bits and scales out and in, x out
        return dict(bytes=T * H * (2 + 2 + 2 + 8 / BLOCK), flops=6 * T * H)
    if op == "act8_norm":                       # x in, hn out; 8 bits out and in; x and hn out
        return dict(bytes=T * H * (2 + 2 + 2 + 8 / BLOCK + 4) + 8 * T + 2 * H, flops=14 * T * H)
    # gate|up in, a out; 8 bits out and in; dout in; dgate|dup and a out
    return dict(bytes=T * H * (4 + 2 + 4 + 16 / BLOCK + 2 + 4 + 2), flops=30 * T * H)


# --------------------------------------------------------------------- exact
def exact(case, seed):
    """The outputs of ``run`` for these inputs from the definitions in 64 bits."""
    s, op = prepare(case, seed), case["op"]
    f8 = torch.float64
    if op == "head":
        T, V, H = case["T"], case["V"], case["H"]
        w, tau = s["w"].to(f8), case["tau"]
        logp, ent, lse, dx = [], [], [], []
        dw = torch.zeros(V, H, dtype=f8, device=DEV) if case["train"] else None
        for i in range(0, T, 1024):
            x, y = s["x"][i:i + 1024].to(f8), s["y"][i:i + 1024]
            lp = torch.log_softmax((x @ w.T).div_(tau), -1)
            z0 = (x * w[y.clamp_min(0)]).sum(-1) / tau
            one = lp.gather(1, y.clamp_min(0)[:, None])[:, 0]
            lse.append(z0 - one)
            logp.append(one * (y >= 0))
            p = lp.exp()
            if not case["train"]:
                ent.append(-(p * lp).sum(-1))
                continue
            p[torch.arange(len(y), device=DEV), y.clamp_min(0)] -= (y >= 0).to(f8)
            p *= (-s["coef"][i:i + 1024].to(f8) / tau)[:, None]
            dx.append(p @ w)
            dw += p.T @ x
        logp, lse = torch.cat(logp), torch.cat(lse)
        return dict(logp=logp, lse=lse, dx=torch.cat(dx), dw=dw) if case["train"] else dict(logp=logp, ent=torch.cat(ent), lse=lse)
    if op == "embed":
        order = torch.argsort(s["ids"], stable=True)
        g = s["before"].to(f8) if case["add"] else torch.zeros(case["V"], case["H"], dtype=f8, device=DEV)
        for i in range(0, case["T"], 4096):
            at = order[i:i + 4096]
            g.index_put_((s["ids"][at],), s["dy"][at].to(f8) * case["scale"], accumulate=True)
        return dict(out=s["table"].index_select(0, s["ids"]).to(f8) * case["scale"], dtable=g)
    if op == "balance":
        E, T = case["E"], case["T"]
        keep = torch.ones(T, dtype=torch.bool, device=DEV) if s["keep"] is None else s["keep"]
        counts = torch.bincount(s["idx"][keep].long().reshape(-1), minlength=E)
        n = max(1, int(keep.sum()))
        gain = 0.001 * E * counts.to(f8) / n ** 2
        p = s["probs"].to(f8)
        dl = p * (gain[None] - (p @ gain)[:, None])
        dl[~keep] = 0
        return dict(loss=torch.dot(gain, p[keep].sum(0)), counts=counts.int(), gain=gain, dlogits=dl)
    x = s["x"].to(f8)
    held = torch.empty_like(x)
    for i in range(0, x.shape[1], BLOCK):
        b = x[:, i:i + BLOCK]
        step = b.abs().max(-1, keepdim=True).values / 127
        held[:, i:i + BLOCK] = torch.where(step > 0, torch.round(b / step) * step, torch.zeros_like(b))
    if op == "act8_hold":
        return dict(x8=held)
    if op == "act8_norm":
        w = s["w"].to(f8)
        r, r8 = ((v * v).mean(-1).add(1e-6).pow(-0.5) for v in (x, held))
        return dict(hn=x * r[:, None] * w, rstd=r, x8=held, hn8=held * r8[:, None] * w, rstd8=r8)
    F = case["H"]
    silu = torch.nn.functional.silu
    g8, u8, d = held[:, :F], held[:, F:], s["dout"].to(f8)
    sg = torch.sigmoid(g8)
    return dict(a=silu(x[:, :F]) * x[:, F:], a8=silu(g8) * u8,
                dgu=torch.cat([d * u8 * sg * (1 + g8 * (1 - sg)), d * silu(g8)], 1))
