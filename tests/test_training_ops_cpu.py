"""The CPU definitions of the vocabulary, balance and 8-bit checkpoint operators
against autograd and differences in 64 bits, and their refusals."""
import math

import pytest
import torch

from kore_b200.ops import act8, moe, vocab

F8 = torch.float64


@pytest.mark.parametrize("T,V,H,tau,piece", [(1, 7, 8, 1.0, 0), (13, 50, 24, 0.7, 16), (40, 33, 8, 1.5, 33), (5, 101, 16, 1.0, 1)])
def test_head_matches_autograd(T, V, H, tau, piece):
    g = torch.Generator().manual_seed(T)
    x, w = torch.randn(T, H, generator=g), torch.randn(V, H, generator=g) / math.sqrt(H)
    y = torch.randint(0, V, (T,), generator=g)
    coef = torch.randn(T, generator=g)
    coef[::3] = 0
    if T > 4:
        y[1] = -1
    a, b = x.to(F8).requires_grad_(True), w.to(F8).requires_grad_(True)
    z = a @ b.t() / tau
    lse = torch.logsumexp(z, -1)
    ok = y >= 0
    logp = torch.where(ok, z.gather(1, y.clamp_min(0)[:, None])[:, 0], torch.zeros((), dtype=F8)) - lse
    (coef.to(F8) * logp).sum().backward()
    lp, ent, l = vocab.head_fwd(x, w, y, tau, want_entropy=True)
    # fp32 products and sums of H and V terms
    assert torch.allclose(l.to(F8), lse.detach(), rtol=1e-5, atol=1e-5)
    assert torch.allclose(lp.to(F8), torch.where(ok, logp.detach(), 0.0), rtol=1e-5, atol=1e-5)
    p = torch.softmax(z.detach(), -1)
    assert torch.allclose(ent.to(F8), -(p * p.log()).sum(-1), rtol=1e-5, atol=1e-5)
    dx, dw = vocab.head_bwd(x, w, y, l, coef, tau, piece=piece)
    assert torch.allclose(dx.to(F8), a.grad, rtol=1e-4, atol=1e-5)
    assert torch.allclose(dw.to(F8), b.grad, rtol=1e-4, atol=1e-5)
    acc = torch.ones_like(w)
    vocab.head_bwd(x, w, y, l, coef, tau, dw=acc, accumulate=True, piece=piece)
    assert torch.allclose(acc.to(F8), 1 + b.grad, rtol=1e-4, atol=1e-5)


def test_head_masked_rows_and_no_rows():
    x, w = torch.randn(4, 8), torch.randn(9, 8)
    y, coef = torch.tensor([1, 2, -1, 4]), torch.tensor([0.5, 0.0, 0.0, -1.0])
    _, _, l = vocab.head_fwd(x, w, y)
    want = vocab.head_bwd(x, w, y, l, coef)
    x[1], x[2] = float("nan"), float("inf")
    _, _, l = vocab.head_fwd(x, w, y)
    got = vocab.head_bwd(x, w, y, l, coef)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    lp, ent, l = vocab.head_fwd(x[:0], w, y[:0], want_entropy=True)
    assert lp.numel() == ent.numel() == l.numel() == 0
    with pytest.raises(ValueError):
        vocab.head_fwd(x, w, y, 0.0)
    with pytest.raises(ValueError):
        vocab.head_bwd(x, w, y, torch.zeros(4), coef, accumulate=True)


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_embedding(dt):
    g = torch.Generator().manual_seed(0)
    table = torch.randn(11, 16, generator=g).to(dt)
    ids = torch.tensor([3, 3, -1, 10, 11, 0, 3])
    ok = (ids >= 0) & (ids < 11)
    out = vocab.embed(ids, table, 2.5)
    assert torch.equal(out[ok], (table[ids[ok]].float() * 2.5).to(dt)) and (out[~ok] == 0).all()
    dy = torch.randn(7, 16, generator=g).to(dt)
    want = torch.zeros(11, 16, dtype=F8).index_add_(0, ids[ok], dy[ok].to(F8)) * 2.5
    unit = 2.0 ** -8 if dt == torch.bfloat16 else 2.0 ** -22
    got = vocab.embed_grad(ids, dy, torch.full((11, 16), float("nan"), dtype=dt), 2.5, accumulate=False)
    assert ((got.to(F8) - want).abs() <= unit * want.abs() + 1e-6).all()
    base = torch.randn(11, 16, generator=g).to(dt)
    acc = vocab.embed_grad(ids, dy, base.clone(), 2.5)
    assert ((acc.to(F8) - base.to(F8) - want).abs() <= unit * (base.to(F8).abs() + want.abs()) + 1e-6).all()
    assert torch.equal(acc[1], base[1])


@pytest.mark.parametrize("masked", [False, True])
def test_balance_gradient_by_differences(masked):
    g = torch.Generator().manual_seed(1)
    T, E, k = 12, 6, 2
    logits = torch.randn(T, E, generator=g, dtype=F8)
    idx = torch.softmax(logits, -1).topk(k, -1).indices.int()
    mask = (torch.arange(T) % 3 != 0) if masked else None
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask
    counts = torch.bincount(idx[keep].long().reshape(-1), minlength=E)

    def f(l):
        p = torch.softmax(l, -1)[keep]
        return 0.3 * E * (counts.to(F8) / keep.sum() * p.mean(0)).sum()

    probs = torch.softmax(logits, -1).float()
    loss, c, gain = moe.balance_loss(probs, idx, mask, 0.3)
    assert torch.equal(c.long(), counts) and abs(loss.to(F8) - f(logits)) < 1e-6
    d = moe.balance_bwd(probs, gain, mask)
    for _ in range(4):
        v = torch.randn(T, E, generator=g, dtype=F8)
        num = (f(logits + 1e-5 * v) - f(logits - 1e-5 * v)) / 2e-5
        assert abs(num - (d.to(F8) * v).sum()) < 1e-6
    base = torch.randn(T, E, generator=g)
    assert torch.allclose(moe.balance_bwd(probs, gain, mask, 2.0, base.clone()), base + 2 * d, atol=1e-6)


def test_balance_even_routing():
    T, E, k = 32, 8, 2
    idx = (torch.arange(T * k) % E).view(T, k).int()
    loss, counts, _ = moe.balance_loss(torch.full((T, E), 1 / E), idx, coef=1.0)
    assert (counts == T * k // E).all() and abs(float(loss) - k) < 1e-6


@pytest.mark.parametrize("T,H", [(0, 8), (1, 8), (5, 136), (9, 384)])
def test_act8_round_trip(T, H):
    x = (torch.randn(T, H) * torch.exp(2 * torch.randn(1, H))).bfloat16()
    a = act8.save(x)
    assert a.q.dtype == torch.int8 and a.s.shape == (T, -(-H // 128)) and a.nbytes() == T * H + 4 * a.s.numel()
    back = act8.load(a, dtype=torch.float32)
    if T:
        amax = torch.nn.functional.pad(x.float().abs(), (0, -H % 128)).view(T, -1, 128).amax(-1)
        lim = amax.repeat_interleave(128, 1)[:, :H] / 254 * (1 + 1e-4)
        assert ((back - x.float()).abs() <= lim).all()


def test_act8_odd_blocks_and_refusals():
    x = torch.zeros(4, 256).bfloat16()
    x[0, 0], x[1, 130], x[2, 5] = 1e-38, float("inf"), float("nan")
    v = act8.load(act8.save(x))
    assert (v[0] == 0).all() and (v[3] == 0).all()
    assert torch.isnan(v[1, 128:]).all() and (v[1, :128] == 0).all() and torch.isnan(v[2, :128]).all()
    with pytest.raises(ValueError):
        act8.save(torch.zeros(2, 12).bfloat16())
    with pytest.raises(ValueError):
        act8.swiglu_save(torch.zeros(2, 24).bfloat16())


def test_act8_in_the_forward_and_backward():
    g = torch.Generator().manual_seed(2)
    x, w = torch.randn(6, 192, generator=g).bfloat16(), torch.randn(192, generator=g).bfloat16()
    hn, rstd, a = act8.rmsnorm_save(x, w, 1e-6)
    r = (x.to(F8).square().mean(-1) + 1e-6).rsqrt()
    assert torch.allclose(rstd.to(F8), r, rtol=1e-6) and torch.equal(a.q, act8.save(x).q)
    assert torch.allclose(hn.to(F8), x.to(F8) * r[:, None] * w.to(F8), rtol=2.0 ** -8, atol=1e-30)
    x8, hn8, rstd8 = act8.rmsnorm_load(a, w, 1e-6)
    v = act8.load(a, dtype=torch.float32).to(F8)
    r = (v.square().mean(-1) + 1e-6).rsqrt()
    assert torch.equal(x8, act8.load(a)) and torch.allclose(rstd8.to(F8), r, rtol=1e-6)
    assert torch.allclose(hn8.to(F8), v * r[:, None] * w.to(F8), rtol=2.0 ** -8, atol=1e-30)

    gu, dout = torch.randn(6, 192, generator=g).bfloat16(), torch.randn(6, 96, generator=g).bfloat16()
    out, held = act8.swiglu_save(gu)
    silu = torch.nn.functional.silu
    assert torch.allclose(out.to(F8), silu(gu[:, :96].to(F8)) * gu[:, 96:].to(F8), rtol=2.0 ** -8, atol=1e-6)
    dgu, again = act8.swiglu_bwd(dout, held)
    v = act8.load(held, dtype=torch.float32).to(F8).requires_grad_(True)
    act = silu(v[:, :96]) * v[:, 96:]
    want, = torch.autograd.grad(act, v, dout.to(F8))
    assert torch.allclose(dgu.to(F8), want, rtol=2.0 ** -8, atol=1e-5)
    assert torch.allclose(again.to(F8), act.detach(), rtol=2.0 ** -8, atol=1e-6)


def test_dependent_launches_read_with_plain_loads():
    """A kernel that starts while the one before it runs may not use read-only
    loads: they are defined only for memory that nobody writes meanwhile."""
    import re
    from pathlib import Path
    waiting = 0
    for f in sorted((Path(moe.__file__).resolve().parents[1] / "csrc").glob("*.cu")):
        text = re.sub(r"__(launch_bounds|cluster_dims)__\([^)]*\)", "", f.read_text())
        funcs = {}                     # device functions: from their qualifier to a brace in the first column
        for m in re.finditer(r"^(?:__global__|KORE_DEV) .*?^}", text, re.M | re.S):
            body = m.group(0)
            funcs[re.search(r"(\w+)\(", body).group(1)] = body
        todo = [n for n, body in funcs.items() if "pdl_wait()" in body]
        waiting += len(todo)
        reach = set()
        while todo:
            n = todo.pop()
            if n not in reach:
                reach.add(n)
                todo += [c for c in re.findall(r"(\w+)(?:<\w+>)?\(", funcs[n]) if c in funcs]
        for n in reach:
            assert "__ldg" not in funcs[n] and not re.search(r"const \w+\s*\*\s*__restrict__", funcs[n]), (f.name, n)
    assert waiting >= 18
