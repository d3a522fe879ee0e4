"""The router's balance loss: the native kernels against the definition in 64 bits."""
import pytest
import torch

from kore_b200.ops import moe

pytestmark = pytest.mark.gpu
F8 = torch.float64


def _case(T, E, k, masked, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + E)
    logits = 2 * torch.randn(T, E, generator=g, device="cuda")
    probs, idx, _ = moe.route(logits, k)
    mask = torch.rand(T, generator=g, device="cuda") >= masked if masked else None
    return logits, probs, idx, mask


def _oracle(probs, idx, mask, coef, E):
    T = probs.shape[0]
    keep = torch.ones(T, dtype=torch.bool, device="cuda") if mask is None else mask
    counts = torch.bincount(idx[keep].long().reshape(-1), minlength=E)
    n = max(1, int(keep.sum()))
    gain = coef * E * counts.to(F8) / n ** 2
    p = probs.to(F8)
    return (gain * p[keep].sum(0)).sum(), counts, gain, torch.where(keep[:, None], p * (gain - (p @ gain)[:, None]), 0.0), keep


@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 8, 2), (7, 8, 8), (64, 60, 4), (1000, 127, 2), (4099, 128, 8),
                                   (33, 256, 16), (20000, 64, 1)])
@pytest.mark.parametrize("masked", [0.0, 0.3, 1.1])
def test_balance(T, E, k, masked):
    _, probs, idx, mask = _case(T, E, k, masked)
    coef = 0.01
    want, counts, gain, dl, keep = _oracle(probs, idx, mask, coef, E)
    loss, c, g = moe.balance_loss(probs, idx, mask, coef)
    assert c.dtype == torch.int32 and torch.equal(c.long(), counts)
    assert torch.allclose(g.to(F8), gain, rtol=1e-6, atol=0)
    # sums of positive fp32 terms, at most 64 + blocks roundings deep
    assert abs(loss.to(F8) - want) <= 4e-5 * want
    d = moe.balance_bwd(probs, g, mask, dloss=2.0)
    tol = 2e-6 * (probs.to(F8) * (gain + (probs.to(F8) @ gain)[:, None])) * 2
    assert ((d.to(F8) - 2 * dl).abs() <= tol + 1e-30).all()
    base = torch.randn(T, E, device="cuda")
    acc = moe.balance_bwd(probs, g, mask, dloss=2.0, dlogits=base.clone())
    assert ((acc.to(F8) - base.to(F8) - 2 * dl).abs() <= tol + 2.0 ** -23 * (base.abs() + 2 * dl.abs())).all()
    assert torch.equal(acc[~keep], base[~keep])
    again = moe.balance_loss(probs, idx, mask, coef)
    assert torch.equal(again[0], loss) and torch.equal(again[2], g)


def test_balance_is_the_gradient():
    logits, _, idx, mask = _case(50, 16, 2, 0.2)
    coef = 0.5

    def loss(l):
        p = torch.softmax(l, -1)
        return _oracle(p, idx, mask, coef, 16)[0]

    probs = torch.softmax(logits, -1)
    _, _, gain = moe.balance_loss(probs, idx, mask, coef)
    d = moe.balance_bwd(probs, gain, mask)
    g = torch.Generator(device="cuda").manual_seed(1)
    h = 1e-5
    for _ in range(4):
        v = torch.randn(50, 16, generator=g, device="cuda", dtype=F8)
        num = (loss(logits.to(F8) + h * v) - loss(logits.to(F8) - h * v)) / (2 * h)
        assert abs(num - (d.to(F8) * v).sum()) <= 1e-5 * (d.to(F8) * v).abs().sum() + 1e-9


def test_masked_tokens_may_hold_anything_and_foreign_choices_do_not_count():
    _, probs, idx, _ = _case(40, 8, 2, 0.0)
    mask = torch.ones(40, dtype=torch.bool, device="cuda")
    mask[3] = mask[17] = False
    want = moe.balance_loss(probs, idx, mask, 1.0)
    dl = moe.balance_bwd(probs, want[2], mask)
    probs[3], idx[17] = float("nan"), -1
    got = moe.balance_loss(probs, idx, mask, 1.0)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert torch.equal(moe.balance_bwd(probs, got[2], mask), dl) and (dl[3] == 0).all()
    idx[0, 0], idx[1, 1] = -1, 8
    assert int(moe.balance_loss(probs, idx, mask, 1.0)[1].sum()) == 2 * 38 - 2


def test_balance_no_tokens_and_refusals():
    p = torch.rand(4, 8, device="cuda")
    i = torch.zeros(4, 2, dtype=torch.int32, device="cuda")
    loss, c, g = moe.balance_loss(p[:0], i[:0])
    assert loss == 0 and (c == 0).all() and (g == 0).all()
    assert moe.balance_bwd(p[:0], g).shape == (0, 8)
    for f in (lambda: moe.balance_loss(p.double(), i), lambda: moe.balance_loss(p, i.long()),
              lambda: moe.balance_loss(p, i[:3]), lambda: moe.balance_loss(p, i, torch.ones(4, device="cuda")),
              lambda: moe.balance_loss(p, i, torch.ones(3, device="cuda").bool()),
              lambda: moe.balance_loss(torch.rand(4, 257, device="cuda"), i),
              lambda: moe.balance_loss(p, torch.zeros(4, 17, dtype=torch.int32, device="cuda")),
              lambda: moe.balance_loss(p.t(), i), lambda: moe.balance_bwd(p, g[:4]),
              lambda: moe.balance_bwd(p, g, dlogits=torch.zeros(4, 7, device="cuda"))):
        with pytest.raises(RuntimeError):
            f()
