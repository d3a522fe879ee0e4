"""Head loss in vocabulary pieces and embedding with sorted gradient: the native
kernels against the definitions in 64 bits."""
import math

import pytest
import torch

from kore_b200 import ops
from kore_b200.ops import vocab

pytestmark = pytest.mark.gpu
F8 = torch.float64


def _inputs(T, V, H, seed=0, lean=8.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = (torch.randn(V, H, generator=g, device="cuda") * 0.5 / math.sqrt(H)).bfloat16()
    y = torch.randint(0, V, (T,), generator=g, device="cuda")
    wy = w[y].float()
    x = torch.randn(T, H, generator=g, device="cuda") + lean * torch.rand(T, 1, generator=g, device="cuda") * wy / \
        wy.square().sum(-1, keepdim=True)
    coef = torch.randn(T, generator=g, device="cuda") / T
    return x.bfloat16(), w, y, coef


def _oracle(x, w, y, coef, tau):
    """64-bit values, and the sums of magnitudes that rounding errors scale with."""
    x, w, coef = x.to(F8), w.to(F8), coef.to(F8)
    lp = torch.log_softmax(x @ w.t() / tau, -1)
    ok = (y >= 0) & (y < w.shape[0])
    yy = torch.where(ok, y, torch.zeros_like(y))
    logp = torch.where(ok, lp.gather(1, yy[:, None])[:, 0], torch.zeros((), dtype=F8, device=x.device))
    lse = torch.logsumexp(x @ w.t() / tau, -1)
    p = lp.exp()
    ent = -(p * lp).sum(-1)
    one = torch.zeros_like(p)
    one[torch.arange(len(y), device=x.device), yy] = ok.to(F8)
    live = (coef != 0)[:, None]
    dz = torch.where(live, (coef / tau)[:, None] * (one - p), torch.zeros_like(p))
    xm = torch.where(live, x, torch.zeros_like(x))
    # a logit is off by delta: the tensor cores add 16 products at a time and truncate the fp32
    # partial sum, by at most 2^-23 of it; dz is off by 2^-8 of itself (bf16) and p delta
    mag = (x.abs() @ w.abs().t()).amax(-1)
    delta = (x.shape[1] / 16 + 2) * 2.0 ** -23 * mag / tau + 2e-6 * (1 + lse.abs())
    slack = 2.0 ** -8 * dz.abs() + torch.where(live, 2 * delta[:, None] * p * (coef.abs() / tau)[:, None], torch.zeros_like(p))
    dx, dw = dz @ w, dz.t() @ xm
    # plus the fp32 sums (2^-18 of the magnitudes is 32 roundings of the partial sums) and the output's own rounding
    tdx = (slack + 2.0 ** -18 * dz.abs()) @ w.abs() + 2.0 ** -8 * dx.abs() + 1e-30
    tdw = (slack + 2.0 ** -18 * dz.abs()).t() @ xm.abs() + 2.0 ** -8 * dw.abs() + 1e-30
    return dict(logp=logp, lse=lse, ent=ent, dx=dx, dw=dw, delta=delta, tdx=tdx, tdw=tdw)


def _check_fwd(o, logp, ent, lse):
    assert ops.check_device_error() == 0
    assert ((lse.to(F8) - o["lse"]).abs() <= o["delta"]).all()
    assert ((logp.to(F8) - o["logp"]).abs() <= 2 * o["delta"]).all()
    if ent is not None:
        # d ent = -sum p (log p + ent) dz: delta times the spread of log p
        spread = 2 + o["lse"].abs() + o["ent"].abs()
        assert ((ent.to(F8) - o["ent"]).abs() <= 4 * o["delta"] * spread).all()


SHAPES = [(1, 8, 8), (1, 1, 64), (3, 17, 72), (129, 1000, 256), (127, 32000, 256), (257, 4097, 264), (300, 513, 1032),
          (1000, 9999, 640), (64, 151936, 128), (2, 5000, 5120),
          (33001, 130, 64), (513, 20011, 5120)]


@pytest.mark.parametrize("T,V,H", SHAPES)
@pytest.mark.parametrize("tau", [1.0, 0.6])
def test_head_forward(T, V, H, tau):
    x, w, y, coef = _inputs(T, V, H)
    if T > 2:
        y[1], y[2] = -1, V
    o = _oracle(x, w, y, coef, tau)
    logp, ent, lse = vocab.head_fwd(x, w, y, tau, want_entropy=True)
    _check_fwd(o, logp, ent, lse)
    logp2, none, lse2 = vocab.head_fwd(x, w, y, tau)
    assert none is None
    _check_fwd(o, logp2, None, lse2)
    nolp, _, lse3 = vocab.head_fwd(x, w, None, tau)
    assert nolp is None and torch.equal(lse2, lse3)


@pytest.mark.parametrize("T,V,H", SHAPES)
@pytest.mark.parametrize("piece", [0, 264])
def test_head_backward(T, V, H, piece):
    if piece and V > 30000:
        piece = 50008
    tau = 0.8
    x, w, y, coef = _inputs(T, V, H, seed=1)
    coef[::4] = 0
    if T > 3:
        y[1] = -1
        coef[1] = 0.3
    o = _oracle(x, w, y, coef, tau)
    _, _, lse = vocab.head_fwd(x, w, y, tau)
    dx, dw = vocab.head_bwd(x, w, y, lse, coef, tau, piece=piece)
    assert ops.check_device_error() == 0
    extra = 2 if piece else 1               # dx of several pieces: fp32 sums of the pieces
    assert ((dx.to(F8) - o["dx"]).abs() <= extra * o["tdx"]).all()
    assert ((dw.to(F8) - o["dw"]).abs() <= o["tdw"]).all()
    assert (dx[coef == 0] == 0).all()
    # fp32 gradient buffer, added to
    base = torch.randn(V, H, device="cuda") * 0.01
    acc = base.clone()
    vocab.head_bwd(x, w, y, lse, coef, tau, dw=acc, accumulate=True, piece=piece)
    assert ((acc.to(F8) - base.to(F8) - o["dw"]).abs() <= o["tdw"] + 2.0 ** -22 * base.abs()).all()


def test_head_backward_is_the_gradient():
    """Directional differences of the loss in 64 bits."""
    T, V, H, tau = 37, 523, 64, 1.3
    x, w, y, coef = _inputs(T, V, H, seed=2, lean=4.0)
    _, _, lse = vocab.head_fwd(x, w, y, tau)
    dx, dw = vocab.head_bwd(x, w, y, lse, coef, tau)

    def loss(x, w):
        return (coef.to(F8) * torch.log_softmax(x @ w.t() / tau, -1).gather(1, y[:, None])[:, 0]).sum()

    g = torch.Generator(device="cuda").manual_seed(3)
    h = 1e-4
    for a, d in ((x, dx), (w, dw)):
        for _ in range(4):
            v = torch.randn(a.shape, generator=g, device="cuda", dtype=F8)
            args = ((x.to(F8) + h * v, w.to(F8)), (x.to(F8) - h * v, w.to(F8))) if a is x else \
                ((x.to(F8), w.to(F8) + h * v), (x.to(F8), w.to(F8) - h * v))
            num = (loss(*args[0]) - loss(*args[1])) / (2 * h)
            # independent roundings of 2^-8 per entry along a random direction: 6 sigma
            assert abs(num - (d.to(F8) * v).sum()) <= 6 * 2.0 ** -8 * (d.to(F8) * v).norm() + 1e-6


@pytest.mark.parametrize("T,H", [(100, 1024), (300, 1024), (300, 2048), (100, 5120), (300, 5120)])
def test_head_backward_of_well_predicted_labels(T, H):
    """The label's entry c (p - 1) with p near 1: it is the difference of the logit, summed
    as the forward summed it, and the forward's lse, so only their last roundings show."""
    V = 6000
    g = torch.Generator(device="cuda").manual_seed(H)
    w = (torch.randn(V, H, generator=g, device="cuda") * 0.02).bfloat16()
    y = torch.randperm(V, generator=g, device="cuda")[:T]
    wy = w[y].float()
    lean = torch.linspace(6.0, 30.0, T, device="cuda")[:, None]         # 1 - p from near 1 down to 1e-9
    x = (torch.randn(T, H, generator=g, device="cuda") + lean * wy / wy.square().sum(-1, keepdim=True)).bfloat16()
    coef = torch.full((T,), -1.0, device="cuda")
    _, _, lse = vocab.head_fwd(x, w, y)
    dx, dw = vocab.head_bwd(x, w, y, lse, coef)
    assert ops.check_device_error() == 0
    z = x.to(F8) @ w.to(F8).t()
    l = torch.logsumexp(z, -1, keepdim=True)
    p = (z - l).exp()
    rows = torch.arange(T, device="cuda")
    mag = (x.to(F8).abs() @ w.to(F8).abs().t()).amax(-1, keepdim=True)
    delta = (H / 16 + 2) * 2.0 ** -23 * mag + 2e-6 * (1 + l.abs())      # of another entry's logit
    slack = (2.0 ** -8 + 2 * delta) * p
    dz = p.clone()
    dz[rows, y] = torch.expm1(z[rows, y] - l[:, 0])
    # eight roundings of 2^-24 of lse between the logit and the exponent, and the exponential's own
    slack[rows, y] = 2.0 ** -8 * dz[rows, y].abs() + 2.0 ** -21 * (1 + l[:, 0].abs())
    slack += 2.0 ** -18 * dz.abs()
    want = dz @ w.to(F8)
    assert ((dx.to(F8) - want).abs() <= slack @ w.to(F8).abs() + 2.0 ** -8 * want.abs() + 1e-30).all()
    want = dz.t() @ x.to(F8)
    assert ((dw.to(F8) - want).abs() <= slack.t() @ x.to(F8).abs() + 2.0 ** -8 * want.abs() + 1e-30).all()


def test_head_strides_streams_and_repeats():
    T, V, H = 200, 3001, 136
    x, w, y, coef = _inputs(T, V, H, seed=4)
    wide = torch.full((T, H + 24), float("nan"), device="cuda", dtype=torch.bfloat16)
    wide[:, 8:8 + H] = x
    ww = torch.full((V, H + 8), float("nan"), device="cuda", dtype=torch.bfloat16)
    ww[:, :H] = w
    logp, _, lse = vocab.head_fwd(x, w, y)
    dx, dw = vocab.head_bwd(x, w, y, lse, coef)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        l2, _, e2 = vocab.head_fwd(wide[:, 8:8 + H], ww[:, :H], y)
        dx2, dw2 = vocab.head_bwd(wide[:, 8:8 + H], ww[:, :H], y, e2, coef)
    torch.cuda.current_stream().wait_stream(s)
    for a, b in ((logp, l2), (lse, e2), (dx, dx2), (dw, dw2)):
        assert torch.equal(a, b)


def test_head_masked_rows_may_hold_anything():
    T, V, H = 70, 777, 64
    x, w, y, coef = _inputs(T, V, H, seed=5)
    coef[5], coef[6], y[6] = 0, 0, -1
    clean = vocab.head_fwd(x, w, y)
    dx, dw = vocab.head_bwd(x, w, y, clean[2], coef)
    bad = x.clone()
    bad[5], bad[6] = float("inf"), float("nan")
    logp, ent, lse = vocab.head_fwd(bad, w, y, want_entropy=True)
    rest = torch.ones(T, dtype=torch.bool, device="cuda")
    rest[5] = rest[6] = False
    assert torch.equal(lse[rest], clean[2][rest]) and torch.equal(logp[rest], clean[0][rest])
    assert torch.isnan(lse[5:7]).all() and torch.isnan(ent[5:7]).all()
    dx2, dw2 = vocab.head_bwd(bad, w, y, lse, coef)
    assert torch.equal(dx2, dx) and torch.equal(dw2, dw)


def test_head_logits_of_minus_inf():
    """Vocabulary entries with logit -inf have probability 0; the rest is as without them."""
    T, V, H = 40, 600, 64
    x, w, y, _ = _inputs(T, V, H, seed=6)
    x[:, 0] = 1.0
    w[:, 0] = 0.0
    keep = torch.ones(V, dtype=torch.bool, device="cuda")
    keep[100:420] = False
    y = y % 100
    want = vocab.head_fwd(x, w[keep].contiguous(), y, want_entropy=True)
    w[100:420, 0] = float("-inf")
    w[100:420, 1:] = 0.0
    got = vocab.head_fwd(x, w, y, want_entropy=True)
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=2e-5, atol=2e-5)


def test_head_without_coefficients_and_into_given_outputs():
    T, V, H = 150, 900, 128
    x, w, y, coef = _inputs(T, V, H, seed=7)
    _, _, lse = vocab.head_fwd(x, w, y)
    dx, dw = vocab.head_bwd(x, w, y, lse, torch.zeros_like(coef))
    assert (dx == 0).all() and (dw == 0).all()
    dx, dw = vocab.head_bwd(x, w, y, lse, coef)
    wide = torch.full((T, H + 8), 3.0, device="cuda", dtype=torch.bfloat16)
    got, _ = vocab.head_bwd(x, w, y, lse, coef, dx=wide[:, :H], dw=torch.full_like(dw, float("nan")))
    assert torch.equal(wide[:, :H], dx) and (wide[:, H:] == 3.0).all() and got.data_ptr() == wide.data_ptr()
    # bf16 dW is added to with one rounding of the sum
    base = torch.randn(V, H, device="cuda").bfloat16()
    exact = torch.zeros(V, H, device="cuda")
    vocab.head_bwd(x, w, y, lse, coef, dw=exact)
    acc = base.clone()
    vocab.head_bwd(x, w, y, lse, coef, dw=acc, accumulate=True)
    assert torch.equal(acc, (base.float() + exact).bfloat16())
    # no targets: the gradient of -coef lse
    dx, _ = vocab.head_bwd(x, w, None, lse, coef)
    p = torch.softmax(x.to(F8) @ w.to(F8).t(), -1)
    want = -(coef.to(F8)[:, None] * p) @ w.to(F8)
    assert ((dx.to(F8) - want).abs() <= 2.0 ** -7 * (coef.to(F8).abs()[:, None] * p) @ w.to(F8).abs() + 1e-9).all()


def test_head_no_rows_and_refusals():
    x, w, y, coef = _inputs(4, 32, 16)
    e = torch.empty(0, 16, device="cuda", dtype=torch.bfloat16)
    n = torch.empty(0, dtype=torch.long, device="cuda")
    logp, ent, lse = vocab.head_fwd(e, w, n, want_entropy=True)
    assert logp.numel() == ent.numel() == lse.numel() == 0
    dx, dw = vocab.head_bwd(e, w, n, lse, torch.empty(0, device="cuda"))
    assert dx.shape == (0, 16) and (dw == 0).all()
    kept = torch.ones_like(w)
    vocab.head_bwd(e, w, n, lse, torch.empty(0, device="cuda"), dw=kept, accumulate=True)
    assert (kept == 1).all()
    lse4 = torch.zeros(4, device="cuda")
    bad = [lambda: vocab.head_fwd(x.float(), w, y), lambda: vocab.head_fwd(x, w[:, :8], y),
           lambda: vocab.head_fwd(x, w, y[:3]), lambda: vocab.head_fwd(x, w, y.int()),
           lambda: vocab.head_fwd(x, w, y, 0.0), lambda: vocab.head_fwd(x, w, y, float("nan")),
           lambda: vocab.head_fwd(x[:, :12], w[:, :12], y), lambda: vocab.head_fwd(x.t(), w[:, :4], None),
           lambda: vocab.head_fwd(x[:, 4:12], w[:, 4:12], y), lambda: vocab.head_fwd(x, w.cpu(), y),
           lambda: vocab.head_fwd(x, w[:0], y),
           lambda: vocab.head_bwd(x, w, y, lse4[:2], coef), lambda: vocab.head_bwd(x, w, y, lse4, coef.half()),
           lambda: vocab.head_bwd(x, w, y, lse4, coef, accumulate=True),
           lambda: vocab.head_bwd(x, w, y, lse4, coef, piece=-1),
           lambda: vocab.head_bwd(x, w, y, lse4, coef, dw=torch.empty(31, 16, device="cuda")),
           lambda: vocab.head_bwd(x, w, y, lse4, coef, dx=torch.empty(4, 16, device="cuda"))]
    for f in bad:
        with pytest.raises((RuntimeError, ValueError)):
            f()


# ------------------------------------------------------------------ embedding
def _ids(T, V, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = torch.exp(torch.rand(T, generator=g, device="cuda") * math.log(V)).long().clamp_(1, V) - 1
    return r


EMBED = [(0, 8, 8), (1, 1, 8), (5, 3, 16), (33, 4, 264), (64, 1000, 256), (4096, 50, 128), (4097, 32000, 256),
         (10001, 100, 1032), (20000, 151936, 64)]


@pytest.mark.parametrize("T,V,H", EMBED)
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_embed_grad(T, V, H, dt):
    g = torch.Generator(device="cuda").manual_seed(T + V)
    ids = _ids(T, V)
    if T > 4:
        ids[2], ids[4] = -1, V
    dy = torch.randn(T, H + 8, generator=g, device="cuda").bfloat16()[:, :H]
    ok = (ids >= 0) & (ids < V)
    want, mag = torch.zeros(V, H, dtype=F8, device="cuda"), torch.zeros(V, H, dtype=F8, device="cuda")
    want.index_put_((ids[ok],), dy[ok].to(F8), accumulate=True)
    mag.index_put_((ids[ok],), dy[ok].to(F8).abs(), accumulate=True)
    count = torch.zeros(V, dtype=F8, device="cuda").index_put_((ids[ok],), torch.ones((), dtype=F8, device="cuda"), accumulate=True)
    unit = 2.0 ** -24 if dt == torch.float32 else 2.0 ** -8
    # an fp32 sum of n terms is off by at most n roundings of its magnitudes
    tol = (count[:, None] + 2) * 2.0 ** -24 * mag
    for scale in (1.0, 3.7):
        got = vocab.embed_grad(ids, dy, torch.full((V, H), float("nan"), device="cuda", dtype=dt), scale, accumulate=False)
        assert ((got.to(F8) - scale * want).abs() <= 1.001 * scale * (tol + unit * want.abs()) + 1e-30).all()
        base = torch.randn(V, H, generator=g, device="cuda").to(dt)
        acc = vocab.embed_grad(ids, dy, base.clone(), scale)
        assert ((acc.to(F8) - base.to(F8) - scale * want).abs()
                <= 1.001 * (scale * tol + 2 * unit * (base.to(F8).abs() + scale * mag)) + 1e-30).all()
        assert torch.equal(acc[count == 0], base[count == 0])
    again = vocab.embed_grad(ids, dy.clone(), torch.empty(V, H, device="cuda", dtype=dt), 3.7, accumulate=False)
    assert torch.equal(again, got)                                   # equal calls, equal bits


@pytest.mark.parametrize("T,V,H", EMBED)
def test_embed_lookup(T, V, H):
    g = torch.Generator(device="cuda").manual_seed(T)
    table = torch.randn(V, H + 16, generator=g, device="cuda").bfloat16()[:, 8:8 + H]
    ids = _ids(T, V)
    if T > 4:
        ids[2], ids[4] = -5, V + 3
    ok = (ids >= 0) & (ids < V)
    for scale in (1.0, 0.3):
        got = vocab.embed(ids, table, scale)
        want = torch.where(ok[:, None], table[torch.where(ok, ids, 0)].float() * scale, torch.zeros((), device="cuda")).bfloat16()
        assert torch.equal(got, want)
        into = torch.full((T, H), 5.0, device="cuda", dtype=torch.bfloat16)
        assert torch.equal(vocab.embed(ids, table, scale, out=into), want) and torch.equal(into, want)


def test_embed_grad_of_one_token_everywhere():
    """A single id: every chunk is one segment; and its neighbours stay zero."""
    for T in (1, 31, 32, 33, 255, 256, 257, 1024, 1025, 5000):
        dy = torch.randn(T, 264, device="cuda").bfloat16()
        ids = torch.full((T,), 2, dtype=torch.long, device="cuda")
        got = vocab.embed_grad(ids, dy, torch.full((5, 264), float("nan"), device="cuda"), accumulate=False)
        want = dy.to(F8).sum(0)
        assert ((got[2].to(F8) - want).abs() <= (T + 2) * 2.0 ** -24 * dy.to(F8).abs().sum(0)).all()
        assert (got[[0, 1, 3, 4]] == 0).all()
        ids = torch.full((T,), 9, dtype=torch.long, device="cuda")          # none in the table
        assert (vocab.embed_grad(ids, dy, torch.full((5, 264), 1.0, device="cuda"), accumulate=False) == 0).all()


def _check_grad(ids, V, H, dt, seed=0):
    T = len(ids)
    g = torch.Generator(device="cuda").manual_seed(seed + T + H)
    dy = torch.randn(T, H, generator=g, device="cuda").bfloat16()
    ok = (ids >= 0) & (ids < V)
    want, mag = torch.zeros(V, H, dtype=F8, device="cuda"), torch.zeros(V, H, dtype=F8, device="cuda")
    want.index_put_((ids[ok],), dy[ok].to(F8), accumulate=True)
    mag.index_put_((ids[ok],), dy[ok].to(F8).abs(), accumulate=True)
    count = torch.bincount(ids[ok], minlength=V).to(F8)[:, None]
    unit = 2.0 ** -24 if dt == torch.float32 else 2.0 ** -8
    # an fp32 sum of n terms is off by at most n roundings of its magnitudes
    tol = (count + 2) * 2.0 ** -24 * mag
    got = vocab.embed_grad(ids, dy, torch.full((V, H), float("nan"), device="cuda", dtype=dt), accumulate=False)
    assert ((got.to(F8) - want).abs() <= 1.001 * (tol + unit * want.abs()) + 1e-30).all()
    base = torch.randn(V, H, generator=g, device="cuda").to(dt)
    acc = vocab.embed_grad(ids, dy, base.clone())
    assert ((acc.to(F8) - base.to(F8) - want).abs() <= 1.001 * (tol + 2 * unit * (base.to(F8).abs() + mag)) + 1e-30).all()
    again = vocab.embed_grad(ids, dy, torch.empty(V, H, device="cuda", dtype=dt), accumulate=False)
    assert torch.equal(again, got)


# widths whose last 1024 columns (128 threads) leave threads of the block without columns, and their neighbours
@pytest.mark.parametrize("H", [8, 16, 24, 32, 40, 48, 1024, 1032, 1040, 1064, 1072, 2056])
@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
def test_embed_grad_of_few_tokens_with_long_runs(H, dt):
    """Runs that begin inside four sorted positions and end several such groups later."""
    for runs in ([6, 14, 3], [1, 13], [2, 3, 9, 1, 17], [5, 40, 1, 1, 30, 7], [3, 200, 53], [64, 65, 66, 61]):
        ids = torch.repeat_interleave(torch.arange(len(runs), device="cuda"), torch.tensor(runs, device="cuda"))
        ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(H)).cuda()]
        _check_grad(ids, len(runs) + 2, H, dt)
        _check_grad(ids, len(runs) - 1, H, dt)              # the last run lies outside the table
    for T in (20, 100, 255, 256):
        _check_grad(_ids(T, 1000, T), 1000, H, dt)


@pytest.mark.parametrize("H,run", [(264, 4200), (512, 2300), (1024, 4300), (1024, 9000)])
def test_embed_grad_of_a_long_run_before_others(H, run):
    """One id on more positions than a block of threads looks at in one turn, and
    many others behind it: its sum takes its own parts only, and repeats."""
    g = torch.Generator(device="cuda").manual_seed(run)
    ids = torch.cat([torch.full((run,), 3, dtype=torch.long, device="cuda"),
                     torch.randint(0, 3, (700,), generator=g, device="cuda"),
                     torch.randint(4, 500, (6000,), generator=g, device="cuda")])
    ids = ids[torch.randperm(len(ids), generator=g, device="cuda")]
    for seed in range(8):
        _check_grad(ids, 500, H, torch.float32, seed)


def test_embed_grad_keeps_rows_apart():
    """inf and NaN stay in the rows of their own tokens."""
    T, V, H = 300, 40, 64
    ids = torch.arange(T, device="cuda") % V
    dy = torch.ones(T, H, device="cuda").bfloat16()
    dy[7] = float("nan")
    dy[9] = float("inf")
    out = vocab.embed_grad(ids, dy, torch.empty(V, H, device="cuda"), accumulate=False)
    assert torch.isnan(out[7]).all() and torch.isinf(out[9]).all()
    assert torch.isfinite(out[10:]).all() and torch.isfinite(out[:7]).all()


def test_embed_refusals():
    ids = torch.zeros(4, dtype=torch.long, device="cuda")
    dy = torch.zeros(4, 16, device="cuda", dtype=torch.bfloat16)
    tab = torch.zeros(8, 16, device="cuda", dtype=torch.bfloat16)
    for f in (lambda: vocab.embed(ids.int(), tab), lambda: vocab.embed(ids, tab.float()),
              lambda: vocab.embed(ids, tab[:, :12]), lambda: vocab.embed(ids.cpu(), tab),
              lambda: vocab.embed_grad(ids[:3], dy, tab), lambda: vocab.embed_grad(ids, dy.float(), tab),
              lambda: vocab.embed_grad(ids, dy, tab[:, :8]), lambda: vocab.embed_grad(ids, dy, tab.half()),
              lambda: vocab.embed_grad(ids, dy, tab.cpu()), lambda: vocab.embed_grad(ids, dy.t(), tab)):
        with pytest.raises(RuntimeError):
            f()
