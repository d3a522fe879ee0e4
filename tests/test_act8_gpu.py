"""8-bit activation checkpoints: the native kernels against the definition."""
import pytest
import torch

from kore_b200.ops import act8

pytestmark = pytest.mark.gpu
F8 = torch.float64


def _x(T, H, seed=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed + T + H)
    col = torch.exp(1.5 * torch.randn(1, H + pad, generator=g, device="cuda"))
    x = (torch.randn(T, H + pad, generator=g, device="cuda") * col).bfloat16()
    return x[:, :H]


def _held(x):
    """The bytes and scales of the definition, computed on the CPU in IEEE fp32."""
    a = act8.empty(x.shape[0], x.shape[1], "cpu")
    act8._quantise(x.cpu(), a)
    return a


def _values(a):
    return a.q.to(F8) * a.s.to(F8).repeat_interleave(128, 1)[:, :a.q.shape[1]]


SHAPES = [(0, 64), (1, 8), (1, 128), (3, 136), (37, 256), (5, 1000), (130, 2048), (9, 5120), (2, 8192), (257, 7168)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("pad", [0, 24])
def test_save_and_load(T, H, pad):
    x = _x(T, H, pad=pad)
    a = act8.save(x)
    want = _held(x)
    assert torch.equal(a.q.cpu(), want.q) and torch.equal(a.s.cpu(), want.s)
    back = act8.load(a)
    assert torch.equal(back.cpu(), (want.q.float() * want.s.repeat_interleave(128, 1)[:, :H]).bfloat16())
    wide = torch.full((T, H + 8), 7.0, device="cuda", dtype=torch.bfloat16)
    act8.load(a, out=wide[:, :H])
    assert torch.equal(wide[:, :H], back) and (wide[:, H:] == 7.0).all()
    into = act8.empty(T, H, "cuda")
    again = act8.save(x, out=into)
    assert torch.equal(into.q, a.q) and torch.equal(into.s, a.s) and again.q.data_ptr() == into.q.data_ptr()
    if T:
        v, xd = _values(a), x.to(F8)
        amax = torch.nn.functional.pad(xd.abs(), (0, -H % 128)).view(T, -1, 128).amax(-1).repeat_interleave(128, 1)[:, :H]
        # half a step, and the roundings of the quotient and of the scale
        assert ((v - xd).abs() <= amax / 254 * (1 + 1e-4)).all()


def test_blocks_without_a_scale():
    x = torch.zeros(6, 264, device="cuda", dtype=torch.bfloat16)
    x[1, 3] = 1e-38                       # denormal range
    x[2, 130] = float("inf")
    x[3, 5] = float("nan")
    x[4, 260] = float("-inf")
    x[5] = 3.3e38
    x[2, 0] = 2.0
    a = act8.save(x)
    v = act8.load(a)
    assert (v[0] == 0).all() and (v[1] == 0).all()
    assert torch.isnan(v[2, 128:256]).all() and v[2, 0] == 2.0 and (v[2, 1:128] == 0).all()
    assert torch.isnan(v[3, :128]).all() and (v[3, 128:] == 0).all()
    assert torch.isnan(v[4, 256:]).all() and (v[4, :256] == 0).all()
    assert torch.isfinite(v[5]).all() and ((v[5].float() / x[5].float() - 1).abs() < 2.0 ** -7).all()


@pytest.mark.parametrize("T,H", SHAPES)
def test_rmsnorm_save_and_load(T, H):
    eps = 1e-6
    x = _x(T, H, seed=1, pad=16)
    w = (1 + 0.1 * torch.randn(H, generator=torch.Generator(device="cuda").manual_seed(H), device="cuda")).bfloat16()
    hn, rstd, a = act8.rmsnorm_save(x, w, eps)
    plain = act8.save(x)
    assert torch.equal(a.q, plain.q) and torch.equal(a.s, plain.s)

    def norm(v):
        r = (v.square().mean(-1) + eps).rsqrt()
        return v * r[:, None] * w.to(F8), r

    # rstd: an fp32 sum of squares and an approximate root; hn: rounded to bf16 once
    want, r = norm(x.to(F8))
    assert torch.allclose(rstd.to(F8), r, rtol=1e-5, atol=0)
    assert ((hn.to(F8) - want).abs() <= (2.0 ** -8 * 1.01 + 2e-5) * want.abs()).all()
    x8, hn8, rstd8 = act8.rmsnorm_load(a, w, eps)
    want, r = norm(_values(a))
    assert torch.equal(x8, act8.load(a))
    assert torch.allclose(rstd8.to(F8), r, rtol=1e-5, atol=0)
    assert ((hn8.to(F8) - want).abs() <= (2.0 ** -8 * 1.01 + 2e-5) * want.abs()).all()


@pytest.mark.parametrize("T,F", [(0, 8), (1, 8), (3, 64), (7, 128), (33, 256), (21, 200), (130, 2048), (5, 17408),
                                 (3, 5000), (9, 11112), (4, 15008), (2, 20488), (40, 1368)])
@pytest.mark.parametrize("pad", [0, 8])
def test_swiglu_save_and_backward(T, F, pad):
    g = torch.Generator(device="cuda").manual_seed(F)
    gu = (3 * torch.randn(T, 2 * F + pad, generator=g, device="cuda")).bfloat16()[:, :2 * F]
    dout = torch.randn(T, F + pad, generator=g, device="cuda").bfloat16()[:, :F]
    a, held = act8.swiglu_save(gu)
    plain = act8.save(gu)
    assert torch.equal(held.q, plain.q) and torch.equal(held.s, plain.s)
    silu = torch.nn.functional.silu
    want = silu(gu[:, :F].to(F8)) * gu[:, F:].to(F8)
    # one bf16 rounding, and exp / reciprocal approximations of a few units in the last fp32 place
    rel = 2.0 ** -8 * 1.01 + 1e-5
    assert ((a.to(F8) - want).abs() <= rel * want.abs() + 1e-37).all()
    dgu, a8 = act8.swiglu_bwd(dout, held)
    v = _values(held).requires_grad_(True)
    act = silu(v[:, :F]) * v[:, F:]
    want, = torch.autograd.grad(act, v, dout.to(F8))
    assert ((a8.to(F8) - act.detach()).abs() <= rel * act.detach().abs() + 1e-37).all()
    # dgate's factor 1 + gate (1 - sg) cancels for negative gates: fp32 roundings of its terms
    gate, up = v[:, :F].detach(), v[:, F:].detach()
    sg = torch.sigmoid(gate)
    terms = dout.to(F8).abs() * up.abs() * sg * (1 + gate.abs())
    tol = rel * want.abs()
    tol[:, :F] += 1e-6 * terms
    assert ((dgu.to(F8) - want).abs() <= tol + 1e-37).all()


def test_swiglu_backward_is_the_gradient():
    g = torch.Generator(device="cuda").manual_seed(3)
    gu = torch.randn(9, 512, generator=g, device="cuda").bfloat16()
    dout = torch.randn(9, 256, generator=g, device="cuda").bfloat16()
    _, held = act8.swiglu_save(gu)
    dgu, _ = act8.swiglu_bwd(dout, held)
    v, h = _values(held), 1e-5

    def f(v):
        return (torch.nn.functional.silu(v[:, :256]) * v[:, 256:] * dout.to(F8)).sum()

    for _ in range(4):
        d = torch.randn(v.shape, generator=g, device="cuda", dtype=F8)
        num = (f(v + h * d) - f(v - h * d)) / (2 * h)
        assert abs(num - (dgu.to(F8) * d).sum()) <= 6 * 2.0 ** -9 * (dgu.to(F8) * d).norm() + 1e-6


def test_other_stream():
    x = _x(1000, 512)
    want = act8.load(act8.save(x))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = act8.load(act8.save(x))
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)


def test_refusals():
    x = _x(4, 64)
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16)
    a = act8.save(x)
    big = torch.zeros(2, 8200, device="cuda", dtype=torch.bfloat16)
    short = act8.Act8(a.q, a.s[:3])
    for f in (lambda: act8.save(x.float()), lambda: act8.save(x[:, :12]), lambda: act8.save(x.t()),
              lambda: act8.save(x[:, 4:20]), lambda: act8.load(short), lambda: act8.load(a, dtype=torch.float32),
              lambda: act8.save(x, out=short), lambda: act8.load(act8.Act8(a.q.float(), a.s)),
              lambda: act8.load(a, out=torch.empty(4, 72, device="cuda", dtype=torch.bfloat16)),
              lambda: act8.rmsnorm_save(x, w[:32], 1e-6), lambda: act8.rmsnorm_save(x, w.float(), 1e-6),
              lambda: act8.rmsnorm_save(big, torch.ones(8200, device="cuda", dtype=torch.bfloat16), 1e-6),
              lambda: act8.rmsnorm_load(a, w[:32], 1e-6), lambda: act8.swiglu_save(x[:, :24]),
              lambda: act8.swiglu_bwd(x, a), lambda: act8.swiglu_bwd(x[:2, :32], a)):
        with pytest.raises((RuntimeError, ValueError)):
            f()
