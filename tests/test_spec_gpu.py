"""Draft verification on the GPU, against the 64-bit definition."""
import math

import pytest
import torch
from test_paged_cpu import check_verify, verify_case

from kore_b200.ops import spec

pytestmark = pytest.mark.gpu


def _i(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("V", [1, 2, 7, 8, 9, 100, 4097, 50257, 151936])
@pytest.mark.parametrize("tau,probs", [(1.0, False), (0.7, True), (0.0, False), (1.3, False), (1.0, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_verify(V, tau, probs, dtype):
    lens = [4, 1, 0, 9, 2, 5] if V < 10 ** 5 else [3, 1, 2]
    check_verify(verify_case(V, V, lens, probs=probs, dtype=dtype, device="cuda"), tau)


@pytest.mark.parametrize("lens", [[1], [40], [8, 9, 16, 17, 1], [0, 0], [2] * 200])
def test_verify_lengths(lens):
    check_verify(verify_case(2, 1000, lens, device="cuda"), 1.0)


def test_long_drafts_are_accepted_past_one_group_of_rows():
    z, tokens, qs, u, _ = verify_case(3, 500, [40, 25], device="cuda")
    z[torch.arange(64), tokens[1:]] = 30.0                     # nearly certain
    v = check_verify((z, tokens, qs, u, None), 1.0)
    assert v.accepted.tolist() == [39, 24]


def test_ties_go_to_the_lowest_index():
    V = 5000
    z = torch.zeros(3, V, device="cuda")
    z[:, [77, 1234, 4999]] = 2.0
    tokens = torch.tensor([0, 77, 1234], device="cuda")
    v = check_verify((z, tokens, _i([0, 3]), torch.rand(3, 2, device="cuda"), None), 0.0)
    assert v.accepted.tolist() == [1] and v.next.tolist() == [77]


def test_draw_hits_every_border():
    """Four equal tokens among masked ones: u at and beside the borders of the running sum."""
    V = 3001
    z = torch.full((8, V), -math.inf, device="cuda")
    z[:, [0, 1500, 1501, 3000]] = 1.0
    u = torch.tensor([0.0, 0.25, 0.2499, 0.5, 0.7499, 0.75, 0.9999999, 0.5001], device="cuda")
    u = torch.stack([u.flip(0), u], 1)
    v = spec.verify(z, torch.zeros(8, dtype=torch.long, device="cuda"), _i(list(range(9))), u)
    assert v.next.tolist() == [0, 1500, 0, 1501, 1501, 3000, 3000, 1501]
    assert torch.allclose(v.logp, torch.full((8,), math.log(0.25), device="cuda"))


def test_rows_without_a_distribution():
    V = 300
    z, tokens, _, u, _ = verify_case(4, V, [15], device="cuda")
    z[0] = -math.inf
    z[4, 17] = math.nan
    z[6, 299] = math.inf
    z[9, :] = -math.inf
    z[9, 5] = 2.0                                              # one token left
    tokens[10] = 5
    tokens[1:4] = torch.tensor([-1, V, 10 ** 12], device="cuda")     # drafts outside the vocabulary
    qs = _i([0, 2, 4, 6, 8, 9, 12, 15])
    for tau in (1.0, 0.0):
        v = check_verify((z, tokens, qs, u, None), tau)
        assert v.next.tolist()[0] == -1 and v.accepted.tolist()[0] == 0


def test_nothing_left_over_draws_from_the_target():
    """A rejected draft where q covers p everywhere (q is no distribution): the next token is drawn from p."""
    V = 64
    z, tokens, qs, u, _ = verify_case(5, V, [2, 2], device="cuda")
    q = torch.full((4, V), 1.0, device="cuda")
    u[:, 0] = 1 - 2.0 ** -24
    v = check_verify((z, tokens, qs, u, q), 1.0)
    assert v.accepted.tolist() == [0, 0]


def test_strided_rows():
    z, tokens, qs, u, q = verify_case(6, 1001, [3, 4, 1], probs=True, dtype=torch.bfloat16, device="cuda")
    zz = torch.full((8, 1013), math.nan, dtype=torch.bfloat16, device="cuda")
    zz[:, 3:1004] = z
    qq = torch.full((8, 1007), math.nan, device="cuda")
    qq[:, 1:1002] = q
    check_verify((zz[:, 3:1004], tokens, qs, u, qq[:, 1:1002]), 0.8)


def test_rows_behind_the_last_sequence():
    z, tokens, qs, u, _ = verify_case(7, 100, [3, 4, 2], device="cuda")
    z[7:] = math.nan
    check_verify((z, tokens, qs[:3].contiguous(), u, None), 1.0)


def test_captured_and_on_two_streams():
    cases = [verify_case(s, 9000, [3, 4, 1, 5], probs=s == 1, device="cuda") for s in (1, 2)]
    want = [check_verify(c, 0.9) for c in cases]
    torch.cuda.synchronize()
    graphs = []
    for z, t, qs, u, q in cases:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, spec.verify(z, t, qs, u, 0.9, draft_probs=q)))
    for _ in range(3):
        for g, _ in graphs:
            g.replay()
    streams, outs = [torch.cuda.Stream() for _ in cases], []
    for _ in range(10):
        for s, (z, t, qs, u, q), w in zip(streams, cases, want):
            with torch.cuda.stream(s):
                outs.append((spec.verify(z, t, qs, u, 0.9, draft_probs=q), w))
    torch.cuda.synchronize()
    outs += [(got, w) for (_, got), w in zip(graphs, want)]
    for got, w in outs:
        assert torch.equal(got.accepted, w.accepted) and torch.equal(got.next, w.next) and torch.equal(got.logp, w.logp)


def test_distribution():
    V, n = 6, 40000
    g = torch.Generator(device="cuda").manual_seed(0)
    z, q = torch.randn(V, generator=g, device="cuda"), torch.softmax(torch.randn(V, generator=g, device="cuda"), -1)
    p = torch.softmax(z.double(), -1)
    for probs in (q, None):
        draft = torch.multinomial(q, n, replacement=True, generator=g) if probs is not None else torch.full((n,), 2, device="cuda")
        tokens = torch.stack([torch.zeros_like(draft), draft], 1).reshape(-1)
        v = spec.verify(z.repeat(2 * n, 1), tokens, _i(list(range(0, 2 * n + 1, 2))), torch.rand(2 * n, 2, generator=g, device="cuda"),
                        draft_probs=None if probs is None else probs.repeat(2 * n, 1))
        first = torch.where(v.accepted > 0, draft, v.next)
        freq = torch.bincount(first, minlength=V).double() / n
        assert (freq - p).abs().max().item() < 5 * math.sqrt(0.25 / n)         # five standard deviations


def test_refusals():
    z, tokens, qs, u, q = verify_case(8, 100, [2, 3], probs=True, device="cuda")
    for bad in (dict(logits=z.half()), dict(logits=z.t()), dict(logits=z[0]), dict(tokens=tokens[:4]), dict(tokens=tokens.int()),
                dict(q_start=qs.long()), dict(u=u[:, :1]), dict(u=u.double()), dict(draft_probs=q.bfloat16()),
                dict(draft_probs=q[:, :99]), dict(tokens=tokens.cpu()), dict(logits=torch.empty(5, 0, device="cuda")),
                dict(logits=torch.empty(1, 1, device="cuda").expand(5, 1 << 21))):
        a = dict(logits=z, tokens=tokens, q_start=qs, u=u, draft_probs=q)
        a.update(bad)
        with pytest.raises(RuntimeError):
            spec.verify(a["logits"], a["tokens"], a["q_start"], a["u"], 1.0, draft_probs=a["draft_probs"])
    with pytest.raises(ValueError):
        spec.verify(z, tokens, qs, u, -0.5)


def test_sequences_without_any_rows():
    z, tokens, _, u, _ = verify_case(9, 50, [2], device="cuda")
    v = spec.verify(z[:0], tokens[:0], _i([0, 0, 0]), u[:0])
    assert v.accepted.tolist() == [0, 0] and v.next.tolist() == [-1, -1] and v.logp.numel() == 0


def test_no_sequences():
    z, tokens, qs, u, _ = verify_case(9, 50, [2], device="cuda")
    v = spec.verify(z, tokens, qs[:1].contiguous(), u)
    assert v.accepted.numel() == 0 and v.next.numel() == 0 and (v.logp == 0).all()
