"""The training step with the vocabulary, balance and 8-bit checkpoint operators
on a B200: gradients against the plain step's, and a short training run."""
import pytest
import torch

from kore_b200 import ops
from kore_b200.engine.qwen3_engine import Batch, Qwen3Engine
from kore_b200.engine.trainer import CausalLMTrainer
from kore_b200.models import Qwen3Config, Qwen3Weights
from kore_b200.parallel.dist import get_context

pytestmark = pytest.mark.gpu


def _cfg(moe=False, tied=False):
    kw = dict(vocab_size=2048, hidden_size=512, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=4,
              num_key_value_heads=2, head_dim=128, max_position_embeddings=1024, tie_word_embeddings=tied)
    if moe:
        kw.update(model_type="qwen3_moe", num_experts=8, num_experts_per_tok=2, moe_intermediate_size=256)
    return Qwen3Config(**kw)


def _batch(cfg):
    g = torch.Generator().manual_seed(0)
    seqs = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (301, 77, 130)]
    return Batch.from_sequences(seqs, [torch.arange(len(s)) > 40 for s in seqs], device="cuda")


def _grads(cfg, b, keep=0, **kw):
    w = Qwen3Weights(cfg, device=torch.device("cuda"), dtype=torch.bfloat16, seed=3)
    eng = Qwen3Engine(w, **kw)
    eng.keep_layers = keep
    eng.zero_grad()
    out = eng.forward_backward(b, coef=eng.sft_coef(b))
    assert ops.check_device_error() == 0
    return out, [g.float().clone() for g in eng.grads], eng


@pytest.mark.parametrize("moe,tied", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("kw,keep,tol", [
    # bf16 logits and gradients against fp32 logits: a few roundings of 2^-8
    (dict(head="pieces", embed_grad="sorted"), 0, 0.02),
    # values of the contexts off by about 0.5%
    (dict(act8=True), 0, 0.04), (dict(act8=True), 2, 0.04),
    (dict(head="pieces", embed_grad="sorted", act8=True), 3, 0.04)])
def test_gradients_stay_near(moe, tied, kw, keep, tol):
    cfg = _cfg(moe, tied)
    b = _batch(cfg)
    a, ga, _ = _grads(cfg, b)
    c, gc, _ = _grads(cfg, b, keep, **kw)
    assert abs(float(a["loss"]) - float(c["loss"])) <= 0.01 * abs(float(a["loss"]))
    for u, (x, y) in enumerate(zip(ga, gc)):
        assert (x - y).norm() <= tol * x.norm(), (u, float((x - y).norm() / x.norm()))


def test_sorted_embedding_gradient_repeats_bit_for_bit():
    cfg = _cfg()
    b = _batch(cfg)
    kw = dict(head="pieces", embed_grad="sorted")
    w = Qwen3Weights(cfg, device=torch.device("cuda"), dtype=torch.bfloat16, seed=3)
    eng = Qwen3Engine(w, **kw)
    dx = torch.randn(b.num_tokens, cfg.hidden_size, device="cuda").bfloat16()
    from kore_b200.ops import vocab
    first = vocab.embed_grad(b.ids, dx, eng.grad_views(0)["embed"].clone(), accumulate=False)
    for _ in range(3):
        assert torch.equal(vocab.embed_grad(b.ids, dx, torch.empty_like(first), accumulate=False), first)


@pytest.mark.parametrize("moe", [False, True])
def test_training_with_all_of_them(moe):
    cfg = _cfg(moe)
    tr = CausalLMTrainer(cfg, get_context(), lr=2e-3, seed=1, head="pieces", embed_grad="sorted", act8=True,
                         router_aux=True)
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, cfg.vocab_size, (4, 128), generator=g)
    losses = [tr.train_step(ids) for _ in range(6)]
    assert losses[-1] < losses[0] - 0.2
    assert ops.check_device_error() == 0
    if moe:
        assert float(tr.eng.aux_loss) > 0
        # 4 micro-batches of 128 tokens, 2 choices each, in every layer
        assert all(int(c.sum()) == 4 * 128 * 2 for c in tr.eng.expert_counts.values())
        assert len(tr.eng.expert_counts) == 3


@pytest.mark.parametrize("T,E,k", [(0, 8, 2), (1, 8, 8), (77, 60, 4), (513, 128, 8), (40, 256, 16)])
@pytest.mark.parametrize("norm", [True, False])
def test_route_with_given_choices(T, E, k, norm):
    from kore_b200.ops import moe
    logits = torch.randn(T, E, device="cuda", generator=torch.Generator(device="cuda").manual_seed(E))
    probs, idx, w = moe.route(logits, k, norm)
    p2, i2, w2 = moe.route(logits, k, norm, idx=idx.clone())
    assert torch.equal(p2, probs) and torch.equal(i2, idx) and torch.equal(w2, w)
    other = torch.argsort(torch.rand(T, E, device="cuda"), -1)[:, :k].int().contiguous()
    _, i3, w3 = moe.route(logits, k, norm, idx=other)
    want = torch.softmax(logits.double(), -1).gather(1, other.long())
    if norm:
        want = want / want.sum(-1, keepdim=True)
    assert torch.equal(i3, other)
    # the exponential is off by up to 2 + |x| / 2 units of 2^-24, twice (entry and sum)
    assert ((w3.double() - want).abs() <= 1e-5 * want).all()
    if T:
        none = other.clone()
        none[:, 0] = -1 if T % 2 else E
        _, _, w4 = moe.route(logits, k, False, idx=none)
        assert (w4[:, 0] == 0).all()
        for bad in (other[:, :k - 1], other.long(), other[:T - 1] if T > 1 else other.float()):
            with pytest.raises(RuntimeError):
                moe.route(logits, k, norm, idx=bad)


def test_act8_backward_takes_the_forwards_routing(monkeypatch):
    from kore_b200.ops import moe
    kw = dict(vocab_size=2048, hidden_size=512, intermediate_size=1024, num_hidden_layers=3, num_attention_heads=4,
              num_key_value_heads=2, head_dim=128, max_position_embeddings=1024, model_type="qwen3_moe",
              num_experts=64, num_experts_per_tok=8, moe_intermediate_size=128)
    cfg = Qwen3Config(**kw)
    b = _batch(cfg)
    seen = []
    real = moe.plan
    monkeypatch.setattr(moe, "plan", lambda idx, *a, **k: (seen.append(idx.clone()), real(idx, *a, **k))[1])
    a, ga, plain = _grads(cfg, b, router_aux_coef=0.1)
    c, gc, held = _grads(cfg, b, router_aux_coef=0.1, act8=True)
    assert len(seen) == 12
    for f, r in zip(seen[6:9], seen[9:][::-1]):
        assert torch.equal(f, r)
    assert torch.equal(a["logp"], c["logp"])
    for u in plain.expert_counts:
        assert torch.equal(held.expert_counts[u], plain.expert_counts[u])
    for u, (x, y) in enumerate(zip(ga, gc)):
        assert (x - y).norm() <= 0.04 * x.norm(), (u, float((x - y).norm() / x.norm()))
