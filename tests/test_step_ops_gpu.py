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
