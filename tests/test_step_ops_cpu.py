"""The training step with the vocabulary, balance and 8-bit checkpoint operators
switched on, against the step without them (fp32 on the CPU)."""
import pytest
import torch

from kore_b200.engine.qwen3_engine import Batch, Qwen3Engine
from kore_b200.engine.trainer import CausalLMTrainer
from kore_b200.models import Qwen3Config, Qwen3Weights
from kore_b200.parallel.dist import get_context
from kore_b200.policy.configs import SFTConfig, step_kwargs


def _cfg(moe=False, tied=False):
    kw = dict(vocab_size=211, hidden_size=64, intermediate_size=128, num_hidden_layers=3, num_attention_heads=4,
              num_key_value_heads=2, head_dim=16, max_position_embeddings=128, tie_word_embeddings=tied)
    if moe:
        kw.update(model_type="qwen3_moe", num_experts=4, num_experts_per_tok=2, moe_intermediate_size=32)
    return Qwen3Config(**kw)


def _engine(cfg, **kw):
    w = Qwen3Weights(cfg, device=torch.device("cpu"), dtype=torch.float32, seed=3)
    return Qwen3Engine(w, **kw)


def _batch(cfg):
    g = torch.Generator().manual_seed(0)
    seqs = [torch.randint(0, cfg.vocab_size, (n,), generator=g) for n in (21, 9)]
    masks = [torch.arange(len(s)) > 4 for s in seqs]
    return Batch.from_sequences(seqs, masks)


def _step(eng, b, coef_fn=None):
    eng.zero_grad()
    out = eng.forward_backward(b, coef_fn=coef_fn) if coef_fn else eng.forward_backward(b, coef=eng.sft_coef(b))
    return out, [g.clone() for g in eng.grads]


@pytest.mark.parametrize("moe", [False, True])
@pytest.mark.parametrize("tied", [False, True])
def test_pieces_and_sorted_give_the_same_step(moe, tied):
    cfg = _cfg(moe, tied)
    b = _batch(cfg)
    plain, other = _engine(cfg), _engine(cfg, head="pieces", embed_grad="sorted")
    for fn in (None, lambda lp: (-0.1 * (1 + lp.exp()), lp.sum())):
        a, ga = _step(plain, b, fn)
        c, gc = _step(other, b, fn)
        assert torch.allclose(a["logp"], c["logp"], atol=1e-5) and torch.allclose(a["loss"], c["loss"], rtol=1e-5)
        for x, y in zip(ga, gc):
            assert torch.allclose(x, y, rtol=1e-4, atol=1e-6)
    # a second micro-batch adds
    other.forward_backward(b, coef=other.sft_coef(b))
    plain.forward_backward(b, coef=plain.sft_coef(b))
    for x, y in zip(plain.grads, other.grads):
        assert torch.allclose(x, y, rtol=1e-4, atol=1e-6)
    lp, ent = plain.token_logprobs(b, want_entropy=True)
    lp2, ent2 = other.token_logprobs(b, want_entropy=True)
    assert torch.allclose(lp, lp2, atol=1e-5) and torch.allclose(ent, ent2, atol=1e-4)


@pytest.mark.parametrize("moe", [False, True])
@pytest.mark.parametrize("keep", [0, 2])
def test_act8_gradients_stay_near(moe, keep):
    cfg = _cfg(moe)
    b = _batch(cfg)
    plain, held = _engine(cfg), _engine(cfg, act8=True)
    held.keep_layers = keep
    a, ga = _step(plain, b)
    c, gc = _step(held, b)
    assert torch.equal(a["logp"], c["logp"])                 # the forward pass is not touched
    for u, (x, y) in enumerate(zip(ga, gc)):
        # values are off by amax / 254 of their block (rms about 0.5% here)
        assert (x - y).norm() <= 0.03 * x.norm(), u
    assert held.activation_bytes_per_layer(1024) < plain.activation_bytes_per_layer(1024) / 4


def test_router_balance_gradient_by_differences():
    cfg = _cfg(moe=True)
    b = _batch(cfg)
    zero = torch.zeros(b.num_tokens)
    eng = _engine(cfg, router_aux_coef=0.5)
    eng.aux_scale = 0.25
    eng.zero_grad()
    eng.forward_backward(b, coef=zero)                        # only the balance loss has a gradient
    total = eng.aux_loss.clone()
    assert sorted(eng.expert_counts) == [1, 2, 3]
    assert all(int(c.sum()) == 2 * b.num_tokens for c in eng.expert_counts.values())
    last = 3                                                  # the last layer's router feeds nothing but its own loss
    grad = eng.grad_views(last)["router"].clone()
    g = torch.Generator().manual_seed(1)
    d = torch.randn(grad.shape, generator=g)
    d *= 1e-3 / d.norm()
    W = eng.w.views(last)["router"]
    vals = []
    for sign in (1, -1):
        W.add_(d, alpha=sign)
        eng.zero_grad()
        eng.forward_backward(b, coef=zero)
        vals.append(float(eng.aux_loss))
        W.add_(d, alpha=-sign)
    num, want = (vals[0] - vals[1]) / 2, float((grad * d).sum())
    assert float(total) > 0 and abs(num - want) <= 0.02 * abs(want) + 1e-7
    off = _engine(cfg)
    off.forward_backward(b, coef=zero)
    assert float(off.aux_loss) == 0 and off.expert_counts == {}


def test_trainer_runs_all_of_them_together():
    cfg = _cfg(moe=True)
    conf = SFTConfig(head="pieces", embed_grad="sorted", act8=True, router_aux=True)
    assert step_kwargs(SFTConfig()) == dict(head="chunks", embed_grad="atomic", act8=False, router_aux=False)
    tr = CausalLMTrainer(cfg, get_context(), lr=1e-2, dtype=torch.float32, seed=1, **step_kwargs(conf))
    assert tr.eng.router_aux_coef == cfg.router_aux_loss_coef
    g = torch.Generator().manual_seed(2)
    ids = torch.randint(0, cfg.vocab_size, (4, 16), generator=g)
    losses = [tr.train_step(ids) for _ in range(8)]
    assert losses[-1] < losses[0] and float(tr.eng.aux_loss) > 0
    seqs = [torch.randint(0, cfg.vocab_size, (n,), generator=g).tolist() for n in (9, 14, 5)]
    assert tr.train_step_sequences(seqs, [[1] * len(s) for s in seqs], micro_tokens=16) > 0
    assert tr.eng.aux_scale == 1 / 3                          # 9 + 14 and 14 + 5 are over 16: three micro-batches


def test_options_are_checked():
    cfg = _cfg()
    for kw in (dict(head="rows"), dict(embed_grad="hash"), dict(router_aux_coef=-1.0)):
        with pytest.raises(ValueError):
            _engine(cfg, **kw)


def _moe_weights(coef=0.5):
    cfg = _cfg(moe=True)
    cfg.router_aux_loss_coef = coef
    return cfg, Qwen3Weights(cfg, device=torch.device("cpu"), dtype=torch.float32, seed=3)


def _same_aux(runs):
    """Equal micro-batches: their mean is the balance loss of all of them at once."""
    (aux, grads), (aux2, grads2) = runs
    assert aux > 0 and abs(aux - aux2) <= 1e-5 * aux
    for a, b in zip(grads, grads2):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-6)


def test_balance_loss_weight_in_dpo():
    from kore_b200.policy.configs import DPOConfig
    from kore_b200.policy.dpo import DPOTrainer
    g = torch.Generator().manual_seed(5)
    cfg, _ = _moe_weights()
    ids = torch.randint(0, cfg.vocab_size, (30,), generator=g).tolist()
    pair = [(ids[:19], 9), (ids[:9] + ids[19:26], 9)]
    runs = []
    for micro in (4, 1):
        dt = DPOTrainer(DPOConfig(beta=0.1, learning_rate=1e-3, use_lora=False, bf16=False, micro_pairs=micro,
                                  router_aux=True), get_context(), _moe_weights()[1])
        dt.tr.opt.step = lambda *a, **k: None
        dt.step([pair] * 4)
        runs.append((float(dt.tr.eng.aux_loss), [x.clone() for x in dt.tr.eng.grads]))
    _same_aux(runs)


def test_balance_loss_weight_in_grpo():
    from kore_b200.env.base import SyntheticRewardEnv
    from kore_b200.policy.configs import GRPOConfig
    from kore_b200.policy.grpo import GRPOTrainer, TrainSample
    g = torch.Generator().manual_seed(6)
    cfg, _ = _moe_weights()
    ids = torch.randint(0, cfg.vocab_size, (24,), generator=g).tolist()
    runs = []
    for budget in (4096, 24):
        tr = GRPOTrainer(GRPOConfig(num_trajectories=4, num_turns=1, tasks_per_step=1, max_response_length=8,
                                    max_prompt_length=64, learning_rate=1e-3, bf16=False, total_steps=2,
                                    overlong_mask=False, pack_trajectories=False, router_aux=True),
                         weights=_moe_weights()[1],
                         env=SyntheticRewardEnv(seed=0, prompt_len=16, feedback_len=4, vocab_size=cfg.vocab_size),
                         rollout_kwargs=dict(num_pages=64, page_size=16, max_seq_len=128))
        tr.trainer.opt.step = lambda *a, **k: None
        samples = [TrainSample(list(ids), 8, ret=0.0, adv=0.5, old_logp=-5.0, ref_logp=-5.0) for _ in range(4)]
        assert len(list(tr._pack(tr._rows(samples), budget))) == (1 if budget == 4096 else 4)
        tr.update(samples, budget)
        runs.append((float(tr.trainer.eng.aux_loss), [x.clone() for x in tr.trainer.eng.grads]))
    _same_aux(runs)


def _wide_moe():
    cfg = Qwen3Config(vocab_size=211, hidden_size=128, intermediate_size=128, num_hidden_layers=3, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=32, max_position_embeddings=512, model_type="qwen3_moe",
                      num_experts=64, num_experts_per_tok=8, moe_intermediate_size=32)
    g = torch.Generator().manual_seed(8)
    return cfg, Batch.from_sequences([torch.randint(0, 211, (n,), generator=g) for n in (301, 99)])


def test_act8_backward_takes_the_forwards_routing(monkeypatch):
    """The 8-bit input moves some tokens over the edge between two experts; the
    backward, the counts and the balance loss follow the forward's choices."""
    from kore_b200.ops import moe
    cfg, b = _wide_moe()
    seen = []
    real = moe.plan
    monkeypatch.setattr(moe, "plan", lambda idx, *a, **k: (seen.append(idx.clone()), real(idx, *a, **k))[1])
    plain, held = _engine(cfg, router_aux_coef=0.1), _engine(cfg, router_aux_coef=0.1, act8=True)
    (_, ga), (_, gc) = _step(plain, b), _step(held, b)
    assert len(seen) == 12
    forward, backward = seen[6:9], seen[9:][::-1]
    for f, r, p in zip(forward, backward, seen[:3]):
        assert torch.equal(f, r) and torch.equal(f, p)
    assert sorted(held.expert_counts) == [1, 2, 3]
    for u in held.expert_counts:
        assert torch.equal(held.expert_counts[u], plain.expert_counts[u])
    assert torch.equal(held.aux_loss, plain.aux_loss)
    for u, (x, y) in enumerate(zip(ga, gc)):
        assert (x - y).norm() <= 0.03 * x.norm(), u


@pytest.mark.parametrize("norm", [True, False])
def test_route_with_given_choices(norm):
    from kore_b200.ops import moe
    logits = torch.randn(9, 12, generator=torch.Generator().manual_seed(4))
    probs, idx, w = moe.route(logits, 3, norm)
    same = moe.route(logits, 3, norm, idx=idx)
    assert all(torch.equal(a, b) for a, b in zip(same, (probs, idx, w)))
    other = (idx + 1) % 12
    p2, i2, w2 = moe.route(logits, 3, norm, idx=other)
    want = torch.softmax(logits.double(), -1).gather(1, other.long())
    if norm:
        want = want / want.sum(-1, keepdim=True)
    assert torch.equal(i2, other) and torch.equal(p2, probs) and torch.allclose(w2.double(), want, rtol=1e-5)


def test_reference_model_uses_the_policys_head():
    """Equal weights have equal log-probs: the frozen reference scores with the same head."""
    from kore_b200.env.base import SyntheticRewardEnv
    from kore_b200.policy.configs import DPOConfig, GRPOConfig
    from kore_b200.policy.dpo import DPOTrainer
    from kore_b200.policy.grpo import GRPOTrainer
    cfg = _cfg()
    b = _batch(cfg)
    for head in ("chunks", "pieces"):
        w = Qwen3Weights(cfg, device=torch.device("cpu"), dtype=torch.float32, seed=3)
        dt = DPOTrainer(DPOConfig(use_lora=False, bf16=False, head=head), get_context(), w.clone())
        gt = GRPOTrainer(GRPOConfig(bf16=False, head=head, ref_anchor_coef=1e-2), weights=w.clone(),
                         env=SyntheticRewardEnv(seed=0, prompt_len=16, feedback_len=4, vocab_size=cfg.vocab_size),
                         rollout_kwargs=dict(num_pages=64, page_size=16, max_seq_len=128))
        for policy, ref in ((dt.tr.eng, dt.ref), (gt.trainer.eng, gt.ref_eng)):
            assert policy.head == ref.head == head and policy.temperature == ref.temperature
            assert torch.equal(policy.token_logprobs(b)[0], ref.token_logprobs(b)[0])


@pytest.mark.parametrize("act8", [False, True])
def test_plan_leaves_room_for_the_layer_in_flight(monkeypatch, act8):
    """The layer that the backward works on is held in the weights' type, whatever its checkpoint is held in."""
    from types import SimpleNamespace
    cfg = _cfg()
    tr = CausalLMTrainer(cfg, get_context(), dtype=torch.float32, act8=act8, activation_reserve_gb=0.0)
    tokens = 1000
    _, ctx = tr.eng._layer_fwd(1, torch.randn(40, cfg.hidden_size), Batch.from_sequences([torch.arange(40)]), keep=True)
    held = ("o", "lse", "rstd1", "rstd2") + (() if act8 else ("x",))       # from 8 bits, x is another tensor
    flight = sum(t.numel() * t.element_size() for k, t in ctx.items() if k not in held) * tokens // 40 + 8 * tokens
    per = tr.eng.activation_bytes_per_layer(tokens)
    free = flight + 2 * per
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda *a: (free, free))
    monkeypatch.setattr(torch.cuda, "memory_reserved", lambda *a: 0)
    monkeypatch.setattr(torch.cuda, "memory_allocated", lambda *a: 0)
    tr.ctx = SimpleNamespace(device=torch.device("cuda"), world=1)
    assert tr.plan_activations(tokens) == 2
    free -= 1
    assert tr.plan_activations(tokens) == 1


def test_ids_outside_the_table_with_the_sorted_gradient():
    """They read a zero row, as their gradient says: no row of the table changes what they give."""
    cfg = _cfg()
    g = torch.Generator().manual_seed(0)
    b = Batch.from_sequences([torch.randint(0, cfg.vocab_size - 1, (21,), generator=g)])
    b.ids[4], b.ids[9] = -1, cfg.vocab_size
    b.targets[3] = b.targets[8] = -1                          # the tokens before them have no label
    eng = _engine(cfg, embed_grad="sorted")
    eng.zero_grad()
    eng.forward_backward(b, coef=eng.sft_coef(b))
    table, grad = eng.w.views(0)["embed"], eng.grad_views(0)["embed"]
    assert (grad[-1] == 0).all()
    lp = eng.token_logprobs(b)[0]
    many = eng.token_logprobs_many([b])[0][0]
    table[-1] += 1.0
    assert torch.equal(eng.token_logprobs(b)[0], lp) and torch.equal(many, lp)
