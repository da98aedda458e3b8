"""A decoder with a sliding window, sinks, positions of several axes and a teacher: the whole step against the definitions."""
import json

import pytest
import torch

from chronicals_b200.config.config import ChronicalsConfig, TrainingConfig
from chronicals_b200.models.decoder import CausalLM
from chronicals_b200.ops import ref
from chronicals_b200.training.chronicals_trainer import ChronicalsTrainer
from test_attention_window_cpu import dense
from test_distillation_cpu import definition
from test_rope_axes_cpu import turned

SECTIONS = {False: (2, 3, 3), True: (4, 2, 2)}


def config(cyclic=False, **kw):
    base = dict(hidden_size=32, intermediate_size=48, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=16,
                vocab_size=97, max_position_embeddings=64, rope_theta=1e3, tie_word_embeddings=True, attention_bias=True,
                sliding_window=7, attention_sinks=2, rope_sections=list(SECTIONS[cyclic]), rope_cyclic=cyclic)
    return ChronicalsConfig(**{**base, **kw})


def batch(B=2, S=23, V=97, K=5, axes=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, V, (B, S), generator=g)
    labels = ids.clone()
    labels[:, :4] = -100
    pos = torch.randint(0, 40, (axes, B, S), generator=g)
    idx = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(B * S)]).view(B, S, K)
    idx[0, 9] = -1
    return dict(input_ids=ids, labels=labels, position_ids=pos, teacher_indices=idx, teacher_logits=torch.randn(B, S, K, generator=g) * 2)


def step_by_hand(model, cfg, b, lens, weight, tau):
    """The loss from the definitions, with the model's own parameters (differentiable)."""
    hq, hk, d = cfg.num_attention_heads, cfg.num_key_value_heads, cfg.head_dim
    T = b["input_ids"].numel()
    cos, sin = ref.rope_cache(64, d, cfg.rope_theta, device=b["input_ids"].device)
    axes = ref.rope_axis_map(cfg.rope_sections, cfg.rope_cyclic)
    pos = b["position_ids"].reshape(len(cfg.rope_sections), T)

    def norm(x, m):
        return x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + m.eps) * m.weight

    h = model.model.embed_tokens.weight[b["input_ids"].reshape(T)]
    for layer in model.model.layers:
        at = layer.self_attn
        qkv = norm(h, layer.input_layernorm) @ at.qkv_proj.weight.t() + at.qkv_proj.bias
        qkv = turned(qkv, cos, sin, pos, axes, hq + hk, d, False).to(h.dtype)
        q, k, v = (t.reshape(T, -1, d) for t in qkv.split((hq * d, hk * d, hk * d), 1))
        h = h + dense(q, k, v, lens, cfg.sliding_window, cfg.attention_sinks).reshape(T, -1) @ at.o_proj.weight.t()
        g, u = (norm(h, layer.post_attention_layernorm) @ layer.mlp.gate_up_proj.weight.t()).chunk(2, -1)
        h = h + (torch.nn.functional.silu(g) * u) @ layer.mlp.down_proj.weight.t()
    z = norm(h, model.model.norm) @ model.output_weight.t()
    y = torch.cat((b["labels"][:, 1:], torch.full_like(b["labels"][:, :1], -100)), 1).reshape(T)
    K = b["teacher_indices"].shape[-1]
    rows, valid = definition(z, b["teacher_indices"].reshape(T, K), b["teacher_logits"].reshape(T, K), tau, y)
    ce = torch.nn.functional.cross_entropy(z, y, ignore_index=-100)
    return (1 - weight) * ce + weight * rows.sum() / valid.sum()


@pytest.mark.parametrize("cyclic", [False, True])
@pytest.mark.parametrize("weight,tau", [(0.5, 1.0), (0.25, 2.0), (1.0, 1.5)])
def test_step(cyclic, weight, tau):
    cfg = config(cyclic)
    model = CausalLM(cfg, dtype=torch.float64)
    model.reset_parameters(std=0.2, seed=3)
    model.distill_weight, model.distill_temperature = weight, tau
    b = batch()
    loss = model(**b).loss
    want = step_by_hand(model, cfg, b, [23, 23], weight, tau)
    # norms, rotation and attention of the plain path compute in 32 bits
    assert abs(loss.item() - want.item()) < 1e-4
    params = list(model.parameters())
    for p, a, r in zip(params, torch.autograd.grad(loss, params), torch.autograd.grad(want, params)):
        assert (a - r).norm() <= 1e-3 * r.norm() + 1e-6, p.shape


def test_documents_flat_ids_and_one_position_a_token():
    cfg = config()
    model = CausalLM(cfg, dtype=torch.float32)
    model.reset_parameters(seed=1)
    b = batch(B=1, S=20)
    cu = torch.tensor([0, 8, 20], dtype=torch.int32)
    whole = model(**b, cu_seqlens=cu, max_seqlen=12, return_logits=True).logits[0]
    flat = model(b["input_ids"][0], position_ids=b["position_ids"][:, 0], cu_seqlens=cu, max_seqlen=12).logits[0]
    assert torch.allclose(whole, flat, atol=1e-5)
    tail = model(b["input_ids"][:, 8:], position_ids=b["position_ids"][:, :, 8:]).logits[0]
    assert torch.allclose(whole[8:], tail, atol=1e-5)
    one = torch.arange(20)[None]
    a = model(b["input_ids"], position_ids=one, cu_seqlens=cu, max_seqlen=12).logits
    assert torch.allclose(a, model(b["input_ids"], position_ids=one.expand(3, 1, 20), cu_seqlens=cu, max_seqlen=12).logits, atol=1e-5)


def test_teacher_alone_and_no_weight():
    model = CausalLM(config(), dtype=torch.float32)
    b = batch()
    teacher = {k: b[k] for k in ("teacher_indices", "teacher_logits")}
    alone = model(b["input_ids"], position_ids=b["position_ids"], **teacher)
    assert alone.loss is not None
    model.distill_weight = 0.0
    with_teacher = model(**b).loss
    del b["teacher_indices"], b["teacher_logits"]
    assert torch.equal(with_teacher, model(**b).loss)


def test_refusals():
    model = CausalLM(config(), dtype=torch.float32)
    b = batch()
    with pytest.raises(ValueError, match="axes"):
        model(b["input_ids"], position_ids=b["position_ids"][:2])
    with pytest.raises(ValueError, match="together"):
        model(b["input_ids"], teacher_indices=b["teacher_indices"])
    with pytest.raises(ValueError, match="without a window"):
        CausalLM(config(sliding_window=None), dtype=torch.float32)(b["input_ids"])


def test_configuration_survives_a_checkpoint_and_other_files_keep_their_meaning():
    cfg = config()
    back = ChronicalsConfig.from_hf_config(json.loads(json.dumps(cfg.to_hf_config())))
    for k in ("sliding_window", "attention_sinks", "rope_sections", "rope_cyclic"):
        assert getattr(back, k) == getattr(cfg, k)
    plain = ChronicalsConfig.from_model_name("tiny-qwen2").to_hf_config()
    assert "chronicals" not in plain
    assert ChronicalsConfig.from_hf_config({**plain, "sliding_window": 4096, "use_sliding_window": False}).sliding_window is None


def test_trainer_takes_a_teacher(tmp_path):
    cfg = config()
    model = CausalLM(cfg, dtype=torch.float32)
    model.reset_parameters(seed=2)
    args = TrainingConfig(output_dir=str(tmp_path), max_steps=2, gradient_accumulation_steps=1, use_gradient_checkpointing=False, fp8=False,
                          save_steps=0, logging_steps=0, distill_weight=0.75, distill_temperature=2.0, z_loss_weight=0.0)
    t = ChronicalsTrainer(model, args, [batch(seed=s) for s in range(2)])
    assert (model.distill_weight, model.distill_temperature) == (0.75, 2.0)
    with torch.no_grad():
        want = model(**batch())
    loss = t._forward_loss(t._prepare_inputs(batch()))
    assert torch.equal(loss.detach().cpu(), want.loss.cpu())


def test_trainer_refuses_a_teacher_for_other_models(tmp_path):
    class Other(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.w = torch.nn.Parameter(torch.zeros(1))

        def forward(self, input_ids, labels=None, **kw):
            return type("O", (), {"loss": self.w.sum()})()
    args = TrainingConfig(output_dir=str(tmp_path), max_steps=1, gradient_accumulation_steps=1, use_gradient_checkpointing=False, fp8=False)
    t = ChronicalsTrainer(Other(), args, [batch()])
    with pytest.raises(ValueError, match="teacher"):
        t._forward_loss(t._prepare_inputs(batch()))
