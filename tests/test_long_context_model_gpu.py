"""The decoder's step with a window, sinks, positions of several axes and a teacher on the kernels, against the definitions."""
import pytest
import torch

from chronicals_b200.config.config import TrainingConfig
from chronicals_b200.models.decoder import CausalLM
from chronicals_b200.ops import _ext
from chronicals_b200.training.chronicals_trainer import ChronicalsTrainer
from test_long_context_model_cpu import batch, config, step_by_hand

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _config(d, cyclic=False):
    sec = {(64, False): [8, 12, 12], (128, False): [16, 24, 24], (64, True): [12, 10, 10]}[d, cyclic]
    return config(hidden_size=256, intermediate_size=512, num_attention_heads=4, num_key_value_heads=2, head_dim=d, vocab_size=2000,
                  sliding_window=70, attention_sinks=3, rope_sections=sec, rope_cyclic=cyclic, tie_word_embeddings=d == 64)


def _batch(seed=0, S=205):
    return {k: v.to(DEV) for k, v in batch(B=2, S=S, V=2000, K=16, seed=seed).items()}


@pytest.mark.parametrize("d,cyclic", [(64, False), (64, True), (128, False)])
def test_step(d, cyclic):
    cfg = _config(d, cyclic)
    model = CausalLM(cfg, dtype=torch.bfloat16, device=DEV)
    model.reset_parameters(std=0.05, seed=3)
    model.distill_weight, model.distill_temperature = 0.5, 2.0
    wide = CausalLM(cfg, dtype=torch.float64, device=DEV)
    wide.load_state_dict({k: v.double() for k, v in model.state_dict().items()})
    b = _batch()
    loss = model(**b).loss
    want = step_by_hand(wide, cfg, b, [205, 205], 0.5, 2.0)
    _ext.check_status()
    # activations are rounded to bf16 at a dozen places (2^-9 on average each); the loss averages over hundreds of rows
    assert abs(loss.item() - want.item()) <= 2.0 ** -7 * abs(want.item())
    got = torch.autograd.grad(loss, list(model.parameters()))
    ref = torch.autograd.grad(want, list(wide.parameters()))
    _ext.check_status()
    for (name, _), a, r in zip(model.named_parameters(), got, ref):
        assert (a.double() - r).norm() <= 2.0 ** -4 * r.norm() + 1e-6, (name, ((a.double() - r).norm() / r.norm()).item())


def test_trainer_step_is_captured_and_follows_the_batches(tmp_path):
    """The CUDA-graph step with a teacher in the batch: every replay sees its own batch's positions and teacher."""
    args = dict(output_dir=str(tmp_path), gradient_accumulation_steps=1, use_gradient_checkpointing=False, fp8=False, learning_rate=0.0,
                weight_decay=0.0, max_grad_norm=0.0, z_loss_weight=0.0, save_steps=0, logging_steps=0, max_steps=8)
    losses = []
    for graphs in (True, False):
        model = CausalLM(_config(64), dtype=torch.bfloat16, device=DEV)
        model.reset_parameters(std=0.05, seed=4)
        t = ChronicalsTrainer(model, TrainingConfig(use_cuda_graphs=graphs, **args), [_batch()])
        losses.append([t.training_step(_batch(s)).item() for s in (0, 1, 2)])
        losses[-1].append(t.training_step(_batch(3, S=130)).item())   # another shape: captured anew
        _ext.check_status()
    assert len(set(losses[0])) == 4
    for a, b in zip(*losses):
        assert abs(a - b) <= 1e-3 * abs(b)
