"""What makes the captured training step be captured anew."""
import pytest
import torch

from chronicals_b200.config.config import TrainingConfig
from chronicals_b200.models.decoder import CausalLM
from chronicals_b200.training.chronicals_trainer import ChronicalsTrainer
from test_long_context_model_cpu import batch, config


class _Replayed(Exception):
    pass


@pytest.fixture
def captures(tmp_path, monkeypatch):
    """``captures(batch)``: whether the step of a batch is captured (instead of replayed)."""
    model = CausalLM(config(), dtype=torch.float32)
    args = TrainingConfig(output_dir=str(tmp_path), max_steps=1, gradient_accumulation_steps=1, use_gradient_checkpointing=False, fp8=False)
    t = ChronicalsTrainer(model, args, [])
    seen = []

    class Graph:
        def replay(self):
            raise _Replayed

    def capture(f, key):
        seen.append(key)
        t._graph = {"key": key, "static": {}, "graph": Graph()}

    def captured(b):
        before = len(seen)
        with pytest.raises(_Replayed):
            t._graphed_step(b)
        return len(seen) > before
    captured.model = model
    monkeypatch.setattr(t, "_capture_graph", capture)
    monkeypatch.setattr(t.optimizer, "prepare_step", lambda: None, raising=False)
    return captured


def test_shapes_and_types(captures):
    assert captures(batch())
    assert not captures(batch(seed=1))
    half = batch(seed=2)
    half["teacher_logits"] = half["teacher_logits"].bfloat16()
    assert captures(half)                                             # and not rounded into, or out of, the other one's buffer
    assert captures(batch(seed=3))
    assert captures(batch(K=4))
    alone = batch(seed=4)
    del alone["teacher_indices"], alone["teacher_logits"]
    assert captures(alone) and not captures(alone)


def test_names(captures):
    """Two optional inputs of one shape are not one another."""
    one, other = batch(axes=2), batch(axes=2)
    del one["teacher_indices"], one["teacher_logits"]
    other["teacher_indices"] = other.pop("position_ids")
    del other["teacher_logits"]
    assert captures(one) and captures(other)


def test_weight_and_temperature(captures):
    assert captures(batch())
    captures.model.distill_weight = 0.125
    assert captures(batch())
    captures.model.distill_temperature = 3.0
    assert captures(batch()) and not captures(batch())
