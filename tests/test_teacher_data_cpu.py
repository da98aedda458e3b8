"""A teacher's top logits go with the tokens through packers, collators and loaders."""
import pytest
import torch

from chronicals_b200.data import DataCollator, DataCollatorWithFlattening, FixedShapeSequencePacker, create_packed_dataloader
from chronicals_b200.data.data_loader import stack_packed_rows
from chronicals_b200.data.sequence_packer_v2 import SequencePackerV2
from chronicals_b200.models.decoder import CausalLM
from chronicals_b200.training.chronicals_trainer import _batch_fields
from test_long_context_model_cpu import config

KEYS = ("teacher_indices", "teacher_logits")


def sample(n, K, seed, V=97, teacher=True):
    g = torch.Generator().manual_seed(seed)
    s = {"input_ids": torch.randint(1, V, (n,), generator=g)}
    s["labels"] = s["input_ids"].clone()
    if teacher:
        s["teacher_indices"] = torch.stack([torch.randperm(V, generator=g)[:K] for _ in range(n)])
        s["teacher_logits"] = torch.randn(n, K, generator=g)
    return s


def samples():
    """One that is cut off at 12 tokens, several widths, and one without a teacher."""
    return [sample(15, 3, 0), sample(4, 5, 1), sample(5, 2, 2, teacher=False), sample(3, 3, 3)]


def check(batch, given, keep):
    """Every token's entries are its sample's; all others are absent."""
    ids, idx, lg = (batch[k].reshape(batch["input_ids"].numel(), *batch[k].shape[batch["input_ids"].dim():]) for k in ("input_ids", *KEYS))
    left = torch.ones(len(ids), dtype=torch.bool)
    for s in given:
        n = min(len(s["input_ids"]), keep)
        want = s["input_ids"][:n]
        at = [a for a in range(len(ids) - n + 1) if torch.equal(ids[a:a + n], want)]
        assert len(at) == 1
        rows = slice(at[0], at[0] + n)
        if KEYS[0] in s:
            left[rows] = False
            K = s[KEYS[0]].shape[1]
            assert torch.equal(idx[rows, :K], s[KEYS[0]][:n]) and torch.equal(lg[rows, :K], s[KEYS[1]][:n]) and (idx[rows, K:] == -1).all()
    assert (idx[left] == -1).all() and lg.isfinite().all()


@pytest.mark.parametrize("how", ["fixed", "list", "stacked", "v2", "v2 filled", "padded", "flat", "loader", "plain loader"])
def test_every_way(how):
    given, keep = samples(), 12
    if how == "list":
        given = [{k: v.tolist() for k, v in s.items()} for s in given]
        batches = [b.to_dict() for b in FixedShapeSequencePacker(keep).pack_all_sequences(given)]
        given = samples()
    elif how in ("fixed", "stacked"):
        rows = FixedShapeSequencePacker(keep).pack_all_sequences(given)
        batches = [_batch_fields(r.to("cpu")) for r in rows] if how == "fixed" else [stack_packed_rows(rows)]
    elif how.startswith("v2"):
        batches = [b.to("cpu").to_dict() for b in SequencePackerV2(keep, fixed_output_shape=how != "v2").pack(given)]
    elif how == "padded":
        batches = [DataCollator(max_length=keep)(given)]
    elif how == "flat":
        given = given[1:]
        batches = [DataCollatorWithFlattening()(given)]
    else:
        batches = list(create_packed_dataloader(given, 2 if how == "loader" else 4, keep, use_packing=how == "loader"))
    seen = 0
    for b in batches:
        here = [s for s in given if any(torch.equal(b["input_ids"].reshape(-1)[a:a + min(len(s["input_ids"]), keep)], s["input_ids"][:keep])
                                        for a in range(b["input_ids"].numel()))]
        seen += len(here)
        if any(KEYS[0] in s for s in here):
            assert b[KEYS[0]].shape[:-1] == b["input_ids"].shape == b[KEYS[1]].shape[:-1]
            check(b, here, keep)
        else:
            assert KEYS[0] not in b and KEYS[1] not in b
    assert seen == len(given)


def test_samples_without_a_teacher_stay_as_they_were():
    given = [sample(n, 1, n, teacher=False) for n in (3, 7, 5)]
    for b in (FixedShapeSequencePacker(12).pack_all_sequences(given)[0].to_dict(), SequencePackerV2(12).pack(given)[0].to_dict(),
              DataCollator()(given), DataCollatorWithFlattening()(given)):
        assert not any(k in b for k in KEYS)


def test_loss_of_packed_documents():
    """The step's loss over a packed batch is the mean over its documents' tokens."""
    model = CausalLM(config(rope_sections=None), dtype=torch.float64)
    model.reset_parameters(std=0.2, seed=1)
    model.distill_weight, model.distill_temperature = 1.0, 2.0
    given = [sample(n, 4, n) for n in (9, 6, 5)]
    (b,) = create_packed_dataloader(given, 1, 24)
    loss = model(**{k: b[k] for k in ("input_ids", "labels", "position_ids", "cu_seqlens", "max_seqlen", *KEYS)}).loss
    alone = [model(**{k: v[None] for k, v in s.items()}).loss for s in given]
    want = sum(a * (len(s["input_ids"]) - 1) for a, s in zip(alone, given)) / sum(len(s["input_ids"]) - 1 for s in given)
    assert abs(loss.item() - want.item()) < 1e-4                      # attention's formula computes in 32 bits


@pytest.mark.parametrize("change,what", [
    (dict(teacher_logits=None), "together"), (dict(teacher_indices=torch.zeros(6, 3, dtype=torch.long)), "wanted"),
    (dict(teacher_logits=torch.zeros(7, 2)), "wanted"), (dict(teacher_indices=torch.zeros(7, 3)), "whole"),
    (dict(teacher_indices=torch.ones(7, 3, dtype=torch.bool)), "whole"), (dict(teacher_logits=torch.zeros(7, 3, dtype=torch.long)), "whole"), (dict(position_ids=torch.zeros(3, 7, dtype=torch.long)), "axes")])
@pytest.mark.parametrize("take", [lambda s: FixedShapeSequencePacker(12).pack_all_sequences(s), lambda s: SequencePackerV2(12).pack(s),
                                  lambda s: DataCollator()(s), lambda s: DataCollatorWithFlattening()(s)])
def test_refusals(change, what, take):
    s = {**sample(7, 3, 0), **change}
    with pytest.raises(ValueError, match=what):
        take([{k: v for k, v in s.items() if v is not None}])
