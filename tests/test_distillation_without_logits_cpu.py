"""A loss from hidden states does not form the logits beside it."""
import pytest
import torch

from chronicals_b200.models.decoder import CausalLM
from test_long_context_model_cpu import batch, config


@pytest.mark.parametrize("given,logits", [((), True), (("labels",), False), (("teacher_indices", "teacher_logits"), False),
                                          (("labels", "teacher_indices", "teacher_logits"), False)])
def test_logits_only_where_there_is_no_loss(given, logits):
    model = CausalLM(config(), dtype=torch.float32)
    b = batch()
    kw = {k: b[k] for k in ("input_ids", "position_ids", *given)}
    out = model(**kw)
    assert (out.loss is None) == logits and (out.logits is not None) == logits
    asked = model(**kw, return_logits=True)
    assert asked.logits.shape == (2, 23, 97) and (out.loss is None or torch.equal(out.loss, asked.loss))
