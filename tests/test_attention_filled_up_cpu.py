"""Lists of boundaries that are filled up with empty documents: what the captured step passes on, and the kernel that is chosen."""
import pytest
import torch

from chronicals_b200.config.config import TrainingConfig
from chronicals_b200.models.decoder import CausalLM
from chronicals_b200.ops import _ext
from chronicals_b200.training.chronicals_trainer import ChronicalsTrainer
from test_long_context_model_cpu import config


def test_kernel_of_the_backward_pass():
    chosen = _ext.lib().cb_attn_window_bwd_pipelined
    # one document of 8192 tokens, alone or in a list of 64, takes the pipelined kernel (14 heads of 64, window 4096: 305 us, not 353)
    assert chosen(8192, 14, 64, 1, 4096, 1, 148) == chosen(8192, 14, 64, 64, 4096, 1, 148) == 1
    # 27 documents of 300 do not (69 us, not 83), however long the list
    assert chosen(8192, 14, 64, 27, 4096, 27, 148) == chosen(8192, 14, 64, 64, 4096, 27, 148) == 0
    assert chosen(8192, 14, 64, 64, 4096, 64, 148) == 0               # nothing known of the list: every entry counts
    assert chosen(8192, 14, 64, 64, 512, 1, 148) == 0                 # short loops
    assert chosen(1024, 14, 64, 64, 512, 64, 148) == 1                # a grid that leaves SMs free
    assert chosen(8192, 28, 128, 64, 128, 64, 148) == 1
    assert chosen(8192, 14, 64, 4, 4096, 99, 148) == 1 and chosen(8192, 14, 64, 4, 4096, 0, 148) == 1


@pytest.mark.parametrize("lens,kept", [([9, 14], True), ([5, 5, 5, 8], False)])
def test_captured_step_fills_the_list_up(tmp_path, monkeypatch, lens, kept):
    model = CausalLM(config(), dtype=torch.float32)
    args = TrainingConfig(output_dir=str(tmp_path), max_steps=1, gradient_accumulation_steps=1, use_gradient_checkpointing=False, fp8=False)
    t = ChronicalsTrainer(model, args, [])
    t.args.cuda_graph_max_documents = 4
    seen = {}

    class Captured(Exception):
        pass

    def capture(f, key):
        seen.update(f)
        raise Captured
    monkeypatch.setattr(t, "_capture_graph", capture)
    cu = torch.tensor([0] + torch.tensor(lens).cumsum(0).tolist(), dtype=torch.int32)
    with pytest.raises(Captured):
        t._graphed_step({"input_ids": torch.zeros(1, 23, dtype=torch.long), "cu_seqlens": cu, "seqlens_host": lens, "max_seqlen": 14})
    assert seen["cu_seqlens"].tolist() == cu.tolist() + [23] * (4 - len(lens))
    # lengths of fewer documents than boundaries say which are not empty; as many would be taken for every batch's
    assert seen["seqlens_host"] == (lens if kept else None)
