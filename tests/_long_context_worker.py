"""Worker on gloo ranks: a window, sinks and positions of several axes in the tensor-parallel model; a teacher through ZeRO-3."""
import json
import sys

import torch

from chronicals_b200.models.decoder import CausalLM
from chronicals_b200.parallel.bootstrap import init_distributed, shutdown
from chronicals_b200.parallel.tensor_parallel import TensorParallelCausalLM, TPState
from chronicals_b200.parallel.zero3 import Zero3Engine
from test_long_context_model_cpu import batch, config


def tensor_parallel(rank, world):
    full = CausalLM(config(vocab_size=96), dtype=torch.float32)
    full.reset_parameters(std=0.2, seed=3)
    model = TensorParallelCausalLM.from_full(full, TPState(backend="nccl"))
    b = batch(B=2, S=16, V=96)
    teacher = {k: b.pop(k) for k in ("teacher_indices", "teacher_logits")}
    loss, want = model(**b).loss, full(**b).loss
    loss.backward()
    want.backward()
    model.sync_replicated_grads()
    refused = 0
    for some in (teacher, {"teacher_logits": teacher["teacher_logits"]}):
        try:
            model(**b, **some)
        except ValueError as e:
            refused += "distillation" in str(e)
    lq = model.layers[0].hq * full.config.head_dim
    qw, fw = model.layers[1].qkv_weight.grad[:lq], full.model.layers[1].self_attn.qkv_proj.weight.grad[rank * lq:(rank + 1) * lq]
    rel = [float((a - r).norm() / r.norm()) for a, r in ((qw, fw), (model.embed_tokens.weight.grad, full.model.embed_tokens.weight.grad))]
    return {"loss": float(loss), "want": float(want), "grads": rel, "refused": refused}


def zero3(rank, world):
    models = [CausalLM(config(), dtype=torch.float32) for _ in range(2)]
    for m in models:
        m.reset_parameters(std=0.2, seed=3)
        m.distill_weight, m.distill_temperature = 0.75, 2.0
    eng = Zero3Engine(models[0], lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.01, max_grad_norm=1.0, backend="fused")
    opt = torch.optim.AdamW(models[1].parameters(), lr=1e-3, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.01)
    losses, want = [], []
    for step in range(2):
        parts = [batch(seed=10 * step + r) for r in range(world)]
        losses.append(float(eng.forward_backward(**parts[rank])))
        eng.step()
        for r, p in enumerate(parts):
            loss = models[1](**p).loss
            (loss / world).backward()
            if r == rank:
                want.append(float(loss))
        torch.nn.utils.clip_grad_norm_(models[1].parameters(), 1.0)
        opt.step()
        opt.zero_grad(set_to_none=True)
    evaluated = float(eng.forward_only(**batch(seed=99)).loss)
    with torch.no_grad():
        losses.append(evaluated)
        want.append(float(models[1](**batch(seed=99)).loss))
    full, ref = eng.gather_full_state_dict(), models[1].hf_state_dict()
    return {"losses": losses, "want": want, "diff": max(float((full[k].float() - ref[k].float()).abs().max()) for k in ref)}


def main():
    rank, _, world = init_distributed("gloo", timeout_s=60)
    res = {"tp": tensor_parallel(rank, world), "zero3": zero3(rank, world)}
    with open(f"{sys.argv[1]}.{rank}", "w") as f:
        json.dump(res, f)
    shutdown()


if __name__ == "__main__":
    main()
