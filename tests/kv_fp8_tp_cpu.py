"""One of two gloo ranks that run the engine with an 8-bit cache, tensor parallel, against the same engine in one process.
Launched by ``test_kv_fp8_cpu.py`` once per rank; prints ``KV_FP8_TP_OK``."""

import os
import sys

import numpy as np
import torch
import torch.distributed as dist

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), ".."))

from multigpu_fused import hf_style_weights  # noqa: E402

from cornserve import ops  # noqa: E402
from cornserve.models.qwen_llm import LLMConfig, QwenLLM  # noqa: E402
from cornserve.parallel.state import init_distributed, single_group  # noqa: E402
from cornserve.task_executors.llm.engine import EngineConfig, LLMEngine, SamplingParams, Sequence  # noqa: E402


def run(cfg, weights, group):
    model = QwenLLM(cfg, group=group, device="cpu").float()
    assert len(model.load_weights(weights.items())) == len(weights)
    eng = LLMEngine(model, EngineConfig(num_pages=8, max_batched_tokens=96, decode_burst=2, max_model_len=512, kv_cache_dtype="fp8"))
    for i in range(2):
        eng.add_request(Sequence(f"s{i}", np.arange(3 + i, 40 + 190 * i, dtype=np.int32), SamplingParams(5, True), return_hidden=True))
    toks, hid = {}, {}
    while eng.has_work():
        for o in eng.step():
            toks.setdefault(o.seq_id, []).extend(o.new_token_ids)
            if o.hidden is not None:
                hid[o.seq_id] = o.hidden
    return eng, toks, hid


def main():
    rank, world, port = int(sys.argv[1]), int(sys.argv[2]), int(sys.argv[3])
    torch.set_num_threads(2)
    g = init_distributed(rank, world, master_port=port, backend="gloo", timeout_s=120, with_fabric=False)
    assert g.size == world
    cfg = LLMConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=32,
                    intermediate_size=256, vocab_size=512, eos_token_id=511)
    weights = hf_style_weights(cfg)
    tp, tp_toks, tp_hid = run(cfg, weights, g)
    one, one_toks, one_hid = run(cfg, weights, single_group())
    assert tp.kv_backing.shape == (2, 8, 2, 1, 128 * 36) and one.kv_backing.shape == (2, 8, 2, 2, 128 * 36)
    for layer in range(2):
        (c, s), (c1, s1) = (ops.kv_cache_fp8_views(e.kv_caches[layer].contiguous()) for e in (tp, one))
        c1, s1 = c1[:, :, rank: rank + 1].float(), s1[:, :, rank: rank + 1]
        # (page 0 takes the padding.)  Sums in another order move a value by its last bits, and a code that lies next to a
        # rounding border by one step; behind such keys and values the second layer's rows move by more than their last bits
        assert s1[1:].any() and torch.allclose(s[1:], s1[1:], rtol=1e-5 if layer == 0 else 1e-2, atol=1e-9)
        assert ((c.float() - c1)[1:].abs() <= c1[1:].abs() * 2 ** -3 + 2 ** -9).all()
        if layer == 0:
            assert (c.float() != c1)[1:].float().mean() < 1e-3
    for sid, want in one_hid.items():
        cos = torch.nn.functional.cosine_similarity(tp_hid[sid].flatten(), want.flatten(), dim=0).item()
        assert cos > 0.999, f"{sid}: hidden states differ (cos {cos:.4f})"
        assert tp_toks[sid][0] == one_toks[sid][0] and len(tp_toks[sid]) == 5
    dist.barrier()
    if rank == 0:
        print("KV_FP8_TP_OK", flush=True)
    dist.destroy_process_group()


if __name__ == "__main__":
    main()
