"""The 8-bit paged key-value cache on the CPU: layout, quantisation, attention, refusals, and the engine on top of it."""

import json
import math
import os
import subprocess
import sys
import types

import numpy as np
import pytest
import torch

from cornserve import ops
from cornserve.models.qwen_llm import BatchMeta, LLMConfig, QwenLLM
from cornserve.ops import reference as ref
from cornserve.services.process import free_port
from cornserve.task_executors.llm.engine import EngineConfig, LLMEngine, PrefilledKV, SamplingParams, Sequence


def _cs(T, d, start=0):
    ang = (start + torch.arange(T, dtype=torch.float64))[:, None] * 1e4 ** (-torch.arange(d // 2, dtype=torch.float64) * 2 / d)
    return torch.stack([ang.cos(), ang.sin()], dim=1).float().contiguous()


def test_layout_is_codes_then_scales_of_every_block():
    cache = ops.kv_cache_fp8(3, 2, 64)
    codes, scales = ops.kv_cache_fp8_views(cache)
    assert cache.shape == (3, 2, 2, 128 * 68) and codes.shape == (3, 2, 2, 128, 64) and scales.shape == (3, 2, 2, 128)
    codes[1, 1, 0, 5, 7] = 1.5
    scales[1, 1, 0, 5] = 2.0
    block = cache[1, 1, 0]
    assert block[5 * 64 + 7] == 0x3C and block[128 * 64:].view(torch.float32)[5] == 2.0
    assert int((cache != 0).sum()) == 2   # the code byte and one byte of 2.0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("norm", [False, True])
def test_append_stores_rows_within_half_a_code_step(d, norm):
    torch.manual_seed(d + norm)
    T, Hq, Hkv = 40, 4, 2
    qkv = torch.randn(T, (Hq + 2 * Hkv) * d) * torch.exp(torch.randn(T, 1))
    cs = _cs(T, d, 100)
    wq, wk = (1 + 0.1 * torch.randn(d) for _ in range(2))
    cache = ops.kv_cache_fp8(3, Hkv, d)
    before = qkv.clone()
    slot = (2 * 128 + 60 + torch.arange(T)).int()
    slot[7] = -1
    kw = dict(q_norm=wq, k_norm=wk, eps=1e-5) if norm else {}
    q = ops.rope_kv_write_fp8_(qkv, Hq, Hkv, d, cs, cache, slot, **kw)
    assert torch.equal(qkv, before)
    x = qkv.double().view(T, -1, d)
    if norm:
        x = torch.cat([x[:, :Hq] / (x[:, :Hq].square().mean(-1, True) + 1e-5).sqrt() * wq,
                       x[:, Hq: Hq + Hkv] / (x[:, Hq: Hq + Hkv].square().mean(-1, True) + 1e-5).sqrt() * wk, x[:, Hq + Hkv:]], 1)
    c, s = cs.double()[:, None, 0], cs.double()[:, None, 1]
    rot = x.clone()
    rot[:, : Hq + Hkv] = torch.cat([x[:, : Hq + Hkv, : d // 2] * c - x[:, : Hq + Hkv, d // 2:] * s,
                                    x[:, : Hq + Hkv, d // 2:] * c + x[:, : Hq + Hkv, : d // 2] * s], -1)
    assert torch.allclose(q.double(), rot[:, :Hq], atol=1e-5, rtol=1e-5)
    codes, scales = ops.kv_cache_fp8_views(cache)
    for t in range(T):
        for i, want in enumerate((rot[t, Hq: Hq + Hkv], rot[t, Hq + Hkv:])):
            got = codes[int(slot[t]) // 128, i, :, int(slot[t]) % 128].double() * scales[int(slot[t]) // 128, i, :, int(slot[t]) % 128, None].double()
            if t == 7:
                continue
            amax = want.abs().amax(-1, keepdim=True)
            # half a step of e4m3 (2^-4 of the value; 2^-10 of the unit among its subnormals), plus fp32 arithmetic
            assert ((got - want).abs() <= want.abs() * (2 ** -4 + 1e-5) + amax / 448 * (2 ** -10 + 1e-3)).all()
    codes[slot[slot >= 0].long() // 128, :, :, slot[slot >= 0].long() % 128] = 0
    assert int((codes.view(torch.uint8) & 0x7f != 0).sum()) == 0   # nothing else was written


def test_rows_of_zeros_tiny_values_and_non_finite_values():
    d, Hkv = 64, 1
    rows = torch.zeros(6, d)
    rows[1] = 1e-30
    rows[2, 3] = float("inf")
    rows[3, 4] = float("nan")
    rows[4] = 3e38
    rows[5] = -2.0 ** -40
    codes, scales = ref.quantize_kv_rows(rows)
    assert scales[0] > 0 and not codes[0].float().any()
    assert scales[1] == scales[0] and not codes[1].float().any()
    assert torch.isnan(scales[2:4]).all() and not codes[2:4].float().any()
    assert torch.isfinite(scales[4]) and (codes[4].float() == 448).all()
    assert (codes[5].float() == -448).all()
    # a row that became NaN shows up in the sequences that read it, and only there
    cache = ops.kv_cache_fp8(3, Hkv, d)
    c, s = ops.kv_cache_fp8_views(cache)
    s.fill_(1.0)
    s[1, 0, 0, 4] = float("nan")
    q = torch.randn(2, 1, d)
    o = ops.attention_paged_fp8(q, cache, torch.tensor([[1], [2]], dtype=torch.int32), torch.tensor([5, 5], dtype=torch.int32),
                                torch.tensor([0, 1, 2], dtype=torch.int32), 1)
    assert torch.isnan(o[0]).all() and not o[1].any()
    o = ops.attention_paged_fp8(q, cache, torch.tensor([[1], [2]], dtype=torch.int32), torch.tensor([4, 5], dtype=torch.int32),
                                torch.tensor([0, 1, 2], dtype=torch.int32), 1)
    assert not o.any()


def test_attention_matches_the_definition_and_leaves_other_rows():
    torch.manual_seed(3)
    d, Hq, Hkv = 64, 6, 2
    lens, new = [130, 0, 5, 200], [3, 2, 5, 1]     # the second has queries and no keys
    cache = ops.kv_cache_fp8(6, Hkv, d)
    codes, scales = ops.kv_cache_fp8_views(cache)
    codes.copy_(torch.randn(codes.shape).to(torch.float8_e4m3fn))
    scales.copy_(torch.rand(scales.shape) + 0.1)
    table = torch.tensor([[3, 1], [0, 0], [5, 0], [2, 4]], dtype=torch.int32)
    cu = [0, 3, 5, 10, 11]
    q = torch.randn(13, Hq, d)
    out = torch.full_like(q, 9.0)
    got = ops.attention_paged_fp8(q, cache, table, torch.tensor(lens, dtype=torch.int32), torch.tensor(cu, dtype=torch.int32), 5, out=out)
    assert got is out and (out[11:] == 9.0).all() and not out[3:5].any()
    for i in (0, 2, 3):
        kv = (codes[table[i].long()].double() * scales[table[i].long()].double()[..., None])    # [blocks, 2, Hkv, 128, d]
        k, v = (kv[:, j].transpose(1, 2).reshape(-1, Hkv, d)[: lens[i]] for j in (0, 1))
        for t in range(new[i]):
            n = lens[i] - new[i] + t + 1
            for h in range(Hq):
                p = torch.softmax(k[:n, h // 3] @ q[cu[i] + t, h].double() / math.sqrt(d), 0)
                assert torch.allclose(out[cu[i] + t, h].double(), p @ v[:n, h // 3], atol=1e-5)


def _good():
    d, Hq, Hkv = 64, 4, 2
    i32 = lambda a: torch.tensor(a, dtype=torch.int32)  # noqa: E731
    append = dict(qkv=torch.zeros(3, (Hq + 2 * Hkv) * d), Hq=Hq, Hkv=Hkv, d=d, cs=_cs(3, d), cache=ops.kv_cache_fp8(2, Hkv, d), slot=i32([0, 1, -1]))
    attend = dict(q=torch.zeros(2, Hq, d), cache=ops.kv_cache_fp8(2, Hkv, d), block_table=i32([[0], [1]]), kv_len=i32([1, 1]),
                  cu_q=i32([0, 1, 2]), max_q_len=1)
    return append, attend


def test_appends_that_are_refused():
    good, _ = _good()
    ops.rope_kv_write_fp8_(**good)
    for bad in (dict(qkv=torch.zeros(3, 511)), dict(cs=_cs(2, 64)), dict(cs=_cs(3, 64).double()), dict(slot=good["slot"].long()),
                dict(slot=good["slot"][:2]), dict(cache=ops.kv_cache_fp8(2, 1, 64)), dict(cache=ops.kv_cache_fp8(2, 2, 128)),
                dict(cache=torch.zeros(2, 2, 2, 128, 64)), dict(cache=ops.kv_cache_fp8(2, 2, 64).transpose(1, 2)),
                dict(q_norm=torch.ones(64)), dict(q_norm=torch.ones(64), k_norm=torch.ones(32)),
                dict(slot=torch.tensor([0, 256, 1], dtype=torch.int32)), dict(slot=torch.zeros(6, dtype=torch.int32)[::2])):
        with pytest.raises(ValueError):
            ops.rope_kv_write_fp8_(**{**good, **bad})


def test_attentions_that_are_refused():
    _, good = _good()
    ops.attention_paged_fp8(**good)
    for bad in (dict(q=torch.zeros(2, 3, 64)), dict(q=torch.zeros(2, 4, 32)), dict(q=torch.zeros(2, 256)), dict(kv_len=good["kv_len"].long()),
                dict(cu_q=good["cu_q"][:2]), dict(block_table=good["block_table"].long()), dict(block_table=good["block_table"][:1]),
                dict(block_table=good["block_table"][:, 0]), dict(max_q_len=-1), dict(out=torch.zeros(1, 4, 64)),
                dict(out=torch.zeros(2, 4, 64, dtype=torch.float64)),
                dict(kv_len=torch.tensor([129, 1], dtype=torch.int32)), dict(block_table=torch.tensor([[2], [1]], dtype=torch.int32)),
                dict(block_table=torch.tensor([[-1], [1]], dtype=torch.int32))):
        with pytest.raises(ValueError):
            ops.attention_paged_fp8(**{**good, **bad})
    with pytest.raises(ValueError):
        ops.kv_cache_fp8_views(torch.zeros(2, 2, 2, 100, dtype=torch.uint8))


# -- the engine ------------------------------------------------------------------------------------------------------
def _model(qk_norm=False):
    torch.manual_seed(0)
    cfg = LLMConfig(hidden_size=128, num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2, head_dim=32,
                    intermediate_size=256, vocab_size=512, mrope_section=[4, 6, 6], rope_theta=10000.0, qk_norm=qk_norm, eos_token_id=511)
    m = QwenLLM(cfg, device="cpu").float()
    for p in m.parameters():
        if p.dim() > 1:
            p.data.normal_(0, 0.1)
    return m


def _full_pass(model, ids):
    """Logits of the last position from one pass over all tokens, through a fresh 8-bit cache."""
    T = len(ids)
    blocks = T // 128 + 1
    meta = BatchMeta(torch.tensor(ids, dtype=torch.int32), torch.arange(T, dtype=torch.int32).expand(3, T).contiguous(),
                     (128 + torch.arange(T)).int(), torch.tensor([0, T], dtype=torch.int32), torch.tensor([T], dtype=torch.int32),
                     torch.arange(1, 1 + blocks, dtype=torch.int32)[None], torch.tensor([T - 1], dtype=torch.int32), T)
    return model.compute_logits(model.forward_hidden(meta, model.alloc_kv_cache(blocks + 1, "fp8"))[-1:])[0]


@pytest.mark.parametrize("qk_norm", [False, True])
def test_engine_with_an_8_bit_cache_matches_full_recompute(qk_norm):
    model = _model(qk_norm)
    prompts = [np.arange(3, 40, dtype=np.int32), np.arange(50, 57, dtype=np.int32), np.arange(100, 250, dtype=np.int32)]
    eng = LLMEngine(model, EngineConfig(num_pages=32, max_batched_tokens=64, decode_burst=3, max_model_len=512, kv_cache_dtype="fp8"))
    assert eng.kv_backing.dtype == torch.uint8 and eng.kv_backing.shape == (2, 32, 2, 2, 128 * 36)
    assert eng.kv_backing[:, 0].numel() == model.kv_bytes_per_page("fp8")
    got = eng.generate([Sequence(f"s{i}", p, SamplingParams(max_tokens=5, ignore_eos=True)) for i, p in enumerate(prompts)])
    for i, p in enumerate(prompts):
        ids = list(p)
        for tok in got[f"s{i}"]:
            logits = _full_pass(model, ids)
            # chunked prefill and decode store the same rows; sums in another order may move a logit by rounding only
            assert logits[tok] >= logits.max() - 1e-4
            ids.append(tok)


def test_transfer_of_8_bit_pages_and_its_geometry():
    model = _model()
    eng = lambda kind="fp8": LLMEngine(model, EngineConfig(num_pages=16, max_batched_tokens=256, decode_burst=2, max_model_len=512,  # noqa: E731
                                                           kv_cache_dtype=kind))
    prompts = [np.arange(3 + i, 150 + 40 * i, dtype=np.int32) for i in range(2)]
    mono = eng().generate([Sequence(f"s{i}", p, SamplingParams(6, True)) for i, p in enumerate(prompts)])
    P, D = eng(), eng()
    P.generate([Sequence(f"s{i}", p, SamplingParams(1, True), hold_kv=True) for i, p in enumerate(prompts)])
    seqs = []
    for i in range(2):
        kp = P.kv_transfer_params(f"s{i}")
        src = dict(src_cache=P.kv_backing) if i == 0 else dict(raw=P.read_pages(kp["pages"]))
        seqs.append(Sequence(f"s{i}", np.zeros(kp["num_tokens"], np.int32), SamplingParams(6, True),
                             prefilled=PrefilledKV(kp["first_token"], kp["next_pos"], kp["pages"], **src)))
    assert D.generate(seqs) == mono
    from cornserve.task_executors.llm.server import LLMServer

    srv = LLMServer.__new__(LLMServer)
    srv.engine = types.SimpleNamespace(kv_geometry=D.kv_geometry)
    meta = {"pages": [3], "first_token": 1, "next_pos": 9, "num_tokens": 100, "request_id": "r"}
    srv._check_transfer({**P.kv_geometry(), **meta})
    with pytest.raises(ValueError):     # a bf16 / fp32 producer cannot feed an 8-bit consumer
        srv._check_transfer({**eng("auto").kv_geometry(), **meta})


def test_unknown_cache_type_is_refused():
    with pytest.raises(ValueError):
        LLMEngine(_model(), EngineConfig(num_pages=4, kv_cache_dtype="int4"))


def test_server_option_reaches_the_engine():
    from cornserve.task_executors.llm.server import parse_args

    assert parse_args(["m"]).kv_cache_dtype == "auto"
    assert parse_args(["m", "--kv-cache-dtype", "fp8"]).kv_cache_dtype == "fp8"
    with pytest.raises(SystemExit):
        parse_args(["m", "--kv-cache-dtype", "int4"])


def test_the_option_is_refused_where_it_would_do_nothing(capsys):
    """The talker allocates its caches in the model's type."""
    from cornserve.task_executors.llm.server import parse_args

    with pytest.raises(SystemExit):
        parse_args(["m", "--run-talker", "--kv-cache-dtype", "fp8"])
    assert "--run-talker" in capsys.readouterr().err
    assert parse_args(["m", "--run-talker"]).run_talker and parse_args(["m", "--run-talker", "--kv-cache-dtype", "auto"]).run_talker


@pytest.mark.timeout(600)
def test_two_tensor_parallel_ranks_cache_their_heads():
    """Two gloo ranks: each caches its own key heads, and the engine's hidden states are those of one process."""
    script = os.path.join(os.path.dirname(__file__), "kv_fp8_tp_cpu.py")
    env = dict(os.environ, OMP_NUM_THREADS="2", CUDA_VISIBLE_DEVICES="")
    port = str(free_port())
    procs = [subprocess.Popen([sys.executable, script, str(r), "2", port], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, env=env)
             for r in range(2)]
    outs = [p.communicate(timeout=500)[0] for p in procs]
    assert all(p.returncode == 0 for p in procs) and "KV_FP8_TP_OK" in outs[0], "\n".join(o[-3000:] for o in outs)


def test_server_builds_an_engine_with_the_option(tmp_path, monkeypatch):
    """From the command line to the cache: its type, and as many pages as a GPU's free memory holds at 8 bits."""
    from cornserve.task_executors.llm import server

    (tmp_path / "config.json").write_text(json.dumps({
        "model_type": "qwen2", "architectures": ["Qwen2ForCausalLM"], "hidden_size": 64, "num_hidden_layers": 2, "num_attention_heads": 4,
        "num_key_value_heads": 2, "head_dim": 16, "intermediate_size": 128, "vocab_size": 512, "rms_norm_eps": 1e-6, "rope_theta": 10000.0,
        "max_position_embeddings": 512, "tie_word_embeddings": False, "eos_token_id": 511, "torch_dtype": "float32"}))
    monkeypatch.setenv("CORNSERVE_DEVICE", "cpu")
    args = [str(tmp_path), "--num-kv-pages", "16", "--max-model-len", "512"]
    eng, _ = server.build_engine(server.parse_args([*args, "--kv-cache-dtype", "fp8"]))
    assert eng.cfg.kv_cache_dtype == "fp8" and eng.kv_backing.dtype == torch.uint8 and eng.kv_backing.shape == (2, 16, 2, 2, 128 * 20)
    seqs = lambda: [Sequence("s", np.arange(3, 150, dtype=np.int32), SamplingParams(max_tokens=3, ignore_eos=True))]  # noqa: E731
    assert len(eng.generate(seqs())["s"]) == 3 and eng.kv_backing[:, 1:].any()
    plain, _ = server.build_engine(server.parse_args(args))
    assert plain.kv_backing.dtype == torch.float32 and plain.kv_backing.shape == (2, 16, 2, 2, 128, 16)
    # without --num-kv-pages the pages come from the free memory of the GPU
    made = []
    monkeypatch.setattr(server, "pick_device", lambda: types.SimpleNamespace(type="cuda"))
    monkeypatch.setattr(server.torch.cuda, "set_device", lambda d: None)
    monkeypatch.setattr(server.torch.cuda, "mem_get_info", lambda d: (100 << 30, 180 << 30))
    monkeypatch.setattr(server, "QwenLLM", lambda cfg, group, device: QwenLLM(cfg, group=group, device="cpu").float())
    monkeypatch.setattr(server, "LLMEngine", lambda model, cfg: made.append((model, cfg)) or types.SimpleNamespace(capture_decode_graphs=lambda: 0))
    for kind in ("auto", "fp8"):
        server.build_engine(server.parse_args([str(tmp_path), "--kv-cache-dtype", kind]))
    for model, cfg in made:
        budget = int((100 << 30) * 0.9) - (4 << 30)
        row = 16 + 4 if cfg.kv_cache_dtype == "fp8" else 2 * 16        # bytes of a token and head
        assert cfg.num_pages == budget // (2 * 2 * 2 * 128 * row)
    assert [cfg.kv_cache_dtype for _, cfg in made] == ["auto", "fp8"]
