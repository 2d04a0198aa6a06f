"""Timed cases of the operators around the 8-bit paged key-value cache.

Three operators belong together here: the append, which rotates the new queries and keys and stores keys and values as
e4m3 codes with one fp32 scale per token and head; the attention of one new token per sequence over such a cache; and the
causal attention of packed prompts (or chunks of them) over it.

A case is a dict of plain values.  ``prepare`` makes its inputs on the GPU, ``run`` makes one pass -- in a plain form from
elementary torch operations in fp32, or, with ``own`` set, through ``cornserve.ops`` -- ``work`` counts the bytes and
operations that a pass cannot do without and ``exact`` evaluates the definition in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

PAGE = 128            # tokens per cache page
FP8_MAX = 448.0       # largest e4m3 value
AMAX_FLOOR = 2.0 ** -40   # rows whose largest magnitude is below this share its scale (so a scale is never zero)
EPS = 1e-6


# ---------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------
def listed() -> list[dict]:
    return [
        # one sequence decoding: the append of a single token is launch latency
        _append("append_one_token", tokens=1, hq=28, hkv=4, d=128, norm=False, padded=0, decode=True),
        # a decode step of a full graph bucket of a model that normalises its query and key heads
        _append("append_decode_128_norm", tokens=128, hq=32, hkv=4, d=128, norm=True, padded=5, decode=True),
        # a prefill step of odd length with narrow heads
        _append("append_chunk_1777_narrow", tokens=1777, hq=16, hkv=2, d=64, norm=False, padded=0, decode=False),
        # the largest prefill step the engine schedules (its default token budget)
        _append("append_full_budget", tokens=18944, hq=28, hkv=4, d=128, norm=False, padded=300, decode=False),
        # one user, short conversation: latency
        _decode("decode_1x500", batch=1, low=500, high=500, hq=28, hkv=4, d=128),
        # one user at the default model length: one long sequence spread over the whole GPU
        _decode("decode_1x32768", batch=1, low=32768, high=32768, hq=28, hkv=4, d=128),
        # a mixed batch with narrow heads and two heads per group
        _decode("decode_33_ragged_narrow", batch=33, low=1, high=5000, hq=16, hkv=8, d=64),
        # the served benchmark's shape: images and text, about 3500 tokens of context, the largest bucket
        _decode("decode_256x3500", batch=256, low=3300, high=3700, hq=28, hkv=4, d=128),
        # a single short prompt
        _prefill("prefill_1x300", batch=1, new=(300, 300), cached=(0, 0), hq=28, hkv=4, d=128),
        # a packed step of prompts of different lengths
        _prefill("prefill_9_ragged", batch=9, new=(17, 2300), cached=(0, 0), hq=32, hkv=4, d=128),
        # chunks of prompts whose beginnings are already in the cache, narrow heads
        _prefill("prefill_3_chunks_narrow", batch=3, new=(500, 2100), cached=(1000, 9000), hq=16, hkv=2, d=64),
        # one long document in a single step
        _prefill("prefill_1x16000", batch=1, new=(16000, 16000), cached=(0, 0), hq=28, hkv=4, d=128),
    ]


def _append(name: str | None, **kw) -> dict:
    return {**({"name": name} if name else {}), "op": "append", **kw}


def _decode(name: str | None, **kw) -> dict:
    return {**({"name": name} if name else {}), "op": "decode", **kw}


def _prefill(name: str | None, batch: int, new: tuple, cached: tuple, **kw) -> dict:
    return {**({"name": name} if name else {}), "op": "prefill", "batch": batch, "new_low": new[0], "new_high": new[1],
            "cached_low": cached[0], "cached_high": cached[1], **kw}


def _log_int(rng: random.Random, low: int, high: int) -> int:
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng: random.Random) -> dict:
    """Another case of the same ranges: head layouts from one to 16 query heads per key head, both head widths, lengths
    from one token up to what the largest listed case of the operator costs."""
    hkv, group = rng.choice([(1, 1), (1, 5), (1, 8), (2, 7), (2, 8), (2, 16), (3, 4), (4, 7), (4, 8), (4, 3), (8, 1), (8, 2), (8, 4)])
    d = rng.choice([64, 128, 128])
    heads = dict(hq=hkv * group, hkv=hkv, d=d)
    op = rng.choice(["append", "decode", "decode", "prefill", "prefill"])
    if op == "append":
        decode = rng.random() < 0.4
        tokens = _log_int(rng, 1, 256 if decode else 12000)
        return _append(None, tokens=tokens, norm=rng.random() < 0.5, padded=rng.randint(0, tokens // 8), decode=decode, **heads)
    if op == "decode":
        batch = _log_int(rng, 1, 256)
        high = _log_int(rng, 1, max(1, min(60000, 850_000 // batch)))
        low = rng.choice([1, high, max(1, high // 2)])
        return _decode(None, batch=batch, low=low, high=high, **heads)
    batch = _log_int(rng, 1, 12)
    new_high = _log_int(rng, 1, max(1, 12000 // batch))
    cached = rng.choice([0, 0, _log_int(rng, 1, 12000 // batch)])
    return _prefill(None, batch, (max(1, new_high // rng.choice([1, 3, 20])), new_high), (cached // rng.choice([1, 2]), cached), **heads)


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Per sequence: new tokens and keys in the cache (new ones included).  Fixed by the case, not by the seed, so that
    ``work`` can count them."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    if case["op"] == "decode":
        lens = [rng.randint(case["low"], case["high"]) for _ in range(case["batch"])]
        return [1] * case["batch"], lens
    new = [rng.randint(case["new_low"], case["new_high"]) for _ in range(case["batch"])]
    return new, [n + rng.randint(case["cached_low"], case["cached_high"]) for n in new]


def work(case: dict) -> dict:
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    row = 2 * hkv * (d + 4)                                # key and value codes and scales of one token
    if case["op"] == "append":
        t, kept = case["tokens"], case["tokens"] - case["padded"]
        norm = 4 * d if case["norm"] else 0
        # q of every token, k and v of the kept ones; cos and sin; slots; q written, cache rows written
        return {"bytes": 2 * t * hq * d + 4 * kept * hkv * d + 4 * t * d + 4 * t + norm + 2 * t * hq * d + kept * row,
                "flops": 3 * t * (hq + hkv) * d + 3 * kept * 2 * hkv * d}
    new, lens = _lengths(case)
    pages = sum(-(-n // PAGE) for n in lens)
    pairs = sum(n * L - n * (n - 1) // 2 for n, L in zip(new, lens))
    return {"bytes": sum(lens) * row + 2 * 2 * sum(new) * hq * d + 4 * pages + 8 * len(lens), "flops": 4 * hq * d * pairs}


# ---------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------
def _quantise(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows of fp32 ``x`` as e4m3 codes with one scale per row (the largest magnitude maps to 448)."""
    amax = x.abs().amax(dim=-1)
    scale = amax.clamp_min(AMAX_FLOOR) * (1.0 / FP8_MAX)
    codes = (x * (1.0 / scale)[..., None]).clamp(-FP8_MAX, FP8_MAX).to(torch.float8_e4m3fn)
    return codes, scale


def _views(cache: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes [pages, 2, hkv, 128, d] and scales [pages, 2, hkv, 128] of a cache [pages, 2, hkv, 128 * (d + 4)] of bytes:
    every block holds its 128 rows of codes, then their 128 fp32 scales."""
    pages, two, hkv, block = cache.shape
    d = block // PAGE - 4
    codes = cache[..., : PAGE * d].view(torch.float8_e4m3fn).unflatten(-1, (PAGE, d))
    return codes, cache[..., PAGE * d:].view(torch.float32)


def _make_cache(pages: int, hkv: int, d: int, gen: torch.Generator) -> torch.Tensor:
    """A cache in use: keys with a few strong channels and an offset, values whose size differs from token to token."""
    cache = torch.zeros((pages, 2, hkv, PAGE * (d + 4)), device="cuda", dtype=torch.uint8)
    codes, scales = _views(cache)
    chan = torch.exp(0.6 * torch.randn(hkv, 1, d, device="cuda", generator=gen))
    bias = 0.7 * torch.randn(hkv, 1, d, device="cuda", generator=gen)
    for p in range(0, pages, 512):
        n = min(512, pages - p)
        k = torch.randn(n, hkv, PAGE, d, device="cuda", generator=gen) * chan + bias
        v = torch.randn(n, hkv, PAGE, d, device="cuda", generator=gen)
        v *= torch.exp(0.5 * torch.randn(n, hkv, PAGE, 1, device="cuda", generator=gen))
        for i, x in enumerate((k, v)):
            c, s = _quantise(x.bfloat16().float())
            codes[p: p + n, i].view(torch.uint8).copy_(c.view(torch.uint8))
            scales[p: p + n, i] = s
    return cache


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "append":
        t = case["tokens"]
        pages = t + 2 if case["decode"] else -(-t // PAGE) + 3
        cache = _make_cache(pages, hkv, d, gen)
        qkv = torch.randn(t, (hq + 2 * hkv) * d, device="cuda", generator=gen)
        qkv[:, : (hq + hkv) * d] *= torch.exp(0.5 * torch.randn((hq + hkv) * d, device="cuda", generator=gen))
        order = list(range(pages))
        host.shuffle(order)
        if case["decode"]:      # every token belongs to its own sequence: one row of one page each
            slots = [order[i] * PAGE + host.randrange(PAGE) for i in range(t)]
            pos = [host.randrange(32768) for _ in range(t)]
        else:                   # consecutive tokens of a chunk that starts inside a page
            first, start = host.randrange(PAGE), host.randrange(8192)
            slots = [order[(first + i) // PAGE] * PAGE + (first + i) % PAGE for i in range(t)]
            pos = [start + i for i in range(t)]
        for i in host.sample(range(t), case["padded"]):
            slots[i] = -1
        inv = 1e6 ** (-torch.arange(d // 2, dtype=torch.float64, device="cuda") * 2.0 / d)
        ang = torch.tensor(pos, dtype=torch.float64, device="cuda")[:, None] * inv[None, :]
        weight = lambda: (1.0 + 0.2 * torch.randn(d, device="cuda", generator=gen)).bfloat16()  # noqa: E731
        return {"op": "append", "hq": hq, "hkv": hkv, "d": d, "qkv": qkv.bfloat16(), "cache": cache,
                "cs": torch.stack([ang.cos(), ang.sin()], dim=1).float().contiguous(),
                "slot": torch.tensor(slots, dtype=torch.int32, device="cuda"),
                "kept": torch.tensor([i for i, s in enumerate(slots) if s >= 0], dtype=torch.int64, device="cuda"),
                "q_norm": weight() if case["norm"] else None, "k_norm": weight() if case["norm"] else None}
    new, lens = _lengths(case)
    blocks = [-(-n // PAGE) for n in lens]
    pages = sum(blocks) + 2
    order = list(range(1, pages))
    host.shuffle(order)
    table = torch.zeros(len(lens), max(blocks) + 1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(blocks):
        table[i, :n] = torch.tensor(order[at: at + n], dtype=torch.int32)
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], hq, d, device="cuda", generator=gen) * torch.exp(0.3 * torch.randn(hq, 1, device="cuda", generator=gen))
    return {"op": case["op"], "hq": hq, "hkv": hkv, "d": d, "q": q.bfloat16(), "cache": _make_cache(pages, hkv, d, gen),
            "table": table.cuda(), "kv_len": torch.tensor(lens, dtype=torch.int32, device="cuda"),
            "cu_q": torch.tensor(cu, dtype=torch.int32, device="cuda"), "new": new, "lens": lens}


# ---------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------
def run(state: dict):
    if own:
        return _run_own(state)
    if state["op"] == "append":
        return _plain_append(state)
    return _plain_decode(state) if state["op"] == "decode" else _plain_prefill(state)


def _run_own(st: dict):
    from cornserve import ops

    if st["op"] == "append":
        q = ops.rope_kv_write_fp8_(st["qkv"], st["hq"], st["hkv"], st["d"], st["cs"], st["cache"], st["slot"],
                                   q_norm=st["q_norm"], k_norm=st["k_norm"], eps=EPS)
        codes, scales = ops.kv_cache_fp8_views(st["cache"])
        return {"q": q, "codes": codes, "scales": scales}
    return ops.attention_paged_fp8(st["q"], st["cache"], st["table"], st["kv_len"], st["cu_q"], max(st["new"]))


def _rotate(x: torch.Tensor, cs: torch.Tensor) -> torch.Tensor:
    half = x.shape[-1] // 2
    cos, sin = cs[:, None, 0], cs[:, None, 1]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_append(st: dict):
    hq, hkv, d = st["hq"], st["hkv"], st["d"]
    x = st["qkv"].float().unflatten(-1, (hq + 2 * hkv, d))
    qk, v = x[:, : hq + hkv], x[:, hq + hkv:]
    if st["q_norm"] is not None:
        w = torch.cat([st["q_norm"].float().expand(hq, d), st["k_norm"].float().expand(hkv, d)])
        qk = qk * torch.rsqrt((qk * qk).mean(dim=-1, keepdim=True) + EPS) * w
    qk = _rotate(qk, st["cs"])
    codes, scales = _views(st["cache"])
    raw = codes.view(torch.uint8)                    # indexed stores move bytes
    kept = st["kept"]
    slot = st["slot"][kept].long()
    page, row = slot // PAGE, slot % PAGE
    for i, rows in enumerate((qk[:, hq:][kept], v[kept])):
        c, s = _quantise(rows)
        raw[page, i, :, row] = c.view(torch.uint8)
        scales[page, i, :, row] = s
    return {"q": qk[:, :hq].bfloat16(), "codes": codes, "scales": scales}


def _gather(st: dict, seqs: slice, blocks: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Keys and values [sequences, hkv, blocks * 128, d] in fp32 of the first ``blocks`` pages of some sequences."""
    codes, scales = _views(st["cache"])
    idx = st["table"][seqs, :blocks].long()
    out = []
    for i in (0, 1):
        c = codes.view(torch.uint8)[idx, i].view(torch.float8_e4m3fn).float()     # [n, blocks, hkv, 128, d]
        out.append((c * scales[idx, i][..., None]).transpose(1, 2).flatten(2, 3))
    return out[0], out[1]


def _plain_decode(st: dict) -> torch.Tensor:
    hq, hkv, d, lens = st["hq"], st["hkv"], st["d"], st["lens"]
    B = len(lens)
    out = torch.empty_like(st["q"])
    step = max(1, 2_000_000 // max(lens))            # sequences at a time: bounds the expanded keys
    for b in range(0, B, step):
        seqs = slice(b, min(B, b + step))
        k, v = _gather(st, seqs, -(-max(lens[seqs]) // PAGE))
        q = st["q"][seqs].float().unflatten(1, (hkv, hq // hkv))
        s = (q @ k.transpose(-1, -2)) * d ** -0.5
        hidden = torch.arange(k.shape[2], device="cuda")[None, :] >= st["kv_len"][seqs, None]
        s = s.masked_fill(hidden[:, None, None, :], float("-inf"))
        p = torch.exp(s - s.amax(dim=-1, keepdim=True))
        out[seqs] = ((p @ v) / p.sum(dim=-1, keepdim=True)).flatten(1, 2).bfloat16()
    return out


def _plain_prefill(st: dict) -> torch.Tensor:
    hq, hkv, d = st["hq"], st["hkv"], st["d"]
    out = torch.empty_like(st["q"])
    at = 0
    for i, (n, L) in enumerate(zip(st["new"], st["lens"])):
        k, v = _gather(st, slice(i, i + 1), -(-L // PAGE))
        step = max(16, 300_000_000 // (hq * L))      # queries at a time: bounds the score matrix
        for a in range(0, n, step):
            m = min(step, n - a)
            end = L - n + a + m                      # keys visible to the last query of the block
            q = st["q"][at + a: at + a + m].float().unflatten(1, (hkv, hq // hkv)).permute(1, 2, 0, 3)
            s = (q @ k[0, :, None, :end].transpose(-1, -2)) * d ** -0.5
            pos = torch.arange(end - m, end, device="cuda")
            s = s.masked_fill(torch.arange(end, device="cuda")[None, :] > pos[:, None], float("-inf"))
            p = torch.exp(s - s.amax(dim=-1, keepdim=True))
            o = (p @ v[0, :, None, :end]) / p.sum(dim=-1, keepdim=True)
            out[at + a: at + a + m] = o.permute(2, 0, 1, 3).flatten(1, 2).bfloat16()
        at += n
    return out


# ---------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ---------------------------------------------------------------------------------------------------------------
def exact(case: dict, seed: int):
    st = prepare(case, seed)
    hq, hkv, d = st["hq"], st["hkv"], st["d"]
    group = hq // hkv
    codes, scales = _views(st["cache"])
    if st["op"] == "append":
        t = case["tokens"]
        x = st["qkv"].double().view(t, hq + 2 * hkv, d)
        if st["q_norm"] is not None:
            rms = torch.sqrt(x.square().sum(dim=2, keepdim=True) / d + EPS)
            x[:, :hq] = x[:, :hq] / rms[:, :hq] * st["q_norm"].double()
            x[:, hq: hq + hkv] = x[:, hq: hq + hkv] / rms[:, hq: hq + hkv] * st["k_norm"].double()
        half = torch.complex(x[:, : hq + hkv, : d // 2], x[:, : hq + hkv, d // 2:])
        turn = torch.complex(st["cs"][:, 0].double(), st["cs"][:, 1].double())
        half = half * turn[:, None, :]
        x[:, : hq + hkv] = torch.cat([half.real, half.imag], dim=2)
        codes, scales = codes.double(), scales.double()
        slot = st["slot"].tolist()
        keep = torch.tensor([s >= 0 for s in slot], device="cuda")
        where = torch.tensor([s for s in slot if s >= 0], device="cuda", dtype=torch.int64)
        for i, lo in ((0, hq), (1, hq + hkv)):
            rows = x[keep, lo: lo + hkv]
            unit = torch.clamp(rows.abs().max(dim=2).values, min=AMAX_FLOOR) / FP8_MAX
            codes[where // PAGE, i, :, where % PAGE] = rows / unit[:, :, None]
            scales[where // PAGE, i, :, where % PAGE] = unit
        return {"q": x[:, :hq].contiguous(), "codes": codes, "scales": scales}
    out = torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64)
    table = st["table"].tolist()
    row = 0
    for i, (n, L) in enumerate(zip(st["new"], st["lens"])):
        ids = torch.tensor(table[i][: (L + PAGE - 1) // PAGE], device="cuda")
        for h in range(hkv):
            k, v = ((codes[ids, j, h].double() * scales[ids, j, h].double()[:, :, None]).reshape(-1, d)[:L] for j in (0, 1))
            step = max(1, 60_000_000 // (group * L))
            for a in range(0, n, step):
                b = min(n, a + step)
                seen = L - n + b
                q = st["q"][row + a: row + b, h * group: (h + 1) * group].double()
                s = torch.einsum("qgd,kd->gqk", q, k[:seen]) / math.sqrt(d)
                if n > 1:
                    first_hidden = torch.arange(L - n + a + 1, L - n + b + 1, device="cuda")
                    s += torch.where(torch.arange(seen, device="cuda")[None, :] < first_hidden[:, None], 0.0, -math.inf)
                out[row + a: row + b, h * group: (h + 1) * group] = torch.einsum("gqk,kd->qgd", torch.softmax(s, dim=-1), v[:seen])
        row += n
    return out
