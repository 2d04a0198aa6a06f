"""The 8-bit paged key-value cache on the GPU: the append and the attention against their definitions in 64 bits.

Tolerances.  A stored code is off by at most half a step of e4m3: 2^-4 of the value, 2^-10 among the subnormal codes.  A
bf16 output is off by 2^-8 of its value.  Inside the attention a key's weight (probability times value scale) may be rounded
to fp16: off by 2^-11 of it, or by half a step of the subnormals, 2^-25, where the largest weight is at least 2^6; so by
2^-31 of the largest, for every code of the row.  With more than one query per sequence the keys and values themselves
(code times scale) are rounded to fp16 once: off by 2^-11 of them, or by half a step of the subnormals, which is at most
2^-30 of the largest scale of their page (a power of two brings that scale to at least 2^6).
Scores are fp32 sums whose error is at most (d + 4) * 2^-24 times the sum of the magnitudes of
their products, and an error e of a score changes its probability, and at most as much the normaliser, by e.
"""

import math

import pytest
import torch

from cornserve import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def _no_kernel_error():
    yield
    torch.cuda.synchronize()
    ops.check_error("after test")


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device=DEV)


def _cs(T, d, start=0):
    ang = (start + torch.arange(T, dtype=torch.float64, device=DEV))[:, None] * \
        1e6 ** (-torch.arange(d // 2, dtype=torch.float64, device=DEV) * 2 / d)
    return torch.stack([ang.cos(), ang.sin()], dim=1).float().contiguous()


def _rows(cache, slots):
    codes, scales = ops.kv_cache_fp8_views(cache)
    p, r = slots.long() // 128, slots.long() % 128
    return codes.view(torch.uint8)[p, :, :, r].view(torch.float8_e4m3fn).double(), scales[p, :, :, r].double()


# ---------------------------------------------------------------------------------------------------------------------
# append
# ---------------------------------------------------------------------------------------------------------------------
def _append_definition(qkv, Hq, Hkv, d, cs, wq, wk, eps):
    x = qkv.double().view(qkv.shape[0], Hq + 2 * Hkv, d)
    qk = x[:, : Hq + Hkv]
    if wq is not None:
        w = torch.cat([wq.double().expand(Hq, d), wk.double().expand(Hkv, d)])
        qk = qk / (qk.square().mean(-1, True) + eps).sqrt() * w
    c, s = cs.double()[:, None, 0], cs.double()[:, None, 1]
    a, b = qk[..., : d // 2], qk[..., d // 2:]
    qk = torch.cat([a * c - b * s, b * c + a * s], -1)
    return qk[:, :Hq], torch.stack([qk[:, Hq:], x[:, Hq + Hkv:]], 1)      # [T, Hq, d], [T, 2, Hkv, d]


@pytest.mark.parametrize("T,Hq,Hkv,d", [(1, 28, 4, 128), (1, 1, 1, 64), (5, 16, 2, 64), (300, 28, 4, 128), (129, 3, 3, 64), (2049, 32, 8, 128)])
@pytest.mark.parametrize("norm", [False, True])
def test_append_matches_the_definition(T, Hq, Hkv, d, norm):
    torch.manual_seed(T + d + norm)
    pages = T // 128 + 4
    qkv = (torch.randn(T, (Hq + 2 * Hkv) * d, device=DEV) * torch.exp(torch.randn(T, 1, device=DEV))).bfloat16()
    cs = _cs(T, d, 77)
    wq, wk = ((1 + 0.1 * torch.randn(d, device=DEV)).bfloat16() for _ in range(2)) if norm else (None, None)
    cache = torch.randint(0, 120, ops.kv_cache_fp8(pages, Hkv, d).shape, device=DEV, dtype=torch.uint8)
    slot = (100 + torch.randperm(pages * 128 - 100, device=DEV)[:T]).int()
    slot[::9] = -1
    before, qkv_before = cache.clone(), qkv.clone()
    q = ops.rope_kv_write_fp8_(qkv, Hq, Hkv, d, cs, cache, slot, wq, wk, 1e-5)
    want_q, want_kv = _append_definition(qkv, Hq, Hkv, d, cs, wq, wk, 1e-5)
    assert torch.equal(qkv, qkv_before)
    amp = want_q.abs().amax(-1, keepdim=True)
    assert ((q.double() - want_q).abs() <= want_q.abs() * 2 ** -8 + amp * 2 ** -20).all()
    kept = slot >= 0
    codes, scales = _rows(cache, slot[kept])
    want = want_kv[kept]
    unit = want.abs().amax(-1).clamp_min(2.0 ** -40) / 448
    assert ((scales - unit).abs() <= unit * 2 ** -20).all()
    assert ((codes - want / unit[..., None]).abs() <= (want / unit[..., None]).abs() * (2 ** -4 + 2 ** -18) + 2 ** -10 + 2 ** -12).all()
    # every byte that belongs to no kept token is as it was
    c, s = ops.kv_cache_fp8_views(cache)
    c0, s0 = ops.kv_cache_fp8_views(before)
    p, r = slot[kept].long() // 128, slot[kept].long() % 128
    c.view(torch.uint8)[p, :, :, r] = c0.view(torch.uint8)[p, :, :, r]
    s.view(torch.int32)[p, :, :, r] = s0.view(torch.int32)[p, :, :, r]
    assert torch.equal(cache, before)


def test_append_zero_tiny_huge_and_non_finite_rows_match_the_cpu():
    d, Hq, Hkv, T = 128, 1, 1, 8
    qkv = torch.zeros(T, 3 * d, device=DEV).bfloat16()
    qkv[1] = 1e-30
    qkv[2, d + 3] = float("inf")
    qkv[3, 2 * d + 4] = float("nan")
    qkv[4] = 3e38
    qkv[5, 2 * d:] = -2.0 ** -40
    qkv[6, 2 * d + 7] = float("-inf")
    qkv[7] = 2.0 ** -133
    cs = _cs(T, d)
    cache = ops.kv_cache_fp8(1, Hkv, d, DEV)
    ops.rope_kv_write_fp8_(qkv, Hq, Hkv, d, cs, cache, _i32(list(range(T))))
    host = ops.kv_cache_fp8(1, Hkv, d)
    ops.rope_kv_write_fp8_(qkv.cpu().float(), Hq, Hkv, d, cs.cpu(), host, torch.arange(T, dtype=torch.int32))
    (c, s), (hc, hs) = ops.kv_cache_fp8_views(cache), ops.kv_cache_fp8_views(host)
    # rows 2, 3 and 6, and the key of row 4: its rotation by 4 radians reaches 3e38 * |cos 4 + sin 4| = 4.2e38, beyond fp32
    assert torch.equal(torch.isnan(s).cpu(), torch.isnan(hs)) and int(torch.isnan(hs).sum()) == 4
    ok = ~torch.isnan(hs)
    assert torch.allclose(s.cpu()[ok], hs[ok], rtol=2 ** -20, atol=0)
    # codes: at most one step apart (their fp32 inputs may differ in the last bit next to a rounding border)
    assert ((c.cpu().double() - hc.double()).abs() <= hc.double().abs() * 2 ** -3 + 2 ** -9).all()


def test_append_takes_strided_and_misaligned_rows_and_empty_batches():
    torch.manual_seed(1)
    d, Hq, Hkv, T = 64, 2, 1, 10
    wide = torch.randn(T, 4 * d + 5, device=DEV).bfloat16()
    cs, slot = _cs(T, d), torch.arange(T, device=DEV, dtype=torch.int32)
    ref_cache = ops.kv_cache_fp8(1, Hkv, d, DEV)
    ref_q = ops.rope_kv_write_fp8_(wide[:, 3: 3 + 4 * d].contiguous(), Hq, Hkv, d, cs, ref_cache, slot)
    cache = ops.kv_cache_fp8(1, Hkv, d, DEV)
    q = ops.rope_kv_write_fp8_(wide[:, 3: 3 + 4 * d], Hq, Hkv, d, cs, cache, slot)
    assert torch.equal(q, ref_q) and torch.equal(cache, ref_cache)
    q = ops.rope_kv_write_fp8_(wide[:0, : 4 * d], Hq, Hkv, d, cs[:0], cache, slot[:0])
    assert q.shape == (0, Hq, d) and torch.equal(cache, ref_cache)


def test_a_slot_beyond_the_cache_is_skipped_and_reported():
    d = 64
    cache = ops.kv_cache_fp8(2, 1, d, DEV)
    x = torch.ones(3, 3 * d, device=DEV).bfloat16()
    ops.rope_kv_write_fp8_(x, 1, 1, d, _cs(3, d), cache, _i32([256, 2**31 - 1, 5]))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.check_error("append")
    codes, _ = ops.kv_cache_fp8_views(cache)
    assert int((codes.float().abs().sum(-1) > 0).sum()) == 2     # the key and value row of slot 5


# ---------------------------------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------------------------------
def _filled_cache(pages, Hkv, d, seed=0):
    """Every byte of the cache is something: rows of different sizes, and rows no sequence may look at."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    cache = ops.kv_cache_fp8(pages, Hkv, d, DEV)
    codes, scales = ops.kv_cache_fp8_views(cache)
    raw = torch.randint(0, 256, codes.shape, device=DEV, generator=g, dtype=torch.int32).to(torch.uint8)
    raw[(raw & 0x7F) == 0x7F] = 0x35
    codes.view(torch.uint8).copy_(raw)
    scales.copy_(torch.exp(0.7 * torch.randn(scales.shape, device=DEV, generator=g)) / 150)
    return cache


def _poison(cache, table, lens):
    """NaN codes and NaN / infinite scales in every row that lies behind a sequence's keys."""
    codes, scales = ops.kv_cache_fp8_views(cache)
    used = torch.zeros(cache.shape[0], 128, dtype=torch.bool)
    for row, n in zip(table.tolist(), lens):
        for b in range(-(-n // 128)):
            used[row[b], : min(128, n - 128 * b)] = True
    hide = (~used).to(DEV)[:, None, None, :].expand(scales.shape)
    codes.view(torch.uint8)[hide] = 0x7F
    scales[hide] = float("nan")
    scales[:, 1][hide[:, 1]] = float("inf")


def _check(out, q, cache, table, lens, new, causal=True, scale=None):
    codes, scales = ops.kv_cache_fp8_views(cache)
    _, Hq, d = q.shape
    Hkv = cache.shape[2]
    group = Hq // Hkv
    scale = scale if scale is not None else 1 / math.sqrt(d)
    at = 0
    for i, (n, L) in enumerate(zip(new, lens)):
        ids = table[i, : -(-L // 128)].long()
        k, v = ((codes[ids, j].double() * scales[ids, j].double()[..., None]).transpose(1, 2).reshape(-1, Hkv, d)[:L]
                .repeat_interleave(group, dim=1) for j in (0, 1))
        vs = scales[ids, 1].double().transpose(1, 2).reshape(-1, Hkv)[:L].repeat_interleave(group, dim=1)     # [keys, Hq]
        qq = q[at: at + n].double()
        got = out[at: at + n].double()
        at += n
        if n == 0:
            continue
        vis = torch.ones(n, L, dtype=torch.bool, device=DEV)
        if causal:
            vis = torch.arange(L, device=DEV)[None] <= torch.arange(n, device=DEV)[:, None] + (L - n)
        dead = ~vis.any(dim=1)
        s = torch.einsum("qhd,khd->hqk", qq, k) * scale
        mag = torch.einsum("qhd,khd->hqk", qq.abs(), k.abs()) * abs(scale)
        p = torch.softmax(s.masked_fill(~vis, float("-inf")), -1).masked_fill(dead[:, None], 0.0)
        want = torch.einsum("hqk,khd->qhd", p, v)
        size = torch.einsum("hqk,khd->qhd", p, v.abs())
        prompt = max(new) > 1
        es = mag * ((d + 4) * 2.0 ** -24 + (2.0 ** -11 if prompt else 0.0))
        tiny_v = 0.0
        if prompt and L:
            ks_top, vs_top = (scales[ids, j].nan_to_num(0.0, 0.0, 0.0).double().masked_fill(
                torch.arange(ids.numel() * 128, device=DEV).view(-1, 1, 128) >= L, 0.0).amax(-1).repeat_interleave(128, dim=0)[:L]
                .repeat_interleave(group, dim=1) for j in (0, 1))                       # [keys, Hq]
            es = es + torch.einsum("qh,kh->hqk", qq.abs().sum(-1), ks_top) * abs(scale) * 2.0 ** -30
            tiny_v = torch.einsum("hqk,kh->qh", p, vs_top)[..., None] * 2.0 ** -30
            # here a key's weight is its probability times a power of two within a factor of two of its page's largest value
            # scale (up to a constant), so the step of the smallest weights is at most 2^-30 of the largest such product
            vs = vs_top.clamp_min(1e-30)
        es = es.masked_fill(~vis, 0.0).amax(-1).transpose(0, 1)[..., None] if L else 0.0
        top = (p * vs.t()[:, None, :]).amax(-1).transpose(0, 1)[..., None] if L else 0.0     # the largest weight of a row
        code_sum = torch.einsum("qk,khd->qhd", vis.double(), (v / vs[..., None]).abs()) if L else 0.0
        tol = want.abs() * 2.0 ** -8 + size * (2.0 ** -11 + (2.0 ** -11 if prompt else 0.0) + 2 * es + 2.0 ** -18) + top * code_sum * 2.0 ** (-30 if prompt else -31) + tiny_v
        assert not got[dead].any()
        err = (got - want).abs()
        assert (err <= tol).all(), f"sequence {i}: {n} of {L} keys, error {err.max().item():.3g} beyond tolerance by {(err - tol).max().item():.3g}"


def _setup(lens, new, Hq, Hkv, d, seed=0, spare=3, poison=True):
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    blocks = [-(-n // 128) for n in lens]
    pages = sum(blocks) + spare
    cache = _filled_cache(pages, Hkv, d, seed)
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = torch.full((len(lens), max(blocks + [1]) + 1), -7, dtype=torch.int32)      # unused entries are never read as pages
    for i, n in enumerate(blocks):
        table[i, :n] = torch.tensor([order.pop() for _ in range(n)], dtype=torch.int32)
    if poison:
        _poison(cache, table, lens)
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    q = torch.randn(cu[-1], Hq, d, device=DEV, generator=g) * torch.exp(torch.randn(cu[-1], Hq, 1, device=DEV, generator=g))
    return q.bfloat16(), cache, table.to(DEV), _i32(lens), _i32(cu)


HEADS = [(28, 4, 128), (16, 16, 64), (8, 1, 128), (32, 2, 64), (6, 2, 64), (5, 1, 128), (20, 1, 64), (40, 2, 128)]


@pytest.mark.parametrize("Hq,Hkv,d", HEADS)
@pytest.mark.parametrize("lens", [[1], [128], [129, 64, 65, 63, 1, 0, 127], [700, 0, 3000, 17], [5000], [300] * 70])
def test_decode_attention(Hq, Hkv, d, lens):
    new = [1] * len(lens)
    q, cache, table, kv_len, cu = _setup(lens, new, Hq, Hkv, d, seed=len(lens))
    out = ops.attention_paged_fp8(q, cache, table, kv_len, cu, 1)
    _check(out, q, cache, table, lens, new)


@pytest.mark.parametrize("Hq,Hkv,d", HEADS)
@pytest.mark.parametrize("lens,new", [([1], [1]), ([2], [2]), ([300], [300]), ([128, 129, 127, 1], [128, 129, 127, 1]),
                                      ([500, 20, 0, 64, 900], [3, 20, 0, 30, 257]), ([10, 5, 300], [12, 9, 2]), ([4100], [37])])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_attention(Hq, Hkv, d, lens, new, causal):
    q, cache, table, kv_len, cu = _setup(lens, new, Hq, Hkv, d, seed=len(lens) + sum(new))
    out = ops.attention_paged_fp8(q, cache, table, kv_len, cu, max(new), causal=causal)
    _check(out, q, cache, table, lens, new, causal)


def test_long_prompt_attention():
    lens, new = [2500, 1700], [2500, 1025]
    q, cache, table, kv_len, cu = _setup(lens, new, 14, 2, 128, seed=5)
    _check(ops.attention_paged_fp8(q, cache, table, kv_len, cu, 2500), q, cache, table, lens, new)


@pytest.mark.parametrize("new", [[1, 1, 1], [40, 3, 77]])
@pytest.mark.parametrize("scale", [None, 0.0, 0.5, -0.1])
def test_strides_given_output_rows_behind_the_last_sequence_and_scale(new, scale):
    lens = [200, 130, 90]
    q, cache, table, kv_len, cu = _setup(lens, new, 8, 2, 64, seed=9)
    T = q.shape[0]
    wide = torch.full((T + 4, 8 * 64 + 11), 3.0, device=DEV, dtype=torch.bfloat16)
    qs = wide[:, 5: 5 + 512].unflatten(1, (8, 64))       # odd row stride, odd start
    qs[:T] = q
    hs = torch.empty(8, T + 4, 64, device=DEV, dtype=torch.bfloat16).transpose(0, 1)     # heads outermost
    hs[:T] = q
    big_table = torch.full((3, 40), -9, device=DEV, dtype=torch.int32)
    big_table[:, : table.shape[1]] = table
    for x in (qs, hs):
        out = torch.full((T + 4, 8, 100), 7.0, device=DEV, dtype=torch.bfloat16)
        if new == [1, 1, 1]:
            x, out = x[:T], out[:T]       # one token per sequence: as many rows as sequences
        got = ops.attention_paged_fp8(x, cache, big_table, kv_len, cu, max(new), scale=scale, out=out[..., 9:73])
        assert got.data_ptr() == out[..., 9:73].data_ptr()
        assert (out[T:] == 7.0).all() and (out[..., :9] == 7.0).all() and (out[..., 73:] == 7.0).all()
        _check(out[:T, :, 9:73], q, cache, table, lens, new, scale=scale)


@pytest.mark.parametrize("Hq,Hkv,d", [(5, 1, 128), (14, 2, 64)])
@pytest.mark.parametrize("offset,width", [(0, 0), (8, 8), (1, 1)])     # 16-byte stores, and single elements
def test_outputs_of_warps_with_rows_that_are_no_queries(Hq, Hkv, d, offset, width):
    """Tiles that end inside a warp (5 and 7 heads do not divide 128 rows, and few tokens do not fill a tile), in items of one
    CTA and in items that are cut: every lane of such a warp takes part in reading the sums, and only queries are written."""
    lens, new = [4100, 130, 70], [37, 3, 26]
    q, cache, table, kv_len, cu = _setup(lens, new, Hq, Hkv, d, seed=19)
    T = q.shape[0]
    out = torch.full((T + 2, Hq, d + width), 7.0, device=DEV, dtype=torch.bfloat16)
    mine = out[..., offset: offset + d]
    ops.attention_paged_fp8(torch.cat([q, q[:2]]), cache, table, kv_len, cu, max(new), out=mine)
    assert (out[T:] == 7.0).all() and (out[..., :offset] == 7.0).all() and (out[..., offset + d:] == 7.0).all()
    _check(mine[:T], q, cache, table, lens, new)


@pytest.mark.parametrize("n", [1, 20])
def test_extreme_scores_scales_and_queries(n):
    """One key that outweighs all others; value rows whose sizes differ by 2^60; queries of 2^-60 and 2^60."""
    lens, new = [700, 700, 700, 700], [n] * 4
    q, cache, table, kv_len, cu = _setup(lens, new, 8, 2, 64, seed=11)
    codes, scales = ops.kv_cache_fp8_views(cache)
    p = table[0].long()
    scales[p[2], 0, :, 17] = 5.0                       # sequence 0: a key far larger than the others
    scales[table[1, :5].long(), 1] *= 2.0 ** 40        # sequence 1: large values, and one page of tiny ones
    scales[table[1, 1].long(), 1] *= 2.0 ** -60
    scales[table[1, 5].long(), 1, :, : 700 - 640] *= 2.0 ** 40
    q[2 * n: 3 * n] *= 2.0 ** -60
    scales[table[3, :5].long(), 0] *= 2.0 ** -60       # sequence 3: tiny keys, huge queries
    scales[table[3, 5].long(), 0, :, : 700 - 640] *= 2.0 ** -60
    q[3 * n:] *= 2.0 ** 60
    _check(ops.attention_paged_fp8(q, cache, table, kv_len, cu, n), q, cache, table, lens, new)


@pytest.mark.parametrize("n", [1, 20])
def test_a_nan_row_spreads_only_to_the_queries_that_see_it(n):
    lens, new = [300, 300], [n, n]
    q, cache, table, kv_len, cu = _setup(lens, new, 4, 2, 128, seed=12)
    codes, scales = ops.kv_cache_fp8_views(cache)
    page, row = int(table[0, 2]), 300 - 257                 # the last key of sequence 0
    scales[page, 0, 1, row] = float("nan")                  # its key, second key head
    scales[page, 1, 0, row] = float("nan")                  # its value, first key head
    codes.view(torch.uint8)[page, :, :, row] = 0
    out = ops.attention_paged_fp8(q, cache, table, kv_len, cu, n)
    assert torch.isnan(out[n - 1]).all()
    assert not torch.isnan(out[: n - 1]).any() and not torch.isnan(out[n:]).any()


@pytest.mark.parametrize("n", [1, 20])
def test_a_query_that_is_no_number_spoils_its_own_row_only(n):
    lens, new = [300, 70], [n, n]
    q, cache, table, kv_len, cu = _setup(lens, new, 14, 2, 128, seed=15)
    q[0, 3, 5] = float("nan")
    q[0, 4, 127] = float("inf")
    q[n, 13, 0] = float("-inf")
    q[2 * n - 1, 0] = 0.0
    out = ops.attention_paged_fp8(q, cache, table, kv_len, cu, n)
    bad = torch.zeros(2 * n, 14, dtype=torch.bool, device=DEV)
    bad[0, 3] = bad[0, 4] = bad[n, 13] = True
    assert torch.isnan(out[bad]).all() and torch.isfinite(out[~bad]).all()
    clean = q.clone()
    clean[bad] = 0.0
    got = torch.where(bad[..., None], ops.attention_paged_fp8(clean, cache, table, kv_len, cu, n), out)
    _check(got, clean, cache, table, lens, new)


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("L", [1, 12, 300, 5000])
def test_scores_that_are_all_minus_infinity_give_nan_and_no_keys_give_zero(n, d, L):
    """As the definition has it (0 / 0), in items of one CTA and in items that are cut; the other head is not touched."""
    blocks = -(-L // 128)
    cache = ops.kv_cache_fp8(blocks, 1, d, DEV)
    codes, scales = ops.kv_cache_fp8_views(cache)
    codes.view(torch.uint8).fill_(0x38)      # 1.0
    scales.fill_(1.0)
    q = torch.zeros(n, 2, d, device=DEV, dtype=torch.bfloat16)
    q[:, 0, 0] = float("-inf")
    out = ops.attention_paged_fp8(q, cache, torch.arange(blocks, device=DEV, dtype=torch.int32)[None], _i32([L]), _i32([0, n]), n)
    unseeing = max(0, n - L)                 # queries ahead of the first key
    assert not out[:unseeing].any()
    assert torch.isnan(out[unseeing:, 0]).all() and (out[unseeing:, 1] == 1.0).all()


@pytest.mark.parametrize("n", [1, 20])
def test_a_scale_that_is_no_number_gives_nan(n):
    q, cache, table, kv_len, cu = _setup([300, 70], [n, n], 14, 2, 128, seed=22)
    assert torch.isnan(ops.attention_paged_fp8(q, cache, table, kv_len, cu, n, scale=math.nan)).all()


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("scale", [None, -0.1])
def test_queries_of_very_different_sizes_leave_each_other_alone(n, d, scale):
    """Queries of one tile 2^20 to 2^100 times larger or smaller than their neighbours, which stay right.

    In the prompt kernel rows share nothing, so they keep every bit.  Where single tokens are decoded, a head that moves the
    reference of its weights moves those of the other heads of its warp with it, which rounds their weights anew: they are held
    to the definition instead (an error e of a weight relative to it is at most 2^-11, as everywhere here)."""
    lens, new = [300, 70], [n, n]
    q, cache, table, kv_len, cu = _setup(lens, new, 14, 2, d, seed=18)
    want = ops.attention_paged_fp8(q, cache, table, kv_len, cu, n, scale=scale)
    _check(want, q, cache, table, lens, new, scale=scale)
    mine = torch.zeros(2 * n, 14, dtype=torch.bool, device=DEV)
    mine[0, 3] = mine[n - 1, 9] = mine[2 * n - 1, 13] = True

    def others_are_right(x):
        got = ops.attention_paged_fp8(x, cache, table, kv_len, cu, n, scale=scale)
        _check(torch.where(mine[..., None], want, got), q, cache, table, lens, new, scale=scale)
        assert n == 1 or torch.equal(got[~mine], want[~mine])
        return got

    for power in (20, 28, 32, 40, 60, 100):
        others_are_right(torch.where(mine[..., None], q * 2.0 ** power, q))
    others_are_right(torch.where(mine[..., None], torch.full_like(q, torch.finfo(q.dtype).max), q))
    for power in (20, 60, 100):     # and the small ones are right themselves: all their scores are next to zero
        quiet = torch.where(mine[..., None], q * 2.0 ** -power, q)
        _check(others_are_right(quiet), quiet, cache, table, lens, new, scale=scale)


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [1.0, 2.0 ** -24, 2.0 ** 24])
def test_scores_too_large_for_fractions_pick_the_best_key(n, d, sign, size):
    """Scores from 2^10 to 2^118, where fp32 has no fraction bits left for an exponent.  The best key is 1/17 ahead of all others,
    so it takes all the weight: the result is its value row, rounded to bf16 once (and to fp16 before, in the prompt kernel)."""
    lens, new = [300, 300, 70], [n] * 3
    best = [20, 210, 45]                                # in the first, the second and the only page; the last page lowers nothing
    q, cache, table, kv_len, cu = _setup(lens, new, 14, 2, d, seed=20, poison=False)
    codes, scales = ops.kv_cache_fp8_views(cache)
    scales[:, 0] = 1 / 256
    scales[:, 1] *= size
    # a negative query is best answered by the smallest key
    codes[:, 0] = 256.0 if sign > 0 else 288.0
    for i, b in enumerate(best):
        codes[int(table[i, b // 128]), 0, :, b % 128] = 288.0 if sign > 0 else 256.0
    want, top = [], []
    for i, b in enumerate(best):
        page = int(table[i, b // 128])
        want.append((codes[page, 1, :, b % 128].double() * scales[page, 1, :, b % 128, None].double()).repeat_interleave(7, 0).expand(n, 14, d))
        top.append(scales[page, 1].double().amax(-1).repeat_interleave(7)[None, :, None].expand(n, 14, d))
    want, top = torch.cat(want), torch.cat(top)
    for power in (10, 16, 20, 22, 24, 26, 28, 32, 40, 60, 100, 111):
        got = ops.attention_paged_fp8(torch.full_like(q, sign * 2.0 ** power), cache, table, kv_len, cu, n)
        # bf16 output, fp16 weight (numerator only), fp16 value row
        tol = want.abs() * (2.0 ** -8 + 2 * 2.0 ** -11 + 2.0 ** -18) + top * 2.0 ** -30
        assert ((got.double() - want).abs() <= tol).all(), power


@pytest.mark.parametrize("n", [1, 20])
def test_pages_shared_by_sequences_and_tables_shared_by_all(n):
    q, cache, table, kv_len, cu = _setup([333], [n], 8, 2, 64, seed=16)
    lens = [333, 200, 129, 333]
    big = torch.cat([q] * 4)
    cu4 = _i32([0, n, 2 * n, 3 * n, 4 * n])
    for shared in (table.expand(4, -1), table.repeat(4, 1)):
        out = ops.attention_paged_fp8(big, cache, shared, _i32(lens), cu4, n)
        _check(out, big, cache, table.repeat(4, 1), lens, [n] * 4)
        assert torch.equal(shared, table.repeat(4, 1))


@pytest.mark.parametrize("new", [[1] * 6, [64, 3, 0, 5, 129, 40]])
def test_tables_and_lengths_that_do_not_fit_are_reported(new):
    lens = [300, 64, 10, 129, 500, 40]
    q, cache, table, kv_len, cu = _setup(lens, new, 8, 2, 64, seed=13, poison=False)
    bad_table = table.clone()
    bad_table[0, 1] = cache.shape[0]
    bad_table[4, 2] = -1
    ops.attention_paged_fp8(q, cache, bad_table, kv_len, cu, max(new))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.check_error("pages")
    bad_len = kv_len.clone()
    bad_len[1] = 128 * table.shape[1] + 1
    out = ops.attention_paged_fp8(q, cache, torch.where(table < 0, 0, table).int(), bad_len, cu, max(new))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="bad argument"):
        ops.check_error("length")
    a, b = sum(new[:1]), sum(new[:2])
    # the others are right (their sums may be cut elsewhere than with the good length, so not the same to the last bit)
    _check(out[:a], q[:a], cache, table[:1], lens[:1], new[:1])
    _check(out[b:], q[b:], cache, table[2:], lens[2:], new[2:])


def test_rows_of_no_sequence_are_left_as_they_were():
    """A padded batch of single tokens: as many rows as sequences, but some sequences have no query."""
    lens = [200, 50, 70, 0, 129]
    q, cache, table, kv_len, _ = _setup(lens, [1] * 5, 8, 2, 64, seed=17)
    for cu, rows in (([0, 1, 2, 2, 2, 2], {0: 0, 1: 1}), ([1, 2, 2, 3, 4, 5], {1: 0, 2: 2, 3: 3, 4: 4}), ([0] * 6, {})):
        out = torch.full_like(q, 5.0)
        ops.attention_paged_fp8(q, cache, table, kv_len, _i32(cu), 1, out=out)
        for r in range(5):
            if r in rows:
                i = rows[r]
                _check(out[r: r + 1], q[r: r + 1], cache, table[i: i + 1], lens[i: i + 1], [1])
            else:
                assert (out[r] == 5.0).all()
    out = torch.full_like(q, 5.0)        # the same rows, for sequences of many queries: rows 0 and 4 are nobody's
    ops.attention_paged_fp8(q, cache, table[1:3], _i32([50, 70]), _i32([1, 3, 4]), 2, out=out)
    assert (out[0] == 5.0).all() and (out[4] == 5.0).all()
    _check(out[1:4], q[1:4], cache, table[1:3], [50, 70], [2, 1])
    for cu in ([0, 1, 2, 3, 4, 6], [0, 2, 2, 3, 4, 5], [-1, 0, 1, 2, 3, 4]):      # not one row each, or not in q
        ops.attention_paged_fp8(q, cache, table, kv_len, _i32(cu), 1)
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match="bad argument"):
            ops.check_error("rows")
    for n in (1, 2):
        ops.attention_paged_fp8(q[:n], cache, table[:1], _i32([-3]), _i32([0, n]), n, out=out[:n])
        assert not out[:n].any()
        with pytest.raises(RuntimeError, match="bad argument"):
            ops.check_error("length")


@pytest.mark.parametrize("B", [479, 481, 1201])
@pytest.mark.parametrize("new", [[1], [3, 0, 1, 2]])
def test_more_sequences_than_threads(B, new):
    """The lengths are added up by the threads of a block, several sequences each in a large batch."""
    lens = [(7 * i * i + 3 * i) % 141 if i % 19 else 0 for i in range(B)]
    new = [min(new[i % len(new)], lens[i]) if len(new) > 1 else 1 for i in range(B)]
    q, cache, table, kv_len, cu = _setup(lens, new, 4, 2, 64, seed=B)
    _check(ops.attention_paged_fp8(q, cache, table, kv_len, cu, max(new)), q, cache, table, lens, new)


@pytest.mark.parametrize("Hq,Hkv,d", [(131, 1, 64), (256, 2, 128), (48, 2, 128)])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 70, 1]])
def test_very_many_heads_to_a_key_head(Hq, Hkv, d, new):
    lens = [260, 70, 1]
    q, cache, table, kv_len, cu = _setup(lens, new, Hq, Hkv, d, seed=Hq)
    _check(ops.attention_paged_fp8(q, cache, table, kv_len, cu, max(new)), q, cache, table, lens, new)


def test_pages_behind_4_gib_of_cache():
    """Offsets of the cache that pass 32 bits: pages at the end of 4.5 GB (zeroed, so nothing but these pages holds a row)."""
    Hkv, d, lens = 8, 128, [300, 129]
    pages = (4608 << 20) // (2 * Hkv * 128 * (d + 4))
    table = torch.arange(pages - 6, pages, device=DEV, dtype=torch.int32).view(2, 3)
    cache = ops.kv_cache_fp8(pages, Hkv, d, DEV)
    cs = _cs(429, d)
    pos = torch.cat([torch.arange(n, device=DEV) for n in lens])
    seq = torch.repeat_interleave(torch.arange(2, device=DEV), torch.tensor(lens, device=DEV))
    slot = (table[seq, pos // 128].long() * 128 + pos % 128).int()
    torch.manual_seed(3)
    qkv = torch.randn(429, 32 * d, device=DEV).bfloat16()
    q = ops.rope_kv_write_fp8_(qkv, 16, Hkv, d, cs, cache, slot)
    assert not cache[: pages - 6].view(torch.int64).any()
    _check(ops.attention_paged_fp8(q, cache, table, _i32(lens), _i32([0, 300, 429]), 300), q, cache, table, lens, lens)
    last = q[[299, 428]]
    _check(ops.attention_paged_fp8(last, cache, table, _i32(lens), _i32([0, 1, 2]), 1), last, cache, table, lens, [1, 1])


def test_results_do_not_depend_on_the_run_or_the_batch_order():
    lens = [5, 2000, 700, 333, 128]
    q, cache, table, kv_len, cu = _setup(lens, [1] * 5, 28, 4, 128, seed=21)
    a = ops.attention_paged_fp8(q, cache, table, kv_len, cu, 1)
    for _ in range(5):
        assert torch.equal(a, ops.attention_paged_fp8(q, cache, table, kv_len, cu, 1))


@pytest.mark.parametrize("Hq,Hkv,d", [(16, 16, 64), (16, 8, 128), (32, 2, 128)])
def test_decode_runs_of_one_cta_over_more_than_32_pages(Hq, Hkv, d):
    """The producers hold 32 table entries at a time: long visits reload them.  (24 x 8 or more items of about 41 pages, and one
    batch whose items fill a CTA's whole run.)"""
    lens = [4500 + 67 * i % 1500 for i in range(24 if Hkv > 2 else 90)]
    q, cache, table, kv_len, cu = _setup(lens, [1] * len(lens), Hq, Hkv, d, seed=24)
    _check(ops.attention_paged_fp8(q, cache, table, kv_len, cu, 1), q, cache, table, lens, [1] * len(lens))


@pytest.mark.parametrize("Hq,d", [(7, 128), (3, 64), (16, 128), (16, 64)])
def test_decode_item_shared_by_more_than_128_ctas(Hq, d):
    """One key head and 40000 keys: every CTA of the GPU leaves a part of the same item, which the join looks for in blocks of 128."""
    assert torch.cuda.get_device_properties(0).multi_processor_count > 129
    q, cache, table, kv_len, cu = _setup([40000], [1], Hq, 1, d, seed=25)
    _check(ops.attention_paged_fp8(q, cache, table, kv_len, cu, 1), q, cache, table, [40000], [1])


@pytest.mark.parametrize("new", [[1] * 5, [5, 300, 64, 33, 128]])
def test_same_call_same_bits_and_any_batch_order_within_tolerance(new):
    """Sums do not depend on timing.  Where a sequence is cut depends on the batch, so another order may change last bits."""
    lens = [5, 2000, 700, 333, 128]
    q, cache, table, kv_len, cu = _setup(lens, new, 28, 4, 128, seed=26)
    a = ops.attention_paged_fp8(q, cache, table, kv_len, cu, max(new))
    for _ in range(5):
        assert torch.equal(a, ops.attention_paged_fp8(q, cache, table, kv_len, cu, max(new)))
    starts = [sum(new[:i]) for i in range(6)]
    for order in ([4, 3, 2, 1, 0], [1, 4, 0, 2, 3]):
        rows = torch.cat([torch.arange(starts[i], starts[i + 1], device=DEV) for i in order])
        lens2, new2 = [lens[i] for i in order], [new[i] for i in order]
        table2, cu2 = table[order].contiguous(), _i32([sum(new2[:i]) for i in range(6)])
        got = ops.attention_paged_fp8(q[rows], cache, table2, _i32(lens2), cu2, max(new))
        _check(got, q[rows], cache, table2, lens2, new2)
        assert torch.equal(got, ops.attention_paged_fp8(q[rows], cache, table2, _i32(lens2), cu2, max(new)))


@pytest.mark.parametrize("Hq,Hkv,d", [(28, 4, 128), (131, 1, 64)])
@pytest.mark.parametrize("new", [[1, 1, 1], [300, 64, 37]])
def test_the_output_may_be_the_queries_themselves(Hq, Hkv, d, new):
    """Every row and head is read by those CTAs alone that work on its item, and written when they have read it."""
    lens = [3000, 64, 700]
    q, cache, table, kv_len, cu = _setup(lens, new, Hq, Hkv, d, seed=27)
    want = ops.attention_paged_fp8(q, cache, table, kv_len, cu, max(new))
    _check(want, q, cache, table, lens, new)
    x = q.clone()
    assert ops.attention_paged_fp8(x, cache, table, kv_len, cu, max(new), out=x) is x
    assert torch.equal(x, want)


@pytest.mark.parametrize("Hq,Hkv,d", [(8, 1, 64), (7, 1, 128)])
@pytest.mark.parametrize("n", [1, 20])
def test_four_million_keys(Hq, Hkv, d, n):
    """A table that names the same 16 pages 2048 times over: the softmax is that over the 16 pages alone."""
    q, cache, table, kv_len, cu = _setup([2048], [n], Hq, Hkv, d, seed=28)
    table = table[:, :16]
    out = ops.attention_paged_fp8(q, cache, table.repeat(1, 2048), _i32([2048 * 2048]), cu, n, causal=False)
    _check(out, q, cache, table, [2048], [n], causal=False)
    # causal: the first query misses 19 keys, one of 2048 occurrences each: 2^-11 of their weights, like a weight's rounding
    out = ops.attention_paged_fp8(q, cache, table.repeat(1, 2048), _i32([2048 * 2048]), cu, n)
    _check(out, q, cache, table, [2048], [n], causal=False)


def test_launches_are_counted_as_they_are_made():
    """A call that one CTA does alone leaves no partial sums, and the kernel that joins them is not launched."""
    for lens, new, Hq, launches in (([2], [2], 64, 1), ([300], [300], 8, 2), ([300, 5], [1, 1], 8, 2)):
        q, cache, table, kv_len, cu = _setup(lens, new, Hq, 1, 128, seed=23)
        before = ops.kernel_launches()
        out = ops.attention_paged_fp8(q, cache, table[:, : -(-max(lens) // 128)], kv_len, cu, max(new))
        assert ops.kernel_launches() - before == launches
        _check(out, q, cache, table, lens, new)


def test_empty_calls():
    q, cache, table, kv_len, cu = _setup([5], [1], 4, 2, 64)
    assert ops.attention_paged_fp8(q[:0], cache, table[:0], kv_len[:0], cu[:1], 0).shape == (0, 4, 64)
    zero = torch.zeros_like(kv_len)
    assert not ops.attention_paged_fp8(q, cache, table, zero, cu, 1).any()
    assert not ops.attention_paged_fp8(q, cache, table[:, :0], zero, cu, 1).any()
    q3 = q.repeat(3, 1, 1)
    assert not ops.attention_paged_fp8(q3, cache, table, zero, _i32([0, 3]), 3).any()
    assert not ops.attention_paged_fp8(q3, cache, table[:, :0], zero, _i32([0, 3]), 3).any()


def test_other_head_widths_are_refused_on_the_gpu():
    cache = ops.kv_cache_fp8(1, 1, 32, DEV)
    with pytest.raises(ValueError, match="head widths"):
        ops.attention_paged_fp8(torch.zeros(1, 1, 32, device=DEV).bfloat16(), cache, _i32([[0]]), _i32([1]), _i32([0, 1]), 1)
    cache = ops.kv_cache_fp8(1, 1, 64, DEV)
    with pytest.raises(ValueError):
        ops.attention_paged_fp8(torch.zeros(1, 1, 64, device=DEV), cache, _i32([[0]]), _i32([1]), _i32([0, 1]), 1)
    with pytest.raises(ValueError):
        ops.attention_paged_fp8(torch.zeros(1, 1, 64).bfloat16(), cache, _i32([[0]]), _i32([1]), _i32([0, 1]), 1)


# ---------------------------------------------------------------------------------------------------------------------
# together: append then attend, on other streams and from graphs
# ---------------------------------------------------------------------------------------------------------------------
def _step(qkv, cs, cache, slot, table, kv_len, cu, n, Hq, Hkv, d):
    q = ops.rope_kv_write_fp8_(qkv, Hq, Hkv, d, cs, cache, slot)
    return ops.attention_paged_fp8(q, cache, table, kv_len, cu, n)


def test_prompt_then_decode_steps_match_one_pass_over_all_tokens():
    torch.manual_seed(2)
    d, Hq, Hkv, T, tail = 128, 8, 2, 333, 6
    qkv = torch.randn(T, (Hq + 2 * Hkv) * d, device=DEV).bfloat16()
    cs = _cs(T, d)
    table = _i32([[2, 0, 3]])
    slot = (table[0].long()[torch.arange(T, device=DEV) // 128] * 128 + torch.arange(T, device=DEV) % 128).int()
    one = ops.kv_cache_fp8(4, Hkv, d, DEV)
    want = _step(qkv, cs, one, slot, table, _i32([T]), _i32([0, T]), T, Hq, Hkv, d)
    cache = ops.kv_cache_fp8(4, Hkv, d, DEV)
    m = T - tail
    parts = [_step(qkv[:100], cs[:100], cache, slot[:100], table, _i32([100]), _i32([0, 100]), 100, Hq, Hkv, d),
             _step(qkv[100:m], cs[100:m], cache, slot[100:m], table, _i32([m]), _i32([0, m - 100]), m - 100, Hq, Hkv, d)]
    for t in range(m, T):
        parts.append(_step(qkv[t: t + 1], cs[t: t + 1], cache, slot[t: t + 1], table, _i32([t + 1]), _i32([0, 1]), 1, Hq, Hkv, d))
    assert torch.equal(cache, one)
    got = torch.cat(parts)
    codes, scales = ops.kv_cache_fp8_views(one)
    v = (codes[table[0].long(), 1].double() * scales[table[0].long(), 1].double()[..., None]).abs().amax()
    # both are within their tolerance of the definition
    assert ((got.double() - want.double()).abs() <= want.double().abs() * 2 ** -7 + v * 2 ** -9).all()
    assert torch.nn.functional.cosine_similarity(got.float().flatten(), want.float().flatten(), dim=0) > 0.9999


@pytest.mark.parametrize("n", [1, 30])
def test_graphs_replayed_at_once_on_two_streams_and_with_new_lengths(n):
    Hq, Hkv, d, B = 28, 4, 128, 3
    sets = []
    for seed in (31, 32):
        q, cache, table, kv_len, cu = _setup([2000, 900, 1500], [n] * B, Hq, Hkv, d, seed=seed, poison=False)
        table = table.clamp_min(0)
        want = ops.attention_paged_fp8(q, cache, table, kv_len, cu, n).clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.attention_paged_fp8(q, cache, table, kv_len, cu, n)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.attention_paged_fp8(q, cache, table, kv_len, cu, n)
        sets.append((g, out, want, side, q, cache, table, kv_len, cu))
    for _ in range(20):
        for g, _, _, side, *_ in sets:
            with torch.cuda.stream(side):
                g.replay()
    torch.cuda.synchronize()
    for _, out, want, *_ in sets:
        assert torch.equal(out, want)
    # the graph reads the lengths on the device: shorter sequences need no new capture
    g, out, _, _, q, cache, table, kv_len, cu = sets[0]
    lens = [40, 900, 777]
    kv_len.copy_(_i32(lens))
    g.replay()
    torch.cuda.synchronize()
    _check(out, q, cache, table, lens, [n] * B)


FIRST_CALLS = """
import torch
from cornserve import ops
d, T, Hq, Hkv = {d}, 40, {Hq}, 2
dev = torch.device("cuda")
i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)
torch.manual_seed(0)
qkv = torch.randn(T, (Hq + 2 * Hkv) * d, device=dev).bfloat16()
ang = torch.arange(T, device=dev)[:, None] * 1e4 ** (-torch.arange(d // 2, device=dev) * 2 / d)
cs = torch.stack([ang.cos(), ang.sin()], dim=1).float().contiguous()
cache, table, slot = ops.kv_cache_fp8(1, Hkv, d, dev), i32([[0]]), torch.arange(T, device=dev, dtype=torch.int32)
lens, cu, one = i32([T]), i32([0, T]), i32([0, 1])

def step():
    q = ops.rope_kv_write_fp8_(qkv, Hq, Hkv, d, cs, cache, slot)
    return ops.attention_paged_fp8(q, cache, table, lens, cu, T), ops.attention_paged_fp8(q[-1:], cache, table, lens, one, 1)

ops.rms_norm(torch.randn(4, 64, device=dev).bfloat16(), torch.ones(64, device=dev).bfloat16())    # the library is in use
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    out = step()
g.replay()
torch.cuda.synchronize()
got = [o.clone() for o in out]
assert all(torch.equal(a, b) for a, b in zip(got, step())) and got[0].any() and got[1].any()
ops.check_error("captured")
print("CAPTURED_OK")
"""


@pytest.mark.parametrize("d,Hq", [(128, 14), (64, 32)])
def test_first_calls_of_a_process_may_be_captured(d, Hq):
    """Append, prompt and decode attention in one graph, none of which ran in this process before."""
    import os
    import subprocess
    import sys

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", FIRST_CALLS.format(d=d, Hq=Hq)], cwd=root, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "CAPTURED_OK" in r.stdout, r.stdout + r.stderr[-3000:]


def test_pages_pulled_into_another_cache_give_the_same_attention():
    lens = [300, 129]
    q, cache, table, kv_len, cu = _setup(lens, [1, 1], 28, 4, 128, seed=41)
    src = torch.stack([cache, cache.flip(0)])                       # two layers
    dst = torch.zeros(2, 9, *cache.shape[1:], device=DEV, dtype=torch.uint8)
    old = [int(p) for row, n in zip(table.tolist(), lens) for p in row[: -(-n // 128)]]
    new = [8, 1, 4, 6, 2]
    ops.kv_copy_pages(dst, src, _i32(old), _i32(new))
    moved = _i32([new[:3], new[3:] + [-7]])
    a = ops.attention_paged_fp8(q, cache, table, kv_len, cu, 1)
    assert torch.equal(a, ops.attention_paged_fp8(q, dst[0], moved, kv_len, cu, 1))
    assert torch.equal(dst[1, new], src[1, old]) and not dst[:, 0].any()


def test_engine_with_an_8_bit_cache_decodes_from_graphs_like_it_does_eagerly():
    import numpy as np

    from cornserve.models.qwen_llm import LLMConfig, QwenLLM
    from cornserve.task_executors.llm.engine import EngineConfig, LLMEngine, SamplingParams, Sequence

    torch.manual_seed(0)
    cfg = LLMConfig(hidden_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2, head_dim=64, intermediate_size=1024,
                    vocab_size=1024, mrope_section=None, qk_norm=True, attention_bias=False, eos_token_id=1023)
    model = QwenLLM(cfg, device=DEV).eval()
    prompts = [np.arange(3, 3 + n, dtype=np.int32) for n in (5, 140, 260)]
    got = []
    for graph in (True, False):
        eng = LLMEngine(model, EngineConfig(num_pages=32, decode_burst=4, max_model_len=512, kv_cache_dtype="fp8", use_cuda_graph=graph))
        assert eng.kv_backing.dtype == torch.uint8
        got.append(eng.generate([Sequence(f"s{i}", p, SamplingParams(max_tokens=9, ignore_eos=True)) for i, p in enumerate(prompts)]))
    assert all(len(t) == 9 for t in got[0].values())
    # the graph pads the batch to its bucket, which changes no row of the attention but may change the projections' kernel
    same = sum(a == b for k in got[0] for a, b in zip(got[0][k], got[1][k]))
    assert same >= 3 and got[0]["s0"][0] == got[1]["s0"][0]


def _tiny_engine(model, graph, **kw):
    from cornserve.task_executors.llm.engine import EngineConfig, LLMEngine

    return LLMEngine(model, EngineConfig(num_pages=32, decode_burst=4, max_model_len=512, kv_cache_dtype="fp8", use_cuda_graph=graph, **kw))


@pytest.mark.parametrize("count", [3, 4])
def test_tokens_decoded_from_graphs_over_an_8_bit_cache(count):
    """Four sequences fill their bucket: graph and eager run the same kernels on the same rows, so every token is the same.  Three
    leave a padding row, which reads and writes the scratch page.  Each decoded token is also held to one pass over all tokens
    before it: the roundings that differ (about 20 to 2^-9 in a row of the hidden states, which add up like their squares)
    move a logit by 2^-7 of the logits' deviation, so half a deviation is far beyond them; a token picked by anything but
    these logits lies there once in some hundred times."""
    import numpy as np

    from cornserve.models.qwen_llm import BatchMeta, LLMConfig, QwenLLM
    from cornserve.task_executors.llm.engine import SamplingParams, Sequence

    torch.manual_seed(0)
    cfg = LLMConfig(hidden_size=512, num_hidden_layers=2, num_attention_heads=8, num_key_value_heads=2, head_dim=64, intermediate_size=1024,
                    vocab_size=1024, mrope_section=None, qk_norm=True, attention_bias=False, eos_token_id=1023)
    model = QwenLLM(cfg, device=DEV).eval()
    prompts = [np.arange(3 + 11 * i, 3 + 11 * i + n, dtype=np.int32) for i, n in enumerate((5, 140, 260, 127)[:count])]
    new = 21                             # the fourth crosses a page while it decodes
    got = []
    for graph in (True, False):
        eng = _tiny_engine(model, graph)
        got.append(eng.generate([Sequence(f"s{i}", p, SamplingParams(max_tokens=new, ignore_eos=True)) for i, p in enumerate(prompts)]))
        assert graph == any(st.graph is not None for st in eng._decode_states.values())
    if count == 4:
        assert got[0] == got[1]
    for tokens in got:
        for i, p in enumerate(prompts):
            ids = torch.tensor([*p.tolist(), *tokens[f"s{i}"]], dtype=torch.int32, device=DEV)
            T = ids.numel() - 1
            meta = BatchMeta(ids[:-1], torch.arange(T, dtype=torch.int32, device=DEV).expand(3, T).contiguous(),
                             (128 + torch.arange(T, device=DEV)).int(), _i32([0, T]), _i32([T]),
                             torch.arange(1, 2 + T // 128, dtype=torch.int32, device=DEV)[None], _i32([T - 1]), T)
            with torch.inference_mode():
                logits = model.compute_logits(model.forward_hidden(meta, model.alloc_kv_cache(2 + T // 128, "fp8")))[len(p):]
            picked = logits.gather(1, ids[len(p) + 1:, None].long())[:, 0]
            assert picked.numel() == new - 1
            assert (picked >= logits.amax(1) - 0.5 * logits.std(1)).all()
