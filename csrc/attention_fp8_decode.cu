// Decode attention over the 8-bit paged key-value cache (layout in kv_fp8.cuh): one new token per sequence, grouped heads.
//
//   o = sum_j w_j vc_j / sum_j 2^(s_j - M),   w_j = 2^(s_j + log2 vs_j - M),   s_j = scale * log2(e) * ks_j * (q . kc_j)
//
// kc, vc are the e4m3 codes and ks, vs the scales of key j.  Codes are exact in fp16, so the two products run on fp16
// fragments: the query is scaled by a power of two per head (exact for every element within 2^-31 of the largest), and M
// follows the maximum of s_j + log2 vs_j, the weight that the second product sees, so that a weight is never too large
// for fp16 whatever the value scales are.  The normaliser needs no vs: it takes its own exponential, in fp32.  (Of scores beyond
// 2^20 the largest is taken off first, see LARGE_EXPONENT.)
//
// The kernel is bound by the cache's bytes, and everything is arranged around reading them once, without a pause:
//
//   * Work is counted in units of 64 keys (128 for the narrow heads) of one (sequence, key head); the list of all units
//     of the batch is cut into runs of equal cost, one per CTA, on the device from kv_len.  So any mix of lengths loads
//     every SM alike (a captured graph adapts to the lengths of each replay), and a single long sequence is spread over the
//     whole GPU.  A CTA has at most two items that it does not own alone, the first and the last of its run: these leave partial
//     sums in a workspace and a second small kernel joins them in the order of the CTAs (no atomics, the result does not
//     depend on timing).
//   * A CTA is three (or two) teams of four consumer warps and one producer warp.  A team has its own ring of stages, kept
//     full by TMA: one copy brings the K and V codes of a unit (through a tensor map with a swizzle), one its scales.
//     Long visits to an item are shared by the teams, unit by unit; short ones are dealt whole to one team each, so that
//     the end of one sequence overlaps the reading of others.
//   * Consumer warp w of a team takes a quarter of the unit's keys, entirely in registers: S^T = K Q^T and O^T += V^T P
//     with mma.m16n8k16, keys (channels) on the 16 side and up to 8 query heads per n tile on the other.  mma.sync and
//     not tcgen05 on purpose: e4m3 becomes fp16 on the way from shared memory to a register fragment, while a tcgen05
//     operand would have to be written back to shared memory twice as wide; tensor time is not what is scarce at 8 to 16
//     heads per byte of K.  The warps share nothing until a visit ends; then their sums meet in shared memory.
//
// Measured inside a graph (28 query heads, 4 key heads, d = 128): 256 sequences of 3300 to 3700 tokens, 954 MB, 151 us =
// 6.3 TB/s, 0.97 of what a copy reaches; issue slots are half full.  64 sequences of 2000, 136 MB, 33 us = 4.1 TB/s.  One of
// 32768, 35 MB over all SMs, 15.5 us; one of 500, 7.7 us.  The short ones are bound by a chain of latencies: lengths, table
// entry, unit, the sums of the warps, and the second kernel (each 0.5 to 1 us).  With 64 query heads (16 to a key head, two n
// tiles) the large batch takes 233 us = 4.1 TB/s, at d = 64 130 us = 3.8 TB/s: twice the exponentials, products and
// accumulators for the same bytes, with spills of about 100 bytes a thread.
#include <math.h>

#include "kv_fp8.cuh"

int cs_encode_tmap_nd(CUtensorMap* out, int elem_bytes, int rank, const void* base, const uint64_t* dims, const uint64_t* strides,
                      const uint32_t* box, int swizzle_bytes);

namespace {

constexpr int MAX_CTAS = 512;
// What an item costs beside its units, in units: queries to load, sums to join.  33 sequences of 1 to 5000 tokens take 30.1 us
// with 1, 25.5 with 3, 25.2 with 5; one of 32768 17.2, 16.6, 15.9.
constexpr int ITEM_COST = 5;
// The cost of a CTA's run is this at least: one sequence of 500 tokens takes 8.1 us with 2, 8.5 with 3 or 4, 9.1 with 6.
constexpr int MIN_RUN = 2;
// Visits of at least this many units are shared by the teams of a CTA, unit by unit, and joined by all of them; shorter ones go
// to one team.  256 sequences of 100 tokens (2 units) take 26.2 us shared, 18.2 dealt; 33 of 1 to 5000 tokens 25.5 us with the
// border at 3, 26.1 at 8.
constexpr int SHARED_VISIT = 3;
constexpr float M_NONE = -3.0e38f;           // running maximum before the first key (finite: differences stay defined)
// Where the maximum passes this, scores and value scales are no longer added up: from 2^24 on the sum is rounded to integers,
// and a weight that is taken relative to it is too large for fp16, or far too small.
constexpr float LARGE_EXPONENT = 1048576.f;

// One instantiation.  TEAMS: as many as registers allow (128 a thread with three teams, 168 with two).
template <int D, int NT>
struct DecShape {
  static constexpr int HEADS = 8 * NT;
  static constexpr int TEAMS = (D == 128 && NT == 2) ? 2 : 3;
  static constexpr int KT = D == 128 ? 1 : 2;                // 16-key tiles per consumer warp and unit
  static constexpr int UNIT = 64 * KT;                       // keys
  static constexpr int WARPS = 4 * TEAMS;                    // consumers
  static constexpr int THREADS = (WARPS + TEAMS) * 32;
  static constexpr int TILE = UNIT * D;                      // bytes of codes of K (or V) per stage
  static constexpr int STAGE = 2 * TILE + 2 * UNIT * 4;
  static constexpr int JOIN_LD = D + 4;                      // floats between two heads of a warp's partial sum
  static constexpr int JOIN = WARPS * HEADS * JOIN_LD * 4;
  static constexpr int Q = HEADS * D * 2;                    // queries of one visit
  static constexpr int QSLOTS = 2;                           // per team
  static constexpr int FIT = (227 * 1024 - 1024 - 4096 - JOIN - TEAMS * QSLOTS * Q) / STAGE;
  static constexpr int RING = FIT / TEAMS < 8 ? FIT / TEAMS : 8;   // stages per team
  static constexpr int SMEM = 1024 + TEAMS * RING * STAGE + TEAMS * QSLOTS * Q + JOIN;
  static_assert(RING >= 3, "a stage in use and two on their way");
};

struct DecParams {
  const __nv_bfloat16* q; long long q_tok;             // heads follow each other; every token on a 16-byte boundary
  __nv_bfloat16* o; long long o_tok, o_head; int o_vec; // o_vec: 8-byte stores are aligned
  int num_pages;
  const int* block_table; long long bt_stride; int bt_width;
  const int* kv_len; const int* cu_q;
  int B, Hq, Hkv, G, head_blocks;                      // G query heads per key head, in blocks of 8 NT
  float scale_log2;
  float* ws_o;        // [ctas, 2, HEADS, D] partial sums: slot 0 = the CTA's first item, slot 1 = its last
  float* ws_ml;       // [ctas, 2, HEADS, 2] their maximum and normaliser
  int* ws_item;       // [ctas, 2] the items they belong to, -1 = none
  int* err;
};

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ float lds32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ void bulk_load(uint32_t smem_dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_dst), "l"(src),
               "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tma_load_4d(uint32_t smem_dst, const CUtensorMap* m, int x, int y, int z, int w, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_5d(uint32_t smem_dst, const CUtensorMap* m, int x, int y, int z, int w, int v, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(smem_dst),
      "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(v), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A sequence: the row of its query (-1: it has none) and the keys of it that can be read (none without a query; a length
// beyond the table is cut).  What does not fit is reported.
struct Seq { int row, len; };
__device__ __forceinline__ Seq get_seq(const DecParams& p, int b) {
  const int n = p.kv_len[b], beg = p.cu_q[b], end = p.cu_q[b + 1], cap = p.bt_width * KV8_PAGE;
  Seq s;
  s.row = end > beg && beg >= 0 && beg < p.B ? beg : -1;
  s.len = s.row < 0 || n < 0 ? 0 : min(n, cap);
  return s;
}
__device__ __forceinline__ bool fits(const DecParams& p, int b) {
  const int n = p.kv_len[b], beg = p.cu_q[b], end = p.cu_q[b + 1];
  return n >= 0 && n <= p.bt_width * KV8_PAGE && beg >= 0 && end <= p.B && (end == beg || end == beg + 1);
}

template <int N> struct Count { static constexpr int value = N; };

// Four channels of one head: sums divided by the normaliser.  (Only sequences with keys come here; the sum is 0 when all their
// scores are -inf, and 0 / 0 is the result.)
__device__ __forceinline__ void store_head(const DecParams& p, int row, int head, int ch4, const float4& acc, float sum) {
  const float inv = 1.0f / sum;
  __nv_bfloat16* dst = p.o + row * p.o_tok + head * p.o_head + ch4 * 4;
  const uint2 v = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (p.o_vec) {
    *reinterpret_cast<uint2*>(dst) = v;
  } else {
    unsigned short* d16 = reinterpret_cast<unsigned short*>(dst);
    d16[0] = v.x & 0xffffu; d16[1] = v.x >> 16; d16[2] = v.y & 0xffffu; d16[3] = v.y >> 16;
  }
}

// A place in the list of units: unit u of head block `head` (of Hkv * head_blocks) of a sequence.
struct Place { int seq, head, u; };

// The place at distance r (cost) into the items of a sequence.  Cuts that would leave less than two units of an item on one
// side move to its edge.
__device__ __forceinline__ Place place_at(int seq, int units, int heads, int r) {
  Place at{seq, r / (units + ITEM_COST), 0};
  const int u = r - at.head * (units + ITEM_COST) - ITEM_COST;
  if (u < 2) return at;
  if (units - u >= 2) { at.u = u; return at; }
  if (++at.head == heads) { at.head = 0; ++at.seq; }
  return at;
}

// One visit of a CTA to an item: units [u, u + n) of `units` of sequence `seq`, head block `head`.  Every role of the CTA
// walks the same list of visits.
template <int UNIT>
struct Walk {
  int seq, head, u;
  Place end;
  int known, row, len, units, n;   // row, len and units are those of sequence `known`
  uint32_t dealt;   // short visits and units of shared visits so far: deals the next ones to the teams in turn
  __device__ __forceinline__ bool settle(const DecParams& p) {   // on to an item with units for this CTA
    const int heads = p.Hkv * p.head_blocks;
    while (seq < p.B) {
      if (known != seq) {
        const Seq s = get_seq(p, seq);
        known = seq;
        row = s.row;
        len = s.len;
        units = (len + UNIT - 1) / UNIT;
      }
      const bool last = seq == end.seq && head == end.head;
      if (seq > end.seq || (last && u >= end.u)) return false;
      n = (last ? min(end.u, units) : units) - u;
      if (n > 0) return true;
      u = 0;
      if (units == 0 || ++head == heads) { head = 0; ++seq; }
    }
    return false;
  }
  __device__ __forceinline__ bool shared() const { return n >= SHARED_VISIT; }
  __device__ __forceinline__ bool next(const DecParams& p) {
    dealt += shared() ? n : 1;
    if (seq == end.seq && head == end.head) return false;
    u = 0;
    if (++head == p.Hkv * p.head_blocks) { head = 0; ++seq; return settle(p); }
    n = (seq == end.seq && head == end.head) ? min(end.u, units) : units;
    return n > 0;
  }
  // the units of this visit that belong to `team`: first, first + step, ... below u + n
  template <int TEAMS>
  __device__ __forceinline__ bool mine(int team, int& first, int& step) const {
    const int turn = static_cast<int>((team + TEAMS - dealt % TEAMS) % TEAMS);
    step = shared() ? TEAMS : 1;
    first = u + (shared() ? turn : 0);
    return shared() || turn == 0;
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(DecShape<D, NT>::THREADS, 1)
attention_decode_fp8_kernel(const __grid_constant__ CUtensorMap tm_codes, const __grid_constant__ CUtensorMap tm_scales, const DecParams p) {
  using Shape = DecShape<D, NT>;
  constexpr int HEADS = Shape::HEADS, TEAMS = Shape::TEAMS, KT = Shape::KT, UNIT = Shape::UNIT, WARPS = Shape::WARPS;
  constexpr int THREADS = Shape::THREADS, ALL_WARPS = THREADS / 32, RING = Shape::RING, QSLOTS = Shape::QSLOTS;
  constexpr int TILE = Shape::TILE, JOIN_LD = Shape::JOIN_LD;
  constexpr int KSTEPS = D / 16, MT = D / 16, VPER = D / 8;   // VPER: channels of a value row per thread

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_codes = smem;                                                   // [team][stage] K tile, V tile
  uint8_t* s_scale = s_codes + TEAMS * RING * 2 * TILE;                      // [team][stage] key scales, value scales
  uint8_t* s_q = s_scale + TEAMS * RING * 2 * UNIT * 4;                      // [team][slot][head][D] bf16
  float* s_join = reinterpret_cast<float*>(s_q + TEAMS * QSLOTS * Shape::Q); // [warp][head][JOIN_LD]
  __shared__ uint64_t full[TEAMS][RING], empty[TEAMS][RING], q_full[TEAMS][QSLOTS], q_empty[TEAMS][QSLOTS];
  __shared__ float s_m[WARPS][HEADS], s_l[WARPS][HEADS];
  __shared__ int abort_flag, s_warp_sum[ALL_WARPS];
  __shared__ Place s_cut[2];       // where the run begins and ends
  __shared__ Seq s_first;          // the sequence it begins in (or ahead of)
  __shared__ int s_first_seq;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    s_cut[0] = s_cut[1] = Place{p.B, 0, 0};
    s_first_seq = -1;
    for (int w = 0; w < TEAMS; ++w) {
      for (int s = 0; s < RING; ++s) { mbar_init(&full[w][s], 1); mbar_init(&empty[w][s], 4); }
      for (int s = 0; s < QSLOTS; ++s) { mbar_init(&q_full[w][s], 1); mbar_init(&q_empty[w][s], 4); }
    }
    mbar_fence_init();
    tma_prefetch_desc(&tm_codes);
    tma_prefetch_desc(&tm_scales);
  }
  // the lengths, the queries and the cache rows of this step come from the kernels ahead in the stream
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x == 0) p.ws_item[blockIdx.x * 2] = p.ws_item[blockIdx.x * 2 + 1] = -1;

  // ------------------------------- this CTA's run of units -------------------------------
  // Thread i adds up the cost of `per` consecutive sequences (one, unless the batch is huge); a scan over the threads gives
  // the total and who owns the two cuts.  The host has checked that 32 bits hold every sum.
  const int heads = p.Hkv * p.head_blocks, per = (p.B + THREADS - 1) / THREADS;
  auto seq_of = [&](int b) { return b < p.B ? get_seq(p, b) : Seq{-1, 0}; };
  auto units_of = [&](const Seq& q) { return (q.len + UNIT - 1) / UNIT; };
  auto cost = [&](int units) { return units > 0 ? (units + ITEM_COST) * heads : 0; };
  const int first = static_cast<int>(threadIdx.x) * per;
  const Seq seq0 = seq_of(first);
  int mine = cost(units_of(seq0));
  for (int i = 1; i < per; ++i) mine += cost(units_of(seq_of(first + i)));
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) s_warp_sum[warp] = incl;
  __syncthreads();
  const int of_lane = lane < ALL_WARPS ? s_warp_sum[lane] : 0;
  const int total = __reduce_add_sync(0xffffffffu, of_lane);
  incl += __reduce_add_sync(0xffffffffu, lane < warp ? of_lane : 0);
  // (at least MIN_RUN each: then the CTAs that share an item are consecutive)
  const int active = max(1, min(total / MIN_RUN, static_cast<int>(gridDim.x))), c = blockIdx.x;
  const int quota = total / active, extra = total - quota * active;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const int r = c + e >= active ? total : quota * (c + e) + min(c + e, extra);
    int at0 = incl - mine;
    if (r >= at0 && r < incl) {
      int i = 0;
      Seq q = seq0;
      while (i + 1 < per && r >= at0 + cost(units_of(q))) {
        at0 += cost(units_of(q));
        q = seq_of(first + ++i);
      }
      s_cut[e] = place_at(first + i, units_of(q), heads, r - at0);
      if (e == 0) { s_first = q; s_first_seq = first + i; }
    }
  }
  __syncthreads();
  volatile int* abortp = &abort_flag;
  Walk<UNIT> wk{};
  wk.seq = s_cut[0].seq;
  wk.head = s_cut[0].head;
  wk.u = s_cut[0].u;
  wk.end = s_cut[1];
  wk.known = s_first_seq;
  wk.row = s_first.row;
  wk.len = s_first.len;
  wk.units = units_of(s_first);
  const bool any = wk.settle(p);

  if (warp >= WARPS) {
    // ------------------------------- producer of one team -------------------------------
    const int team = warp - WARPS;
    uint32_t n = 0, nv = 0;   // running counts: units, visits
    bool ok = true;
    if (any) do {
      int first, step;
      if (!wk.template mine<TEAMS>(team, first, step)) continue;
      const int hk = wk.head / p.head_blocks, hb = wk.head - hk * p.head_blocks;
      const int* table = p.block_table + wk.seq * p.bt_stride;
      const int blocks = (wk.len + KV8_PAGE - 1) / KV8_PAGE;
      int page_base = first / (KV8_PAGE / UNIT);    // the 32 table entries held by the lanes start at page_base
      int page_lane = page_base + lane < blocks ? table[page_base + lane] : 0;
      if (lane == 0) {
        const uint32_t slot = nv % QSLOTS;
        ok = ok && mbar_wait(&q_empty[team][slot], ((nv / QSLOTS) & 1) ^ 1, abortp, p.err, CS_ERR_TIMEOUT_SLOT);
        if (ok) {
          const uint32_t bytes = min(HEADS, p.G - hb * HEADS) * D * 2;
          mbar_arrive_expect_tx(&q_full[team][slot], bytes);
          bulk_load(smem_u32(s_q + (team * QSLOTS + slot) * Shape::Q), p.q + wk.row * p.q_tok + (hk * p.G + hb * HEADS) * D, bytes,
                    &q_full[team][slot]);
        }
      }
      ++nv;
      for (int u = first; u < wk.u + wk.n; u += step, ++n) {
        const int blk = u / (KV8_PAGE / UNIT), part = u % (KV8_PAGE / UNIT);
        if (blk >= page_base + 32) {
          page_base = blk;
          page_lane = blk + lane < blocks ? table[blk + lane] : 0;
        }
        int page = __shfl_sync(0xffffffffu, page_lane, blk - page_base);
        if (lane == 0 && ok) {
          if (page < 0 || page >= p.num_pages) { cs_set_error(p.err, CS_ERR_BAD_ARG); page = 0; }
          const uint32_t s = n % RING;
          ok = mbar_wait(&empty[team][s], ((n / RING) & 1) ^ 1, abortp, p.err, CS_ERR_TIMEOUT_SLOT);
          if (ok) {
            const int stage = team * RING + s;
            mbar_arrive_expect_tx(&full[team][s], Shape::STAGE);
            tma_load_5d(smem_u32(s_codes + stage * 2 * TILE), &tm_codes, 0, part * UNIT, hk, 0, page, &full[team][s]);
            tma_load_4d(smem_u32(s_scale + stage * 2 * UNIT * 4), &tm_scales, part * UNIT, hk, 0, page, &full[team][s]);
          }
        }
      }
    } while (wk.next(p));
  } else {
    // ------------------------------- consumers -------------------------------
    const int g = lane >> 2, t = lane & 3;
    const int team = warp >> 2, kw = (warp & 3) * 16 * KT;
    // Fragment row r (0..7) of a 16-key tile holds key ord(r) (and row r + 8 key ord(r) + 8).  The order is such that the
    // eight threads of a shared-memory phase touch all banks: the K rows of neighbouring fragment rows (their 16-byte
    // chunks differ by the swizzle), and the V rows ord(2t), ord(2t + 1) of the threads of a quad.
    auto ord = [](int r) {
      if (D == 128) return (r & 6) ^ ((r & 1) * 5);
      const int q = r >> 1;
      return ((q & 1) | ((q & 2) << 1)) ^ ((r & 1) * 3);
    };
    // byte offset of 16-byte chunk c of row r in a tile, as the tensor map's swizzle leaves it
    auto at = [](int row, int c) { return row * D + ((D == 128 ? c ^ (row & 7) : c ^ ((row >> 1) & 3)) << 4); };
    const int key0 = kw + ord(g);
    const int va = kw + ord(2 * t), vb = kw + ord(2 * t + 1);
    const uint32_t k_off = at(key0, t);                                             // chunks t and (D = 128) t + 4: ^ 64
    const uint32_t v_off_a = TILE + (D == 128 ? at(va, g) : at(va, g >> 1) + (g & 1) * 8);
    const uint32_t v_off_b = TILE + (D == 128 ? at(vb, g) : at(vb, g >> 1) + (g & 1) * 8);

    uint32_t n = 0, nv = 0;   // running counts of this team: units, visits
    if (any) do {
      int first, step;
      if (!wk.template mine<TEAMS>(team, first, step)) continue;
      const int hk = wk.head / p.head_blocks, hb = wk.head - hk * p.head_blocks;
      const int h0 = hk * p.G + hb * HEADS, n_heads = min(HEADS, p.G - hb * HEADS);
      // queries of this item as B fragments: thread (g, t) holds head g (+ 8), the channels of chunks t (and t + 4)
      uint32_t qf[NT][KSTEPS][2];
      float qs[NT][2];   // scale * log2(e) / power of two of heads 2t and 2t + 1
      const uint32_t slot = nv % QSLOTS;
      mbar_wait(&q_full[team][slot], (nv / QSLOTS) & 1, abortp, p.err, CS_ERR_TIMEOUT_TMA);
      ++nv;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + g;
        uint32_t raw[KSTEPS * 2];
        const uint32_t src = smem_u32(s_q + (team * QSLOTS + slot) * Shape::Q) + (h * D + t * 16) * 2;
#pragma unroll
        for (int c = 0; c < KSTEPS / 4; ++c)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4 v = h < n_heads ? lds128(src + c * 128 + half * 16) : make_uint4(0, 0, 0, 0);
            raw[c * 8 + half * 4] = v.x; raw[c * 8 + half * 4 + 1] = v.y;
            raw[c * 8 + half * 4 + 2] = v.z; raw[c * 8 + half * 4 + 3] = v.w;
          }
        uint32_t mx = 0;   // largest exponent, as the sign-less bits of the largest magnitude
#pragma unroll
        for (int i = 0; i < KSTEPS * 2; ++i) mx = max(mx, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        // bring the largest element into [2^14, 2^15): as far from fp16's subnormals as its range allows
        const int shift = min(max(127 + 14 - static_cast<int>(mx >> 7), -120), 120);
        const float up = __uint_as_float(static_cast<uint32_t>(127 + shift) << 23);
#pragma unroll
        for (int i = 0; i < KSTEPS; ++i) {
          qf[nt][i][0] = pack_half2(bf16lo(raw[2 * i]) * up, bf16hi(raw[2 * i]) * up);
          qf[nt][i][1] = pack_half2(bf16lo(raw[2 * i + 1]) * up, bf16hi(raw[2 * i + 1]) * up);
        }
        const float down = p.scale_log2 * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
        qs[nt][0] = __shfl_sync(0xffffffffu, down, t * 8);
        qs[nt][1] = __shfl_sync(0xffffffffu, down, t * 8 + 4);
      }
      if (lane == 0) mbar_arrive(&q_empty[team][slot]);
      // Weights are relative to the exponent r, 6 below the maximum m, so they reach up to 2^14.  Of large scores m itself is taken
      // first, and r is what is left to take.
      float o[NT][MT][4], m[NT][2], r[NT][2], l[NT][2];
      bool large = false;                       // of the warp
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = r[nt][0] = r[nt][1] = M_NONE;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      }

      for (int u = first; u < wk.u + wk.n; u += step, ++n) {
        const uint32_t s = n % RING;
        const uint32_t codes = smem_u32(s_codes + (team * RING + s) * 2 * TILE);
        const uint32_t scale = smem_u32(s_scale + (team * RING + s) * 2 * UNIT * 4);
        mbar_wait(&full[team][s], (n / RING) & 1, abortp, p.err, CS_ERR_TIMEOUT_TMA);
        __syncwarp();                          // every lane polls for itself; the products below are warp-wide
        const int valid = wk.len - u * UNIT;   // keys of the unit that exist (may exceed UNIT)
        if (kw < valid) {
          // ---- S^T = K Q^T for KT tiles of 16 keys; two chains of products per tile
          float c[KT][NT][4], ks[KT][2], lv[KT][2];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            uint32_t k0[KSTEPS], k1[KSTEPS];   // codes of keys key0 and key0 + 8, four channels per word
#pragma unroll
            for (int i = 0; i < KSTEPS / 4; ++i) {
              const uint32_t addr = codes + (k_off ^ (i * 64)) + kt * 16 * D;
              const uint4 x = lds128(addr), y = lds128(addr + 8 * D);
              k0[i * 4] = x.x; k0[i * 4 + 1] = x.y; k0[i * 4 + 2] = x.z; k0[i * 4 + 3] = x.w;
              k1[i * 4] = y.x; k1[i * 4 + 1] = y.y; k1[i * 4 + 2] = y.z; k1[i * 4 + 3] = y.w;
            }
            const uint32_t sc = scale + (key0 + kt * 16) * 4;
            ks[kt][0] = lds32(sc); ks[kt][1] = lds32(sc + 32);
            lv[kt][0] = lds32(sc + UNIT * 4); lv[kt][1] = lds32(sc + UNIT * 4 + 32);
            float c2[NT][4];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) c[kt][nt][j] = c2[nt][j] = 0.f;
#pragma unroll
            for (int i = 0; i < KSTEPS; ++i) {
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_half2x2(k0[i], a0, a2);
              e4m3x4_to_half2x2(k1[i], a1, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816((i & 1) ? c2[nt] : c[kt][nt], a0, a1, a2, a3, qf[nt][i][0], qf[nt][i][1]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) c[kt][nt][j] = (c[kt][nt][j] + c2[nt][j]) * (ks[kt][j >> 1] * qs[nt][j & 1]);
#pragma unroll
            for (int j = 0; j < 2; ++j) lv[kt][j] = lv[kt][j] < 1.2e-38f ? -126.f : __log2f(lv[kt][j]);
          }
          // the value rows of this thread: keys va, vb and those 8 further, per tile
          uint32_t x[KT][4][VPER / 4];
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const uint32_t addr = codes + ((r & 1) ? v_off_b : v_off_a) + (kt * 16 + (r >> 1) * 8) * D;
              if constexpr (D == 128) {
                const uint4 v = lds128(addr);
                x[kt][r][0] = v.x; x[kt][r][1] = v.y; x[kt][r][2] = v.z; x[kt][r][3] = v.w;
              } else {
                const uint2 v = lds64(addr);
                x[kt][r][0] = v.x; x[kt][r][1] = v.y;
              }
            }
          if (valid < UNIT) {   // the sequence ends in this unit: what lies behind it may be anything
#pragma unroll
            for (int kt = 0; kt < KT; ++kt) {
#pragma unroll
              for (int j = 0; j < 2; ++j)
                if (key0 + kt * 16 + j * 8 >= valid) {
                  lv[kt][j] = 0.f;
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt) c[kt][nt][2 * j] = c[kt][nt][2 * j + 1] = -INFINITY;
                }
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (((r & 1) ? vb : va) + kt * 16 + (r >> 1) * 8 >= valid) {
#pragma unroll
                  for (int j = 0; j < VPER / 4; ++j) x[kt][r][j] = 0u;
                }
            }
          }
          bool grow = false;
#pragma unroll
          for (int kt = 0; kt < KT; ++kt)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 4; ++j) grow |= c[kt][nt][j] + lv[kt][j >> 1] > m[nt][j & 1] + 8.f;
          // The reference moves only when a weight would pass 2^14, which after the first tiles is rare
          if (__any_sync(0xffffffffu, grow || large)) {
            auto all_keys = [](float x) {            // the maximum over the lanes of a head
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
              x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
              return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            };
            const bool was_large = large;
            bool far = false;
            float mx[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                mx[nt][j] = m[nt][j];
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) mx[nt][j] = fmaxf(mx[nt][j], fmaxf(c[kt][nt][j] + lv[kt][0], c[kt][nt][2 + j] + lv[kt][1]));
                mx[nt][j] = all_keys(mx[nt][j]);
                far |= fabsf(mx[nt][j]) > LARGE_EXPONENT && mx[nt][j] != M_NONE;
              }
            large = __any_sync(0xffffffffu, far);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const float had = was_large ? -r[nt][j] : 6.f;
                float room = 6.f;
                if (large) {
                  float top = -INFINITY;             // the largest weight relative to mx
#pragma unroll
                  for (int kt = 0; kt < KT; ++kt) {
                    c[kt][nt][j] -= mx[nt][j];
                    c[kt][nt][2 + j] -= mx[nt][j];
                    top = fmaxf(top, fmaxf(c[kt][nt][j] + lv[kt][0], c[kt][nt][2 + j] + lv[kt][1]));
                  }
                  top = all_keys(top);
                  room = mx[nt][j] > m[nt][j] || top + had > 14.f ? 6.f - top : had;
                }
                const float alpha = ex2((m[nt][j] - mx[nt][j]) + (room - had));
                m[nt][j] = mx[nt][j];
                r[nt][j] = large ? -room : mx[nt][j] - 6.f;
                l[nt][j] *= alpha;
#pragma unroll
                for (int i = 0; i < MT; ++i) { o[nt][i][j] *= alpha; o[nt][i][2 + j] *= alpha; }
              }
          }
#pragma unroll
          for (int kt = 0; kt < KT; ++kt) {
            uint32_t b0[NT], b1[NT];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float w[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float e = c[kt][nt][j] - r[nt][j & 1];
                l[nt][j & 1] += ex2(e);
                w[j] = ex2(e + lv[kt][j >> 1]);
              }
              b0[nt] = transpose8x8(pack_half2(w[0], w[1]));
              b1[nt] = transpose8x8(pack_half2(w[2], w[3]));
            }
            // ---- O^T += V^T P: fragment row g of tile i is channel VPER g + 2 i, row g + 8 the next one
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
              uint32_t a0, a1, a2, a3;
              e4m3x4_to_half2x2(__byte_perm(x[kt][0][i >> 1], x[kt][1][i >> 1], sel), a0, a1);
              e4m3x4_to_half2x2(__byte_perm(x[kt][2][i >> 1], x[kt][3][i >> 1], sel), a2, a3);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][i], a0, a1, a2, a3, b0[nt], b1[nt]);
            }
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[team][s]);
      }

      // ---- the warps' sums meet in shared memory, [warp][head][channel]; then every warp finishes some heads
      const bool shared = wk.shared();
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
          const int h = nt * 8 + 2 * t + j;
          if (g == 0) { s_m[warp][h] = large ? m[nt][j] + r[nt][j] : r[nt][j]; s_l[warp][h] = l[nt][j]; }
          float* dst = s_join + (warp * HEADS + h) * JOIN_LD + g * VPER;
#pragma unroll
          for (int i = 0; i < MT; i += 2)
            *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[nt][i][j], o[nt][i][2 + j], o[nt][i + 1][j], o[nt][i + 1][2 + j]);
        }
      auto meet = [&]() {
        if (shared) asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
        else asm volatile("bar.sync %0, 128;" ::"r"(2 + team) : "memory");
      };
      meet();
      const bool whole = wk.u == 0 && wk.n == wk.units;
      const int out_slot = c * 2 + (wk.u == 0 ? 1 : 0);   // an item that began before the run is its first, one that goes on its last
      auto finish = [&](auto count, int w0) {             // `count` warps from w0 on took part and share the outputs
        constexpr int W = decltype(count)::value;
        const int part = out_slot * HEADS;
        if (!whole && warp == w0 && lane == 0) p.ws_item[out_slot] = wk.seq * heads + wk.head;
#pragma unroll
        for (int i = 0; i < (HEADS * D / 4 + W * 32 - 1) / (W * 32); ++i) {
          const int idx = (warp - w0 + i * W) * 32 + lane, h = idx / (D / 4), ch = idx % (D / 4);
          if (h >= n_heads) continue;
          float f[W], mx = M_NONE, sum = 0.f;
#pragma unroll
          for (int w = 0; w < W; ++w) { f[w] = s_m[w0 + w][h]; mx = fmaxf(mx, f[w]); }
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < W; ++w) {
            const float e = ex2(f[w] - mx);
            sum += s_l[w0 + w][h] * e;
            const float4 v = *reinterpret_cast<const float4*>(s_join + ((w0 + w) * HEADS + h) * JOIN_LD + ch * 4);
            acc.x += v.x * e; acc.y += v.y * e; acc.z += v.z * e; acc.w += v.w * e;
          }
          if (whole) {
            store_head(p, wk.row, h0 + h, ch, acc, sum);
          } else {
            *reinterpret_cast<float4*>(p.ws_o + (part + h) * D + ch * 4) = acc;
            if (ch == 0) { p.ws_ml[(part + h) * 2] = mx; p.ws_ml[(part + h) * 2 + 1] = sum; }
          }
        }
      };
      if (shared) finish(Count<WARPS>{}, 0); else finish(Count<4>{}, team * 4);
      meet();   // the join area is written again at the end of the next visit
    } while (wk.next(p));

    // queries without keys give zeros
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
      if (threadIdx.x == 0 && !fits(p, b)) cs_set_error(p.err, CS_ERR_BAD_ARG);
      const Seq s = get_seq(p, b);
      if (s.row >= 0 && s.len == 0)
        for (int i = threadIdx.x; i < p.Hq * D; i += WARPS * 32) p.o[s.row * p.o_tok + (i / D) * p.o_head + i % D] = __float2bfloat16(0.f);
    }
  }
}

// Joins the items that several CTAs worked on: block (c, h) takes head h of the item whose first part is the last of
// decode CTA c.  Its parts are slot 1 of CTA c and slot 0 of the CTAs behind it; warp w reads parts w, w + 4, ...
template <int D, int NT>
__global__ void __launch_bounds__(128) attention_decode_fp8_join_kernel(const DecParams p, int ctas) {
  constexpr int HEADS = 8 * NT;
  __shared__ float s_acc[4][D], s_ml[4][2];
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int item = p.ws_item[c * 2 + 1];
  int behind = c + 1 + threadIdx.x < ctas ? p.ws_item[(c + 1 + threadIdx.x) * 2] : -1;
  if (item < 0) return;
  const int heads = p.Hkv * p.head_blocks, seq = item / heads, head = item - seq * heads;
  const int hk = head / p.head_blocks, hb = head - hk * p.head_blocks;
  if (hb * HEADS + h >= p.G) return;
  int parts = 1 + __syncthreads_count(behind == item);
  for (int first = c + 129; parts % 128 == 1 && parts > 1 && first < ctas; first += 128) {   // more than 128 CTAs on one item
    behind = first + threadIdx.x < ctas ? p.ws_item[(first + threadIdx.x) * 2] : -1;
    const int more = __syncthreads_count(behind == item);
    parts += more;
    if (more < 128) break;
  }
  float m = M_NONE, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = warp; i < parts; i += 4) {
    const long long row = ((c + i) * 2 + (i == 0 ? 1 : 0)) * HEADS + h;
    const float mi = p.ws_ml[row * 2], li = p.ws_ml[row * 2 + 1];
    const float4 v = lane * 4 < D ? *reinterpret_cast<const float4*>(p.ws_o + row * D + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float mx = fmaxf(m, mi), a = ex2(m - mx), b = ex2(mi - mx);
    m = mx;
    l = l * a + li * b;
    acc.x = acc.x * a + v.x * b; acc.y = acc.y * a + v.y * b; acc.z = acc.z * a + v.z * b; acc.w = acc.w * a + v.w * b;
  }
  if (lane * 4 < D) *reinterpret_cast<float4*>(&s_acc[warp][lane * 4]) = acc;
  if (lane == 0) { s_ml[warp][0] = m; s_ml[warp][1] = l; }
  __syncthreads();
  if (warp != 0 || lane * 4 >= D) return;
  m = fmaxf(fmaxf(s_ml[0][0], s_ml[1][0]), fmaxf(s_ml[2][0], s_ml[3][0]));
  l = 0.f;
  acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float e = ex2(s_ml[w][0] - m);
    const float4 v = *reinterpret_cast<const float4*>(&s_acc[w][lane * 4]);
    l += s_ml[w][1] * e;
    acc.x += v.x * e; acc.y += v.y * e; acc.z += v.z * e; acc.w += v.w * e;
  }
  store_head(p, get_seq(p, seq).row, hk * p.G + hb * HEADS + h, lane, acc, l);
}

template <int D, int NT>
int launch_decode(const void* cache, DecParams& p, int ctas, cudaStream_t stream) {
  using Shape = DecShape<D, NT>;
  static bool attr_done[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -10;
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(attention_decode_fp8_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM) != cudaSuccess)
      return -10;
    attr_done[dev] = true;
  }
  // no more CTAs than runs that full tables would make
  const long long most = static_cast<long long>(p.B) * p.Hkv * p.head_blocks * (p.bt_width * (KV8_PAGE / Shape::UNIT) + ITEM_COST) / MIN_RUN;
  if (most < ctas) ctas = most > 0 ? static_cast<int>(most) : 1;
  // one box = the K and V codes (or scales) of one unit of one head and page
  CUtensorMap tm_codes, tm_scales;
  const uint64_t blk = kv8_block_bytes(D), pages = p.num_pages, hkv = p.Hkv;
  const uint64_t dims[5] = {D, KV8_PAGE, hkv, 2, pages}, strides[4] = {D, blk, hkv * blk, 2 * hkv * blk};
  const uint32_t box[5] = {D, Shape::UNIT, 1, 2, 1};
  const uint64_t sdims[4] = {KV8_PAGE, hkv, 2, pages}, sstrides[3] = {blk, hkv * blk, 2 * hkv * blk};
  const uint32_t sbox[4] = {Shape::UNIT, 1, 2, 1};
  if (cs_encode_tmap_nd(&tm_codes, 1, 5, cache, dims, strides, box, D)) return -3;
  if (cs_encode_tmap_nd(&tm_scales, 4, 4, static_cast<const uint8_t*>(cache) + KV8_PAGE * D, sdims, sstrides, sbox, 0)) return -3;
  if (cs_launch_pdl(attention_decode_fp8_kernel<D, NT>, dim3(ctas), dim3(Shape::THREADS), Shape::SMEM, stream, tm_codes, tm_scales, p) !=
      cudaSuccess)
    return -10;
  return cs_launch_pdl(attention_decode_fp8_join_kernel<D, NT>, dim3(ctas, p.G < Shape::HEADS ? p.G : Shape::HEADS), dim3(128), 0, stream, p,
                       ctas) == cudaSuccess ? 0 : -10;
}

}  // namespace

// Scratch of one call (any sequence count): partial sums, their maxima and normalisers, and the items they belong to.
CS_API long long cs_attention_decode_fp8_ws_bytes(int Hq, int Hkv, int d) {
  if (Hkv <= 0) return 0;
  const int heads = Hq / Hkv <= 8 ? 8 : 16;
  const long long ctas = cs_num_sms() < MAX_CTAS ? cs_num_sms() : MAX_CTAS;
  return ctas * 2 * (heads * (d + 2LL) * 4 + 4);
}

// q: [B, Hq, d] with contiguous heads, tokens q_tok elements apart and on 16-byte boundaries; o: [B, Hq, d] with token and
// head strides in elements.  Sequence b has the query of row cu_q[b], which sees all kv_len[b] keys, or none if cu_q[b + 1] is
// the same; rows of no sequence are left as they are.  ws: cs_attention_decode_fp8_ws_bytes
// of scratch that no call on another stream uses.
CS_API int cs_attention_decode_fp8(const void* q, long long q_tok, const void* cache, long long num_pages, void* o, long long o_tok,
                                   long long o_head, const void* cu_q, const void* kv_len, const void* block_table, long long bt_stride, int bt_width, int B,
                                   int Hq, int Hkv, int d, float scale, void* ws, long long ws_bytes, void* stream) {
  if (B <= 0) return 0;
  if ((d != 64 && d != 128) || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || num_pages <= 0 || num_pages > 0x7fffffffLL) return -1;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_tok & 7)) return -1;
  DecParams p{};
  p.q = (const __nv_bfloat16*)q; p.q_tok = q_tok;
  p.o = (__nv_bfloat16*)o; p.o_tok = o_tok; p.o_head = o_head;
  p.o_vec = (reinterpret_cast<uintptr_t>(o) & 7) == 0 && (o_tok & 3) == 0 && (o_head & 3) == 0;
  p.num_pages = static_cast<int>(num_pages);
  p.block_table = (const int*)block_table; p.bt_stride = bt_stride; p.bt_width = bt_width;
  p.kv_len = (const int*)kv_len; p.cu_q = (const int*)cu_q;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
  const int heads = p.G <= 8 ? 8 : 16;
  p.head_blocks = (p.G + heads - 1) / heads;
  // lengths, and the cost of the whole batch were every table full, are added up in 32 bits on the device
  if (bt_width < 0 || bt_width > KV8_MAX_PAGES) return -1;
  if (static_cast<long long>(B) * Hkv * p.head_blocks > 0x7fffffffLL / (2LL * bt_width + ITEM_COST)) return -1;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = cs_error_word();
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < cs_attention_decode_fp8_ws_bytes(Hq, Hkv, d)) return -5;
  const int ctas = cs_num_sms() < MAX_CTAS ? cs_num_sms() : MAX_CTAS;
  p.ws_o = reinterpret_cast<float*>(ws);
  p.ws_ml = p.ws_o + static_cast<long long>(ctas) * 2 * heads * d;
  p.ws_item = reinterpret_cast<int*>(p.ws_ml + static_cast<long long>(ctas) * 2 * heads * 2);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (d == 128) return heads == 8 ? launch_decode<128, 1>(cache, p, ctas, st) : launch_decode<128, 2>(cache, p, ctas, st);
  return heads == 8 ? launch_decode<64, 1>(cache, p, ctas, st) : launch_decode<64, 2>(cache, p, ctas, st);
}
