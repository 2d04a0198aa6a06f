// Attention of packed prompts (or chunks of them) over the 8-bit paged key-value cache (layout in kv_fp8.cuh):
//
//   o_i = sum_j w_ij V_j / sum_j w_ij 2^-F_j,   w_ij = 2^(s_ij + F_j - M_i),   s_ij = scale * log2(e) * 2^E_j * (q_i . K_j)
//
// over the keys j that query i sees (all, or those up to its own position).  K_j = kc_j ks_j 2^-E and V_j = vc_j vs_j 2^-F
// are the cached rows (e4m3 codes times the fp32 scale of the row) in fp16, with one power of two per page that brings the
// page's largest scale to the top of fp16's range: code times scale is rounded once, to 11 bits, and the page's factors
// enter in fp32 as scalars.  (Scales could stay exact as a vector over the keys that the softmax applies, but every row's
// thread would have to read it from shared memory: 3 x 128 values per row and page made that the slowest part, at 8400
// cycles a page and tile pair.)  M_i follows the largest weight, not the largest score, so weights fit fp16 whatever the
// value scales are.  Queries become fp16 too, with a power of two per row that brings the row's largest element to the top of
// the range (every element within 2^-31 of that one is exact); its inverse is part of the row's factor in the softmax, so that
// rows do not touch each other, however far apart they are.
//
// One CTA works on 2 x 128 query rows of one sequence and one key head (rows = tokens x the query heads that share the
// key head) against pages of 128 keys:
//   warps 0-3, 4-7 : softmax of tile 0 / tile 1, one thread per row; scores come from TMEM, weights go back to TMEM over
//                    them and are the A operand of the second product there
//   warps 8-11, 12-15 : operand preparation, K tiles (and the queries of an item) / V tiles: codes and scales from global
//                    memory through registers to fp16 tiles in shared memory (128-byte swizzle)
//   warp 16        : issues tcgen05.mma: S_t = Q_t K^T (t = 0, 1) and O_t += P_t V.  While one tile's softmax runs, the
//                    tensor cores work for the other.
// The codes are converted once per 256 query rows.  They are not staged in shared memory as bytes: its bandwidth is what
// the products need most of (192 KB of operands per page and tile pair), so the preparation warps load them straight into
// registers.
//
// Work: the items (a tile pair of one sequence and key head, and all its pages) form one list; the CTAs cut it, on the
// device from the lengths, into runs of equal cost (visible keys, plus a constant per item).  An item that a cut goes
// through is worked on by two or more CTAs, which leave partial sums that a second kernel joins.  So prompts of any mix of
// lengths load all SMs alike, and a short chunk over a long cache is spread over the whole GPU.
//
// Measured inside a graph (28 query heads, 4 key heads, d = 128): one prompt of 16000 tokens 1.91 ms = 0.96 PFLOP/s (called for
// seconds, at the power limit, 2.16 ms = 0.85), 8 of 2000 tokens 358 us = 0.64 PFLOP/s, one of 300 24.4 us; 16 query and 2 key
// heads, d = 64: 3 chunks of 500 to 2100 tokens over 1000 to 9000 cached ones 214 us = 0.45 PFLOP/s.  A page of a tile pair takes
// 4300 cycles, of which the products are 2048 (1024 with d = 64) and the exponentials keep their unit busy for 2048; each softmax
// warp spends 1500 cycles waiting for its next scores, 600 on their maximum and 2000 on the weights.  An item costs 8000 to 13000
// cycles beside its pages, a good half of it for the output.
#include <math.h>

#include "kv_fp8.cuh"

namespace {

constexpr int ATOM = 128 * 128;            // 128 rows x 64 fp16, 128-byte swizzle
constexpr int RING = 2;                    // fp16 tiles of K and of V
constexpr int SRING = 4;                   // the two scalars of a page; at least RING + 2
constexpr int THREADS = 17 * 32;
constexpr float M_NONE = -3.0e38f;         // running maximum before the first key (finite: differences stay defined)
// Where exponents pass this, scores are taken relative to their page's largest before they are multiplied by their factor: the
// rounding of the product (2^-4 here, 1 at 2^24) would make weights that fp16 cannot hold, or none at all.
constexpr float LARGE_EXPONENT = 1048576.f;

static_assert(SRING >= RING + 2, "scalars outlive their tile by a page");

// What an item costs beside its keys, in keys.  8 prompts of 2000 tokens take 390 us with 2 pages, 367 with 3, 363 with 3.5, 373
// with 4.5; one of 16000 2.08 ms, 1.94, 1.91, 1.92.
constexpr int ITEM_COST = 7 * KV8_PAGE / 2;
// The cost of a CTA's run is this at least: one prompt of 300 tokens takes 27.2 us with 2 pages, 24.7 with 4, 35.2 with 8.
constexpr int MIN_RUN = 4 * KV8_PAGE;
constexpr int PAIR_ROWS = 256;

struct PrefillParams {
  const __nv_bfloat16* q; long long q_tok;              // heads follow each other; every token on a 16-byte boundary
  __nv_bfloat16* o; long long o_tok, o_head; int o_vec; // o_vec: 16-byte stores are aligned
  const uint8_t* cache; int num_pages;
  const int* block_table; long long bt_stride; int bt_width;
  const int* kv_len; const int* cu_q;
  int B, Tq, Hq, Hkv, G, blocks, causal;                // G query heads of a key head per tile row block; blocks = Hkv * row blocks
  int tok_per_tile;
  float scale_log2;
  float* ws_o;     // [ctas, 2, 256, D] partial sums: slot 0 = the first item of a CTA, begun by another, slot 1 = its last
  float* ws_ml;    // [ctas, 2, 256, 2] their maximum and normaliser
  int4* ws_item;   // [ctas, 2] the items (sequence, row block, pair), sequence -1 = none
  uint32_t idesc_s, idesc_pv;
  int* err;
};

// Lengths of a sequence, brought into the bounds of q and of the table.
struct Seq {
  int q_beg, q_len, k_len, shift;           // causal: query i sees keys j <= i + shift
};
__device__ __forceinline__ Seq get_seq(const PrefillParams& p, int s) {
  const int a = min(max(p.cu_q[s], 0), p.Tq), b = min(p.cu_q[s + 1], p.Tq), len = max(p.kv_len[s], 0);
  Seq q;
  q.q_beg = a;
  q.q_len = max(b - a, 0);
  q.k_len = min(len, p.bt_width * KV8_PAGE);
  q.shift = len - q.q_len;
  return q;
}
__device__ __forceinline__ int pairs_of(const PrefillParams& p, const Seq& q) { return (q.q_len + 2 * p.tok_per_tile - 1) / (2 * p.tok_per_tile); }
// Pages that pair k of a sequence looks at.
__device__ __forceinline__ int pages_of(const PrefillParams& p, const Seq& q, int k) {
  const int end = p.causal ? min(q.k_len, min(q.q_len, (k + 1) * 2 * p.tok_per_tile) + q.shift) : q.k_len;
  return end > 0 ? (end + KV8_PAGE - 1) / KV8_PAGE : 0;
}
// a / b for a >= 0 and b > 0; costs fit 32 bits but for huge batches
__device__ __forceinline__ long long quotient(long long a, long long b) {
  if (((a | b) >> 32) == 0) return static_cast<uint32_t>(a) / static_cast<uint32_t>(b);
  return a / b;
}
// Cost of the first n pairs of a sequence (one row block): a sum over an arithmetic progression.
__device__ __forceinline__ long long cost_of(const PrefillParams& p, const Seq& q, int n) {
  if (!p.causal) return static_cast<long long>(n) * (q.k_len + ITEM_COST);
  const int step = 2 * p.tok_per_tile;
  const int k0 = q.shift >= 0 ? 0 : min(n, (-q.shift) / step);       // pairs that end before the first key
  const long long m = n - k0;
  return m * q.shift + step * (m * (k0 + 1) + m * (m - 1) / 2) + static_cast<long long>(n) * ITEM_COST;
}

// A place in the list: page `page` of pair `pair` of row block `blk` of a sequence.
struct Pos { int seq, blk, pair, page; };

// The place at distance r (cost units) into the row blocks of sequence `seq`.  Cuts that would leave less than two pages of
// an item on one side move to its edge.
__device__ __forceinline__ Pos place_at(const PrefillParams& p, int seq, const Seq& q, long long r) {
  const int pairs = pairs_of(p, q);
  const long long per_blk = cost_of(p, q, pairs);
  Pos at{seq, static_cast<int>(quotient(r, per_blk)), 0, 0};
  r -= at.blk * per_blk;
  int lo = 0, hi = pairs;                   // the pair with cost_of(lo) <= r < cost_of(lo + 1)
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cost_of(p, q, mid) <= r) lo = mid; else hi = mid;
  }
  at.pair = lo;
  const int pages = pages_of(p, q, lo), cut = static_cast<int>(max(0ll, r - cost_of(p, q, lo) - ITEM_COST + KV8_PAGE / 2) / KV8_PAGE);
  if (cut < 2) return at;
  if (pages - cut >= 2) { at.page = cut; return at; }
  if (++at.pair == pairs) {                 // on to the next item
    at.pair = 0;
    if (++at.blk == p.blocks) { at.blk = 0; ++at.seq; }
  }
  return at;
}

// One visit of a CTA to an item: pages [j0, j0 + n) of a pair of query tiles of one sequence and key head (row block).
struct Item {
  int seq, hk, h0, n_heads, q_beg, q_len, t0, k_len, shift, j0, n;
  bool whole;                               // all pages of the item
};
struct Walk { Pos at, end; };               // of one warp, in shared memory

__device__ __forceinline__ void make_item(const PrefillParams& p, const Seq& q, int seq, int blk, int pair, Item& it) {
  const int group = p.Hq / p.Hkv, per = p.blocks / p.Hkv;
  it.seq = seq;
  it.hk = blk / per;
  const int first = (blk - it.hk * per) * p.G;
  it.h0 = it.hk * group + first;
  it.n_heads = min(p.G, group - first);
  it.q_beg = q.q_beg; it.q_len = q.q_len; it.k_len = q.k_len; it.shift = q.shift;
  it.t0 = pair * 2 * p.tok_per_tile;
}

// The next visit of this warp's walk (all lanes), or false.
__device__ __forceinline__ bool next_visit(const PrefillParams& p, Walk* w, Item* out) {
  Pos at = w->at;
  const Pos end = w->end;
  bool found = false;
  Item it;
  while (!found && at.seq < p.B) {
    const Seq q = get_seq(p, at.seq);
    const int pairs = pairs_of(p, q);
    if (at.pair >= pairs) { at = Pos{at.seq + 1, 0, 0, 0}; continue; }     // no queries
    const bool last = at.seq == end.seq && at.blk == end.blk && at.pair == end.pair;
    if (at.seq > end.seq || (last && (end.page == 0 || at.page >= end.page))) break;
    const int pages = pages_of(p, q, at.pair), stop = last ? min(end.page, pages) : pages;
    make_item(p, q, at.seq, at.blk, at.pair, it);
    it.j0 = at.page;
    it.n = stop - at.page;
    it.whole = at.page == 0 && stop == pages;
    found = it.n > 0 || pages == 0;
    if (last) {
      at.page = max(end.page, 1);           // behind the end
    } else {
      at.page = 0;
      if (++at.pair == pairs) {
        at.pair = 0;
        if (++at.blk == p.blocks) { at.blk = 0; ++at.seq; }
      }
    }
  }
  __syncwarp();
  if ((threadIdx.x & 31) == 0) w->at = at;
  __syncwarp();
  if (found) *out = it;
  return found;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint64_t pack2(float lo, float hi) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
  return v;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// D[tmem] (+)= A[tmem] * B[smem], fp16 inputs, fp32 accumulate
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Takes the scores of the rows of a warp whose limit is not 0 relative to the largest of their first `limit` ones, in place;
// that one is returned (0 for the other rows).  A function of its own: inside the loop over pages its registers cost 16000
// tokens 1.2 % and ragged prompts 1 to 2 %, although it hardly ever runs.
__device__ __noinline__ float relative_scores(uint32_t tS, int limit) {
  float top = limit > 0 ? M_NONE : 0.f;
#pragma unroll 1
  for (int c = 0; c < 2 * KV8_PAGE; c += 16) {
    uint32_t x[16];
    tmem_ld16(tS + (c & (KV8_PAGE - 1)), x);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if (c < KV8_PAGE) top = c + i < limit ? fmaxf(top, __uint_as_float(x[i])) : top;
      else x[i] = __float_as_uint(__uint_as_float(x[i]) - top);
    }
    if (c >= KV8_PAGE) tmem_st16(tS + c - KV8_PAGE, x);
  }
  tmem_wait_st();
  return top;
}

// Shared memory: queries (two tiles), ring of fp16 tiles.
template <int D>
struct Shape {
  static constexpr int ATOMS = D / 64, TILE = ATOMS * ATOM;
  static constexpr int Q = 2 * TILE;
  static constexpr int SMEM = 1024 + Q + 2 * RING * TILE;
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1) attention_prefill_fp8_kernel(const PrefillParams p) {
  constexpr int TILE = Shape<D>::TILE;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_q = smem;
  uint8_t* s_kv = smem + Shape<D>::Q;    // K tiles, V tiles
  __shared__ uint64_t q_full, q_empty, kv_full[2][RING], kv_empty[2][RING], sc_full[SRING], s_full[2], p_full[2], o_full[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;
  __shared__ Walk s_walk[THREADS / 32];
  __shared__ Pos s_pos[2];
  __shared__ long long s_sum[THREADS / 32], s_cut[2];
  __shared__ int s_cut_seq[2];
  __shared__ Seq s_cut_q[2];
  __shared__ uint32_t s_row[128];       // token in tile | head << 16 of a tile row
  __shared__ float s_qscale[2][2][128]; // [item parity][tile][row]: factor from S 2^E to base-2 exponents
  __shared__ float4 s_scale[SRING];     // of a page: 2^E, F, 2^-F

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    mbar_init(&q_full, 256);
    mbar_init(&q_empty, 1);
    for (int i = 0; i < 2 * RING; ++i) { mbar_init(&kv_full[i / RING][i % RING], 128); mbar_init(&kv_empty[i / RING][i % RING], 1); }
    for (int i = 0; i < SRING; ++i) mbar_init(&sc_full[i], 2);
    for (int t = 0; t < 2; ++t) { mbar_init(&s_full[t], 1); mbar_init(&p_full[t], 128); mbar_init(&o_full[t], 1); }
    mbar_fence_init();
  }
  if (warp == 16) { tmem_alloc(&tmem_slot, 512); tmem_relinquish(); }
  if (threadIdx.x < 128) s_row[threadIdx.x] = threadIdx.x / p.G | (threadIdx.x % p.G) << 16;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_wait();
  pdl_launch_dependents();
  if (threadIdx.x < 2) p.ws_item[blockIdx.x * 2 + threadIdx.x] = make_int4(-1, 0, 0, 0);

  // ------------------------------- this CTA's run of the list -------------------------------
  // Thread i adds up the cost of `per` consecutive sequences (one, unless the batch is huge); a scan over the threads gives
  // the total and who owns the two cuts.
  {
    const int per = (p.B + THREADS - 1) / THREADS, b0 = min(static_cast<int>(threadIdx.x) * per, p.B), b1 = min(b0 + per, p.B);
    auto seq_cost = [&](const Seq& q) { return cost_of(p, q, pairs_of(p, q)) * p.blocks; };
    const Seq first = b0 < b1 ? get_seq(p, b0) : Seq{0, 0, 0, 0};
    long long mine = seq_cost(first);
    for (int b = b0 + 1; b < b1; ++b) mine += seq_cost(get_seq(p, b));
    long long incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_sum[warp] = incl;
    if (threadIdx.x < 2) { s_cut_seq[threadIdx.x] = p.B; s_cut[threadIdx.x] = 0; }
    __syncthreads();
    long long total = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
      if (w == warp) incl += total;
      total += s_sum[w];
    }
    const long long active = max(1ll, min(static_cast<long long>(gridDim.x), total / MIN_RUN)), quota = quotient(total, active), extra = total - quota * active;
    for (int e = 0; e < 2; ++e) {
      const long long c = blockIdx.x + e, r = c >= active ? total : quota * c + min(c, extra);
      if (r >= incl - mine && r < incl) {
        long long at = incl - mine;
        int b = b0;
        Seq q = first;
        while (b + 1 < b1) {
          const long long x = seq_cost(q);
          if (r < at + x) break;
          at += x;
          q = get_seq(p, ++b);
        }
        s_cut_seq[e] = b;
        s_cut[e] = r - at;
        s_cut_q[e] = q;
      }
    }
    __syncthreads();
    if (warp < 2 && lane == 0) s_pos[warp] = s_cut_seq[warp] < p.B ? place_at(p, s_cut_seq[warp], s_cut_q[warp], s_cut[warp]) : Pos{p.B, 0, 0, 0};
    __syncthreads();
    if (lane == 0) s_walk[warp] = Walk{s_pos[0], s_pos[1]};
    __syncwarp();
  }
  Walk* walk = &s_walk[warp];
  const uint32_t tmem = tmem_slot;      // S_0, S_1 at columns 0, 128 (P_t over the first half of S_t), O_0, O_1 at 256, 384
  volatile int* abortp = &abort_flag;

  // No role leaves its loops early when a wait gives up: later waits return at once, and all keep their barriers company.
  if (warp == 16) {
    const bool leader = elect_one();
    {
      // -------------------------------- MMA issuer --------------------------------
      const uint32_t q_addr = smem_u32(s_q), kv_addr = smem_u32(s_kv);
      uint32_t n_item = 0, n_p = 0;     // running counts: items, pages (steps of the softmax)
      auto wait_kv = [&](int kv, uint32_t n) {
        mbar_wait(&kv_full[kv][n % RING], (n / RING) & 1, abortp, p.err, CS_ERR_TIMEOUT_TMA);
        tc_fence_after();
      };
      // (short loops: three roles run through their code in turn, and what does not stay in the instruction cache costs
      // more than the loop does)
      auto issue_s = [&](int t, uint32_t n) {
        uint64_t a = umma_smem_desc(q_addr + t * TILE, 16, 1024), b = umma_smem_desc(kv_addr + (n % RING) * TILE, 16, 1024);
#pragma unroll 1
        for (int atom = 0; atom < D / 64; ++atom, a += ATOM / 16, b += ATOM / 16)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f16_ss(tmem + t * 128, a + kk * 2, b + kk * 2, p.idesc_s, (atom | kk) != 0);
        umma_commit(&s_full[t]);
      };
      auto issue_pv = [&](int t, uint32_t n, bool first) {
        uint64_t b = umma_smem_desc(kv_addr + (RING + n % RING) * TILE, ATOM, 1024);
        uint32_t a = tmem + t * 128;
#pragma unroll 1
        for (int k4 = 0; k4 < 2; ++k4, a += 32, b += 4 * 128)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk) umma_f16_ts(tmem + 256 + t * 128, a + kk * 8, b + kk * 128, p.idesc_pv, !(first && (k4 | kk) == 0));
      };
      Item visit;      // (copied: what has its address taken lives in memory)
      while (next_visit(p, walk, &visit)) {
        const Item it = visit;
        if (it.n == 0 || !leader) continue;
        mbar_wait(&q_full, n_item & 1, abortp, p.err, CS_ERR_TIMEOUT_TMA);
        ++n_item;
        wait_kv(0, n_p);
        issue_s(0, n_p);
        issue_s(1, n_p);
        umma_commit(&kv_empty[0][n_p % RING]);
        if (it.n == 1) umma_commit(&q_empty);
        for (int j = 0; j < it.n; ++j, ++n_p) {
          const bool more = j + 1 < it.n;
          wait_kv(1, n_p);
          if (more) wait_kv(0, n_p + 1);
#pragma unroll 1
          for (int t = 0; t < 2; ++t) {
            mbar_wait(&p_full[t], n_p & 1, abortp, p.err, CS_ERR_TIMEOUT_EPI);
            tc_fence_after();
            issue_pv(t, n_p, j == 0);
            if (t == 1) umma_commit(&kv_empty[1][n_p % RING]);
            if (more) issue_s(t, n_p + 1); else umma_commit(&o_full[t]);
          }
          if (more) {
            umma_commit(&kv_empty[0][(n_p + 1) % RING]);
            if (j + 2 == it.n) umma_commit(&q_empty);
          }
        }
      }
    }
  } else if (warp >= 8) {
    // ------------------------------ operand preparation ------------------------------
    constexpr int CHUNKS = D / 16;                 // 16-byte chunks of codes per row
    constexpr int ITER = CHUNKS;                   // chunks per thread and tile (128 rows, 128 threads)
    const int kv = (warp - 8) >> 2, tid = threadIdx.x - 256 - kv * 128;     // 0: keys, 1: values
    // This thread's chunks are chunk c0 of rows row0, row0 + STEP, ...  The eight threads of a shared-memory phase write
    // two rows of different parity, so that the swizzle sends their stores to different banks.
    constexpr int STEP = 128 / CHUNKS;
    const int row0 = D == 128 ? (tid >> 5) * 4 + ((tid >> 4) & 1) * 2 + ((tid >> 2) & 1) : tid >> 2;
    const int c0 = D == 128 ? ((tid >> 3) & 1) * 4 + (tid & 3) : tid & 3;
    const int off_a = (c0 >> 2) * ATOM + row0 * 128 + ((((c0 & 3) * 2) ^ (row0 & 7)) << 4), off_b = off_a ^ 16;   // STEP is a multiple of 8
    // Lane L looks after the scale of one of the 32 rows of its warp (rows row0 + i * STEP over the warp's threads).
    constexpr int RPW = 32 / ITER;
    const int my_row = (warp & 3) * RPW + lane % RPW + STEP * (lane / RPW);
    uint32_t n = 0, n_item = 0;                    // running counts: pages, items
    // A tile in registers: codes, the scale of row `my_row` (with keys that of the value row too), the scales of keys 4 lane .. + 3
    constexpr int PART = 4, PARTS = ITER / PART;   // a tile is converted in parts, with the next part's codes on their way
    uint4 code[PART];
    float row_s, row_vs = 0.f;
    float4 all_s;
    int rows = 0;                                  // rows that are keys of the sequence (may exceed 128)
    auto page_of = [&](const Item& it, int j) { return j < it.j0 + it.n ? p.block_table[it.seq * p.bt_stride + j] : 0; };
    const long long page_bytes = 2 * p.Hkv * kv8_block_bytes(D);
    auto block_of = [&](const uint8_t* head, int page) {
      if (static_cast<unsigned>(page) >= static_cast<unsigned>(p.num_pages)) {
        if (tid == 0) cs_set_error(p.err, CS_ERR_BAD_ARG);
        page = 0;
      }
      return head + page * page_bytes;
    };
    auto fetch_scales = [&](const uint8_t* block) {
      const float* scales = reinterpret_cast<const float*>(block + KV8_PAGE * D);
      row_s = __ldg(scales + my_row);
      all_s = __ldg(reinterpret_cast<const float4*>(scales) + lane);
      if (kv == 0) {
        const float* values = reinterpret_cast<const float*>(block + p.Hkv * kv8_block_bytes(D) + KV8_PAGE * D);
        row_vs = __ldg(values + my_row);
      }
    };
    auto fetch_codes = [&](const uint8_t* from, int i) {
      code[i] = __ldg(reinterpret_cast<const uint4*>(from + row0 * D + c0 * 16 + i * STEP * D));
    };
    auto finite_bits = [](float f) { const uint32_t b = __float_as_uint(f) & 0x7fffffffu; return b < 0x7f800000u ? b : 0u; };
    auto is_finite = [](float f) { return (__float_as_uint(f) & 0x7fffffffu) < 0x7f800000u; };
    // The multiplier of row `my_row` as two fp16 parts, and the exponent E (or F) of the page.  Rows behind the sequence's
    // keys become 0, whatever is there.  A key row or value row with a scale that is no number makes the key a NaN, so that
    // queries that see it, and only those, become NaN; in V such a row is 0 (0 * NaN is not 0).
    auto multiplier = [&](uint32_t& parts) {
      const float a4[4] = {all_s.x, all_s.y, all_s.z, all_s.w};
      uint32_t mx = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) mx = max(mx, lane * 4 + k < rows ? finite_bits(a4[k]) : 0u);
      mx = __reduce_max_sync(0xffffffffu, mx);
      const int e = min(max(static_cast<int>(mx >> 23) - 127 - 6, -110), 120);      // the largest scale into [2^6, 2^7): codes reach 448
      float v = row_s * __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      if (!is_finite(row_s) || !is_finite(row_vs)) v = kv == 0 ? __uint_as_float(0x7fffffffu) : 0.f;
      if (my_row >= rows) v = 0.f;
      const __half h = __float2half_rn(v), r = __float2half_rn(v - __half2float(h));
      parts = __half_as_ushort(h) | static_cast<uint32_t>(__half_as_ushort(r)) << 16;
      return e;
    };
    auto scaled = [](uint32_t c, uint32_t hi, uint32_t lo) {      // c * (hi + lo), rounded once
      const __half2 x = *reinterpret_cast<const __half2*>(&c), h = *reinterpret_cast<const __half2*>(&hi), l = *reinterpret_cast<const __half2*>(&lo);
      const __half2 y = __hfma2(x, h, __hmul2(x, l));
      return *reinterpret_cast<const uint32_t*>(&y);
    };
    // The scalars of page n, once its tile's place was free.  Their own place was that of page n - SRING, which both softmax
    // groups are done with: the tile of page n - RING is free only behind products that waited for the weights of page
    // n - RING - 1 or a later one.
    auto publish = [&](int e) {
      if (tid != 0) return;
      const uint32_t s = n % SRING;
      if (kv == 0) {
        s_scale[s].x = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
      } else {
        s_scale[s].y = static_cast<float>(e);
        s_scale[s].z = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
      }
      mbar_arrive(&sc_full[s]);
    };
    // Convert a tile and, chunk by chunk, fetch the next part into the registers that become free.  (Parts of 64 of 128 rows at
    // d = 128: half the registers and code of a whole tile at once, 9 prompts of 17 to 2300 tokens 180 -> 178 us; quarters 182.)
    auto convert = [&](uint32_t parts, const uint8_t* block, const uint8_t* next, int e, bool pub) {
      const uint32_t slot = n % RING;
      mbar_wait(&kv_empty[kv][slot], ((n / RING) & 1) ^ 1, abortp, p.err, CS_ERR_TIMEOUT_SLOT);
      if (pub) publish(e);
      uint8_t* tile = s_kv + (kv * RING + slot) * TILE;
#pragma unroll 1
      for (int k = 0; k < PARTS; ++k, tile += PART * STEP * 128) {
        const uint8_t* from = k + 1 < PARTS ? block + (k + 1) * PART * STEP * D : next;
        const int row = row0 + k * PART * STEP, first = k * PART * RPW + row0 % RPW;
        if (rows < KV8_PAGE) {                     // what lies behind the keys may be anything
#pragma unroll
          for (int i = 0; i < PART; ++i)
            if (row + i * STEP >= rows) code[i] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < PART; ++i) {
          const uint32_t f = __shfl_sync(0xffffffffu, parts, first + i * RPW);
          const uint32_t hi = __byte_perm(f, 0, 0x1010), lo = __byte_perm(f, 0, 0x3232);
          const uint32_t w[4] = {code[i].x, code[i].y, code[i].z, code[i].w};
          fetch_codes(from, i);
          uint32_t h[8];
#pragma unroll
          for (int c = 0; c < 4; ++c) e4m3x4_to_half2x2(w[c], h[2 * c], h[2 * c + 1]);
#pragma unroll
          for (int c = 0; c < 8; ++c) h[c] = scaled(h[c], hi, lo);
          *reinterpret_cast<uint4*>(tile + off_a + i * STEP * 128) = make_uint4(h[0], h[1], h[2], h[3]);
          *reinterpret_cast<uint4*>(tile + off_b + i * STEP * 128) = make_uint4(h[4], h[5], h[6], h[7]);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&kv_full[kv][slot]);
    };
    // Queries, one tile per group, D / 8 lanes per row: copied as they are to the place where their fp16 form will be, all
    // in flight at once.
    constexpr int LANES = D / 8, PER = 32 / LANES, PASSES = 32 / PER;     // lanes per row, rows per warp and pass, passes
    const int ch = lane % LANES, row_w = (warp & 3) * PER + lane / LANES;
    // row i * 4 * PER + row_w: its swizzle is the same in all passes (4 * PER is a multiple of 8)
    uint8_t* q_at = s_q + kv * TILE + (ch >> 3) * ATOM + row_w * 128 + (((ch & 7) ^ (row_w & 7)) << 4);
    auto fetch_queries = [&](const Item& it) {
      const int t0 = it.t0 + kv * p.tok_per_tile, n_tok = min(p.tok_per_tile, it.q_len - t0);
      const __nv_bfloat16* src0 = p.q + (it.q_beg + (n_tok > 0 ? t0 : 0)) * p.q_tok + it.h0 * D + ch * 8;
      const uint32_t q_sm = smem_u32(q_at);
#pragma unroll 8
      for (int i = 0; i < PASSES; ++i) {
        const uint32_t rc = s_row[i * 4 * PER + row_w];                   // token in tile | head << 16
        const int tl = rc & 0xffff, g = rc >> 16;
        const bool ok = tl < n_tok && g < it.n_heads;
        const __nv_bfloat16* src = ok ? src0 + tl * p.q_tok + g * D : src0;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(q_sm + i * 4 * PER * 128), "l"(src), "r"(ok ? 16 : 0) : "memory");
      }
    };
    Item visit;
    while (next_visit(p, walk, &visit)) {
      const Item it = visit;
      if (it.n == 0) continue;
      if (n_item == 0) fetch_queries(it);            // their place is free (one prompt of 300 tokens: 24.5 -> 24.1 us)
      const uint8_t* head = p.cache + (static_cast<long long>(kv) * p.Hkv + it.hk) * kv8_block_bytes(D);
      const uint8_t* block = block_of(head, page_of(it, it.j0));
      fetch_scales(block);
#pragma unroll
      for (int i = 0; i < PART; ++i) fetch_codes(block, i);
      int page = page_of(it, it.j0 + 1);
#pragma unroll 1
      for (int j = it.j0; j < it.j0 + it.n; ++j, ++n) {
        // the tile of a page, and the next page's scales and codes on their way
        uint32_t parts;
        rows = it.k_len - j * KV8_PAGE;
        const int e = multiplier(parts);
        const uint8_t* here = block;
        if (j + 1 < it.j0 + it.n) block = block_of(head, page);   // (behind the last page the same one is read again)
        fetch_scales(block);
        page = page_of(it, j + 2);
        convert(parts, here, block, e, j > it.j0);
        if (j > it.j0) continue;
        // The queries of later items come behind the first tile, which does not need them: the item before is still at work on
        // its own.  Then the largest magnitude of every row, and fp16 scaled by the row's power of two in place.
        if (n_item > 0) {
          mbar_wait(&q_empty, (n_item & 1) ^ 1, abortp, p.err, CS_ERR_TIMEOUT_SLOT);
          fetch_queries(it);
        }
        // (two sets of factors: the item before the last is done with its own, since the wait above is behind its softmax)
        float* row_scale = s_qscale[n_item & 1][kv];
        ++n_item;
        asm volatile("cp.async.wait_all;" ::: "memory");
        asm volatile("bar.sync %0, 128;" ::"r"(1 + kv) : "memory");     // the rows of this tile are there
        uint8_t* row_at = s_q + kv * TILE + tid * 128;                  // one thread per row
        const int swizzle = (tid & 7) << 4;
        auto chunk = [&](int c) { return reinterpret_cast<uint4*>(row_at + (c >> 3) * ATOM + (((c & 7) << 4) ^ swizzle)); };
        uint32_t m2 = 0;                             // largest magnitudes as bf16, of even and odd channels
#pragma unroll 4
        for (int c = 0; c < D / 8; ++c) {
          const uint4 v = *chunk(c);
          m2 = __vmaxu2(m2, __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu)));
        }
        const int ex = static_cast<int>(max(m2 & 0xffffu, m2 >> 16) >> 7);     // (255: the row is no number)
        const int shift = min(127 + 14 - ex, 120);                             // the largest element into [2^14, 2^15)
        // a negative scale turns the queries around, so that the largest score is the largest S
        const float up = copysignf(__uint_as_float(static_cast<uint32_t>(127 + shift) << 23), p.scale_log2);
        row_scale[tid] = fabsf(p.scale_log2) * __uint_as_float(static_cast<uint32_t>(127 - shift) << 23);
#pragma unroll 1
        for (int c = 0; c < D / 8; c += 4) {
          uint4 v[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) v[i] = *chunk(c + i);
#pragma unroll
          for (int i = 0; i < 4; ++i)
            *chunk(c + i) = make_uint4(half2_bits(bf16lo(v[i].x) * up, bf16hi(v[i].x) * up), half2_bits(bf16lo(v[i].y) * up, bf16hi(v[i].y) * up),
                                       half2_bits(bf16lo(v[i].z) * up, bf16hi(v[i].z) * up), half2_bits(bf16lo(v[i].w) * up, bf16hi(v[i].w) * up));
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_full);
        asm volatile("bar.sync %0, 128;" ::"r"(1 + kv) : "memory");     // the factors of all rows of this tile
        publish(e);
      }
    }
  } else {
    // ---------------------------------- softmax -----------------------------------
    const int t = warp >> 2, r = (warp & 3) * 32 + lane;         // tile, row == TMEM lane
    const int tl = r / p.G, g = r - tl * p.G;                    // token in tile, head within group
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lane_off, tO = tmem + 256 + t * 128 + lane_off;
    uint32_t n_step = 0, n_item = 0;
    Item visit;
    while (next_visit(p, walk, &visit)) {
      const Item it = visit;
      const int tok = it.t0 + t * p.tok_per_tile + tl;
      const bool row_ok = tl < p.tok_per_tile && tok < it.q_len && g < it.n_heads;
      const int lim = p.causal ? min(it.k_len, tok + it.shift + 1) : it.k_len;     // keys [0, lim) are visible
      const int wmin = __reduce_min_sync(0xffffffffu, lim);                        // ... to all rows of the warp
      float m = M_NONE;
      float l = 0.f;
      for (int j = 0; j < it.n; ++j, ++n_step) {
        const uint32_t s = n_step % SRING;
        mbar_wait(&sc_full[s], (n_step / SRING) & 1, abortp, p.err, CS_ERR_TIMEOUT_SLOT);
        mbar_wait(&s_full[t], n_step & 1, abortp, p.err, CS_ERR_TIMEOUT_MMA);
        __syncwarp();                                // every lane polls for itself; tcgen05.ld / st below are warp-wide
        tc_fence_after();
        const float4 sc = s_scale[s];
        // (not 0, also for a scale of 0: a hidden key's -inf times the factor has to stay -inf)
        const float product = s_qscale[n_item & 1][t][r] * sc.x, factor = product < 1e-37f ? 1e-37f : product;   // (a NaN stays one)
        const int nvalid = lim - (it.j0 + j) * KV8_PAGE;       // visible keys of the page (may be negative or beyond 128)
        const int wvalid = wmin - (it.j0 + j) * KV8_PAGE;      // the same for every row of the warp: no divergent branch
        // first pass: the largest S of the row
        float mx0 = -INFINITY, mx1 = -INFINITY;
        auto largest = [&](uint32_t (&x)[32], int c) {
          if (wvalid < c + 32) {                     // hidden keys: whatever is there
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c + i >= nvalid) x[i] = 0xff800000u;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            mx0 = fmaxf(fmaxf(mx0, __uint_as_float(x[i])), __uint_as_float(x[i + 1]));
            mx1 = fmaxf(fmaxf(mx1, __uint_as_float(x[i + 2])), __uint_as_float(x[i + 3]));
          }
        };
#pragma unroll 1
        for (int c = 0; c < KV8_PAGE; c += 64) {
          uint32_t x[32], y[32];
          tmem_ld32(tS + c, x);
          tmem_ld32(tS + c + 32, y);
          tmem_wait_ld();
          largest(x, c);
          largest(y, c + 32);
        }
        const float mx = fmaxf(mx0, mx1) * factor + sc.y;
        // The reference m - 6 moves only when a weight would pass 2^14
        const float m_new = mx > m + 8.f ? mx : m;
        if (__any_sync(0xffffffffu, m_new != m)) {   // tcgen05.ld / st are warp-wide: the warp decides together
          const float alpha = ex2(m - m_new);
          l *= alpha;
          if (j > 0) {                               // PV of the last page is complete: S of this one was issued behind it
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
              uint32_t o[16];
              tmem_ld16(tO + c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              tmem_st16(tO + c, o);
            }
          }
        }
        m = m_new;
        // second pass: weights and their sum; the weights of 32 keys take 16 columns and stay behind the scores still to be read
        float add = sc.y + (6.f - m);
        const bool large = fabsf(m) > LARGE_EXPONENT && nvalid > 0;
        if (__any_sync(0xffffffffu, large)) {
          const float top = relative_scores(tS, large ? nvalid : 0);
          if (large) add = ((top * factor + sc.y) - m) + 6.f;
        }
        const uint64_t mul2 = pack2(factor, factor), ref2 = pack2(add, add);
        uint64_t sum_a = pack2(0.f, 0.f), sum_b = sum_a;
        auto weigh = [&](uint32_t (&x)[32], int c) {
          if (wvalid < c + 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c + i >= nvalid) x[i] = 0xff800000u;
          }
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float e0, e1, e2, e3;
            unpack2(fma2(pack2(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), mul2, ref2), e0, e1);
            unpack2(fma2(pack2(__uint_as_float(x[i + 2]), __uint_as_float(x[i + 3])), mul2, ref2), e2, e3);
            e0 = ex2(e0); e1 = ex2(e1); e2 = ex2(e2); e3 = ex2(e3);
            sum_a = add2(sum_a, pack2(e0, e1));
            sum_b = add2(sum_b, pack2(e2, e3));
            pk[i >> 1] = half2_bits(e0, e1);
            pk[(i >> 1) + 1] = half2_bits(e2, e3);
          }
          tmem_st16(tS + (c >> 1), pk);
        };
#pragma unroll 1
        for (int c = 0; c < KV8_PAGE; c += 32) {
          uint32_t x[32];
          tmem_ld32(tS + c, x);
          tmem_wait_ld();
          weigh(x, c);
        }
        {
          float s0, s1;
          unpack2(add2(sum_a, sum_b), s0, s1);
          l += (s0 + s1) * sc.z;
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[t]);
      }
      // ---------------------------------- output ------------------------------------
      if (it.n > 0) {
        mbar_wait(&o_full[t], n_item & 1, abortp, p.err, CS_ERR_TIMEOUT_MMA);
        __syncwarp();
        ++n_item;
        tc_fence_after();
      }
      // a partial sum goes to slot 0 when another CTA began the item, to slot 1 when this one did
      const int slot = blockIdx.x * 2 + (it.j0 == 0 ? 1 : 0);
      const long long row = static_cast<long long>(slot) * PAIR_ROWS + t * 128 + r;
      if (!it.whole) {
        if (row_ok) { p.ws_ml[row * 2] = m; p.ws_ml[row * 2 + 1] = l; }
        if (threadIdx.x == 0) p.ws_item[slot] = make_int4(it.seq, it.h0, it.t0, 0);
      }
      // (a row that sees no key is 0; one whose scores are all -inf has a sum of 0 and becomes 0 / 0)
      const float inv = !it.whole ? 1.f : (lim > 0 ? 1.f / l : 0.f);
      __nv_bfloat16* dst = p.o + static_cast<long long>(it.q_beg + tok) * p.o_tok + (it.h0 + g) * p.o_head;
      float* part = p.ws_o + row * D;
      const bool mate_ok = __shfl_xor_sync(0xffffffffu, row_ok, 1);
      __nv_bfloat16* mate = reinterpret_cast<__nv_bfloat16*>(__shfl_xor_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), 1));
      const bool even_ok = (lane & 1) ? mate_ok : row_ok, odd_ok = (lane & 1) ? row_ok : mate_ok;
      __nv_bfloat16 *dst_even = ((lane & 1) ? mate + 8 : dst), *dst_odd = ((lane & 1) ? dst + 8 : mate);
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {
        uint32_t o[16];
        if (it.n > 0) {
          tmem_ld16(tO + c * 16, o);
          tmem_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) o[i] = 0u;
        }
        float f[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) f[i] = __uint_as_float(o[i]) * inv;
        if (!it.whole) {
          if (row_ok) {
#pragma unroll
            for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(part + c * 16 + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
          }
        } else if (p.o_vec) {
          // Neighbours trade halves, so that a store covers whole sectors (32 bytes of 16 rows, not 16 of 32: 9 prompts of
          // 17 to 2300 tokens 188 -> 183 us, one of 300 26.3 -> 24.9 us).
          uint32_t w[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) w[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
          const bool odd = lane & 1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? w[i] : w[4 + i], 1);
            if (odd) w[i] = got; else w[4 + i] = got;
          }
          if (even_ok) *reinterpret_cast<uint4*>(dst_even + c * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          if (odd_ok) *reinterpret_cast<uint4*>(dst_odd + c * 16) = make_uint4(w[4], w[5], w[6], w[7]);
        } else if (row_ok) {
#pragma unroll
          for (int i = 0; i < 16; ++i) dst[c * 16 + i] = __float2bfloat16(f[i]);
        }
        __syncwarp();                              // the next read of TMEM is the whole warp's
      }
      tc_fence_before();
    }
    // lengths that do not fit the table or the queries are reported
    for (int b = blockIdx.x * 256 + threadIdx.x; b < p.B; b += gridDim.x * 256)
      if (p.kv_len[b] < 0 || p.kv_len[b] > p.bt_width * KV8_PAGE || p.cu_q[b] < 0 || p.cu_q[b + 1] < p.cu_q[b] || p.cu_q[b + 1] > p.Tq)
        cs_set_error(p.err, CS_ERR_BAD_ARG);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) { tc_fence_after(); tmem_dealloc(tmem, 512); }
}

// Joins the items that several CTAs worked on: blocks (c, y) take rows 8 y .. + 7 of the item whose first part is the last of
// CTA c, one warp per row.  The parts are slot 1 of CTA c and slot 0 of the CTAs behind it, read in order.
template <int D>
__global__ void __launch_bounds__(256) attention_prefill_fp8_join_kernel(const PrefillParams p, int ctas) {
  pdl_wait();
  pdl_launch_dependents();
  const int c = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int4 item = p.ws_item[c * 2 + 1];
  if (item.x < 0) return;
  const int r = blockIdx.y * 8 + warp, rr = r & 127;
  const int tl = rr / p.G, g = rr - tl * p.G;
  const Seq q = get_seq(p, item.x);
  const int group = p.Hq / p.Hkv, tok = item.z + (r >> 7) * p.tok_per_tile + tl;
  if (tl >= p.tok_per_tile || tok >= q.q_len || item.y % group + g >= group) return;
  auto same = [&](int4 o) { return o.x == item.x && o.y == item.y && o.z == item.z; };
  auto row_of = [&](int i) { return (static_cast<long long>(c + i) * 2 + (i == 0 ? 1 : 0)) * PAIR_ROWS + r; };
  float m = M_NONE, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i = 0; c + i < ctas; ++i) {
    if (i > 0 && !same(p.ws_item[(c + i) * 2])) break;
    const long long row = row_of(i);
    const float mi = p.ws_ml[row * 2], li = p.ws_ml[row * 2 + 1];
    const float4 v = lane * 4 < D ? *reinterpret_cast<const float4*>(p.ws_o + row * D + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    const float mx = fmaxf(m, mi), a = ex2(m - mx), b = ex2(mi - mx);
    m = mx;
    l = l * a + li * b;
    acc.x = acc.x * a + v.x * b; acc.y = acc.y * a + v.y * b; acc.z = acc.z * a + v.z * b; acc.w = acc.w * a + v.w * b;
  }
  if (lane * 4 >= D) return;
  const bool sees_keys = (p.causal ? min(q.k_len, tok + q.shift + 1) : q.k_len) > 0;
  const float inv = sees_keys ? 1.0f / l : 0.f;
  __nv_bfloat16* dst = p.o + static_cast<long long>(q.q_beg + tok) * p.o_tok + (item.y + g) * p.o_head + lane * 4;
  const float f[4] = {acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv};
  if (p.o_vec) {
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) dst[i] = __float2bfloat16(f[i]);
  }
}

template <int D>
int launch_prefill(const PrefillParams& p, int grid, cudaStream_t stream) {
  static bool ready[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -10;
  if (!ready[dev]) {
    if (cudaFuncSetAttribute(attention_prefill_fp8_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::SMEM) != cudaSuccess)
      return -10;
    ready[dev] = true;
  }
  if (cs_launch_pdl(attention_prefill_fp8_kernel<D>, dim3(grid), dim3(THREADS), Shape<D>::SMEM, stream, p) != cudaSuccess) return -10;
  if (grid == 1) return 1;
  return cs_launch_pdl(attention_prefill_fp8_join_kernel<D>, dim3(grid, PAIR_ROWS / 8), dim3(256), 0, stream, p, grid) == cudaSuccess ? 2 : -10;
}

// CTAs of a call: no more than runs of the least length that the queries and tables could make up.
int prefill_ctas(long long Tq, long long B, int Hq, int Hkv, long long bt_width) {
  const int group = Hq / Hkv, G = group < 128 ? group : 128, pair = 2 * (128 / G);
  const long long items = (Tq / pair + B) * Hkv * ((group + G - 1) / G);
  const long long most = (items * (bt_width * KV8_PAGE + pair + ITEM_COST)) / MIN_RUN;
  const int sms = cs_num_sms();
  return most >= sms ? sms : (most < 1 ? 1 : static_cast<int>(most));
}

}  // namespace

// Scratch of a call.
CS_API long long cs_attention_prefill_fp8_ws_bytes(long long Tq, long long B, int Hq, int Hkv, int d, long long bt_width) {
  if (Hkv <= 0 || Hq <= 0) return 0;
  return prefill_ctas(Tq, B, Hq, Hkv, bt_width) * 2LL * (PAIR_ROWS * (d + 2LL) * 4 + 16);
}

// q: [Tq, Hq, d] with contiguous heads, tokens q_tok elements apart and on 16-byte boundaries; o: [Tq, Hq, d] with token and
// head strides in elements; d is 64 or 128.  ws: cs_attention_prefill_fp8_ws_bytes of scratch that no call on another stream
// uses.  Returns how many kernels were launched, or a negative error.
CS_API int cs_attention_prefill_fp8(const void* q, long long q_tok, const void* cache, long long num_pages, void* o, long long o_tok,
                                    long long o_head, const void* cu_q, const void* kv_len, const void* block_table, long long bt_stride,
                                    int bt_width, int B, int Tq, int Hq, int Hkv, int d, float scale, int causal, void* ws,
                                    long long ws_bytes, void* stream) {
  if (B <= 0 || Tq <= 0) return 0;
  if ((d != 64 && d != 128) || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || num_pages <= 0 || num_pages > 0x7fffffffLL || bt_width < 0 ||
      bt_width > KV8_MAX_PAGES)
    return -1;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_tok & 7)) return -1;
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < cs_attention_prefill_fp8_ws_bytes(Tq, B, Hq, Hkv, d, bt_width))
    return -5;
  PrefillParams p{};
  p.q = (const __nv_bfloat16*)q; p.q_tok = q_tok;
  p.o = (__nv_bfloat16*)o; p.o_tok = o_tok; p.o_head = o_head;
  p.o_vec = (reinterpret_cast<uintptr_t>(o) & 15) == 0 && (o_tok & 7) == 0 && (o_head & 7) == 0;
  p.cache = (const uint8_t*)cache; p.num_pages = static_cast<int>(num_pages);
  p.block_table = (const int*)block_table; p.bt_stride = bt_stride; p.bt_width = bt_width;
  p.kv_len = (const int*)kv_len; p.cu_q = (const int*)cu_q;
  const int group = Hq / Hkv;
  p.B = B; p.Tq = Tq; p.Hq = Hq; p.Hkv = Hkv; p.G = group < 128 ? group : 128; p.causal = causal;
  p.blocks = Hkv * ((group + p.G - 1) / p.G);
  p.tok_per_tile = 128 / p.G;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = cs_error_word();
  p.idesc_s = umma_idesc_f16(128, 128, 0, 0);
  p.idesc_pv = umma_idesc_f16(128, d, 0, 1);
  const int ctas = prefill_ctas(Tq, B, Hq, Hkv, bt_width);
  p.ws_item = reinterpret_cast<int4*>(ws);
  p.ws_o = reinterpret_cast<float*>(p.ws_item + ctas * 2);
  p.ws_ml = p.ws_o + ctas * 2LL * PAIR_ROWS * d;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return d == 128 ? launch_prefill<128>(p, ctas, st) : launch_prefill<64>(p, ctas, st);
}
