// Decode attention over the 8-bit paged key-value cache (layout in kv_fp8.cuh): one new token per sequence, grouped heads.
//
//   o = sum_j w_j vc_j / sum_j 2^(s_j - M),   w_j = 2^(s_j + log2 vs_j - M),   s_j = scale * log2(e) * ks_j * (q . kc_j)
//
// kc, vc are the e4m3 codes and ks, vs the scales of key j.  Codes are exact in fp16, so the two products run on fp16
// fragments: the query is scaled by a power of two per head (exact for every element within 2^-38 of the largest), and M
// follows the maximum of s_j + log2 vs_j, the weight that the second product sees, so that a weight is never too large
// for fp16 whatever the value scales are.  The normaliser needs no vs: it takes its own exponential, in fp32.
//
// The kernel is bound by the cache's bytes, and everything is arranged around reading them once, without a pause:
//
//   * Work is counted in units of 64 keys of one (sequence, key head); the list of all units of the batch is cut into
//     equal runs, one per CTA, on the device from kv_len.  So any mix of lengths loads every SM alike (a captured graph
//     adapts to the lengths of each replay), and a single long sequence is spread over the whole GPU.  A CTA has at most
//     two items that it does not own alone, the first and the last of its run: these leave partial sums in a workspace
//     and a second small kernel joins them in the order of the CTAs (no atomics, the result does not depend on timing).
//   * One producer warp keeps a ring of stages full by TMA (K and V codes through a tensor map with a swizzle, scales by
//     plain bulk copies).
//   * Eight consumer warps: warp w takes keys 16 (w % 4) .. + 15 of every second unit, entirely in registers: S^T = K Q^T
//     and O^T += V^T P with mma.m16n8k16, keys (channels) on the 16 side and up to 8 query heads per n tile on the other.
//     mma.sync and not tcgen05 on purpose: e4m3 becomes fp16 on the way from shared memory to a register fragment, while
//     a tcgen05 operand would have to be written back to shared memory twice as wide; tensor time is not what is scarce
//     at 8 to 16 heads per byte of K.  The warps share nothing until an item ends; then their sums meet in shared memory.
#include <math.h>

#include "kv_fp8.cuh"

int cs_encode_tmap_3d_u8(CUtensorMap* out, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1_bytes,
                         uint64_t s2_bytes, uint32_t b0, uint32_t b1, uint32_t b2, int swizzle_bytes);

namespace {

constexpr int UNIT = 64;                     // keys per unit of work
constexpr int CONSUMERS = 8;                 // warps
constexpr int DEC_THREADS = (CONSUMERS + 1) * 32;
constexpr int MAX_CTAS = 512;
constexpr float M_NONE = -3.0e38f;           // running maximum before the first key (finite: differences stay defined)

// Shared memory of one instantiation.
template <int D, int NT>
struct DecShape {
  static constexpr int HEADS = 8 * NT;
  static constexpr int TILE = UNIT * D;                      // bytes of codes of K (or V) per stage
  static constexpr int JOIN_LD = D + 4;                      // floats between two heads of a warp's partial sum
  static constexpr int JOIN = CONSUMERS * HEADS * JOIN_LD * 4;
  static constexpr int STAGE = 2 * TILE + 2 * UNIT * 4;
  static constexpr int FIT = (227 * 1024 - 2048 - 2 * CONSUMERS * HEADS * 4 - JOIN) / STAGE;
  static constexpr int STAGES = FIT < 16 ? FIT : 16;
  static constexpr int SMEM = 1024 + STAGES * STAGE + JOIN;
};

struct DecParams {
  const __nv_bfloat16* q; long long q_tok, q_head;     // strides in elements, rows on 16-byte boundaries
  __nv_bfloat16* o; long long o_tok, o_head; int o_vec; // o_vec: 8-byte stores are aligned
  const uint8_t* cache; int num_pages;
  const int* block_table; long long bt_stride; int bt_width;
  const int* kv_len;
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
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
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
__device__ __forceinline__ uint32_t pack_half2(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Keys of sequence b that can be read (a length beyond the table is cut and reported), and its units.
__device__ __forceinline__ int dec_len(const DecParams& p, int b) {
  const int n = p.kv_len[b];
  const long long cap = static_cast<long long>(p.bt_width) * KV8_PAGE;
  return n < 0 ? 0 : (n > cap ? static_cast<int>(cap) : n);
}
__device__ __forceinline__ int dec_units(const DecParams& p, int b) { return (dec_len(p, b) + UNIT - 1) / UNIT; }

// One visit of a CTA to an item: units [u, u + n) of `units` of sequence `seq`, head block `head` (of Hkv * head_blocks).
// Every role of the CTA walks the same list of visits.
struct Walk {
  int seq, head, units, len, u, n;
  long long left;   // units of the CTA's run not yet handed out, this visit included
  __device__ __forceinline__ bool settle(const DecParams& p) {   // on to a sequence with keys
    for (; seq < p.B; ++seq) {
      len = dec_len(p, seq);
      units = (len + UNIT - 1) / UNIT;
      if (u < units) {
        n = static_cast<int>(min(static_cast<long long>(units - u), left));
        return true;
      }
    }
    return false;
  }
  __device__ __forceinline__ bool next(const DecParams& p) {
    left -= n;
    if (left <= 0) return false;
    u = 0;
    if (++head == p.Hkv * p.head_blocks) { head = 0; ++seq; return settle(p); }
    n = static_cast<int>(min(static_cast<long long>(units), left));
    return true;
  }
};

template <int D, int NT>
__global__ void __launch_bounds__(DEC_THREADS, 1)
attention_decode_fp8_kernel(const __grid_constant__ CUtensorMap tm, const DecParams p) {
  using Shape = DecShape<D, NT>;
  constexpr int HEADS = Shape::HEADS, STAGES = Shape::STAGES, TILE = Shape::TILE, JOIN_LD = Shape::JOIN_LD;
  constexpr int KSTEPS = D / 16, MT = D / 16, VPER = D / 8;   // VPER: channels of a value row per thread

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* s_codes = smem;                                              // STAGES x (K tile, V tile)
  float* s_scale = reinterpret_cast<float*>(smem + STAGES * 2 * TILE);  // STAGES x (64 key scales, 64 value scales)
  float* s_join = s_scale + STAGES * 2 * UNIT;                          // [warp][head][JOIN_LD]
  __shared__ uint64_t full[STAGES], empty[STAGES];
  __shared__ float s_m[CONSUMERS][HEADS], s_l[CONSUMERS][HEADS];
  __shared__ int abort_flag, s_start_seq;
  __shared__ long long s_warp_sum[CONSUMERS + 1], s_start_off;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    abort_flag = 0;
    s_start_seq = 0;
    s_start_off = 0;
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], CONSUMERS / 2); }
    mbar_fence_init();
    tma_prefetch_desc(&tm);
  }
  // the lengths, the queries and the cache rows of this step come from the kernels ahead in the stream
  pdl_wait();
  pdl_launch_dependents();

  // ------------------------------- this CTA's run of units -------------------------------
  const int heads = p.Hkv * p.head_blocks;
  long long mine = 0;
  for (int b = threadIdx.x; b < p.B; b += DEC_THREADS) mine += dec_units(p, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
  if (lane == 0) s_warp_sum[warp] = mine;
  __syncthreads();
  long long total = 0;
#pragma unroll
  for (int w = 0; w <= CONSUMERS; ++w) total += s_warp_sum[w];
  total *= heads;
  // no CTA of the first `active` is without a unit, so the CTAs that share an item are consecutive
  const long long active = min(total, static_cast<long long>(gridDim.x));
  long long r0 = 0, r1 = 0;
  if (blockIdx.x < active) { r0 = total * blockIdx.x / active; r1 = total * (blockIdx.x + 1) / active; }
  long long before = 0;   // units (all heads) of the sequences ahead of this chunk
  for (int base = 0; base < p.B && r1 > r0; base += DEC_THREADS) {
    __syncthreads();
    const int b = base + threadIdx.x;
    const long long units = b < p.B ? static_cast<long long>(dec_units(p, b)) * heads : 0;
    long long incl = units;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_warp_sum[warp] = incl;
    __syncthreads();
    for (int w = 0; w < warp; ++w) incl += s_warp_sum[w];
    incl += before;
    if (r0 < incl && r0 >= incl - units) { s_start_seq = b; s_start_off = r0 - (incl - units); }
    for (int w = 0; w <= CONSUMERS; ++w) before += s_warp_sum[w];
    if (before > r0) break;
  }
  __syncthreads();
  volatile int* abortp = &abort_flag;
  Walk wk{};
  wk.seq = s_start_seq;
  wk.left = r1 - r0;
  const int start_units = max(1, dec_units(p, wk.seq));
  wk.head = static_cast<int>(s_start_off / start_units);
  wk.u = static_cast<int>(s_start_off - static_cast<long long>(wk.head) * start_units);
  const bool any = r1 > r0 && wk.settle(p);
  if (threadIdx.x == 0) p.ws_item[blockIdx.x * 2] = p.ws_item[blockIdx.x * 2 + 1] = -1;

  if (warp == CONSUMERS) {
    // ------------------------------- producer -------------------------------
    if (any) {
      uint32_t n = 0;
      bool ok = true;
      do {
        const int hk = wk.head / p.head_blocks;
        const int* table = p.block_table + wk.seq * p.bt_stride;
        int page_lane = 0, page_base = -64;   // the 32 table entries held by the lanes start at page_base
        for (int u = wk.u; u < wk.u + wk.n && ok; ++u, ++n) {
          const int blk = u / (KV8_PAGE / UNIT), half = u % (KV8_PAGE / UNIT);
          if (blk >= page_base + 32 || page_base < 0) {
            page_base = blk;
            page_lane = blk + lane < (wk.len + KV8_PAGE - 1) / KV8_PAGE ? table[blk + lane] : 0;
          }
          int page = __shfl_sync(0xffffffffu, page_lane, blk - page_base);
          if (lane == 0) {
            if (page < 0 || page >= p.num_pages) { cs_set_error(p.err, CS_ERR_BAD_ARG); page = 0; }
            const uint32_t s = n % STAGES;
            if (mbar_wait(&empty[s], ((n / STAGES) & 1) ^ 1, abortp, p.err, CS_ERR_TIMEOUT_SLOT)) {
              const int block = (page * 2) * p.Hkv + hk;
              uint8_t* codes = s_codes + s * 2 * TILE;
              float* scale = s_scale + s * 2 * UNIT;
              const uint8_t* src = p.cache + block * kv8_block_bytes(D) + KV8_PAGE * D + half * UNIT * 4;
              mbar_arrive_expect_tx(&full[s], 2 * TILE + 2 * UNIT * 4);
              tma_load_3d(codes, &tm, 0, half * UNIT, block, &full[s]);
              bulk_load(smem_u32(scale), src, UNIT * 4, &full[s]);
              tma_load_3d(codes + TILE, &tm, 0, half * UNIT, block + p.Hkv, &full[s]);
              bulk_load(smem_u32(scale + UNIT), src + p.Hkv * kv8_block_bytes(D), UNIT * 4, &full[s]);
            } else {
              ok = false;
            }
          }
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
      } while (ok && wk.next(p));
    }
  } else {
    // ------------------------------- consumers -------------------------------
    const int g = lane >> 2, t = lane & 3;
    const int kw = (warp & 3) * 16, team = warp >> 2;
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
    const uint32_t codes0 = smem_u32(s_codes), scale0 = smem_u32(s_scale);
    const uint32_t k_off = at(key0, t);                                             // chunks t and (D = 128) t + 4: ^ 64
    const uint32_t v_off_a = TILE + (D == 128 ? at(va, g) : at(va, g >> 1) + (g & 1) * 8);
    const uint32_t v_off_b = TILE + (D == 128 ? at(vb, g) : at(vb, g >> 1) + (g & 1) * 8);

    uint32_t n = 0;   // running unit of this CTA
    if (any) do {
      const int hk = wk.head / p.head_blocks, hb = wk.head - hk * p.head_blocks;
      const int h0 = hk * p.G + hb * HEADS, n_heads = min(HEADS, p.G - hb * HEADS);
      // queries of this item as B fragments: thread (g, t) holds head g (+ 8), the channels of chunks t (and t + 4)
      uint32_t qf[NT][KSTEPS][2];
      float qs[NT][2];   // scale * log2(e) / power of two of heads 2t and 2t + 1
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + g;
        uint32_t raw[KSTEPS * 2];
        const __nv_bfloat16* src = p.q + wk.seq * p.q_tok + (h0 + h) * p.q_head + t * 16;
#pragma unroll
        for (int c = 0; c < KSTEPS / 4; ++c)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint4 v = h < n_heads ? *reinterpret_cast<const uint4*>(src + c * 64 + half * 8) : make_uint4(0, 0, 0, 0);
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
      float o[NT][MT][4], m[NT][2], l[NT][2];   // m: the reference exponent is m - 6, so weights reach up to 2^14
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        m[nt][0] = m[nt][1] = M_NONE;
        l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int i = 0; i < MT; ++i) o[nt][i][0] = o[nt][i][1] = o[nt][i][2] = o[nt][i][3] = 0.f;
      }

      for (int u = wk.u; u < wk.u + wk.n; ++u, ++n) {
        if ((n & 1) != team) continue;
        const uint32_t s = n % STAGES;
        mbar_wait(&full[s], (n / STAGES) & 1, abortp, p.err, CS_ERR_TIMEOUT_TMA);
        const int valid = wk.len - u * UNIT;   // keys of the unit that exist (may exceed 64)
        if (kw < valid) {
          const uint32_t codes = codes0 + s * 2 * TILE, scale = scale0 + s * 2 * UNIT * 4;
          // ---- S^T = K Q^T for 16 keys
          uint32_t k0[KSTEPS], k1[KSTEPS];   // codes of keys key0 and key0 + 8, four channels per word
#pragma unroll
          for (int c = 0; c < KSTEPS / 4; ++c) {
            const uint4 x = lds128(codes + (k_off ^ (c * 64))), y = lds128(codes + (k_off ^ (c * 64)) + 8 * D);
            k0[c * 4] = x.x; k0[c * 4 + 1] = x.y; k0[c * 4 + 2] = x.z; k0[c * 4 + 3] = x.w;
            k1[c * 4] = y.x; k1[c * 4 + 1] = y.y; k1[c * 4 + 2] = y.z; k1[c * 4 + 3] = y.w;
          }
          const float ks0 = lds32(scale + key0 * 4), ks1 = lds32(scale + (key0 + 8) * 4);
          const float vs0 = lds32(scale + (UNIT + key0) * 4), vs1 = lds32(scale + (UNIT + key0 + 8) * 4);
          float c[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
          for (int i = 0; i < KSTEPS; ++i) {
            const uint32_t a0 = e4m3x2_to_half2(k0[i]), a1 = e4m3x2_to_half2(k1[i]);
            const uint32_t a2 = e4m3x2_to_half2(k0[i] >> 16), a3 = e4m3x2_to_half2(k1[i] >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(c[nt], a0, a1, a2, a3, qf[nt][i][0], qf[nt][i][1]);
          }
          // the value rows of this thread: keys va, vb and those 8 further
          uint32_t x[4][VPER / 4];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const uint32_t addr = codes + ((r & 1) ? v_off_b : v_off_a) + (r >> 1) * 8 * D;
            if constexpr (D == 128) {
              const uint4 v = lds128(addr);
              x[r][0] = v.x; x[r][1] = v.y; x[r][2] = v.z; x[r][3] = v.w;
            } else {
              const uint2 v = lds64(addr);
              x[r][0] = v.x; x[r][1] = v.y;
            }
          }
          const float lv0 = vs0 < 1.2e-38f ? -126.f : __log2f(vs0), lv1 = vs1 < 1.2e-38f ? -126.f : __log2f(vs1);
          float tt[NT][4];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            c[nt][0] *= ks0 * qs[nt][0]; c[nt][1] *= ks0 * qs[nt][1];
            c[nt][2] *= ks1 * qs[nt][0]; c[nt][3] *= ks1 * qs[nt][1];
          }
          if (valid < UNIT) {   // the sequence ends in this unit: what lies behind it may be anything
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              if (key0 >= valid) c[nt][0] = c[nt][1] = -INFINITY;
              if (key0 + 8 >= valid) c[nt][2] = c[nt][3] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (((r & 1) ? vb : va) + (r >> 1) * 8 >= valid) {
#pragma unroll
                for (int j = 0; j < VPER / 4; ++j) x[r][j] = 0u;
              }
          }
          const float w0 = key0 < valid ? lv0 : 0.f, w1 = key0 + 8 < valid ? lv1 : 0.f;
          bool grow = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            tt[nt][0] = c[nt][0] + w0; tt[nt][1] = c[nt][1] + w0;
            tt[nt][2] = c[nt][2] + w1; tt[nt][3] = c[nt][3] + w1;
            grow |= fmaxf(tt[nt][0], tt[nt][2]) > m[nt][0] + 8.f || fmaxf(tt[nt][1], tt[nt][3]) > m[nt][1] + 8.f;
          }
          // The reference moves only when a weight would pass 2^14, which after the first tiles is rare
          if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                float mx = fmaxf(tt[nt][j], tt[nt][2 + j]);
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                mx = fmaxf(mx, m[nt][j]);
                const float alpha = ex2(m[nt][j] - mx);
                m[nt][j] = mx;
                l[nt][j] *= alpha;
#pragma unroll
                for (int i = 0; i < MT; ++i) { o[nt][i][j] *= alpha; o[nt][i][2 + j] *= alpha; }
              }
          }
          uint32_t b0[NT], b1[NT];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const float r0_ = m[nt][0] - 6.f, r1_ = m[nt][1] - 6.f;
            l[nt][0] += ex2(c[nt][0] - r0_) + ex2(c[nt][2] - r0_);
            l[nt][1] += ex2(c[nt][1] - r1_) + ex2(c[nt][3] - r1_);
            b0[nt] = transpose8x8(pack_half2(ex2(tt[nt][0] - r0_), ex2(tt[nt][1] - r1_)));
            b1[nt] = transpose8x8(pack_half2(ex2(tt[nt][2] - r0_), ex2(tt[nt][3] - r1_)));
          }
          // ---- O^T += V^T P: fragment row g of tile i is channel VPER g + 2 i, row g + 8 the next one
#pragma unroll
          for (int i = 0; i < MT; ++i) {
            const uint32_t sel = (i & 1) ? 0x7362u : 0x5140u;
            const uint32_t ab = __byte_perm(x[0][i >> 1], x[1][i >> 1], sel), cd = __byte_perm(x[2][i >> 1], x[3][i >> 1], sel);
            const uint32_t a0 = e4m3x2_to_half2(ab), a1 = e4m3x2_to_half2(ab >> 16);
            const uint32_t a2 = e4m3x2_to_half2(cd), a3 = e4m3x2_to_half2(cd >> 16);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma16816(o[nt][i], a0, a1, a2, a3, b0[nt], b1[nt]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&empty[s]);
      }

      // ---- the warps' sums meet: [warp][head][channel] in shared memory, then warp w finishes head w (and w + 8)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 4);
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 8);
          l[nt][j] += __shfl_xor_sync(0xffffffffu, l[nt][j], 16);
          const int h = nt * 8 + 2 * t + j;
          if (g == 0) { s_m[warp][h] = m[nt][j]; s_l[warp][h] = l[nt][j]; }
          float* dst = s_join + (warp * HEADS + h) * JOIN_LD + g * VPER;
#pragma unroll
          for (int i = 0; i < MT; i += 2)
            *reinterpret_cast<float4*>(dst + 2 * i) = make_float4(o[nt][i][j], o[nt][i][2 + j], o[nt][i + 1][j], o[nt][i + 1][2 + j]);
        }
      asm volatile("bar.sync 1, 256;" ::: "memory");
      const bool whole = wk.u == 0 && wk.n == wk.units;
      const int slot = blockIdx.x * 2 + (wk.u == 0 ? 1 : 0);   // an item that began before the run is its first, one that goes on its last
      const long long part = static_cast<long long>(slot) * HEADS;
      if (!whole && threadIdx.x == 0) p.ws_item[slot] = wk.seq * heads + wk.head;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int h = nt * 8 + warp;
        if (h < n_heads) {
          float mx = M_NONE, sum = 0.f, f[CONSUMERS];
#pragma unroll
          for (int w = 0; w < CONSUMERS; ++w) mx = fmaxf(mx, s_m[w][h]);
#pragma unroll
          for (int w = 0; w < CONSUMERS; ++w) { f[w] = ex2(s_m[w][h] - mx); sum += s_l[w][h] * f[w]; }
          if (lane * 4 < D) {
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < CONSUMERS; ++w) {
              const float4 v = *reinterpret_cast<const float4*>(s_join + (w * HEADS + h) * JOIN_LD + lane * 4);
              acc.x += v.x * f[w]; acc.y += v.y * f[w]; acc.z += v.z * f[w]; acc.w += v.w * f[w];
            }
            if (whole) {
              const float inv = sum == 0.f ? 0.f : 1.0f / sum;
              __nv_bfloat16* dst = p.o + wk.seq * p.o_tok + (h0 + h) * p.o_head + lane * 4;
              const uint2 v = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
              if (p.o_vec) {
                *reinterpret_cast<uint2*>(dst) = v;
              } else {
                unsigned short* d16 = reinterpret_cast<unsigned short*>(dst);
                d16[0] = v.x & 0xffffu; d16[1] = v.x >> 16; d16[2] = v.y & 0xffffu; d16[3] = v.y >> 16;
              }
            } else {
              *reinterpret_cast<float4*>(p.ws_o + (part + h) * D + lane * 4) = acc;
            }
          }
          if (!whole && lane == 0) { p.ws_ml[(part + h) * 2] = mx; p.ws_ml[(part + h) * 2 + 1] = sum; }
        }
      }
      asm volatile("bar.sync 1, 256;" ::: "memory");   // the join area is written again at the end of the next item
    } while (wk.next(p));

    // sequences without keys give zeros; lengths that do not fit the table are reported
    for (int b = blockIdx.x; b < p.B; b += gridDim.x) {
      const int len = p.kv_len[b];
      if (len > static_cast<long long>(p.bt_width) * KV8_PAGE && threadIdx.x == 0) cs_set_error(p.err, CS_ERR_BAD_ARG);
      if (dec_len(p, b) == 0)
        for (int i = threadIdx.x; i < p.Hq * D; i += CONSUMERS * 32) p.o[b * p.o_tok + (i / D) * p.o_head + i % D] = __float2bfloat16(0.f);
    }
  }
}

// Joins the items that several CTAs worked on: CTA c takes the item whose first part is the last of decode CTA c.  One
// warp per head; the parts are read in the order of the CTAs.
template <int D, int NT>
__global__ void __launch_bounds__(256 * NT) attention_decode_fp8_join_kernel(const DecParams p) {
  constexpr int HEADS = 8 * NT;
  pdl_wait();
  pdl_launch_dependents();
  const int item = p.ws_item[blockIdx.x * 2 + 1];
  if (item < 0) return;
  const int h = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int heads = p.Hkv * p.head_blocks, seq = item / heads, head = item - seq * heads;
  const int hk = head / p.head_blocks, hb = head - hk * p.head_blocks;
  if (h >= min(HEADS, p.G - hb * HEADS)) return;
  int end = blockIdx.x + 1;   // the parts are slot 1 of this CTA and slot 0 of those up to `end`
  while (end < gridDim.x) {
    const int c = end + lane;
    const unsigned same = __ballot_sync(0xffffffffu, c < gridDim.x && p.ws_item[c * 2] == item);
    end += __popc(same);     // the CTAs of an item are consecutive
    if (same != 0xffffffffu) break;
  }
  auto part = [&](int c) { return (static_cast<long long>(c) * 2 + (c == blockIdx.x ? 1 : 0)) * HEADS + h; };
  float mx = M_NONE;
  for (int c = blockIdx.x + lane; c < end; c += 32) mx = fmaxf(mx, p.ws_ml[part(c) * 2]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  float sum = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = blockIdx.x; c0 < end; c0 += 32) {
    const int c = c0 + lane;
    float f = 0.f;
    if (c < end) {
      f = ex2(p.ws_ml[part(c) * 2] - mx);
      sum += p.ws_ml[part(c) * 2 + 1] * f;
    }
    const int cnt = min(32, end - c0);
#pragma unroll 8
    for (int i = 0; i < cnt; ++i) {
      const float fi = __shfl_sync(0xffffffffu, f, i);
      if (lane * 4 < D) {
        const float4 v = *reinterpret_cast<const float4*>(p.ws_o + part(c0 + i) * D + lane * 4);
        acc.x += v.x * fi; acc.y += v.y * fi; acc.z += v.z * fi; acc.w += v.w * fi;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane * 4 >= D) return;
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  __nv_bfloat16* dst = p.o + seq * p.o_tok + (hk * p.G + hb * HEADS + h) * p.o_head + lane * 4;
  const uint2 v = make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
  if (p.o_vec) {
    *reinterpret_cast<uint2*>(dst) = v;
  } else {
    unsigned short* d16 = reinterpret_cast<unsigned short*>(dst);
    d16[0] = v.x & 0xffffu; d16[1] = v.x >> 16; d16[2] = v.y & 0xffffu; d16[3] = v.y >> 16;
  }
}

template <int D, int NT>
int launch_decode(const CUtensorMap& tm, const DecParams& p, int ctas, cudaStream_t stream) {
  using Shape = DecShape<D, NT>;
  static bool attr_done[64] = {false};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return -10;
  if (!attr_done[dev]) {
    if (cudaFuncSetAttribute(attention_decode_fp8_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape::SMEM) != cudaSuccess)
      return -10;
    attr_done[dev] = true;
  }
  if (cs_launch_pdl(attention_decode_fp8_kernel<D, NT>, dim3(ctas), dim3(DEC_THREADS), Shape::SMEM, stream, tm, p) != cudaSuccess) return -10;
  return cs_launch_pdl(attention_decode_fp8_join_kernel<D, NT>, dim3(ctas), dim3(256 * NT), 0, stream, p) == cudaSuccess ? 0 : -10;
}

}  // namespace

// Scratch of one call (any sequence count): partial sums, their maxima and normalisers, and the items they belong to.
CS_API long long cs_attention_decode_fp8_ws_bytes(int Hq, int Hkv, int d) {
  if (Hkv <= 0) return 0;
  const int heads = Hq / Hkv <= 8 ? 8 : 16;
  const long long ctas = cs_num_sms() < MAX_CTAS ? cs_num_sms() : MAX_CTAS;
  return ctas * 2 * (heads * (d + 2LL) * 4 + 4);
}

// q, o: [B, Hq, d] with token and head strides in elements; q rows lie on 16-byte boundaries.  One query per sequence,
// which sees all kv_len[b] keys.  ws: cs_attention_decode_fp8_ws_bytes of scratch that no call on another stream uses.
CS_API int cs_attention_decode_fp8(const void* q, long long q_tok, long long q_head, const void* cache, long long num_pages, void* o,
                                   long long o_tok, long long o_head, const void* kv_len, const void* block_table, long long bt_stride,
                                   int bt_width, int B, int Hq, int Hkv, int d, float scale, void* ws, long long ws_bytes, void* stream) {
  if (B <= 0) return 0;
  if ((d != 64 && d != 128) || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || num_pages <= 0 || num_pages * 2 * Hkv > 0x7fffffffLL) return -1;
  if ((reinterpret_cast<uintptr_t>(q) & 15) || (q_tok & 7) || (q_head & 7)) return -1;
  DecParams p{};
  p.q = (const __nv_bfloat16*)q; p.q_tok = q_tok; p.q_head = q_head;
  p.o = (__nv_bfloat16*)o; p.o_tok = o_tok; p.o_head = o_head;
  p.o_vec = (reinterpret_cast<uintptr_t>(o) & 7) == 0 && (o_tok & 3) == 0 && (o_head & 3) == 0;
  p.cache = (const uint8_t*)cache; p.num_pages = static_cast<int>(num_pages);
  p.block_table = (const int*)block_table; p.bt_stride = bt_stride; p.bt_width = bt_width;
  p.kv_len = (const int*)kv_len;
  p.B = B; p.Hq = Hq; p.Hkv = Hkv; p.G = Hq / Hkv;
  const int heads = p.G <= 8 ? 8 : 16;
  p.head_blocks = (p.G + heads - 1) / heads;
  if (static_cast<long long>(B) * Hkv * p.head_blocks > 0x7fffffffLL) return -1;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = cs_error_word();
  if (ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 15) || ws_bytes < cs_attention_decode_fp8_ws_bytes(Hq, Hkv, d)) return -5;
  int ctas = cs_num_sms() < MAX_CTAS ? cs_num_sms() : MAX_CTAS;
  p.ws_o = reinterpret_cast<float*>(ws);
  p.ws_ml = p.ws_o + static_cast<long long>(ctas) * 2 * heads * d;
  p.ws_item = reinterpret_cast<int*>(p.ws_ml + static_cast<long long>(ctas) * 2 * heads * 2);
  // no more CTAs than units that the tables could hold
  const long long most = static_cast<long long>(B) * Hkv * p.head_blocks * bt_width * (KV8_PAGE / UNIT);
  if (most < ctas) ctas = most > 0 ? static_cast<int>(most) : 1;
  CUtensorMap tm;
  if (cs_encode_tmap_3d_u8(&tm, cache, d, KV8_PAGE, static_cast<uint64_t>(num_pages) * 2 * Hkv, d, kv8_block_bytes(d), d, UNIT, 1, d)) return -3;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (d == 128) return heads == 8 ? launch_decode<128, 1>(tm, p, ctas, st) : launch_decode<128, 2>(tm, p, ctas, st);
  return heads == 8 ? launch_decode<64, 1>(tm, p, ctas, st) : launch_decode<64, 2>(tm, p, ctas, st);
}
