// Attention of packed queries over the 8-bit paged key-value cache (layout in kv_fp8.cuh):
//
//   o_i = sum_j 2^(s_ij - m_i) vs_j vc_j / sum_j 2^(s_ij - m_i),   s_ij = scale * log2(e) * ks_j * (q_i . kc_j)
//
// over the keys j that query i sees (all, or those up to its own position), with the codes kc, vc and the scales ks, vs
// of the cache.  One warp per (token, query head), all arithmetic in fp32.
#include <math.h>

#include "kv_fp8.cuh"

namespace {

struct PagedParams {
  const __nv_bfloat16* q; long long q_tok, q_head;   // strides in elements
  __nv_bfloat16* o; long long o_tok, o_head;
  const uint8_t* cache; long long num_pages;
  const int* block_table; long long bt_stride; int bt_width;
  const int* kv_len;
  const int* cu_q;
  int B, Tq, Hq, Hkv, causal;
  float scale_log2;
  int* err;
};

template <int D>
__global__ void __launch_bounds__(128) attention_paged_fp8_kernel(const PagedParams p) {
  constexpr int PER = D / 32;   // channels per lane in the value product
  __shared__ float sq[4][D];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long item = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (item >= static_cast<long long>(p.Tq) * p.Hq) return;
  const int t = static_cast<int>(item / p.Hq), h = static_cast<int>(item % p.Hq), hk = h / (p.Hq / p.Hkv);
  if (t >= p.cu_q[p.B]) return;   // a row behind the last sequence
  int lo = 0, hi = p.B;           // the sequence with cu_q[lo] <= t < cu_q[lo + 1]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (p.cu_q[mid] <= t) lo = mid; else hi = mid;
  }
  const int seq = lo;
  int k_len = p.kv_len[seq];
  if (k_len > p.bt_width * KV8_PAGE) {
    if (lane == 0) cs_set_error(p.err, CS_ERR_BAD_ARG);
    k_len = p.bt_width * KV8_PAGE;
  }
  const int shift = p.kv_len[seq] - (p.cu_q[seq + 1] - p.cu_q[seq]);
  const int lim = p.causal ? min(k_len, t - p.cu_q[seq] + shift + 1) : k_len;
  const __nv_bfloat16* q = p.q + t * p.q_tok + h * p.q_head;
  for (int i = lane; i < D; i += 32) sq[warp][i] = __bfloat162float(q[i]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) acc[i] = 0.f;
  for (int base = 0; base < lim; base += 32) {
    const int j = base + lane;
    long long page = p.block_table[seq * p.bt_stride + (base / KV8_PAGE)];
    if (page < 0 || page >= p.num_pages) {
      if (lane == 0) cs_set_error(p.err, CS_ERR_BAD_ARG);
      page = 0;
    }
    const uint8_t* kb = p.cache + (page * 2 * p.Hkv + hk) * kv8_block_bytes(D);
    const uint8_t* vb = p.cache + ((page * 2 + 1) * p.Hkv + hk) * kv8_block_bytes(D);
    float s = -INFINITY;
    if (j < lim) {
      const int r = j % KV8_PAGE;
      float dot = 0.f;
      for (int i = 0; i < D; i += 4) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(kb + r * D + i);
        const uint32_t x = e4m3x2_to_half2(w & 0xffffu), y = e4m3x2_to_half2(w >> 16);
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x)), g = __half22float2(*reinterpret_cast<const __half2*>(&y));
        dot += f.x * sq[warp][i] + f.y * sq[warp][i + 1] + g.x * sq[warp][i + 2] + g.y * sq[warp][i + 3];
      }
      s = dot * reinterpret_cast<const float*>(kb + KV8_PAGE * D)[r] * p.scale_log2;
    }
    float mx = s;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    const float m_new = fmaxf(m, mx), m_use = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = exp2f(m - m_use), e = exp2f(s - m_use);
    m = m_new;
    l = l * alpha + e;
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] *= alpha;
    const int n = min(32, lim - base), r0 = base % KV8_PAGE;
    for (int jj = 0; jj < n; ++jj) {
      const float w = __shfl_sync(0xffffffffu, e, jj) * reinterpret_cast<const float*>(vb + KV8_PAGE * D)[r0 + jj];
#pragma unroll
      for (int i = 0; i < PER; i += 2) {
        const uint32_t x = e4m3x2_to_half2(*reinterpret_cast<const uint16_t*>(vb + (r0 + jj) * D + lane * PER + i));
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x));
        acc[i] += w * f.x;
        acc[i + 1] += w * f.y;
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  __nv_bfloat16* out = p.o + t * p.o_tok + h * p.o_head + lane * PER;
#pragma unroll
  for (int i = 0; i < PER; ++i) out[i] = __float2bfloat16(acc[i] * inv);
}

}  // namespace

// q, o: [Tq, Hq, d] with token and head strides in elements (channels contiguous); d is 64 or 128.
CS_API int cs_attention_paged_fp8(const void* q, long long q_tok, long long q_head, const void* cache, long long num_pages, void* o,
                                  long long o_tok, long long o_head, const void* cu_q, const void* kv_len, const void* block_table,
                                  long long bt_stride, int bt_width, int B, int Tq, int Hq, int Hkv, int d, float scale, int causal,
                                  void* stream) {
  if (B <= 0 || Tq <= 0) return 0;
  if ((d != 64 && d != 128) || Hkv <= 0 || Hq % Hkv != 0) return -1;
  PagedParams p{};
  p.q = (const __nv_bfloat16*)q; p.q_tok = q_tok; p.q_head = q_head;
  p.o = (__nv_bfloat16*)o; p.o_tok = o_tok; p.o_head = o_head;
  p.cache = (const uint8_t*)cache; p.num_pages = num_pages;
  p.block_table = (const int*)block_table; p.bt_stride = bt_stride; p.bt_width = bt_width;
  p.kv_len = (const int*)kv_len; p.cu_q = (const int*)cu_q;
  p.B = B; p.Tq = Tq; p.Hq = Hq; p.Hkv = Hkv; p.causal = causal;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.err = cs_error_word();
  const long long blocks = (static_cast<long long>(Tq) * Hq + 3) / 4;
  if (blocks > 0x7fffffffLL) return -1;
  cudaError_t e;
  if (d == 128) e = cs_launch_pdl(attention_paged_fp8_kernel<128>, dim3((unsigned)blocks), dim3(128), 0, (cudaStream_t)stream, p);
  else e = cs_launch_pdl(attention_paged_fp8_kernel<64>, dim3((unsigned)blocks), dim3(128), 0, (cudaStream_t)stream, p);
  return e == cudaSuccess ? 0 : -10;
}
