// Append of keys and values to the 8-bit paged cache (layout in kv_fp8.cuh), with the query and key heads normalised
// (optionally) and rotated on the way.  Per token t:
//
//   q head : y = rope(norm(x))                      -> bf16 [T, Hq, d]
//   k head : y = rope(norm(x)), s = amax|y| / 448   -> e4m3(y / s) and s in the row `slot[t]` of the cache
//   v head : y = x,             s = amax|y| / 448   -> the same
//
// norm(x) = x * rsqrt(mean(x^2) + eps) * w; rope rotates the channel pairs (i, i + d/2) by the angle whose cosine and
// sine are cs[t].  All of it is fp32; nothing is rounded between the norm, the rotation and the quantisation, so a query
// is rounded once and a cache row twice less than through bf16.  amax is at least 2^-40, so a scale is never zero; a row
// that holds an infinity or NaN gets the scale NaN, which spreads into every score or output that reads the row.
//
// Bound by its bytes: 18944 tokens of 28 query and 4 key heads (d = 128), 339 MB, take 61.3 us = 5.5 TB/s, 0.85 of what a copy
// reaches; most of a warp's time is the wait for its row.  Blocks of 128 threads, 12 to an SM (40 registers): 256 threads 70 us,
// 64 threads 90, 512 threads 87, 16 blocks of 128 65.  Several rows of a token to a team, so that they share cos and sin: 72 to
// 78 us against 71 for one, when blocks had 256 threads.  One token takes 1.9 us.
#include "kv_fp8.cuh"

namespace {

constexpr int APPEND_THREADS = 128;

struct AppendParams {
  const __nv_bfloat16* qkv; long long ld;
  const float* cs;                        // [T, 2, d/2]
  const __nv_bfloat16* q_norm; const __nv_bfloat16* k_norm;   // [d] or null
  const int* slot;                        // [T]
  __nv_bfloat16* q_out;                   // [T, Hq, d]
  uint8_t* cache;
  unsigned rows;                          // T * (Hq + 2 Hkv)
  long long num_slots;                    // pages * 128
  int Hq, Hkv;
  float eps;
  int* err;
};

// A team of D/16 lanes owns one head row: lane c holds channels [8c, 8c+8) of the lower and of the upper half, so that
// both members of every rotated pair are in one thread and all accesses are 8 or 16 bytes wide.
template <int D>
__global__ void __launch_bounds__(APPEND_THREADS, 12) rope_kv_write_fp8_kernel(const AppendParams p) {
  constexpr int LANES = D / 16, HALF = D / 2;
  pdl_wait();
  pdl_launch_dependents();
  const unsigned row = blockIdx.x * (APPEND_THREADS / LANES) + threadIdx.x / LANES;
  const int c = threadIdx.x % LANES;
  const unsigned team = (LANES == 8 ? 0xffu : 0xfu) << ((threadIdx.x & 31) / LANES * LANES);
  if (row >= p.rows) return;
  const unsigned heads = p.Hq + 2 * p.Hkv;
  const long long t = row / heads;              // (32 bits: a 64-bit division is a third of this kernel's instructions)
  const int h = static_cast<int>(row - static_cast<unsigned>(t) * heads);
  long long slot = 0;
  if (h >= p.Hq) {
    slot = p.slot[t];
    if (slot < 0) return;
    if (slot >= p.num_slots) {   // a bad slot must not touch memory
      if (c == 0) cs_set_error(p.err, CS_ERR_BAD_ARG);
      return;
    }
  }
  const __nv_bfloat16* src = p.qkv + t * p.ld + static_cast<long long>(h) * D + c * 8;
  const uint4 va = *reinterpret_cast<const uint4*>(src), vb = *reinterpret_cast<const uint4*>(src + HALF);
  float a[8], b[8];
  {
    const uint32_t wa[4] = {va.x, va.y, va.z, va.w}, wb[4] = {vb.x, vb.y, vb.z, vb.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      a[2 * i] = bf16lo(wa[i]); a[2 * i + 1] = bf16hi(wa[i]);
      b[2 * i] = bf16lo(wb[i]); b[2 * i + 1] = bf16hi(wb[i]);
    }
  }
  if (h < p.Hq + p.Hkv) {
    const __nv_bfloat16* w = h < p.Hq ? p.q_norm : p.k_norm;
    if (w != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += a[i] * a[i] + b[i] * b[i];
#pragma unroll
      for (int o = LANES / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(team, ss, o);
      const float inv = rsqrtf(ss * (1.0f / D) + p.eps);
      const uint4 ua = *reinterpret_cast<const uint4*>(w + c * 8), ub = *reinterpret_cast<const uint4*>(w + HALF + c * 8);
      const uint32_t wa[4] = {ua.x, ua.y, ua.z, ua.w}, wb[4] = {ub.x, ub.y, ub.z, ub.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        a[2 * i] *= inv * bf16lo(wa[i]); a[2 * i + 1] *= inv * bf16hi(wa[i]);
        b[2 * i] *= inv * bf16lo(wb[i]); b[2 * i + 1] *= inv * bf16hi(wb[i]);
      }
    }
    const float4* cosp = reinterpret_cast<const float4*>(p.cs + t * D + c * 8);
    const float4* sinp = reinterpret_cast<const float4*>(p.cs + t * D + HALF + c * 8);
    const float4 c0 = cosp[0], c1 = cosp[1], s0 = sinp[0], s1 = sinp[1];
    const float cv[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
    const float sv[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = a[i], y = b[i];
      a[i] = x * cv[i] - y * sv[i];
      b[i] = y * cv[i] + x * sv[i];
    }
  }
  if (h < p.Hq) {
    __nv_bfloat16* dst = p.q_out + (t * p.Hq + h) * D + c * 8;
    *reinterpret_cast<uint4*>(dst) = make_uint4(pack_bf16x2(a[0], a[1]), pack_bf16x2(a[2], a[3]), pack_bf16x2(a[4], a[5]), pack_bf16x2(a[6], a[7]));
    *reinterpret_cast<uint4*>(dst + HALF) = make_uint4(pack_bf16x2(b[0], b[1]), pack_bf16x2(b[2], b[3]), pack_bf16x2(b[4], b[5]), pack_bf16x2(b[6], b[7]));
    return;
  }
  // largest magnitude of the row as an integer maximum of the sign-less bits: an infinity or NaN in the row stays visible
  unsigned mx = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) mx = max(mx, max(__float_as_uint(a[i]) & 0x7fffffffu, __float_as_uint(b[i]) & 0x7fffffffu));
#pragma unroll
  for (int o = LANES / 2; o > 0; o >>= 1) mx = max(mx, __shfl_xor_sync(team, mx, o));
  const bool finite = mx < 0x7f800000u;
  const float scale = fmaxf(__uint_as_float(mx), 9.094947017729282e-13f) * (1.0f / 448.0f);   // 2^-40
  const float inv = 1.0f / scale;
  uint32_t code[4];   // lower half: words 0, 1; upper half: words 2, 3
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float* y = i < 2 ? a + i * 4 : b + (i - 2) * 4;
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(y[0] * inv, y[1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(y[2] * inv, y[3] * inv), __NV_SATFINITE, __NV_E4M3);
    code[i] = finite ? (lo | (hi << 16)) : 0u;
  }
  const int kv = h < p.Hq + p.Hkv ? 0 : 1;
  const int hh = kv == 0 ? h - p.Hq : h - p.Hq - p.Hkv;
  uint8_t* block = p.cache + (((slot / KV8_PAGE) * 2 + kv) * p.Hkv + hh) * kv8_block_bytes(D);
  const int r = static_cast<int>(slot % KV8_PAGE);
  uint8_t* dst = block + r * D + c * 8;
  *reinterpret_cast<uint2*>(dst) = make_uint2(code[0], code[1]);
  *reinterpret_cast<uint2*>(dst + HALF) = make_uint2(code[2], code[3]);
  if (c == 0) reinterpret_cast<float*>(block + KV8_PAGE * D)[r] = finite ? scale : __uint_as_float(0x7fffffffu);
}

}  // namespace

// qkv: [T, (Hq + 2 Hkv) * d] with row stride ld (a multiple of 8, 16-byte aligned rows); q_out: [T, Hq, d] contiguous.
// q_norm / k_norm: both null, or two weights [d].  slot[t] = page * 128 + row, negative = the token is not cached; two
// tokens with one slot leave a mix of their rows in it (decode graphs park padding rows on the scratch page).
CS_API int cs_rope_kv_write_fp8(const void* qkv, long long ld, int T, int Hq, int Hkv, int d, const void* cs, const void* q_norm,
                                const void* k_norm, float eps, const void* slot, void* q_out, void* cache, long long num_pages,
                                void* stream) {
  if (T <= 0) return 0;
  if ((d != 64 && d != 128) || Hq <= 0 || Hkv <= 0 || (ld & 7) || (q_norm == nullptr) != (k_norm == nullptr)) return -1;
  AppendParams p{};
  p.qkv = (const __nv_bfloat16*)qkv; p.ld = ld;
  p.cs = (const float*)cs;
  p.q_norm = (const __nv_bfloat16*)q_norm; p.k_norm = (const __nv_bfloat16*)k_norm;
  p.slot = (const int*)slot;
  p.q_out = (__nv_bfloat16*)q_out;
  p.cache = (uint8_t*)cache;
  const long long rows = static_cast<long long>(T) * (Hq + 2 * Hkv);
  if (rows > 0x7fffffffLL) return -1;
  p.rows = static_cast<unsigned>(rows);
  p.num_slots = num_pages * KV8_PAGE;
  p.Hq = Hq; p.Hkv = Hkv; p.eps = eps;
  p.err = cs_error_word();
  const int rows_per_block = APPEND_THREADS / (d / 16);
  const long long blocks = (rows + rows_per_block - 1) / rows_per_block;
  cudaError_t e;
  if (d == 128) e = cs_launch_pdl(rope_kv_write_fp8_kernel<128>, dim3((unsigned)blocks), dim3(APPEND_THREADS), 0, (cudaStream_t)stream, p);
  else e = cs_launch_pdl(rope_kv_write_fp8_kernel<64>, dim3((unsigned)blocks), dim3(APPEND_THREADS), 0, (cudaStream_t)stream, p);
  return e == cudaSuccess ? 0 : -10;
}
