// Layout of the 8-bit paged key-value cache, shared by the kernels that fill it and the kernels that read it.
//
// A cache is [pages, 2, Hkv] blocks of 128 * (d + 4) bytes; block (page, kv, head) holds the 128 rows of one page of the
// keys (kv = 0) or values (kv = 1) of one head:
//
//   byte 0        : 128 rows of d e4m3 codes
//   byte 128 * d  : 128 fp32 scales; row r stands for  code[r][:] * scale[r]
//
// A row and its scale travel with the page (pages are what executors copy from one cache to another), a block is one run
// of bytes, and both parts of it start on a 512-byte boundary relative to the cache.  The scale is per token and head:
// it needs no calibration, and a token with large keys costs no other token any precision.
#pragma once
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"

constexpr int KV8_PAGE = 128;
constexpr int KV8_MAX_PAGES = (1 << 24) - 16;   // of a sequence: positions, and a little more, fit 31 bits

__host__ __device__ __forceinline__ constexpr long long kv8_block_bytes(int d) { return static_cast<long long>(KV8_PAGE) * (d + 4); }

// Four e4m3 codes as fp16 numbers (every finite code is exact in fp16): the lower two and the upper two.
__device__ __forceinline__ void e4m3x4_to_half2x2(uint32_t codes, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(codes));
}
