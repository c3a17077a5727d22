// The 4-bit paged cache as the kernels see it (format: include/b200kv_kv4.h).
#pragma once

#include "b200kv_kv4.h"
#include "common.cuh"

namespace b200kv {
namespace kv4 {

constexpr int kHeadDim = 128;
constexpr int kPageTok = 16;
constexpr int kRowBytes = kHeadDim / 2;                 // codes of one token of one head
constexpr int kScaleOffset = kPageTok * kRowBytes;      // 1024
constexpr int kScaleBytes = 8;                          // four fp16 scales per token and head
constexpr int kBlockBytes = kScaleOffset + kPageTok * kScaleBytes;
static_assert(kBlockBytes == B200KV_KV4_BLOCK_BYTES, "one page of one head");

// Byte offset, inside a block, of the 16-byte chunk j (elements 32 g + 8 j + n for every g and n) of
// token row t.  The XOR spreads the chunks that one shared-memory access of the attention kernels
// touches over all banks; the blocks are copied there as they are.
__host__ __device__ __forceinline__ int chunk_offset(int t, int j) {
  return t * kRowBytes + ((j ^ ((t >> 1) & 3)) << 4);
}

#ifdef __CUDACC__
// The eight codes of a word as four fp16 pairs (elements 2i, 2i+1) of code - 8, exact.  A nibble k
// under the exponent of 1024 reads as 1024 + k (low nibble of a byte) or 1024 + 16 k (high nibble), so
// one logical operation and one packed add or multiply-add give two elements.
__device__ __forceinline__ uint32_t lop_and_or(uint32_t a, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;\n" : "=r"(d) : "r"(a), "r"(mask), "r"(bits));
  return d;
}
__device__ __forceinline__ uint32_t h2_sub(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("sub.rn.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_fma(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.f16x2 %0, %1, %2, %3;\n" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
__device__ __forceinline__ uint32_t h2_mul(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ void unpack_word(uint32_t w, uint32_t (&pair)[4]) {
  constexpr uint32_t kLow = 0x000F000Fu, kHigh = 0x00F000F0u, kExp = 0x64006400u;   // 1024 in both halves
  constexpr uint32_t k1032 = 0x64086408u;      // 1024 + 8
  constexpr uint32_t kSixteenth = 0x2C002C00u; // 1 / 16
  constexpr uint32_t kMinus72 = 0xD480D480u;   // -(64 + 8)
  const uint32_t w8 = w >> 8;
  pair[0] = h2_sub(lop_and_or(w, kLow, kExp), k1032);
  pair[1] = h2_fma(lop_and_or(w, kHigh, kExp), kSixteenth, kMinus72);
  pair[2] = h2_sub(lop_and_or(w8, kLow, kExp), k1032);
  pair[3] = h2_fma(lop_and_or(w8, kHigh, kExp), kSixteenth, kMinus72);
}

// Position of page `page` of row `row` in the pool.
__device__ __forceinline__ const uint8_t* block_at(const uint8_t* pool, int64_t page, int64_t page_stride, int row) {
  return pool + page * page_stride + static_cast<int64_t>(row) * kBlockBytes;
}
#endif

}  // namespace kv4
}  // namespace b200kv
