// Writers of the 4-bit paged cache, and the read-back of its rows.
//
// Append: the K and V rows of a token, as they are or straight from the projections (per-head RMSNorm
// and rotary embedding on the way, as in qk_prologue.cu), quantised in groups of 32 elements and
// scattered by slot_mapping.  With x the fp16 values of a group:
//   s = min(fp16(max |x| / 7), 9352),   code = clamp(floor(x / s + 1/2), -8, 7) + 8.
// K is rounded to fp16 after the rotation, as the fp16 pool would hold it, so a cache filled through
// this launch and one filled from an fp16 pool's rows hold the same codes.
//
// The codes have to be exactly those of the definition, although x / s is evaluated as x * (1 / s):
// x and s have 11-bit significands, so x / s is either exactly a border k + 1/2 or at least 2^-13
// away from it, and the product is off by less than 2^-20; adding 2^-14 before the floor therefore
// puts ties on the upper side and moves nothing else.  max|x| / 7 is at least 2^-15 (relative) away from
// every tie of its rounding to fp16, so the product with the rounded 1/7 rounds the same.  The norm's
// mean square of a K row is summed in 64 bits: a reciprocal root that is one unit off would move
// about one K in 4000 to the neighbouring fp16 number and now and then a code with it.  Q keeps
// 32-bit statistics: its rows are rounded once and nothing is decided by them.
//
// A warp takes kRows (one, or four where there are enough tokens to fill the GPU with them) head rows of
// four neighbouring tokens, eight lanes to a row, the loads in flight before they are used.
// A lane owns 8 elements of the first half of head_dim and the 8 they rotate with, i.e. one 32-bit word
// of codes in each of two groups; the words of lanes l and l ^ 4 make up one 16-byte chunk of the row.
// Four neighbouring tokens of a page are 256 contiguous bytes of codes and one 32-byte sector of scales.
// The arithmetic is kept short, or it and not HBM would bound the launch (3 instructions per element: to 32
// bits, half a packed multiply-add, half a packed directed addition for the floor, shift-add into the word).
// HBM-bound: per token 2 * KH * 256 B read and 2 * KH * 72 B written (+ 2 * QH * 256 B of Q and 256 B of
// cos / sin for the fused form).
#include "kv4.cuh"
#include "launch.h"

namespace b200kv {

namespace {

constexpr int kThreads = 256;
constexpr int kD = kv4::kHeadDim;
constexpr int kHalf = kD / 2;
constexpr int kTokPerWarp = 4;
// CTAs per SM that a grid is capped at; warps stride above it.  The copies balance best in many short CTAs
// (4 / 8 / 32 / unlimited per SM: 124 / 123 / 119 / 122 us for 65 536 tokens appended and read back), the
// fused form, whose warps set up more, in the four that are resident (64.6 / 64.9 / 66.3 / 66.9 us for 8205).
constexpr int kCopyCtas = 32;
constexpr int kPrologueCtas = 4;
constexpr float kMaxScale = 9352.f;   // 7 * 9352 = 65464 is a value fp16 can hold after rounding

struct AppendParams {
  const __half* k;            // kFused: the kv projection's rows (K heads, then V heads)
  const __half* v;
  int64_t k_tok_stride, v_tok_stride;
  const int32_t* slots;
  uint8_t* pool;
  int64_t pool_tokens, page_stride;
  int n_tokens, q_heads, kv_heads;
  int rows_per_token;         // head rows of a token: 2 * kv_heads (+ q_heads)
  int groups;                 // warps a token quad needs: rows_per_token / kRows, rounded up (fused: by kind of row)
  int quads;                  // ceil(n_tokens / 4)
  int step_quad, step_grp;    // (warps in the grid) / and % groups
  int32_t* status;
  // fused form only
  const __half* q;
  __half* q_out;
  int64_t q_tok_stride, q_out_tok_stride;
  const __half* q_weight;     // nullptr: no norm
  const __half* k_weight;
  const __half* cos;
  const __half* sin;
  int64_t cs_tok_stride;
  float eps;
};

__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
// c + a * b of the low (high) halves, the product exact, one rounding to 32 bits.
__device__ __forceinline__ float fma_lo(uint32_t a, uint32_t b, float c) {
  float d;
  asm("{\n\t.reg .b16 al, ah, bl, bh;\n\tmov.b32 {al, ah}, %1;\n\tmov.b32 {bl, bh}, %2;\n\t"
      "fma.rn.f32.f16 %0, al, bl, %3;\n\t}\n" : "=f"(d) : "r"(a), "r"(b), "f"(c));
  return d;
}
__device__ __forceinline__ float fma_hi(uint32_t a, uint32_t b, float c) {
  float d;
  asm("{\n\t.reg .b16 al, ah, bl, bh;\n\tmov.b32 {al, ah}, %1;\n\tmov.b32 {bl, bh}, %2;\n\t"
      "fma.rn.f32.f16 %0, ah, bh, %3;\n\t}\n" : "=f"(d) : "r"(a), "r"(b), "f"(c));
  return d;
}
__device__ __forceinline__ void words(const uint4& u, uint32_t (&w)[4]) {
  w[0] = u.x;
  w[1] = u.y;
  w[2] = u.z;
  w[3] = u.w;
}
// x * rrms rounded to fp16, times the fp16 weight in fp16 (the reference's roundings, qk_prologue.cu).
__device__ __forceinline__ void norm8(uint32_t (&x)[4], float rrms, const uint32_t (&w)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
    x[i] = kv4::h2_mul(pack_half2(f.x * rrms, f.y * rrms), w[i]);
  }
}
__device__ __forceinline__ uint32_t h2_max_nan(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.NaN.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
__device__ __forceinline__ uint32_t h2_abs(uint32_t a) { return a & 0x7fff7fffu; }
__device__ __forceinline__ uint32_t abs_max8(const uint4& h) {
  return h2_max_nan(h2_max_nan(h2_abs(h.x), h2_abs(h.y)), h2_max_nan(h2_abs(h.z), h2_abs(h.w)));
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Floors of eight numbers (1 .. 15), given as pairs, as the nibbles of a word.  Adding 2^23 rounding down leaves a floor in the low bits of
// 0x4B000000; the eight are shifted into place and added up, and the constant parts taken off (all but two
// are shifted out).
__device__ __forceinline__ uint32_t pack_floors(const uint64_t (&t)[4]) {
  uint32_t word = 0u - 0x4B000000u - (0x4B000000u << 4);
  const uint64_t two23 = pack_f32x2(8388608.f, 8388608.f);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float even, odd;
    unpack_f32x2(add_down_f32x2(t[i], two23), even, odd);
    word += __float_as_uint(even) << (4 * i);
    word += __float_as_uint(odd) << (4 * (i + 4));
  }
  return word;
}

// One head row of four tokens, eight lanes each: this lane's 8 + 8 elements (fp16 in ha and hb, 32-bit in a and
// b) are quantised and stored.  Lane `sub` of a row owns the words of groups sub / 4 and 2 + sub / 4; lane
// sub ^ 4 has the others of the same chunk.  Called by whole warps; nothing is stored where slot_ok is
// false.
__device__ __forceinline__ void store_row(const uint4& ha, const uint4& hb, const float (&a)[8], const float (&b)[8],
                                          int sub, bool slot_ok, uint8_t* block, int t) {
  // the largest magnitudes of both groups travel as one pair through the four lanes of a group
  const uint32_t ma = abs_max8(ha), mb = abs_max8(hb);
  uint32_t m = h2_max_nan(__byte_perm(ma, mb, 0x5410), __byte_perm(ma, mb, 0x7632));
  m = h2_max_nan(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = h2_max_nan(m, __shfl_xor_sync(0xffffffffu, m, 2));
  const float2 top = __half22float2(*reinterpret_cast<const __half2*>(&m));
  const bool fine1 = top.x <= 65504.f, fine2 = top.y <= 65504.f;   // false for infinities and NaN
  const __half2 sh = __floats2half2_rn(fminf(top.x * (1.f / 7.f), kMaxScale), fminf(top.y * (1.f / 7.f), kMaxScale));
  const float2 s = __half22float2(sh);
  const float inv1 = s.x > 0.f ? rcp_approx(s.x) : 0.f, inv2 = s.y > 0.f ? rcp_approx(s.y) : 0.f;
  const uint64_t inv11 = pack_f32x2(inv1, inv1), inv22 = pack_f32x2(inv2, inv2);
  const uint64_t half = pack_f32x2(8.5f + 1.f / 16384.f, 8.5f + 1.f / 16384.f);
  uint64_t t1[4], t2[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    t1[i] = fma_f32x2(pack_f32x2(a[2 * i], a[2 * i + 1]), inv11, half);
    t2[i] = fma_f32x2(pack_f32x2(b[2 * i], b[2 * i + 1]), inv22, half);
  }
  // floor(x / s + 8.5) is 1 .. 15 when s is a normal number (|x| / s <= 7 (1 + 2^-11)); only a subnormal s,
  // rounded coarsely, can be exceeded by more, and then the sum is limited first.
  if (__any_sync(0xffffffffu, fminf(s.x, s.y) < 6.104e-5f)) {
    auto limit = [](uint64_t& t) {
      float lo, hi;
      unpack_f32x2(t, lo, hi);
      t = pack_f32x2(fminf(fmaxf(lo, 0.f), 15.5f), fminf(fmaxf(hi, 0.f), 15.5f));
    };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      limit(t1[i]);
      limit(t2[i]);
    }
  }
  const uint32_t w1 = fine1 ? pack_floors(t1) : 0x88888888u, w2 = fine2 ? pack_floors(t2) : 0x88888888u;
  uint32_t sc = *reinterpret_cast<const uint32_t*>(&sh);   // a scale of NaN is never read as a number
  if (!fine1) sc = (sc & 0xffff0000u) | 0x7E00u;
  if (!fine2) sc = (sc & 0xffffu) | 0x7E000000u;
  const uint32_t pw1 = __shfl_xor_sync(0xffffffffu, w1, 4), pw2 = __shfl_xor_sync(0xffffffffu, w2, 4);
  const uint32_t ps = __shfl_xor_sync(0xffffffffu, sc, 4);
  if (slot_ok && sub < 4) {
    *reinterpret_cast<uint4*>(block + kv4::chunk_offset(t, sub)) = make_uint4(w1, pw1, w2, pw2);
    if (sub == 0)
      *reinterpret_cast<uint2*>(block + kv4::kScaleOffset + t * kv4::kScaleBytes) =
          make_uint2(__byte_perm(sc, ps, 0x5410), __byte_perm(sc, ps, 0x7632));
  }
}

// Four CTAs per SM, whose 64 registers four rows just fit into (65 536 tokens of 8 K and 8 V heads appended and read
// back: 72 registers and three CTAs 118.3 us, 64 and four 113.3, 48 and five, with spills, 130).  The append alone
// 59.4 us = 5786 GB/s, 0.88 of a plain copy's rate; a step's 33 tokens 1.5 us, a launch's latency.
template <int kRows>
__global__ void __launch_bounds__(kThreads, 4) kv4_append_kernel(AppendParams p) {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int lane = threadIdx.x & 31;
  const int sub = lane & 7;
  const unsigned warp = (blockIdx.x * kThreads + threadIdx.x) >> 5;
  int quad = static_cast<int>(warp / static_cast<unsigned>(p.groups));
  int grp = static_cast<int>(warp % static_cast<unsigned>(p.groups));
  while (quad < p.quads) {
    const int64_t tok = static_cast<int64_t>(quad) * kTokPerWarp + (lane >> 3);
    const bool live = tok < p.n_tokens;
    const int row0 = grp * kRows;
    const int64_t src_tok = live ? tok : p.n_tokens - 1;   // lanes past the last token load it again and store nothing
    uint4 ua[kRows], ub[kRows];
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      const int row = row0 + i;   // K heads, then V heads
      if (row < p.rows_per_token) {
        const __half* src = (row >= p.kv_heads ? p.v + src_tok * p.v_tok_stride + (row - p.kv_heads) * kD
                                               : p.k + src_tok * p.k_tok_stride + row * kD) + sub * 8;
        ua[i] = __ldg(reinterpret_cast<const uint4*>(src));
        ub[i] = __ldg(reinterpret_cast<const uint4*>(src + kHalf));
      }
    }
    const int64_t slot = live ? __ldg(p.slots + src_tok) : -1;
    const bool slot_ok = slot >= 0 && slot < p.pool_tokens;
    if (live && !slot_ok && sub == 0) set_status(p.status, B200KV_DEV_BAD_SLOT);
    const int t = static_cast<int>(slot & (kv4::kPageTok - 1));
    uint8_t* page = p.pool + (slot_ok ? slot / kv4::kPageTok : 0) * p.page_stride;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if (row0 + i >= p.rows_per_token) break;
      float a[8], b[8];
      unpack8(ua[i], a);
      unpack8(ub[i], b);
      store_row(ua[i], ub[i], a, b, sub, slot_ok, page + (row0 + i) * kv4::kBlockBytes, t);
    }
    quad += p.step_quad;
    grp += p.step_grp;
    if (grp >= p.groups) {
      grp -= p.groups;
      ++quad;
    }
  }
}

// The fused form.  A warp's rows are all Q, all K or all V heads of its four tokens (a row kind has a body
// of its own and the loops are not unrolled: the kernel has to stay inside the instruction cache), and
// the next row is on its way while one is worked on.  8205 tokens, 64 Q and 8 + 8 KV heads: 54.0 us = 5819 GB/s, issue
// slots 68 % busy (64-bit sums and exact reciprocal roots of K, 16-bit roundings of the norm); four tokens 2.4 us.
template <int kRows>
__global__ void __launch_bounds__(kThreads, kPrologueCtas) kv4_prologue_kernel(AppendParams p) {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int lane = threadIdx.x & 31;
  const int sub = lane & 7;
  const unsigned warp = (blockIdx.x * kThreads + threadIdx.x) >> 5;
  int quad = static_cast<int>(warp / static_cast<unsigned>(p.groups));
  int grp = static_cast<int>(warp % static_cast<unsigned>(p.groups));
  const int q_groups = (p.q_heads + kRows - 1) / kRows, kv_groups = (p.kv_heads + kRows - 1) / kRows;
  while (quad < p.quads) {
    const int64_t tok = static_cast<int64_t>(quad) * kTokPerWarp + (lane >> 3);
    const bool live = tok < p.n_tokens;
    const bool is_q = grp < q_groups;
    const bool is_v = grp >= q_groups + kv_groups;
    const int row0 = (is_q ? grp : is_v ? grp - q_groups - kv_groups : grp - q_groups) * kRows;   // head of its kind
    const int rows = min(kRows, (is_q ? p.q_heads : p.kv_heads) - row0);
    const __half* src = (is_q ? p.q + tok * p.q_tok_stride : (is_v ? p.v + tok * p.v_tok_stride : p.k + tok * p.k_tok_stride)) +
                        row0 * kD + sub * 8;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    uint4 na = zero, nb = zero;
    if (live) {
      na = __ldg(reinterpret_cast<const uint4*>(src));
      nb = __ldg(reinterpret_cast<const uint4*>(src + kHalf));
    }
    auto next_row = [&](int i, uint4& ha, uint4& hb) {   // hands row i out and requests row i + 1
      ha = na;
      hb = nb;
      if (live && i + 1 < rows) {
        src += kD;
        na = __ldg(reinterpret_cast<const uint4*>(src));
        nb = __ldg(reinterpret_cast<const uint4*>(src + kHalf));
      }
    };
    int64_t slot = -1;
    if (live && !is_q) slot = __ldg(p.slots + tok);
    const bool slot_ok = slot >= 0 && slot < p.pool_tokens;
    if (live && !is_q && !slot_ok && sub == 0) set_status(p.status, B200KV_DEV_BAD_SLOT);
    const int t = static_cast<int>(slot & (kv4::kPageTok - 1));
    uint8_t* block = p.pool + (slot_ok ? slot / kv4::kPageTok : 0) * p.page_stride +
                     ((is_v ? p.kv_heads : 0) + row0) * kv4::kBlockBytes;
    if (is_v) {
#pragma unroll 1
      for (int i = 0; i < rows; ++i, block += kv4::kBlockBytes) {
        uint4 ha, hb;
        next_row(i, ha, hb);
        float a[8], b[8];
        unpack8(ha, a);
        unpack8(hb, b);
        store_row(ha, hb, a, b, sub, slot_ok, block, t);
      }
    } else {
      uint32_t c[4], sn[4], neg[4];   // cos, sin and -sin of the token, for all of the warp's rows
      {
        uint4 uc = zero, us = zero;
        if (live) {
          uc = __ldg(reinterpret_cast<const uint4*>(p.cos + tok * p.cs_tok_stride + sub * 8));
          us = __ldg(reinterpret_cast<const uint4*>(p.sin + tok * p.cs_tok_stride + sub * 8));
        }
        words(uc, c);
        words(us, sn);
#pragma unroll
        for (int i = 0; i < 4; ++i) neg[i] = sn[i] ^ 0x80008000u;
      }
      const __half* weight = is_q ? p.q_weight : p.k_weight;
      uint32_t wa[4] = {}, wb[4] = {};
      if (weight != nullptr) {
        words(__ldg(reinterpret_cast<const uint4*>(weight + sub * 8)), wa);
        words(__ldg(reinterpret_cast<const uint4*>(weight + kHalf + sub * 8)), wb);
      }
      // Products of fp16 numbers are exact in 32 bits, so each rotated element is rounded once there and
      // once to fp16.
      auto rotate = [&](const uint32_t (&a)[4], const uint32_t (&b)[4], uint4& ha, uint4& hb) {
        uint32_t x[4], y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[i] = pack_half2(fma_lo(a[i], c[i], fma_lo(b[i], neg[i], 0.f)), fma_hi(a[i], c[i], fma_hi(b[i], neg[i], 0.f)));
          y[i] = pack_half2(fma_lo(b[i], c[i], fma_lo(a[i], sn[i], 0.f)), fma_hi(b[i], c[i], fma_hi(a[i], sn[i], 0.f)));
        }
        ha = make_uint4(x[0], x[1], x[2], x[3]);
        hb = make_uint4(y[0], y[1], y[2], y[3]);
      };
      if (is_q) {
        __half* dst = p.q_out + tok * p.q_out_tok_stride + row0 * kD + sub * 8;
#pragma unroll 1
        for (int i = 0; i < rows; ++i, dst += kD) {
          uint4 ha, hb;
          next_row(i, ha, hb);
          uint32_t a[4], b[4];
          words(ha, a);
          words(hb, b);
          if (weight != nullptr) {
            float s0 = 0.f, s1 = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              s0 = fma_lo(a[e], a[e], fma_lo(b[e], b[e], s0));
              s1 = fma_hi(a[e], a[e], fma_hi(b[e], b[e], s1));
            }
            float ss = s0 + s1;
#pragma unroll
            for (int m = 1; m < 8; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            const float rrms = rsqrtf(ss * (1.f / kD) + p.eps);
            norm8(a, rrms, wa);
            norm8(b, rrms, wb);
          }
          rotate(a, b, ha, hb);
          if (live) {
            *reinterpret_cast<uint4*>(dst) = ha;
            *reinterpret_cast<uint4*>(dst + kHalf) = hb;
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < rows; ++i, block += kv4::kBlockBytes) {
          uint4 ha, hb;
          next_row(i, ha, hb);
          uint32_t a[4], b[4];
          words(ha, a);
          words(hb, b);
          if (weight != nullptr) {
            double ss = 0.;
#pragma unroll
            for (int e = 0; e < 4; ++e)
              ss += (static_cast<double>(fma_lo(a[e], a[e], 0.f)) + static_cast<double>(fma_hi(a[e], a[e], 0.f))) +
                    (static_cast<double>(fma_lo(b[e], b[e], 0.f)) + static_cast<double>(fma_hi(b[e], b[e], 0.f)));
#pragma unroll
            for (int m = 1; m < 8; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            const float rrms = __fdiv_rn(1.f, __fsqrt_rn(static_cast<float>(ss * (1. / kD)) + p.eps));
            norm8(a, rrms, wa);
            norm8(b, rrms, wb);
          }
          rotate(a, b, ha, hb);
          float x[8], y[8];
          unpack8(ha, x);
          unpack8(hb, y);
          store_row(ha, hb, x, y, sub, slot_ok, block, t);
        }
      }
    }
    quad += p.step_quad;
    grp += p.step_grp;
    if (grp >= p.groups) {
      grp -= p.groups;
      ++quad;
    }
  }
}

// Read-back: four lanes to a row, a lane reads one 16-byte chunk (8 elements in each of the four
// groups) and the row's four scales and writes four 16-byte pieces; the four lanes of a row write 64
// contiguous bytes per store.  A warp takes kRows head rows of eight neighbouring tokens, all loads in
// flight first.  HBM-bound: per token 2 * KH * (72 + 256) B; 65 536 tokens of 8 + 8 heads 55.4 us = 6210 GB/s, 0.95 of
// a plain copy's rate.
struct GatherParams {
  const uint8_t* pool;
  int64_t pool_tokens, page_stride;
  const int32_t* slots;
  __half* out;
  int64_t out_tok_stride;
  int n, rows;
  int octets, groups, step_octet, step_grp;
  int32_t* status;
};

template <int kRows>
__global__ void __launch_bounds__(kThreads) kv4_gather_kernel(GatherParams p) {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
  const int lane = threadIdx.x & 31;
  const int j = lane & 3;
  const unsigned warp = (blockIdx.x * kThreads + threadIdx.x) >> 5;
  int octet = static_cast<int>(warp / static_cast<unsigned>(p.groups));
  int grp = static_cast<int>(warp % static_cast<unsigned>(p.groups));
  while (octet < p.octets) {
    const int64_t tok = static_cast<int64_t>(octet) * 8 + (lane >> 2);
    if (tok < p.n) {
      const int row0 = grp * kRows;
      const int64_t slot = __ldg(p.slots + tok);
      const bool ok = slot >= 0 && slot < p.pool_tokens;
      if (!ok && j == 0) set_status(p.status, B200KV_DEV_BAD_SLOT);
      const int t = static_cast<int>(slot & (kv4::kPageTok - 1));
      const uint8_t* block = kv4::block_at(p.pool, ok ? slot / kv4::kPageTok : 0, p.page_stride, row0);
      uint4 codes[kRows];
      uint2 scales[kRows];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        codes[i] = make_uint4(0x88888888u, 0x88888888u, 0x88888888u, 0x88888888u);
        scales[i] = make_uint2(0, 0);
        if (ok && row0 + i < p.rows) {
          codes[i] = *reinterpret_cast<const uint4*>(block + i * kv4::kBlockBytes + kv4::chunk_offset(t, j));
          scales[i] = *reinterpret_cast<const uint2*>(block + i * kv4::kBlockBytes + kv4::kScaleOffset + t * kv4::kScaleBytes);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        if (row0 + i < p.rows) {
          const uint32_t w[4] = {codes[i].x, codes[i].y, codes[i].z, codes[i].w};
          const uint32_t s2[4] = {__byte_perm(scales[i].x, 0, 0x1010), __byte_perm(scales[i].x, 0, 0x3232),
                                  __byte_perm(scales[i].y, 0, 0x1010), __byte_perm(scales[i].y, 0, 0x3232)};
          __half* dst = p.out + tok * p.out_tok_stride + (row0 + i) * kD + 8 * j;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t v[4];
            kv4::unpack_word(w[g], v);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = kv4::h2_mul(v[e], s2[g]);
            *reinterpret_cast<uint4*>(dst + 32 * g) = make_uint4(v[0], v[1], v[2], v[3]);
          }
        }
      }
    }
    octet += p.step_octet;
    grp += p.step_grp;
    if (grp >= p.groups) {
      grp -= p.groups;
      ++octet;
    }
  }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Grid of one warp per work item, at most `per_sm` CTAs of 256 threads per SM (grid-stride above).
int grid_for(int64_t items, int per_sm, unsigned* blocks) {
  const int sms = device_sm_count();
  if (sms <= 0) return B200KV_ECUDA;
  int64_t b = (items + kThreads / 32 - 1) / (kThreads / 32);
  const int64_t cap = static_cast<int64_t>(sms) * per_sm;
  if (b > cap) b = cap;
  *blocks = static_cast<unsigned>(b);
  return B200KV_OK;
}

template <typename Kernel, typename Params>
int launch(Kernel kernel, const Params& p, unsigned blocks, cudaStream_t stream) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

// Rows per warp: four when that still gives every SM this many warps, one otherwise.  One / four rows, us, 64/8
// heads: append of 32 tokens 1.6 / 2.7, 4096 5.8 / 6.1, 32 768 38.2 / 36.4; read-back of 32 1.6 / 2.5, 32 768
// 28.8 / 28.4; fused append of 256 3.7 / 5.2, 1024 9.2 / 9.4, 8192 64.1 / 54.0.
constexpr int kWarpsForFour = 16;
inline bool four_rows(int64_t token_groups, int rows, int sms) {
  return token_groups * ((rows + 3) / 4) >= static_cast<int64_t>(sms) * kWarpsForFour;
}

template <bool kFused, int kRows>
int launch_append_rows(AppendParams p, cudaStream_t stream) {
  p.groups = kFused ? (p.q_heads + kRows - 1) / kRows + 2 * ((p.kv_heads + kRows - 1) / kRows)
                    : (p.rows_per_token + kRows - 1) / kRows;
  unsigned blocks = 0;
  const int rc = grid_for(static_cast<int64_t>(p.quads) * p.groups, kFused ? kPrologueCtas : kCopyCtas, &blocks);
  if (rc != B200KV_OK) return rc;
  const int64_t warps = static_cast<int64_t>(blocks) * (kThreads / 32);
  p.step_quad = static_cast<int>(warps / p.groups);
  p.step_grp = static_cast<int>(warps % p.groups);
  if (kFused) return launch(kv4_prologue_kernel<kRows>, p, blocks, stream);
  return launch(kv4_append_kernel<kRows>, p, blocks, stream);
}

template <bool kFused>
int launch_append(AppendParams p, cudaStream_t stream) {
  const int sms = device_sm_count();
  if (sms <= 0) return B200KV_ECUDA;
  p.rows_per_token = 2 * p.kv_heads + (kFused ? p.q_heads : 0);
  p.quads = (p.n_tokens + kTokPerWarp - 1) / kTokPerWarp;
  return four_rows(p.quads, p.rows_per_token, sms) ? launch_append_rows<kFused, 4>(p, stream)
                                                   : launch_append_rows<kFused, 1>(p, stream);
}

template <int kRows>
int launch_gather(GatherParams p, cudaStream_t stream) {
  p.groups = (p.rows + kRows - 1) / kRows;
  unsigned blocks = 0;
  const int rc = grid_for(static_cast<int64_t>(p.octets) * p.groups, kCopyCtas, &blocks);
  if (rc != B200KV_OK) return rc;
  const int64_t warps = static_cast<int64_t>(blocks) * (kThreads / 32);
  p.step_octet = static_cast<int>(warps / p.groups);
  p.step_grp = static_cast<int>(warps % p.groups);
  return launch(kv4_gather_kernel<kRows>, p, blocks, stream);
}

}  // namespace

int kv4_check_pool(const void* pool, int64_t pool_pages, int64_t page_stride_bytes, int kv_heads) {
  if (!pool || pool_pages <= 0 || kv_heads <= 0) return B200KV_EINVAL;
  if (pool_pages > (int64_t{1} << 27)) return B200KV_ETOOLARGE;   // slots are int32
  if (kv_heads > 1024) return B200KV_ETOOLARGE;
  if (!aligned16(pool) || page_stride_bytes % 16 != 0) return B200KV_EALIGN;
  if (page_stride_bytes > (int64_t{1} << 31) - 16) return B200KV_ETOOLARGE;   // kernels multiply 32 x 32 bits
  if (page_stride_bytes < static_cast<int64_t>(2) * kv_heads * kv4::kBlockBytes) return B200KV_EINVAL;
  return B200KV_OK;
}

int kv4_append(const Kv4AppendArgs& a, cudaStream_t stream) {
  if (a.n_tokens < 0 || a.kv_heads <= 0) return B200KV_EINVAL;
  if (a.head_dim != kD) return B200KV_EUNSUPPORTED;
  if (a.n_tokens == 0) return B200KV_OK;
  if (a.n_tokens > (1 << 30)) return B200KV_ETOOLARGE;
  if (!a.k || !a.v || !a.slots) return B200KV_EINVAL;
  int rc = kv4_check_pool(a.pool, a.pool_pages, a.page_stride_bytes, a.kv_heads);
  if (rc != B200KV_OK) return rc;
  if (a.k_tok_stride % 8 || a.v_tok_stride % 8 || !aligned16(a.k) || !aligned16(a.v)) return B200KV_EALIGN;
  const int64_t half = static_cast<int64_t>(a.kv_heads) * kD;
  if (a.k_tok_stride < half || a.v_tok_stride < half) return B200KV_EINVAL;
  AppendParams p{};
  p.k = static_cast<const __half*>(a.k);
  p.v = static_cast<const __half*>(a.v);
  p.k_tok_stride = a.k_tok_stride;
  p.v_tok_stride = a.v_tok_stride;
  p.slots = a.slots;
  p.pool = static_cast<uint8_t*>(a.pool);
  p.pool_tokens = a.pool_pages * kv4::kPageTok;
  p.page_stride = a.page_stride_bytes;
  p.n_tokens = static_cast<int>(a.n_tokens);
  p.kv_heads = a.kv_heads;
  p.status = a.status;
  if (a.q == nullptr) return launch_append<false>(p, stream);

  if (!a.q_out || !a.cos || !a.sin || a.q_heads <= 0 || !(a.eps >= 0.f)) return B200KV_EINVAL;
  if (a.q_heads > 65536) return B200KV_ETOOLARGE;
  if (a.q_tok_stride % 8 || a.q_out_tok_stride % 8 || a.cs_tok_stride % 8) return B200KV_EALIGN;
  if (!aligned16(a.q) || !aligned16(a.q_out) || !aligned16(a.cos) || !aligned16(a.sin) ||
      (a.q_weight && !aligned16(a.q_weight)) || (a.k_weight && !aligned16(a.k_weight)))
    return B200KV_EALIGN;
  if (a.q_tok_stride < static_cast<int64_t>(a.q_heads) * kD || a.q_out_tok_stride < static_cast<int64_t>(a.q_heads) * kD ||
      a.cs_tok_stride < kHalf)
    return B200KV_EINVAL;
  p.q = static_cast<const __half*>(a.q);
  p.q_out = static_cast<__half*>(a.q_out);
  p.q_tok_stride = a.q_tok_stride;
  p.q_out_tok_stride = a.q_out_tok_stride;
  p.q_heads = a.q_heads;
  p.q_weight = static_cast<const __half*>(a.q_weight);
  p.k_weight = static_cast<const __half*>(a.k_weight);
  p.cos = static_cast<const __half*>(a.cos);
  p.sin = static_cast<const __half*>(a.sin);
  p.cs_tok_stride = a.cs_tok_stride;
  p.eps = a.eps;
  return launch_append<true>(p, stream);
}

int kv4_gather(const void* pool, int64_t pool_pages, int64_t page_stride_bytes, const int32_t* slots, int64_t n,
               void* out, int64_t out_tok_stride, int kv_heads, int head_dim, int32_t* status, cudaStream_t stream) {
  if (n < 0 || kv_heads <= 0) return B200KV_EINVAL;
  if (head_dim != kD) return B200KV_EUNSUPPORTED;
  if (n == 0) return B200KV_OK;
  if (n > (1 << 30)) return B200KV_ETOOLARGE;
  if (!slots || !out) return B200KV_EINVAL;
  int rc = kv4_check_pool(pool, pool_pages, page_stride_bytes, kv_heads);
  if (rc != B200KV_OK) return rc;
  if (!aligned16(out) || out_tok_stride % 8 != 0) return B200KV_EALIGN;
  if (out_tok_stride < static_cast<int64_t>(2) * kv_heads * kD) return B200KV_EINVAL;
  GatherParams p{};
  p.pool = static_cast<const uint8_t*>(pool);
  p.pool_tokens = pool_pages * kv4::kPageTok;
  p.page_stride = page_stride_bytes;
  p.slots = slots;
  p.out = static_cast<__half*>(out);
  p.out_tok_stride = out_tok_stride;
  p.n = static_cast<int>(n);
  p.rows = 2 * kv_heads;
  p.octets = static_cast<int>((n + 7) / 8);
  p.status = status;
  const int sms = device_sm_count();
  if (sms <= 0) return B200KV_ECUDA;
  return four_rows(p.octets, p.rows, sms) ? launch_gather<4>(p, stream) : launch_gather<1>(p, stream);
}

}  // namespace b200kv
