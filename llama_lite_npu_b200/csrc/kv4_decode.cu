// Paged flash-decoding over the 4-bit cache (format: include/b200kv_kv4.h), one launch.
//
// The page line, its cut into teams and the merge of the partials are those of paged_decode.cu
// (decode_plan.cuh): a CTA owns one KV head over a contiguous range of pages and serves the head's
// whole query group from one pass over them.  What differs is a warp's work on a page:
//
//   S^T[tok, head] = sum_g s_K[tok, g] * (C_K[tok, d in g] . Q^T[d in g, head])
//   O^T[d, head]  += C_V^T[d, tok] . (P^T[tok, head] * s_V[tok, g(d)])
//
// with C the codes minus 8, integers that fp16 holds exactly.  No element is ever multiplied by its
// scale: K's scales multiply the four partial scores of a token in 32 bits, V's scales go into P,
// where 16 tokens meet 8 heads instead of 128 elements.  A code costs 9/8 of an instruction (one
// logical operation and one packed add per pair, a shift per word) on its way to mma.sync m16n8k16
// (fp16 in, fp32 accumulate; tokens or head_dim are the M rows, the query heads the N columns).
//
// P * s_V is an fp16 operand, so its range matters: P is at most 2^8 (the running maximum is moved only
// when it has grown by more than that) and s_V is multiplied by 2^a with the largest scale seen so far
// below 2^(6 - a), a <= 15; products are at most 2^14 and lose bits only below 2^-14, 2^28 under the
// largest.  A new largest scale rescales O, as a new maximum does.
//
// A warp streams its own pages: page k of a piece belongs to warp k % 4, and every warp keeps a ring of
// kStages pages (K block + V block, 2304 bytes) filled by two bulk copies per page that its lane 0
// issues as soon as the page's ring slot has been read.  No producer warp, no CTA-wide barrier in the
// steady state; the blocks are stored in the order in which the lanes read them (conflict-free 16-byte
// shared loads).  The page table is read 32 entries at a time, one block of entries ahead of use.
// Every wait is an mbarrier wait bounded by ~2 s.
//
// Bytes per token and KV head: 2 * 72 (a page is 2304 B where fp16 has 8192).
#include "common.cuh"
#include "decode_plan.cuh"
#include "kv4.cuh"
#include "launch.h"
#include "tma.h"

namespace b200kv {

namespace {

constexpr int kThreads = kConsumerThreads;
constexpr int kStages = 4;
constexpr int kPageBytes = 2 * kv4::kBlockBytes;   // K and V block of one page of one head
constexpr int kRingBytes = kConsumerWarps * kStages * kPageBytes;
constexpr int kSeqCache = kThreads;                // lengths and table rows kept in shared memory
constexpr int kDefaultPieceCost = 8;
constexpr int kMaxTeams = kConsumerWarps * kD;     // a sequence's weights must fit the merge buffer
static_assert(kPS == kv4::kPageTok && kD == kv4::kHeadDim, "one geometry");

struct Kv4DecodeParams : DecodePlan {
  const __half* q;
  int64_t q_stride_b, q_stride_h;
  const uint8_t* pool;
  int64_t pool_pages, page_stride;
  const int32_t* table;
  int64_t table_row_stride;
  int table_kind;
  float scale_log2;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;\n"
      :
      : "r"(dst), "l"(src), "r"(bytes), "r"(bar), "l"(policy)
      : "memory");
}
__device__ __forceinline__ void bulk_prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" : : "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
// D = A * B (no accumulator input)
__device__ __forceinline__ void mma_16816_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float half_bits_to_float(uint32_t bits) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(bits & 0xffffu)));
}
__device__ __forceinline__ uint32_t h2_max(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A piece: the part of one sequence that lies in the team's range.
struct Piece {
  int b, row, len, np;   // sequence, table row, tokens, pages
  int begin, end;        // pages [begin, end) of the sequence
  int64_t flat;          // position of page `begin` on the page line
  int kseq;              // non-empty sequences before b
  bool valid;
};

// Lengths and table rows of the sequences from `first` on, from shared memory for the first kSeqCache.
struct SeqCache {
  const int* len;
  const int* row;
  int first;
  __device__ __forceinline__ int len_of(const Kv4DecodeParams& p, int b) const {
    return b - first < kSeqCache ? len[b - first] : seq_len_checked(p, b);
  }
  __device__ __forceinline__ int row_of(const Kv4DecodeParams& p, int b) const {
    return b - first < kSeqCache ? row[b - first] : (p.row_ids ? __ldg(p.row_ids + b) : b);
  }
};

__device__ __forceinline__ void enter_piece(const Kv4DecodeParams& p, const SeqCache& seq, int64_t range_end, Piece& pc,
                                            int b, int first_page) {
  pc.b = b;
  pc.len = seq.len_of(p, b);
  pc.row = seq.row_of(p, b);
  pc.np = pages_of(pc.len);
  pc.begin = first_page;
  const int64_t room = range_end - pc.flat;
  pc.end = (pc.np - first_page <= room) ? pc.np : first_page + static_cast<int>(room);
  pc.valid = true;
}
__device__ __forceinline__ void next_piece(const Kv4DecodeParams& p, const SeqCache& seq, int64_t range_end, Piece& pc) {
  pc.flat += pc.end - pc.begin;
  pc.valid = false;
  if (pc.flat >= range_end) return;
  int b = pc.b + 1;
  while (b < p.batch && seq.len_of(p, b) == 0) ++b;
  if (b >= p.batch) return;   // cannot happen for consistent lengths; stop rather than overrun
  ++pc.kseq;
  enter_piece(p, seq, range_end, pc, b, 0);
}
// Pages of a piece that belong to a warp.
__device__ __forceinline__ int warp_pages(const Piece& pc, int warp) {
  return pc.valid ? (pc.end - pc.begin - warp + kConsumerWarps - 1) / kConsumerWarps : 0;
}

// The pages a warp requests, in order, with their table entries: lane l holds the entry of page
// begin + warp + 4 * (32 * block + l) of the piece; the next block of entries (of this piece, or
// the first of the next piece) is already on its way.
struct PageStream {
  Piece pc, nx;
  int m, cnt;            // next page of this warp in pc, and how many it has there
  int32_t ids, ids_next;

  __device__ __forceinline__ int32_t load_ids(const Kv4DecodeParams& p, const Piece& from, int warp, int lane, int first) const {
    const int page = from.begin + warp + kConsumerWarps * (first + lane);
    if (!from.valid || page >= from.end) return 0;
    const int64_t at = p.table_kind == B200KV_TABLE_BLOCK ? page : static_cast<int64_t>(page) * kPS;
    return __ldg(p.table + static_cast<int64_t>(from.row) * p.table_row_stride + at);
  }
  __device__ __forceinline__ void refill(const Kv4DecodeParams& p, const SeqCache& seq, int64_t range_end, int warp, int lane) {
    if (m + 32 < cnt) {
      ids_next = load_ids(p, pc, warp, lane, m + 32);
    } else {
      nx = pc;
      do {
        next_piece(p, seq, range_end, nx);
      } while (nx.valid && warp_pages(nx, warp) <= 0);   // short pieces have no page for the later warps
      ids_next = load_ids(p, nx, warp, lane, 0);
    }
  }
  __device__ __forceinline__ void start(const Kv4DecodeParams& p, const SeqCache& seq, int64_t range_end, const Piece& first,
                                        int warp, int lane) {
    pc = first;
    while (pc.valid && warp_pages(pc, warp) <= 0) next_piece(p, seq, range_end, pc);
    m = 0;
    cnt = warp_pages(pc, warp);
    ids = load_ids(p, pc, warp, lane, 0);
    if (pc.valid) refill(p, seq, range_end, warp, lane);
  }
  __device__ __forceinline__ bool more() const { return pc.valid; }
  __device__ __forceinline__ void advance(const Kv4DecodeParams& p, const SeqCache& seq, int64_t range_end, int warp, int lane) {
    ++m;
    if (m == cnt) {
      pc = nx;
      m = 0;
      cnt = warp_pages(pc, warp);
      ids = ids_next;
      if (pc.valid) refill(p, seq, range_end, warp, lane);
    } else if ((m & 31) == 0) {
      ids = ids_next;
      refill(p, seq, range_end, warp, lane);
    }
  }
};

template <int ROWS>
__global__ void __launch_bounds__(kThreads, ROWS == 8 ? 4 : 3) kv4_decode_kernel(Kv4DecodeParams p) {
  static_assert(ROWS == 8 || ROWS == 16, "query-group heads are padded to 8 or 16");
  constexpr int NB = ROWS / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  float* merge_o = reinterpret_cast<float*>(smem + kRingBytes);            // [4][128][ROWS]
  float* merge_ml = merge_o + kConsumerWarps * kD * ROWS;                  // [4][ROWS][2]
  uint64_t* bars = reinterpret_cast<uint64_t*>(merge_ml + kConsumerWarps * ROWS * 2);   // [4][kStages]
  int* arrival = reinterpret_cast<int*>(bars + kConsumerWarps * kStages);
  int* seq_len_s = arrival + 4;                                            // [kSeqCache]
  int* seq_row_s = seq_len_s + kSeqCache;
  int* scan = reinterpret_cast<int*>(merge_o);

  const int tid = threadIdx.x;
  const int lane = tid & 31;
  const int warp = tid >> 5;
  const int team = blockIdx.x / p.kv_heads;
  const int head = blockIdx.x - team * p.kv_heads;
  const uint32_t ring = smem_u32(smem) + warp * (kStages * kPageBytes);
  const uint32_t bar = smem_u32(bars) + warp * (kStages * 8);
  if (tid == 0) {
    for (int i = 0; i < kConsumerWarps * kStages; ++i) mbar_init(smem_u32(bars) + 8 * i, 1);
    fence_barrier_init();
  }
  const TeamRange range = plan_team_range(p, team, tid, scan);
  if (range.any) {
    const int b = range.start_b + tid;
    seq_len_s[tid] = b < p.batch ? seq_len_checked(p, b) : 0;
    seq_row_s[tid] = b < p.batch ? (p.row_ids ? __ldg(p.row_ids + b) : b) : 0;
  }
  __syncthreads();
  const SeqCache seq{seq_len_s, seq_row_s, range.start_b};
  Piece pc;
  pc.flat = range.begin;
  pc.kseq = range.start_k;
  pc.valid = false;
  PageStream st;
  if (range.any) {
    enter_piece(p, seq, range.end, pc, range.start_b, range.start_page);
    st.start(p, seq, range.end, pc, warp, lane);
  }
  // Raw table entry -> page number; an entry that names no page is reported and page 0 read instead.
  auto page_of = [&](int32_t id) -> int64_t {
    int64_t page = id;
    bool ok = true;
    if (p.table_kind == B200KV_TABLE_TOKEN) {
      ok = (id & (kPS - 1)) == 0;
      page = id >> 4;
    }
    if (!ok || page < 0 || page >= p.pool_pages) {
      set_status(p.status, B200KV_DEV_BAD_PAGE);
      page = 0;
    }
    return page;
  };
  const uint8_t* k_rows = p.pool + static_cast<int64_t>(head) * kv4::kBlockBytes;
  const int64_t v_from_k = static_cast<int64_t>(p.kv_heads) * kv4::kBlockBytes;
  // First pages towards L2 while the previous kernel is still finishing: L2 is the point of coherence,
  // so rows that kernel writes afterwards are still seen by the copies below.
  if (range.any && st.more() && lane < min(st.cnt, kStages)) {
    const uint8_t* src = k_rows + page_of(st.ids) * p.page_stride;
    bulk_prefetch_l2(src, kv4::kBlockBytes);
    bulk_prefetch_l2(src + v_from_k, kv4::kBlockBytes);
  }
  pdl_wait_then_trigger();   // q, the pool, the workspace and out belong to earlier kernels until here
  if (team == 0 && range.any_empty) {
    // No keys: the output rows are defined as zero, and nobody else writes them.
    for (int b = 0; b < p.batch; ++b) {
      if (seq_len_checked(p, b) != 0) continue;
      for (int g = 0; g < p.group; ++g)
        p.out[static_cast<int64_t>(b) * p.out_stride_b +
              (static_cast<int64_t>(head) * p.group + g) * p.out_stride_h + tid] = __float2half_rn(0.f);
    }
  }
  if (!range.any) return;

  const uint64_t policy = l2_evict_first_policy();
  auto request = [&](int stage) {
    const int32_t id = __shfl_sync(0xffffffffu, st.ids, st.m & 31);
    if (lane == 0) {
      const uint8_t* src = k_rows + page_of(id) * p.page_stride;
      const uint32_t dst = ring + stage * kPageBytes;
      mbar_arrive_expect_tx(bar + 8 * stage, kPageBytes);
      bulk_load(dst, src, kv4::kBlockBytes, bar + 8 * stage, policy);
      bulk_load(dst + kv4::kBlockBytes, src + v_from_k, kv4::kBlockBytes, bar + 8 * stage, policy);
    }
    st.advance(p, seq, range.end, warp, lane);
  };
  int pending = 0;             // pages requested and not yet waited for
  for (int s = 0; s < kStages && st.more(); ++s, ++pending) request(s);

  const int r = lane >> 2;     // fragment row: token (S^T) or one of the 8 row pairs of head_dim (O^T); also a head column
  const int jq = lane & 3;     // fragment column pair
  const int jv = r >> 1;       // V: chunk of the token rows that holds this lane's elements ...
  const uint32_t vsel = (r & 1) ? 0x7632u : 0x5410u;   // ... and which half of its words
  const uint32_t k_off = static_cast<uint32_t>(kv4::chunk_offset(r, jq));      // token r; token r + 8 is 512 bytes on
  const uint32_t v_off = static_cast<uint32_t>(kv4::chunk_offset(2 * jq, jv)); // token 2 jq; 2 jq + 1 is 64 bytes on
  bool alive = true;           // false once a wait of this warp ran out: keep walking, stop computing
  unsigned seen_arrivals = 0;
  int stage = 0;
  uint32_t parity = 0;

  while (pc.valid) {
    uint32_t qf[NB][8][2];     // Q^T as B fragments
    float o[8][NB][4];         // O^T * 2^a: 8 M blocks of 16 along head_dim
    float m_run[NB][2], l_run[NB][2];
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int hq = nb * 8 + r;
      const __half* qh = p.q + static_cast<int64_t>(pc.b) * p.q_stride_b +
                         (static_cast<int64_t>(head) * p.group + hq) * p.q_stride_h + 8 * jq;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint4 v = hq < p.group ? __ldg(reinterpret_cast<const uint4*>(qh + 32 * g)) : make_uint4(0, 0, 0, 0);
        qf[nb][2 * g][0] = v.x;
        qf[nb][2 * g][1] = v.y;
        qf[nb][2 * g + 1][0] = v.z;
        qf[nb][2 * g + 1][1] = v.w;
      }
      m_run[nb][0] = m_run[nb][1] = -INFINITY;
      l_run[nb][0] = l_run[nb][1] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) o[j][nb][0] = o[j][nb][1] = o[j][nb][2] = o[j][nb][3] = 0.f;
    int shift = 15;            // a: V scales are multiplied by 2^a
    const bool whole = pc.begin == 0 && pc.end == pc.np;
    const int cnt = warp_pages(pc, warp);

#pragma unroll 1
    for (int m = 0; m < cnt; ++m) {
      if (tid == 0 && m == cnt - 1 && !whole) {
        // How many of the other pieces have arrived already (see emit_piece).
        asm volatile("ld.relaxed.gpu.global.u32 %0, [%1];\n"
                     : "=r"(seen_arrivals)
                     : "l"(p.piece_ctr + static_cast<int64_t>(pc.b) * p.kv_heads + head)
                     : "memory");
      }
      if (alive) {
        if (!mbar_wait_bounded(bar + 8 * stage, parity)) {
          set_status(p.status, B200KV_DEV_WAIT_TIMEOUT);
          alive = false;
          for (int i = 1; i < pending; ++i) {   // what else is in flight lands (or gives up) before the CTA may end
            const int s2 = stage + i < kStages ? stage + i : stage + i - kStages;
            mbar_wait_bounded(bar + 8 * s2, stage + i < kStages ? parity : parity ^ 1);
          }
        }
        --pending;
      }
      if (alive) {
        const int wtok = min(kPS, pc.len - (pc.begin + warp + kConsumerWarps * m) * kPS);   // valid tokens of the page
        const uint32_t kb = ring + stage * kPageBytes;
        const uint32_t vb = kb + kv4::kBlockBytes;
        // ---- S^T = K Q^T ----------------------------------------------------------------------
        float s[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) s[nb][0] = s[nb][1] = s[nb][2] = s[nb][3] = 0.f;
        {
          const uint4 k0 = lds128(kb + k_off), k1 = lds128(kb + k_off + 8 * kv4::kRowBytes);
          const uint2 c0 = lds64(kb + kv4::kScaleOffset + r * kv4::kScaleBytes);
          const uint2 c1 = lds64(kb + kv4::kScaleOffset + (r + 8) * kv4::kScaleBytes);
          const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
          const uint32_t sc0[4] = {c0.x, c0.x >> 16, c0.y, c0.y >> 16}, sc1[4] = {c1.x, c1.x >> 16, c1.y, c1.y >> 16};
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint32_t a[4], b[4];
            kv4::unpack_word(w0[g], a);
            kv4::unpack_word(w1[g], b);
            const float f0 = half_bits_to_float(sc0[g]), f1 = half_bits_to_float(sc1[g]);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
              float d[4];
              mma_16816_first(d, a[0], b[0], a[1], b[1], qf[nb][2 * g][0], qf[nb][2 * g][1]);
              const uint32_t a2[4] = {a[2], b[2], a[3], b[3]};
              mma_16816(d, a2, qf[nb][2 * g + 1][0], qf[nb][2 * g + 1][1]);
              s[nb][0] += f0 * d[0];
              s[nb][1] += f0 * d[1];
              s[nb][2] += f1 * d[2];
              s[nb][3] += f1 * d[3];
            }
          }
        }
        // ---- V scales of tokens 2jq, 2jq+1 | 2jq+8, 2jq+9 as fp16 pairs per group ----------------
        uint32_t sv[4][2];
        {
          const uint4 t0 = lds128(vb + kv4::kScaleOffset + 2 * jq * kv4::kScaleBytes);
          const uint4 t1 = lds128(vb + kv4::kScaleOffset + (2 * jq + 8) * kv4::kScaleBytes);
          sv[0][0] = __byte_perm(t0.x, t0.z, 0x5410);
          sv[1][0] = __byte_perm(t0.x, t0.z, 0x7632);
          sv[2][0] = __byte_perm(t0.y, t0.w, 0x5410);
          sv[3][0] = __byte_perm(t0.y, t0.w, 0x7632);
          sv[0][1] = __byte_perm(t1.x, t1.z, 0x5410);
          sv[1][1] = __byte_perm(t1.x, t1.z, 0x7632);
          sv[2][1] = __byte_perm(t1.y, t1.w, 0x5410);
          sv[3][1] = __byte_perm(t1.y, t1.w, 0x7632);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[nb][i] *= p.scale_log2;
        if (wtok < kPS) {
          // Rows past the length were never written and may hold anything, NaN scales included.
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            if (r >= wtok) s[nb][0] = s[nb][1] = -INFINITY;
            if (r + 8 >= wtok) s[nb][2] = s[nb][3] = -INFINITY;
          }
          const uint32_t keep0 = (2 * jq < wtok ? 0xffffu : 0u) | (2 * jq + 1 < wtok ? 0xffff0000u : 0u);
          const uint32_t keep1 = (2 * jq + 8 < wtok ? 0xffffu : 0u) | (2 * jq + 9 < wtok ? 0xffff0000u : 0u);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            sv[g][0] &= keep0;
            sv[g][1] &= keep1;
          }
        }
        // ---- has a maximum, or the largest V scale, outgrown its reference? ------------------------
        uint32_t sv_max = h2_max(h2_max(sv[0][0], sv[0][1]), h2_max(sv[1][0], sv[1][1]));
        sv_max = h2_max(sv_max, h2_max(h2_max(sv[2][0], sv[2][1]), h2_max(sv[3][0], sv[3][1])));
        const float sv_hi = fmaxf(half_bits_to_float(sv_max), half_bits_to_float(sv_max >> 16));
        const float sv_lim = __int_as_float((127 + 6 - shift) << 23);   // 2^(6 - a)
        bool grow = sv_hi > sv_lim;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) grow |= s[nb][i] > m_run[nb][i & 1] + 8.f;
        if (__any_sync(0xffffffffu, grow)) {
          float hi = sv_hi;
          hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
          hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 2));
          int new_shift = shift;
          if (hi > sv_lim) {   // smallest power of two that is not below the scale: exponent of hi rounded up
            const int e = static_cast<int>((__float_as_uint(hi) + 0x7fffffu) >> 23) - 127;
            new_shift = max(6 - e, -8);
          }
          const float re = __int_as_float((127 + new_shift - shift) << 23);
          shift = new_shift;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float mx = fmaxf(s[nb][h], s[nb][h + 2]);
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
              mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
              const float m_new = fmaxf(m_run[nb][h], mx);
              const float alpha = m_run[nb][h] == -INFINITY ? 0.f : fast_exp2(m_run[nb][h] - m_new);
              m_run[nb][h] = m_new;
              l_run[nb][h] *= alpha;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                o[j][nb][h] *= alpha * re;
                o[j][nb][h + 2] *= alpha * re;
              }
            }
        }
        // ---- P^T -> B fragments ----------------------------------------------------------------------
        uint32_t pb[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          float pr[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const float msub = m_run[nb][h] == -INFINITY ? 0.f : m_run[nb][h];
            pr[h] = fast_exp2(s[nb][h] - msub);
            pr[h + 2] = fast_exp2(s[nb][h + 2] - msub);
            l_run[nb][h] += pr[h] + pr[h + 2];
          }
          pb[nb][0] = movmatrix_trans(pack_half2(pr[0], pr[1]));
          pb[nb][1] = movmatrix_trans(pack_half2(pr[2], pr[3]));
        }
        // ---- O^T += V^T P^T ------------------------------------------------------------------------------
        const uint32_t up = static_cast<uint32_t>(shift + 15) << 10;   // 2^a in fp16
        const uint32_t up2 = up | (up << 16);
        const uint4 v0 = lds128(vb + v_off), v1 = lds128(vb + v_off + kv4::kRowBytes);
        const uint4 v2 = lds128(vb + v_off + 8 * kv4::kRowBytes), v3 = lds128(vb + v_off + 9 * kv4::kRowBytes);
        const uint32_t x0[4] = {v0.x, v0.y, v0.z, v0.w}, x1[4] = {v1.x, v1.y, v1.z, v1.w};
        const uint32_t x2[4] = {v2.x, v2.y, v2.z, v2.w}, x3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint32_t a[4], b[4];
          kv4::unpack_word(__byte_perm(x0[g], x1[g], vsel), a);
          kv4::unpack_word(__byte_perm(x2[g], x3[g], vsel), b);
          const uint32_t u0 = kv4::h2_mul(sv[g][0], up2), u1 = kv4::h2_mul(sv[g][1], up2);
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const uint32_t q0 = kv4::h2_mul(pb[nb][0], u0), q1 = kv4::h2_mul(pb[nb][1], u1);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const uint32_t av[4] = {a[2 * e], a[2 * e + 1], b[2 * e], b[2 * e + 1]};
              mma_16816(o[2 * g + e][nb], av, q0, q1);
            }
          }
        }
      }
      __syncwarp();   // every lane has read the slot
      if (alive && st.more()) {
        request(stage);
        ++pending;
      }
      if (++stage == kStages) {
        stage = 0;
        parity ^= 1;
      }
    }

    // ---- the piece is done: this warp's state to the merge buffer ----------------------------------
    const float down = __int_as_float((127 - shift) << 23);   // 2^-a
    consumer_bar();
    float* mo = merge_o + warp * kD * ROWS;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = l_run[nb][h];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        if (r == 0) {
          float* ml = merge_ml + (warp * ROWS + nb * 8 + 2 * jq + h) * 2;
          ml[0] = m_run[nb][h];
          ml[1] = l;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {   // M block j = 2 g + e: rows r and r + 8 are elements d0 and d0 + 2
        const int d0 = 32 * (j >> 1) + 8 * jv + 4 * (j & 1) + (r & 1);
        *reinterpret_cast<float2*>(mo + d0 * ROWS + nb * 8 + 2 * jq) = make_float2(o[j][nb][0] * down, o[j][nb][1] * down);
        *reinterpret_cast<float2*>(mo + (d0 + 2) * ROWS + nb * 8 + 2 * jq) =
            make_float2(o[j][nb][2] * down, o[j][nb][3] * down);
      }
    }
    Tile t{};
    t.b = pc.b;
    t.np = pc.np;
    t.units0 = (pc.flat - pc.begin) + static_cast<int64_t>(p.piece_cost) * pc.kseq;
    t.whole = whole;
    emit_piece<ROWS>(p, t, team, head, tid, range.nteams_eff, range.units_total, seen_arrivals, merge_o, merge_ml, arrival);
    next_piece(p, seq, range.end, pc);
  }
}

inline int rows_for_group(int group) { return group <= 8 ? 8 : 16; }
inline int ctas_per_sm(int rows) { return rows == 8 ? 4 : 3; }
inline int max_teams(int sms, int kv_heads, int rows) {
  int t = sms * ctas_per_sm(rows) / kv_heads;
  if (t > kMaxTeams) t = kMaxTeams;
  return t < 1 ? 1 : t;
}
inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

template <int ROWS>
int launch_decode(const Kv4DecodeParams& p, bool programmatic, cudaStream_t stream) {
  constexpr int smem = kRingBytes + kConsumerWarps * ROWS * kD * 4 + kConsumerWarps * ROWS * 2 * 4 +
                       kConsumerWarps * kStages * 8 + 4 * 4 + 2 * kSeqCache * 4;
  static bool attr_done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return record_cuda_error(cudaGetLastError());
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kv4_decode_kernel<ROWS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev >= 0 && dev < 64) attr_done[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.nteams * p.kv_heads));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = programmatic ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_decode_kernel<ROWS>, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

}  // namespace

size_t kv4_decode_workspace_bytes(int batch, int q_heads, int kv_heads, int head_dim) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || head_dim != kD) return 0;
  if (q_heads % kv_heads != 0 || q_heads / kv_heads > 16) return 0;
  if (static_cast<int64_t>(batch) * kv_heads > kMaxCounters) return 0;
  const int sms = device_sm_count();
  if (sms <= 0) return 0;
  const int rows = rows_for_group(q_heads / kv_heads);
  const size_t nslots = static_cast<size_t>(max_teams(sms, kv_heads, rows)) + static_cast<size_t>(batch);
  return kCounterBytes + align_up(nslots * kv_heads * rows * kD * sizeof(float), 256) +
         align_up(nslots * kv_heads * rows * sizeof(float), 256);
}

int kv4_paged_decode(const Kv4DecodeArgs& a, cudaStream_t stream) {
  if (a.batch < 0 || a.q_heads <= 0 || a.kv_heads <= 0 || a.max_seq_len < 0) return B200KV_EINVAL;
  if (a.batch == 0) return B200KV_OK;
  if (!a.q || !a.table || !a.seq_lens || !a.out || !a.workspace) return B200KV_EINVAL;
  if (a.table_kind != B200KV_TABLE_BLOCK && a.table_kind != B200KV_TABLE_TOKEN) return B200KV_EINVAL;
  if (a.head_dim != kD || a.page_size != kPS) return B200KV_EUNSUPPORTED;
  if (a.q_heads % a.kv_heads != 0) return B200KV_EUNSUPPORTED;
  const int group = a.q_heads / a.kv_heads;
  if (group > 16) return B200KV_EUNSUPPORTED;
  if (a.batch > 4096) return B200KV_ETOOLARGE;
  if (static_cast<int64_t>(a.batch) * a.kv_heads > kMaxCounters) return B200KV_ETOOLARGE;
  if (a.max_seq_len > (int64_t{1} << 30)) return B200KV_ETOOLARGE;
  if (a.table_rows <= 0 || a.table_cols <= 0 || a.table_row_stride < a.table_cols) return B200KV_EINVAL;
  if (a.row_ids == nullptr && a.batch > a.table_rows) return B200KV_EINVAL;
  if (a.max_seq_len > a.table_cols * (a.table_kind == B200KV_TABLE_BLOCK ? kPS : 1)) return B200KV_EINVAL;
  if (a.flags & ~B200KV_DECODE_SERIALIZED) return B200KV_EINVAL;
  int rc = kv4_check_pool(a.pool, a.pool_pages, a.page_stride_bytes, a.kv_heads);
  if (rc != B200KV_OK) return rc;
  auto mis = [](const void* ptr, uintptr_t al) { return (reinterpret_cast<uintptr_t>(ptr) & (al - 1)) != 0; };
  if (mis(a.q, 16) || mis(a.out, 8) || mis(a.workspace, 16)) return B200KV_EALIGN;
  if (a.q_stride_b % 8 != 0 || a.q_stride_h % 8 != 0) return B200KV_EALIGN;
  if (a.out_stride_b % 4 != 0 || a.out_stride_h % 4 != 0) return B200KV_EALIGN;
  const size_t need = kv4_decode_workspace_bytes(a.batch, a.q_heads, a.kv_heads, a.head_dim);
  if (need == 0) return B200KV_ECUDA;
  if (a.workspace_bytes < need) return B200KV_EWORKSPACE;

  const int sms = device_sm_count();
  const int rows = rows_for_group(group);
  const int teams_cap = max_teams(sms, a.kv_heads, rows);
  // Do not launch more teams than the page bound can feed.
  const int64_t pages_bound = static_cast<int64_t>(a.batch) * ((a.max_seq_len + kPS - 1) / kPS);
  int64_t teams = pages_bound / kMinPagesPerTeam;
  if (teams > teams_cap) teams = teams_cap;
  if (teams < 1) teams = 1;

  Kv4DecodeParams p{};
  p.q = static_cast<const __half*>(a.q);
  p.q_stride_b = a.q_stride_b;
  p.q_stride_h = a.q_stride_h;
  p.pool = static_cast<const uint8_t*>(a.pool);
  p.pool_pages = a.pool_pages;
  p.page_stride = a.page_stride_bytes;
  p.table = a.table;
  p.table_row_stride = a.table_row_stride;
  p.table_kind = a.table_kind;
  p.table_rows = a.table_rows;
  p.row_ids = a.row_ids;
  p.seq_lens = a.seq_lens;
  p.seq_lens_i64 = a.seq_lens_i64;
  p.batch = a.batch;
  p.q_heads = a.q_heads;
  p.kv_heads = a.kv_heads;
  p.group = group;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.max_seq_len = a.max_seq_len;
  p.nteams = static_cast<int>(teams);
  p.piece_cost = kDefaultPieceCost;
  const size_t nslots = static_cast<size_t>(teams_cap) + static_cast<size_t>(a.batch);
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.piece_ctr = reinterpret_cast<unsigned*>(ws);
  p.part_o = reinterpret_cast<float*>(ws + kCounterBytes);
  p.part_lse = reinterpret_cast<float*>(ws + kCounterBytes + align_up(nslots * a.kv_heads * rows * kD * sizeof(float), 256));
  p.out = static_cast<__half*>(a.out);
  p.out_stride_b = a.out_stride_b;
  p.out_stride_h = a.out_stride_h;
  p.status = a.status;
  const bool programmatic = (a.flags & B200KV_DECODE_SERIALIZED) == 0;
  return rows == 8 ? launch_decode<8>(p, programmatic, stream) : launch_decode<16>(p, programmatic, stream);
}

}  // namespace b200kv
