// Paged flash-decoding over the 4-bit cache (format: include/b200kv_kv4.h), one launch; also the short
// chunks of a packed prefill, whose few query rows would fill a small part of a tensor-core tile.
//
// Queries are columns: column c of a request is query token c / G and head c % G of a KV head's group of G
// (a decode step has one token).  A CTA serves ROWS (8 or 16) columns of one KV head in one pass over a
// contiguous range of pages:
//
//   S^T[tok, col] = sum_g s_K[tok, g] * (C_K[tok, d in g] . Q^T[d in g, col])
//   O^T[d, col]  += C_V^T[d, tok] . (P^T[tok, col] * s_V[tok, g(d)])
//
// with C the codes minus 8, integers that fp16 holds exactly.  No element is ever multiplied by its
// scale: K's scales multiply the four partial scores of a token in 32 bits, V's scales go into P,
// where 16 tokens meet 8 columns instead of 128 elements.  A code costs 9/8 of an instruction (one
// logical operation and one packed add per pair, a shift per word) on its way to mma.sync m16n8k16
// (fp16 in, fp32 accumulate; tokens or head_dim are the M rows, the columns N): tcgen05 would want
// the codes as fp16 in shared memory first, and 64 rows to work on.
//
// P * s_V is an fp16 operand, so its range matters.  P = 2^(score - m) with a reference m that is kept
// about 2^7 under the running maximum (it cancels between O and the sum of P): P is at most 2^14 and
// P * s_V at most 2^15, and m is moved, and O rescaled, only when a score or a V scale would
// exceed that.  V scales of 2 and more (values of 14 and more) lower the bound on P accordingly.  A
// product loses bits only below 2^-14, i.e. where it is 2^-21 of the largest weight times one scale unit;
// the absolute error of such a token, 2^-25 * 2^-7 * 8 per code, is far under half a step of the output.
//
// Scheduling.  All sequences' pages are laid end to end and measured in units (pages, plus kPieceCost per
// non-empty sequence: ending a piece costs about that many pages of streaming); team i of kv_heads x
// column-block CTAs takes the i-th equal part.  A part holds tails, whole sequences and heads of sequences
// ("pieces"); a piece that is a whole sequence yields final rows, any other a partial that the CTA which
// arrives last combines.  The plan is made by every CTA from the lengths (one load per sequence and two
// scans), so nothing is synchronised with the host and a captured launch replays with new lengths.
//
// A warp streams its own pages: page k of a piece belongs to warp k % 4, two of them make up one step
// (one wait, one look at the maxima, one request, and twice the independent arithmetic in flight).  Every
// warp keeps a ring of kStages page pairs (2 x (K block + V block), 4608 bytes) that its own lanes fill with
// 16-byte asynchronous copies, nine per lane and pair, as soon as the slot has been read (bulk copies, and
// cache hints, cost several times the instructions here: their operands are uniform registers).  No producer
// warp, no barrier in the steady state; the blocks are stored in the order in which the lanes read
// them (conflict-free 16-byte shared loads).  The page table is read 32 entries at a time, one block of
// entries ahead of use.
//
// Bytes per token and KV head: 2 * 72 (a page is 2304 B where fp16 has 8192).  32 sequences of 1-4 k tokens, 64/8
// heads: 25.9 us = 3.68 TB/s where the fp16 cache takes 57.9; 48 sequences of up to 16 k 34.2 us (fp16 76.9).  Half of the
// rate of a copy: a step's chain (wait, unpack, two products, exponentials) over the 12 warps of an SM bounds it, issue
// slots are 52 % busy, and leaving out the unpacking (22.9 us), V (21.7) or K (21.1) shortens it little.
#include <climits>
#include <cmath>

#include "common.cuh"
#include "kv4.cuh"
#include "launch.h"

namespace b200kv {

namespace {

constexpr int kD = kv4::kHeadDim;
constexpr int kPS = kv4::kPageTok;
constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kStages = 2;
constexpr int kPageBytes = 2 * kv4::kBlockBytes;   // K and V block of one page of one head
constexpr int kPairBytes = 2 * kPageBytes;
constexpr int kRingBytes = kWarps * kStages * kPairBytes;
constexpr int kMinPagesPerTeam = 4;                // a team is not worth launching for fewer pages
constexpr int kPieceCost = 16;
constexpr float kNoScore = -3.0e38f;               // the reference of sums over no token; finite, so that differences are
// Resident CTAs per SM.  Three of them leave 168 registers, which a step of two pages needs (32 sequences of 1-4 k
// tokens, 64/8 heads, us: four, with spills, 31.0; three 25.9; two with 184 registers 26.6).
constexpr int ctas_per_sm(int rows) { return rows == 8 ? 3 : 2; }
constexpr size_t kCounterBytes = B200KV_DECODE_COUNTER_BYTES;
constexpr int64_t kMaxCounters = static_cast<int64_t>(kCounterBytes / sizeof(unsigned));

struct Kv4Params {
  const __half* q;
  int64_t q_stride_t, q_stride_h;
  const uint8_t* pool;
  int pool_pages;
  int64_t page_stride;
  const int32_t* table;
  int64_t table_row_stride;
  int table_kind, table_rows;
  const int32_t* row_ids;
  // Decode: lens are the sequences' lengths, sequence b has query row b.  Chunk (q_lens != nullptr): lens are the
  // contexts, request b has query rows q_start[b] .. + q_lens[b], of which the last sees everything.
  const void* lens;
  const void* q_lens;
  const int32_t* q_start;
  int lens_i64;
  int batch, kv_heads, group;
  int blocks;               // column blocks of ROWS columns
  int max_seq_len;          // decode: bound of the lengths; chunk: positions a table row can name
  int max_q_len;
  int64_t total_q;
  int nteams;
  float scale_log2;
  float4* part_o;           // [nteams + batch][kv_heads][blocks][8 * NB][32] O^T fragments
  float2* part_ml;          // [nteams + batch][kv_heads][blocks][ROWS] (m, l)
  unsigned* piece_ctr;      // [batch][kv_heads][blocks], zero between launches
  __half* out;
  int64_t out_stride_t, out_stride_h;
  int32_t* status;
};

// What every part of the kernel takes a sequence to be.  A table row that does not exist, or a length or
// chunk out of bounds, is reported and never turns into an address: a decode length is limited, anything
// else makes the sequence empty.
struct Seq {
  int len, row, ql;
};
template <bool kChunk>
__device__ __forceinline__ Seq seq_of(const Kv4Params& p, int b) {
  Seq s;
  s.row = p.row_ids ? __ldg(p.row_ids + b) : b;
  int64_t len = load_len(p.lens, p.lens_i64, b);
  bool bad = s.row < 0 || s.row >= p.table_rows || len < 0;
  int64_t ql = 1;
  if (kChunk) {
    ql = load_len(p.q_lens, p.lens_i64, b);
    const int64_t start = __ldg(p.q_start + b);
    bad = bad || ql < 0 || ql > p.max_q_len || len > p.max_seq_len || len + ql > p.max_seq_len || start < 0 ||
          start + ql > p.total_q;
    len = ql > 0 ? len + ql : 0;
  }
  if (bad || len > p.max_seq_len) {
    set_status(p.status, B200KV_DEV_BAD_LENGTH);
    len = bad ? 0 : p.max_seq_len;
  }
  s.len = static_cast<int>(len);
  s.ql = static_cast<int>(ql);
  return s;
}
__device__ __forceinline__ int pages_of(int len) { return (len + kPS - 1) / kPS; }

// a * b / c for 0 <= a, b, c < 2^31 (a 64-bit division only where it takes one).
__device__ __forceinline__ int mul_div(int a, int b, int c) {
  const uint64_t m = static_cast<uint64_t>(static_cast<uint32_t>(a)) * static_cast<uint32_t>(b);
  if (m >> 32) return static_cast<int>(m / static_cast<uint32_t>(c));
  return static_cast<int>(static_cast<uint32_t>(m) / static_cast<uint32_t>(c));
}
// Team whose part of `total` units holds unit x.
__device__ __forceinline__ int team_of(int x, int nteams, int total) {
  const uint64_t m = static_cast<uint64_t>(x + 1) * static_cast<uint32_t>(nteams) - 1;
  if (m >> 32) return static_cast<int>(m / static_cast<uint32_t>(total));
  return static_cast<int>(static_cast<uint32_t>(m) / static_cast<uint32_t>(total));
}

__device__ __forceinline__ void cta_bar() { __syncthreads(); }

// Programmatic dependent launch: what comes before this call may overlap the tail of the previous kernel
// and reads launch metadata only (lengths, rows, page table); every thread makes the call on every path.
__device__ __forceinline__ void pdl_wait_then_trigger() {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
}

__device__ __forceinline__ void async_copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" : : "r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void async_commit() { asm volatile("cp.async.commit_group;\n" : : : "memory"); }
template <int N>
__device__ __forceinline__ void async_wait() {
  asm volatile("cp.async.wait_group %0;\n" : : "n"(N) : "memory");
}
__device__ __forceinline__ void bulk_prefetch_l2(const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;\n" : : "l"(src), "r"(bytes) : "memory");
}
// The tensor instructions are pure functions of registers: not volatile, so that the compiler may
// interleave the two pages of a step.  D = A * B + C.
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                    uint32_t b1, float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
  return d;
}
__device__ __forceinline__ float2 h2_to_f2(uint32_t h2) { return __half22float2(*reinterpret_cast<const __half2*>(&h2)); }
__device__ __forceinline__ uint32_t h2_max(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("max.f16x2 %0, %1, %2;\n" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// A team's part of the page line.
struct TeamRange {
  int b, page, kseq, flat;   // first sequence, its first page, non-empty sequences before it, flat page position
  int end;                   // flat page position of the end
  int units_total, nteams;
  bool any_empty, any;
};
struct PlanScratch {
  int4 sums[kWarps];         // units, non-empty sequences, fewest and most pages of one
  int2 scan[kWarps];
  int4 found[2];             // sequence, page, flat position, kseq at the part's begin and end
};
// Lengths, rows and query rows of kThreads sequences from `first` on.
struct SeqCache {
  int len[kThreads], row[kThreads], ql[kThreads];
};

// Where is this team's part?  Called by the whole CTA (it holds barriers).
template <bool kChunk>
__device__ __forceinline__ TeamRange plan_team_range(const Kv4Params& p, int team, int tid, PlanScratch& sc, SeqCache& cache,
                                                     int& cache_first) {
  const int lane = tid & 31, warp = tid >> 5;
  int units = 0, cnt = 0, lo = INT_MAX, hi = 0, own_np = 0;
  for (int b = tid; b < p.batch; b += kThreads) {
    const Seq s = seq_of<kChunk>(p, b);
    const int np = pages_of(s.len);
    if (b == tid) {
      own_np = np;
      cache.len[tid] = s.len;
      cache.row[tid] = s.row;
      cache.ql[tid] = s.ql;
    }
    if (np > 0) {
      units += np + kPieceCost;
      ++cnt;
      lo = min(lo, np);
      hi = max(hi, np);
    }
  }
  units = __reduce_add_sync(0xffffffffu, units);
  cnt = __reduce_add_sync(0xffffffffu, cnt);
  lo = __reduce_min_sync(0xffffffffu, lo);
  hi = __reduce_max_sync(0xffffffffu, hi);
  if (lane == 0) sc.sums[warp] = make_int4(units, cnt, lo, hi);
  cta_bar();
  units = cnt = hi = 0;
  lo = INT_MAX;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    const int4 v = sc.sums[w];
    units += v.x;
    cnt += v.y;
    lo = min(lo, v.z);
    hi = max(hi, v.w);
  }
  const int pages = units - kPieceCost * cnt;
  TeamRange r;
  r.units_total = units;
  r.any_empty = cnt < p.batch;
  r.nteams = max(1, min(p.nteams, pages / kMinPagesPerTeam));
  // Sequences of one length whose count divides into about as many groups as there are teams: one team per
  // group of whole sequences.  Nothing is then published, counted or combined, at the price of leaving
  // up to a quarter of the CTA slots empty.
  if (cnt > 0 && lo == hi) {
    const int k = (cnt + p.nteams - 1) / p.nteams;
    const int groups = cnt / k;
    if (groups * k == cnt && 4 * groups >= 3 * p.nteams) r.nteams = groups;
  }
  const bool mine = pages > 0 && team < r.nteams;
  int x[2] = {0, 0};
  if (mine) {
    x[0] = mul_div(team, units, r.nteams);
    x[1] = mul_div(team + 1, units, r.nteams);
  }
  if (tid < 2) sc.found[tid] = make_int4(0, 0, pages, 0);   // x[1] == units: the end of the line
  cta_bar();
  if (mine) {
    int before_u = 0, before_c = 0;    // units and non-empty sequences before this round's
    for (int base = 0; base < p.batch && before_u <= x[1]; base += kThreads) {
      const int b = base + tid;
      const int np = base == 0 ? own_np : (b < p.batch ? pages_of(seq_of<kChunk>(p, b).len) : 0);
      const int u = np > 0 ? np + kPieceCost : 0;
      int inc = u;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int o = __shfl_up_sync(0xffffffffu, inc, d);
        if (lane >= d) inc += o;
      }
      const unsigned non_empty = __ballot_sync(0xffffffffu, np > 0);
      if (lane == 31) sc.scan[warp] = make_int2(inc, __popc(non_empty));
      cta_bar();
      int eu = before_u + inc - u, ec = before_c + __popc(non_empty & ((1u << lane) - 1));
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const int2 v = sc.scan[w];
        if (w < warp) {
          eu += v.x;
          ec += v.y;
        }
        before_u += v.x;
        before_c += v.y;
      }
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        if (u > 0 && eu <= x[side] && x[side] < eu + u) {   // positions in a sequence's extra units are its start
          const int page = max(0, x[side] - eu - kPieceCost);
          sc.found[side] = make_int4(b, page, eu - kPieceCost * ec + page, ec);
        }
      }
      cta_bar();
    }
  }
  const int4 f0 = sc.found[0], f1 = sc.found[1];
  r.b = f0.x;
  r.page = f0.y;
  r.flat = f0.z;
  r.kseq = f0.w;
  r.end = f1.z;
  r.any = mine && r.end > r.flat;
  cache_first = 0;
  if (p.batch > kThreads && r.any) {   // the cache holds the sequences from this part's first on
    cta_bar();
    cache_first = r.b;
    const int b = r.b + tid;
    Seq s{0, 0, 0};
    if (b < p.batch) s = seq_of<kChunk>(p, b);
    cache.len[tid] = s.len;
    cache.row[tid] = s.row;
    cache.ql[tid] = s.ql;
  }
  cta_bar();
  return r;
}

// Where a CTA stands: its sequences, the end of its part, its column block.
struct Walk {
  const SeqCache* cache;
  int first;                 // sequence of the cache's first entry
  int end;                   // flat end of the part
  int col0;                  // first column of the block
};
template <bool kChunk>
__device__ __forceinline__ Seq walk_seq(const Kv4Params& p, const Walk& w, int b) {
  const int i = b - w.first;
  if (i < kThreads) return Seq{w.cache->len[i], w.cache->row[i], w.cache->ql[i]};
  return seq_of<kChunk>(p, b);
}

// A piece: the part of one sequence that lies in the team's part.
struct Piece {
  int b, row, len, ql;
  int begin, end;            // pages [begin, end) of the sequence
  int flat;                  // position of page `begin` on the page line
  int kseq;                  // non-empty sequences before b
  bool valid;
};
// The piece that starts at page `page` of sequence pc.b, or the first one after it that has a column for this
// CTA (a shorter chunk may have none in the block).
template <bool kChunk>
__device__ __forceinline__ void settle_piece(const Kv4Params& p, const Walk& w, Piece& pc, int page) {
  for (;;) {
    const Seq s = walk_seq<kChunk>(p, w, pc.b);
    if (s.len > 0) {
      pc.len = s.len;
      pc.row = s.row;
      pc.ql = s.ql;
      pc.begin = page;
      pc.end = min(pages_of(s.len), page + (w.end - pc.flat));
      pc.valid = true;
      if (!kChunk || s.ql * p.group > w.col0) return;
      pc.flat += pc.end - pc.begin;
      ++pc.kseq;
    }
    ++pc.b;
    page = 0;
    if (pc.flat >= w.end || pc.b >= p.batch) {
      pc.valid = false;
      return;
    }
  }
}
template <bool kChunk>
__device__ __forceinline__ void next_piece(const Kv4Params& p, const Walk& w, Piece& pc) {
  pc.flat += pc.end - pc.begin;
  pc.valid = false;
  ++pc.kseq;
  ++pc.b;
  if (pc.flat < w.end && pc.b < p.batch) settle_piece<kChunk>(p, w, pc, 0);
}
// Pages of a piece that belong to a warp.
__device__ __forceinline__ int warp_pages(const Piece& pc, int warp) {
  return pc.valid ? (pc.end - pc.begin - warp + kWarps - 1) / kWarps : 0;
}

// The pages a warp requests, in order and two at a time: lane l holds the number of page
// begin + warp + 4 * (32 * block + l) of the piece; the next block of table entries (of this piece, or
// the first of the next piece) is already on its way.
template <bool kChunk>
struct PageStream {
  Piece pc, nx;
  int m, cnt;            // next page of this warp in pc, and how many it has there
  int32_t ids, ids_next; // page numbers in use; raw table entries of the next block

  // Raw table entry -> page number; an entry that names no page is reported and page 0 read instead.
  __device__ __forceinline__ static int32_t checked(const Kv4Params& p, int32_t id) {
    int32_t page = id;
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
  }
  __device__ __forceinline__ int32_t load_ids(const Kv4Params& p, const Piece& from, int warp, int lane, int first) const {
    const int page = from.begin + warp + kWarps * (first + lane);
    if (!from.valid || page >= from.end) return 0;
    const int64_t at = p.table_kind == B200KV_TABLE_BLOCK ? page : static_cast<int64_t>(page) * kPS;
    return __ldg(p.table + static_cast<int64_t>(from.row) * p.table_row_stride + at);
  }
  __device__ __forceinline__ void refill(const Kv4Params& p, const Walk& w, int warp, int lane) {
    if (m + 32 < cnt) {
      ids_next = load_ids(p, pc, warp, lane, m + 32);
    } else {
      nx = pc;
      do {
        next_piece<kChunk>(p, w, nx);
      } while (nx.valid && warp_pages(nx, warp) <= 0);   // short pieces have no page for the later warps
      ids_next = load_ids(p, nx, warp, lane, 0);
    }
  }
  __device__ __forceinline__ void start(const Kv4Params& p, const Walk& w, const Piece& first,
                                        int warp, int lane) {
    pc = first;
    while (pc.valid && warp_pages(pc, warp) <= 0) next_piece<kChunk>(p, w, pc);
    m = 0;
    cnt = warp_pages(pc, warp);
    ids = checked(p, load_ids(p, pc, warp, lane, 0));
    if (pc.valid) refill(p, w, warp, lane);
  }
  __device__ __forceinline__ bool more() const { return pc.valid; }
  __device__ __forceinline__ void advance(const Kv4Params& p, const Walk& w, int warp, int lane) {
    m += 2;
    const bool done = m >= cnt;
    if (!done && (m & 31) != 0) return;
    if (done) {
      pc = nx;
      m = 0;
      cnt = warp_pages(pc, warp);
    }
    ids = checked(p, ids_next);
    if (pc.valid) refill(p, w, warp, lane);
  }
};

// S^T of 16 tokens: k_at and c_at are this lane's chunk of token r and that token's scales.
template <int NB>
__device__ __forceinline__ void page_scores(const uint8_t* k_at, const uint8_t* c_at, const uint32_t (&qf)[NB][8][2],
                                            float (&s)[NB][4]) {
  const uint4 k0 = *reinterpret_cast<const uint4*>(k_at), k1 = *reinterpret_cast<const uint4*>(k_at + 8 * kv4::kRowBytes);
  const uint2 c0 = *reinterpret_cast<const uint2*>(c_at), c1 = *reinterpret_cast<const uint2*>(c_at + 8 * kv4::kScaleBytes);
  const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
  const float2 f0a = h2_to_f2(c0.x), f0b = h2_to_f2(c0.y), f1a = h2_to_f2(c1.x), f1b = h2_to_f2(c1.y);
  const float f0[4] = {f0a.x, f0a.y, f0b.x, f0b.y}, f1[4] = {f1a.x, f1a.y, f1b.x, f1b.y};
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint32_t a[4], b[4];
    kv4::unpack_word(w0[g], a);
    kv4::unpack_word(w1[g], b);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float d[4];
      mma(d, a[0], b[0], a[1], b[1], qf[nb][2 * g][0], qf[nb][2 * g][1], 0.f, 0.f, 0.f, 0.f);
      mma(d, a[2], b[2], a[3], b[3], qf[nb][2 * g + 1][0], qf[nb][2 * g + 1][1], d[0], d[1], d[2], d[3]);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = i < 2 ? f0[g] : f1[g];
        s[nb][i] = g == 0 ? f * d[i] : s[nb][i] + f * d[i];
      }
    }
  }
}

// V scales of tokens 2jq, 2jq+1 | 2jq+8, 2jq+9 as fp16 pairs per group.
__device__ __forceinline__ void page_v_scales(const uint8_t* at, uint32_t (&sv)[4][2]) {
  const uint4 t0 = *reinterpret_cast<const uint4*>(at), t1 = *reinterpret_cast<const uint4*>(at + 8 * kv4::kScaleBytes);
  sv[0][0] = __byte_perm(t0.x, t0.z, 0x5410);
  sv[1][0] = __byte_perm(t0.x, t0.z, 0x7632);
  sv[2][0] = __byte_perm(t0.y, t0.w, 0x5410);
  sv[3][0] = __byte_perm(t0.y, t0.w, 0x7632);
  sv[0][1] = __byte_perm(t1.x, t1.z, 0x5410);
  sv[1][1] = __byte_perm(t1.x, t1.z, 0x7632);
  sv[2][1] = __byte_perm(t1.y, t1.w, 0x5410);
  sv[3][1] = __byte_perm(t1.y, t1.w, 0x7632);
}

// O^T += V^T (P^T s_V) of 16 tokens.  kMasked: `seen` has all ones where this lane's column (as a B fragment)
// sees the token, so that a V scale of NaN reaches no column that does not.
template <int NB, bool kMasked>
__device__ __forceinline__ void page_pv(const uint8_t* v_at, uint32_t vsel, const uint32_t (&sv)[4][2],
                                        const uint32_t (&pb)[NB][2], const uint32_t (&seen)[NB][2],
                                        float (&o)[8][NB][4]) {
  const uint4 v0 = *reinterpret_cast<const uint4*>(v_at), v1 = *reinterpret_cast<const uint4*>(v_at + kv4::kRowBytes);
  const uint4 v2 = *reinterpret_cast<const uint4*>(v_at + 8 * kv4::kRowBytes);
  const uint4 v3 = *reinterpret_cast<const uint4*>(v_at + 9 * kv4::kRowBytes);
  const uint32_t x0[4] = {v0.x, v0.y, v0.z, v0.w}, x1[4] = {v1.x, v1.y, v1.z, v1.w};
  const uint32_t x2[4] = {v2.x, v2.y, v2.z, v2.w}, x3[4] = {v3.x, v3.y, v3.z, v3.w};
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    uint32_t a[4], b[4];
    kv4::unpack_word(__byte_perm(x0[g], x1[g], vsel), a);
    kv4::unpack_word(__byte_perm(x2[g], x3[g], vsel), b);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      uint32_t q0 = kv4::h2_mul(pb[nb][0], sv[g][0]), q1 = kv4::h2_mul(pb[nb][1], sv[g][1]);
      if (kMasked) {
        q0 &= seen[nb][0];
        q1 &= seen[nb][1];
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float(&acc)[4] = o[2 * g + e][nb];
        mma(acc, a[2 * e], a[2 * e + 1], b[2 * e], b[2 * e + 1], q0, q1, acc[0], acc[1], acc[2], acc[3]);
      }
    }
  }
}

// Column sums of what `n` contributors hold, in the order of the O^T fragments: a thread takes 16-byte
// pieces (M block j, lane) with the head columns 2 jq and 2 jq + 1 of N block nb.
struct Weighted {
  float m[2], l[2];
  float acc[4];
  __device__ __forceinline__ void add(const float4& v, float w0, float w1) {
    acc[0] += w0 * v.x;
    acc[1] += w1 * v.y;
    acc[2] += w0 * v.z;
    acc[3] += w1 * v.w;
  }
};

// The end of a piece.  The four warps put their O^T fragments, as they are, and their (m, l) into shared
// memory; every thread then combines 2 * NB of the 16-byte pieces over the warps and writes the final
// rows (whole sequence) or the partial, in the same fragment order (16-byte accesses without bank
// conflicts or strides all the way).  A partial is published by one release-acquire count on the
// (sequence, head, column block) counter, which wraps to zero on the last arrival; the CTA that arrives last
// combines the partials of all pieces the same way.
template <int ROWS, bool kChunk>
__device__ __forceinline__ void finish_piece(const Kv4Params& p, const Piece& pc, bool whole, int team, int head, int blk, int q_row0, int tid,
                                             const float (&o)[8][ROWS / 8][4], const float (&m_ref)[ROWS / 8][2],
                                             const float (&l_run)[ROWS / 8][2], float4* merge_o, float2* merge_ml,
                                             int* note) {
  constexpr int NB = ROWS / 8;
  constexpr int kParts = 8 * NB;               // fragments of a warp
  const int lane = tid & 31, warp = tid >> 5;
  const int r = lane >> 2, jq = lane & 3;
  cta_bar();   // the previous piece's merge has read the buffers
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      merge_o[(warp * kParts + nb * 8 + j) * 32 + lane] = make_float4(o[j][nb][0], o[j][nb][1], o[j][nb][2], o[j][nb][3]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float l = l_run[nb][h];
      l += __shfl_xor_sync(0xffffffffu, l, 4);
      l += __shfl_xor_sync(0xffffffffu, l, 8);
      l += __shfl_xor_sync(0xffffffffu, l, 16);
      if (r == 0) merge_ml[warp * ROWS + nb * 8 + 2 * jq + h] = make_float2(l == 0.f ? kNoScore : m_ref[nb][h], l);
    }
  }
  cta_bar();
  // O / l of one fragment (M block j = 2 g + e: elements d0 and d0 + 2, heads 2 jq, 2 jq + 1) -> out
  auto write_out = [&](int nb, int j, const Weighted& w) {
    const int d0 = 32 * (j >> 1) + 8 * (r >> 1) + 4 * (j & 1) + (r & 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int col = blk * ROWS + nb * 8 + 2 * jq + h;
      if (col < (kChunk ? pc.ql * p.group : p.group)) {
        const int tok = kChunk ? col / p.group : 0;
        __half* dst = p.out + static_cast<int64_t>(q_row0 + tok) * p.out_stride_t +
                      static_cast<int64_t>(head * p.group + col - tok * p.group) * p.out_stride_h + d0;
        dst[0] = __float2half_rn(w.acc[h] / w.l[h]);
        dst[2] = __float2half_rn(w.acc[h + 2] / w.l[h]);
      }
    }
  };
  const int64_t slot = ((static_cast<int64_t>(team) + pc.b) * p.kv_heads + head) * p.blocks + blk;
  float4* part = p.part_o + slot * kParts * 32;
  float2* part_ml = p.part_ml + slot * ROWS;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    // (m, l) of the four warps for this lane's two heads
    float2 ml[kWarps][2];
    float top[2] = {kNoScore, kNoScore};
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 v = *reinterpret_cast<const float4*>(merge_ml + w * ROWS + nb * 8 + 2 * jq);
      ml[w][0] = make_float2(v.x, v.y);
      ml[w][1] = make_float2(v.z, v.w);
      top[0] = fmaxf(top[0], v.x);
      top[1] = fmaxf(top[1], v.z);
    }
    float wt[kWarps][2];
    Weighted sum[2];
    float l[2] = {0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kWarps; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        wt[w][h] = fast_exp2(ml[w][h].x - top[h]);
        l[h] += wt[w][h] * ml[w][h].y;
      }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int j = 2 * warp + k;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[k].acc[i] = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w)
        sum[k].add(merge_o[(w * kParts + nb * 8 + j) * 32 + lane], wt[w][0], wt[w][1]);
      if (whole) {
        sum[k].l[0] = l[0];
        sum[k].l[1] = l[1];
        write_out(nb, j, sum[k]);
      } else {
        __stcg(part + (nb * 8 + j) * 32 + lane, make_float4(sum[k].acc[0], sum[k].acc[1], sum[k].acc[2], sum[k].acc[3]));
      }
    }
    if (!whole && warp == 0 && r == 0)
      __stcg(reinterpret_cast<float4*>(part_ml + nb * 8 + 2 * jq), make_float4(top[0], l[0], top[1], l[1]));
  }
  if (whole) return;
  const int first_team = note[1], pieces = note[2];   // thread 0 rewrites both when the next piece begins
  cta_bar();   // all of the CTA's partial is written; the count below publishes it
  if (tid == 0)
    note[0] = atomic_inc_acq_rel(p.piece_ctr + (static_cast<int64_t>(pc.b) * p.kv_heads + head) * p.blocks + blk,
                                 static_cast<unsigned>(pieces - 1)) == static_cast<unsigned>(pieces - 1);
  cta_bar();
  if (note[0] == 0) return;
  // Last to arrive: the partials of all pieces (this CTA's own among them) lie in neighbouring slots.
  const int64_t slot0 = ((static_cast<int64_t>(first_team) + pc.b) * p.kv_heads + head) * p.blocks + blk;
  const int64_t step = static_cast<int64_t>(p.kv_heads) * p.blocks;
  constexpr int kBatch = 4;                    // partials in flight
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    Weighted sum[2];
    float top[2] = {kNoScore, kNoScore}, l[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[k].acc[i] = 0.f;
#pragma unroll 1
    for (int p0 = 0; p0 < pieces; p0 += kBatch) {
      float4 ml[kBatch], v[kBatch][2];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        if (p0 + i < pieces) {
          const int64_t sl = slot0 + (p0 + i) * step;
          ml[i] = __ldcg(reinterpret_cast<const float4*>(p.part_ml + sl * ROWS + nb * 8 + 2 * jq));
#pragma unroll
          for (int k = 0; k < 2; ++k)
            v[i][k] = __ldcg(p.part_o + (sl * kParts + nb * 8 + 2 * warp + k) * 32 + lane);
        } else {
          ml[i] = make_float4(kNoScore, 0.f, kNoScore, 0.f);
          v[i][0] = v[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
      }
      float was[2] = {top[0], top[1]};
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        top[0] = fmaxf(top[0], ml[i].x);
        top[1] = fmaxf(top[1], ml[i].z);
      }
      float re[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        re[h] = fast_exp2(was[h] - top[h]);
        l[h] *= re[h];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[k].acc[i] *= re[i & 1];
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const float w0 = fast_exp2(ml[i].x - top[0]), w1 = fast_exp2(ml[i].z - top[1]);
        l[0] += w0 * ml[i].y;
        l[1] += w1 * ml[i].w;
#pragma unroll
        for (int k = 0; k < 2; ++k) sum[k].add(v[i][k], w0, w1);
      }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sum[k].l[0] = l[0];
      sum[k].l[1] = l[1];
      write_out(nb, 2 * warp + k, sum[k]);
    }
  }
}

// kChunk: query rows come in chunks (p.q_lens); a decode step has one per sequence, and its code none of the
// arithmetic that several take.
template <int ROWS, bool kChunk>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(ROWS)) kv4_decode_kernel(Kv4Params p) {
  static_assert(ROWS == 8 || ROWS == 16, "columns are padded to 8 or 16");
  constexpr int NB = ROWS / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  float4* merge_o = reinterpret_cast<float4*>(smem + kRingBytes);          // [4 warps][8 * NB][32 lanes]
  float2* merge_ml = reinterpret_cast<float2*>(merge_o + kWarps * 8 * NB * 32);   // [4][ROWS] (m, l)
  int* note = reinterpret_cast<int*>(merge_ml + kWarps * ROWS);            // [0] this CTA merges, [1] first team, [2] pieces
  SeqCache& cache = *reinterpret_cast<SeqCache*>(note + 4);
  PlanScratch& scratch = *reinterpret_cast<PlanScratch*>(merge_o);

  const int tid = threadIdx.x;
  const int lane = tid & 31;
  const int warp = tid >> 5;
  const int unit = kChunk ? blockIdx.x / p.blocks : blockIdx.x;
  const int blk = kChunk ? blockIdx.x - unit * p.blocks : 0;
  const int team = unit / p.kv_heads;
  const int head = unit - team * p.kv_heads;
  const uint8_t* ring = smem + warp * (kStages * kPairBytes);
  if (kChunk) pdl_wait_then_trigger();   // a chunk's lengths may come straight from the kernel before
  Walk walk;
  const TeamRange range = plan_team_range<kChunk>(p, team, tid, scratch, cache, walk.first);
  walk.cache = &cache;
  walk.end = range.end;
  walk.col0 = blk * ROWS;
  Piece pc;
  pc.valid = false;
  PageStream<kChunk> st;
  if (range.any) {
    pc.b = range.b;
    pc.flat = range.flat;
    pc.kseq = range.kseq;
    settle_piece<kChunk>(p, walk, pc, range.page);
    st.start(p, walk, pc, warp, lane);
  }
  const uint8_t* k_rows = p.pool + static_cast<int64_t>(head) * kv4::kBlockBytes;
  const int64_t v_from_k = static_cast<int64_t>(p.kv_heads) * kv4::kBlockBytes;
  // First pages towards L2 while the previous kernel is still finishing: L2 is the point of coherence,
  // so rows that kernel writes afterwards are still seen by the copies below.
  if (range.any && st.more() && lane < min(st.cnt, 2 * kStages)) {
    const uint8_t* src = k_rows + st.ids * p.page_stride;
    bulk_prefetch_l2(src, kv4::kBlockBytes);
    bulk_prefetch_l2(src + v_from_k, kv4::kBlockBytes);
  }
  pdl_wait_then_trigger();   // q, the pool, the workspace and out belong to earlier kernels until here
  if (!kChunk && team == 0 && range.any_empty) {
    // No keys: the output rows of a decode step are defined as zero, and nobody else writes them.
    for (int b = 0; b < p.batch; ++b) {
      if (seq_of<kChunk>(p, b).len != 0) continue;
      for (int g = 0; g < p.group; ++g)
        p.out[static_cast<int64_t>(b) * p.out_stride_t +
              (static_cast<int64_t>(head) * p.group + g) * p.out_stride_h + tid] = __float2half_rn(0.f);
    }
  }
  if (!range.any) return;

  // The next two pages into ring slot `stage`.  The pair is four blocks (K and V of the first page, K and V of
  // the second); eight lanes copy a block, each of them every eighth of its 72 16-byte pieces, so that a lane
  // has one address.
  const int my_block = lane >> 3;
  const uint8_t* my_rows = k_rows + ((my_block & 1) ? v_from_k : 0) + (lane & 7) * 16;
  const uint32_t my_dst = smem_u32(ring) + my_block * kv4::kBlockBytes + (lane & 7) * 16;
  const uint32_t page_stride = static_cast<uint32_t>(p.page_stride);   // the host refuses strides of 2^31 and more
  auto request = [&](int stage) {
    if (st.more()) {
      const bool two = st.cnt - st.m >= 2;
      const int32_t id = __shfl_sync(0xffffffffu, st.ids, (st.m & 31) + (my_block >> 1));
      if (two || my_block < 2) {
        const uint8_t* src = my_rows + static_cast<uint64_t>(static_cast<uint32_t>(id)) * page_stride;
        const uint32_t dst = my_dst + stage * kPairBytes;
#pragma unroll
        for (int i = 0; i < kv4::kBlockBytes / 128; ++i) async_copy16(dst + i * 128, src + i * 128);
      }
      st.advance(p, walk, warp, lane);
    }
    async_commit();   // an empty group too: the wait below counts groups
  };
  for (int s = 0; s < kStages; ++s) request(s);

  const int r = lane >> 2;     // fragment row: token (S^T) or one of the 8 row pairs of head_dim (O^T); also a head column
  const int jq = lane & 3;     // fragment column pair
  const int jv = r >> 1;       // V: chunk of the token rows that holds this lane's elements ...
  const uint32_t vsel = (r & 1) ? 0x7632u : 0x5410u;   // ... and which half of its words
  // this lane's places in a pair: K chunk and scales of token r, V chunk and scales of token 2 jq
  const uint8_t* k_at = ring + kv4::chunk_offset(r, jq);
  const uint8_t* kc_at = ring + kv4::kScaleOffset + r * kv4::kScaleBytes;
  const uint8_t* v_at = ring + kv4::kBlockBytes + kv4::chunk_offset(2 * jq, jv);
  const uint8_t* vc_at = ring + kv4::kBlockBytes + kv4::kScaleOffset + 2 * jq * kv4::kScaleBytes;
  int stage = 0;

  while (pc.valid) {
    uint32_t qf[NB][8][2];     // Q^T as B fragments
    float o[8][NB][4];         // O^T: 8 M blocks of 16 along head_dim
    float m_ref[NB][2], l_run[NB][2];
    const int q_row0 = kChunk ? __ldg(p.q_start + pc.b) : pc.b;
    const int cols = kChunk ? pc.ql * p.group : p.group;
    const int pos0 = pc.len - (kChunk ? pc.ql : 1);     // position of the first query token: column c sees positions <= pos0 + c / group
    int lim[NB][2], lim_r[NB];           // of columns 2 jq, 2 jq + 1 (S^T) and r (P^T as B fragment) of each N block
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      lim[nb][0] = lim[nb][1] = lim_r[nb] = pos0;
      const int col = walk.col0 + nb * 8 + r;
      int tok = 0, hq = col;
      if (kChunk) {
        tok = col / p.group;
        hq = col - tok * p.group;
        lim_r[nb] += tok;
        lim[nb][0] += (walk.col0 + nb * 8 + 2 * jq) / p.group;
        lim[nb][1] += (walk.col0 + nb * 8 + 2 * jq + 1) / p.group;
      }
      const __half* qh = p.q + static_cast<int64_t>(q_row0 + tok) * p.q_stride_t +
                         (static_cast<int64_t>(head) * p.group + hq) * p.q_stride_h + 8 * jq;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const uint4 v = col < cols ? __ldg(reinterpret_cast<const uint4*>(qh + 32 * g)) : make_uint4(0, 0, 0, 0);
        qf[nb][2 * g][0] = v.x;
        qf[nb][2 * g][1] = v.y;
        qf[nb][2 * g + 1][0] = v.z;
        qf[nb][2 * g + 1][1] = v.w;
      }
      m_ref[nb][0] = m_ref[nb][1] = 0.f;
      l_run[nb][0] = l_run[nb][1] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) o[j][nb][0] = o[j][nb][1] = o[j][nb][2] = o[j][nb][3] = 0.f;
    float p_room = 14.f;       // log2 of the largest P allowed: P * (largest V scale) stays under 2^15
    uint32_t sv_lim = 0x4000u; // V scales seen are below this fp16 number (2 to begin with)
    // positions up to here are seen by every column of the block
    const int all_see = pos0 + (kChunk ? walk.col0 / p.group : 0);
    const int np = pages_of(pc.len);
    const bool whole = pc.begin == 0 && pc.end == np;
    const int cnt = warp_pages(pc, warp);
    if (tid == 0 && !whole) {   // the teams that hold a piece of this sequence; read at the end of the piece
      const int u0 = pc.flat - pc.begin + kPieceCost * (pc.kseq + 1);
      note[1] = team_of(u0, range.nteams, range.units_total);
      note[2] = team_of(u0 + np - 1, range.nteams, range.units_total) - note[1] + 1;
    }

#pragma unroll 1
    for (int m = 0; m < cnt; m += 2) {
      const int page = pc.begin + warp + kWarps * m;      // the step's pages are this one and the fourth after it
      const bool masked = m + 1 >= cnt || (page + kWarps) * kPS + kPS - 1 > all_see;
      async_wait<kStages - 1>();
      __syncwarp();   // the pair's pieces were copied by all lanes
      const int pair = stage * kPairBytes;
      float s[2][NB][4];
      uint32_t sv[2][4][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        page_scores<NB>(k_at + pair + h * kPageBytes, kc_at + pair + h * kPageBytes, qf, s[h]);
        page_v_scales(vc_at + pair + h * kPageBytes, sv[h]);
      }
      // scores relative to the reference, in the log2 domain
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[h][nb][i] = fmaf(s[h][nb][i], p.scale_log2, -m_ref[nb][i & 1]);
      if (masked) {
        // Rows past the length were never written and a missing second page was not loaded: they may
        // hold anything, NaN scales included.  Positions past a column's own are not for it.
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int at = m + h < cnt ? (page + kWarps * h) * kPS : INT_MAX - kPS;   // position of the page's first token
#pragma unroll
          for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (at + r > lim[nb][i]) s[h][nb][i] = -INFINITY;
              if (at + r + 8 > lim[nb][i]) s[h][nb][i + 2] = -INFINITY;
            }
          const int n = pc.len - at - 2 * jq;
          const uint32_t keep0 = (0 < n ? 0xffffu : 0u) | (1 < n ? 0xffff0000u : 0u);
          const uint32_t keep1 = (8 < n ? 0xffffu : 0u) | (9 < n ? 0xffff0000u : 0u);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            sv[h][g][0] &= keep0;
            sv[h][g][1] &= keep1;
          }
        }
      }
      // ---- would a weight, or a weight times its V scale, leave fp16's range? --------------------
      uint32_t any_sv = 0;     // bitwise or of non-negative numbers: not below the largest
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int g = 0; g < 4; ++g) any_sv |= sv[h][g][0] | sv[h][g][1];
      // (The first step of a piece always goes there: it sets the reference.)
      bool grow = m == 0 || ((any_sv + (0x8000u - sv_lim) * 0x10001u) & 0x80008000u) != 0;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float top = fmaxf(fmaxf(s[0][nb][i], s[0][nb][i + 2]), fmaxf(s[1][nb][i], s[1][nb][i + 2]));
          grow |= top > p_room;
        }
      if (__any_sync(0xffffffffu, grow)) {
        uint32_t top2 = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int g = 0; g < 4; ++g) top2 = h2_max(top2, h2_max(sv[h][g][0], sv[h][g][1]));   // NaN is passed over
        const float2 tf = h2_to_f2(top2);
        float hi = fmaxf(tf.x, tf.y);
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 1));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, 2));
        const int e = min(static_cast<int>(__float_as_uint(hi) >> 23) - 127 + 1, 16);   // hi < 2^e
        if (e > 1) {
          p_room = fminf(p_room, static_cast<float>(15 - e));
          sv_lim = max(sv_lim, static_cast<uint32_t>(e + 15) << 10);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float mx = fmaxf(fmaxf(s[0][nb][i], s[0][nb][i + 2]), fmaxf(s[1][nb][i], s[1][nb][i + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            // the largest weight so far becomes 2^(p_room - 7), unless the reference is higher already
            float up = mx - (p_room - 7.f);
            if (m == 0) up = mx > -INFINITY ? up : 0.f;   // nothing seen: nothing will be, positions only grow
            else up = fmaxf(0.f, up);
            const float alpha = m == 0 ? 0.f : fast_exp2(-up);
            m_ref[nb][i] += up;
            l_run[nb][i] *= alpha;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              s[h][nb][i] -= up;
              s[h][nb][i + 2] -= up;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              o[j][nb][i] *= alpha;
              o[j][nb][i + 2] *= alpha;
            }
          }
      }
      // ---- P^T -> B fragments, O^T += V^T (P^T s_V) -------------------------------------------------
      uint32_t pb[2][NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = fast_exp2(s[h][nb][0]), p1 = fast_exp2(s[h][nb][1]);
          const float p2 = fast_exp2(s[h][nb][2]), p3 = fast_exp2(s[h][nb][3]);
          l_run[nb][0] += p0 + p2;
          l_run[nb][1] += p1 + p3;
          pb[h][nb][0] = movmatrix_trans(pack_half2(p0, p1));
          pb[h][nb][1] = movmatrix_trans(pack_half2(p2, p3));
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint32_t seen[NB][2];
        if (kChunk && masked) {
          const int at = m + h < cnt ? (page + kWarps * h) * kPS + 2 * jq : INT_MAX - kPS;
#pragma unroll
          for (int nb = 0; nb < NB; ++nb) {
            const int n = lim_r[nb] - at;
            seen[nb][0] = (0 <= n ? 0xffffu : 0u) | (1 <= n ? 0xffff0000u : 0u);
            seen[nb][1] = (8 <= n ? 0xffffu : 0u) | (9 <= n ? 0xffff0000u : 0u);
          }
          page_pv<NB, true>(v_at + pair + h * kPageBytes, vsel, sv[h], pb[h], seen, o);
        } else {
          page_pv<NB, false>(v_at + pair + h * kPageBytes, vsel, sv[h], pb[h], seen, o);
        }
      }
      __syncwarp();   // every lane has read the slot
      request(stage);
      if (++stage == kStages) stage = 0;
    }

    finish_piece<ROWS, kChunk>(p, pc, whole, team, head, blk, q_row0, tid, o, m_ref, l_run, merge_o, merge_ml, note);
    next_piece<kChunk>(p, walk, pc);
  }
}

inline int64_t align_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }

// How a launch is cut: columns per CTA, column blocks, teams at most.
struct Shape {
  int rows, blocks, teams;
};
int shape_of(int max_q_len, int q_heads, int kv_heads, Shape* s) {
  const int sms = device_sm_count();
  if (sms <= 0) return B200KV_ECUDA;
  const int cols = max_q_len * (q_heads / kv_heads);
  s->rows = cols <= 8 ? 8 : 16;
  s->blocks = (cols + s->rows - 1) / s->rows;
  const int t = sms * ctas_per_sm(s->rows) / (kv_heads * s->blocks);
  s->teams = t < 1 ? 1 : t;
  return B200KV_OK;
}

// Byte offsets of the workspace's parts: counters, partial outputs, (m, l).
struct Layout {
  int64_t ml, total;
};
Layout layout_of(const Shape& s, int batch, int kv_heads) {
  const int64_t slots = (static_cast<int64_t>(s.teams) + batch) * kv_heads * s.blocks;
  Layout l;
  l.ml = static_cast<int64_t>(kCounterBytes) + slots * s.rows * kD * 4;
  l.total = l.ml + align_up(slots * s.rows * 8, 256);
  return l;
}

template <int ROWS, bool kChunk>
int launch_decode(const Kv4Params& p, bool programmatic, cudaStream_t stream) {
  constexpr int smem = kRingBytes + kWarps * ROWS * kD * 4 + kWarps * ROWS * 2 * 4 + 4 * 4 + static_cast<int>(sizeof(SeqCache));
  static bool attr_done[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return record_cuda_error(cudaGetLastError());
  if (dev < 0 || dev >= 64 || !attr_done[dev]) {
    cudaError_t e = cudaFuncSetAttribute(kv4_decode_kernel<ROWS, kChunk>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return record_cuda_error(e);
    if (dev >= 0 && dev < 64) attr_done[dev] = true;
  }
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(p.nteams * p.kv_heads * p.blocks));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = programmatic ? 1 : 0;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_decode_kernel<ROWS, kChunk>, p);
  if (e != cudaSuccess) return record_cuda_error(e);
  return check_launch();
}

int run_decode(Kv4Params& p, int q_heads, const Shape& s, void* workspace, size_t workspace_bytes, int64_t max_kv_len,
               bool programmatic, cudaStream_t stream) {
  if (static_cast<int64_t>(p.batch) * p.kv_heads * s.blocks > kMaxCounters) return B200KV_ETOOLARGE;
  const int64_t pages_bound = static_cast<int64_t>(p.batch) * ((max_kv_len + kPS - 1) / kPS + kPieceCost);
  if (pages_bound > INT_MAX) return B200KV_ETOOLARGE;   // the page line is counted in 32 bits
  const Layout l = layout_of(s, p.batch, p.kv_heads);
  if (workspace_bytes < static_cast<size_t>(l.total)) return B200KV_EWORKSPACE;
  // Do not launch more teams than the page bound can feed, nor cut a sequence of n pages into many more than
  // 0.8 sqrt(n) pieces: a piece more saves streaming as 1 / pieces^2 and costs its share of the combination
  // that ends the sequence (one KV head, one sequence, us for 48 / 96 / 128 / 444 pieces: 13 / 16 / 19 / 52 at
  // 2048 pages, 25 / 22 / 24 / 58 at 8192).
  const int64_t pages = (max_kv_len + kPS - 1) / kPS;
  int64_t teams = static_cast<int64_t>(p.batch) * pages / kMinPagesPerTeam;
  const int64_t fine = static_cast<int64_t>(p.batch * (1. + 0.8 * std::sqrt(static_cast<double>(pages))));
  if (teams > fine) teams = fine;
  if (teams > s.teams) teams = s.teams;
  p.nteams = static_cast<int>(teams < 1 ? 1 : teams);
  p.blocks = s.blocks;
  p.group = q_heads / p.kv_heads;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  p.piece_ctr = reinterpret_cast<unsigned*>(ws);
  p.part_o = reinterpret_cast<float4*>(ws + kCounterBytes);
  p.part_ml = reinterpret_cast<float2*>(ws + l.ml);
  if (p.q_lens != nullptr)
    return s.rows == 8 ? launch_decode<8, true>(p, programmatic, stream) : launch_decode<16, true>(p, programmatic, stream);
  return s.rows == 8 ? launch_decode<8, false>(p, programmatic, stream) : launch_decode<16, false>(p, programmatic, stream);
}

inline bool misaligned(const void* ptr, uintptr_t al) { return (reinterpret_cast<uintptr_t>(ptr) & (al - 1)) != 0; }

// A chunk is streamed like a decode step when it has at most kChunkRows rows, and at most kChunkColumns columns (rows
// x heads of a group) or at most kChunkWork columns over all KV heads and requests.  Streaming costs a pass over
// the keys per 16 columns; the 128-row tiles cost the same whatever part of them is filled, but have few CTAs to
// spread over when there are few heads and requests.  Streamed / tiles, us, contexts of 2 k and 12 k:
//   128 columns: 1 request, 32/4 heads 13.7 / 27.8 and 26.8 / 54.6; 4 requests, 64/8 heads 30.3 / 42.1 and 141 / 211
//   256 columns: 1 request, 32/4 heads 16.7 / 27.8 and 43.6 / 55.2; 4 requests, 64/8 heads 56.5 / 42.4 and 278 / 213
//   1024 columns in all, contexts of 1 k and 12 k: 1 request, 8/1 heads 14.1 / 23.9 and 45.0 / 54.8; 2048: 2 requests
//   18.0 / 24.9 and 79.3 / 60.2
constexpr int kChunkRows = 128;
constexpr int kChunkColumns = 128;
constexpr int kChunkWork = 1024;

}  // namespace

size_t kv4_decode_workspace_bytes(int batch, int q_heads, int kv_heads, int head_dim) {
  if (batch <= 0 || batch > 4096 || q_heads <= 0 || kv_heads <= 0 || head_dim != kD) return 0;
  if (q_heads % kv_heads != 0 || q_heads / kv_heads > 16) return 0;
  if (static_cast<int64_t>(batch) * kv_heads > kMaxCounters) return 0;
  Shape s;
  if (shape_of(1, q_heads, kv_heads, &s) != B200KV_OK) return 0;
  return static_cast<size_t>(layout_of(s, batch, kv_heads).total);
}

// Does a chunk of at most max_q_len rows go through this file's kernel (given a workspace)?
bool kv4_streams_chunk(int batch, int64_t max_q_len, int q_heads, int kv_heads) {
  if (batch > 4096 || max_q_len > kChunkRows) return false;
  const int64_t cols = max_q_len * (q_heads / kv_heads);
  if (cols > kChunkColumns && cols * kv_heads * batch > kChunkWork) return false;
  Shape s;
  return shape_of(static_cast<int>(max_q_len), q_heads, kv_heads, &s) == B200KV_OK &&
         static_cast<int64_t>(batch) * kv_heads * s.blocks <= kMaxCounters;
}

size_t kv4_chunk_workspace_bytes(int batch, int64_t max_q_len, int q_heads, int kv_heads, int head_dim) {
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || max_q_len <= 0 || head_dim != kD) return 0;
  if (batch > 65535 || max_q_len > (int64_t{1} << 31) - 1 || q_heads % kv_heads != 0) return 0;
  if (!kv4_streams_chunk(batch, max_q_len, q_heads, kv_heads)) return kv4_split_workspace_bytes(batch, max_q_len, q_heads, kv_heads);
  Shape s;
  if (shape_of(static_cast<int>(max_q_len), q_heads, kv_heads, &s) != B200KV_OK) return 0;
  return static_cast<size_t>(layout_of(s, batch, kv_heads).total);
}

int kv4_paged_decode(const Kv4DecodeArgs& a, cudaStream_t stream) {
  if (a.batch < 0 || a.q_heads <= 0 || a.kv_heads <= 0 || a.max_seq_len < 0) return B200KV_EINVAL;
  if (a.batch == 0) return B200KV_OK;
  if (!a.q || !a.table || !a.seq_lens || !a.out || !a.workspace) return B200KV_EINVAL;
  if (a.table_kind != B200KV_TABLE_BLOCK && a.table_kind != B200KV_TABLE_TOKEN) return B200KV_EINVAL;
  if (a.head_dim != kD || a.page_size != kPS) return B200KV_EUNSUPPORTED;
  if (a.q_heads % a.kv_heads != 0) return B200KV_EUNSUPPORTED;
  if (a.q_heads / a.kv_heads > 16) return B200KV_EUNSUPPORTED;
  if (a.batch > 4096) return B200KV_ETOOLARGE;
  if (a.max_seq_len > (int64_t{1} << 30)) return B200KV_ETOOLARGE;
  if (a.table_rows <= 0 || a.table_cols <= 0 || a.table_row_stride < a.table_cols) return B200KV_EINVAL;
  if (a.row_ids == nullptr && a.batch > a.table_rows) return B200KV_EINVAL;
  if (a.max_seq_len > a.table_cols * (a.table_kind == B200KV_TABLE_BLOCK ? kPS : 1)) return B200KV_EINVAL;
  if (a.flags & ~B200KV_DECODE_SERIALIZED) return B200KV_EINVAL;
  int rc = kv4_check_pool(a.pool, a.pool_pages, a.page_stride_bytes, a.kv_heads);
  if (rc != B200KV_OK) return rc;
  if (misaligned(a.q, 16) || misaligned(a.out, 8) || misaligned(a.workspace, 16)) return B200KV_EALIGN;
  if (a.q_stride_b % 8 != 0 || a.q_stride_h % 8 != 0) return B200KV_EALIGN;
  if (a.out_stride_b % 4 != 0 || a.out_stride_h % 4 != 0) return B200KV_EALIGN;
  Shape s;
  rc = shape_of(1, a.q_heads, a.kv_heads, &s);
  if (rc != B200KV_OK) return rc;
  Kv4Params p{};
  p.q = static_cast<const __half*>(a.q);
  p.q_stride_t = a.q_stride_b;
  p.q_stride_h = a.q_stride_h;
  p.pool = static_cast<const uint8_t*>(a.pool);
  p.pool_pages = static_cast<int>(a.pool_pages);
  p.page_stride = a.page_stride_bytes;
  p.table = a.table;
  p.table_row_stride = a.table_row_stride;
  p.table_kind = a.table_kind;
  p.table_rows = a.table_rows;
  p.row_ids = a.row_ids;
  p.lens = a.seq_lens;
  p.lens_i64 = a.seq_lens_i64;
  p.batch = a.batch;
  p.kv_heads = a.kv_heads;
  p.max_seq_len = static_cast<int>(a.max_seq_len);
  p.max_q_len = 1;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  p.out = static_cast<__half*>(a.out);
  p.out_stride_t = a.out_stride_b;
  p.out_stride_h = a.out_stride_h;
  p.status = a.status;
  return run_decode(p, a.q_heads, s, a.workspace, a.workspace_bytes, a.max_seq_len,
                    (a.flags & B200KV_DECODE_SERIALIZED) == 0, stream);
}

// A chunk that is streamed (kv4_streams_chunk); the arguments have been checked (kv4_paged_prefill).
int kv4_paged_chunk(const Kv4PrefillArgs& k, cudaStream_t stream) {
  const PrefillArgs& a = k.args;
  if (misaligned(a.q, 16) || a.q_stride_t % 8 != 0 || a.q_stride_h % 8 != 0 || misaligned(k.workspace, 16)) return B200KV_EALIGN;
  Shape s;
  const int rc = shape_of(static_cast<int>(a.max_q_len), a.q_heads, a.kv_heads, &s);
  if (rc != B200KV_OK) return rc;
  Kv4Params p{};
  p.q = static_cast<const __half*>(a.q);
  p.q_stride_t = a.q_stride_t;
  p.q_stride_h = a.q_stride_h;
  p.pool = static_cast<const uint8_t*>(k.pool);
  p.pool_pages = static_cast<int>(k.pool_pages);
  p.page_stride = k.page_stride_bytes;
  p.table = a.table;
  p.table_row_stride = a.table_row_stride;
  p.table_kind = a.table_kind;
  p.table_rows = a.table_rows;
  p.row_ids = a.req_ids;
  p.lens = a.ctx_lens;
  p.q_lens = a.q_lens;
  p.q_start = a.q_start;
  p.lens_i64 = a.lens_i64;
  p.batch = a.batch;
  p.kv_heads = a.kv_heads;
  const int64_t width = a.table_cols * (a.table_kind == B200KV_TABLE_BLOCK ? kPS : 1);
  p.max_seq_len = static_cast<int>(width < (1 << 30) ? width : (1 << 30));
  p.max_q_len = static_cast<int>(a.max_q_len);
  p.total_q = a.total_q;
  p.scale_log2 = a.scale_log2;
  p.out = static_cast<__half*>(a.out);
  p.out_stride_t = a.out_stride_t;
  p.out_stride_h = a.out_stride_h;
  p.status = a.status;
  return run_decode(p, a.q_heads, s, k.workspace, k.workspace_bytes, p.max_seq_len, true, stream);
}

}  // namespace b200kv
