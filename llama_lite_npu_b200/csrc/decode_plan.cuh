// What every paged split-KV decode kernel of this library shares: the flat page line and its cut into
// teams, the walk over a team's tiles, and the end of a piece (the four warps' state merged, the rows
// or the partial written, the partials of a sequence merged by the CTA that arrives last).
//
// A kernel that uses it runs kConsumerWarps warps that each hold an online-softmax state, numbers its
// CTAs team * kv_heads + head, and fills a merge buffer [warp][head_dim][ROWS] + (m, l) pairs at the
// end of a piece.  The scheduling itself is explained at the head of paged_decode.cu.
#pragma once

#include <climits>

#include "common.cuh"

namespace b200kv {

constexpr int kD = 128;
constexpr int kPS = 16;
constexpr int kTileTok = 64;
constexpr int kTilePages = kTileTok / kPS;
constexpr int kConsumerWarps = 4;
constexpr int kConsumerThreads = kConsumerWarps * 32;
constexpr int kScanThreads = 128;
constexpr int kMinPagesPerTeam = 4;   // a team is not worth launching for fewer pages
// The first bytes of the workspace hold one arrival counter per (sequence, KV head).
constexpr size_t kCounterBytes = B200KV_DECODE_COUNTER_BYTES;
constexpr int64_t kMaxCounters = static_cast<int64_t>(kCounterBytes / sizeof(unsigned));

// The part of a decode kernel's arguments that the functions below read.
struct DecodePlan {
  int table_rows;
  const int32_t* row_ids;
  const void* seq_lens;
  int seq_lens_i64;
  int batch, q_heads, kv_heads, group;
  int64_t max_seq_len;
  int nteams;
  int piece_cost;
  float* part_o;        // [nslots][kv_heads][ROWS][128]
  float* part_lse;      // [nslots][kv_heads][ROWS]
  unsigned* piece_ctr;  // [batch][kv_heads], zero between launches
  __half* out;
  int64_t out_stride_b, out_stride_h;
  int32_t* status;
};

// Length of sequence b as every part of the kernel sees it: clamped to [0, max_seq_len] (the
// host made sure max_seq_len fits the table's width), and 0 when its table row does not exist,
// so a stale length or request id can never turn into a read outside the table.
__device__ __forceinline__ int seq_len_checked(const DecodePlan& p, int b) {
  int64_t len = load_len(p.seq_lens, p.seq_lens_i64, b);
  if (len < 0) {
    set_status(p.status, B200KV_DEV_BAD_LENGTH);
    len = 0;
  } else if (len > p.max_seq_len) {
    set_status(p.status, B200KV_DEV_BAD_LENGTH);
    len = p.max_seq_len;
  }
  if (p.row_ids != nullptr) {
    const int row = __ldg(p.row_ids + b);
    if (row < 0 || row >= p.table_rows) {
      set_status(p.status, B200KV_DEV_BAD_LENGTH);
      len = 0;
    }
  }
  return static_cast<int>(len);
}
__device__ __forceinline__ int pages_of(int len) { return (len + kPS - 1) / kPS; }

// Number of teams that actually get work for NP pages (host launched `nteams`).
__device__ __forceinline__ int effective_teams(int nteams, int64_t np_total) {
  int64_t t = np_total / kMinPagesPerTeam;
  if (t > nteams) t = nteams;
  if (t < 1) t = 1;
  return static_cast<int>(t);
}
__device__ __forceinline__ int64_t team_begin(int team, int nteams_eff, int64_t total) {
  return (static_cast<int64_t>(team) * total) / nteams_eff;
}
// Team whose range holds position x (0 <= x < total).
__device__ __forceinline__ int team_of(int64_t x, int nteams_eff, int64_t total) {
  return static_cast<int>(((x + 1) * nteams_eff - 1) / total);
}

struct Tile {
  int b;        // sequence (batch position)
  int row;      // table row of that sequence
  int page0;    // first logical page of the tile
  int npages;   // pages in the tile (1..4)
  int ntok;     // valid tokens in the tile
  int np;       // pages of the whole sequence
  int len;      // tokens of the whole sequence
  int64_t units0;  // unit position of the sequence's start on the line
  bool first;   // first tile of its piece
  bool last;    // last tile of its piece
  bool whole;   // the piece is the whole sequence
};

// Walks the tiles of flat page range [flat, flat_end) in order.  Producer and consumer each
// own one walker; both visit exactly the same tiles.
struct Walker {
  int b;
  int64_t flat, flat_end;
  int page, piece_begin, piece_end, np, len, row;
  int kseq;   // non-empty sequences before b

  __device__ __forceinline__ void enter(const DecodePlan& p, int seq, int first_page) {
    b = seq;
    len = seq_len_checked(p, b);
    np = pages_of(len);
    row = p.row_ids ? __ldg(p.row_ids + b) : b;
    page = piece_begin = first_page;
    const int64_t room = flat_end - flat;
    piece_end = (np - first_page <= room) ? np : first_page + static_cast<int>(room);
  }
  __device__ __forceinline__ bool next(const DecodePlan& p, Tile& t) {
    if (flat >= flat_end) return false;
    if (page == piece_end) {
      int nb = b + 1;
      while (nb < p.batch && pages_of(seq_len_checked(p, nb)) == 0) ++nb;
      if (nb >= p.batch) {  // cannot happen for consistent lengths; stop rather than overrun
        flat = flat_end;
        return false;
      }
      ++kseq;
      enter(p, nb, 0);
    }
    t.b = b;
    t.row = row;
    t.page0 = page;
    t.npages = min(kTilePages, piece_end - page);
    const int tok_end = min(len, (page + t.npages) * kPS);
    t.ntok = tok_end - page * kPS;
    t.np = np;
    t.len = len;
    t.units0 = (flat - page) + static_cast<int64_t>(p.piece_cost) * kseq;
    t.first = (page == piece_begin);
    t.last = (page + t.npages == piece_end);
    t.whole = (piece_begin == 0 && piece_end == np);
    page += t.npages;
    flat += t.npages;
    return true;
  }
};
// A team's range of the page line.
struct TeamRange {
  int start_b, start_page, start_k;   // first sequence, its first page, non-empty sequences before it
  int64_t begin, end;                 // flat page positions
  int64_t units_total;
  int nteams_eff;
  bool any_empty;
  bool any;                           // false also for a range wholly inside a sequence's extra units
};

// Where does this team's range start and end?  Called by the whole CTA (it holds CTA barriers); `scan`
// is shared-memory scratch of 4 * (kScanThreads + 1) ints that may be reused after the call.
//
// Thread t < 128 sums the units (pages + piece_cost per non-empty sequence) and the non-empty
// sequences of [t*per, (t+1)*per); scans over the 128 sums give the totals and the chunk holding
// a boundary, then a short linear walk finds the sequence.
__device__ __forceinline__ TeamRange plan_team_range(const DecodePlan& p, int team, int tid, int* scan) {
  const int lane = tid & 31;
  const int warp = tid >> 5;
  int* scan_k = scan + kScanThreads + 1;   // non-empty sequences, same indexing
  int* scan_lo = scan_k + kScanThreads + 1;  // fewest / most pages of a non-empty sequence per thread,
  int* scan_hi = scan_lo + kScanThreads + 1; // reduced into entry [0]
  const int per = (p.batch + kScanThreads - 1) / kScanThreads;
  if (tid < kScanThreads) {
    int sum = 0, cnt = 0, lo_np = INT_MAX, hi_np = 0;
    const int lo = tid * per;
    const int hi = min(p.batch, lo + per);
    for (int b = lo; b < hi; ++b) {
      const int np = pages_of(seq_len_checked(p, b));
      sum += np + (np > 0 ? p.piece_cost : 0);
      cnt += np > 0;
      if (np > 0) {
        lo_np = min(lo_np, np);
        hi_np = max(hi_np, np);
      }
    }
    scan[tid + 1] = sum;
    scan_k[tid + 1] = cnt;
    scan_lo[tid + 1] = lo_np;
    scan_hi[tid + 1] = hi_np;
    if (tid == 0) scan[0] = scan_k[0] = 0;
  }
  __syncthreads();
  if (warp == 2 || warp == 3) {  // fewest / most pages over the 128 entries
    int* arr = warp == 2 ? scan_lo : scan_hi;
    int v = arr[1 + lane * 4];
#pragma unroll
    for (int i = 1; i < 4; ++i) v = warp == 2 ? min(v, arr[1 + lane * 4 + i]) : max(v, arr[1 + lane * 4 + i]);
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) {
      const int o = __shfl_xor_sync(0xffffffffu, v, d);
      v = warp == 2 ? min(v, o) : max(v, o);
    }
    if (lane == 0) arr[0] = v;
  }
  if (warp < 2) {  // inclusive scans of [1..128] by one warp each, 4 values per lane
    int* arr = warp == 0 ? scan : scan_k;
    int v[4];
    int run = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      run += arr[1 + lane * 4 + i];
      v[i] = run;
    }
    int incl = run;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int o = __shfl_up_sync(0xffffffffu, incl, d);
      if (lane >= d) incl += o;
    }
    const int excl = incl - run;
#pragma unroll
    for (int i = 0; i < 4; ++i) arr[1 + lane * 4 + i] = v[i] + excl;
  }
  __syncthreads();
  const int64_t units_total = scan[kScanThreads];
  const int nonempty_total = scan_k[kScanThreads];
  const int64_t np_total = units_total - static_cast<int64_t>(p.piece_cost) * nonempty_total;
  int nteams_eff = effective_teams(p.nteams, np_total);
  // Sequences of one length whose count divides into about as many groups as there are teams: one
  // team per group of k whole sequences.  Every piece is then a whole sequence — nothing is
  // published, counted or merged — at the price of leaving up to a quarter of the CTA slots empty,
  // which the streaming rate survives.
  if (nonempty_total > 0 && scan_lo[0] == scan_hi[0]) {
    const int k = (nonempty_total + p.nteams - 1) / p.nteams;   // sequences per team
    const int groups = nonempty_total / k;
    if (groups * k == nonempty_total && 4 * groups >= 3 * p.nteams) nteams_eff = groups;
  }
  const bool any_empty = nonempty_total < p.batch;

  // Unit position x -> (sequence, page inside it, flat page index).  Positions inside a sequence's
  // piece_cost extra units map to its first page.
  int start_b = 0, start_page = 0, start_k = 0;
  int64_t r_begin = 0, r_end = 0;
  if (np_total > 0 && team < nteams_eff) {
#pragma unroll 1
    for (int side = 0; side < 2; ++side) {
      const int64_t x = team_begin(team + side, nteams_eff, units_total);
      int64_t flat = np_total;
      int sb = 0, sp = 0, sk = 0;
      if (x < units_total) {
        int lo = 0, hi = kScanThreads - 1;   // last chunk whose unit prefix <= x
        while (lo < hi) {
          const int mid = (lo + hi + 1) >> 1;
          if (scan[mid] <= x) lo = mid; else hi = mid - 1;
        }
        int64_t acc = scan[lo];
        sk = scan_k[lo];
        int64_t pages_before = acc - static_cast<int64_t>(p.piece_cost) * sk;
        int b = lo * per;
        for (; b < p.batch; ++b) {   // ends before the batch does when the lengths are consistent
          const int np = pages_of(seq_len_checked(p, b));
          const int w = np + (np > 0 ? p.piece_cost : 0);
          if (acc + w > x) break;
          acc += w;
          pages_before += np;
          sk += np > 0;
        }
        if (b < p.batch) {
          const int64_t o = x - acc - p.piece_cost;
          sb = b;
          sp = o > 0 ? static_cast<int>(o) : 0;
          flat = pages_before + sp;
        }
      }
      if (side == 0) {
        start_b = sb;
        start_page = sp;
        start_k = sk;
        r_begin = flat;
      } else {
        r_end = flat;
      }
    }
  }
  __syncthreads();  // the scratch may be reused; barrier inits of the caller are visible
  TeamRange r;
  r.start_b = start_b;
  r.start_page = start_page;
  r.start_k = start_k;
  r.begin = r_begin;
  r.end = r_end;
  r.units_total = units_total;
  r.nteams_eff = nteams_eff;
  r.any_empty = any_empty;
  r.any = r_end > r_begin;
  return r;
}

// Programmatic dependent launch, used by every kernel of this library the same way: whatever
// a kernel does BEFORE this call may overlap the tail of the previous kernel in the stream, so
// it must only read launch metadata (lengths, row ids, page table) that an earlier, already
// completed operation produced.  Every thread of every CTA makes this call on every path, early
// exits included, and a kernel releases its own dependents only after its own wait: when a
// dependent's prologue runs, everything two or more kernels back has completed.
__device__ __forceinline__ void pdl_wait_then_trigger() {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();
}
__device__ __forceinline__ void consumer_bar() {
  asm volatile("bar.sync 1, %0;\n" ::"n"(kConsumerThreads) : "memory");
}

// Merge the `npieces` partials of (sequence b, KV head `head`) held in slots t_first + b ...:
// out = sum_p 2^(lse_p - M) o_p / sum_p 2^(lse_p - M).  Run by the 128 consumer threads of the CTA
// that delivered the last partial; everything it reads was written by other CTAs, so the loads go
// past L1, and the whole merge costs about three memory round trips whatever the piece count:
//   A. thread (piece j, row r) fetches lse[j][r] (128 / ROWS pieces per sweep) into shared memory
//      and the row maxima are reduced with shuffles and one pass through shared memory;
//   B. the same threads turn their entries into weights 2^(lse - M) in place and reduce the row sums;
//   C. thread = output column: the partial outputs are loaded kMergeBatch pieces at a time, every
//      load of a batch issued before any arithmetic (the first batch before step A even), and
//      weighted with the shared-memory weights.
// `wbuf` (npieces * ROWS floats) and `red` (2 * 4 * ROWS floats) are shared-memory scratch that
// nobody else uses between the surrounding consumer barriers.
constexpr int kMergeBatch = 6;
template <int ROWS>
__device__ __forceinline__ void merge_pieces(const DecodePlan& p, int b, int head, int t_first,
                                             int npieces, int tid, float* wbuf, float* red) {
  constexpr int kPerSweep = kConsumerThreads / ROWS;
  const int my_r = tid % ROWS;
  const int lane = tid & 31;
  const int warp = tid >> 5;
  auto slot_of = [&](int pc) { return (static_cast<int64_t>(t_first + pc) + b) * p.kv_heads + head; };
  auto load_batch = [&](float (&ov)[kMergeBatch][8], int r0, int p0) {
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      if (p0 + j < npieces) {   // the same for every thread of the CTA
        const int64_t slot = slot_of(p0 + j);
#pragma unroll
        for (int r = 0; r < 8; ++r) ov[j][r] = __ldcg(p.part_o + (slot * ROWS + r0 + r) * kD + tid);
      } else {
#pragma unroll
        for (int r = 0; r < 8; ++r) ov[j][r] = 0.f;
      }
    }
  };
  // The first batch of partial outputs needs no weights to be requested: its loads are issued
  // now and are in flight under steps A and B.
  float first[kMergeBatch][8];
  load_batch(first, 0, 0);
  // ---- A: log-sum-exp values -> shared memory, row maxima --------------------------------------
  float m = -INFINITY;
  for (int j = tid / ROWS; j < npieces; j += kPerSweep) {
    const float v = __ldcg(p.part_lse + slot_of(j) * ROWS + my_r);
    wbuf[j * ROWS + my_r] = v;
    m = fmaxf(m, v);
  }
#pragma unroll
  for (int d = ROWS; d < 32; d <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
  if (lane < ROWS) red[warp * ROWS + lane] = m;
  consumer_bar();
  const float M = fmaxf(fmaxf(red[my_r], red[ROWS + my_r]), fmaxf(red[2 * ROWS + my_r], red[3 * ROWS + my_r]));
  // ---- B: weights in place, row sums --------------------------------------------------------------
  float sum = 0.f;
  for (int j = tid / ROWS; j < npieces; j += kPerSweep) {
    const float w = fast_exp2(wbuf[j * ROWS + my_r] - M);
    wbuf[j * ROWS + my_r] = w;
    sum += w;
  }
#pragma unroll
  for (int d = ROWS; d < 32; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
  float* red_sum = red + kConsumerWarps * ROWS;
  if (lane < ROWS) red_sum[warp * ROWS + lane] = sum;
  consumer_bar();
  // ---- C: weighted sum of the partial outputs, thread = column -----------------------------------
  auto add_batch = [&](float (&acc)[8], const float (&ov)[kMergeBatch][8], int r0, int p0) {
#pragma unroll
    for (int j = 0; j < kMergeBatch; ++j) {
      if (p0 + j < npieces) {
        const float4 w0 = *reinterpret_cast<const float4*>(wbuf + (p0 + j) * ROWS + r0);
        const float4 w1 = *reinterpret_cast<const float4*>(wbuf + (p0 + j) * ROWS + r0 + 4);
        acc[0] += w0.x * ov[j][0]; acc[1] += w0.y * ov[j][1]; acc[2] += w0.z * ov[j][2]; acc[3] += w0.w * ov[j][3];
        acc[4] += w1.x * ov[j][4]; acc[5] += w1.y * ov[j][5]; acc[6] += w1.z * ov[j][6]; acc[7] += w1.w * ov[j][7];
      }
    }
  };
#pragma unroll 1
  for (int r0 = 0; r0 < ROWS && r0 < p.group; r0 += 8) {
    float acc[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) acc[r] = 0.f;
    if (r0 == 0) add_batch(acc, first, 0, 0);
#pragma unroll 1
    for (int p0 = (r0 == 0 ? kMergeBatch : 0); p0 < npieces; p0 += kMergeBatch) {
      float ov[kMergeBatch][8];
      load_batch(ov, r0, p0);
      add_batch(acc, ov, r0, p0);
    }
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      if (r0 + r < p.group) {
        const float L = red_sum[r0 + r] + red_sum[ROWS + r0 + r] + red_sum[2 * ROWS + r0 + r] + red_sum[3 * ROWS + r0 + r];
        p.out[static_cast<int64_t>(b) * p.out_stride_b +
              (static_cast<int64_t>(head) * p.group + r0 + r) * p.out_stride_h + tid] =
            __float2half_rn(acc[r] / L);
      }
    }
  }
}
// The end of a piece, run by the kConsumerThreads threads after every warp has written its unnormalised
// output and its (m, l) pairs to the merge buffer: the warps' states are merged, the rows (whole
// sequence) or the partial are written, and the partials of a sequence are merged by the CTA that
// arrives last.  `seen_arrivals` (thread 0): the piece counter as read when the piece's last tile began.
template <int ROWS>
__device__ __forceinline__ void emit_piece(const DecodePlan& p, const Tile& t, int team, int head, int tid,
                                           int nteams_eff, int64_t units_total, unsigned seen_arrivals,
                                           float* merge_o, float* merge_ml, int* arrival) {
        // (thread 0, partial pieces) had every other piece of the sequence arrived when this piece's
        // last tile began?  The flag rides on the barrier below.
        const int64_t u0 = t.units0 + p.piece_cost;
        const int t_first = team_of(u0, nteams_eff, units_total);
        const int t_last = team_of(u0 + t.np - 1, nteams_eff, units_total);
        const int npieces = t_last - t_first + 1;
        if (tid == 0 && !t.whole) {
          const bool others_in = seen_arrivals == static_cast<unsigned>(npieces - 1);
          if (others_in) __threadfence();   // acquire: their published rows come before what follows
          arrival[2] = others_in ? 1 : 0;
        }
        consumer_bar();
        const int64_t slot = (static_cast<int64_t>(team) + t.b) * p.kv_heads + head;
        // Thread = output column; its ROWS values of a warp's O are contiguous in the merge buffer
        // (vector loads), the (m, l) pairs are broadcast loads, and all rows are merged in registers.
  #pragma unroll 1
        for (int r0 = 0; r0 < ROWS; r0 += 8) {   // eight rows at a time keeps the registers modest
          float M[8], L[8], acc[8];
          float mw[kConsumerWarps][8], lw[kConsumerWarps][8];
  #pragma unroll
          for (int r = 0; r < 8; ++r) {
            M[r] = -INFINITY;
            L[r] = acc[r] = 0.f;
          }
  #pragma unroll
          for (int w = 0; w < kConsumerWarps; ++w) {
  #pragma unroll
            for (int r2 = 0; r2 < 4; ++r2) {
              const float4 v = *reinterpret_cast<const float4*>(merge_ml + (w * ROWS + r0 + 2 * r2) * 2);
              mw[w][2 * r2] = v.x;
              lw[w][2 * r2] = v.y;
              mw[w][2 * r2 + 1] = v.z;
              lw[w][2 * r2 + 1] = v.w;
              M[2 * r2] = fmaxf(M[2 * r2], v.x);
              M[2 * r2 + 1] = fmaxf(M[2 * r2 + 1], v.z);
            }
          }
  #pragma unroll
          for (int w = 0; w < kConsumerWarps; ++w) {
            const float4 v0 = *reinterpret_cast<const float4*>(merge_o + (w * kD + tid) * ROWS + r0);
            const float4 v1 = *reinterpret_cast<const float4*>(merge_o + (w * kD + tid) * ROWS + r0 + 4);
            const float ov[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
  #pragma unroll
            for (int r = 0; r < 8; ++r) {
              const float sc = (mw[w][r] == -INFINITY) ? 0.f : fast_exp2(mw[w][r] - M[r]);
              L[r] += sc * lw[w][r];
              acc[r] += sc * ov[r];
            }
          }
  #pragma unroll
          for (int r = 0; r < 8; ++r) {
            if (r0 + r < p.group) {
              const float val = acc[r] / L[r];
              if (t.whole) {
                p.out[static_cast<int64_t>(t.b) * p.out_stride_b +
                      (static_cast<int64_t>(head) * p.group + r0 + r) * p.out_stride_h + tid] =
                    __float2half_rn(val);
              } else {
                p.part_o[(slot * ROWS + r0 + r) * kD + tid] = val;
                if (tid == 0) p.part_lse[slot * ROWS + r0 + r] = M[r] + log2f(L[r]);
              }
            }
          }
        }
        if (!t.whole) {
          // A partial: publish it, count it, and merge the sequence if it was the last one to arrive.
          // The counter wraps to zero on the last arrival, so it needs no reset between launches.
          unsigned* ctr = p.piece_ctr + static_cast<int64_t>(t.b) * p.kv_heads + head;
          if (arrival[2] != 0) {
            // Everybody else had arrived before this piece's last tile: nobody waits for this
            // partial but this CTA itself, which reads it back through L2 in the merge (a barrier,
            // not a fence, orders that).  The count still has to wrap the counter to zero.
            consumer_bar();
            if (tid == 0) atomicInc(ctr, static_cast<unsigned>(npieces - 1));
            merge_pieces<ROWS>(p, t.b, head, t_first, npieces, tid, merge_o, merge_ml);
          } else {
            __threadfence();
            consumer_bar();
            if (tid == 0) {
              const unsigned old = atomicInc(ctr, static_cast<unsigned>(npieces - 1));
              const bool last_arrival = old == static_cast<unsigned>(npieces - 1);
              arrival[0] = last_arrival ? npieces : 0;
              // Acquire side of the hand-over, paid by the merging CTA only: this thread saw the other
              // pieces' counts; the fence orders their published rows before everything that follows,
              // and the named barrier below extends that to the other 127 threads.
              if (last_arrival) __threadfence();
            }
            consumer_bar();
            if (arrival[0] > 0) merge_pieces<ROWS>(p, t.b, head, t_first, npieces, tid, merge_o, merge_ml);
          }
        }
}

}  // namespace b200kv
