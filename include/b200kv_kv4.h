/*
 * b200kv — C ABI of the 4-bit paged KV cache ("kv4") for NVIDIA B200 (sm_100a).
 *
 * The cache holds the same pages, heads and slots as the fp16 pool of b200kv.h, at 4.5 bits per
 * element instead of 16: per page of 16 tokens and per head row one block of
 * B200KV_KV4_BLOCK_BYTES bytes,
 *
 *   pool[page][row]   row in [0, 2*kv_heads): K heads first, then V heads
 *     bytes    0..1023   16 token rows of 64 bytes of codes
 *     bytes 1024..1151   16 token rows of 4 fp16 scales
 *
 * A group is 32 neighbouring elements of a token's head row.  With d = 32 g + 8 j + n
 * (g, j < 4, n < 8) the code of (token-in-page t, element d) is nibble n/2 + 4 (n & 1) of the 32-bit
 * little-endian word at byte 64 t + 16 (j ^ ((t >> 1) & 3)) + 4 g, the scale of (t, g) is the fp16 at
 * byte 1024 + 8 t + 2 g, and the element stands for scale * (code - 8).
 *
 * Quantisation of a group of fp16 values x: amax = max |x|; scale = min(fp16(amax / 7), 9352) (so
 * that every value the cache stands for is a finite fp16 number); code - 8 = floor(x / scale + 1/2)
 * limited to [-8, 7], and 0 for every element when the scale rounds to zero.  The error of an
 * element is at most half a scale step, amax / 14, plus the rounding of the scale.  A group that
 * holds an infinity or a NaN gets a NaN scale: it reads back as NaN, never as a number.
 *
 * A block is contiguous and 16-byte aligned, the rows of a page follow one another, and pages are
 * page_stride_bytes apart (a multiple of 16, at least 2*kv_heads*B200KV_KV4_BLOCK_BYTES, below 2^31).  Slots, page
 * tables, lengths, status words, return codes, stream ordering and the programmatic-launch rule are
 * those of b200kv.h.  head_dim is 128 and page_size 16.
 *
 * The reference project has no 4-bit cache; the operators stand beside the fp16 ones it has
 * (lite_llama/kernels/update_kv_buffer.py:47-81, rope_emb.py:6-87, flashdecoding.py:295-342,
 * paged_chunk_flashattention.py:227-327).
 */
#ifndef B200KV_KV4_H_
#define B200KV_KV4_H_

#include "b200kv.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200KV_KV4_BLOCK_BYTES 1152
#define B200KV_KV4_GROUP 32

/*
 * Quantise and append: the rows of token i go to slot slots[i].
 *   k_values, v_values  fp16 [n_tokens, kv_heads, 128] each, row-contiguous inside a token, token
 *              strides in elements (multiples of 8), pointers 16-byte aligned.  For one combined
 *              [n_tokens, 2*kv_heads, 128] tensor pass v_values = k_values + kv_heads*128
 *   slots      int32 [n_tokens]; a slot outside the pool is skipped and sets B200KV_DEV_BAD_SLOT
 * n_tokens == 0 is a no-op.  Two tokens of one call may name the same slot only with identical
 * rows; otherwise what that slot holds afterwards is a mixture of the two.
 */
int b200kv_kv4_append(const void* k_values, const void* v_values, int64_t n_tokens,
                      int64_t k_tok_stride, int64_t v_tok_stride, const int32_t* slots,
                      void* pool, int64_t pool_pages, int64_t page_stride_bytes,
                      int kv_heads, int head_dim, int32_t* status, void* stream);

/*
 * The attention prologue in one launch: per-head RMSNorm of Q and K, rotary embedding of Q and K, and
 * the quantising append of K (normalised, rotated, rounded to fp16 as the fp16 pool would hold it)
 * and V.  Arguments as for b200kv_qk_norm_rope_append (b200kv.h); head_dim is 128.
 */
int b200kv_kv4_qk_norm_rope_append(const void* q, void* q_out, int64_t q_tok_stride,
                                   int64_t q_out_tok_stride, const void* kv, int64_t kv_tok_stride,
                                   const void* q_weight, const void* k_weight, float eps,
                                   const void* cos, const void* sin, int64_t cs_tok_stride,
                                   const int32_t* slots,
                                   void* pool, int64_t pool_pages, int64_t page_stride_bytes,
                                   int64_t n_tokens, int q_heads, int kv_heads, int head_dim,
                                   int32_t* status, void* stream);

/*
 * The rows the cache stands for: out[i] = fp16 rows of slot slots[i], rounded once.
 *   out        fp16 [n, 2*kv_heads, 128], row-contiguous inside a token, token stride
 *              out_tok_stride (a multiple of 8 elements), 16-byte aligned
 * A slot outside the pool gives a row of zeros and sets B200KV_DEV_BAD_SLOT.
 */
int b200kv_kv4_gather(const void* pool, int64_t pool_pages, int64_t page_stride_bytes,
                      const int32_t* slots, int64_t n, void* out, int64_t out_tok_stride,
                      int kv_heads, int head_dim, int32_t* status, void* stream);

/*
 * *id = the identifier of the stream capture that `stream` is recording, 0 when it records none.  A
 * caller that keeps a decode workspace gives every captured graph one of its own with it: two
 * graphs may be replayed at the same time.
 */
int b200kv_stream_capture_id(void* stream, uint64_t* id);

/*
 * Bytes of scratch of b200kv_kv4_paged_decode for `batch` sequences on the CURRENT device: arrival
 * counters (B200KV_DECODE_COUNTER_BYTES, zeroed once by the caller, left at zero by every call) and
 * split-KV partials, under the rules of b200kv_decode_workspace_bytes.  Returns 0 on bad input.
 */
size_t b200kv_kv4_decode_workspace_bytes(int batch, int q_heads, int kv_heads, int head_dim);

/*
 * Bytes of scratch that b200kv_kv4_paged_prefill can use for chunks of at most max_q_len rows on the CURRENT
 * device; 0 where it has no use for any (many long chunks), or on bad input.  Above 128 rows only the
 * number of 128-row tiles matters.
 */
size_t b200kv_kv4_chunk_workspace_bytes(int batch, int64_t max_q_len, int q_heads, int kv_heads, int head_dim);

/*
 * Paged flash-decoding over a kv4 pool: arguments, limits and meaning as for b200kv_paged_decode, with
 * the pool given as base, pages and page stride.  A token table's entries at page starts must be
 * multiples of 16; one that is not, or a page outside the pool, sets B200KV_DEV_BAD_PAGE and page 0 is
 * read in its place.  out strides are multiples of 4, q strides multiples of 8 elements, q 16-byte
 * aligned.
 */
int b200kv_kv4_paged_decode(const void* q, int64_t q_stride_b, int64_t q_stride_h,
                            const void* pool, int64_t pool_pages, int64_t page_stride_bytes,
                            const int32_t* table, int64_t table_row_stride, int table_kind,
                            int table_rows, int64_t table_cols,
                            const int32_t* row_ids,
                            const void* seq_lens, int seq_lens_i64,
                            int batch, int q_heads, int kv_heads, int head_dim, int page_size,
                            float scale, int64_t max_seq_len,
                            void* workspace, size_t workspace_bytes,
                            void* out, int64_t out_stride_b, int64_t out_stride_h,
                            int flags, int32_t* status, void* stream);

/*
 * Packed causal prefill with history over a kv4 pool: arguments and meaning as for
 * b200kv_paged_prefill (the chunk's own rows are already in the pool), table kinds BLOCK and TOKEN.
 * Lengths, rows and tables may come from the kernel launched immediately before.  A request whose chunk
 * is longer than max_q_len is skipped (B200KV_DEV_BAD_LENGTH).  A K or V group that reads as NaN reaches
 * the rows that see its token and no others.  scale_log2 is positive and finite.
 *   workspace  NULL, or scratch of b200kv_kv4_chunk_workspace_bytes() bytes under the rules of the decode
 *              workspace (the same buffer may serve both).  With it chunks of a few rows -- drafted tokens,
 *              the end of a prompt -- are streamed like a decode step instead of filling a small part of
 *              128-row tiles (then q is 16-byte aligned with strides that are multiples of 8), and where
 *              the query tiles leave most SMs empty their keys are cut into parts that are joined at the end
 */
int b200kv_kv4_paged_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h,
                             const void* pool, int64_t pool_pages, int64_t page_stride_bytes,
                             const int32_t* table, int64_t table_row_stride, int table_kind,
                             int table_rows, int64_t table_cols,
                             const int32_t* req_ids, const int32_t* q_start,
                             const void* ctx_lens, const void* q_lens, int lens_i64,
                             int batch, int64_t total_q, int64_t max_q_len,
                             int q_heads, int kv_heads, int head_dim, int page_size,
                             float scale_log2,
                             void* out, int64_t out_stride_t, int64_t out_stride_h,
                             void* workspace, size_t workspace_bytes,
                             int32_t* status, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* B200KV_KV4_H_ */
