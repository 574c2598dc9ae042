/*
 * nvfp4kv_serving -- C ABI of the serving operators around the NVFP4 paged cache: the tables of a
 * step, rotary positions on one axis or several, rotated keys into the rope side-pool, attention
 * of a ragged chunk of new tokens over the paged pool, whole or in a window, and the upkeep of the
 * cache's pages.  Same library (libnvfp4kv.so),
 * conventions, return codes and device error bits as nvfp4kv.h.  The reference has none of
 * these: its model is NoPE and vLLM schedules its prefill and its pages.
 */
#ifndef NVFP4KV_SERVING_H_
#define NVFP4KV_SERVING_H_

#include "nvfp4kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* a third element type, for nvfp4kv_rope */
#define NVFP4KV_DTYPE_F32 2
/* caches one page call can name */
#define NVFP4KV_MAX_CACHES 8
/* position axes of one rotation, and the widest rotated part that several axes can share */
#define NVFP4KV_MAX_AXES 4
#define NVFP4KV_MAX_AXES_DIM 256
/* a block table's entry for a page that nvfp4kv_trim_pages gave back behind a window */
#define NVFP4KV_PAGE_TRIMMED (-2)

/*
 * Rotary positions.  x: [num_tokens, num_heads, head_dim] of `dtype` (bf16, fp16 or fp32) with
 * element strides (x_stride_t, x_stride_h) and a contiguous last dim.  Dims [rope_offset,
 * rope_offset + rotary_dim) of every head of token t are rotated by the angles of
 * positions[t], the others copied:
 *   interleaved: pairs (2i, 2i + 1);  else: pairs (i, i + rotary_dim / 2)
 *   (a, b) -> (a c - b s, b c + a s),  c = cos_sin[pos][i], s = cos_sin[pos][rotary_dim / 2 + i]
 * `inverse` rotates by the negative angles: the gradient with respect to x of the forward call.
 * cos_sin: fp32 [max_positions, rotary_dim] (cos | sin; scaled frequencies and attention factors
 * are in it).  Arithmetic in fp32, one rounding to dtype.  out: same shape and dtype, its own
 * strides; it may be x itself (then only the rotated dims are touched), otherwise the two must
 * not overlap.  A position < 0 or >= max_positions leaves its token unrotated and sets
 * NVFP4KV_DEVERR_BAD_INDEX.  num_tokens == 0 is a no-op.
 */
int nvfp4kv_rope(const void* x, int dtype, int64_t num_tokens, int num_heads, int head_dim,
                 int64_t x_stride_t, int64_t x_stride_h, const void* positions, int pos_dtype,
                 const float* cos_sin, int64_t max_positions, int rotary_dim, int rope_offset,
                 int interleaved, int inverse, void* out, int64_t out_stride_t, int64_t out_stride_h,
                 int32_t* err_flag, nvfp4kv_stream_t stream);

/*
 * The rope part of a step in one launch: k_pe [num_tokens, >= 64] bf16 rotated by the angles of
 * positions[t] into rope_pool[slot[t]] (as nvfp4kv_append_rope: slot < 0 skips, slot >=
 * pool_rows skips and sets NVFP4KV_DEVERR_BAD_SLOT), and, where q_pe is given, the 64 rope dims
 * of the queries q_pe [num_tokens, num_heads, >= 64] bf16 rotated into q_out (same shape, its
 * own strides; q_out may be q_pe).  cos_sin, positions and the pairing as in nvfp4kv_rope with
 * rotary_dim 64.
 */
int nvfp4kv_append_rope_rotated(const void* k_pe, int64_t num_tokens, int64_t k_stride, void* rope_pool,
                                int64_t pool_rows, const void* slot_mapping, int slot_dtype,
                                const void* positions, int pos_dtype, const float* cos_sin,
                                int64_t max_positions, int interleaved, const void* q_pe, int num_heads,
                                int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t qo_stride_t,
                                int64_t qo_stride_h, int32_t* err_flag, nvfp4kv_stream_t stream);

/*
 * The two above with positions on several axes (time, height and width of an image's or a video's
 * tokens): positions [num_axes, num_tokens] with stride positions_stride between axes, and
 * pair_axes, a host array of rotary_dim / 2 axis numbers: pair i turns by row
 * positions[pair_axes[i]][t] of the table.  1 <= num_axes <= NVFP4KV_MAX_AXES, rotary_dim <=
 * NVFP4KV_MAX_AXES_DIM.  A token with a position outside the table on any axis is left unrotated
 * and sets NVFP4KV_DEVERR_BAD_INDEX.
 */
int nvfp4kv_rope_axes(const void* x, int dtype, int64_t num_tokens, int num_heads, int head_dim,
                      int64_t x_stride_t, int64_t x_stride_h, const void* positions, int pos_dtype,
                      int64_t positions_stride, int num_axes, const uint8_t* pair_axes,
                      const float* cos_sin, int64_t max_positions, int rotary_dim, int rope_offset,
                      int interleaved, int inverse, void* out, int64_t out_stride_t, int64_t out_stride_h,
                      int32_t* err_flag, nvfp4kv_stream_t stream);
int nvfp4kv_append_rope_rotated_axes(const void* k_pe, int64_t num_tokens, int64_t k_stride, void* rope_pool,
                                     int64_t pool_rows, const void* slot_mapping, int slot_dtype,
                                     const void* positions, int pos_dtype, int64_t positions_stride,
                                     int num_axes, const uint8_t* pair_axes, const float* cos_sin,
                                     int64_t max_positions, int interleaved, const void* q_pe, int num_heads,
                                     int64_t q_stride_t, int64_t q_stride_h, void* q_out, int64_t qo_stride_t,
                                     int64_t qo_stride_h, int32_t* err_flag, nvfp4kv_stream_t stream);

/*
 * Causal MLA attention of a ragged batch of new tokens over the paged pool (their own rows
 * already appended).  Sequence b has the query tokens [cu_seqlens_q[b], cu_seqlens_q[b + 1]) of
 * q, which are the last of its seq_lens[b] tokens: query i of n sees tokens t <= seq_lens[b] -
 * n + i.  Any mix of single tokens and long chunks; n may be 0.
 * q: bf16 [total_q, num_heads, head_dim_qk] with element strides (q_stride_t, q_stride_h),
 *    multiples of 8, 16-byte aligned.  The first 512 dims meet the latent rows; with rope_pool
 *    (the rope side-pool, may be NULL) dims [512, 576) meet its rows.
 * tables [batch, >= ceil(max_seq_len / page_size)] page ids (row stride tables_stride).
 *    seq_lens and cu_seqlens_q stay on the device; max_q_len and max_seq_len bound them.  What
 *    goes past them sets NVFP4KV_DEVERR_SEQ_LEN: a sequence ends at max_seq_len tokens (and at
 *    2^31 - 4,096), and of more than max_q_len new tokens only the first max_q_len get their rows of
 *    out and lse.
 * out: bf16 [total_q, num_heads, 512] with strides (out_stride_t, out_stride_h), multiples of
 *    8, 16-byte aligned: softmax(bmm1_scale * q.k) . v * bmm2_scale.  A row that sees no token
 *    is zeros.  lse (may be NULL): fp32 [total_q, num_heads], the natural log of the sum of
 *    exp(bmm1_scale * q.k), -inf for such a row.
 * Tokens on a missing page (id outside the pool) are masked and set NVFP4KV_DEVERR_BAD_PAGE.
 * A hidden token never reaches a row, whatever its bytes hold.
 * Rows of out and lse that belong to no sequence (those from cu_seqlens_q[batch] on) or to a new
 * token past max_q_len are not written; every other row is.
 * pool_rows is a multiple of page_size below 2^31, page_size a power of two up to 4096.
 * workspace: nvfp4kv_mla_prefill_workspace_size() bytes, 256-byte aligned: a dequantised image
 *    of the contexts (1,152 bytes a token, max_seq_len for each sequence, at most 1 GiB or one
 *    sequence's; a larger batch runs in groups of sequences) and partial results.  Give the
 *    batch's own max_q_len and max_seq_len: they size both the workspace and the grid.
 */
int nvfp4kv_mla_prefill(const void* q, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* pool,
                        int64_t pool_rows, const void* rope_pool, const int32_t* tables,
                        int64_t tables_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                        int batch, int total_q, int num_heads, int head_dim_qk, int kv_lora_rank,
                        int page_size, int max_q_len, int max_seq_len, float bmm1_scale,
                        float bmm2_scale, void* out, int64_t out_stride_t, int64_t out_stride_h,
                        float* lse, void* workspace, size_t workspace_bytes, int32_t* err_flag,
                        nvfp4kv_stream_t stream);

/* Workspace bytes nvfp4kv_mla_prefill needs for this shape on the current device. */
int nvfp4kv_mla_prefill_workspace_size(int batch, int total_q, int num_heads, int max_q_len,
                                       int max_seq_len, size_t* bytes);

/*
 * The same with a sliding window: the query at position p sees the tokens t <= p with t > p -
 * window, and those with t < sinks.  window >= 1, sinks >= 0.  Tokens that no query of the call
 * sees are never read, and their pages may be missing (nvfp4kv_trim_pages gives them back) without
 * an error.  The workspace holds images of what the windows cover, not of whole contexts.
 * Where there are images (many query rows), q is used as it is, without the power of two that each row
 * is scaled by elsewhere: queries past 2^106 can pass fp32's range there.
 */
int nvfp4kv_mla_prefill_window(const void* q, int64_t q_stride_t, int64_t q_stride_h, const uint8_t* pool,
                               int64_t pool_rows, const void* rope_pool, const int32_t* tables,
                               int64_t tables_stride, const int32_t* cu_seqlens_q, const int32_t* seq_lens,
                               int batch, int total_q, int num_heads, int head_dim_qk, int kv_lora_rank,
                               int page_size, int max_q_len, int max_seq_len, int window, int sinks,
                               float bmm1_scale, float bmm2_scale, void* out, int64_t out_stride_t,
                               int64_t out_stride_h, float* lse, void* workspace, size_t workspace_bytes,
                               int32_t* err_flag, nvfp4kv_stream_t stream);

/* Workspace bytes nvfp4kv_mla_prefill_window needs for this shape on the current device. */
int nvfp4kv_mla_prefill_window_workspace_size(int batch, int total_q, int num_heads, int max_q_len,
                                              int max_seq_len, int window, int sinks, size_t* bytes);

/*
 * Page upkeep.  A cache is a set of pools that share page ids (latent rows, rope rows, indexer
 * rows ...): caches[c] (a host array of device pointers, num_caches <= NVFP4KV_MAX_CACHES) is
 * [num_pages] pages of page_bytes[c] bytes, a multiple of page_size.  block_tables [num_slots,
 * >= table_width] int32 page ids, -1 padded (row stride tables_stride); seq_lens [num_slots]
 * tokens of each slot; ref_counts [num_pages] int32, how many tables name a page, 0 = free.
 * Everything is on the device and in stream order; the results do not depend on the order in
 * which blocks run.
 */

/* Pages src[k] -> dst[k] of every cache, k < num_pairs.  A pair with a negative id is skipped;
 * an id >= num_pages skips the pair and sets NVFP4KV_DEVERR_BAD_PAGE.  No page may be both a
 * source and a destination, nor a destination twice. */
int nvfp4kv_copy_pages(const void* const* caches, const int64_t* page_bytes, int num_caches,
                       int64_t num_pages, const int32_t* src, const int32_t* dst, int64_t num_pairs,
                       int32_t* err_flag, nvfp4kv_stream_t stream);

/* Empties slots[k] (k < num): every page its table names loses one reference, its table row
 * becomes -1 and its seq_len 0.  A slot outside [0, num_slots) is skipped with
 * NVFP4KV_DEVERR_BAD_SLOT; a page outside the pool, or one that has no reference left, sets
 * NVFP4KV_DEVERR_BAD_PAGE (counts stay >= 0). */
int nvfp4kv_free_pages(int32_t* block_tables, int64_t tables_stride, int table_width, int64_t num_slots,
                       int32_t* seq_lens, const int32_t* slots, int num, int32_t* ref_counts,
                       int64_t num_pages, int32_t* err_flag, nvfp4kv_stream_t stream);

/* Makes slot dst[k] a copy of the sequence in slot src[k] (k < num; a parent may be named often):
 * its full pages are shared (one reference more each) and a partly filled last page is copied,
 * its filled rows only, into the lowest free pages in order of k.  dst[k] must be empty
 * (seq_len 0) and named once; a fork with a bad or non-empty slot is skipped with
 * NVFP4KV_DEVERR_BAD_SLOT (of equal dst the first counts), one that finds no free page is
 * skipped with NVFP4KV_DEVERR_CAPACITY, a missing page of the parent stays missing and sets
 * NVFP4KV_DEVERR_BAD_PAGE (one trimmed by a window stays so without).  workspace: 3 * num int32. */
int nvfp4kv_fork_pages(const void* const* caches, const int64_t* page_bytes, int num_caches, int page_size,
                       int32_t* block_tables, int64_t tables_stride, int table_width, int64_t num_slots,
                       int32_t* seq_lens, const int32_t* src, const int32_t* dst, int num,
                       int32_t* ref_counts, int64_t num_pages, int32_t* workspace,
                       int64_t workspace_ints, int32_t* err_flag, nvfp4kv_stream_t stream);

/*
 * The tables of a step.  Request k (k < num) appends new_lens[k] tokens to the sequence in
 * slots[k], whose length before the step is lens[k], or its seq_len where lens is NULL; lens[k] <
 * seq_len takes the tokens past it back (drafts that were not accepted) and gives their pages
 * back first.  In order of k every page that begins in the new tokens is the lowest free one
 * (ref_count 0 becomes 1); seq_lens[slots[k]] becomes the length with them.  For the step's kernels:
 *   cu_seqlens_q [num + 1], out_lens [num]: the requests' first tokens, their lengths with the new ones
 *   out_tables   [num, table_width]: their table rows
 *   slot_mapping [num_tokens] int64, positions [num_tokens] int32: of every new token; -1 and 0
 *                from cu_seqlens_q[num] on (the padding of a captured batch)
 * A request is skipped, with no tokens, length 0 and a table of -1, if its slot is bad or named
 * by an earlier request (NVFP4KV_DEVERR_BAD_SLOT), if a length is negative or lens[k] is above
 * seq_len (NVFP4KV_DEVERR_SEQ_LEN), if the page that its first new token falls into is missing or
 * shared (NVFP4KV_DEVERR_BAD_PAGE), if table_width pages cannot hold it, if the tokens of the
 * requests up to it pass num_tokens, or if it needs pages and those of the requests up to it are
 * more than there are (NVFP4KV_DEVERR_CAPACITY; in the last two cases its tokens past lens[k] are
 * still taken back).  Table entries past a sequence's end must name no page.
 * workspace: nvfp4kv_extend_workspace_ints() int32.
 */
int nvfp4kv_extend_pages(int32_t* block_tables, int64_t tables_stride, int table_width, int64_t num_slots,
                         int32_t* seq_lens, const int32_t* slots, const int32_t* new_lens, const int32_t* lens,
                         int num, int page_size, int32_t* ref_counts, int64_t num_pages, int64_t num_tokens,
                         int64_t* slot_mapping, int32_t* positions, int32_t* cu_seqlens_q, int32_t* out_lens,
                         int32_t* out_tables, int32_t* workspace, int64_t workspace_ints, int32_t* err_flag,
                         nvfp4kv_stream_t stream);

/* int32 workspace size of nvfp4kv_extend_pages. */
int nvfp4kv_extend_workspace_ints(int num, int64_t num_slots, int64_t num_pages, int64_t* ints);

/* Gives back pages of the sequences in slots[k] (k < num) that no later step reads: with window >
 * 0 those whose tokens are all at or past `sinks` and behind the window of the next token, at
 * position seq_len (their entries become NVFP4KV_PAGE_TRIMMED), and those that begin at or past
 * seq_len (-1).  Where tokens may still be taken back or asked for again, window has to be longer by
 * their number.
 * Bad slots and pages as in nvfp4kv_free_pages. */
int nvfp4kv_trim_pages(int32_t* block_tables, int64_t tables_stride, int table_width, int64_t num_slots,
                       const int32_t* seq_lens, const int32_t* slots, int num, int page_size, int window,
                       int sinks, int32_t* ref_counts, int64_t num_pages, int32_t* err_flag,
                       nvfp4kv_stream_t stream);

/* Moves the pages in use to the front: with n = pages whose ref_count is > 0, the k-th of them
 * past page n goes to the k-th free page before it, in every cache.  out_tables (own row stride)
 * and out_ref_counts receive the tables and counts that go with it (they may be block_tables
 * and ref_counts themselves), *num_live n.  A table entry that names no page in use becomes -1
 * and sets NVFP4KV_DEVERR_BAD_PAGE; NVFP4KV_PAGE_TRIMMED stays.  workspace:
 * nvfp4kv_compact_workspace_ints() int32. */
int nvfp4kv_compact_pages(const void* const* caches, const int64_t* page_bytes, int num_caches,
                          const int32_t* block_tables, int64_t tables_stride, int table_width,
                          int64_t num_slots, const int32_t* ref_counts, int64_t num_pages,
                          int32_t* out_tables, int64_t out_tables_stride, int32_t* out_ref_counts,
                          int32_t* num_live, int32_t* workspace, int64_t workspace_ints,
                          int32_t* err_flag, nvfp4kv_stream_t stream);

/* int32 workspace size of nvfp4kv_compact_pages. */
int nvfp4kv_compact_workspace_ints(int64_t num_pages, int64_t* ints);

/* An entry above that takes a stream, by its number, with its arguments in `args`, 8 bytes each and in
 * order: int64 for numbers, pointers and streams, double for floats.  For callers whose foreign calls
 * convert one argument at a time.  nvfp4kv_packed_entry gives an entry's number and how many
 * arguments it has; they do not change while the library is loaded. */
int nvfp4kv_packed_entry(const char* name, int* entry, int* num_args);
int nvfp4kv_call_packed(int entry, int num_args, const void* args);

#ifdef __cplusplus
}
#endif

#endif /* NVFP4KV_SERVING_H_ */
