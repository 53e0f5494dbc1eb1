/*
 * hsattn_ops.h -- what a prompt and its sequences need around the paged
 * attention of hsattn.h: rotary positions and the cache write, attention over
 * whole prompts, the cache's pages while their sequences live, a cache held in 4
 * bits, and decode through a window.  The
 * conventions (pointers, streams, status codes, dtype codes, block tables) are
 * hsattn.h's.  Nothing here replaces a function of the reference.
 */
#ifndef HSATTN_OPS_H
#define HSATTN_OPS_H

#include "hsattn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Rotary positions with several axes.  Pair i (of `pairs`) of every head of
 * row r is turned by theta = positions[pair_axis[i]][r] * inv_freq[i]:
 *   (a, b) -> (a cos theta - b sin theta, b cos theta + a sin theta)
 * where a and b are elements i and pairs + i of the head, or 2 i and 2 i + 1
 * with interleaved != 0; elements from 2 * pairs on are cast as they are.
 * Arithmetic in fp32 (the angle in fp64, so far positions lose nothing),
 * rounded once to each output's type.  No reference counterpart: its models
 * learn their positions.
 *   q, k        [n, H, D] and [n, Hkv, D] of src_dtype; rows q_row_stride and
 *               k_row_stride elements apart (slices of the fused projection
 *               work as they are)
 *   positions   [axes, n] int32 (1 axis for text; time, height, width for
 *               images and video); inv_freq [pairs] float32
 *   pair_axis   [pairs] int32, the axis of each pair (entries outside
 *               [0, axes) are read as axis 0), or NULL: all on axis 0
 *   pairs       1 .. D / 2, at most 1024
 *   q_out       [n, H, D] of out_dtype; k_out [n, Hkv, D] of out_dtype.  An
 *               output may be its own source (same type, rows without gaps),
 *               and must not overlap the sources otherwise.
 */
int hs_rotary(const void* q, const void* k, int src_dtype, int64_t q_row_stride,
              int64_t k_row_stride, const int32_t* positions, int axes, const float* inv_freq,
              const int32_t* pair_axis, int pairs, int interleaved, int64_t n, int H, int Hkv,
              int D, void* q_out, void* k_out, int out_dtype, void* stream);

/*
 * hs_rotary, and in the same launch hs_kv_append of the rotated keys and of
 * the values: row i of k (rotated in fp32, then cast to kv_dtype) and of v
 * goes to position cache_positions[i] of sequence seq_ids[i] (row i of the
 * tables when seq_ids is NULL, which needs n <= B).  Rows that hs_kv_append
 * would skip are not written; their q_out and k_out are.  k_out may be NULL
 * where only the cache needs the keys.  The cache must not overlap the
 * sources or outputs, and rows must not share a slot.
 */
int hs_rotary_append(const void* q, const void* k, const void* v, int src_dtype,
                     int64_t q_row_stride, int64_t k_row_stride, int64_t v_row_stride,
                     const int32_t* positions, int axes, const float* inv_freq,
                     const int32_t* pair_axis, int pairs, int interleaved, int64_t n, int H,
                     int Hkv, int D, void* q_out, void* k_out, int out_dtype, void* k_cache,
                     void* v_cache, int kv_dtype, int NB, int BS, const int32_t* block_tables,
                     int B, int MB, const int32_t* cache_positions, const int32_t* seq_ids,
                     void* stream);

/*
 * Causal attention over whole prompts, packed one behind the other, K and V as
 * the projection left them (hs_prefill_varlen reads them from the cache):
 *   out[i,h,:] = softmax_j(scale * q[i,h,:] . k[j,kvh,:]) . v[j,kvh,:]
 * over the rows j <= i of row i's own sequence; sequence b owns the rows
 * [cu_seqlens[b], cu_seqlens[b+1]) of [0, total).  Rows of no sequence, and
 * rows of a sequence from max_seqlen on, are left as they were.  What k and v
 * hold behind a row never reaches it, infinities and NaN included; rows that see
 * such a value are right and slow (a walk of their keys one by one).  Finite
 * values under finite scores give finite rows, up to the type's largest.
 * No reference counterpart (its engine prefills through the cache).
 *   q, k, v     [total, H, D], [total, Hkv, D] twice, of dtype; rows and
 *               heads are the given strides apart (elements, at most 2^22;
 *               multiples of 16 bytes), D elements of a head contiguous,
 *               16-byte aligned
 *   out         [total, H, D] of dtype, contiguous, 16-byte aligned; must not
 *               overlap the inputs
 *   D           32, 64, 128 or 256;  H % Hkv == 0;  scale finite, and times
 *               log2(e) as well (below 2.35e38)
 */
int hs_prompt_attention(const void* q, const void* k, const void* v, int dtype,
                        int64_t q_row_stride, int64_t q_head_stride, int64_t k_row_stride,
                        int64_t k_head_stride, int64_t v_row_stride, int64_t v_head_stride,
                        const int32_t* cu_seqlens, int B, int64_t total, int max_seqlen, int H,
                        int Hkv, int D, float scale, void* out, void* stream);

/*
 * Pages while their sequences live.  The state is the pool [L, 2, NB, page]
 * (page_bytes a page), the block tables [B, MB] (-1 padded), the context
 * lengths [B] and one count per block, ref_counts [NB]: how many table rows
 * (or other holders, such as a prefix cache) keep the block.  A block whose
 * count is not above 0 is free.  All of it stays on the device; the calls
 * below run in stream order and may be captured.  The reference keeps the
 * counts and tables on the host (heteroserve/kv/blocks.py:62) and has no copy
 * inside the pool.
 */

/*
 * pool[l, c, dst_ids[i]] = pool[l, c, src_ids[i]] for every layer, K and V.
 * Pairs with an id outside [0, NB) are skipped.  A destination must not repeat
 * nor be a source.
 */
int hs_kv_copy(void* pool, int L, int NB, int64_t page_bytes, const int64_t* src_ids,
               const int64_t* dst_ids, int n, void* stream);

/* out[0 .. n): the n lowest free blocks in ascending order, -1 past the last
 * one.  NB is at most 2^22.  Nothing is reserved: a count goes up where the
 * block is first held (hs_kv_fork, or the caller). */
int hs_kv_find_free(const int32_t* ref_counts, int NB, int32_t* out, int n, void* stream);

/*
 * Row children[i] of the tables becomes a fork of row parents[i], for i < n:
 * it shares the parent's full blocks (their counts go up by 1), and the tokens
 * of the parent's last, unfinished block (context_lens % BS of them; the rest
 * of the block is left as it was), if there is one, are copied for all layers
 * to block fresh[i], whose count goes up by 1.  The rest of the child's row is
 * -1 and its context length the parent's.  forked[i] is 1; it is 0, the
 * child's row -1 and its length 0, where the parent's last block or fresh[i] is
 * outside the pool (so -1 from hs_kv_find_free is safe), and 0 with nothing
 * written where a row is outside [0, B) or its own parent.  Contexts past the
 * table count as its end.
 * A parent may have several children.  A child must not repeat nor be a parent
 * in the same call, its row must hold no blocks (hs_kv_free it first), and
 * fresh blocks must not repeat.
 */
int hs_kv_fork(void* pool, int L, int NB, int64_t page_bytes, int BS, int32_t* block_tables, int B,
               int MB, int32_t* context_lens, int32_t* ref_counts, const int32_t* parents,
               const int32_t* children, const int32_t* fresh, int n, int32_t* forked,
               void* stream);

/* Rows `rows` [n] of the tables give up their blocks: every count goes down by
 * 1 (and never below 0), the row becomes -1 and its context length 0.  Row
 * indexes outside [0, B) are skipped, and one that repeats is freed once. */
int hs_kv_free(int32_t* block_tables, int B, int MB, int32_t* context_lens, int32_t* ref_counts,
               int NB, const int32_t* rows, int n, void* stream);

/*
 * The live blocks (count above 0) move into blocks [0, live), the highest one
 * into the lowest hole and so on; blocks below `live` stay where they are.
 * Pages (all layers, K and V), counts and table entries follow; an entry of a
 * free block becomes -1.  moved_to [NB] gets every live block's new id and -1
 * for the others, live [1] the number of live blocks.  NB is at most 2^22.
 *   workspace  device scratch of hs_kv_compact_workspace_bytes(NB) bytes
 */
size_t hs_kv_compact_workspace_bytes(int NB);
int hs_kv_compact(void* pool, int L, int NB, int64_t page_bytes, int32_t* block_tables, int B,
                  int MB, int32_t* ref_counts, int32_t* moved_to, int32_t* live, void* workspace,
                  size_t workspace_bytes, void* stream);

/*
 * A cache held in 4 bits.  A cache is [NB, BS, Hkv, HS_Q4_RECORD_BYTES(D)] bytes,
 * one record for each token and KV head, so its pages are copied, forked, packed
 * and moved as the bytes of any other.  Every 32 elements of a head share a step s
 * and a lowest value lo, both fp16:
 *   lo = min x,  s = max(0, (max x - lo) / 15)
 *   n  = (x - lo) / s to the nearest of 0 .. 15, ties to even (0 where s is 0)
 * and x is held as n s + lo.  Values beyond fp16's largest count as that; a group
 * that holds a NaN is NaN as a whole.  lo, s (through fp32) and n are rounded from
 * the exact quotients.  A record is D / 8 32-bit words of 8 elements n (element e in
 * bits 4 e .. 4 e + 3), then D / 32 steps, then D / 32 lowest values.  Word w holds
 * elements 8 w .. of a value's head, and elements 32 (w % G) + 8 (w / G) .. of a
 * key's, G = D / 32.  D is 32, 64, 128 or 256.  Caches are aligned to D / 8 bytes, at
 * most 16.  No reference counterpart.
 */
#define HS_Q4_RECORD_BYTES(D) ((D) / 2 + (D) / 8)

/*
 * hs_kv_append into a 4-bit cache: row i of k_src and v_src (n rows of Hkv * D
 * elements of src_dtype, rows the given strides of elements apart) goes to position
 * positions[i] of sequence seq_ids[i] (row i of the tables when seq_ids is NULL,
 * which needs n <= B).  Rows that hs_kv_append would skip are not written; rows must
 * not share a slot.
 */
int hs_q4_append(void* k_cache, void* v_cache, int NB, int BS, int Hkv, int D,
                 const int32_t* block_tables, int B, int MB, const int32_t* positions,
                 const int32_t* seq_ids, int64_t n, const void* k_src, const void* v_src,
                 int src_dtype, int64_t k_row_stride, int64_t v_row_stride, void* stream);

/*
 * The way back: row i of k_out and v_out [n, Hkv, D] of out_dtype (16-byte aligned,
 * no part of the caches) is what the cache holds at position positions[i] of
 * sequence seq_ids[i], n s + lo rounded to fp32 and then to out_dtype, or zeros where
 * hs_q4_append would skip.  In fp16 values beyond its largest count as that here too (15 s +
 * lo may be: s is rounded).  Rows may share a slot.
 */
int hs_q4_read(const void* k_cache, const void* v_cache, int NB, int BS, int Hkv, int D,
               const int32_t* block_tables, int B, int MB, const int32_t* positions,
               const int32_t* seq_ids, int64_t n, void* k_out, void* v_out, int out_dtype,
               void* stream);

/*
 * hs_decode over what a sequence's new token sees through a window: of the ctx_b
 * cached tokens (the new one among them) the last `window` and the first `sinks`.
 * window 0: all of them.  What other tokens' slots hold never reaches a row,
 * infinities and NaN included.  hs_q4_decode reads a 4-bit cache, hs_window_decode
 * one of kv_dtype; scores, softmax and sums are fp32, products as near as fp32's (of
 * a 4-bit cache: relative to their group's range), of a query's elements to 2^-22 or
 * to 2^-35 of the largest of their head, whichever is larger.
 * A row that sees an infinity or a NaN may be NaN in the elements that it reaches.
 * A call repeated gives the same bits; how a row's sums are split, and so its last
 * bits, depends on the sizes and on the lengths of all rows.
 *   q, out      [B, H, D] float32, 16-byte aligned
 *   D           32, 64, 128 or 256;  H % Hkv == 0;  MB * BS at most 2^30, num_blocks
 *               * BS below 2^31;  scale finite, and times log2(e) as well
 *   workspace   device scratch of the query's size for the same arguments, with the
 *               launch device current (may be NULL when that is 0), 16-byte aligned
 */
size_t hs_q4_decode_workspace_bytes(int B, int H, int Hkv, int D, int BS, int MB, int window,
                                    int sinks);
int hs_q4_decode(const float* q, const void* k_cache, const void* v_cache, int num_blocks,
                 const int32_t* block_tables, const int32_t* context_lens, float* out, int B,
                 int H, int Hkv, int D, int BS, int MB, float scale, int window, int sinks,
                 void* workspace, size_t workspace_bytes, void* stream);
size_t hs_window_decode_workspace_bytes(int kv_dtype, int B, int H, int Hkv, int D, int BS, int MB,
                                        int window, int sinks);
int hs_window_decode(const float* q, const void* k_cache, const void* v_cache, int kv_dtype,
                     int num_blocks, const int32_t* block_tables, const int32_t* context_lens,
                     float* out, int B, int H, int Hkv, int D, int BS, int MB, float scale,
                     int window, int sinks, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* HSATTN_OPS_H */
