/*
 * pbattn.h - C ABI of the MI355X (gfx950) attention operators: the windowed
 * attention that a hybrid layer runs beside its Gated DeltaNet recurrence
 * (the operators of pbgdn.h), over plain keys and over a paged cache.
 *
 *   pbattn_window_fwd      attention with a sliding window and a few first
 *                          tokens that stay visible (sinks); prefill, training
 *   pbattn_window_bwd      its gradients
 *   pbattn_paged_decode    the newest token (or a few drafted ones) of each
 *                          sequence over a paged key-value cache, split over
 *                          the cache's length and joined
 *   pbattn_paged_write     new keys and values into the cache's pages
 *   pbattn_fp4_decode, pbattn_fp4_write, pbattn_fp4_read
 *                          the cache held in 4 bits: decoding over it, its writes,
 *                          its contexts read back
 *   pbattn_pages_extend, pbattn_pages_release
 *                          the pages, slots and positions of new tokens from the
 *                          requests' lengths; pages given back
 *   pbattn_qk_norm_rope, pbattn_qk_norm_rope_bwd
 *                          what queries and keys go through before they are attended:
 *                          norms of each head and the rotation by position
 *
 * The reference computes this half of WindowedHybridLayer.mix
 * (pseudobrain/transplant.py:989-997) with PyTorch's attention in training and
 * leaves it to vLLM in serving (serving/pb27_vllm/pb27_vllm/model.py:481-490).
 *
 * What a query sees: Tq queries are the last Tq positions of their sequence's
 * Tk keys, so query i stands at position p = Tk - Tq + i. It sees key j when
 * j <= p and (j > p - window or j < sinks); window <= 0 means no window. With
 * s_ij = scale q_i . k_j over the keys that i sees, p_ij = exp(s_ij - lse_i)
 * and lse_i = log sum_j exp(s_ij), o_i = sum_j p_ij v_j. A query that sees no
 * key gets o = 0 and lse = -infinity, and adds nothing to any gradient; no other
 * query has that lse (one past float32's range ends at its largest values).
 * Query head h reads key head h / (Hq / Hk).
 *
 * Conventions: those of pbgdn.h (its dtype and status codes; caller-owned
 * device memory, nothing allocated, launches asynchronous on `stream`, no
 * state kept between calls, no exception across the ABI). Scores, softmax
 * statistics and every accumulation are float32; with 16-bit inputs the
 * weights p (and in the backward ds) are rounded to that type as matrix
 * operands, with float32 inputs nothing is rounded below float32. Strides are
 * in elements; the innermost axis (the head width) is dense. Results do not
 * depend on scheduling: no sum is taken by atomics.
 *
 * Infinities and NaN. What no query of the call sees (keys past a sequence's
 * length, absent pages, tokens of no sequence) is never used, whatever it
 * holds. The forward and the decoding call also keep a key's or value's infinity
 * or NaN from the queries that do not see that key. The backward call does not: a key,
 * value, query or grad_o that is not finite may reach the gradients of its
 * neighbours (within 128 positions) that it has no part in.
 */
#ifndef PBATTN_H_
#define PBATTN_H_

#include <stddef.h>
#include <stdint.h>

#include "pbgdn.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Raised with every function that is added or changed. */
#define PBATTN_ABI_VERSION 4

/* Most query tokens a sequence may have in pbattn_paged_decode. */
#define PBATTN_MAX_DRAFT 16

/* Version of this ABI (PBATTN_ABI_VERSION). */
int pbattn_abi_version(void);

/*
 * Forward.
 *
 *   q          [B, Tq, Hq, D]   dtype F32, BF16 or F16, any strides whose
 *   k, v       [B, Tk, Hk, D]   values are multiples of 16 bytes; bases
 *                               aligned to 16 bytes
 *   strides    (batch, token, head) strides of q, k, v: 9 values, elements;
 *              a token stride below 2^24 bytes
 *   cu_q, cu_k [N + 1] int32 boundaries of N packed sequences in the token
 *              axes (B must be 1, nondecreasing, from 0 to Tq / Tk), or NULL:
 *              then N = B sequences of Tq and Tk tokens. cu_k NULL with cu_q
 *              given: the same boundaries (Tk must equal Tq). Tokens past the
 *              last boundary belong to no sequence: such a query sees nothing,
 *              such a key is seen by none
 *   o          [B, Tq, Hq, D] dense, dtype, written
 *   lse        [B, Tq, Hq] dense float32, written; may be NULL
 *   D          64, 128 or 256 (narrower heads zero-padded by the caller)
 *
 * A call without sequences or queries (B, num_seqs or Tq 0) launches nothing and
 * writes nothing, the backward call's neither: where tokens of no sequence are
 * left (num_seqs 0), or keys without queries (Tq 0), the caller fills o with
 * zeros, lse with -infinity and the gradients with zeros.
 */
int pbattn_window_fwd(const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                      const int32_t *cu_q, const int32_t *cu_k, int num_seqs, void *o, float *lse, int B, int Tq,
                      int Tk, int Hq, int Hk, int D, float scale, int window, int sinks, void *stream);

/*
 * Gradients of pbattn_window_fwd. With delta_i = do_i . o_i - dlse_i,
 * dp_ij = do_i . v_j and ds_ij = p_ij (dp_ij - delta_i):
 *   dv_j = sum_i p_ij do_i,  dk_j = scale sum_i ds_ij q_i,  dq_i = scale sum_j ds_ij k_j,
 * the sums of dk and dv over every query head of the key head's group.
 *
 *   q .. num_seqs, B .. sinks   as in the forward call; besides, 32 rows of q
 *              (h = min(Hq / Hk, 32) heads of 32 / h tokens) must lie within
 *              0x7ffffff0 bytes by its strides, and as many of grad_o
 *   o, lse     the forward call's results (dense)
 *   grad_o     [B, Tq, Hq, D] dense, dtype
 *   grad_lse   [B, Tq, Hq] dense float32, or NULL for zeros
 *   dq         [B, Tq, Hq, D] dense, dtype, written
 *   dk, dv     [B, Tk, Hk, D] dense, dtype, written (zeros for keys
 *              that no query sees)
 *   workspace  device scratch of at least pbattn_window_bwd_workspace_size
 *              bytes, 16-byte aligned; needs no initialisation
 *
 * With dtype F16, ds is scaled by a power of two found on the device from the
 * largest finite |do|, |v| and |dlse| of the queries that see a key and the
 * keys that a query sees, before it is rounded, and the results scaled back, so
 * that neither small nor large gradients leave float16's range there. It is one
 * power of two for the call: the largest of them all sets it.
 */
int pbattn_window_bwd(const void *q, const void *k, const void *v, int dtype, const int64_t *strides,
                      const int32_t *cu_q, const int32_t *cu_k, int num_seqs, const void *o, const float *lse,
                      const void *grad_o, const float *grad_lse, void *dq, void *dk, void *dv, int B, int Tq, int Tk,
                      int Hq, int Hk, int D, float scale, int window, int sinks, void *workspace,
                      size_t workspace_bytes, void *stream);

/* Bytes of workspace pbattn_window_bwd needs: 12 bytes per (token, query head)
 * and, where the sums over queries are split, their float32 parts. 0 for
 * invalid sizes. `packed`: cu_q is given. */
size_t pbattn_window_bwd_workspace_size(int B, int Tq, int Tk, int Hq, int Hk, int D, int num_seqs, int dtype,
                                        int packed, int window, int sinks);

/*
 * One step of decoding over a paged cache: the T newest tokens of each of B
 * sequences (1, or a sampled token and drafted ones to verify) against its
 * cached keys and values, theirs among them.
 *
 *   q            [B, T, Hq, D] dtype; 1 <= T <= PBATTN_MAX_DRAFT
 *   k_cache,     pages of page_size tokens: token i of page g at element
 *   v_cache      g strides[0] + i strides[1], key head h strides[2] further on
 *                (both caches by the same three strides, multiples of 16
 *                bytes, strides[0] a multiple of strides[1]: [pages, page,
 *                heads, D] and [pages, heads, page, D] alike), dtype
 *   num_pages    pages in the caches
 *   page_table   [B, max_pages] int32: key j of sequence b is token
 *                j % page_size of page page_table[b][j / page_size]; entries
 *                that no query sees are not read, and the keys of an entry
 *                outside [0, num_pages) count as absent
 *   lengths      [B] int32 keys of each sequence; query t stands at position
 *                lengths[b] - T + t. A sequence of length <= 0 sees nothing
 *   o            [B, T, Hq, D] dense, dtype, written
 *   lse          [B, T, Hq] dense float32, written; may be NULL
 *   workspace    at least pbattn_paged_decode_workspace_size bytes, 16-byte
 *                aligned; needs no initialisation
 *
 * The visible keys of all sequences are divided over the GPU on the device,
 * from lengths alone, in parts whose partial softmax a second kernel joins in
 * a fixed order: equal inputs give equal results.
 */
int pbattn_paged_decode(const void *q, const void *k_cache, const void *v_cache, int dtype, const int64_t *strides,
                        int page_size, int num_pages, const int32_t *page_table, int max_pages,
                        const int32_t *lengths, void *o, float *lse, int B, int T, int Hq, int Hk, int D, float scale,
                        int window, int sinks, void *workspace, size_t workspace_bytes, void *stream);

/* Bytes of workspace pbattn_paged_decode needs; 0 for invalid sizes. */
size_t pbattn_paged_decode_workspace_size(int B, int T, int Hq, int Hk, int D);

/*
 * Writes N tokens' keys and values into the caches.
 *
 *   k, v       [N, Hk, D] dtype by kv_strides (token, head of k, then of v;
 *              elements, multiples of 16 bytes)
 *   k_cache .. num_pages   as above, written
 *   slots      [N] int64: token i goes to token slots[i] % page_size of page
 *              slots[i] / page_size; a slot outside [0, num_pages page_size)
 *              (e.g. -1 for padding) is skipped; the others must be distinct
 */
int pbattn_paged_write(const void *k, const void *v, int dtype, const int64_t *kv_strides, void *k_cache,
                       void *v_cache, const int64_t *strides, int page_size, int num_pages, const int64_t *slots,
                       int N, int Hk, int D, void *stream);

/* Most sequences of a call that works packed sequences out from their lengths
 * (pbattn_fp4_read, pbattn_pages_extend, pbattn_pages_release). */
#define PBATTN_MAX_REQUESTS 4096

/*
 * The cache held in 4 bits. 32 consecutive values of a head share a scale s, a
 * power of two; each is held as the nearest of +-{0, 0.5, 1, 1.5, 2, 3, 4, 6} s
 * (ties to the even code; codes 0 to 7, 8 more for a negative value). s is
 * 2^(e - 2), where 2^e <= x < 2^(e + 1) for the largest |x| of the 32, and twice
 * that where x >= 1.75 2^e, held as the byte e - 2 + 127 kept within [2, 252]
 * (smaller values round to zero or 2^-126, larger ones are cut to 6 2^125). A byte
 * of 255 marks 32 values among which one is infinite or NaN: all of them read as
 * NaN. Byte i of a row of codes holds value 2 i in its lower half and 2 i + 1 in the
 * upper one.
 *
 *   k_cache, v_cache   codes: pages of page_size tokens, rows of D / 2 bytes; token
 *                      i of page g at byte g strides[0] + i strides[1], key head h
 *                      strides[2] further on. Strides are multiples of D / 2,
 *                      strides[0] of strides[1] too
 *   k_scale, v_scale   their scales, laid out alike: rows of D / 32 bytes, every
 *                      stride a sixteenth of the codes'
 *   D                  64, 128 or 256; bases aligned to 16 bytes
 */

/*
 * pbattn_paged_decode over such a cache: the same arguments besides, and the same
 * results for the values that the cache stands for. q in any of the three types.
 * Queries enter the products exactly (float16 and float32 rows in two and three
 * parts), the weights of 16-bit rows in two parts, rounded to 16 bits (off by 2^-16
 * at most), those of float32 rows in three, with all of their 24.
 */
int pbattn_fp4_decode(const void *q, int dtype, const void *k_cache, const void *v_cache, const void *k_scale,
                      const void *v_scale, const int64_t *strides, int page_size, int num_pages,
                      const int32_t *page_table, int max_pages, const int32_t *lengths, void *o, float *lse, int B,
                      int T, int Hq, int Hk, int D, float scale, int window, int sinks, void *workspace,
                      size_t workspace_bytes, void *stream);

/* Bytes of workspace pbattn_fp4_decode needs; 0 for invalid sizes. */
size_t pbattn_fp4_decode_workspace_size(int B, int T, int Hq, int Hk, int D);

/* pbattn_paged_write into such a cache: k, v of `dtype` by kv_strides are rounded as
 * said above. */
int pbattn_fp4_write(const void *k, const void *v, int dtype, const int64_t *kv_strides, void *k_cache, void *v_cache,
                     void *k_scale, void *v_scale, const int64_t *strides, int page_size, int num_pages,
                     const int64_t *slots, int N, int Hk, int D, void *stream);

/*
 * Reads B sequences back, packed in their order: the first lengths[b] keys and
 * values of each, as pbattn_window_fwd takes them for a prompt's next queries.
 *
 *   page_table, lengths   as in pbattn_paged_decode (a length below 0 counts as 0)
 *   k, v         [tokens, Hk, D] dense, dtype (exact in bfloat16 and float32; float16
 *                ends at its own range), written: zeros for the keys of absent pages
 *                and for tokens past the last sequence
 *   cu_seqlens   [B + 1] int32, written: where each sequence starts and ends, cut at
 *                `tokens`
 *   B            at most PBATTN_MAX_REQUESTS
 */
int pbattn_fp4_read(const void *k_cache, const void *v_cache, const void *k_scale, const void *v_scale,
                    const int64_t *strides, int page_size, int num_pages, const int32_t *page_table, int max_pages,
                    const int32_t *lengths, void *k, void *v, int dtype, int32_t *cu_seqlens, int B, int tokens, int Hk,
                    int D, void *stream);

/*
 * The pages of a paged cache from its requests' lengths, on the device: a pool of free
 * pages, kept as a stack, from which requests take pages as they grow and to which they
 * give them back. Page i of a request holds its tokens i page_size .. (i + 1) page_size
 * - 1, entry i of its row of page_table (rows table_row entries apart) says which it is.
 *
 *   free_pages   [capacity] int32, the pool's pages from its bottom up
 *   num_free     [1] int32, how many of them there are (kept within [0, capacity])
 *   B            at most PBATTN_MAX_REQUESTS; max_pages page_size at most 2^31 - 1
 *
 * pbattn_pages_extend: request b, of lengths[b] tokens, gets counts[b] more (none where
 * it is not positive). Requests are gone through in order; one is granted if
 *   its tokens, and those asked for by all requests before it, are at most `tokens`,
 *   they and its lengths[b] (not negative) fit max_pages pages, and
 *   it needs no new page, or the pages that requests up to it need (those of requests
 *   that fail the first two left out) are no more than the pool's.
 * The others get nothing. New pages come off the top of the stack, in the requests'
 * order, and are entered in page_table; the granted tokens are packed in that order:
 *   slots        [tokens] int64, written: page_table entry times page_size plus the
 *                place there, as pbattn_paged_write takes it (-1 where the entry is
 *                negative), and -1 past the last token
 *   positions    [tokens] int32, written: the token's place in its request, -1 past the last
 *   cu_seqlens   [B + 1] int32, written: where each request's new tokens start and end
 *   new_lengths  [B] int32, written: lengths with what was granted
 *   new_num_free [1] int32, written
 * pbattn_pages_release: the pages of request b whose last token lies in [first[b],
 * end[b]) are pushed, in the requests' order (capacity ends it); entries below 0, which
 * are no pages, are left out, and page_table stays as it is. Ranges of one request that follow each other so give every page back once: the
 * tokens that a window has left, or, up to a multiple of page_size, all of a finished
 * request's.
 * Which pages a request holds follows from its length: whoever lowers one (drafted tokens
 * that were not accepted) releases [new length, old length), both rounded up to a multiple
 * of page_size, before the next pbattn_pages_extend, which takes pages past the new length
 * as not yet held and would enter others in their place.
 *
 * Neither changes lengths, counts, num_free: the same call again gives the same results.
 * The outputs must not overlap the inputs.
 */
int pbattn_pages_extend(int32_t *page_table, int64_t table_row, int max_pages, const int32_t *lengths,
                        const int32_t *counts, int B, int page_size, const int32_t *free_pages, int capacity,
                        const int32_t *num_free, int tokens, int64_t *slots, int32_t *positions, int32_t *cu_seqlens,
                        int32_t *new_lengths, int32_t *new_num_free, void *stream);
int pbattn_pages_release(const int32_t *page_table, int64_t table_row, int max_pages, const int32_t *first,
                         const int32_t *end, int B, int page_size, int32_t *free_pages, int capacity,
                         const int32_t *num_free, int32_t *new_num_free, void *stream);

/*
 * Norms of queries and keys for each head, and the rotation by their positions, in one
 * pass: for a row x of D values, with r = (mean x^2 + eps)^(-1/2) and the weight w,
 *   y_i = x_i r (w_i + weight_offset),
 *   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin)   for the R / 2 pairs (a, b)
 * of the first R values: i and R / 2 + i, or with `interleaved` 2 i and 2 i + 1; the
 * others stay. float32 throughout, rounded once; rows whose squares float32 does not hold
 * are scaled by a power of two for them.
 *
 *   q, k         [B, T, Hq, D] and [B, T, Hk, D] dtype by `strides` (batch, token, head of
 *                q, then of k: 6 values, elements, not negative), the innermost axis
 *                dense. Where strides and bases are multiples of 16 bytes and D and R of
 *                16 (float32: of 8) rows are moved in whole units; any others work too,
 *                slower
 *   q_weight, k_weight   [D] of weight_dtype
 *   cos, sin     [rows, R / 2] float32: the angles of position i in row i
 *   positions    int32, or int64 with positions64, by pos_strides (batch, token;
 *                elements, 0 to repeat): rows of the tables. A token whose position lies
 *                outside them (-1 for padding) gets zeros
 *   q_out, k_out dense, dtype, written; 16-byte aligned
 *   D            up to 256; R even, 0 (norms alone) to D
 */
int pbattn_qk_norm_rope(const void *q, const void *k, int dtype, const int64_t *strides, const void *q_weight,
                        const void *k_weight, int weight_dtype, float weight_offset, const float *cos, const float *sin,
                        int rows, const void *positions, int positions64, const int64_t *pos_strides, void *q_out,
                        void *k_out, int B, int T, int Hq, int Hk, int D, int R, float eps, int interleaved, void *stream);

/*
 * Its gradients: with g the gradient of an output row turned back by its angles and
 * u = g (w + weight_offset),
 *   dx = r (u - x r^2 mean(u x)),  dw = sum over tokens and heads of g x r
 *   grad_q, grad_k        dense, dtype, 16-byte aligned
 *   dq, dk                dense, dtype, written (zeros for tokens without a position,
 *                         which add nothing to dw)
 *   dq_weight, dk_weight  [D] weight_dtype, written, 16-byte aligned
 *   workspace             at least pbattn_qk_norm_rope_bwd_workspace_size bytes, 16-byte
 *                         aligned; needs no initialisation
 * Sums are taken in a fixed order. A call without tokens writes nothing, the weights'
 * gradients neither.
 */
int pbattn_qk_norm_rope_bwd(const void *q, const void *k, int dtype, const int64_t *strides, const void *q_weight,
                            const void *k_weight, int weight_dtype, float weight_offset, const float *cos,
                            const float *sin, int rows, const void *positions, int positions64, const int64_t *pos_strides,
                            const void *grad_q, const void *grad_k, void *dq, void *dk, void *dq_weight, void *dk_weight,
                            int B, int T, int Hq, int Hk, int D, int R, float eps, int interleaved, void *workspace,
                            size_t workspace_bytes, void *stream);

/* Bytes of workspace pbattn_qk_norm_rope_bwd needs on the current device; 0 for an invalid width. */
size_t pbattn_qk_norm_rope_bwd_workspace_size(int D);

#ifdef __cplusplus
}
#endif

#endif /* PBATTN_H_ */
