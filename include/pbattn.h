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
#define PBATTN_ABI_VERSION 2

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

#ifdef __cplusplus
}
#endif

#endif /* PBATTN_H_ */
