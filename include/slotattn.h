/* C-ABI of the MI355X (gfx950) exact attention of any range, part of libslotscan.so.
 *
 * Scaled dot-product attention whose scores may be capped and biased and whose visibility is a band, documents and a
 * prefix; the rolling window of slotwin.h is the special case of a short causal window alone.  For query i at position
 * p_i and key j at position j:
 *     s = scale <q_i, k_j>;   cap > 0:  s = cap tanh(s / cap);   slopes:  s -= slopes[head] |p_i - j|
 *     out_i = sum_j softmax_j(s) v_j  over the visible keys, 0 where there is none
 * key j is visible to query i when
 *     0 <= p_i - j < window  (causal)   or   |p_i - j| < window  (not causal),   or   j < prefix[b]
 * and, with documents, both belong to the same one (a negative id is padding: sees nothing and is not seen), and j < lens[b].
 * The Tq queries are the last ones of the Tk keys, or of each sequence's lens[b] keys:  p_i = i + Tk - Tq  or  i + lens[b] - Tq
 * (a query of negative position sees nothing; lens[b] > Tk reads Tk keys).
 *
 * Conventions as in slotscan.h (device pointers, caller-allocated, launched on `stream`, 0 or a SLOTSCAN_ERR_* code).
 *   dtype   SLOTSCAN_BF16 or SLOTSCAN_F16; scores, softmax statistics and sums are fp32
 *   q (B, Hq, Tq, D), k, v (B, Hk, Tk, D) by strides in elements (batch, head, token), every row 16-byte aligned; D = 64 or 128;
 *           Hq a multiple of Hk: query head h reads key/value head h / (Hq / Hk)
 *   |scale| in [1e-30, 1e30], cap too and at most 1e36 |scale|, or 0: none; window >= 1 (2^31 - 1: none); slopes (Hq) fp32, prefix (B), lens (B) int32 or NULL
 *   out, dq (B, Tq, Hq, D), dk, dv (B, Tk, Hk, D) contiguous;  lse, delta (B, Hq, Tq) fp32, the rows' log-sum-exp in base 2
 *           (+inf where nothing is visible) and sum(dout o out), kept between the calls
 *   docs    what slotattn_docs left: slotattn_docs_bytes(B, Tk) bytes, or NULL
 */
#ifndef SLOTATTN_H
#define SLOTATTN_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* The document ids (B, T) int32 in the form that the kernels read: padded to whole 64-key tiles, each with the range of its
 * ids, so that tiles of other documents are skipped.  Ids may come in any order. */
size_t slotattn_docs_bytes(int64_t B, int64_t T);
int slotattn_docs(const int32_t* ids, int64_t B, int64_t T, void* docs, void* stream);

/* Forward.  res (as out: what rounding took from it, so that delta is as exact as the sums) and lse may be NULL where no backward follows.  workspace: slotattn_fwd_workspace(...) bytes, 256-byte aligned: partial results where few query
 * rows meet many keys and the keys are split over workgroups (0 bytes otherwise). */
size_t slotattn_fwd_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, int causal, int64_t window,
                              int has_docs, int has_prefix, int has_lens);
int slotattn_fwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                 int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, int64_t B, int64_t Tq,
                 int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, float scale, int causal, int64_t window, float cap,
                 const float* slopes, const void* docs, const int32_t* prefix, const int32_t* lens, void* workspace,
                 void* out, void* res, float* lse, void* stream);

/* Backward for the upstream gradient dout (B, Hq, Tq, D) by strides, without lens.  delta is written on the way.  Two kernels, one walking the
 * keys of every query tile (dq), one the queries of every key tile (dk, dv; where there are few key tiles, parts of the queries, whose sums a
 * third kernel adds in order): no atomics, bitwise reproducible.  workspace: slotattn_bwd_workspace(...) bytes, 256-byte aligned. */
size_t slotattn_bwd_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, int causal, int64_t window,
                              int has_prefix);
int slotattn_bwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                 int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, int64_t B, int64_t Tq,
                 int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, float scale, int causal, int64_t window, float cap,
                 const float* slopes, const void* docs, const int32_t* prefix, const void* out, const void* res,
                 const float* lse, const void* dout, int64_t do_sb, int64_t do_sh, int64_t do_st, void* workspace, float* delta, void* dq,
                 void* dk, void* dv, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SLOTATTN_H */
