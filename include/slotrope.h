/* C-ABI of the MI355X (gfx950) head norm and position rotation of queries and keys, part of libslotscan.so.
 *
 * One pass over the queries and keys as a layer's projection leaves them.  Every head's row x of D values:
 *     y = x * rsqrt(mean(x^2) + eps) * w          (w: the gain of the queries' or the keys' heads, NULL: none)
 *     (a, b) -> (a cos - b sin, b cos + a sin)    for the rot / 2 pairs of the first rot values, angle = position * freqs[i]
 * pair i is (i, i + rot / 2), or with `interleaved` (2 i, 2 i + 1); the values behind rot are normed only.  Sums, angles'
 * sines and products are fp32, the angles themselves fp64 (a far position times a frequency keeps its fraction of a turn);
 * the result is rounded once.
 *
 * Conventions as in slotscan.h (device pointers, caller-allocated, launched on `stream`, 0 or a SLOTSCAN_ERR_* code).
 *   dtype   SLOTSCAN_F32, SLOTSCAN_BF16 or SLOTSCAN_F16: of every token tensor and cache
 *   wdtype  the same codes: of both gains and their gradients
 *   q (B, Hq, T, D), k, v (B, Hk, T, D) by strides in elements (batch, head, token; the D values of a row are contiguous), every row
 *           16-byte aligned; D = 64 or 128; rot a multiple of 16, 0 <= rot <= D; freqs (rot / 2) fp64
 *   outputs without strides are token-major and contiguous, (B, T, H, D)
 */
#ifndef SLOTROPE_H
#define SLOTROPE_H
#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Forward: qo (B, T, Hq, D), ko (B, T, Hk, D).  pos: the positions of the tokens, int64 (pos64) or int32, row b at
 * pos + b * pos_sb (0: the same for every sequence), or NULL: 0 .. T - 1. */
int slotrope_fwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                 int64_t k_st, int dtype, const void* wq, const void* wk, int wdtype, const double* freqs, int64_t rot,
                 int interleaved, const void* pos, int pos64, int64_t pos_sb, int64_t B, int64_t T, int64_t Hq,
                 int64_t Hk, int64_t D, float eps, void* qo, void* ko, void* stream);

/* Backward: the gradients dqo, dko of the two outputs (by strides) in; dq (B, T, Hq, D), dk (B, T, Hk, D) and dwq, dwk
 * (D, in wdtype; NULL: not wanted) out.  The gains' gradients are summed in fp32 in a fixed order (no atomics).
 * workspace: slotrope_bwd_workspace(B, T, Hq, Hk, D) bytes, 16-byte aligned. */
size_t slotrope_bwd_workspace(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D);
int slotrope_bwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                 int64_t k_st, int dtype, const void* wq, const void* wk, int wdtype, const double* freqs, int64_t rot,
                 int interleaved, const void* pos, int pos64, int64_t pos_sb, int64_t B, int64_t T, int64_t Hq,
                 int64_t Hk, int64_t D, float eps, const void* dqo, int64_t dq_sb, int64_t dq_sh, int64_t dq_st,
                 const void* dko, int64_t dk_sb, int64_t dk_sh, int64_t dk_st, void* workspace, void* dq, void* dk,
                 void* dwq, void* dwk, void* stream);

/* The serving form: the tokens are the newest T of lens[b] tokens of sequence b (token t at position lens[b] - T + t).
 * qo (B, T, Hq, D) is written whole; the prepared keys and the values go to rows `position` of the caches kc, vc
 * (B, Hk, S, D) by strides.  A token whose position is negative (a first prompt's padding on the left) or >= S writes no cache row; one
 * of a sequence that has tokens already has a position of theirs and overwrites it. */
int slotrope_cache(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                   int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, const void* wq,
                   const void* wk, int wdtype, const double* freqs, int64_t rot, int interleaved, const int32_t* lens,
                   int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t S, float eps, void* qo, void* kc,
                   int64_t kc_sb, int64_t kc_sh, int64_t kc_st, void* vc, int64_t vc_sb, int64_t vc_sh, int64_t vc_st,
                   void* stream);

#ifdef __cplusplus
}
#endif
#endif /* SLOTROPE_H */
