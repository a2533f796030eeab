// Argument checks and kernel arguments shared by the attention entry points (slotattn.hip, slotattn_bwd.hip).
#pragma once
#include <algorithm>
#include <cmath>

#include "slot_attn.h"
#include "slot_host.h"
#include "slotscan.h"

#define SLOTATTN_MAX_T 0x3fffffffLL                  // positions and their differences stay in 31 bits
#define SLOTATTN_MAX_ST (1LL << 25)                  // elements between tokens: 32 rows' offsets in bytes stay in 32 bits

namespace slotattn_host {

inline int check(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh, int64_t k_st,
                 const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, int64_t B, int64_t Tq, int64_t Tk, int64_t Hq,
                 int64_t Hk, int64_t D, float scale, int64_t window, float cap) {
    using slothost::fail;
    using slothost::al16;
    if (B < 1 || Tq < 1 || Tk < 1 || Hq < 1 || Hk < 1) return fail(SLOTSCAN_ERR_SHAPE, "slotattn: B, Tq, Tk, Hq, Hk must be >= 1");
    if (Hq % Hk) return fail(SLOTSCAN_ERR_SHAPE, "slotattn: Hq must be a multiple of Hk");
    if (D != 64 && D != 128) return fail(SLOTSCAN_ERR_SHAPE, "slotattn: D must be 64 or 128");
    if (window < 1 || window > 0x7fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn: window must be in [1, 2^31)");
    if (!(cap == 0.f || (cap >= 1e-30f && cap <= 1e30f))) return fail(SLOTSCAN_ERR_SHAPE, "slotattn: cap must be 0 or in [1e-30, 1e30]");
    if (!(std::fabs(scale) >= 1e-30f && std::fabs(scale) <= 1e30f)) return fail(SLOTSCAN_ERR_SHAPE, "slotattn: |scale| must be in [1e-30, 1e30]");
    if (cap > 1.000001e36 * std::fabs((double)scale))                 // (both are rounded to 32 bits here)
        return fail(SLOTSCAN_ERR_SHAPE, "slotattn: cap must be at most 1e36 |scale|");
    if (Tq > SLOTATTN_MAX_T || Tk > SLOTATTN_MAX_T || B > 0x7fffffffLL / Hq || Hq / Hk * Tq > SLOTATTN_MAX_T)
        return fail(SLOTSCAN_ERR_SHAPE, "slotattn: shape too large");
    if (std::max(std::max(q_st, k_st), v_st) >= SLOTATTN_MAX_ST || std::min(std::min(q_st, k_st), v_st) < 0)
        return fail(SLOTSCAN_ERR_SHAPE, "slotattn: token strides must be in [0, 2^25)");
    if (dtype != SLOTSCAN_BF16 && dtype != SLOTSCAN_F16) return fail(SLOTSCAN_ERR_DTYPE, "slotattn: dtype must be bf16 or fp16");
    if (!q || !k || !v) return fail(SLOTSCAN_ERR_NULL, "slotattn: a required pointer is NULL");
    if (!al16(q) || !al16(k) || !al16(v) || (q_sb | q_sh | q_st | k_sb | k_sh | k_st | v_sb | v_sh | v_st) % 8)
        return fail(SLOTSCAN_ERR_ALIGN, "slotattn: rows of q, k and v must be 16-byte aligned");
    return 0;
}

inline slotattn::AttnArgs args(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                               int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int64_t B, int64_t Tq, int64_t Tk,
                               int64_t Hq, int64_t Hk, float scale, int causal, int64_t window, float cap, const float* slopes,
                               const void* docs, const int32_t* prefix) {
    slotattn::AttnArgs a{};
    a.q = q; a.k = k; a.v = v;
    a.q_sb = q_sb; a.q_sh = q_sh; a.q_st = q_st;
    a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
    a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
    a.B = (int)B; a.Tq = (int)Tq; a.Tk = (int)Tk; a.Hq = (int)Hq; a.Hk = (int)Hk; a.R = (int)(Hq / Hk);
    a.causal = causal != 0;
    a.W = (int)std::min<int64_t>(window, 1 << 30);      // any distance is less
    a.slopes = slopes;
    a.ntd = (int)((Tk + KT - 1) / KT);
    a.ids = (const int32_t*)docs;
    a.range = docs ? (const int2*)((const int32_t*)docs + B * a.ntd * KT) : nullptr;
    a.prefix = prefix;
    a.scale = scale;
    a.f = scale * LOG2E;
    if (cap > 0.f) {
        a.f = cap * LOG2E;
        const double k = std::min(std::max((double)scale / cap, -1e37), 1e37), m = std::fabs(k);       // (at the ends tanh is 1, or its argument 0)
        a.kc = (float)k;
        a.ct = (float)(2.0 * k * 1.4426950408889634);
        a.mix = cap > 64.f;
        a.lim = -1.f;                                 // powers of k that leave fp32: no score takes the shorter polynomial
        if (m >= 1e-4 && m <= 1e3) {                  // in the products <q, k> themselves
            const double t[5] = {TANH0, TANH1, TANH2, TANH3, TANH4};
            double f = k;
            float* c[5] = {&a.t0, &a.t1, &a.t2, &a.t3, &a.t4};
            for (int i = 0; i < 5; i++, f *= k * k) *c[i] = (float)(t[i] * f);
            a.lim = (float)(0.75 / m);
        }
    }
    a.nsplit = 1;
    return a;
}

}  // namespace slotattn_host
