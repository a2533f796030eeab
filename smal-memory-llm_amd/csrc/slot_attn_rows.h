// The running softmax of 32 query rows a wave, one row a lane and half (l and l + 32 share row l & 31), for the attention over pages.
#pragma once
#include "slot_attn.h"

namespace slotattn {

// A row's sums keep their reference maximum until a score passes it by this much (base 2): probabilities then reach 2^8, far
// from any type's end, and the sums are rescaled a few times a row instead of in most tiles.
#define LAZY 8.f
// Scores are taken to base 2 and from their reference by one multiply-add.  The reference's own product is rounded, which moves a row's
// probabilities by a common factor of up to 2^(|reference| 2^-24): nothing, until scores of millions.  From FAR on the difference is formed first.
#define FAR 4194304.f
// In fp16 the reference is 2^7 below the maximum, so that probabilities reach 2^7 to 2^15: fp16's smallest step is 2^-24, and below a largest
// one of 1 those under 2^-25 would add to a row's sum but not to its output (8,192 of them at 2^-26: 1.2e-4 of the values).
template <typename T> constexpr float HEAD = 0.f;
template <> inline constexpr float HEAD<f16_t> = 7.f;

template <typename T, int D, bool BIAS> struct RowSums {
    static constexpr int DT = D / 32;
    f32x16 o[DT];
    float m, mu, l;                                   // a row's reference, the same in base 2, its sum
    bool far;
    float F, lazy, head;                              // from a row's values to base 2
    __device__ __forceinline__ RowSums(float f2) : F(BIAS ? 1.f : f2), lazy(LAZY / F), head(HEAD<T> / F) { clear(); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[dt] = zero16();
        m = -INFINITY;
        mu = l = 0.f;
        far = false;
    }
    // NB tiles of 32 scores become probabilities as operands of the next product; the sums move to a new reference where they must
    template <int NB> __device__ __forceinline__ void weigh(f32x16 (&s)[NB], uint4 (&pf)[NB][2]) {
        float mx = s[0][0];
#pragma unroll
        for (int u = 0; u < NB; u++)
#pragma unroll
            for (int r = 0; r < 16; r++) mx = fmaxf(mx, s[u][r]);
        mx = half_max(mx) - head;
        if (__any(mx > m + lazy)) {
            const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : exp2_((m - mn) * F);
            m = mn;
            mu = m == -INFINITY ? 0.f : m * F;
            far = __any(fabsf(mu) > FAR);
            l *= f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int r = 0; r < 16; r++) o[dt][r] *= f;
        }
        if (far) {
#pragma unroll
            for (int u = 0; u < NB; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[u][r] = (s[u][r] - (m == -INFINITY ? 0.f : m)) * F;
        } else {
#pragma unroll
            for (int u = 0; u < NB; u++)
#pragma unroll
                for (int r = 0; r < 16; r++) s[u][r] = fmaf(s[u][r], F, -mu);
        }
#pragma unroll
        for (int u = 0; u < NB; u++) {
#pragma unroll
            for (int r = 0; r < 16; r++) {
                s[u][r] = exp2_(s[u][r]);
                l += s[u][r];
            }
            pf[u][0] = pack8<T>(s[u], 0);
            pf[u][1] = pack8<T>(s[u], 1);
        }
    }
    // a row's sum over both halves, and its reference in base 2 from here on
    __device__ __forceinline__ void close() {
        l = half_sum(l);
        m = m == -INFINITY ? m : mu;
    }
};

}  // namespace slotattn
