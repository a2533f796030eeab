// Exact attention of any range for MI355X (gfx950), backward (semantics: slotattn.h).  With P = softmax, dP = dO V^T,
// delta = rowsum(dO o O) and the cap's slope 1 - tanh^2:
//     dS = P (dP - delta) (1 - tanh^2),   dV = P^T dO,   dQ = scale dS K,   dK = scale dS^T Q
// P comes back from the rows' log-sum-exp.  Two kernels, each of which owns what it sums, so nothing is added atomically:
//   attn_dq    128 queries of one head per workgroup, walking the visible key tiles (as the forward does); it forms delta
//   attn_dkv   128 keys of one key/value head per workgroup, walking the query tiles of every head of the group that see them
// The price is that the scores and dP are formed twice (with dQ's in two parts 8 products, where one kernel with atomic dQ would need 5 or 6).
#include <algorithm>

#include "slot_attn.h"
#include "slotscan.h"
#include "slotattn.h"
#include "slot_attn_host.h"

using namespace slotattn;
using slothost::fail;
using slothost::hip_fail;
using slothost::al16;

#define BW 4                                         // waves per workgroup
#define BT (64 * BW)
#define BQ (32 * BW)                                 // queries (attn_dq) or keys (attn_dkv) per workgroup
#define QT 32                                        // query rows of a tile of attn_dkv

namespace {

__device__ __forceinline__ void dot8(const uint4& x, const uint4& y, float& s, bf16_t) {
    const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        s = fmaf(__uint_as_float(xs[i] << 16), __uint_as_float(ys[i] << 16), s);
        s = fmaf(__uint_as_float(xs[i] & 0xffff0000u), __uint_as_float(ys[i] & 0xffff0000u), s);
    }
}
__device__ __forceinline__ void dot8(const uint4& x, const uint4& y, float& s, f16_t) {
    const f16x8 a = __builtin_bit_cast(f16x8, x), b = __builtin_bit_cast(f16x8, y);
#pragma unroll
    for (int i = 0; i < 8; i++) s = fmaf((float)a[i], (float)b[i], s);
}

// P and dS of one 32 x 32 tile, in the place of its products s = <q, k> and dp = <dO, v> - delta; ld(g): the log-sum-exp of
// registers 4 g .. 4 g + 3, so that no more of them are held than a few scores need.  dist: the lane's own position; d0: the
// position of register row 0.  ok(): which rows are visible, as bits (only asked if !all).
template <bool CAP, bool BIAS, class LD, class OK>
__device__ __forceinline__ void probs(f32x16& s, f32x16& dp, const AttnArgs& a, float slope, int dist, int d0, int h, bool all, LD ld, OK ok) {
    scores<CAP>(s, a);
    const float d = BIAS ? (float)(dist - d0 - 4 * h) : 0.f;
#pragma unroll
    for (int g = 0; g < 4; g++) {
        const f32x4 L = ld(g);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int r = 4 * g + i;
            const float t = s[r];                     // capped: the tanh, whose slope is 1 - t^2
            float x = fmaf(t, a.f, -L[i]);
            if constexpr (BIAS) x = fmaf(-slope, fabsf(d - (float)key_of(r, 0)), x);
            s[r] = exp2_(x);
            dp[r] *= s[r];
            if constexpr (CAP) dp[r] *= fmaf(-t, t, 1.f);
        }
    }
    if (!all) {
        const uint32_t m = ok();
#pragma unroll
        for (int r = 0; r < 16; r++) {
            s[r] = bit(m, r) ? s[r] : 0.f;
            dp[r] = bit(m, r) ? dp[r] : 0.f;
        }
    }
}

// what rounding took from x to y = pack8() of it
template <typename T> __device__ __forceinline__ void minus(f32x16& x, const uint4 (&y)[2]) {
#pragma unroll
    for (int m = 0; m < 2; m++) {
        const uint32_t w[4] = {y[m].x, y[m].y, y[m].z, y[m].w};
#pragma unroll
        for (int i = 0; i < 8; i++) x[8 * m + i] -= unpack<T>(w[i / 2], i & 1);
    }
}

// fp16 has 30 powers of two, and dS is about 1/T of dP: unscaled it falls among the subnormals, or to zero, long before the
// gradients do.  So each sum's dS -- a query's for dQ, a key's for dK -- is held at a power of two of its own: large at first, lowered
// when the largest |dS| passes fp16's range, to where that one has the exponent DS_AT, and taken out at the end: half a step of the
// smallest dS is then 2^-35 of the sum's largest.  P, at most 1, enters dV's product at 2^P_UP.  Measured, 2,048 tokens, an upstream gradient of
// 1e-4: dQ and dK off by 7.5e-4 and 7.8e-4 (2-norm; the results' own rounding is 7.5e-4), unscaled 3.9e-3; 8,192 tokens, 12 heads of 128 on 4:
// attn_dq 404 and attn_dkv 610 us, unscaled 371 and 573.  bf16 has fp32's range and needs none of it.
#define DS_FROM 60
#define DS_AT 10
#define DS_TOP 32768.f
#define P_UP 14
template <typename T> struct Half { static constexpr bool value = false; };
template <> struct Half<f16_t> { static constexpr bool value = true; };
__device__ __forceinline__ float max_abs(const f32x16& x) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r++) m = fmaxf(m, fabsf(x[r]));
    return half_max(m);
}
__device__ __forceinline__ float pow2(int e) { return __builtin_amdgcn_ldexpf(1.f, e); }
// by how many powers of two the largest |dS|, scaled, has to be lowered; 0: it is in range
__device__ __forceinline__ int lower_by(float mx) { return mx > DS_TOP ? DS_AT + 127 - (int)(__float_as_uint(mx) >> 23) : 0; }

// ------------------------------------------------------------------------------------------- dQ
// Four products of 32 x 32 x D per wave and half tile (S, dP, dQ twice) beside about 12 vector instructions a score; K and V tiles are
// staged once for 128 queries, two workgroups a CU.  8,192 causal tokens, 12 query heads of 128 on 4, capped: 435 us (kernel trace; the three products
// that cannot be left out take 224 us at a large library product's rate; with dS rounded once 370 us).  (GR groups of waves as in
// the forward.)
template <typename T, int D, bool CAP, bool BIAS, int GR>
__global__ __launch_bounds__(BT * GR, 2) void attn_dq(AttnArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = KT * 2 * D;
    typedef TileLoad<D, KT, BW> Load;
    __shared__ __align__(1024) unsigned char smem[GR][2][2][STAGE];
    const int tid = threadIdx.x & (BT - 1), lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), grp = GR == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / BT);
    const int heads = a.B * a.Hq;
    const int qt = uni((int)(a.tiles - 1 - blockIdx.x / heads)), bh = uni((int)(blockIdx.x % heads));
    const int b = uni(bh / a.Hq), hq = bh - b * a.Hq, hk = uni(hq / a.R);
    const int t0 = qt * BQ, off = a.Tk - a.Tq;
    const int t = t0 + 32 * w + (lane & 31), tc = min(t, a.Tq - 1), p = tc + off;
    Mask mk{a.causal, a.W, prefix_of(a, b), a.Tk};
    uint4 qf[KK], df[KK];
    float delta = 0.f;
    {
        const T* q = (const T*)a.q + b * a.q_sb + hq * a.q_sh + tc * a.q_st + 8 * h;
        const T* g = (const T*)a.dout + b * a.do_sb + hq * a.do_sh + tc * a.do_st + 8 * h;
        const int64_t at = (((int64_t)b * a.Tq + tc) * a.Hq + hq) * D + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            qf[kk] = ld16(q + 16 * kk);
            df[kk] = ld16(g + 16 * kk);
        }
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            dot8(df[kk], ld16((const T*)a.out + at + 16 * kk), delta, T{});
            dot8(df[kk], ld16((const T*)a.res + at + 16 * kk), delta, T{});
        }
    }
    delta = half_sum(delta);
    const int64_t row = (int64_t)bh * a.Tq + tc;
    int up = Half<T>::value ? DS_FROM : 0;            // dS and its sums are held at 2^up
    float lse = a.lse[row] - up;
    if (t < a.Tq && h == 0 && grp == 0) a.delta[row] = -delta;  // as attn_dkv starts its products
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
    const bool docs = a.ids != nullptr;
    const int64_t idb = (int64_t)b * a.ntd * KT;
    Span sw{t0 + off, min(t0 + BQ, a.Tq) - 1 + off, 0, 0, true}, sv{t0 + 32 * w + off, min(t0 + 32 * w + 32, a.Tq) - 1 + off, 0, 0, true};
    int dq = 0;
    if (docs) {
        const int2* range = a.range + (int64_t)b * a.ntd;
        doc_span(range, sw);
        if (sv.p0 <= sv.p1) doc_span(range, sv);
        dq = a.ids[idb + p];
        if (dq < 0) dq = -2;
    }
    const Sees see = Sees::query(mk, p);
    Walk walk(mk, sw, sv, docs ? a.range + (int64_t)b * a.ntd : nullptr, lane);
    const unsigned lds = lds_addr(smem[grp]);
    const Load lk(a.k_st, w, lane), lv(a.v_st, w, lane);
    auto load = [&](int jt, int buf) {
        lk.issue(kb, jt * KT, mk.klen - 1, lds + (2 * buf) * STAGE);
        lv.issue(vb, jt * KT, mk.klen - 1, lds + (2 * buf + 1) * STAGE);
    };
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();
    auto next = [&](int& jt, bool& some, bool& all) -> bool {
        walk.next(jt, some, all);
        const bool any = jt >= 0;
        if constexpr (GR == 2) {
            int j1 = -1;
            bool s1 = false, a1 = false;
            if (any) walk.next(j1, s1, a1);
            if (grp) { jt = j1; some = s1; all = a1; }
        }
        some = some && jt >= 0;
        return any;
    };
    int jt, jn;
    bool some = false, all = false, some_n = false, all_n = false;
    const Ops<D> ops(lane);
    bool go = next(jt, some, all), more;
    if (jt >= 0) load(jt, 0);
    for (int buf = 0; go; buf ^= 1, jt = jn, some = some_n, all = all_n, go = more) {
        more = next(jn, some_n, all_n);
        wait_vm<0>();
        tile_barrier();
        if (jn >= 0) load(jn, buf ^ 1);
        if (some) {
            const unsigned bo = lds + (2 * buf) * STAGE, rk = bo + ops.row, c = bo + ops.col, c8 = bo + ops.col8;
            // operands are read ahead of their products, the columns' before the probabilities, the second half's rows before the first
            // half's last products
            uint4 kr[4], vr[4], cr[5];
            auto rows = [&](int u, int kk) {
                const unsigned x = Ops<D>::k_step(rk, kk) + 32 * u * Tile<D>::ROWB;
                kr[kk & 3] = lds16(x);
                vr[kk & 3] = lds16(x + STAGE);
            };
            auto cols = [&](int u, int i) {           // operand i: column block i % DT of 16 keys i / DT
                cr[i % 5] = Ops<D>::at_col(Ops<D>::block(c, i % DT), Ops<D>::block(c8, i % DT), (32 * u + 16 * (i / DT)) * Tile<D>::ROWB);
            };
            rows(0, 0);
            rows(0, 1);
            rows(0, 2);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int j0 = jt * KT + 32 * u;
                f32x16 s = zero16(), dp;
#pragma unroll
                for (int r = 0; r < 16; r++) dp[r] = -delta;
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    if (kk + 3 < KK) rows(u, kk + 3);
                    s = mfma32<T>(kr[kk & 3], qf[kk], s);
                    dp = mfma32<T>(vr[kk & 3], df[kk], dp);
                    __builtin_amdgcn_sched_barrier(0);
                }
                cols(u, 0);
                cols(u, 1);
                cols(u, 2);
                probs<CAP, BIAS>(s, dp, a, slope, p, j0, h, all, [&](int) { return f32x4{lse, lse, lse, lse}; }, [&]() { return seen16(see, j0, h, j0 < mk.prefix, docs ? a.ids + idb + j0 : nullptr, dq); });
                if constexpr (Half<T>::value) {
                    const int e = lower_by(max_abs(dp));
                    if (__any(e < 0)) {
                        up += e;
                        lse = a.lse[(int64_t)bh * a.Tq + tc] - up;
                        const float f = pow2(e);
#pragma unroll
                        for (int r = 0; r < 16; r++) dp[r] *= f;
#pragma unroll
                        for (int dt = 0; dt < DT; dt++)
#pragma unroll
                            for (int r = 0; r < 16; r++) acc[dt][r] *= f;
                    }
                }
                // dS in two parts, its rounding and what that took away: a row's dS sum to zero, so that what the keys with the large
                // weights have in common (they lie along the query) cancels in dQ, but not the roundings of their dS.
                const uint4 ds[2] = {pack8<T>(dp, 0), pack8<T>(dp, 1)};
                minus<T>(dp, ds);
                const uint4 dl[2] = {pack8<T>(dp, 0), pack8<T>(dp, 1)};
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int i = 0; i <= 2 * DT; i++) {   // the second part a step behind, so that no product waits for the one before
                    if (i < 2 * DT) acc[i % DT] = mfma32<T>(cr[i % 5], ds[i / DT], acc[i % DT]);
                    if (i > 0) acc[(i - 1) % DT] = mfma32<T>(cr[(i - 1) % 5], dl[(i - 1) / DT], acc[(i - 1) % DT]);
                    if (i + 3 < 2 * DT) cols(u, i + 3);
                    else if (u == 0 && i < 2 * DT) rows(1, i + 3 - 2 * DT);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
    }
    if constexpr (GR == 2) {
        float4* so = reinterpret_cast<float4*>(smem);                 // [4 DT][thread], then the rows' powers of two
        int* su = reinterpret_cast<int*>(so + 4 * DT * BT);
        static_assert((16 * DT + 1) * BT * 4 <= (int)sizeof(smem), "a group's sums fit");
        __syncthreads();
        if (grp) {
            su[tid] = up;
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++) so[(4 * dt + g) * BT + tid] = make_float4(acc[dt][4 * g], acc[dt][4 * g + 1], acc[dt][4 * g + 2], acc[dt][4 * g + 3]);
        }
        __syncthreads();
        if (grp) return;
        float f0 = 1.f, f1 = 1.f;                     // to the smaller of the groups' powers of two
        if constexpr (Half<T>::value) {
            const int u1 = su[tid], u = min(up, u1);
            f0 = pow2(u - up);
            f1 = pow2(u - u1);
            up = u;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float4 x = so[(4 * dt + g) * BT + tid];
                acc[dt][4 * g] = fmaf(x.x, f1, acc[dt][4 * g] * f0);
                acc[dt][4 * g + 1] = fmaf(x.y, f1, acc[dt][4 * g + 1] * f0);
                acc[dt][4 * g + 2] = fmaf(x.z, f1, acc[dt][4 * g + 2] * f0);
                acc[dt][4 * g + 3] = fmaf(x.w, f1, acc[dt][4 * g + 3] * f0);
            }
    }
    float bad = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) bad = nonfinite(acc[dt], bad);
    // (a NaN log-sum-exp or, where anything is visible, delta makes all of a row NaN)
    uint32_t rows = row_bits(bad != 0.f && t < a.Tq && lse == lse && (delta == delta || lse == INFINITY));
    if (rows)
        rows &= ~row_bits(keeps<T, D>(kb, a.k_st, vb, a.v_st, kb, a.k_st, 0, mk.klen, mk.klen % KT ? mk.klen - 1 : -1, lane,
                                      [&](int j) { return sees1(see, j, docs ? a.ids + idb : nullptr, dq); }, [&](int j) { return walk.computes(j / KT); }));
    for (uint32_t left = rows; left; left &= left - 1) {              // (exact_row's, with dS in the place of P)
        const int i = __builtin_ctz(left), ti = t0 + 32 * w + i, pi = ti + off, id = lane_of(dq, i);
        const T* q = (const T*)a.q + b * a.q_sb + hq * a.q_sh + ti * a.q_st;
        const T* g = (const T*)a.dout + b * a.do_sb + hq * a.do_sh + ti * a.do_st;
        const Sees v = Sees::query(mk, pi);
        const float L = a.lse[(int64_t)bh * a.Tq + ti], de = lane_of(delta, i);
        float o1[D / 64];
        for (int e = 0; e < D / 64; e++) o1[e] = 0.f;
        for (int j1 = 0; j1 < mk.klen; j1 += 64) {
            const int j = j1 + lane;
            const bool ok = j < mk.klen && sees1(v, j, docs ? a.ids + idb : nullptr, id);
            const uint64_t m = __ballot(ok);
            if (!m) continue;
            float d = 0.f, tang;
            if (ok) {
                d = exp2_(score1<CAP, BIAS>(dot_row<T, D>(q, kb + j * a.k_st), a, slope, pi - j, tang) - L);
                d *= (dot_row<T, D>(g, vb + j * a.v_st) - de) * tang;
            }
            if (__ballot(d != d)) {
                for (int e = 0; e < D / 64; e++) o1[e] = NAN;
                break;
            }
            add_rows<T, D>(o1, d, m, kb + j1 * a.k_st, a.k_st, mk.klen - j1, lane);
        }
        for (int e = 0; e < D / 64; e++) o1[e] *= a.scale;
        put_row<T, D>((T*)a.dq + (((int64_t)b * a.Tq + ti) * a.Hq + hq) * D, lane, o1);
    }
    if (t < a.Tq && !bit(rows, lane & 31)) {
        T* out = (T*)a.dq + (((int64_t)b * a.Tq + t) * a.Hq + hq) * D;
        const float f = a.scale * pow2(-up);
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<uint2*>(out + 32 * dt + 8 * g + 4 * h) =
                    make_uint2(pack2<T>(acc[dt][4 * g] * f, acc[dt][4 * g + 1] * f), pack2<T>(acc[dt][4 * g + 2] * f, acc[dt][4 * g + 3] * f));
    }
}

// ------------------------------------------------------------------------------------------- dK, dV
// the query tiles [x0, x1) of a head that may see keys j0 .. j1
__device__ __forceinline__ void tile_rows(const AttnArgs& a, const Mask& mk, int j0, int j1, int off, int& x0, int& x1) {
    x0 = 0;
    x1 = (a.Tq + QT - 1) / QT;
    if (j0 >= mk.prefix) {
        const int lo = a.causal ? j0 : max(0, j0 - a.W + 1);          // the first position
        x0 = max(0, lo - off) / QT;
        if (a.W < a.Tk) x1 = min(x1, max(0, j1 + a.W - off + QT - 1) / QT);
    }
}
// whether tiles [x0, x1) of any head, numbered head * nx + tile, fall into [u0, u1)
__device__ __forceinline__ bool meets(int x0, int x1, int nx, int u0, int u1) {
    if (x0 >= x1) return false;
    for (int r = u0 / nx; r * nx < u1; r++)
        if (max(x0, u0 - r * nx) < min(x1, u1 - r * nx)) return true;
    return false;
}

// Two waves share 32 keys, on one SIMD: the first forms the scores and P, and sums dV = P^T dO; the second dP and dS, and sums
// dK = dS^T Q, a tile behind, with P (times the cap's slope) handed over in LDS.  Each holds one operand and one sum -- one wave
// with both had 250 registers and no room to read operands ahead: 3,100 cycles a tile of 32 x 32 pairs, with 1,024 of
// matrix work -- and one's matrix instructions run beside the other's vector ones.  Measured (as above): 658 us, 627 TFLOP/s; 176 KB
// pass through the LDS per step of four 32 x 32 tiles, which is about as long as their products take.  With dV summed by the
// second wave, too: 698 us; one wave a SIMD with a pipeline of three tiles: 681 us.
#define RING 4                                       // tiles: the two at work, two on their way

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(2 * BT, 2) void attn_dkv(AttnArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = QT * 2 * D, SLOT = 2 * STAGE, EX = 4096;
    typedef TileLoad<D, QT, BW> Load;
    __shared__ __align__(1024) unsigned char smem[RING * SLOT];      // [slot][queries, dout]
    __shared__ __align__(1024) unsigned char s_ex[2][BW][EX];        // P on its way: [tile % 2][pair][register quad][lane]
    __shared__ uint32_t s_mk[2][BW][64];                             // which pairs of a masked tile are visible: [tile % 2][pair][lane]
    __shared__ __align__(16) float s_st[RING][2][QT];                // log-sum-exp, minus delta
    __shared__ __align__(16) int s_id[RING][2 * QT];                 // the queries' documents (twice)
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const int role = uni((int)threadIdx.x / BT), w = uni((int)(threadIdx.x & (BT - 1)) >> 6);
    const int kvh = a.B * a.Hk;
    // Workgroups that read the same queries -- one part of one key/value head's -- run on one XCD, at the same time, so that its L2
    // serves them: XCD i % 8 takes every 8th (part, head).  Where those are no multiple of 8, heads alternate.
    int jt, bh, part;
    if (a.nsplit * kvh % 8 == 0) {
        const int x = blockIdx.x & 7, k = blockIdx.x >> 3, g = k / a.tiles * 8 + x;
        jt = k % a.tiles;
        part = g / kvh;
        bh = g % kvh;
    } else {
        jt = blockIdx.x / kvh % a.tiles;
        bh = blockIdx.x % kvh;
        part = blockIdx.x / (kvh * a.tiles);
    }
    jt = uni(jt);
    bh = uni(bh);
    part = uni(part);
    const int b = uni(bh / a.Hk), hk = bh - b * a.Hk;
    const int j0 = jt * BQ, j1 = min(j0 + BQ, a.Tk) - 1, off = a.Tk - a.Tq;
    const int jw = j0 + 32 * w, j = jw + (lane & 31), jc = min(j, a.Tk - 1);
    const int jw1 = min(jw + 31, a.Tk - 1);
    Mask mk{a.causal, a.W, prefix_of(a, b), a.Tk};
    int x0, x1;
    tile_rows(a, mk, j0, j1, off, x0, x1);
    const int nx = (a.Tq + QT - 1) / QT, u0 = part * a.units, u1 = min(u0 + a.units, a.R * nx);
    if (a.nsplit > 1 && !meets(x0, x1, nx, u0, u1)) return;           // the whole workgroup; attn_add knows it too
    uint4 of[KK];                                     // this wave's keys, or values, as operands
    {
        const T* x = (role ? (const T*)a.v + b * a.v_sb + hk * a.v_sh + jc * a.v_st : (const T*)a.k + b * a.k_sb + hk * a.k_sh + jc * a.k_st) + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) of[kk] = ld16(x + 16 * kk);
    }
    const bool docs = a.ids != nullptr;
    const int64_t idb = (int64_t)b * a.ntd * KT;
    Span kw{j0, j1, 0, 0, true}, kv{jw, jw1, 0, 0, true};             // document ranges of the keys
    const int2* range = docs ? a.range + (int64_t)b * a.ntd : nullptr;
    int id = 0;
    if (docs) {
        doc_span(range, kw);
        if (jw <= jw1) doc_span(range, kv);
        id = a.ids[idb + jc];
        if (id < 0) id = -2;
    }
    const Sees see = Sees::key(mk, j, a.Tk - 1);
    // the walk: heads of the group x query tiles, those of this workgroup's part.  A tile: its number, twice, plus whether every
    // pair of the wave's keys is visible, and its head; -1: none
    int r = u0 / nx - 1, base = 0, xe = 0;
    uint64_t act = 0, full = 0;
    auto next = [&]() -> int2 {
        while (!act) {
            base += 64;
            if (base >= xe) {
                if (++r * nx >= u1) return make_int2(-1, 0);
                base = max(x0, u0 - r * nx);
                xe = min(x1, u1 - r * nx);
            }
            const int x = base + lane;
            const bool in = x < xe;
            Span s{x * QT + off, min(x * QT + QT, a.Tq) - 1 + off, 0, 0, true};
            if (range && in) {
                const int2 ra = range[s.p0 / KT], rb = range[s.p1 / KT];
                s.lo = min(range_lo(ra), range_lo(rb));
                s.hi = max(ra.y, rb.y);
                s.one = range_one(ra) && range_one(rb) && ra.y == rb.y;
            }
            act = __ballot(in && mk.some(s, j0, j1) && (!range || (s.lo <= kw.hi && kw.lo <= s.hi)));
            full = __ballot(in && x * QT + QT <= a.Tq && mk.all(s, jw, jw + 31) && (!range || (s.one && kv.one && s.lo == kv.lo)));
        }
        const int i = __builtin_ctzll(act);
        act &= act - 1;
        return make_int2(2 * (base + i) + (int)(full >> i & 1), r);
    };
    const unsigned lds = lds_addr(smem), lst = lds_addr(s_st), lid = lds_addr(s_id), lex = lds_addr(s_ex) + w * EX + 16 * lane;
    // the first kind of wave loads the queries, the second dout
    const int64_t xst = role ? a.do_st : a.q_st, xsh = role ? a.do_sh : a.q_sh;
    const Load ldx(xst, w, lane);
    const T* xb = role ? (const T*)a.dout + b * a.do_sb + (int64_t)hk * a.R * xsh : (const T*)a.q + b * a.q_sb + (int64_t)hk * a.R * xsh;
    const int64_t sb = ((int64_t)b * a.Hq + hk * a.R) * a.Tq;
    auto load = [&](int2 c, int slot) {
        const int t0 = (c.x >> 1) * QT;
        ldx.issue(xb + c.y * xsh, t0, a.Tq - 1, lds + slot * SLOT + role * STAGE);
        const int t = min(t0 + (lane & 31), a.Tq - 1);                // rows past the last repeat it and are masked
        if (w == 0 && !role) dma4((h ? a.delta : a.lse) + sb + (int64_t)c.y * a.Tq + t, lst + slot * 2 * QT * 4);
        if (w == 0 && role && docs) dma4(a.ids + idb + t + off, lid + slot * 2 * QT * 4);
    };
    f32x16 sum[DT];                                   // dV, or dK
#pragma unroll
    for (int dt = 0; dt < DT; dt++) sum[dt] = zero16();
    const Ops<D> ops(lane);
    // x = sum over D of the tile's rows (the queries', or dout's) and this wave's operands, read three products ahead
    auto product = [&](f32x16& x, unsigned rows) {
        uint4 o[4];
#pragma unroll
        for (int kk = 0; kk < 3; kk++) o[kk] = lds16(Ops<D>::k_step(rows, kk));
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            if (kk + 3 < KK) o[(kk + 3) & 3] = lds16(Ops<D>::k_step(rows, kk + 3));
            x = mfma32<T>(o[kk & 3], of[kk], x);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // sum += the tile's columns times y; the first operands come with the tile
    struct Cols { uint4 o[5]; } cols;
    auto col = [&](unsigned tile, int i) {            // operand i: column block i % DT of 16 rows i / DT
        cols.o[i % 5] = Ops<D>::at_col(Ops<D>::block(tile + ops.col, i % DT), Ops<D>::block(tile + ops.col8, i % DT), 16 * (i / DT) * Tile<D>::ROWB);
    };
    auto add = [&](unsigned tile, const uint4 (&y)[2]) {
#pragma unroll
        for (int i = 0; i < 2 * DT; i++) {
            sum[i % DT] = mfma32<T>(cols.o[i % 5], y[i / DT], sum[i % DT]);
            if (i + 4 < 2 * DT) col(tile, i + 4);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    // tiles n - 1 (the second wave's), n (the first's), n + 1, n + 2
    int2 last = make_int2(-1, 0), cur = next(), nxt = make_int2(-1, 0), nn;
    if (cur.x >= 0) {
        load(cur, 0);
        nxt = next();
        if (nxt.x >= 0) load(nxt, 1);
    }
    int n = 0;
    // tile n is there, tile n - 2 is read, P of tile n - 1 handed over; the next one's loads on their way
    auto arrive = [&]() {
        if (nxt.x >= 0) wait_vm<Load::N>();
        else wait_vm<0>();
        tile_barrier();
        nn = nxt.x >= 0 ? next() : make_int2(-1, 0);
        if (nn.x >= 0) load(nn, (n + 2) & (RING - 1));
    };
    auto leave = [&]() {
        n++;
        last = cur;
        cur = nxt;
        nxt = nn;
    };
    int up = !Half<T>::value ? 0 : role ? DS_FROM + P_UP : P_UP;      // the sums are held at 2^up
    // (a loop for each kind of wave, with the same barriers: in one loop the sums were copied where its branches meet)
    if (!role) {
        while (cur.x >= 0) {
            arrive();
            const int slot = n & (RING - 1), t0 = (cur.x >> 1) * QT;
            const unsigned tile = lds + slot * SLOT;
            f32x16 s = zero16();
            product(s, tile + ops.row);
#pragma unroll
            for (int i = 0; i < 4; i++) col(tile + STAGE, i);
            f32x4 L[4];
#pragma unroll
            for (int g = 0; g < 4; g++) {
                L[g] = lds4f(lst + slot * 2 * QT * 4 + 32 * g + 16 * h);
                if constexpr (Half<T>::value) L[g] -= (float)P_UP;
            }
            __builtin_amdgcn_sched_barrier(0);
            scores<CAP>(s, a);
            const float slope = BIAS ? a.slopes[hk * a.R + cur.y] * LOG2E : 0.f, d = (float)(j - t0 - off - 4 * h);
            f32x16 g;                                 // what dP becomes dS by
#pragma unroll
            for (int e = 0; e < 16; e++) {
                const float t = s[e];                 // capped: the tanh, whose slope is 1 - t^2
                float x = fmaf(t, a.f, -L[e >> 2][e & 3]);
                if constexpr (BIAS) x = fmaf(-slope, fabsf(d - (float)key_of(e, 0)), x);
                s[e] = exp2_(x);
                if constexpr (CAP) g[e] = s[e] * fmaf(-t, t, 1.f);
            }
            if (!(cur.x & 1)) {
                const uint32_t m = seen16(see, t0 + off, h, false, docs ? s_id[slot] : nullptr, id);
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = bit(m, e) ? s[e] : 0.f;
                s_mk[n & 1][w][lane] = m;
            }
            if constexpr (!CAP) g = s;
            unsigned char* ex = s_ex[n & 1][w] + 16 * lane;
#pragma unroll
            for (int q = 0; q < 4; q++) *reinterpret_cast<float4*>(ex + 1024 * q) = make_float4(g[4 * q], g[4 * q + 1], g[4 * q + 2], g[4 * q + 3]);
            const uint4 y[2] = {pack8<T>(s, 0), pack8<T>(s, 1)};
            __builtin_amdgcn_sched_barrier(0);
            add(tile + STAGE, y);
            leave();
        }
        if (n) arrive();                              // the second wave's last tile
    } else if (cur.x >= 0) {
        arrive();
        leave();
        while (last.x >= 0) {
            arrive();
            const int slot = (n - 1) & (RING - 1);
            const unsigned tile = lds + slot * SLOT;
            f32x16 dp;
#pragma unroll
            for (int g = 0; g < 4; g++) {             // minus delta
                const f32x4 y = lds4f(lst + slot * 2 * QT * 4 + QT * 4 + 32 * g + 16 * h);
                dp[4 * g] = y.x; dp[4 * g + 1] = y.y; dp[4 * g + 2] = y.z; dp[4 * g + 3] = y.w;
            }
            product(dp, tile + STAGE + ops.row);
            f32x4 p[4];
#pragma unroll
            for (int q = 0; q < 4; q++) p[q] = lds4f(lex + ((n - 1) & 1) * BW * EX + 1024 * q);
#pragma unroll
            for (int i = 0; i < 4; i++) col(tile, i);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int e = 0; e < 16; e++) dp[e] *= p[e >> 2][e & 3];
            if (!(last.x & 1)) {                      // a masked pair's dP, and with a cap its P, may be anything
                const uint32_t m = s_mk[(n - 1) & 1][w][lane];
#pragma unroll
                for (int e = 0; e < 16; e++) {
                    asm volatile("" : "+v"(dp[e]));   // (not ahead of the branch)
                    dp[e] = __uint_as_float(__float_as_uint(dp[e]) & (uint32_t)((int)(m << (31 - e)) >> 31));
                }
            }
            if constexpr (Half<T>::value) {           // (P comes at 2^P_UP)
                const float mx = max_abs(dp);
                const int e = lower_by(mx * pow2(up - P_UP));
                if (__any(e < 0)) {
                    up += e;
                    const float g = pow2(e);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++)
#pragma unroll
                        for (int r = 0; r < 16; r++) sum[dt][r] *= g;
                }
                const float g = pow2(up - P_UP);
#pragma unroll
                for (int r = 0; r < 16; r++) dp[r] *= g;
            }
            const uint4 y[2] = {pack8<T>(dp, 0), pack8<T>(dp, 1)};
            __builtin_amdgcn_sched_barrier(0);
            add(tile, y);
            leave();
        }
    }
    const float one = role ? a.scale : 1.f, f = one * pow2(-up);
    float bad = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) bad = nonfinite(sum[dt], bad);
    uint32_t rows = row_bits(bad != 0.f && j < a.Tk);
    if (rows) {
        Ill<T, D> ill;
        auto met = [&](int x) {                       // tile x was walked
            const Span s{x * QT + off, min(x * QT + QT, a.Tq) - 1 + off, 0, 0, true};
            if (!mk.some(s, j0, j1)) return false;
            if (!range) return true;
            const int2 ra = range[s.p0 / KT], rb = range[s.p1 / KT];
            return min(range_lo(ra), range_lo(rb)) <= kw.hi && kw.lo <= max(ra.y, rb.y);
        };
        auto open = [&]() { return (rows & row_bits(!ill.lost)) != 0; };               // some row is not decided yet
        for (int rr = u0 / nx; rr * nx < u1 && open(); rr++) {
            const int hq = hk * a.R + rr, te = min(min(x1, u1 - rr * nx) * QT, a.Tq);
            const T* qh = (const T*)a.q + b * a.q_sb + hq * a.q_sh;
            const T* gh = (const T*)a.dout + b * a.do_sb + hq * a.do_sh;
            const int64_t at = ((int64_t)b * a.Hq + hq) * a.Tq;
            for (int t1 = max(x0, u0 - rr * nx) * QT; t1 < te && open(); t1 += 64) {
                const int t = t1 + lane;
                bool is = false, gone = false;        // not finite; all of what it adds is NaN
                if (t < te) {
                    const float L = a.lse[at + t], de = role ? a.delta[at + t] : 0.f;
                    gone = L != L || de != de;
                    is = gone || !(fabsf(de) < INFINITY) || !finite_row<T, D>(qh + t * a.q_st) || !finite_row<T, D>(gh + t * a.do_st);
                }
                const uint64_t all = __ballot(gone);
                for (uint64_t m = __ballot(is); m; m &= m - 1) {
                    const int i = __builtin_ctzll(m), ti = t1 + i;
                    const bool sees = sees1(see, ti + off, docs ? a.ids + idb : nullptr, id);
                    ill.lost = ill.lost || (sees && (all >> i & 1));
                    ill.add(role ? qh + ti * a.q_st : gh + ti * a.do_st, sees, met(ti / QT), ti == a.Tq - 1 && a.Tq % QT, lane);
                }
            }
        }
        rows &= ~row_bits(ill.kept());
    }
    float* const po = a.part + ((int64_t)(part * a.tiles + jt) * kvh + bh) * 2 * BQ * D + (role ? 0 : BQ * D) + 32 * w * D;
    for (uint32_t left = rows; left; left &= left - 1) {              // a key's sums from the queries that see it, of this part
        const int i = __builtin_ctz(left), ji = jw + i, idi = lane_of(id, i);
        const T* k = (const T*)a.k + b * a.k_sb + hk * a.k_sh + ji * a.k_st;
        const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh + ji * a.v_st;
        const Sees se = lane_of(see, i);
        float o1[D / 64];
        for (int e = 0; e < D / 64; e++) o1[e] = 0.f;
        for (int rr = u0 / nx; rr * nx < u1; rr++) {
            const int hq = hk * a.R + rr;
            const T* qh = (const T*)a.q + b * a.q_sb + hq * a.q_sh;
            const T* gh = (const T*)a.dout + b * a.do_sb + hq * a.do_sh;
            const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
            const int te = min(min(x1, u1 - rr * nx) * QT, a.Tq);
            for (int t1 = max(x0, u0 - rr * nx) * QT; t1 < te; t1 += 64) {
                const int t = t1 + lane;
                const bool ok = t < te && sees1(se, t + off, docs ? a.ids + idb : nullptr, idi);
                const uint64_t m = __ballot(ok);
                if (!m) continue;
                float d = 0.f, tang;
                if (ok) {
                    const int64_t at = ((int64_t)b * a.Hq + hq) * a.Tq + t;
                    d = exp2_(score1<CAP, BIAS>(dot_row<T, D>(qh + t * a.q_st, k), a, slope, t + off - ji, tang) - a.lse[at]);
                    if (role) d *= (dot_row<T, D>(gh + t * a.do_st, v) + a.delta[at]) * tang;
                }
                if (__ballot(d != d)) {
                    for (int e = 0; e < D / 64; e++) o1[e] = NAN;
                    rr = a.R;
                    break;
                }
                add_rows<T, D>(o1, d, m, role ? qh + t1 * a.q_st : gh + t1 * a.do_st, role ? a.q_st : a.do_st, te - t1, lane);
            }
        }
        for (int e = 0; e < D / 64; e++) o1[e] *= one;
        if (a.nsplit > 1) {
            for (int e = 0; e < D / 64; e++) po[i * D + lane * (D / 64) + e] = o1[e];
        } else {
            put_row<T, D>((T*)(role ? a.dk : a.dv) + (((int64_t)b * a.Tk + ji) * a.Hk + hk) * D, lane, o1);
        }
    }
    if (bit(rows, lane & 31)) return;
    if (a.nsplit > 1) {
        float* o = po + (lane & 31) * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<float4*>(o + 32 * dt + 8 * g) = make_float4(sum[dt][4 * g] * f, sum[dt][4 * g + 1] * f, sum[dt][4 * g + 2] * f, sum[dt][4 * g + 3] * f);
    } else if (j < a.Tk) {
        T* o = (T*)(role ? a.dk : a.dv) + (((int64_t)b * a.Tk + j) * a.Hk + hk) * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<uint2*>(o + 32 * dt + 8 * g) =
                    make_uint2(pack2<T>(sum[dt][4 * g] * f, sum[dt][4 * g + 1] * f), pack2<T>(sum[dt][4 * g + 2] * f, sum[dt][4 * g + 3] * f));
    }
}

// dK and dV of 32 keys from the parts' sums, added in order; 32 rows x D / 4 lanes of 4 values
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_add(AttnArgs a) {
    const int kvh = a.B * a.Hk, bh = blockIdx.x % kvh, q4 = blockIdx.x / kvh, jt = q4 / (BQ / 32);
    const int b = bh / a.Hk, hk = bh - b * a.Hk, off = a.Tk - a.Tq;
    const int j0 = jt * BQ, j1 = min(j0 + BQ, a.Tk) - 1;
    const Mask mk{a.causal, a.W, prefix_of(a, b), a.Tk};
    int x0, x1;
    tile_rows(a, mk, j0, j1, off, x0, x1);
    const int nx = (a.Tq + QT - 1) / QT, lane = threadIdx.x & 63;
    const uint64_t parts = __ballot(lane < a.nsplit && meets(x0, x1, nx, lane * a.units, min((lane + 1) * a.units, a.R * nx)));
    for (int e = threadIdx.x; e < 32 * (D / 4) * 2; e += 256) {
        const int which = e / (32 * (D / 4)), i = e % (32 * (D / 4)), row = (q4 % (BQ / 32)) * 32 + i / (D / 4), c = 4 * (i % (D / 4));
        if (j0 + row >= a.Tk) continue;
        const float* from = a.part + ((int64_t)jt * kvh + bh) * 2 * BQ * D + which * BQ * D + row * D + c;
        const int64_t st = (int64_t)a.tiles * kvh * 2 * BQ * D;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint64_t m = parts; m;) {                // in order, four loads on their way
            float4 x[4];
            bool in[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                in[k] = m != 0;
                x[k] = *reinterpret_cast<const float4*>(from + (in[k] ? __builtin_ctzll(m) : __builtin_ctzll(parts)) * st);
                m &= m - 1;
            }
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (in[k]) { s.x += x[k].x; s.y += x[k].y; s.z += x[k].z; s.w += x[k].w; }
        }
        put4<T>(which ? a.dv : a.dk, nullptr, (((int64_t)b * a.Tk + j0 + row) * a.Hk + hk) * D + c, s.x, s.y, s.z, s.w);
    }
}

template <typename T, int D, bool CAP, bool BIAS>
void launch_one(AttnArgs a, bool keys, hipStream_t st) {
    if (keys) {
        a.tiles = (a.Tk + BQ - 1) / BQ;
        slothost::launch(attn_dkv<T, D, CAP, BIAS>, dim3((unsigned)((int64_t)a.tiles * a.nsplit * a.B * a.Hk)), dim3(2 * BT), 0, st, a);
    } else {
        a.tiles = (a.Tq + BQ - 1) / BQ;
        if (a.groups == 2) slothost::launch(attn_dq<T, D, CAP, BIAS, 2>, dim3((unsigned)((int64_t)a.tiles * a.B * a.Hq)), dim3(2 * BT), 0, st, a);
        else slothost::launch(attn_dq<T, D, CAP, BIAS, 1>, dim3((unsigned)((int64_t)a.tiles * a.B * a.Hq)), dim3(BT), 0, st, a);
    }
}
template <typename T, int D>
void launch_bwd(const AttnArgs& a, bool cap, bool keys, hipStream_t st) {
    if (cap) a.slopes ? launch_one<T, D, true, true>(a, keys, st) : launch_one<T, D, true, false>(a, keys, st);
    else a.slopes ? launch_one<T, D, false, true>(a, keys, st) : launch_one<T, D, false, false>(a, keys, st);
}

template <typename T, int D>
void launch_add(AttnArgs a, hipStream_t st) {
    a.tiles = (a.Tk + BQ - 1) / BQ;
    slothost::launch(attn_add<T, D>, dim3((unsigned)((int64_t)a.tiles * (BQ / 32) * a.B * a.Hk)), dim3(256), 0, st, a);
}

// Parts of the queries per key tile, 64 at most.  A part costs the write and the read of its sums, about as long as 20 query tiles take, so
// where the key tiles fill the card, keys are split into parts of 48 query tiles at least.  Where they leave CUs idle (under 400 / 2 tiles), a part
// of 8 pays already: 4 heads of 128 x 4,096 tokens 145 -> 78 us with the addition, 12 heads on 4 x 1,024 tokens 111 -> 41, 2 heads of 64 on
// 1 x 2,048 tokens 109 -> 29, 3 x 6 heads of 64 x 1,111 tokens 36 -> 30.
void parts(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int causal, int64_t W, bool prefix, int& nsplit, int& units) {
    const int64_t R = Hq / Hk, nx = (Tq + QT - 1) / QT, tiles = (Tk + BQ - 1) / BQ * B * Hk;
    int64_t rows = causal ? Tq - Tq / 2 : Tq;                         // of a head that see a key tile, about
    if (!prefix && W < Tk) rows = std::min(rows, (causal ? W : 2 * W) + BQ);
    const int64_t work = R * ((rows + QT - 1) / QT);
    const int64_t n = tiles >= 512 ? 1 : std::max({(int64_t)1, std::min({(int64_t)64, (1023 + tiles) / tiles, work / 48}), std::min({(int64_t)64, 400 / tiles, work / 8})});
    units = (int)((R * nx + n - 1) / n);
    nsplit = (int)((R * nx + units - 1) / units);
}

}  // namespace

// ======================================================================================== C-ABI
extern "C" size_t slotattn_bwd_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, int causal, int64_t window,
                                         int has_prefix) {
    if (B < 1 || Tq < 1 || Tk < 1 || Hk < 1 || Hq < Hk || Hq % Hk) return 0;
    int n, u;
    parts(B, Tq, Tk, Hq, Hk, causal, window, has_prefix, n, u);
    return n == 1 ? 0 : (size_t)((Tk + BQ - 1) / BQ * B * Hk * n) * 2 * BQ * D * sizeof(float);
}

extern "C" int slotattn_bwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                            int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, int64_t B, int64_t Tq,
                            int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, float scale, int causal, int64_t window, float cap,
                            const float* slopes, const void* docs, const int32_t* prefix, const void* out, const void* res,
                            const float* lse, const void* dout, int64_t do_sb, int64_t do_sh, int64_t do_st, void* workspace, float* delta, void* dq,
                            void* dk, void* dv, void* stream) {
    if (int r = slotattn_host::check(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st, dtype, B, Tq, Tk, Hq, Hk, D, scale, window, cap)) return r;
    if (Tq > Tk) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: more queries than keys");
    if (!out || !res || !lse || !dout || !delta || !dq || !dk || !dv) return fail(SLOTSCAN_ERR_NULL, "slotattn_bwd: a required pointer is NULL");
    if (!al16(out) || !al16(res) || !al16(dout) || !al16(dq) || !al16(dk) || !al16(dv) || !al16(docs) || !al16(workspace) || (do_sb | do_sh | do_st) % 8)
        return fail(SLOTSCAN_ERR_ALIGN, "slotattn_bwd: rows of out, res, dout, dq, dk and dv, docs and the workspace must be 16-byte aligned");
    if (do_st < 0 || do_st >= SLOTATTN_MAX_ST) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: token strides must be in [0, 2^25)");
    if ((Tq + BQ - 1) / BQ * B * Hq > 0x7fffffffLL || (Tk + BQ - 1) / BQ * B * Hk > 0x7fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: shape too large");
    AttnArgs a = slotattn_host::args(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st, B, Tq, Tk, Hq, Hk, scale, causal, window, cap,
                                     slopes, docs, prefix);
    parts(B, Tq, Tk, Hq, Hk, causal, window, prefix != nullptr, a.nsplit, a.units);
    if (a.nsplit > 1 && !workspace) return fail(SLOTSCAN_ERR_NULL, "slotattn_bwd: workspace is NULL");
    if ((Tk + BQ - 1) / BQ * B * Hk * std::max(a.nsplit, BQ / 32) > 0x7fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: shape too large");
    a.part = (float*)workspace;
    a.groups = (Tq + BQ - 1) / BQ * B * Hq <= 256 ? 2 : 1;           // as in the forward
    a.out = (void*)out;
    a.res = (void*)res;
    a.lse = (float*)lse;
    a.dout = dout;
    a.do_sb = do_sb; a.do_sh = do_sh; a.do_st = do_st;
    a.delta = delta;
    a.dq = dq; a.dk = dk; a.dv = dv;
    hipStream_t st = (hipStream_t)stream;
    const bool cp = cap > 0.f;
    for (int keys = 0; keys < 2; keys++) {
        slothost::Scope sc(keys ? SLOTSCAN_K_ATTN_DKV : SLOTSCAN_K_ATTN_DQ, st);
        if (dtype == SLOTSCAN_BF16) D == 128 ? launch_bwd<bf16_t, 128>(a, cp, keys, st) : launch_bwd<bf16_t, 64>(a, cp, keys, st);
        else D == 128 ? launch_bwd<f16_t, 128>(a, cp, keys, st) : launch_bwd<f16_t, 64>(a, cp, keys, st);
        hipError_t e = hipGetLastError();
        if (e != hipSuccess) return hip_fail(e, keys ? "attn_dkv launch" : "attn_dq launch");
    }
    if (a.nsplit == 1) return 0;
    slothost::Scope sc(SLOTSCAN_K_ATTN_JOIN, st);
    if (dtype == SLOTSCAN_BF16) D == 128 ? launch_add<bf16_t, 128>(a, st) : launch_add<bf16_t, 64>(a, st);
    else D == 128 ? launch_add<f16_t, 128>(a, st) : launch_add<f16_t, 64>(a, st);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "attn_add launch");
}
