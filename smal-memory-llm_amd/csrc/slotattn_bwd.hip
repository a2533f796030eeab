// Exact attention of any range for MI355X (gfx950), backward (semantics: slotattn.h).  With P = softmax, dP = dO V^T,
// delta = rowsum(dO o O) and the cap's slope 1 - tanh^2:
//     dS = P (dP - delta) (1 - tanh^2),   dV = P^T dO,   dQ = scale dS K,   dK = scale dS^T Q
// P comes back from the rows' log-sum-exp.  Two kernels, each of which owns what it sums, so nothing is added atomically:
//   attn_dq    128 queries of one head per workgroup, walking the visible key tiles (as the forward does); it forms delta
//   attn_dkv   128 keys of one key/value head per workgroup, walking the query tiles of every head of the group that see them
// The price is that the scores and dP are formed twice: 7 products where one kernel with atomic dQ would need 5.
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
#define QT 64                                        // query rows of a tile of attn_dkv

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
// position of register row 0.  ok(g, o): which of those four are visible (only asked if !all).
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
#pragma unroll
        for (int g = 0; g < 4; g++) {
            bool o[4];
            ok(g, o);
#pragma unroll
            for (int i = 0; i < 4; i++) {
                s[4 * g + i] = o[i] ? s[4 * g + i] : 0.f;
                dp[4 * g + i] = o[i] ? dp[4 * g + i] : 0.f;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------- dQ
template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(BT, 2) void attn_dq(AttnArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = KT * 2 * D;
    typedef TileLoad<D, KT, BW> Load;
    __shared__ __align__(1024) unsigned char smem[2][2][STAGE];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int heads = a.B * a.Hq;
    const int qt = a.tiles - 1 - blockIdx.x / heads, bh = blockIdx.x % heads;
    const int b = bh / a.Hq, hq = bh - b * a.Hq, hk = hq / a.R;
    const int t0 = qt * BQ, off = a.Tk - a.Tq;
    const int t = t0 + 32 * w + (lane & 31), tc = min(t, a.Tq - 1), p = tc + off;
    Mask mk{a.causal, a.W, a.prefix ? a.prefix[b] : 0, a.Tk};
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
    const float lse = a.lse[row];
    if (t < a.Tq && h == 0) a.delta[row] = -delta;  // as attn_dkv starts its products
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
    const bool docs = a.ids != nullptr;
    const int64_t idb = (int64_t)b * a.ntd * KT;
    Span sw{t0 + off, min(t0 + BQ, a.Tq) - 1 + off, 0, 0, true}, sv{t0 + 32 * w + off, min(t0 + 32 * w + 32, a.Tq) - 1 + off, 0, 0, true};
    int dq = 0;
    if (docs) {
        rows_range(a.ids, idb, sw.p0, sw.p1 - sw.p0 + 1, lane, sw);
        rows_range(a.ids, idb, min(sv.p0, sw.p1), max(sv.p1 - sv.p0 + 1, 1), lane, sv);
        dq = a.ids[idb + p];
        if (dq < 0) dq = -2;
    }
    Walk walk(mk, sw, sv, docs ? a.range + (int64_t)b * a.ntd : nullptr, lane);
    const unsigned lds = lds_addr(smem);
    const Load lk(a.k_st, w, lane), lv(a.v_st, w, lane);
    auto load = [&](int jt, int buf) {
        lk.issue(kb, jt * KT, mk.klen - 1, lds + (2 * buf) * STAGE);
        lv.issue(vb, jt * KT, mk.klen - 1, lds + (2 * buf + 1) * STAGE);
    };
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();
    int jt, jn;
    bool some, all, some_n = false, all_n = false;
    const Ops<D> ops(lane);
    walk.next(jt, some, all);
    if (jt >= 0) load(jt, 0);
    for (int buf = 0; jt >= 0; buf ^= 1, jt = jn, some = some_n, all = all_n) {
        walk.next(jn, some_n, all_n);
        wait_vm<0>();
        tile_barrier();
        if (jn >= 0) load(jn, buf ^ 1);
        if (some) {
            const unsigned bo = lds + (2 * buf) * STAGE, rk = bo + ops.row, c = bo + ops.col, c8 = bo + ops.col8;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int j0 = jt * KT + 32 * u, at = 32 * u * Tile<D>::ROWB;
                f32x16 s = zero16(), dp;
#pragma unroll
                for (int r = 0; r < 16; r++) dp[r] = -delta;
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    const unsigned x = Ops<D>::k_step(rk, kk);
                    s = mfma32<T>(lds16(x + at), qf[kk], s);
                    dp = mfma32<T>(lds16(x + at + STAGE), df[kk], dp);
                }
                probs<CAP, BIAS>(s, dp, a, slope, p, j0, h, all, [&](int) { return f32x4{lse, lse, lse, lse}; }, [&](int g, bool (&o)[4]) {
                    const int j = j0 + 8 * g + 4 * h;
                    const int4 id = docs ? *reinterpret_cast<const int4*>(a.ids + idb + j) : make_int4(0, 0, 0, 0);
                    o[0] = mk.sees(p, j) && id.x == dq;
                    o[1] = mk.sees(p, j + 1) && id.y == dq;
                    o[2] = mk.sees(p, j + 2) && id.z == dq;
                    o[3] = mk.sees(p, j + 3) && id.w == dq;
                });
                const uint4 ds[2] = {pack8<T>(dp, 0), pack8<T>(dp, 1)};
#pragma unroll
                for (int dt = 0; dt < DT; dt++) {
                    const unsigned x = Ops<D>::block(c, dt), x8 = Ops<D>::block(c8, dt);
#pragma unroll
                    for (int mm = 0; mm < 2; mm++) acc[dt] = mfma32<T>(Ops<D>::at_col(x, x8, at + 16 * mm * Tile<D>::ROWB), ds[mm], acc[dt]);
                }
            }
        }
    }
    if (t < a.Tq) {
        T* out = (T*)a.dq + (((int64_t)b * a.Tq + t) * a.Hq + hq) * D;
        const float f = a.scale;
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

// Each wave holds 32 keys and values as operands and their dK, dV as sums, one wave per SIMD.  A step interleaves three
// blocks of 32 queries: the products of block m + 1, P and dS of block m, the sums of block m - 1, which do not depend on each
// other, so the matrix and the vector units run at the same time within the wave.  The queries' and dout's tiles of 64 rows
// come through a ring of RING, up to FLY of them in flight behind the one that is needed next.
#define RING 4
#define FLY 2

template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(BT, 1) void attn_dkv(AttnArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = QT * 2 * D, SLOT = 2 * STAGE, RC = 16 / KK, HALF = 32 * 2 * D;
    static_assert(KK == 2 * DT, "a step's chunks: one k step of the next tile's products, one operand of the last one's sums");
    typedef TileLoad<D, QT, BW> Load;
    constexpr int PER = 2 * Load::N;
    __shared__ __align__(1024) unsigned char smem[RING * SLOT];      // [slot][queries, dout]
    __shared__ __align__(16) float s_st[RING][2][QT];                // log-sum-exp, minus delta
    __shared__ __align__(16) int s_id[RING][QT];                     // the queries' documents
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
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
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int j0 = jt * BQ, j1 = min(j0 + BQ, a.Tk) - 1, off = a.Tk - a.Tq;
    const int jw = j0 + 32 * w, j = jw + (lane & 31), jc = min(j, a.Tk - 1);
    const int jw1 = min(jw + 31, a.Tk - 1);
    Mask mk{a.causal, a.W, a.prefix ? a.prefix[b] : 0, a.Tk};
    int x0, x1;
    tile_rows(a, mk, j0, j1, off, x0, x1);
    const int nx = (a.Tq + QT - 1) / QT, u0 = part * a.units, u1 = min(u0 + a.units, a.R * nx);
    if (a.nsplit > 1 && !meets(x0, x1, nx, u0, u1)) return;           // the whole workgroup; attn_add knows it too
    uint4 kf[KK], vf[KK];
    {
        const T* k = (const T*)a.k + b * a.k_sb + hk * a.k_sh + jc * a.k_st + 8 * h;
        const T* v = (const T*)a.v + b * a.v_sb + hk * a.v_sh + jc * a.v_st + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            kf[kk] = ld16(k + 16 * kk);
            vf[kk] = ld16(v + 16 * kk);
        }
    }
    const bool docs = a.ids != nullptr;
    const int64_t idb = (int64_t)b * a.ntd * KT;
    Span kw{j0, j1, 0, 0, true}, kv{jw, jw1, 0, 0, true};             // document ranges of the keys
    int dk_ = 0;
    if (docs) {
        rows_range(a.ids, idb, j0, j1 - j0 + 1, lane, kw);
        rows_range(a.ids, idb, min(jw, j1), max(jw1 - jw + 1, 1), lane, kv);
        dk_ = a.ids[idb + jc];
        if (dk_ < 0) dk_ = -2;
    }
    const int2* range = docs ? a.range + (int64_t)b * a.ntd : nullptr;
    // the walk: heads of the group x query tiles, those of this workgroup's part.  A tile as one number: head of the group,
    // tile, whether every pair of the wave's keys is visible; -1: none
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
    const unsigned lds = lds_addr(smem), lst = lds_addr(s_st), lid = lds_addr(s_id);
    const Load lq(a.q_st, w, lane), ld(a.do_st, w, lane);
    const T* qb = (const T*)a.q + b * a.q_sb + (int64_t)hk * a.R * a.q_sh;
    const T* db = (const T*)a.dout + b * a.do_sb + (int64_t)hk * a.R * a.do_sh;
    const int64_t sb = ((int64_t)b * a.Hq + hk * a.R) * a.Tq;
    auto load = [&](int2 c, int slot) {
        const int t0 = (c.x >> 1) * QT;
        lq.issue(qb + c.y * a.q_sh, t0, a.Tq - 1, lds + slot * SLOT);
        ld.issue(db + c.y * a.do_sh, t0, a.Tq - 1, lds + slot * SLOT + STAGE);
        const int t = min(t0 + lane, a.Tq - 1);                       // rows past the last repeat it and are masked
        if (w < 2) dma4((w ? a.delta : a.lse) + sb + (int64_t)c.y * a.Tq + t, lst + (2 * slot + w) * QT * 4);
        if (w == 2 && docs) dma4(a.ids + idb + t + off, lid + slot * QT * 4);
    };
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) dk[dt] = dv[dt] = zero16();
    const Ops<D> ops(lane);
    uint4 pp[2], ds[2];                               // P and dS of the last tile as operands
    // a block of 32 query rows: its tile's slot and which half.  Its products start from 0 and minus delta.
    auto start = [&](f32x16& s, f32x16& dp, int blk) {
        s = zero16();
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const f32x4 y = lds4f(lst + (blk >> 1) * 2 * QT * 4 + QT * 4 + (blk & 1) * 128 + 32 * g + 16 * h);
            dp[4 * g] = y.x; dp[4 * g + 1] = y.y; dp[4 * g + 2] = y.z; dp[4 * g + 3] = y.w;
        }
        asm volatile("s_nop 3" : "+v"(s), "+v"(dp)); // between a register's write and a matrix instruction of an asm block
    };
    auto at = [&](int blk) { return lds + (blk >> 1) * SLOT + (blk & 1) * HALF; };
    // P and dS of a block whose pairs are not all visible: 0 for the others
    auto mask = [&](f32x16& s, f32x16& dp, int blk, int t0) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int tq = t0 + 8 * g + 4 * h;
            const int4 id = docs ? *reinterpret_cast<const int4*>(&s_id[blk >> 1][(blk & 1) * 32 + 8 * g + 4 * h]) : make_int4(0, 0, 0, 0);
            const int ids[4] = {id.x, id.y, id.z, id.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const bool o = tq + i < a.Tq && mk.sees(tq + i + off, j) && ids[i] == dk_;
                s[4 * g + i] = o ? s[4 * g + i] : 0.f;
                dp[4 * g + i] = o ? dp[4 * g + i] : 0.f;
            }
        }
    };
    // One step: the products of block bn into (sN, dN), P and dS of block bc (rows from t0, head r of the group) from (s, dp), the
    // sums of block bp.
    auto step = [&](f32x16& s, f32x16& dp, f32x16& sN, f32x16& dN, int bp, int bc, int bn, int t0, int r, bool all) {
        const unsigned rn = at(bn) + ops.row, cp = at(bp) + ops.col, cp8 = at(bp) + ops.col8;
        float c0 = 1.f, c1 = 0.f, c2 = 0.f, c3 = 0.f, c4 = 0.f;
        if constexpr (CAP) {
            if (poly_holds(s, a)) {
                c0 = a.t0; c1 = a.t1; c2 = a.t2; c3 = a.t3; c4 = a.t4;
            } else {                                  // the polynomial below then is its argument
#pragma unroll
                for (int e = 0; e < 16; e++) s[e] = tanh_any(s[e], a);
            }
        }
        f32x4 L[4];
#pragma unroll
        for (int g = 0; g < 4; g++) L[g] = lds4f(lst + (bc >> 1) * 2 * QT * 4 + (bc & 1) * 128 + 32 * g + 16 * h);
        start(sN, dN, bn);
        const float slope = BIAS ? a.slopes[hk * a.R + r] * LOG2E : 0.f, d = (float)(j - t0 - off - 4 * h);
        uint4 oq = lds16(Ops<D>::k_step(rn, 0)), od = lds16(Ops<D>::k_step(rn, 0) + STAGE);
        uint4 xq = Ops<D>::at_col(cp, cp8, 0), xd = Ops<D>::at_col(cp, cp8, STAGE);
        float t;
        // half of a score's way to P and dS: its tanh where it is capped, then the rest
        auto half = [&](int x) {
            const int e = x >> 1;
            if ((x & 1) == 0) {
                t = s[e];                             // capped: the tanh, whose slope is 1 - t^2
                if constexpr (CAP) {
                    const float y = t * t;
                    t *= fmaf(fmaf(fmaf(fmaf(c4, y, c3), y, c2), y, c1), y, c0);
                }
                return;
            }
            float z = fmaf(t, a.f, -L[e >> 2][e & 3]);
            if constexpr (BIAS) z = fmaf(-slope, fabsf(d - (float)key_of(e, 0)), z);
            s[e] = exp2_(z);
            dp[e] *= s[e];
            if constexpr (CAP) dp[e] *= fmaf(-t, t, 1.f);
        };
#pragma unroll
        for (int i = 0; i < KK; i++) {
            const uint4 pq = oq, pd = od, yq = xq, yd = xd;
            // one matrix instruction, then as much of the vector work as hides it
#pragma unroll
            for (int x = 0; x < 4; x++) {
                if (x == 0) mfma_vec<T>(sN, pq, kf[i]);
                if (x == 1) mfma_acc<T>(dv[i / 2], yd, pp[i & 1]);
                if (x == 2) mfma_vec<T>(dN, pd, vf[i]);
                if (x == 3) mfma_acc<T>(dk[i / 2], yq, ds[i & 1]);
                if (i + 1 < KK) {
                    // column block (i + 1) / 2, rows 16 ((i + 1) % 2) ..
                    const int ro = 16 * ((i + 1) & 1) * Tile<D>::ROWB;
                    if (x == 0) oq = lds16(Ops<D>::k_step(rn, i + 1));
                    if (x == 1) xd = Ops<D>::at_col(Ops<D>::block(cp, (i + 1) / 2), Ops<D>::block(cp8, (i + 1) / 2), ro + STAGE);
                    if (x == 2) od = lds16(Ops<D>::k_step(rn, i + 1) + STAGE);
                    if (x == 3) xq = Ops<D>::at_col(Ops<D>::block(cp, (i + 1) / 2), Ops<D>::block(cp8, (i + 1) / 2), ro);
                }
#pragma unroll
                for (int y = 0; y < RC / 2; y++) half(2 * RC * i + x * (RC / 2) + y);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (!all) mask(s, dp, bc, t0);
#pragma unroll
        for (int m = 0; m < 2; m++) {
            pp[m] = pack8<T>(s, m);
            ds[m] = pack8<T>(dp, m);
        }
        mfma_settle();
    };
    // tiles n (at hand), n + 1 .. n + 1 + FLY (loaded or on their way)
    int2 tile[FLY + 2];
    int fly = 0;                                      // tiles issued and not yet waited for
#pragma unroll
    for (int i = 0; i < FLY + 1; i++) {
        tile[i] = i && tile[i - 1].x < 0 ? make_int2(-1, 0) : next();
        if (tile[i].x >= 0) {
            load(tile[i], i);
            fly++;
        }
    }
    // the oldest of the tiles in flight has landed: at most the younger ones' loads are outstanding
    auto landed = [&]() {
        fly--;
        if (fly >= 2) wait_vm<2 * PER>();
        else if (fly == 1) wait_vm<PER>();
        else wait_vm<0>();
        tile_barrier();
    };
    if (tile[0].x >= 0) {
        f32x16 s, dp, sN, dN;
        // the step before the first: nothing, from a slot of zeros (the ring reaches it only behind another barrier)
        pp[0] = pp[1] = ds[0] = ds[1] = make_uint4(0u, 0u, 0u, 0u);
        for (int i = tid; i < SLOT / 16; i += BT) *reinterpret_cast<uint4*>(smem + (RING - 1) * SLOT + 16 * i) = make_uint4(0u, 0u, 0u, 0u);
        landed();
        start(s, dp, 0);
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            const unsigned x = Ops<D>::k_step(lds + ops.row, kk);
            mfma_vec<T>(s, lds16(x), kf[kk]);
            mfma_vec<T>(dp, lds16(x + STAGE), vf[kk]);
        }
        mfma_settle();
        int n = 0;
        for (bool more = true; more; n++) {
            const int b0 = 2 * (n & (RING - 1)), t0 = (tile[0].x >> 1) * QT, rr = tile[0].y;
            const bool all = tile[0].x & 1;
            step(s, dp, sN, dN, (b0 - 1) & (2 * RING - 1), b0, b0 + 1, t0, rr, all);
            more = tile[1].x >= 0;
            if (more) {
                landed();                             // tile n + 1 is there, tile n - 1 is read
                tile[FLY + 1] = tile[FLY].x < 0 ? make_int2(-1, 0) : next();
                if (tile[FLY + 1].x >= 0) {
                    load(tile[FLY + 1], (n + FLY + 1) & (RING - 1));
                    fly++;
                }
#pragma unroll
                for (int i = 0; i <= FLY; i++) tile[i] = tile[i + 1];
            }
            step(sN, dN, s, dp, b0, b0 + 1, more ? (b0 + 2) & (2 * RING - 1) : b0, t0 + 32, rr, all);
        }
        // the sums of the last block
        const int bl = 2 * ((n - 1) & (RING - 1)) + 1;
        const unsigned cp = at(bl) + ops.col, cp8 = at(bl) + ops.col8;
#pragma unroll
        for (int i = 0; i < KK; i++) {
            const unsigned xc = Ops<D>::block(cp, i / 2), x8 = Ops<D>::block(cp8, i / 2);
            mfma_acc<T>(dv[i / 2], Ops<D>::at_col(xc, x8, 16 * (i & 1) * Tile<D>::ROWB + STAGE), pp[i & 1]);
            mfma_acc<T>(dk[i / 2], Ops<D>::at_col(xc, x8, 16 * (i & 1) * Tile<D>::ROWB), ds[i & 1]);
        }
        mfma_settle();
    }
    const float f = a.scale;
    if (a.nsplit > 1) {
        float* o = a.part + ((int64_t)(part * a.tiles + jt) * kvh + bh) * 2 * BQ * D + (32 * w + (lane & 31)) * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                *reinterpret_cast<float4*>(o + 32 * dt + 8 * g) = make_float4(dk[dt][4 * g] * f, dk[dt][4 * g + 1] * f, dk[dt][4 * g + 2] * f, dk[dt][4 * g + 3] * f);
                *reinterpret_cast<float4*>(o + BQ * D + 32 * dt + 8 * g) = make_float4(dv[dt][4 * g], dv[dt][4 * g + 1], dv[dt][4 * g + 2], dv[dt][4 * g + 3]);
            }
    } else if (j < a.Tk) {
        const int64_t o = (((int64_t)b * a.Tk + j) * a.Hk + hk) * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                *reinterpret_cast<uint2*>((T*)a.dk + o + 32 * dt + 8 * g) =
                    make_uint2(pack2<T>(dk[dt][4 * g] * f, dk[dt][4 * g + 1] * f), pack2<T>(dk[dt][4 * g + 2] * f, dk[dt][4 * g + 3] * f));
                *reinterpret_cast<uint2*>((T*)a.dv + o + 32 * dt + 8 * g) =
                    make_uint2(pack2<T>(dv[dt][4 * g], dv[dt][4 * g + 1]), pack2<T>(dv[dt][4 * g + 2], dv[dt][4 * g + 3]));
            }
    }
}

// dK and dV of 32 keys from the parts' sums, added in order; 32 rows x D / 4 lanes of 4 values
template <typename T, int D>
__global__ __launch_bounds__(256) void attn_add(AttnArgs a) {
    const int kvh = a.B * a.Hk, bh = blockIdx.x % kvh, q4 = blockIdx.x / kvh, jt = q4 / (BQ / 32);
    const int b = bh / a.Hk, hk = bh - b * a.Hk, off = a.Tk - a.Tq;
    const int j0 = jt * BQ, j1 = min(j0 + BQ, a.Tk) - 1;
    const Mask mk{a.causal, a.W, a.prefix ? a.prefix[b] : 0, a.Tk};
    int x0, x1;
    tile_rows(a, mk, j0, j1, off, x0, x1);
    const int nx = (a.Tq + QT - 1) / QT;
    for (int e = threadIdx.x; e < 32 * (D / 4) * 2; e += 256) {
        const int which = e / (32 * (D / 4)), i = e % (32 * (D / 4)), row = (q4 % (BQ / 32)) * 32 + i / (D / 4), c = 4 * (i % (D / 4));
        if (j0 + row >= a.Tk) continue;
        float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < a.nsplit; p++) {
            if (!meets(x0, x1, nx, p * a.units, min((p + 1) * a.units, a.R * nx))) continue;
            const float4 x = *reinterpret_cast<const float4*>(a.part + ((int64_t)(p * a.tiles + jt) * kvh + bh) * 2 * BQ * D + which * BQ * D + row * D + c);
            s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        }
        put4<T>(which ? a.dv : a.dk, nullptr, (((int64_t)b * a.Tk + j0 + row) * a.Hk + hk) * D + c, s.x, s.y, s.z, s.w);
    }
}

template <typename T, int D, bool CAP, bool BIAS>
void launch_one(AttnArgs a, bool keys, hipStream_t st) {
    if (keys) {
        a.tiles = (a.Tk + BQ - 1) / BQ;
        slothost::launch(attn_dkv<T, D, CAP, BIAS>, dim3((unsigned)((int64_t)a.tiles * a.nsplit * a.B * a.Hk)), dim3(BT), 0, st, a);
    } else {
        a.tiles = (a.Tq + BQ - 1) / BQ;
        slothost::launch(attn_dq<T, D, CAP, BIAS>, dim3((unsigned)((int64_t)a.tiles * a.B * a.Hq)), dim3(BT), 0, st, a);
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

// Parts of the queries per key tile: where the key tiles alone do not give the card's 512 workgroup slots a round and a half, each
// workgroup takes about 1 / 1024 of all (key tile, query tile) pairs, 8 at least (a part costs the write and the read of its sums).
void parts(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int causal, int64_t W, bool prefix, int& nsplit, int& units) {
    const int64_t R = Hq / Hk, nx = (Tq + QT - 1) / QT, tiles = (Tk + BQ - 1) / BQ * B * Hk;
    nsplit = 1;
    units = (int)(R * nx);
    if (tiles >= 768) return;
    int64_t rows = causal ? Tq - Tq / 2 : Tq;                         // of a head that see a key tile, about
    if (!prefix && W < Tk) rows = std::min(rows, (causal ? W : 2 * W) + BQ);
    const int64_t c = std::max<int64_t>(8, tiles * R * ((rows + QT - 1) / QT) / 1024);
    nsplit = (int)((R * nx + c - 1) / c);
    units = (int)c;
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
    if (!al16(out) || !al16(res) || !al16(dout) || !al16(dq) || !al16(dk) || !al16(dv) || !al16(docs) || (do_sb | do_sh | do_st) % 8)
        return fail(SLOTSCAN_ERR_ALIGN, "slotattn_bwd: rows of out, res, dout, dq, dk and dv, and docs, must be 16-byte aligned");
    if (do_st < 0 || do_st >= SLOTATTN_MAX_ST) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: token strides must be in [0, 2^25)");
    if ((Tq + BQ - 1) / BQ * B * Hq > 0x7fffffffLL || (Tk + BQ - 1) / BQ * B * Hk > 0x7fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: shape too large");
    AttnArgs a = slotattn_host::args(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st, B, Tq, Tk, Hq, Hk, scale, causal, window, cap,
                                     slopes, docs, prefix);
    parts(B, Tq, Tk, Hq, Hk, causal, window, prefix != nullptr, a.nsplit, a.units);
    if (a.nsplit > 1 && !workspace) return fail(SLOTSCAN_ERR_NULL, "slotattn_bwd: workspace is NULL");
    if ((Tk + BQ - 1) / BQ * B * Hk * std::max(a.nsplit, BQ / 32) > 0x7fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: shape too large");
    a.part = (float*)workspace;
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
