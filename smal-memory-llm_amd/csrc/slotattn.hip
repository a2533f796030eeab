// Exact attention of any range for MI355X (gfx950), forward: scores optionally capped by a tanh and biased by the
// distance, visible in a band, within documents and in a prefix (semantics: slotattn.h).
//
//   attn_fwd    many query rows: 128 queries of one head per workgroup, 32 per wave; one pass over the visible 64-key
//               tiles with the running maximum and sum of the softmax.
//   attn_split  few query rows against many keys (a generated token, a short chunk): the rows of a key/value head's query
//               heads together, the keys split over waves and workgroups; attn_join combines the parts.
#include "slot_attn_rows.h"
#include "slotscan.h"
#include "slotattn.h"
#include "slot_attn_host.h"

using namespace slotattn;
using slothost::fail;
using slothost::hip_fail;
using slothost::al16;

#define FW 4                                         // waves per workgroup
#define FT (64 * FW)
#define FQ (32 * FW)                                 // query rows per workgroup
#define SW 2                                         // waves per workgroup where the keys are split

namespace {

// ------------------------------------------------------------------------------------------- documents
// One wave per 64 ids: the padded copy (-1 past the end and for every padding id) and the range of the tile's ids.
__global__ __launch_bounds__(64) void attn_docs(const int32_t* ids, int T, int ntd, int32_t* out, int2* range) {
    const int b = blockIdx.y, lane = threadIdx.x, i = blockIdx.x * KT + lane;
    int x = i < T ? ids[(int64_t)b * T + i] : -1;
    x = x < 0 ? -1 : x;
    out[((int64_t)b * ntd) * KT + i] = x;
    int lo = x < 0 ? 0x7fffffff : x, hi = x;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        lo = min(lo, __shfl_xor(lo, m));
        hi = max(hi, __shfl_xor(hi, m));
    }
    const bool pad = __ballot(x < 0) != 0;
    if (lane == 0) range[(int64_t)b * ntd + blockIdx.x] = make_int2(pad ? (int)((unsigned)lo | 0x80000000u) : lo, hi < 0 ? -2 : hi);
}

// ------------------------------------------------------------------------------------------- many rows
// Per 64 keys a wave has 2 D / 16 + D / 8 matrix instructions of 32 cycles (S = K Q^T, O += V^T P^T; 1,024 cycles at D = 128) and
// about 350 vector ones for the softmax of 32 x 64 scores; both share a SIMD's issue, so two waves a SIMD (64 KB of LDS a
// workgroup) fill one's gaps with the other's work.  Measured (kernel trace): 8,192 causal tokens, 12 query heads of 128 on 4, capped:
// 284 us (2.06e11 operations in products: 726 TFLOP/s; they alone would take 149 us at the rate of a large library product);
// 4 x 2,000 tokens with prefixes, capped: 104 us.
// GR groups of 4 waves share a workgroup's rows, each taking every GR-th of their key tiles; their sums meet in LDS.  Two
// groups halve the longest rows' steps where every tile has a CU of its own (up to 256 tiles); with more tiles their
// lockstep costs more than the balance gives (8,192 tokens: 340 against 295 us).
template <typename T, int D, bool CAP, bool BIAS, int GR>
__global__ __launch_bounds__(FT * GR, 2) void attn_fwd(AttnArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = KT * 2 * D;
    typedef TileLoad<D, KT, FW> Load;
    __shared__ __align__(1024) unsigned char smem[GR][2][2][STAGE];  // [group][buffer][keys, values]
    const int tid = threadIdx.x & (FT - 1), lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), grp = GR == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / FT);
    // the longest rows (the last tiles under causality) first
    const int heads = a.B * a.Hq;
    const int qt = uni((int)(a.tiles - 1 - blockIdx.x / heads)), bh = uni((int)(blockIdx.x % heads));
    const int b = uni(bh / a.Hq), hq = bh - b * a.Hq, hk = uni(hq / a.R);
    const int len = length_of(a, b), t0 = qt * FQ, off = len - a.Tq;
    const int t = t0 + 32 * w + (lane & 31), tc = min(t, a.Tq - 1), p = tc + off;
    Mask mk{a.causal, a.W, prefix_of(a, b), min(len, a.Tk)};
    // this wave's queries, in operand order
    uint4 qf[KK];
    {
        const T* q = (const T*)a.q + b * a.q_sb + hq * a.q_sh + tc * a.q_st + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) qf[kk] = ld16(q + 16 * kk);
        if (a.f < 0.f)                                // a negative scale: of the queries' sign, so that larger products are larger scores
#pragma unroll
            for (int kk = 0; kk < KK; kk++) { qf[kk].x ^= 0x80008000u; qf[kk].y ^= 0x80008000u; qf[kk].z ^= 0x80008000u; qf[kk].w ^= 0x80008000u; }
    }
    const float f2 = fabsf(a.f);
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
    const bool docs = a.ids != nullptr;
    const int64_t idb = (int64_t)b * a.ntd * KT;
    Span sw{t0 + off, min(t0 + FQ, a.Tq) - 1 + off, 0, 0, true}, sv{t0 + 32 * w + off, min(t0 + 32 * w + 32, a.Tq) - 1 + off, 0, 0, true};
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
    const float F = BIAS ? 1.f : f2;                  // from a row's values to base 2
    const unsigned lds = lds_addr(smem[grp]);
    const Load lk(a.k_st, w, lane), lv(a.v_st, w, lane);
    auto load = [&](int jt, int buf) {
        lk.issue(kb, jt * KT, mk.klen - 1, lds + (2 * buf) * STAGE);
        lv.issue(vb, jt * KT, mk.klen - 1, lds + (2 * buf + 1) * STAGE);
    };
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = zero16();
    float m = -INFINITY, mu = 0.f, l = 0.f;           // a row's reference, the same in base 2, its sum
    const float lazy = LAZY / F, head = HEAD<T> / F;
    bool far = false;
    // this group's next tile, and whether any group has one
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
    // one barrier a tile: behind it the tile is there for every wave and the other buffer is read, so the next one's loads
    // run during this one's products
    for (int buf = 0; go; buf ^= 1, jt = jn, some = some_n, all = all_n, go = more) {
        more = next(jn, some_n, all_n);
        wait_vm<0>();
        tile_barrier();
        if (jn >= 0) load(jn, buf ^ 1);
        if (some) {
            const unsigned bo = lds + (2 * buf) * STAGE, rk = bo + ops.row, c = bo + ops.col, c8 = bo + ops.col8;
            const int j0 = jt * KT;
            // operands are read three steps (six products) ahead: an LDS read takes as long as four or five products
            f32x16 s[2] = {zero16(), zero16()};
            uint4 kr[4][2];
            auto rows = [&](int kk) {
                const unsigned x = Ops<D>::k_step(rk, kk);
                kr[kk & 3][0] = lds16(x);
                kr[kk & 3][1] = lds16(x + 32 * Tile<D>::ROWB);
            };
            rows(0);
            rows(1);
            rows(2);
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                if (kk + 3 < KK) rows(kk + 3);
                s[0] = mfma32<T>(kr[kk & 3][0], qf[kk], s[0]);
                s[1] = mfma32<T>(kr[kk & 3][1], qf[kk], s[1]);
                __builtin_amdgcn_sched_barrier(0);
            }
            uint4 vr[5];                              // operand i: column block i % DT of 16 keys i / DT
            auto cols = [&](int i) {
                vr[i % 5] = Ops<D>::at_col(Ops<D>::block(c, i % DT), Ops<D>::block(c8, i % DT), STAGE + 16 * (i / DT) * Tile<D>::ROWB);
            };
            cols(0);
            cols(1);
            cols(2);
            cols(3);
#pragma unroll
            for (int u = 0; u < 2; u++) {
                scores<CAP>(s[u], a);
                if constexpr (BIAS) bias(s[u], f2, slope, p, j0 + 32 * u, h);
            }
            if (!all) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const uint32_t ok = seen16(see, j0 + 32 * u, h, j0 < mk.prefix, docs ? a.ids + idb + j0 + 32 * u : nullptr, dq);
#pragma unroll
                    for (int r = 0; r < 16; r++) s[u][r] = bit(ok, r) ? s[u][r] : -INFINITY;
                }
            }
            float mx = s[0][0];
#pragma unroll
            for (int u = 0; u < 2; u++)
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
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[u][r] = (s[u][r] - (m == -INFINITY ? 0.f : m)) * F;
            } else {
#pragma unroll
                for (int u = 0; u < 2; u++)
#pragma unroll
                    for (int r = 0; r < 16; r++) s[u][r] = fmaf(s[u][r], F, -mu);
            }
            uint4 pf[2][2];
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int r = 0; r < 16; r++) {
                    s[u][r] = exp2_(s[u][r]);
                    l += s[u][r];
                }
                pf[u][0] = pack8<T>(s[u], 0);
                pf[u][1] = pack8<T>(s[u], 1);
            }
#pragma unroll
            for (int i = 0; i < 4 * DT; i++) {
                o[i % DT] = mfma32<T>(vr[i % 5], pf[i / DT >> 1][i / DT & 1], o[i % DT]);
                if (i + 4 < 4 * DT) cols(i + 4);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
    }
    l = half_sum(l);
    m = m == -INFINITY ? m : mu;                      // in base 2 from here on
    if constexpr (GR == 2) {
        float4* so = reinterpret_cast<float4*>(smem);                 // [4 DT][thread], then the rows' maxima and sums
        float* sm = reinterpret_cast<float*>(so + 4 * DT * FT);
        static_assert((16 * DT + 2) * FT * 4 <= (int)sizeof(smem), "a group's sums fit");
        __syncthreads();
        if (grp) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++) so[(4 * dt + g) * FT + tid] = make_float4(o[dt][4 * g], o[dt][4 * g + 1], o[dt][4 * g + 2], o[dt][4 * g + 3]);
            sm[tid] = m;
            sm[FT + tid] = l;
        }
        __syncthreads();
        if (grp) return;
        const float m1 = sm[tid], l1 = sm[FT + tid], M = fmaxf(m, m1), Mu = M == -INFINITY ? 0.f : M;
        const float f0 = exp2_(m - Mu), f1 = exp2_(m1 - Mu);
        m = M;
        l = l * f0 + l1 * f1;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++) {
                const float4 x = so[(4 * dt + g) * FT + tid];
                o[dt][4 * g] = fmaf(x.x, f1, o[dt][4 * g] * f0);
                o[dt][4 * g + 1] = fmaf(x.y, f1, o[dt][4 * g + 1] * f0);
                o[dt][4 * g + 2] = fmaf(x.z, f1, o[dt][4 * g + 2] * f0);
                o[dt][4 * g + 3] = fmaf(x.w, f1, o[dt][4 * g + 3] * f0);
            }
    }
    float bad = l * 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) bad = nonfinite(o[dt], bad);
    uint32_t rows = row_bits(bad != 0.f && l == l && t < a.Tq);       // (a NaN in its sum makes all of a row NaN)
    if (rows)
        rows &= ~row_bits(keeps<T, D>(kb, a.k_st, vb, a.v_st, vb, a.v_st, 0, mk.klen, mk.klen % KT ? mk.klen - 1 : -1, lane,
                                      [&](int j) { return sees1(see, j, docs ? a.ids + idb : nullptr, dq); }, [&](int j) { return walk.computes(j / KT); }));
    for (uint32_t left = rows; left; left &= left - 1) {
        const int i = __builtin_ctz(left), ti = t0 + 32 * w + i;
        float m1, l1, o1[D / 64], rest[D / 64];
        exact_row<T, D, CAP, BIAS>(a, (const T*)a.q + b * a.q_sb + hq * a.q_sh + ti * a.q_st, kb, vb, lane_of(see, i), docs ? a.ids + idb : nullptr,
                                   lane_of(dq, i), slope, ti + off, 0, mk.klen, lane, m1, l1, o1);
        const float inv1 = l1 > 0.f || l1 != l1 ? 1.f / l1 : 0.f;
        const int64_t at = (((int64_t)b * a.Tq + ti) * a.Hq + hq) * D;
        for (int e = 0; e < D / 64; e++) {
            o1[e] *= inv1;
            rest[e] = o1[e] - unpack<T>(pack2<T>(o1[e], 0.f), 0);
        }
        put_row<T, D>((T*)a.out + at, lane, o1);
        if (a.res) put_row<T, D>((T*)a.res + at, lane, rest);
        if (a.lse && lane == 0) a.lse[(int64_t)bh * a.Tq + ti] = l1 > 0.f || l1 != l1 ? m1 + __builtin_amdgcn_logf(l1) : INFINITY;
    }
    const float inv = l > 0.f || l != l ? 1.f / l : 0.f;
    if (t < a.Tq && !bit(rows, lane & 31)) {
        const int64_t at = (((int64_t)b * a.Tq + t) * a.Hq + hq) * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                put4<T>(a.out, a.res, at + 32 * dt + 8 * g, o[dt][4 * g] * inv, o[dt][4 * g + 1] * inv, o[dt][4 * g + 2] * inv, o[dt][4 * g + 3] * inv);
        if (a.lse && h == 0) a.lse[(int64_t)bh * a.Tq + t] = l > 0.f || l != l ? m + __builtin_amdgcn_logf(l) : INFINITY;
    }
}

// ------------------------------------------------------------------------------------------- few rows
// Rows of a key/value head packed as (token, query head of the group); a workgroup takes `chunk` keys of 32 rows, its waves every
// SW-th 32-key tile of them, each through a ring of its own of two tiles (no barrier in the loop); the waves' results meet
// in LDS, the workgroups' in attn_join.  Bound by the bytes of the keys and values: two workgroups a CU keep about 100 KB
// on their way.  Measured (kernel trace): 32 sequences of up to 8,192 tokens, 12 query heads of 128 on 4: 66 + 5
// us (join), 4.8 TB/s in the kernel; one of 131,072: 44 + 9 us, 6.1 TB/s.  (Four waves a workgroup, one workgroup a CU, tiles fetched one
// ahead: 92 and 57 us.)
template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(64 * SW) void attn_split(AttnArgs a) {
    constexpr int KK = D / 16, DT = D / 32, ST = 32 * 2 * D;
    typedef TileLoad<D, 32, 1> Load;
    __shared__ __align__(1024) unsigned char smem[SW][2][2][ST];     // [wave][buffer][keys, values]
    __shared__ float s_m[SW][32], s_l[SW][32];                       // the waves' maxima and sums of every row
    __shared__ float s_M[32], s_L[32];                               // the workgroup's
    __shared__ uint32_t s_bad[SW];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int sp = blockIdx.x % a.nsplit, rt = blockIdx.x / a.nsplit;
    const int hk = blockIdx.y, b = blockIdx.z;
    const int rows = a.Tq * a.R, r0 = rt * 32, row = min(r0 + (lane & 31), rows - 1);
    const int t = row / a.R, hq = hk * a.R + row - t * a.R;
    const int len = length_of(a, b), klen = min(len, a.Tk), off = len - a.Tq, p = t + off;
    Mask mk{a.causal, a.W, prefix_of(a, b), klen};
    const Span s{r0 / a.R + off, (min(r0 + 32, rows) - 1) / a.R + off, 0, 0, true};
    // this workgroup's keys
    const int end = a.causal ? min(klen, max(s.p1 + 1, mk.prefix)) : klen;
    const int lo = (mk.prefix > 0 ? 0 : max(0, max(s.p0, 0) - a.W + 1) & ~31) + sp * a.chunk, hi = min(end, lo + a.chunk);
    const T* kb = (const T*)a.k + b * a.k_sb + hk * a.k_sh;
    const T* vb = (const T*)a.v + b * a.v_sb + hk * a.v_sh;
    const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
    const float f2 = fabsf(a.f), F = BIAS ? 1.f : f2;
    const unsigned lds = lds_addr(smem[w]);
    const Load lk(a.k_st, 0, lane), lv(a.v_st, 0, lane);
    auto load = [&](int j0, int buf) {
        lk.issue(kb, j0, klen - 1, lds + (2 * buf) * ST);
        lv.issue(vb, j0, klen - 1, lds + (2 * buf + 1) * ST);
    };
    auto seen = [&](int j0) {                         // the next of this wave's tiles that any row sees
        while (j0 < hi && !mk.some(s, j0, j0 + 31)) j0 += 32 * SW;
        return j0;
    };
    const Ops<D> ops(lane);
    const Sees see = Sees::query(mk, p);
    int j0 = seen(lo + 32 * w);
    if (j0 < hi) load(j0, 0);
    uint4 qf[KK];
    {
        const T* q = (const T*)a.q + b * a.q_sb + hq * a.q_sh + t * a.q_st + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) qf[kk] = ld16(q + 16 * kk);
        if (a.f < 0.f)                                // a negative scale: of the queries' sign, so that larger products are larger scores
#pragma unroll
            for (int kk = 0; kk < KK; kk++) { qf[kk].x ^= 0x80008000u; qf[kk].y ^= 0x80008000u; qf[kk].z ^= 0x80008000u; qf[kk].w ^= 0x80008000u; }
    }
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) o[dt] = zero16();
    float m = -INFINITY, mu = 0.f, l = 0.f;           // a row's reference, the same in base 2, its sum
    const float lazy = LAZY / F, head = HEAD<T> / F;
    bool far = false;
    // Keys and values are fetched two tiles ahead, each into the place that it has just been read from: a wave has one and a
    // half to two tiles (24 to 32 KB at D = 128) on their way while it computes.
    int j1 = j0 < hi ? seen(j0 + 32 * SW) : hi;
    if (j1 < hi) load(j1, 1);
    for (int buf = 0; j0 < hi; buf ^= 1) {
        const int j2 = j1 < hi ? seen(j1 + 32 * SW) : hi;
        if (j1 < hi) wait_vm<3 * Load::N>();          // behind this tile's keys: its values, the next keys and values
        else wait_vm<Load::N>();
        asm volatile("" ::: "memory");
        const unsigned bo = lds + (2 * buf) * ST, rk = bo + ops.row, c = bo + ops.col, c8 = bo + ops.col8;
        f32x16 x = zero16();
#pragma unroll
        for (int kk = 0; kk < KK; kk++) x = mfma32<T>(lds16(Ops<D>::k_step(rk, kk)), qf[kk], x);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");            // the keys are read before their place is filled again
        if (j2 < hi) lk.issue(kb, j2, klen - 1, lds + (2 * buf) * ST);
        scores<CAP>(x, a);
        if constexpr (BIAS) bias(x, f2, slope, p, j0, h);
        if (j0 + 32 > hi || !mk.all(s, j0, j0 + 31)) {
            const uint32_t ok = seen16(see, j0, h, j0 < mk.prefix, nullptr, 0);
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = j0 + key_of(r, h) < hi && bit(ok, r) ? x[r] : -INFINITY;
        }
        float mx = x[0];
#pragma unroll
        for (int r = 1; r < 16; r++) mx = fmaxf(mx, x[r]);
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
            for (int r = 0; r < 16; r++) x[r] = (x[r] - (m == -INFINITY ? 0.f : m)) * F;
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) x[r] = fmaf(x[r], F, -mu);
        }
#pragma unroll
        for (int r = 0; r < 16; r++) {
            x[r] = exp2_(x[r]);
            l += x[r];
        }
        const uint4 pf[2] = {pack8<T>(x, 0), pack8<T>(x, 1)};
        if (j2 < hi) wait_vm<3 * Load::N>();          // behind the values: the next tile, the keys after it
        else if (j1 < hi) wait_vm<2 * Load::N>();
        else wait_vm<0>();
        asm volatile("" ::: "memory");
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int mm = 0; mm < 2; mm++)
                o[dt] = mfma32<T>(Ops<D>::at_col(Ops<D>::block(c, dt), Ops<D>::block(c8, dt), ST + 16 * mm * Tile<D>::ROWB), pf[mm], o[dt]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");            // the values, too
        if (j2 < hi) lv.issue(vb, j2, klen - 1, lds + (2 * buf + 1) * ST);
        j0 = j1;
        j1 = j2;
    }
    l = half_sum(l);
    m = m == -INFINITY ? m : mu;                      // in base 2 from here on
    // the waves' parts: (m, l) of every row to all, then the weighted sums through LDS (its tiles are read)
    if (h == 0) { s_m[w][lane] = m; s_l[w][lane] = l; }
    __syncthreads();
    float M = -INFINITY, Ls = 0.f;
#pragma unroll
    for (int i = 0; i < SW; i++) M = fmaxf(M, s_m[i][lane & 31]);
    const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < SW; i++) Ls += s_l[i][lane & 31] * exp2_(s_m[i][lane & 31] - Mu);
    const float f = exp2_(m - Mu);
    float* so = reinterpret_cast<float*>(smem);       // [wave][row][D + 4]
    constexpr int SO = D + 4;
    static_assert(SW * 32 * SO * 4 <= (int)sizeof(smem), "the waves' sums fit");
#pragma unroll
    for (int dt = 0; dt < DT; dt++)
#pragma unroll
        for (int g = 0; g < 4; g++)
            *reinterpret_cast<float4*>(so + (w * 32 + (lane & 31)) * SO + 32 * dt + 8 * g + 4 * h) =
                make_float4(o[dt][4 * g] * f, o[dt][4 * g + 1] * f, o[dt][4 * g + 2] * f, o[dt][4 * g + 3] * f);
    if (w == 0 && h == 0) { s_M[lane] = M; s_L[lane] = Ls; }          // not over s_m and s_l, which the other waves may still read
    float bad = l * 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) bad = nonfinite(o[dt], bad);
    const uint32_t odd = row_bits(bad != 0.f && r0 + (lane & 31) < rows);
    if (lane == 0) s_bad[w] = odd;
    __syncthreads();
    uint32_t left = 0;
#pragma unroll
    for (int i = 0; i < SW; i++) left |= s_bad[i];
    if (left) {                                       // the same in every wave
        const int last = (klen - lo) % 32 ? klen - 1 : -1;            // keys past hi are in the last tile, too
        const bool kept = keeps<T, D>(kb, a.k_st, vb, a.v_st, vb, a.v_st, lo, min(klen, lo + (hi - lo + 31) / 32 * 32), last, lane,
                                      [&](int j) { return j < hi && sees1(see, j, nullptr, 0); },
                                      [&](int j) { const int x = lo + (j - lo) / 32 * 32; return mk.some(s, x, x + 31); });      // (by all lanes)
        left &= ~row_bits(kept || Ls != Ls);
        for (; left; left &= left - 1) {
            const int i = __builtin_ctz(left);
            if (i % SW != w) continue;
            float m1, l1, o1[D / 64];
            exact_row<T, D, CAP, BIAS>(a, (const T*)a.q + b * a.q_sb + lane_of(hq, i) * a.q_sh + lane_of(t, i) * a.q_st, kb, vb, lane_of(see, i),
                                       nullptr, 0, lane_of(slope, i), lane_of(p, i), lo, hi, lane, m1, l1, o1);
            for (int ww = 0; ww < SW; ww++)
                for (int e = 0; e < D / 64; e++) so[(ww * 32 + i) * SO + lane * (D / 64) + e] = ww ? 0.f : o1[e];
            if (lane == 0) { s_M[i] = m1; s_L[i] = l1; }
        }
        __syncthreads();
    }
    // 32 rows x D values: 8 lanes a row
    for (int rr = tid >> 3; rr < 32; rr += 8 * SW) {
        const int c8 = tid & 7, g = r0 + rr;
        if (g >= rows) break;
        const float lr = s_L[rr], mr = s_M[rr];
        const bool got = lr > 0.f || lr != lr;
        const float inv = got ? 1.f / lr : 0.f;
        const int gt = g / a.R, gh = hk * a.R + g - gt * a.R;
        const int64_t orow = ((int64_t)b * a.Tq + gt) * a.Hq + gh;
#pragma unroll
        for (int i = 0; i < D / 32; i++) {
            const int d = 4 * c8 + 32 * i;
            float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int ww = 0; ww < SW; ww++) {
                const float4 y = *reinterpret_cast<const float4*>(so + (ww * 32 + rr) * SO + d);
                v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
            }
            if (a.nsplit == 1) {
                put4<T>(a.out, a.res, orow * D + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
            } else if (got) {
                *reinterpret_cast<float4*>(a.po + (orow * a.nsplit + sp) * D + d) = v;
            }
        }
        if (c8 == 0) {
            if (a.nsplit == 1) {
                if (a.lse) a.lse[((int64_t)b * a.Hq + gh) * a.Tq + gt] = got ? mr + __builtin_amdgcn_logf(lr) : INFINITY;
            } else {
                *reinterpret_cast<float2*>(a.pm + (orow * a.nsplit + sp) * 2) = make_float2(mr, lr);
            }
        }
    }
}

// One workgroup per row: out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s.  Groups of D / 4 lanes take every NG-th part,
// so that a row of hundreds of parts is as many short chains of loads; their sums meet in LDS in order.
template <typename T, int D>
__global__ __launch_bounds__(FT) void attn_join(AttnArgs a) {
    constexpr int LN = D / 4, NG = FT / LN;
    __shared__ __align__(16) float s_o[NG][D];
    __shared__ float s_l[NG], s_m[FW];
    const int tid = threadIdx.x, c = tid % LN, g = tid / LN;
    const int64_t row = blockIdx.x;
    const float2* pm = reinterpret_cast<const float2*>(a.pm) + row * a.nsplit;
    float M = -INFINITY;
    for (int s = tid; s < a.nsplit; s += FT) M = fmaxf(M, pm[s].x);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) M = fmaxf(M, __shfl_xor(M, i));
    if ((tid & 63) == 0) s_m[tid >> 6] = M;
    __syncthreads();
    M = s_m[0];
#pragma unroll
    for (int i = 1; i < FW; i++) M = fmaxf(M, s_m[i]);
    const float Mu = M == -INFINITY ? 0.f : M;
    float L = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = g; s < a.nsplit; s += NG) {
        const float2 x = pm[s];
        const bool in = x.y != 0.f;                   // otherwise nothing is visible in this part, and no sum was written
        const float f = in ? exp2_(x.x - Mu) : 0.f;
        const float4 o = in ? *reinterpret_cast<const float4*>(a.po + (row * a.nsplit + s) * D + 4 * c) : make_float4(0.f, 0.f, 0.f, 0.f);
        L = fmaf(x.y, f, L);
        acc.x = fmaf(o.x, f, acc.x);
        acc.y = fmaf(o.y, f, acc.y);
        acc.z = fmaf(o.z, f, acc.z);
        acc.w = fmaf(o.w, f, acc.w);
    }
    *reinterpret_cast<float4*>(&s_o[g][4 * c]) = acc;
    if (c == 0) s_l[g] = L;
    __syncthreads();
    if (tid >= LN) return;
    L = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < NG; i++) {
        const float4 o = *reinterpret_cast<const float4*>(&s_o[i][4 * c]);
        L += s_l[i];
        acc.x += o.x;
        acc.y += o.y;
        acc.z += o.z;
        acc.w += o.w;
    }
    const bool got = L > 0.f || L != L;
    const float inv = got ? 1.f / L : 0.f;
    put4<T>(a.out, a.res, row * D + 4 * c, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    if (a.lse && c == 0) {
        const int64_t tok = row / a.Hq;
        const int hq = (int)(row - tok * a.Hq);
        const int64_t b = tok / a.Tq;
        a.lse[(b * a.Hq + hq) * a.Tq + tok - b * a.Tq] = got ? M + __builtin_amdgcn_logf(L) : INFINITY;
    }
}

template <typename T, int D, bool CAP, bool BIAS>
void launch_one(const AttnArgs& a, bool split, hipStream_t st) {
    if (split) slothost::launch(attn_split<T, D, CAP, BIAS>, dim3((unsigned)(a.nsplit * a.tiles), (unsigned)a.Hk, (unsigned)a.B), dim3(64 * SW), 0, st, a);
    else if (a.groups == 2) slothost::launch(attn_fwd<T, D, CAP, BIAS, 2>, dim3((unsigned)((int64_t)a.tiles * a.B * a.Hq)), dim3(2 * FT), 0, st, a);
    else slothost::launch(attn_fwd<T, D, CAP, BIAS, 1>, dim3((unsigned)((int64_t)a.tiles * a.B * a.Hq)), dim3(FT), 0, st, a);
}
template <typename T, int D>
void launch_fwd(const AttnArgs& a, bool cap, bool split, hipStream_t st) {
    if (cap) a.slopes ? launch_one<T, D, true, true>(a, split, st) : launch_one<T, D, true, false>(a, split, st);
    else a.slopes ? launch_one<T, D, false, true>(a, split, st) : launch_one<T, D, false, false>(a, split, st);
}
template <typename T, int D>
void launch_join(const AttnArgs& a, hipStream_t st) {
    slothost::launch(attn_join<T, D>, dim3((unsigned)((int64_t)a.B * a.Tq * a.Hq)), dim3(FT), 0, st, a);
}

// How the forward runs.  split: the packed rows and split keys, where a key/value head has at most 32 rows (a tile of 128 would be
// mostly empty), or where few rows in all meet many keys: unsplit, a call takes about 8 us and 15 ns a key while CUs idle (D = 128; 128
// to 512 rows of 12 heads alike), split about 14 us and 2.5 ns for 1,000 rows and a key.  Measured, split / unsplit: 768 rows (64 tokens of 12
// heads) x 1,024 / 3,500 keys 16 / 22 and 18 / 55 us, 1,536 rows x 1,024 / 2,048 keys 17 / 22 and 19 / 35, 6,144 rows x 2,048 / 3,500 keys 43 / 37 and
// 65 / 60; 256 rows x 512 keys 16 / 14.  groups: two groups of waves per tile while every tile has a CU of its own anyway.
struct Plan { bool split; int chunk, nsplit, rtiles, groups; };
Plan plan(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int causal, int64_t W, bool docs, bool prefix, bool ragged) {
    Plan p{false, 0, 1, 0, 1};
    const int64_t rows = Tq * (Hq / Hk), tiles = (Tq + FQ - 1) / FQ * Hq * B;
    // keys that one row tile can see
    int64_t keys = Tk;
    if (causal && !prefix && W < Tk) keys = W + Tq + 32 < Tk ? W + Tq + 32 : Tk;
    const int64_t all = rows * Hk * B;
    if (docs || !(rows <= 32 || (all <= 4096 && keys >= 1024 && 3 * keys >= 2 * all))) {
        if (tiles <= 256) p.groups = 2;
        return p;
    }
    p.split = true;
    p.rtiles = (int)((rows + 31) / 32);
    // Two workgroups a CU (their rings fill the LDS).  One round of them where the lengths are equal; where they may be ragged, pieces
    // small enough that the last round is short, not so small that a workgroup's start (about 5 us) counts: 32 sequences of
    // 1,024 to 8,192 keys, pieces of 512 / 768 / 1,024 / 2,048 keys: 81 / 62 / 77 / 70 us.
    const int64_t total = ragged && B > 1 ? 1408 : 512, want = (total + p.rtiles * Hk * B - 1) / (p.rtiles * Hk * B);
    int64_t chunk = (keys + want - 1) / want;
    chunk = (chunk + 63) / 64 * 64;
    if (chunk < 256) chunk = 256;
    p.chunk = (int)chunk;
    p.nsplit = (int)((keys + chunk - 1) / chunk);
    return p;
}
size_t split_bytes(const Plan& p, int64_t B, int64_t Tq, int64_t Hq, int64_t D) {
    return p.nsplit == 1 ? 0 : (size_t)(B * Tq * Hq * p.nsplit) * (D + 2) * sizeof(float);
}

}  // namespace

// ======================================================================================== C-ABI
extern "C" size_t slotattn_docs_bytes(int64_t B, int64_t T) {
    if (B < 1 || T < 1) return 0;
    const int64_t n = (T + KT - 1) / KT;
    return (size_t)(B * n) * (KT * 4 + 8);
}

extern "C" int slotattn_docs(const int32_t* ids, int64_t B, int64_t T, void* docs, void* stream) {
    if (B < 1 || T < 1 || B > 65535 || T > SLOTATTN_MAX_T) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_docs: B in [1, 65535], T in [1, 2^30)");
    if (!ids || !docs) return fail(SLOTSCAN_ERR_NULL, "slotattn_docs: a required pointer is NULL");
    if (!al16(docs)) return fail(SLOTSCAN_ERR_ALIGN, "slotattn_docs: docs must be 16-byte aligned");
    const int n = (int)((T + KT - 1) / KT);
    slothost::launch(attn_docs, dim3((unsigned)n, (unsigned)B), dim3(64), 0, (hipStream_t)stream, ids, (int)T, n, (int32_t*)docs,
                     (int2*)((int32_t*)docs + B * n * KT));
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "attn_docs launch");
}

extern "C" size_t slotattn_fwd_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, int causal, int64_t window,
                                         int has_docs, int has_prefix, int has_lens) {
    if (B < 1 || Tq < 1 || Tk < 1 || Hk < 1 || Hq < Hk || Hq % Hk) return 0;
    return split_bytes(plan(B, Tq, Tk, Hq, Hk, causal, window, has_docs, has_prefix, has_lens), B, Tq, Hq, D);
}

extern "C" int slotattn_fwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                            int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, int64_t B, int64_t Tq,
                            int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, float scale, int causal, int64_t window, float cap,
                            const float* slopes, const void* docs, const int32_t* prefix, const int32_t* lens, void* workspace,
                            void* out, void* res, float* lse, void* stream) {
    if (int r = slotattn_host::check(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st, dtype, B, Tq, Tk, Hq, Hk, D, scale, window, cap)) return r;
    if (lens && (docs || !causal)) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_fwd: lens goes with causality and without documents");
    if (!lens && Tq > Tk) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_fwd: more queries than keys");
    if (!out) return fail(SLOTSCAN_ERR_NULL, "slotattn_fwd: a required pointer is NULL");
    if (!al16(out) || !al16(res) || !al16(workspace) || !al16(docs)) return fail(SLOTSCAN_ERR_ALIGN, "slotattn_fwd: out, res, docs and workspace must be 16-byte aligned");
    Plan p = plan(B, Tq, Tk, Hq, Hk, causal, window, docs != nullptr, prefix != nullptr, lens != nullptr);
    if (split_bytes(p, B, Tq, Hq, D) && !workspace) return fail(SLOTSCAN_ERR_NULL, "slotattn_fwd: workspace is NULL");
    AttnArgs a = slotattn_host::args(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st, B, Tq, Tk, Hq, Hk, scale, causal, window, cap,
                                     slopes, docs, prefix);
    a.lens = lens;
    a.out = out;
    a.res = res;
    a.lse = lse;
    a.tiles = p.split ? p.rtiles : (int)((Tq + FQ - 1) / FQ);
    a.chunk = p.chunk;
    a.nsplit = p.nsplit;
    a.groups = p.groups;
    a.po = (float*)workspace;
    a.pm = a.po ? a.po + B * Tq * Hq * p.nsplit * D : nullptr;
    const bool split = p.split;
    if ((int64_t)a.tiles * (split ? a.nsplit : B * Hq) > 0x7fffffffLL || (split && (Hk > 65535 || B > 65535 || B * Tq * Hq > 0x7fffffffLL)))
        return fail(SLOTSCAN_ERR_SHAPE, "slotattn_fwd: shape too large");
    hipStream_t st = (hipStream_t)stream;
    const bool cp = cap > 0.f;
    hipError_t e;
    {
        slothost::Scope sc(SLOTSCAN_K_ATTN, st);
        if (dtype == SLOTSCAN_BF16) D == 128 ? launch_fwd<bf16_t, 128>(a, cp, split, st) : launch_fwd<bf16_t, 64>(a, cp, split, st);
        else D == 128 ? launch_fwd<f16_t, 128>(a, cp, split, st) : launch_fwd<f16_t, 64>(a, cp, split, st);
        e = hipGetLastError();
    }
    if (e != hipSuccess) return hip_fail(e, "attn_fwd launch");
    if (!split || a.nsplit == 1) return 0;
    {
        slothost::Scope sc(SLOTSCAN_K_ATTN_JOIN, st);
        if (dtype == SLOTSCAN_BF16) D == 128 ? launch_join<bf16_t, 128>(a, st) : launch_join<bf16_t, 64>(a, st);
        else D == 128 ? launch_join<f16_t, 128>(a, st) : launch_join<f16_t, 64>(a, st);
        e = hipGetLastError();
    }
    return e == hipSuccess ? 0 : hip_fail(e, "attn_join launch");
}
