// Exact attention of any range for MI355X (gfx950), backward (semantics: slotattn.h).  With P = softmax, dP = dO V^T,
// delta = rowsum(dO o O) and the cap's slope 1 - tanh^2:
//     dS = P (dP - delta) (1 - tanh^2),   dV = P^T dO,   dQ = scale dS K,   dK = scale dS^T Q
// P comes back from the rows' log-sum-exp.  Two kernels, each of which owns what it sums, so nothing is added atomically:
//   attn_dq    128 queries of one head per workgroup, walking the visible key tiles (as the forward does); it forms delta
//   attn_dkv   128 keys of one key/value head per workgroup, walking the query tiles of every head of the group that see them
// The price is that the scores and dP are formed twice: 7 products where one kernel with atomic dQ would need 5.
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

// P and dS of one 32 x 32 tile from its products s = <q, k> and dp = <dO, v>; lse and delta of register r's row through
// L(r), Dl(r).  dist: the lane's own position; d0: the position of register row 0.  ok(r): visible (only asked if !all).
template <bool CAP, bool BIAS, class LF, class DF, class OK>
__device__ __forceinline__ void probs(f32x16& s, f32x16& dp, const AttnArgs& a, float slope, int dist, int d0, int h, bool all, LF L, DF Dl, OK ok) {
    f32x16 x = s;
    scores<CAP, BIAS>(x, a, slope, dist, d0, h);
#pragma unroll
    for (int r = 0; r < 16; r++) {
        float g = 1.f;
        if constexpr (CAP) {                          // 1 - tanh^2 = 4 z (1 - z), z = 1 / (1 + e^2x)
            const float z = __builtin_amdgcn_rcpf(1.f + exp2_(s[r] * a.ct));
            g = 4.f * z * (1.f - z);
        }
        float p = exp2_(x[r] - L(r));
        float ds = p * (dp[r] - Dl(r)) * g;
        if (!all) {
            const bool o = ok(r);
            p = o ? p : 0.f;
            ds = o ? ds : 0.f;
        }
        s[r] = p;
        dp[r] = ds;
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
        const T* o = (const T*)a.out + (((int64_t)b * a.Tq + tc) * a.Hq + hq) * D + 8 * h;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            qf[kk] = ld16(q + 16 * kk);
            df[kk] = ld16(g + 16 * kk);
        }
#pragma unroll
        for (int kk = 0; kk < KK; kk++) dot8(df[kk], ld16(o + 16 * kk), delta, T{});
    }
    delta = half_sum(delta);
    const int64_t row = (int64_t)bh * a.Tq + tc;
    const float lse = a.lse[row];
    if (t < a.Tq && h == 0) a.delta[row] = delta;
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
    auto load = [&](int jt, int buf) {
        Load::issue(kb, a.k_st, jt * KT, mk.klen - 1, lds + (2 * buf) * STAGE, w, lane);
        Load::issue(vb, a.v_st, jt * KT, mk.klen - 1, lds + (2 * buf + 1) * STAGE, w, lane);
    };
    f32x16 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) acc[dt] = zero16();
    int jt, jn;
    bool some, all, some_n = false, all_n = false;
    walk.next(jt, some, all);
    if (jt >= 0) load(jt, 0);
    for (int buf = 0; jt >= 0; buf ^= 1, jt = jn, some = some_n, all = all_n) {
        walk.next(jn, some_n, all_n);
        if (jn >= 0) {
            load(jn, buf ^ 1);
            wait_vm<2 * Load::N>();
        } else {
            wait_vm<0>();
        }
        tile_barrier();
        if (some) {
            const unsigned char* sk = smem[buf][0];
            const unsigned char* sx = smem[buf][1];
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const int j0 = jt * KT + 32 * u;
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    s = mfma32<T>(Tile<D>::row_op(sk, 32 * u, kk, lane), qf[kk], s);
                    dp = mfma32<T>(Tile<D>::row_op(sx, 32 * u, kk, lane), df[kk], dp);
                }
                probs<CAP, BIAS>(s, dp, a, slope, p, j0, h, all, [&](int) { return lse; }, [&](int) { return delta; }, [&](int r) {
                    const int j = j0 + key_of(r, h);
                    return mk.sees(p, j) && (!docs || a.ids[idb + j] == dq);
                });
#pragma unroll
                for (int mm = 0; mm < 2; mm++) {
                    const uint4 ds = pack8<T>(dp, mm);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) acc[dt] = mfma32<T>(Tile<D>::col_op(sk, 32 * u, dt, mm, lane), ds, acc[dt]);
                }
            }
        }
        tile_barrier();
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
template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(BT, 1) void attn_dkv(AttnArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = KT * 2 * D;
    typedef TileLoad<D, KT, BW> Load;
    __shared__ __align__(1024) unsigned char smem[2][2][STAGE];      // [buffer][queries, dout]
    __shared__ __align__(16) float s_lse[2][KT], s_del[2][KT];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = a.B * a.Hk;
    const int jt = blockIdx.x / kvh, bh = blockIdx.x % kvh;           // the first tiles have the most queries under causality
    const int b = bh / a.Hk, hk = bh - b * a.Hk;
    const int j0 = jt * BQ, j1 = min(j0 + BQ, a.Tk) - 1, off = a.Tk - a.Tq;
    const int jw = j0 + 32 * w, j = jw + (lane & 31), jc = min(j, a.Tk - 1);
    const int jw1 = min(jw + 31, a.Tk - 1);
    Mask mk{a.causal, a.W, a.prefix ? a.prefix[b] : 0, a.Tk};
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
    // query tiles of 64 rows that may see these keys
    const bool pre = j0 < mk.prefix;
    int x0 = 0, x1 = (a.Tq + KT - 1) / KT;
    if (!pre) {
        const int lo = a.causal ? j0 : max(0, j0 - a.W + 1);          // the first position
        x0 = max(0, lo - off) / KT;
        if (a.W < a.Tk) x1 = min(x1, max(0, j1 + a.W - off + KT - 1) / KT);
    }
    const int2* range = docs ? a.range + (int64_t)b * a.ntd : nullptr;
    const unsigned lds = lds_addr(smem);
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int dt = 0; dt < DT; dt++) dk[dt] = dv[dt] = zero16();
    // the walk: heads of the group x query tiles
    int r = -1, base = x1;
    uint64_t act = 0, mine = 0, full = 0;
    auto next = [&](int& hq, int& xt, bool& some, bool& all) {
        while (!act) {
            base += 64;
            if (base >= x1) {
                if (++r >= a.R) { xt = -1; return; }
                base = x0;
            }
            const int x = base + lane;
            const bool in = x < x1;
            Span s{x * KT + off, min(x * KT + KT, a.Tq) - 1 + off, 0, 0, true};
            if (range && in) {
                const int2 ra = range[s.p0 / KT], rb = range[s.p1 / KT];
                s.lo = min(range_lo(ra), range_lo(rb));
                s.hi = max(ra.y, rb.y);
                s.one = range_one(ra) && range_one(rb) && ra.y == rb.y;
            }
            act = __ballot(in && mk.some(s, j0, j1) && (!range || (s.lo <= kw.hi && kw.lo <= s.hi)));
            mine = __ballot(in && jw <= jw1 && mk.some(s, jw, jw1) && (!range || (s.lo <= kv.hi && kv.lo <= s.hi)));
            full = __ballot(in && x * KT + KT <= a.Tq && mk.all(s, jw, jw + 31) && (!range || (s.one && kv.one && s.lo == kv.lo)));
        }
        const int i = __builtin_ctzll(act);
        act &= act - 1;
        xt = base + i;
        hq = hk * a.R + r;
        some = mine >> i & 1;
        all = full >> i & 1;
    };
    auto load = [&](int hq, int xt, int buf) {
        Load::issue((const T*)a.q + b * a.q_sb + hq * a.q_sh, a.q_st, xt * KT, a.Tq - 1, lds + (2 * buf) * STAGE, w, lane);
        Load::issue((const T*)a.dout + b * a.do_sb + hq * a.do_sh, a.do_st, xt * KT, a.Tq - 1, lds + (2 * buf + 1) * STAGE, w, lane);
    };
    auto stat = [&](int hq, int xt) {                 // threads 0..63 the log-sum-exp, 64..127 delta of a row
        const int t = xt * KT + (tid & 63);
        const int64_t i = ((int64_t)b * a.Hq + hq) * a.Tq + min(t, a.Tq - 1);
        const float v = tid < 64 ? a.lse[i] : a.delta[i];
        return t < a.Tq ? v : (tid < 64 ? INFINITY : 0.f);
    };
    int hq, xt, hn = 0, xn;
    bool some, all, some_n = false, all_n = false;
    next(hq, xt, some, all);
    float st = 0.f;
    if (xt >= 0) {
        if (tid < 128) st = stat(hq, xt);
        load(hq, xt, 0);
    }
    for (int buf = 0; xt >= 0; buf ^= 1, hq = hn, xt = xn, some = some_n, all = all_n) {
        if (tid < 64) s_lse[buf][tid] = st;
        else if (tid < 128) s_del[buf][tid - 64] = st;
        next(hn, xn, some_n, all_n);
        if (xn >= 0) {
            if (tid < 128) st = stat(hn, xn);
            load(hn, xn, buf ^ 1);
            wait_vm<2 * Load::N>();
        } else {
            wait_vm<0>();
        }
        __syncthreads();
        if (some) {
            const unsigned char* sq = smem[buf][0];
            const unsigned char* sd = smem[buf][1];
            const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
#pragma unroll
            for (int u = 0; u < 2; u++) {
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    s = mfma32<T>(Tile<D>::row_op(sq, 32 * u, kk, lane), kf[kk], s);
                    dp = mfma32<T>(Tile<D>::row_op(sd, 32 * u, kk, lane), vf[kk], dp);
                }
                const int t0 = xt * KT + 32 * u;
                float L[16], Dl[16];
#pragma unroll
                for (int g = 0; g < 4; g++) {
                    const float4 x = *reinterpret_cast<const float4*>(&s_lse[buf][32 * u + 8 * g + 4 * h]);
                    const float4 y = *reinterpret_cast<const float4*>(&s_del[buf][32 * u + 8 * g + 4 * h]);
                    L[4 * g] = x.x; L[4 * g + 1] = x.y; L[4 * g + 2] = x.z; L[4 * g + 3] = x.w;
                    Dl[4 * g] = y.x; Dl[4 * g + 1] = y.y; Dl[4 * g + 2] = y.z; Dl[4 * g + 3] = y.w;
                }
                probs<CAP, BIAS>(s, dp, a, slope, j, t0 + off, h, all, [&](int r_) { return L[r_]; }, [&](int r_) { return Dl[r_]; }, [&](int r_) {
                    const int tq = t0 + key_of(r_, h), pq = tq + off;
                    return tq < a.Tq && mk.sees(pq, j) && (!docs || a.ids[idb + min(pq, a.Tk - 1)] == dk_);
                });
#pragma unroll
                for (int mm = 0; mm < 2; mm++) {
                    const uint4 pp = pack8<T>(s, mm), ds = pack8<T>(dp, mm);
#pragma unroll
                    for (int dt = 0; dt < DT; dt++) {
                        dv[dt] = mfma32<T>(Tile<D>::col_op(sd, 32 * u, dt, mm, lane), pp, dv[dt]);
                        dk[dt] = mfma32<T>(Tile<D>::col_op(sq, 32 * u, dt, mm, lane), ds, dk[dt]);
                    }
                }
            }
        }
        __syncthreads();
    }
    if (j < a.Tk) {
        const int64_t o = (((int64_t)b * a.Tk + j) * a.Hk + hk) * D + 4 * h;
        const float f = a.scale;
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

template <typename T, int D, bool CAP, bool BIAS>
void launch_one(AttnArgs a, bool keys, hipStream_t st) {
    if (keys) {
        a.tiles = (a.Tk + BQ - 1) / BQ;
        slothost::launch(attn_dkv<T, D, CAP, BIAS>, dim3((unsigned)((int64_t)a.tiles * a.B * a.Hk)), dim3(BT), 0, st, a);
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

}  // namespace

// ======================================================================================== C-ABI
extern "C" size_t slotattn_bwd_workspace(int64_t B, int64_t Tq, int64_t Tk, int64_t Hq, int64_t Hk, int64_t D) { return 0; }

extern "C" int slotattn_bwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                            int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, int64_t B, int64_t Tq,
                            int64_t Tk, int64_t Hq, int64_t Hk, int64_t D, float scale, int causal, int64_t window, float cap,
                            const float* slopes, const void* docs, const int32_t* prefix, const void* out, const float* lse,
                            const void* dout, int64_t do_sb, int64_t do_sh, int64_t do_st, void* workspace, float* delta, void* dq,
                            void* dk, void* dv, void* stream) {
    if (int r = slotattn_host::check(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st, dtype, B, Tq, Tk, Hq, Hk, D, window, cap)) return r;
    if (Tq > Tk) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: more queries than keys");
    if (!out || !lse || !dout || !delta || !dq || !dk || !dv) return fail(SLOTSCAN_ERR_NULL, "slotattn_bwd: a required pointer is NULL");
    if (!al16(out) || !al16(dout) || !al16(dq) || !al16(dk) || !al16(dv) || !al16(docs) || (do_sb | do_sh | do_st) % 8)
        return fail(SLOTSCAN_ERR_ALIGN, "slotattn_bwd: rows of out, dout, dq, dk and dv, and docs, must be 16-byte aligned");
    if ((Tq + BQ - 1) / BQ * B * Hq > 0x7fffffffLL || (Tk + BQ - 1) / BQ * B * Hk > 0x7fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_bwd: shape too large");
    AttnArgs a = slotattn_host::args(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, v, v_sb, v_sh, v_st, B, Tq, Tk, Hq, Hk, scale, causal, window, cap,
                                     slopes, docs, prefix);
    a.out = (void*)out;
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
    return 0;
}
