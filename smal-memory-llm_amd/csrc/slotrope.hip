// Norm of every query and key head with the position rotation in the same pass, for MI355X (gfx950).
//
// Per row x of D values:  y = x r w,  r = rsqrt(mean x^2 + eps);  then every pair (a, b) of the first rot values turns:
// (a cos - b sin, b cos + a sin).  Backward, with the upstream gradient turned back to g (the transposed rotation),
// u = x r and h = g w:   dx = r (h - u mean(h u)),   dw = sum over all rows of g u.
//
// Memory-bound: each direction reads its rows once and writes them once.  A group of D / 8 consecutive lanes owns a
// token and walks over its heads with 8 consecutive values a lane (one 16-byte access for 16-bit types), so the angles --
// an fp64 product reduced to a fraction of a turn, then one sine and cosine per pair -- are formed once per token, not
// once per row.  Row sums are DPP sums over the group; the partner of a pair (i, i + rot / 2) sits rot / 16 lanes away in
// the same group and is fetched as the raw 16-byte piece.
#include "slot_common.h"
#include "slotscan.h"
#include "slotrope.h"
#include "slot_host.h"

using namespace slot;
using slothost::fail;
using slothost::hip_fail;
using slothost::al16;

#define RT 256                                       // threads per workgroup
#define RU 4                                         // rows in flight per group
#define RB_BLOCKS 1024                               // backward: workgroups at most (partials of the gains' gradients)

namespace {

typedef _Float16 f16_t;

// 8 consecutive values of one row as they lie in memory
template <typename T> struct Raw8 { uint4 v; };
template <> struct Raw8<float> { uint4 v, w; };

template <typename T> __device__ __forceinline__ Raw8<T> ldr(const T* p) { return {*reinterpret_cast<const uint4*>(p)}; }
template <> __device__ __forceinline__ Raw8<float> ldr<float>(const float* p) {
    return {*reinterpret_cast<const uint4*>(p), *reinterpret_cast<const uint4*>(p + 4)};
}
template <typename T> __device__ __forceinline__ void str(T* p, const Raw8<T>& r) { *reinterpret_cast<uint4*>(p) = r.v; }
template <> __device__ __forceinline__ void str<float>(float* p, const Raw8<float>& r) {
    *reinterpret_cast<uint4*>(p) = r.v;
    *reinterpret_cast<uint4*>(p + 4) = r.w;
}
__device__ __forceinline__ void widen(const Raw8<bf16_t>& r, float (&f)[8]) {
    const uint32_t x[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
    for (int i = 0; i < 4; i++) { f[2 * i] = __uint_as_float(x[i] << 16); f[2 * i + 1] = __uint_as_float(x[i] & 0xffff0000u); }
}
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ void widen(const Raw8<f16_t>& r, float (&f)[8]) {
    const f16x8 x = __builtin_bit_cast(f16x8, r.v);
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = (float)x[i];
}
__device__ __forceinline__ void widen(const Raw8<float>& r, float (&f)[8]) {
    const uint32_t x[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
    for (int i = 0; i < 8; i++) f[i] = __uint_as_float(x[i]);
}
__device__ __forceinline__ void narrow(const float (&f)[8], Raw8<bf16_t>& r) {
    r.v = make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
}
__device__ __forceinline__ void narrow(const float (&f)[8], Raw8<f16_t>& r) {
    f16x8 x;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = (f16_t)f[i];
    r.v = __builtin_bit_cast(uint4, x);
}
__device__ __forceinline__ void narrow(const float (&f)[8], Raw8<float>& r) {
    r.v = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
    r.w = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
}
template <int LPR> __device__ __forceinline__ uint4 from_lane(uint4 v, int src) {
    return make_uint4(__shfl((int)v.x, src, LPR), __shfl((int)v.y, src, LPR), __shfl((int)v.z, src, LPR), __shfl((int)v.w, src, LPR));
}
template <int LPR, typename T> __device__ __forceinline__ Raw8<T> from_lane(const Raw8<T>& r, int src) { return {from_lane<LPR>(r.v, src)}; }
template <int LPR> __device__ __forceinline__ Raw8<float> from_lane(const Raw8<float>& r, int src) {
    return {from_lane<LPR>(r.v, src), from_lane<LPR>(r.w, src)};
}
// sum over the LPR (8 or 16) lanes of a group, at every lane
template <int LPR> __device__ __forceinline__ float groupsum(float v) {
    v += dppf<SLOT_DPP_XOR1>(v);
    v += dppf<SLOT_DPP_XOR2>(v);
    v += dppf<SLOT_DPP_HMIR>(v);
    if constexpr (LPR == 16) v += dppf<SLOT_DPP_MIR>(v);
    return v;
}

struct RopeArgs {
    const void* q; const void* k; const void* v;
    int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;
    const void* wq; const void* wk;
    int wdtype, rot, pos64;
    const double* freqs;
    const void* pos;
    int64_t pos_sb;
    const int32_t* lens;
    int64_t BT;
    int T, Hq, Hk, S, hs;                            // hs: heads per workgroup (grid y)
    float eps;
    void* qo; void* ko; void* vo;
    int64_t ko_sb, ko_sh, ko_st, vo_sb, vo_sh, vo_st;   // the caches
    const void* dqo; const void* dko;
    int64_t dq_sb, dq_sh, dq_st, dk_sb, dk_sh, dk_st;
    float* part;
};

__device__ __forceinline__ void load_gain(const void* w, int dtype, int e, float (&f)[8]) {
    if (!w) {
#pragma unroll
        for (int i = 0; i < 8; i++) f[i] = 1.f;
    } else if (dtype == SLOTSCAN_F32) {
        widen(ldr((const float*)w + e), f);
    } else if (dtype == SLOTSCAN_BF16) {
        widen(ldr((const bf16_t*)w + e), f);
    } else {
        widen(ldr((const f16_t*)w + e), f);
    }
}
__device__ __forceinline__ int64_t position(const RopeArgs& a, int64_t b, int t) {
    if (a.lens) return (int64_t)a.lens[b] - a.T + t;
    if (!a.pos) return t;
    return a.pos64 ? ((const int64_t*)a.pos)[b * a.pos_sb + t] : ((const int32_t*)a.pos)[b * a.pos_sb + t];
}
// A lane's part of the rotation: cosine and sine of the angles of its 8 values (halves: value e0 + j pairs with lane
// `partner`, the first half's sine negated) or of its 4 pairs (neighbours).  The turn is reduced in fp64: a position
// times a frequency keeps 53 bits, its fraction of a turn is exact to 2^-30 at positions of 2^23.
template <int D, bool PAIRS> struct Turn {
    float cs[PAIRS ? 4 : 8], sn[PAIRS ? 4 : 8];
    bool on;                                          // the lane's values are rotated
    int partner;
    __device__ __forceinline__ void set(const RopeArgs& a, int64_t pos, int c) {
        const int e0 = 8 * c, half = a.rot / 2;
        on = e0 < a.rot;
        const bool second = e0 >= half;
        partner = !on ? c : second ? c - half / 8 : c + half / 8;
        const double turns = (double)pos * 0.15915494309189533577;    // 1 / (2 pi)
        const int f0 = PAIRS ? e0 / 2 : (second ? e0 - half : e0);
#pragma unroll
        for (int i = 0; i < (PAIRS ? 4 : 8); i++) {
            cs[i] = 1.f;
            sn[i] = 0.f;
            if (on) {
                const double x = turns * a.freqs[f0 + i];
                sincospif(2.f * (float)(x - rint(x)), &sn[i], &cs[i]);
                if (!PAIRS && !second) sn[i] = -sn[i];
            }
        }
    }
    // y (own values) and p (the partner lane's, halves only), turned by the angle (dir 1) or back (dir -1)
    __device__ __forceinline__ void apply(const float (&y)[8], const float (&p)[8], float dir, float (&o)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            if constexpr (PAIRS) {
                const float s = dir * sn[i / 2];
                o[i] = (i & 1) ? fmaf(y[i], cs[i / 2], y[i - 1] * s) : fmaf(y[i], cs[i / 2], -y[i + 1] * s);
            } else {
                o[i] = fmaf(y[i], cs[i], dir * sn[i] * p[i]);
            }
        }
    }
};

// ------------------------------------------------------------------------------------------- forward
template <typename T, int D, bool PAIRS, bool CACHE>
__global__ __launch_bounds__(RT) void rope_fwd(RopeArgs a) {
    constexpr int LPR = D / 8, GPB = RT / LPR;
    const int c = threadIdx.x % LPR, e0 = 8 * c;
    const int64_t tok = (int64_t)blockIdx.x * GPB + threadIdx.x / LPR;
    if (tok >= a.BT) return;                          // whole groups: nothing below crosses a group
    const int64_t b = tok / a.T;
    const int t = (int)(tok - b * a.T);
    const int64_t pos = position(a, b, t);
    const int all = a.Hq + (CACHE ? 2 : 1) * a.Hk;
    const int h0 = blockIdx.y * a.hs, h1 = min(h0 + a.hs, all);
    Turn<D, PAIRS> turn;
    turn.set(a, pos, c);
    const T* xq = (const T*)a.q + b * a.q_sb + t * a.q_st + e0;
    const T* xk = (const T*)a.k + b * a.k_sb + t * a.k_st + e0;
    const T* xv = CACHE ? (const T*)a.v + b * a.v_sb + t * a.v_st + e0 : nullptr;
    T* oq = (T*)a.qo + (tok * a.Hq) * D + e0;
    const bool kept = !CACHE || (pos >= 0 && pos < a.S);
    T* ok;
    T* ov = nullptr;
    if constexpr (CACHE) {
        ok = (T*)a.ko + b * a.ko_sb + (kept ? pos : 0) * a.ko_st + e0;
        ov = (T*)a.vo + b * a.vo_sb + (kept ? pos : 0) * a.vo_st + e0;
    } else {
        ok = (T*)a.ko + (tok * a.Hk) * D + e0;
    }
    const int64_t ok_sh = CACHE ? a.ko_sh : D;
    // one kind of head at a time: its gain (the partner's too) stays in registers
    auto rows = [&](const T* x, int64_t sh, const void* w, T* o, int64_t osh, int lo, int hi, bool put) {
        if (lo >= hi) return;
        float wo[8], wp[8];
        load_gain(w, a.wdtype, e0, wo);
        load_gain(w, a.wdtype, 8 * turn.partner, wp);
        for (int h = lo; h < hi; h += RU) {
            Raw8<T> r[RU];
#pragma unroll
            for (int u = 0; u < RU; u++) r[u] = ldr(x + min(h + u, hi - 1) * sh);
#pragma unroll
            for (int u = 0; u < RU; u++) {
                float f[8], p[8], y[8];
                widen(r[u], f);
                float ss = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++) ss = fmaf(f[i], f[i], ss);
                const float rr = 1.f / sqrtf(groupsum<LPR>(ss) * (1.f / D) + a.eps);
                if constexpr (!PAIRS) {
                    widen(from_lane<LPR>(r[u], turn.partner), p);
#pragma unroll
                    for (int i = 0; i < 8; i++) p[i] *= rr * wp[i];
                }
#pragma unroll
                for (int i = 0; i < 8; i++) f[i] *= rr * wo[i];
                turn.apply(f, p, 1.f, y);
                Raw8<T> out;
                narrow(y, out);
                if (put && h + u < hi) str(o + (h + u) * osh, out);
            }
        }
    };
    rows(xq, a.q_sh, a.wq, oq, D, h0, min(h1, a.Hq), true);
    rows(xk, a.k_sh, a.wk, ok, ok_sh, max(h0 - a.Hq, 0), min(h1 - a.Hq, a.Hk), kept);
    if constexpr (CACHE) {
        const int lo = max(h0 - a.Hq - a.Hk, 0), hi = h1 - a.Hq - a.Hk;
        if (kept)
            for (int h = lo; h < hi; h++) str(ov + h * a.vo_sh, ldr(xv + h * a.v_sh));
    }
}

// ------------------------------------------------------------------------------------------- backward
// The gains' gradients: every lane sums g u of its 8 columns over the rows it meets, a workgroup sums its groups in
// order, and rope_reduce the workgroups' partials in order: fixed, whatever the schedule.
template <typename T, int D, bool PAIRS>
__global__ __launch_bounds__(RT) void rope_bwd(RopeArgs a) {
    constexpr int LPR = D / 8, GPB = RT / LPR;
    __shared__ float s_part[2][GPB][D];
    const int c = threadIdx.x % LPR, e0 = 8 * c, grp = threadIdx.x / LPR;
    const int h0 = blockIdx.y * a.hs, h1 = min(h0 + a.hs, a.Hq + a.Hk);
    float dw[2][8];
#pragma unroll
    for (int i = 0; i < 8; i++) dw[0][i] = dw[1][i] = 0.f;
    for (int64_t tok = (int64_t)blockIdx.x * GPB + grp; tok < a.BT; tok += (int64_t)gridDim.x * GPB) {
        const int64_t b = tok / a.T;
        const int t = (int)(tok - b * a.T);
        Turn<D, PAIRS> turn;
        turn.set(a, position(a, b, t), c);
        auto rows = [&](const T* x, int64_t sh, const T* dy, int64_t dsh, const void* w, T* o, int lo, int hi, float (&dwa)[8]) {
            if (lo >= hi) return;
            float wo[8];
            load_gain(w, a.wdtype, e0, wo);
            for (int h = lo; h < hi; h += RU) {
                Raw8<T> r[RU], d[RU];
#pragma unroll
                for (int u = 0; u < RU; u++) {
                    r[u] = ldr(x + min(h + u, hi - 1) * sh);
                    d[u] = ldr(dy + min(h + u, hi - 1) * dsh);
                }
#pragma unroll
                for (int u = 0; u < RU; u++) {
                    float f[8], p[8], y[8], g[8];
                    widen(r[u], f);
                    widen(d[u], y);
                    float ss = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) ss = fmaf(f[i], f[i], ss);
                    const float rr = 1.f / sqrtf(groupsum<LPR>(ss) * (1.f / D) + a.eps);
                    if constexpr (!PAIRS) widen(from_lane<LPR>(d[u], turn.partner), p);
                    turn.apply(y, p, -1.f, g);
                    const bool in = h + u < hi;
                    float hu = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        f[i] *= rr;                   // u
                        if (in) dwa[i] = fmaf(g[i], f[i], dwa[i]);
                        g[i] *= wo[i];                // h
                        hu = fmaf(g[i], f[i], hu);
                    }
                    hu = groupsum<LPR>(hu) * (1.f / D);
#pragma unroll
                    for (int i = 0; i < 8; i++) y[i] = rr * fmaf(-f[i], hu, g[i]);
                    Raw8<T> out;
                    narrow(y, out);
                    if (in) str(o + (h + u) * D, out);
                }
            }
        };
        rows((const T*)a.q + b * a.q_sb + t * a.q_st + e0, a.q_sh, (const T*)a.dqo + b * a.dq_sb + t * a.dq_st + e0, a.dq_sh,
             a.wq, (T*)a.qo + tok * a.Hq * D + e0, h0, min(h1, a.Hq), dw[0]);
        rows((const T*)a.k + b * a.k_sb + t * a.k_st + e0, a.k_sh, (const T*)a.dko + b * a.dk_sb + t * a.dk_st + e0, a.dk_sh,
             a.wk, (T*)a.ko + tok * a.Hk * D + e0, max(h0 - a.Hq, 0), min(h1 - a.Hq, a.Hk), dw[1]);
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        s_part[0][grp][e0 + i] = dw[0][i];
        s_part[1][grp][e0 + i] = dw[1][i];
    }
    __syncthreads();
    if ((int)threadIdx.x < 2 * D) {
        const int which = threadIdx.x / D, col = threadIdx.x % D;
        float s = 0.f;
        for (int i = 0; i < GPB; i++) s += s_part[which][i][col];
        a.part[((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * D + threadIdx.x] = s;
    }
}

__device__ __forceinline__ void put_gain(void* w, int dtype, int i, float v) {
    if (!w) return;
    if (dtype == SLOTSCAN_F32) ((float*)w)[i] = v;
    else if (dtype == SLOTSCAN_BF16) ((bf16_t*)w)[i] = f2bf(v);
    else ((f16_t*)w)[i] = (f16_t)v;
}
// 16 columns a workgroup, its 16 lanes of a column over every 16th partial
__global__ __launch_bounds__(256) void rope_reduce(const float* part, int n, int D, int wdtype, void* dwq, void* dwk) {
    __shared__ float s[16][17];
    const int i = threadIdx.x & 15, j = threadIdx.x >> 4, col = blockIdx.x * 16 + i;
    float v = 0.f;
#pragma unroll 8
    for (int r = j; r < n; r += 16) v += part[(int64_t)r * 2 * D + col];
    s[j][i] = v;
    __syncthreads();
    if (j == 0) {
        v = 0.f;
        for (int r = 0; r < 16; r++) v += s[r][i];
        put_gain(col < D ? dwq : dwk, wdtype, col % D, v);
    }
}

template <typename T, int D, bool PAIRS>
void launch_kind(const RopeArgs& a, int dir, dim3 grid, hipStream_t st) {
    if (dir == 0) slothost::launch(rope_fwd<T, D, PAIRS, false>, grid, dim3(RT), 0, st, a);
    else if (dir == 1) slothost::launch(rope_fwd<T, D, PAIRS, true>, grid, dim3(RT), 0, st, a);
    else slothost::launch(rope_bwd<T, D, PAIRS>, grid, dim3(RT), 0, st, a);
}
template <typename T>
void launch_type(const RopeArgs& a, int D, int pairs, int dir, dim3 grid, hipStream_t st) {
    if (D == 128) pairs ? launch_kind<T, 128, true>(a, dir, grid, st) : launch_kind<T, 128, false>(a, dir, grid, st);
    else pairs ? launch_kind<T, 64, true>(a, dir, grid, st) : launch_kind<T, 64, false>(a, dir, grid, st);
}
int launch_rope(const RopeArgs& a, int dtype, int D, int pairs, int dir, dim3 grid, hipStream_t st) {
    if (dtype == SLOTSCAN_F32) launch_type<float>(a, D, pairs, dir, grid, st);
    else if (dtype == SLOTSCAN_BF16) launch_type<bf16_t>(a, D, pairs, dir, grid, st);
    else launch_type<f16_t>(a, D, pairs, dir, grid, st);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "rope launch");
}

// Heads per workgroup: a group walks over all of a token's heads (its angles are formed once) unless the tokens alone do
// not give every CU a few waves; then the heads are split, down to the RU rows that a group has in flight anyway.
int heads_per_group(int64_t BT, int heads, int D) {
    const int64_t waves = (BT * (D / 8) + 63) / 64;
    int hs = heads;
    while (hs > RU && waves * ((heads + hs - 1) / hs) < 2048) hs = (hs + 1) / 2;
    return (hs + RU - 1) / RU * RU;
}

int check_rope(const void* q, const void* k, int dtype, int wdtype, const void* wq, const void* wk, const double* freqs,
               int64_t rot, int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, const char* what) {
    if (B < 1 || T < 1 || Hq < 1 || Hk < 1) return fail(SLOTSCAN_ERR_SHAPE, "slotrope: B, T, Hq, Hk must be >= 1");
    if (D != 64 && D != 128) return fail(SLOTSCAN_ERR_SHAPE, "slotrope: D must be 64 or 128");
    if (rot < 0 || rot > D || rot % 16) return fail(SLOTSCAN_ERR_SHAPE, "slotrope: rot must be a multiple of 16 in [0, D]");
    if (T > 0x7fffffffLL || Hq + 2 * Hk > 65535 || B > 0x7fffffffLL || B * T > (0x7fffffffLL - 1024) * 16)
        return fail(SLOTSCAN_ERR_SHAPE, "slotrope: shape too large");
    if (dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2) return fail(SLOTSCAN_ERR_DTYPE, "slotrope: unknown dtype");
    if (!q || !k || (rot && !freqs)) return fail(SLOTSCAN_ERR_NULL, "slotrope: a required pointer is NULL");
    if (!al16(q) || !al16(k) || !al16(wq) || !al16(wk)) return fail(SLOTSCAN_ERR_ALIGN, "slotrope: q, k, wq and wk must be 16-byte aligned");
    return 0;
}
// rows 16-byte aligned: every stride a multiple of 16 bytes
bool rows16(int dtype, int64_t a, int64_t b, int64_t c) {
    const int64_t m = dtype == SLOTSCAN_F32 ? 4 : 8;
    return a % m == 0 && b % m == 0 && c % m == 0;
}

RopeArgs base_args(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                   int64_t k_st, const void* wq, const void* wk, int wdtype, const double* freqs, int64_t rot, int64_t B,
                   int64_t T, int64_t Hq, int64_t Hk, float eps) {
    RopeArgs a{};
    a.q = q; a.k = k;
    a.q_sb = q_sb; a.q_sh = q_sh; a.q_st = q_st; a.k_sb = k_sb; a.k_sh = k_sh; a.k_st = k_st;
    a.wq = wq; a.wk = wk; a.wdtype = wdtype; a.rot = (int)rot; a.freqs = freqs;
    a.BT = B * T; a.T = (int)T; a.Hq = (int)Hq; a.Hk = (int)Hk; a.eps = eps;
    return a;
}
// workgroups of the backward: tokens x heads
void bwd_grid(int64_t B, int64_t T, int64_t heads, int64_t D, int& hs, dim3& grid) {
    hs = heads_per_group(B * T, (int)heads, (int)D);
    const int64_t gy = (heads + hs - 1) / hs, gpb = RT / (D / 8), need = (B * T + gpb - 1) / gpb;
    int64_t gx = RB_BLOCKS / gy < 1 ? 1 : RB_BLOCKS / gy;
    if (gx > need) gx = need;
    grid = dim3((unsigned)gx, (unsigned)gy);
}

}  // namespace

// ======================================================================================== C-ABI
extern "C" int slotrope_fwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                            int64_t k_st, int dtype, const void* wq, const void* wk, int wdtype, const double* freqs,
                            int64_t rot, int interleaved, const void* pos, int pos64, int64_t pos_sb, int64_t B, int64_t T,
                            int64_t Hq, int64_t Hk, int64_t D, float eps, void* qo, void* ko, void* stream) {
    if (int r = check_rope(q, k, dtype, wdtype, wq, wk, freqs, rot, B, T, Hq, Hk, D, "slotrope_fwd")) return r;
    if (!qo || !ko) return fail(SLOTSCAN_ERR_NULL, "slotrope_fwd: a required pointer is NULL");
    if (!al16(qo) || !al16(ko) || !rows16(dtype, q_sb, q_sh, q_st) || !rows16(dtype, k_sb, k_sh, k_st))
        return fail(SLOTSCAN_ERR_ALIGN, "slotrope_fwd: rows of q, k, qo and ko must be 16-byte aligned");
    RopeArgs a = base_args(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, wq, wk, wdtype, freqs, rot, B, T, Hq, Hk, eps);
    a.pos = pos; a.pos64 = pos64; a.pos_sb = pos_sb;
    a.qo = qo; a.ko = ko;
    const int heads = (int)(Hq + Hk), gpb = RT / (int)(D / 8);
    a.hs = heads_per_group(B * T, heads, (int)D);
    hipStream_t st = (hipStream_t)stream;
    slothost::Scope sc(SLOTSCAN_K_ROPE, st);
    return launch_rope(a, dtype, (int)D, interleaved, 0, dim3((unsigned)((B * T + gpb - 1) / gpb), (unsigned)((heads + a.hs - 1) / a.hs)), st);
}

extern "C" size_t slotrope_bwd_workspace(int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D) {
    if (B < 1 || T < 1 || Hq < 1 || Hk < 1 || (D != 64 && D != 128)) return 0;
    int hs;
    dim3 g;
    bwd_grid(B, T, Hq + Hk, D, hs, g);
    return (size_t)g.x * g.y * 2 * D * sizeof(float);
}

extern "C" int slotrope_bwd(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                            int64_t k_st, int dtype, const void* wq, const void* wk, int wdtype, const double* freqs,
                            int64_t rot, int interleaved, const void* pos, int pos64, int64_t pos_sb, int64_t B, int64_t T,
                            int64_t Hq, int64_t Hk, int64_t D, float eps, const void* dqo, int64_t dq_sb, int64_t dq_sh,
                            int64_t dq_st, const void* dko, int64_t dk_sb, int64_t dk_sh, int64_t dk_st, void* workspace,
                            void* dq, void* dk, void* dwq, void* dwk, void* stream) {
    if (int r = check_rope(q, k, dtype, wdtype, wq, wk, freqs, rot, B, T, Hq, Hk, D, "slotrope_bwd")) return r;
    if (!dqo || !dko || !dq || !dk || ((dwq || dwk) && !workspace))
        return fail(SLOTSCAN_ERR_NULL, "slotrope_bwd: a required pointer is NULL");
    if (!al16(dqo) || !al16(dko) || !al16(dq) || !al16(dk) || !al16(workspace) || !rows16(dtype, q_sb, q_sh, q_st) ||
        !rows16(dtype, k_sb, k_sh, k_st) || !rows16(dtype, dq_sb, dq_sh, dq_st) || !rows16(dtype, dk_sb, dk_sh, dk_st))
        return fail(SLOTSCAN_ERR_ALIGN, "slotrope_bwd: rows of every token tensor and the workspace must be 16-byte aligned");
    RopeArgs a = base_args(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, wq, wk, wdtype, freqs, rot, B, T, Hq, Hk, eps);
    a.pos = pos; a.pos64 = pos64; a.pos_sb = pos_sb;
    a.dqo = dqo; a.dko = dko;
    a.dq_sb = dq_sb; a.dq_sh = dq_sh; a.dq_st = dq_st; a.dk_sb = dk_sb; a.dk_sh = dk_sh; a.dk_st = dk_st;
    a.qo = dq; a.ko = dk;
    a.part = (dwq || dwk) ? (float*)workspace : nullptr;
    dim3 grid;
    bwd_grid(B, T, Hq + Hk, D, a.hs, grid);
    hipStream_t st = (hipStream_t)stream;
    {
        slothost::Scope sc(SLOTSCAN_K_ROPE_BWD, st);
        if (int r = launch_rope(a, dtype, (int)D, interleaved, 2, grid, st)) return r;
    }
    if (!a.part) return 0;
    slothost::launch(rope_reduce, dim3((unsigned)(2 * D / 16)), dim3(256), 0, st, (const float*)a.part, (int)(grid.x * grid.y),
                     (int)D, wdtype, dwq, dwk);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "rope_reduce launch");
}

extern "C" int slotrope_cache(const void* q, int64_t q_sb, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sb, int64_t k_sh,
                              int64_t k_st, const void* v, int64_t v_sb, int64_t v_sh, int64_t v_st, int dtype, const void* wq,
                              const void* wk, int wdtype, const double* freqs, int64_t rot, int interleaved, const int32_t* lens,
                              int64_t B, int64_t T, int64_t Hq, int64_t Hk, int64_t D, int64_t S, float eps, void* qo, void* kc,
                              int64_t kc_sb, int64_t kc_sh, int64_t kc_st, void* vc, int64_t vc_sb, int64_t vc_sh, int64_t vc_st,
                              void* stream) {
    if (int r = check_rope(q, k, dtype, wdtype, wq, wk, freqs, rot, B, T, Hq, Hk, D, "slotrope_cache")) return r;
    if (S < 1 || S > 0x7fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotrope_cache: S must be in [1, 2^31)");
    if (!v || !lens || !qo || !kc || !vc) return fail(SLOTSCAN_ERR_NULL, "slotrope_cache: a required pointer is NULL");
    if (!al16(v) || !al16(qo) || !al16(kc) || !al16(vc) || !rows16(dtype, q_sb, q_sh, q_st) || !rows16(dtype, k_sb, k_sh, k_st) ||
        !rows16(dtype, v_sb, v_sh, v_st) || !rows16(dtype, kc_sb, kc_sh, kc_st) || !rows16(dtype, vc_sb, vc_sh, vc_st))
        return fail(SLOTSCAN_ERR_ALIGN, "slotrope_cache: rows of q, k, v, qo and the caches must be 16-byte aligned");
    RopeArgs a = base_args(q, q_sb, q_sh, q_st, k, k_sb, k_sh, k_st, wq, wk, wdtype, freqs, rot, B, T, Hq, Hk, eps);
    a.v = v; a.v_sb = v_sb; a.v_sh = v_sh; a.v_st = v_st;
    a.lens = lens; a.S = (int)S;
    a.qo = qo; a.ko = kc; a.vo = vc;
    a.ko_sb = kc_sb; a.ko_sh = kc_sh; a.ko_st = kc_st; a.vo_sb = vc_sb; a.vo_sh = vc_sh; a.vo_st = vc_st;
    const int heads = (int)(Hq + 2 * Hk), gpb = RT / (int)(D / 8);
    a.hs = heads_per_group(B * T, heads, (int)D);
    hipStream_t st = (hipStream_t)stream;
    slothost::Scope sc(SLOTSCAN_K_ROPE, st);
    return launch_rope(a, dtype, (int)D, interleaved, 1, dim3((unsigned)((B * T + gpb - 1) / gpb), (unsigned)((heads + a.hs - 1) / a.hs)), st);
}
