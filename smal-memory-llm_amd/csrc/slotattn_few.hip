// Attention over a cache in pages where a sequence has few query rows: a generated token, a few guessed ones (slot_attn_pages.h).
//
// One 32-row tile of a key/value head against 32-key tiles, each wave through a ring of its own of two tiles without a barrier in the loop.
//   SHARED  every wave is a worker with an equal share of all units' tiles; keys are fetched across the units' borders
//   SINGLE  a workgroup's NW waves share one unit, every NW-th tile each, and meet in LDS: no join behind it
#include "slot_attn_pages.h"
#include "slotscan.h"
#include "slot_attn_few.h"

using namespace slotattn;

namespace {

__device__ __forceinline__ int scan_up(int x, int lane) {            // sum over the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}
// 32-row tiles of a sequence, and 32-key tiles of each: those that its tokens see together, so that no table of them is needed
__device__ __forceinline__ int few_tiles(const PagedArgs& a, const Seq& x, int& per) {
    int lo, hi;
    keys_of<32>(a, x, x.end - x.n, x.end - 1, lo, hi);
    per = max(1, (hi - lo + 31) >> 5);
    return (x.n * a.rep + 31) >> 5;
}
__device__ __forceinline__ int few_cost(const PagedArgs& a, int r) {
    if (r >= a.R) return 0;
    int per;
    const int t = few_tiles(a, seq_of(a, r), per);
    return t * per;
}

// A wave's way through its tiles.  unit() enters the next unit, tile() finds the next of its tiles (every `step` / 32-th) that any row sees.
struct Walker {
    int r, base, x, end;                              // row, tiles of one head in front of it, the worker's next tile and its end
    Seq sq;
    int per, hk, t, ka, kb, lo, hi, j;
    Span s;
    __device__ __forceinline__ void enter(const PagedArgs& a) {       // tile rows t, key tiles [ka, kb)
        const int rows = sq.n * a.rep, off = sq.end - sq.n, r0 = 32 * t;
        keys_of<32>(a, sq, off, sq.end - 1, lo, hi);
        s = {r0 / a.rep + off, (min(r0 + 32, rows) - 1) / a.rep + off, 0, 0, true};
        hi = min(hi, lo + 32 * kb);
    }
    __device__ __forceinline__ bool unit(const PagedArgs& a) {
        while (x < end) {
            sq = seq_uni(a, r);
            const int cost = few_tiles(a, sq, per) * per, y = x - base * a.Hk;
            if (y >= cost * a.Hk) {                   // the next row
                if (++r >= a.R) return false;
                base += cost;
                continue;
            }
            hk = y / cost;
            const int z = y - hk * cost;
            t = z / per;
            ka = z - t * per;
            kb = min(per, ka + end - x);
            x += kb - ka;
            enter(a);
            j = lo + 32 * ka - 32;
            return true;
        }
        return false;
    }
    __device__ __forceinline__ bool tile(const Mask& mk, int step) {
        do j += step; while (j < hi && !mk.some(s, j, j + 31));
        return j < hi;
    }
};

template <typename T, int D, bool CAP, bool BIAS, int NW, bool SHARED>
__global__ __launch_bounds__(64 * NW) void pages_few(PagedArgs a) {
    constexpr int KK = D / 16, DT = D / 32, ST = 32 * 2 * D;
    typedef PageLoad<D, 32, 1> Load;
    __shared__ __align__(1024) unsigned char smem[NW][2][2][ST];     // [wave][buffer][keys, values]
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
    Walker c{};                                       // the tiles that are computed
    int me = 0, total = 0, G = 1;
    if constexpr (SHARED) {
        const int C = (a.R + 63) / 64;
        int mine = 0;
        for (int i = 0; i < C; i++) mine += few_cost(a, lane * C + i);
        const int upto = scan_up(mine, lane);
        total = lane_of(upto, 63) * a.Hk;
        G = min((int)gridDim.x, max(total / FS, 1));
        me = blockIdx.x;
        if (me < G) {
            if (G % 8 == 0) me = (me & 7) * (G / 8) + (me >> 3);     // workers that follow each other run on one XCD
            const Shares sh(total, G);
            c.x = sh.begin(me);
            c.end = sh.begin(me + 1);
            const int y = c.x / a.Hk, L = 63 - __builtin_clzll(__ballot(upto - mine <= y) | 1);
            c.base = lane_of(upto - mine, L);
            c.r = L * C;
            for (int i0 = 0; C > 1 && i0 < C; i0 += 64) {            // the row within the lane's rows
                const int cost = i0 + lane < C ? few_cost(a, c.r + i0 + lane) : 0, u = scan_up(cost, lane), all = lane_of(u, 63);
                if (c.base + all <= y) { c.base += all; continue; }
                const int k = 63 - __builtin_clzll(__ballot(c.base + u - cost <= y) | 1);
                c.base += lane_of(u - cost, k);
                c.r += i0 + k;
                break;
            }
        }
    } else {
        c.r = blockIdx.z;
        c.hk = blockIdx.y;
        c.t = blockIdx.x;
    }
    const unsigned lds = lds_addr(smem[w]);
    const Load lk(a.k_sp, a.k_st, a.shift, 0, lane), lv(a.v_sp, a.v_st, a.shift, 0, lane);
    const Ops<D> ops(lane);
    const float f2 = fabsf(a.s.f);
    RowSums<T, D, BIAS> sum(f2);
    // the tiles that are loaded, two ahead
    Walker f;
    Pages<2> pg;
    const T* fk = nullptr;
    const T* fv = nullptr;
    bool open = false;                                // f is in a unit
    auto fetch = [&]() -> bool {
        for (;;) {
            if (!open) {
                if (!SHARED || !f.unit(a)) return false;
                open = true;
                fk = (const T*)a.k + f.hk * a.k_sh;
                fv = (const T*)a.v + f.hk * a.v_sh;
            }
            if (f.tile(Mask{1, a.W, f.sq.pre, f.sq.klen}, 32 * NW)) break;
            open = false;
        }
        pg.fetch(a, f.r * a.t_sr, f.j, f.sq.klen);
        return true;
    };
    auto keys = [&](int buf) { lk.issue(fk, pg, f.j, f.sq.klen - 1, lds + (2 * buf) * ST); };
    auto values = [&](int buf) { lv.issue(fv, pg, f.j, f.sq.klen - 1, lds + (2 * buf + 1) * ST); };
    bool e0 = false, e1 = false, e2 = false;          // this tile and the next are on their way, the one after them is known
    uint32_t lost0 = 0, lost1 = 0;
    auto begin = [&]() {
        e0 = fetch();
        if (e0) {
            keys(0);
            values(0);
            lost0 = pg.lost;
            e1 = fetch();
        }
        if (e1) {
            keys(1);
            values(1);
            lost1 = pg.lost;
            e2 = fetch();
        }
    };
    int buf = 0;
    if constexpr (SHARED) {
        f = c;
        begin();
    }
    for (;;) {
        if constexpr (SHARED) {
            if (!c.unit(a)) break;
        } else {
            c.sq = seq_uni(a, c.r);
            if (c.t >= few_tiles(a, c.sq, c.per)) break;
            c.ka = 0;
            c.kb = c.per;
            c.enter(a);
            c.j = c.lo + 32 * (w - NW);
            f = c;
            open = true;
            fk = (const T*)a.k + f.hk * a.k_sh;
            fv = (const T*)a.v + f.hk * a.v_sh;
            e1 = e2 = false;
            buf = 0;
            begin();
        }
        const int rows = c.sq.n * a.rep, off = c.sq.end - c.sq.n, r0 = 32 * c.t, row = min(r0 + (lane & 31), rows - 1);
        const int tok = row / a.rep, hq = c.hk * a.rep + row - tok * a.rep, p = tok + off;
        const Mask mk{1, a.W, c.sq.pre, c.sq.klen};
        const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
        uint4 qf[KK];
        {
            const T* q = (const T*)a.q + hq * a.q_sh + (int64_t)(c.sq.s + tok) * a.q_st + 8 * h;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) qf[kk] = ld16(q + 16 * kk);
        }
        if (a.s.f < 0.f)                              // a negative scale: of the queries' sign, so that larger products are larger scores
#pragma unroll
            for (int kk = 0; kk < KK; kk++) { qf[kk].x ^= 0x80008000u; qf[kk].y ^= 0x80008000u; qf[kk].z ^= 0x80008000u; qf[kk].w ^= 0x80008000u; }
        const Rows rw{c.sq.s, tok, hq, p, min(32, rows - r0), Sees::query(mk, p), slope};
        sum.clear();
        // Keys and values are fetched two tiles ahead, each into the place that it has just been read from: a wave has one and a half to two
        // tiles on their way while it computes.
        for (; c.tile(mk, 32 * NW); buf ^= 1) {
            const int j0 = c.j;
            if (e1) wait_vm<3 * Load::N>();           // behind this tile's keys: its values, the next keys and values
            else wait_vm<Load::N>();
            asm volatile("" ::: "memory");
            const unsigned bo = lds + (2 * buf) * ST, rk = bo + ops.row, cc = bo + ops.col, c8 = bo + ops.col8;
            f32x16 sc[1] = {zero16()};
#pragma unroll
            for (int kk = 0; kk < KK; kk++) sc[0] = mfma32<T>(lds16(Ops<D>::k_step(rk, kk)), qf[kk], sc[0]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the keys are read before their place is filled again
            if (e2) keys(buf);
            scores<CAP>(sc[0], a.s);
            if constexpr (BIAS) bias(sc[0], f2, slope, p, j0, h);
            if (lost0 || j0 + 32 > c.hi || !mk.all(c.s, j0, j0 + 31)) {
                uint32_t ok = seen16(rw.see, j0, h, j0 < mk.prefix, nullptr, 0);
                if (bit(lost0, 0)) ok &= ~0xffu;      // registers 0 .. 7 are keys of the first 16
                if (bit(lost0, 1)) ok &= 0xffu;
#pragma unroll
                for (int e = 0; e < 16; e++) sc[0][e] = j0 + key_of(e, h) < c.hi && bit(ok, e) ? sc[0][e] : -INFINITY;
            }
            uint4 pf[1][2];
            sum.template weigh<1>(sc, pf);
            if (e2) wait_vm<3 * Load::N>();           // behind the values: the next tile, the keys after it
            else if (e1) wait_vm<2 * Load::N>();
            else wait_vm<0>();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int mm = 0; mm < 2; mm++)
                    sum.o[dt] = mfma32<T>(Ops<D>::at_col(Ops<D>::block(cc, dt), Ops<D>::block(c8, dt), ST + 16 * mm * Tile<D>::ROWB), pf[0][mm], sum.o[dt]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the values, too
            lost0 = lost1;
            e1 = e2;
            if (e2) {
                values(buf);
                lost1 = pg.lost;
                e2 = fetch();
            }
        }
        const T* kb = (const T*)a.k + c.hk * a.k_sh;
        const T* vb = (const T*)a.v + c.hk * a.v_sh;
        const int32_t* tab = a.table + c.r * a.t_sr;
        if constexpr (SHARED) {
            finish<T, D, CAP, BIAS>(a, sum, rw, kb, vb, tab, c.lo + 32 * c.ka, c.hi, c.ka == 0 && c.kb == c.per, (int64_t)(2 * me + (c.ka == 0)) * 32, lane);
            if (c.ka == 0 && lane == 0)
                a.pieces[(((c.sq.s * a.rep) >> 5) + c.r + c.t) * a.Hk + c.hk] = {me, c.kb == c.per ? 1 : Shares(total, G).owner(c.end + c.per - c.kb - 1) - me + 1};
        } else {
            // the waves' parts: (m, l) of every row to all, then the weighted sums through LDS (its tiles are read)
            __shared__ float s_m[NW][32], s_l[NW][32], s_M[32], s_L[32];     // the waves' maxima and sums of every row, the workgroup's
            __shared__ uint32_t s_bad[NW];
            sum.close();
            if (h == 0) { s_m[w][lane] = sum.m; s_l[w][lane] = sum.l; }
            __syncthreads();
            float M = -INFINITY, Ls = 0.f;
#pragma unroll
            for (int i = 0; i < NW; i++) M = fmaxf(M, s_m[i][lane & 31]);
            const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
            for (int i = 0; i < NW; i++) Ls += s_l[i][lane & 31] * exp2_(s_m[i][lane & 31] - Mu);
            const float fm = exp2_(sum.m - Mu);
            float* so = reinterpret_cast<float*>(smem);               // [wave][row][D + 4]
            constexpr int SO = D + 4;
            static_assert(NW * 32 * SO * 4 <= (int)sizeof(smem), "the waves' sums fit");
            if ((lane & 31) < rw.used) {
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *reinterpret_cast<float4*>(so + (w * 32 + (lane & 31)) * SO + 32 * dt + 8 * g + 4 * h) =
                            make_float4(sum.o[dt][4 * g] * fm, sum.o[dt][4 * g + 1] * fm, sum.o[dt][4 * g + 2] * fm, sum.o[dt][4 * g + 3] * fm);
            }
            if (w == 0 && h == 0) s_L[lane] = Ls;     // not over s_l, which the other waves may still read
            float nf = sum.l * 0.f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) nf = nonfinite(sum.o[dt], nf);
            const uint32_t odd = row_bits(nf != 0.f && (lane & 31) < rw.used);
            if (lane == 0) s_bad[w] = odd;
            __syncthreads();
            uint32_t bad = 0;
#pragma unroll
            for (int i = 0; i < NW; i++) bad |= s_bad[i];
            if (bad) {                                // rows next to infinities and NaN, from their visible pairs alone; the same in every wave
                bad &= ~row_bits(Ls != Ls);
                for (; bad; bad &= bad - 1) {
                    const int i = __builtin_ctz(bad);
                    if (i % NW != w) continue;
                    float m1, l1, o1[D / 64];
                    exact_paged<T, D, CAP, BIAS>(a, (const T*)a.q + lane_of(hq, i) * a.q_sh + (int64_t)(c.sq.s + lane_of(tok, i)) * a.q_st, kb, vb, tab,
                                                 lane_of(rw.see, i), lane_of(slope, i), lane_of(p, i), c.lo, c.hi, lane, m1, l1, o1);
                    for (int ww = 0; ww < NW; ww++)
                        for (int e = 0; e < D / 64; e++) so[(ww * 32 + i) * SO + lane * (D / 64) + e] = ww ? 0.f : o1[e];
                    if (lane == 0) s_L[i] = l1;
                }
                __syncthreads();
            }
            // used rows x D values: 8 lanes a row
            for (int rr = tid >> 3; rr < rw.used; rr += 8 * NW) {
                const int c4 = 4 * (tid & 7), g = r0 + rr;
                const float lr = s_L[rr], inv = lr > 0.f || lr != lr ? 1.f / lr : 0.f;
                const int gt = g / a.rep, gh = c.hk * a.rep + g - gt * a.rep;
                const int64_t at = ((int64_t)(c.sq.s + gt) * a.Hq + gh) * D;
#pragma unroll
                for (int i = 0; i < D / 32; i++) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                    for (int ww = 0; ww < NW; ww++) {
                        const float4 y = *reinterpret_cast<const float4*>(so + (ww * 32 + rr) * SO + c4 + 32 * i);
                        v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
                    }
                    put4<T>(a.out, nullptr, at + c4 + 32 * i, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                }
            }
            c.t += gridDim.x;
            __syncthreads();                          // the sums are read before the next unit's tiles take their place
        }
    }
    fill_rest<D>(a, ((int64_t)(blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * 64 * NW + tid, (int64_t)gridDim.x * gridDim.y * gridDim.z * 64 * NW);
}

template <typename T, int D, bool CAP, bool BIAS>
void launch_one(const PagedArgs& a, int G, int tiles, hipStream_t st) {
    if (G) slothost::launch(pages_few<T, D, CAP, BIAS, 1, true>, dim3((unsigned)G), dim3(64), 0, st, a);
    else slothost::launch(pages_few<T, D, CAP, BIAS, FW, false>, dim3((unsigned)tiles, (unsigned)a.Hk, (unsigned)a.R), dim3(64 * FW), 0, st, a);
}
template <typename T, int D>
void launch_attn(const PagedArgs& a, bool cap, int G, int tiles, hipStream_t st) {
    if (cap) a.slopes ? launch_one<T, D, true, true>(a, G, tiles, st) : launch_one<T, D, true, false>(a, G, tiles, st);
    else a.slopes ? launch_one<T, D, false, true>(a, G, tiles, st) : launch_one<T, D, false, false>(a, G, tiles, st);
}

}  // namespace

void slotattn_few::launch(const PagedArgs& a, int dtype, int D, bool cap, int G, int tiles, hipStream_t st) {
    if (dtype == SLOTSCAN_BF16) D == 128 ? launch_attn<bf16_t, 128>(a, cap, G, tiles, st) : launch_attn<bf16_t, 64>(a, cap, G, tiles, st);
    else D == 128 ? launch_attn<f16_t, 128>(a, cap, G, tiles, st) : launch_attn<f16_t, 64>(a, cap, G, tiles, st);
}
