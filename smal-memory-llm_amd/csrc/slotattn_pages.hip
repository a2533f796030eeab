// Attention of the newest tokens of many sequences over a cache in pages, for MI355X (gfx950); semantics: include/slotattn.h.
//
// The query rows of a key/value head -- the tokens of a sequence times the query heads of the group -- are cut into tiles; a tile against the keys
// that it sees is a unit, and all units' key tiles in a row are shared out to the workers in equal contiguous pieces, so that neither
// ragged lengths nor causality leave a worker more than another.  A piece that is not a whole unit leaves its rows' maxima, sums and
// weighted values in the workspace, two such pieces a worker at most, and pages_join combines a unit's pieces in order.
//
//   pages_many   128 rows a workgroup, 32 per wave, 64-key tiles; pages_plan before it: the units' costs and their running sums
//   pages_few    32 rows, 32-key tiles
//   pages_join   pieces of one unit
#include "slot_attn_rows.h"
#include "slotscan.h"
#include "slotattn.h"
#include "slotpage.h"
#include "slot_attn_host.h"

using namespace slotattn;
using slothost::fail;
using slothost::hip_fail;
using slothost::al16;

#define MW 4                                         // waves of a workgroup of pages_many
#define MT (64 * MW)
#define MQ (32 * MW)                                 // its query rows
#define MG 512                                       // workgroups: two a CU
#define LT 1024                                      // threads of pages_plan
#define FG 1024                                      // waves of pages_few that share all units
#define FS 4                                         // tiles of one of them at least
#define FW 4                                         // waves of pages_few that share one
#define UNIT_KEYS 2048                               // keys of a row up to which they do

namespace {

struct Unit { int r, hk, t, n, parts; };             // what a worker leaves for the join: row, head, tile, tokens, pieces (0: nothing)

struct PagedArgs {
    AttnArgs s;                                       // the scores' constants
    const void* q; const void* k; const void* v;
    int64_t q_sh, q_st, k_sp, k_sh, k_st, v_sp, v_sh, v_st;
    const int32_t* table; int64_t t_sr;
    const int32_t* starts; const int32_t* ends; const int32_t* prefix; const float* slopes;
    int N, R, M, P, Hq, Hk, rep, W, shift, units;     // units: room for them in the plan
    int* plan;                                        // running costs of the rows (R + 1), first units of the rows (R + 1), running costs (units + 1)
    Unit* join; float* po; float2* pm;                // of every worker; (worker, head or tail, row of the tile)
    void* out;
};

// A sequence's part of the batch, whatever the tensors hold: tokens s .. s + n - 1 of [0, N), the first at position off
struct Seq { int s, n, end, klen, pre; };
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int r) {
    Seq x;
    x.s = min(max(a.starts[r], 0), a.N);
    x.n = min(max(a.starts[r + 1], x.s), a.N) - x.s;
    x.end = min(max(a.ends[r], 0), (1 << 30) - 1);
    x.klen = (int)min((int64_t)x.end, (int64_t)a.M << a.shift);
    x.pre = a.prefix ? a.prefix[r] : 0;
    return x;
}
// Keys that rows [r0, r1] of a tile see lie in [lo, hi), lo a multiple of STEP
template <int STEP> __device__ __forceinline__ void keys_of(const PagedArgs& a, const Seq& x, int p0, int p1, int& lo, int& hi) {
    lo = x.pre > 0 ? 0 : max(0, max(p0, 0) - a.W + 1) & ~(STEP - 1);
    hi = p1 < 0 ? lo : min(x.klen, max(p1 + 1, x.pre));
}

// A wave's 64 NR pages of a sequence from page wb on, NR a lane.  An id outside of the pages stands for page 0, and its keys are not seen.
template <int NR> struct Window {
    const int32_t* tab;
    int M, P, shift, used, lane, wb, ids[NR];         // used: pages that hold keys
    uint64_t bad[NR];
    __device__ __forceinline__ Window(const PagedArgs& a, int r, int klen, int l)
        : tab(a.table + r * a.t_sr), M(a.M), P(a.P), shift(a.shift), used((klen + (1 << a.shift) - 1) >> a.shift), lane(l), wb(-65536) {}
    __device__ __forceinline__ void at(int j0, int keys) {
        const int first = j0 >> shift, last = (j0 + keys - 1) >> shift;
        if (first >= wb && last - wb < 64 * NR) return;
        wb = first;
#pragma unroll
        for (int n = 0; n < NR; n++) ids[n] = tab[min(wb + 64 * n + lane, M - 1)];
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const bool in = wb + 64 * n + lane < used, b = in && (unsigned)ids[n] >= (unsigned)P;
            bad[n] = __ballot(b);
            ids[n] = in && !b ? ids[n] : 0;
        }
    }
    __device__ __forceinline__ int page(int j) const {                // j: of the wave
        const int i = (j >> shift) - wb;
        int x = __builtin_amdgcn_readlane(ids[0], i & 63);
#pragma unroll
        for (int n = 1; n < NR; n++) {
            const int y = __builtin_amdgcn_readlane(ids[n], i & 63);
            x = i >= 64 * n ? y : x;
        }
        return x;
    }
    // the groups of 16 keys from j0 on, as bits, that lie in no page
    __device__ __forceinline__ uint32_t lost(int j0, int keys) const {
        uint32_t x = 0;
        uint64_t any = bad[0];
#pragma unroll
        for (int n = 1; n < NR; n++) any |= bad[n];
        if (any)
            for (int g = 0; g < keys / 16; g++) {
                const int i = ((j0 + 16 * g) >> shift) - wb;
                uint64_t b = bad[0];
#pragma unroll
                for (int n = 1; n < NR; n++) b = i >= 64 * n ? bad[n] : b;
                x |= (uint32_t)(b >> (i & 63) & 1) << g;
            }
        return x;
    }
};

// Direct loads of a tile of ROWS keys by wave w of NW, as TileLoad's; a load's rows (4 or 8 aligned ones) are of one page.
template <int D, int ROWS, int NW> struct PageLoad {
    static constexpr int N = ROWS * 2 * D / 1024 / NW, RPL = 512 / D;  // loads per wave, rows per load
    static constexpr int VAR = RPL * NW >= 16 ? 1 : 16 / (RPL * NW);
    unsigned off[VAR];
    int64_t sp, st;
    int w, lane;
    __device__ __forceinline__ PageLoad(int64_t page_stride, int64_t stride, int wave, int l) : sp(page_stride), st(stride), w(wave), lane(l) {
#pragma unroll
        for (int i = 0; i < VAR; i++) off[i] = (unsigned)(lane / Tile<D>::CH) * (unsigned)(2 * st) + 16 * chunk(i);
    }
    __device__ __forceinline__ int row(int i) const { return RPL * (NW * i + w) + lane / Tile<D>::CH; }
    __device__ __forceinline__ int chunk(int i) const { return Tile<D>::pos(row(i), lane % Tile<D>::CH); }
    // keys j0 .. (a multiple of 32), `last` the sequence's last (>= j0), which stands for those behind it
    template <typename T, int NR> __device__ __forceinline__ void issue(const T* base, const Window<NR>& win, int j0, int last, unsigned lds) const {
        const int in = (1 << win.shift) - 1;
        if (last - j0 >= ROWS - 1) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int j = j0 + RPL * (NW * i + w);
                dma16s(base + win.page(j) * sp + (j & in) * st, off[i % VAR], lds + 1024u * (NW * i + w));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int j = min(j0 + RPL * (NW * i + w), last), jl = min(j0 + row(i), last);
                dma16(base + win.page(j) * sp + (jl & in) * st + 8 * chunk(i), lds + 1024u * (NW * i + w));
            }
        }
    }
};

// One query's softmax over keys [lo, hi) from its visible pairs alone (slot_attn.h's exact_row, the rows found through the table)
template <typename T, int D, bool CAP, bool BIAS>
__device__ __forceinline__ void exact_paged(const PagedArgs& a, const T* q, const T* kb, const T* vb, const int32_t* tab, const Sees& v, float slope, int p,
                                            int lo, int hi, int lane, float& m, float& l, float (&o)[D / 64]) {
    constexpr int N = D / 64;
    const int in = (1 << a.shift) - 1;
    m = -INFINITY;
    l = 0.f;
    for (int i = 0; i < N; i++) o[i] = 0.f;
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        int id = -1;
        if (j < hi && sees1(v, j, nullptr, 0)) id = tab[j >> a.shift];
        const bool ok = (unsigned)id < (unsigned)a.P;
        uint64_t b = __ballot(ok);
        if (!b) continue;
        const int64_t row = ok ? id : 0;
        float x = -INFINITY, tang;
        if (ok) x = score1<CAP, BIAS>(dot_row<T, D>(q, kb + row * a.k_sp + (j & in) * a.k_st), a.s, slope, p - j, tang);
        float mx = x;
        for (int i = 1; i < 64; i <<= 1) mx = fmaxf(mx, __shfl_xor(mx, i));
        const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn, f = m == -INFINITY ? 0.f : exp2_(m - mn);
        const float e = ok ? exp2_(x - mu) : 0.f;
        m = mn;
        l = l * f + wavesum(e);
        for (int i = 0; i < N; i++) o[i] *= f;
        if (l != l) {                                 // its own query, or an overflow
            for (int i = 0; i < N; i++) o[i] = NAN;
            return;
        }
        for (; b; b &= b - 1) {
            const int k = __builtin_ctzll(b);
            const T* z = vb + lane_of(id, k) * a.v_sp + ((j0 + k) & in) * a.v_st + lane * N;
            const float y = lane_of(e, k);
            for (int i = 0; i < N; i++) o[i] = fmaf(y, widen1(z[i]), o[i]);
        }
    }
}

// ------------------------------------------------------------------------------------------- plan
// One workgroup: the rows' tiles of MQ query rows in a row (units), then their key tiles.  Latency: two running sums.
__device__ __forceinline__ int before_sum(int x, int* s, int& all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int v = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(v, d);
        if (lane >= d) v += y;
    }
    __syncthreads();
    if (lane == 63) s[w] = v;
    __syncthreads();
    int base = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < LT / 64; i++) {
        if (i == w) base = sum;
        sum += s[i];
    }
    all = sum;
    return base + v - x;
}

__global__ __launch_bounds__(LT) void pages_plan(PagedArgs a) {
    __shared__ int s_sum[LT / 64];
    int* cost_r = a.plan;                             // running costs in front of each row
    int* first = a.plan + a.R + 1;
    int* cost = first + a.R + 1;
    const int tid = threadIdx.x;
    int u0 = 0, all;
    for (int r0 = 0; r0 < a.R; r0 += LT) {
        const int r = r0 + tid;
        int tiles = 0;
        if (r < a.R) {
            const Seq x = seq_of(a, r);
            tiles = (x.n * a.rep + MQ - 1) / MQ;
        }
        const int u = min(u0 + before_sum(tiles, s_sum, all), a.units);
        if (r < a.R) first[r] = u;
        u0 = min(u0 + all, a.units);
    }
    if (tid == 0) first[a.R] = u0;
    __syncthreads();
    int c0 = 0;
    for (int i0 = 0; i0 < u0; i0 += LT) {
        const int i = i0 + tid;
        int c = 0, lo = 0, hi = a.R;
        if (i < u0) {
            while (hi - lo > 1) {                     // the last row whose first unit is at or before i
                const int mid = (lo + hi) >> 1;
                if (first[mid] <= i) lo = mid; else hi = mid;
            }
            const Seq x = seq_of(a, lo);
            const int t = i - first[lo], off = x.end - x.n, last = min(MQ * (t + 1), x.n * a.rep) - 1;
            int k0, k1;
            keys_of<KT>(a, x, MQ * t / a.rep + off, last / a.rep + off, k0, k1);
            c = max(1, (k1 - k0 + KT - 1) / KT);
        }
        const int at = c0 + before_sum(c, s_sum, all);
        if (i < u0) {
            cost[i] = at;
            if (i == first[lo]) cost_r[lo] = at;
        }
        c0 += all;
    }
    if (tid == 0) cost[u0] = c0;
    __syncthreads();
    // rows without units stand where the next row stands
    for (int r = tid; r <= a.R; r += LT)
        if (r == a.R || first[r] == first[r + 1]) cost_r[r] = cost[first[r]];
}

// the last i of [lo, hi) with mul x[i] <= y (x ascending, x[lo] does), by all lanes
__device__ __forceinline__ int find(const int* x, int lo, int hi, int64_t mul, int64_t y, int lane) {
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, i = lo + lane * step;
        const uint64_t b = __ballot(i < hi && mul * x[min(i, hi - 1)] <= y);
        const int k = 63 - __builtin_clzll(b | 1);
        lo += k * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// ------------------------------------------------------------------------------------------- many rows
template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(MT, 2) void pages_many(PagedArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = KT * 2 * D;
    typedef PageLoad<D, KT, MW> Load;
    __shared__ __align__(1024) unsigned char smem[2][2][STAGE];      // [buffer][keys, values]
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    // tokens of no row
    {
        const int s0 = min(max(uni(a.starts[0]), 0), a.N), s1 = min(max(uni(a.starts[a.R]), s0), a.N);
        const int64_t row = (int64_t)a.Hq * D / 8, n0 = s0 * row, n1 = n0 + (a.N - s1) * row;
        for (int64_t i = (int64_t)blockIdx.x * MT + tid; i < n1; i += (int64_t)gridDim.x * MT)
            reinterpret_cast<uint4*>(a.out)[i < n0 ? i : i - n0 + s1 * row] = make_uint4(0, 0, 0, 0);
    }
    const int* cost_r = a.plan;
    const int* first = a.plan + a.R + 1;
    const int* cost = first + a.R + 1;
    const int64_t total = (int64_t)uni(cost_r[a.R]) * a.Hk;
    // workers that follow each other run on one XCD (workgroup i on XCD i % 8): they share keys
    const int G = (int)min((int64_t)gridDim.x, max((total + 3) / 4, (int64_t)1));
    int me = blockIdx.x;
    if (me >= G) {
        if (tid == 0 && me < (int)gridDim.x) a.join[me].parts = 0;
        return;
    }
    if (G % 8 == 0) me = (me & 7) * (G / 8) + (me >> 3);
    int64_t x = total * me / G;
    const int64_t end = total * (me + 1) / G;
    Unit left{0, 0, 0, 0, 0};
    int r = uni(find(cost_r, 0, a.R, a.Hk, x, lane));
    while (r + 1 < a.R && (int64_t)uni(cost_r[r + 1]) * a.Hk <= x) r++;      // (rows without tokens)
    const unsigned lds = lds_addr(smem);
    const Load lk(a.k_sp, a.k_st, w, lane), lv(a.v_sp, a.v_st, w, lane);
    const Ops<D> ops(lane);
    const float f2 = fabsf(a.s.f);
    RowSums<T, D, BIAS> sum(f2);
    while (x < end) {
        // the unit of x, and this worker's key tiles [ka, kb) of its c
        const int cr = uni(cost_r[r]), per = uni(cost_r[r + 1]) - cr;
        const int64_t y = x - (int64_t)cr * a.Hk;
        if (per == 0 || y >= (int64_t)per * a.Hk) { r++; continue; }
        const int hk = uni((int)(y / per)), z = uni((int)(y - (int64_t)hk * per) + cr);
        const int u0 = uni(first[r]), u = uni(find(cost, u0, uni(first[r + 1]), 1, z, lane));
        const int cu = uni(cost[u]), c = uni(cost[u + 1]) - cu, ka = z - cu, kb = (int)min((int64_t)c, ka + end - x);
        const int t = u - u0;
        Seq sq = seq_of(a, r);
        sq = {uni(sq.s), uni(sq.n), uni(sq.end), uni(sq.klen), uni(sq.pre)};
        const int rows = sq.n * a.rep, off = sq.end - sq.n, row0 = MQ * t + 32 * w, row = min(row0 + (lane & 31), rows - 1);
        const int tok = row / a.rep, hq = hk * a.rep + row - tok * a.rep, p = tok + off;
        const Mask mk{1, a.W, sq.pre, sq.klen};
        const Span sw{MQ * t / a.rep + off, (min(MQ * (t + 1), rows) - 1) / a.rep + off, 0, 0, true};
        const bool mine = row0 < rows;
        const Span sv{uni(row0 / a.rep + off), uni((min(row0 + 32, rows) - 1) / a.rep + off), 0, 0, true};
        int lo, hi;
        keys_of<KT>(a, sq, sw.p0, sw.p1, lo, hi);
        const int j_end = min(hi, lo + kb * KT);
        const T* kbase = (const T*)a.k + hk * a.k_sh;
        const T* vbase = (const T*)a.v + hk * a.v_sh;
        Window<1> win(a, r, sq.klen, lane);
        auto seen = [&](int j) {                      // the next tile that any of the workgroup's rows sees
            while (j < j_end && !mk.some(sw, j, j + KT - 1)) j += KT;
            return j;
        };
        auto load = [&](int j, int buf) {
            lk.issue(kbase, win, j, sq.klen - 1, lds + (2 * buf) * STAGE);
            lv.issue(vbase, win, j, sq.klen - 1, lds + (2 * buf + 1) * STAGE);
        };
        const T* qrow = (const T*)a.q + hq * a.q_sh + (int64_t)(sq.s + tok) * a.q_st;
        uint4 qf[KK];
#pragma unroll
        for (int kk = 0; kk < KK; kk++) qf[kk] = ld16(qrow + 8 * h + 16 * kk);
        if (a.s.f < 0.f)                              // a negative scale: of the queries' sign, so that larger products are larger scores
#pragma unroll
            for (int kk = 0; kk < KK; kk++) { qf[kk].x ^= 0x80008000u; qf[kk].y ^= 0x80008000u; qf[kk].z ^= 0x80008000u; qf[kk].w ^= 0x80008000u; }
        const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
        const Sees see = Sees::query(mk, p);
        sum.clear();
        int j0 = seen(lo + ka * KT);
        __syncthreads();                              // the last unit's tiles are read
        if (j0 < j_end) {
            win.at(j0, KT);
            load(j0, 0);
        }
        // one barrier a tile: behind it the tile is there for every wave and the other buffer is read, so the next one's loads
        // run during this one's products
        for (int buf = 0; j0 < j_end; buf ^= 1) {
            const int j1 = seen(j0 + KT);
            const uint32_t lost = win.lost(j0, KT);
            if (j1 < j_end) win.at(j1, KT);
            wait_vm<0>();
            tile_barrier();
            if (j1 < j_end) load(j1, buf ^ 1);
            if (mine && mk.some(sv, j0, j0 + KT - 1)) {
                const unsigned bo = lds + (2 * buf) * STAGE, rk = bo + ops.row, cc = bo + ops.col, c8 = bo + ops.col8;
                // operands are read three steps (six products) ahead: an LDS read takes as long as four or five products
                f32x16 s[2] = {zero16(), zero16()};
                uint4 kr[4][2];
                auto rowop = [&](int kk) {
                    const unsigned q = Ops<D>::k_step(rk, kk);
                    kr[kk & 3][0] = lds16(q);
                    kr[kk & 3][1] = lds16(q + 32 * Tile<D>::ROWB);
                };
                rowop(0);
                rowop(1);
                rowop(2);
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    if (kk + 3 < KK) rowop(kk + 3);
                    s[0] = mfma32<T>(kr[kk & 3][0], qf[kk], s[0]);
                    s[1] = mfma32<T>(kr[kk & 3][1], qf[kk], s[1]);
                    __builtin_amdgcn_sched_barrier(0);
                }
                uint4 vr[5];                          // operand i: column block i % DT of 16 keys i / DT
                auto colop = [&](int i) {
                    vr[i % 5] = Ops<D>::at_col(Ops<D>::block(cc, i % DT), Ops<D>::block(c8, i % DT), STAGE + 16 * (i / DT) * Tile<D>::ROWB);
                };
                colop(0);
                colop(1);
                colop(2);
                colop(3);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    scores<CAP>(s[i], a.s);
                    if constexpr (BIAS) bias(s[i], f2, slope, p, j0 + 32 * i, h);
                }
                if (lost || !mk.all(sv, j0, j0 + KT - 1)) {
#pragma unroll
                    for (int i = 0; i < 2; i++) {
                        uint32_t ok = seen16(see, j0 + 32 * i, h, j0 < mk.prefix, nullptr, 0);
                        if (bit(lost, 2 * i)) ok &= ~0xffu;           // registers 0 .. 7 are keys of the first 16
                        if (bit(lost, 2 * i + 1)) ok &= 0xffu;
#pragma unroll
                        for (int e = 0; e < 16; e++) s[i][e] = bit(ok, e) ? s[i][e] : -INFINITY;
                    }
                }
                uint4 pf[2][2];
                sum.template weigh<2>(s, pf);
#pragma unroll
                for (int i = 0; i < 4 * DT; i++) {
                    sum.o[i % DT] = mfma32<T>(vr[i % 5], pf[i / DT >> 1][i / DT & 1], sum.o[i % DT]);
                    if (i + 4 < 4 * DT) colop(i + 4);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            j0 = j1;
        }
        sum.close();
        const bool whole = ka == 0 && kb == c, in = row0 + (lane & 31) < rows;
        const int64_t at = ((int64_t)(sq.s + tok) * a.Hq + hq) * D;
        const int64_t part = ((int64_t)(2 * me + (ka == 0)) * MW + w) * 32;   // a piece's rows
        float nf = sum.l * 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) nf = nonfinite(sum.o[dt], nf);
        // rows next to infinities and NaN, from their visible pairs alone
        const uint32_t odd = row_bits(nf != 0.f && sum.l == sum.l && in);
        for (uint32_t b = odd; b; b &= b - 1) {
            const int i = __builtin_ctz(b);
            float m1, l1, o1[D / 64];
            exact_paged<T, D, CAP, BIAS>(a, (const T*)a.q + lane_of(hq, i) * a.q_sh + (int64_t)(sq.s + lane_of(tok, i)) * a.q_st, kbase, vbase, win.tab,
                                         lane_of(see, i), lane_of(slope, i), lane_of(p, i), lo + ka * KT, j_end, lane, m1, l1, o1);
            if (whole) {
                const float inv1 = l1 > 0.f || l1 != l1 ? 1.f / l1 : 0.f;
                for (int e = 0; e < D / 64; e++) o1[e] *= inv1;
                put_row<T, D>((T*)a.out + ((int64_t)(sq.s + lane_of(tok, i)) * a.Hq + lane_of(hq, i)) * D, lane, o1);
            } else {
                for (int e = 0; e < D / 64; e++) a.po[(part + i) * D + lane * (D / 64) + e] = o1[e];
                if (lane == 0) a.pm[part + i] = make_float2(m1, l1);
            }
        }
        if (in && !bit(odd, lane & 31)) {
            if (whole) {
                const float inv = sum.l > 0.f || sum.l != sum.l ? 1.f / sum.l : 0.f;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        put4<T>(a.out, nullptr, at + 32 * dt + 8 * g + 4 * h, sum.o[dt][4 * g] * inv, sum.o[dt][4 * g + 1] * inv, sum.o[dt][4 * g + 2] * inv,
                                sum.o[dt][4 * g + 3] * inv);
            } else {
                float* po = a.po + (part + (lane & 31)) * D + 4 * h;
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
#pragma unroll
                    for (int g = 0; g < 4; g++)
                        *reinterpret_cast<float4*>(po + 32 * dt + 8 * g) =
                            make_float4(sum.o[dt][4 * g], sum.o[dt][4 * g + 1], sum.o[dt][4 * g + 2], sum.o[dt][4 * g + 3]);
                if (h == 0) a.pm[part + lane] = make_float2(sum.m, sum.l);
            }
        }
        if (ka == 0 && kb < c) {                      // its other pieces are those of the workers up to the one of its last tile
            const int64_t last = x + c - 1;
            left = {r, hk, t, sq.n, (int)(((last + 1) * G - 1) / total) - me + 1};
        }
        x += kb - ka;
    }
    if (tid == 0) a.join[me] = left;
}

// ------------------------------------------------------------------------------------------- few rows
// One 32-row tile of a key/value head (a generated token's query heads, a few tokens') against 32-key tiles, each wave through a ring of its own of
// two tiles without a barrier in the loop.  NW = 1, STREAM: every wave is a worker with an equal share of all units' tiles.  Otherwise a
// workgroup's NW waves share one unit, every NW-th tile each, and meet in LDS.
__device__ __forceinline__ int scan_up(int x, int lane) {            // sum over the lanes up to this one
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x += y;
    }
    return x;
}
// 32-row tiles of row r, and 32-key tiles of each (of its whole row, so that no table of them is needed)
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

template <typename T, int D, bool CAP, bool BIAS, int NW, bool STREAM>
__global__ __launch_bounds__(64 * NW) void pages_few(PagedArgs a) {
    constexpr int KK = D / 16, DT = D / 32, ST = 32 * 2 * D;
    typedef PageLoad<D, 32, 1> Load;
    __shared__ __align__(1024) unsigned char smem[NW][2][2][ST];     // [wave][buffer][keys, values]
    __shared__ float s_m[NW][32], s_l[NW][32];                       // the waves' maxima and sums of every row
    __shared__ float s_M[32], s_L[32];                               // the workgroup's
    __shared__ uint32_t s_bad[NW];
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
    int r = 0, base = 0, me = 0, G = 1;               // base: tiles of one head in front of row r
    int64_t x = 0, end = 1, total = 1;
    Unit left{0, 0, 0, 0, 0};
    if constexpr (STREAM) {
        const int C = (a.R + 63) / 64;
        int mine = 0;
        for (int i = 0; i < C; i++) mine += few_cost(a, lane * C + i);
        const int upto = scan_up(mine, lane);
        total = (int64_t)lane_of(upto, 63) * a.Hk;
        G = (int)min((int64_t)gridDim.x, max(total / FS, (int64_t)1));
        me = blockIdx.x;
        if (me < G) {
            if (G % 8 == 0) me = (me & 7) * (G / 8) + (me >> 3);     // workers that follow each other run on one XCD
            x = total * me / G;
            end = total * (me + 1) / G;
            const int y = (int)(x / a.Hk), L = 63 - __builtin_clzll(__ballot(upto - mine <= y) | 1);
            base = lane_of(upto - mine, L);
            r = L * C;
            for (int i0 = 0; C > 1 && i0 < C; i0 += 64) {            // the row within the lane's rows
                const int c = i0 + lane < C ? few_cost(a, r + i0 + lane) : 0, u = scan_up(c, lane), all = lane_of(u, 63);
                if (base + all <= y) { base += all; continue; }
                const int k = 63 - __builtin_clzll(__ballot(base + u - c <= y) | 1);
                base += lane_of(u - c, k);
                r += i0 + k;
                break;
            }
        } else {
            x = end;
        }
    }
    const unsigned lds = lds_addr(smem[w]);
    const Load lk(a.k_sp, a.k_st, 0, lane), lv(a.v_sp, a.v_st, 0, lane);
    const Ops<D> ops(lane);
    const float f2 = fabsf(a.s.f);
    RowSums<T, D, BIAS> sum(f2);
    int t = STREAM ? 0 : blockIdx.x, hk = STREAM ? 0 : blockIdx.y;
    if constexpr (!STREAM) r = blockIdx.z;
    while (x < end) {
        Seq sq = seq_of(a, r);
        sq = {uni(sq.s), uni(sq.n), uni(sq.end), uni(sq.klen), uni(sq.pre)};
        const int rows = sq.n * a.rep, off = sq.end - sq.n;
        int per, ka = 0, kb, lo, hi;
        const int tiles = few_tiles(a, sq, per);
        if constexpr (STREAM) {
            const int64_t y = x - (int64_t)base * a.Hk;
            const int cost = tiles * per;
            if (y >= (int64_t)cost * a.Hk) {          // the next row
                if (++r >= a.R) break;
                base += cost;
                continue;
            }
            hk = (int)(y / cost);
            const int z = (int)(y - (int64_t)hk * cost);
            t = z / per;
            ka = z - t * per;
            kb = (int)min((int64_t)per, ka + end - x);
        } else {
            if (t >= tiles) break;
            kb = per;
        }
        keys_of<32>(a, sq, off, sq.end - 1, lo, hi);
        const int r0 = 32 * t, row = min(r0 + (lane & 31), rows - 1);
        const int tok = row / a.rep, hq = hk * a.rep + row - tok * a.rep, p = tok + off;
        const Mask mk{1, a.W, sq.pre, sq.klen};
        const Span s{r0 / a.rep + off, (min(r0 + 32, rows) - 1) / a.rep + off, 0, 0, true};
        const int first = lo + 32 * ka;
        hi = min(hi, lo + 32 * kb);
        const T* kbase = (const T*)a.k + hk * a.k_sh;
        const T* vbase = (const T*)a.v + hk * a.v_sh;
        Window<2> win(a, r, sq.klen, lane);
        auto seen = [&](int j) {                      // the next of this wave's tiles that any row sees
            while (j < hi && !mk.some(s, j, j + 31)) j += 32 * NW;
            return j;
        };
        auto keys = [&](int j, int buf) { lk.issue(kbase, win, j, sq.klen - 1, lds + (2 * buf) * ST); };
        auto values = [&](int j, int buf) { lv.issue(vbase, win, j, sq.klen - 1, lds + (2 * buf + 1) * ST); };
        // a tile's groups of 16 keys in no page; the window stands at the tile that is loaded last
        auto look = [&](int j) -> uint32_t {
            win.at(j, 32);
            return win.lost(j, 32);
        };
        uint32_t lost0 = 0, lost1 = 0, lost2 = 0;
        int j0 = seen(first + 32 * w);
        if (j0 < hi) {
            lost0 = look(j0);
            keys(j0, 0);
            values(j0, 0);
        }
        const float slope = BIAS ? a.slopes[hq] * LOG2E : 0.f;
        const T* qrow = (const T*)a.q + hq * a.q_sh + (int64_t)(sq.s + tok) * a.q_st;
        uint4 qf[KK];
#pragma unroll
        for (int kk = 0; kk < KK; kk++) qf[kk] = ld16(qrow + 8 * h + 16 * kk);
        if (a.s.f < 0.f)                              // a negative scale: of the queries' sign, so that larger products are larger scores
#pragma unroll
            for (int kk = 0; kk < KK; kk++) { qf[kk].x ^= 0x80008000u; qf[kk].y ^= 0x80008000u; qf[kk].z ^= 0x80008000u; qf[kk].w ^= 0x80008000u; }
        const Sees see = Sees::query(mk, p);
        sum.clear();
        // Keys and values are fetched two tiles ahead, each into the place that it has just been read from.
        int j1 = j0 < hi ? seen(j0 + 32 * NW) : hi;
        if (j1 < hi) {
            lost1 = look(j1);
            keys(j1, 1);
            values(j1, 1);
        }
        for (int buf = 0; j0 < hi; buf ^= 1) {
            const int j2 = j1 < hi ? seen(j1 + 32 * NW) : hi;
            if (j2 < hi) lost2 = look(j2);
            if (j1 < hi) wait_vm<3 * Load::N>();      // behind this tile's keys: its values, the next keys and values
            else wait_vm<Load::N>();
            asm volatile("" ::: "memory");
            const unsigned bo = lds + (2 * buf) * ST, rk = bo + ops.row, c = bo + ops.col, c8 = bo + ops.col8;
            f32x16 sc[1] = {zero16()};
#pragma unroll
            for (int kk = 0; kk < KK; kk++) sc[0] = mfma32<T>(lds16(Ops<D>::k_step(rk, kk)), qf[kk], sc[0]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the keys are read before their place is filled again
            if (j2 < hi) keys(j2, buf);
            scores<CAP>(sc[0], a.s);
            if constexpr (BIAS) bias(sc[0], f2, slope, p, j0, h);
            if (lost0 || j0 + 32 > hi || !mk.all(s, j0, j0 + 31)) {
                uint32_t ok = seen16(see, j0, h, j0 < mk.prefix, nullptr, 0);
                if (bit(lost0, 0)) ok &= ~0xffu;      // registers 0 .. 7 are keys of the first 16
                if (bit(lost0, 1)) ok &= 0xffu;
#pragma unroll
                for (int e = 0; e < 16; e++) sc[0][e] = j0 + key_of(e, h) < hi && bit(ok, e) ? sc[0][e] : -INFINITY;
            }
            uint4 pf[1][2];
            sum.template weigh<1>(sc, pf);
            if (j2 < hi) wait_vm<3 * Load::N>();      // behind the values: the next tile, the keys after it
            else if (j1 < hi) wait_vm<2 * Load::N>();
            else wait_vm<0>();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int mm = 0; mm < 2; mm++)
                    sum.o[dt] = mfma32<T>(Ops<D>::at_col(Ops<D>::block(c, dt), Ops<D>::block(c8, dt), ST + 16 * mm * Tile<D>::ROWB), pf[0][mm], sum.o[dt]);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the values, too
            if (j2 < hi) values(j2, buf);
            j0 = j1;
            j1 = j2;
            lost0 = lost1;
            lost1 = lost2;
        }
        sum.close();
        // the waves' parts: (m, l) of every row to all, then the weighted sums through LDS (its tiles are read)
        if (h == 0) { s_m[w][lane] = sum.m; s_l[w][lane] = sum.l; }
        __syncthreads();
        float M = -INFINITY, Ls = 0.f;
#pragma unroll
        for (int i = 0; i < NW; i++) M = fmaxf(M, s_m[i][lane & 31]);
        const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < NW; i++) Ls += s_l[i][lane & 31] * exp2_(s_m[i][lane & 31] - Mu);
        const float f = exp2_(sum.m - Mu);
        float* so = reinterpret_cast<float*>(smem);   // [wave][row][D + 4]
        constexpr int SO = D + 4;
        static_assert(NW * 32 * SO * 4 <= (int)sizeof(smem), "the waves' sums fit");
        const int used = min(32, rows - r0);
        if ((lane & 31) < used) {
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
#pragma unroll
                for (int g = 0; g < 4; g++)
                    *reinterpret_cast<float4*>(so + (w * 32 + (lane & 31)) * SO + 32 * dt + 8 * g + 4 * h) =
                        make_float4(sum.o[dt][4 * g] * f, sum.o[dt][4 * g + 1] * f, sum.o[dt][4 * g + 2] * f, sum.o[dt][4 * g + 3] * f);
        }
        if (w == 0 && h == 0) { s_M[lane] = M; s_L[lane] = Ls; }      // not over s_m and s_l, which the other waves may still read
        float nf = sum.l * 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) nf = nonfinite(sum.o[dt], nf);
        const uint32_t odd = row_bits(nf != 0.f && (lane & 31) < used);
        if (lane == 0) s_bad[w] = odd;
        __syncthreads();
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < NW; i++) bad |= s_bad[i];
        if (bad) {                                    // rows next to infinities and NaN, from their visible pairs alone; the same in every wave
            bad &= ~row_bits(Ls != Ls);
            for (; bad; bad &= bad - 1) {
                const int i = __builtin_ctz(bad);
                if (i % NW != w) continue;
                float m1, l1, o1[D / 64];
                exact_paged<T, D, CAP, BIAS>(a, (const T*)a.q + lane_of(hq, i) * a.q_sh + (int64_t)(sq.s + lane_of(tok, i)) * a.q_st, kbase, vbase,
                                             win.tab, lane_of(see, i), lane_of(slope, i), lane_of(p, i), first, hi, lane, m1, l1, o1);
                for (int ww = 0; ww < NW; ww++)
                    for (int e = 0; e < D / 64; e++) so[(ww * 32 + i) * SO + lane * (D / 64) + e] = ww ? 0.f : o1[e];
                if (lane == 0) { s_M[i] = m1; s_L[i] = l1; }
            }
            __syncthreads();
        }
        const bool whole = ka == 0 && kb == per;
        const int64_t part = (int64_t)(2 * me + (ka == 0)) * 32;      // a piece's rows
        // used rows x D values: 8 lanes a row
        for (int rr = tid >> 3; rr < used; rr += 8 * NW) {
            const int c8 = tid & 7, g = r0 + rr;
            const float lr = s_L[rr], inv = lr > 0.f || lr != lr ? 1.f / lr : 0.f;
            const int gt = g / a.rep, gh = hk * a.rep + g - gt * a.rep;
            const int64_t at = ((int64_t)(sq.s + gt) * a.Hq + gh) * D;
#pragma unroll
            for (int i = 0; i < D / 32; i++) {
                const int d = 4 * c8 + 32 * i;
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int ww = 0; ww < NW; ww++) {
                    const float4 y = *reinterpret_cast<const float4*>(so + (ww * 32 + rr) * SO + d);
                    v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
                }
                if (whole) put4<T>(a.out, nullptr, at + d, v.x * inv, v.y * inv, v.z * inv, v.w * inv);
                else *reinterpret_cast<float4*>(a.po + (part + rr) * D + d) = v;
            }
            if (!whole && c8 == 0) a.pm[part + rr] = make_float2(s_M[rr], lr);
        }
        if constexpr (STREAM) {
            if (ka == 0 && kb < per) left = {r, hk, t, sq.n, (int)(((x + per) * G - 1) / total) - me + 1};
            x += kb - ka;
        } else {
            t += gridDim.x;
        }
        __syncthreads();                              // the sums are read before the next unit's tiles take their place
    }
    // tokens of no row, by workers that are through
    {
        const int s0 = min(max(uni(a.starts[0]), 0), a.N), s1 = min(max(uni(a.starts[a.R]), s0), a.N);
        const int64_t n = (int64_t)a.Hq * D / 8, n0 = s0 * n, n1 = n0 + (a.N - s1) * n, all = (int64_t)gridDim.x * gridDim.y * gridDim.z * 64 * NW;
        for (int64_t i = ((int64_t)(blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * 64 * NW + tid; i < n1; i += all)
            reinterpret_cast<uint4*>(a.out)[i < n0 ? i : i - n0 + s1 * n] = make_uint4(0, 0, 0, 0);
    }
    if constexpr (STREAM) {
        if (tid == 0) a.join[me] = left;
    }
}

// ------------------------------------------------------------------------------------------- join
// out = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s over a unit's pieces.  A row is D / 4 lanes times NG groups, which take every NG-th piece: a
// row of hundreds of pieces is as many short chains of loads.  Their sums meet in LDS in order.
template <typename T, int D, int ROWS, int NG>
__global__ __launch_bounds__(256) void pages_join(PagedArgs a) {
    constexpr int LN = D / 4, RW = 256 / (LN * NG);
    static_assert(RW >= 1, "whole rows");
    __shared__ __align__(16) float s_o[NG > 1 ? NG : 1][D];
    __shared__ float s_l[NG];
    const int me = blockIdx.x;
    const Unit u = a.join[me];
    if (u.parts < 2) return;
    const int c = threadIdx.x % LN, g = NG == 1 ? 0 : threadIdx.x / LN;
    for (int i = blockIdx.y * RW + (NG == 1 ? threadIdx.x / LN : 0); i < ROWS; i += gridDim.y * RW) {
        const int row = ROWS * u.t + i;
        if (row >= u.n * a.rep) return;               // (with several groups: all threads alike)
        auto slot = [&](int s) { return (int64_t)(s ? 2 * (me + s) : 2 * me + 1) * ROWS + i; };
        float M = -INFINITY, L = 0.f;
        if constexpr (NG == 1) {
            for (int s = 0; s < u.parts; s++) M = fmaxf(M, a.pm[slot(s)].x);
        } else {
            for (int s = threadIdx.x & 63; s < u.parts; s += 64) M = fmaxf(M, a.pm[slot(s)].x);
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) M = fmaxf(M, __shfl_xor(M, d));
        }
        const float Mu = M == -INFINITY ? 0.f : M;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
        for (int s = g; s < u.parts; s += NG) {
            const float2 x = a.pm[slot(s)];
            const float f = x.y != 0.f ? exp2_(x.x - Mu) : 0.f;       // otherwise nothing is visible in this piece
            const float4 o = *reinterpret_cast<const float4*>(a.po + slot(s) * D + 4 * c);
            L = fmaf(x.y, f, L);
            acc.x = fmaf(o.x, f, acc.x);
            acc.y = fmaf(o.y, f, acc.y);
            acc.z = fmaf(o.z, f, acc.z);
            acc.w = fmaf(o.w, f, acc.w);
        }
        if constexpr (NG > 1) {
            __syncthreads();                          // the last row's sums are read
            *reinterpret_cast<float4*>(&s_o[g][4 * c]) = acc;
            if (c == 0) s_l[g] = L;
            __syncthreads();
            if (g) continue;
            acc = make_float4(0.f, 0.f, 0.f, 0.f);
            L = 0.f;
#pragma unroll
            for (int k = 0; k < NG; k++) {
                const float4 o = *reinterpret_cast<const float4*>(&s_o[k][4 * c]);
                L += s_l[k];
                acc.x += o.x;
                acc.y += o.y;
                acc.z += o.z;
                acc.w += o.w;
            }
        }
        const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
        const int tok = row / a.rep, hq = u.hk * a.rep + row - tok * a.rep;
        const int s = min(max(a.starts[u.r], 0), a.N);
        put4<T>(a.out, nullptr, ((int64_t)(s + tok) * a.Hq + hq) * D + 4 * c, acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
    }
}

// How a call runs.
//   MANY    tiles of 128 query rows
//   SHARED  one tile of 32 rows a key/value head (one or a few tokens of each sequence): equal shares of all keys, and a join
//   SINGLE  the same where no row has many keys: a workgroup a unit, no join
enum { MANY, SHARED, SINGLE };
struct Plan { int kind, G; int64_t units; size_t join, pm, po, all; };
Plan plan(int64_t N, int64_t R, int64_t M, int64_t page, int64_t Hq, int64_t Hk, int64_t D, int64_t most, int64_t W, bool prefix) {
    Plan x{};
    const int64_t rep = Hq / Hk, rows = std::min(N, R);
    const int64_t keys = prefix ? M * page : std::min(M * page, W + most + 32);
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    x.kind = most * rep > 32 ? MANY : keys <= UNIT_KEYS ? SINGLE : SHARED;
    if (x.kind == SINGLE && (R > 65535 || Hk > 65535)) x.kind = SHARED;
    if (x.kind == SHARED && (N * rep / 32 + rows) * Hk * ((M * page + 31) / 32) > 0x3fffffffLL) x.kind = MANY;      // (its sums are 32-bit ones)
    const int64_t Q = x.kind == MANY ? MQ : 32, K = x.kind == MANY ? KT : 32;
    x.units = N * rep / Q + rows;
    if (x.kind == SINGLE) return x;
    const int64_t tiles = x.units * Hk * ((M * page + K - 1) / K);
    x.G = x.kind == MANY ? (int)std::min<int64_t>(MG, (tiles + 3) / 4) : (int)std::min<int64_t>(FG, std::max<int64_t>(tiles / FS, 1));
    x.join = x.kind == MANY ? up((size_t)(2 * (R + 1) + x.units + 1) * 4) : 0;
    x.pm = x.join + up((size_t)x.G * sizeof(Unit));
    x.po = x.pm + up((size_t)x.G * 2 * Q * sizeof(float2));
    x.all = x.po + up((size_t)x.G * 2 * Q * D * sizeof(float));
    return x;
}

template <typename T, int D, bool CAP, bool BIAS>
void launch_one(const PagedArgs& a, const Plan& x, int tiles, hipStream_t st) {
    if (x.kind == MANY) slothost::launch(pages_many<T, D, CAP, BIAS>, dim3((unsigned)x.G), dim3(MT), 0, st, a);
    else if (x.kind == SHARED) slothost::launch(pages_few<T, D, CAP, BIAS, 1, true>, dim3((unsigned)x.G), dim3(64), 0, st, a);
    else slothost::launch(pages_few<T, D, CAP, BIAS, FW, false>, dim3((unsigned)tiles, (unsigned)a.Hk, (unsigned)a.R), dim3(64 * FW), 0, st, a);
}
template <typename T, int D>
void launch_attn(const PagedArgs& a, bool cap, const Plan& x, int tiles, hipStream_t st) {
    if (cap) a.slopes ? launch_one<T, D, true, true>(a, x, tiles, st) : launch_one<T, D, true, false>(a, x, tiles, st);
    else a.slopes ? launch_one<T, D, false, true>(a, x, tiles, st) : launch_one<T, D, false, false>(a, x, tiles, st);
}
template <typename T, int D>
void launch_join(const PagedArgs& a, const Plan& x, int rows, hipStream_t st) {
    if (x.kind == MANY) slothost::launch(pages_join<T, D, MQ, 1>, dim3((unsigned)x.G, (unsigned)(MQ * (D / 4) / 256)), dim3(256), 0, st, a);
    else slothost::launch(pages_join<T, D, 32, 1024 / D>, dim3((unsigned)x.G, (unsigned)std::min(rows, 8)), dim3(256), 0, st, a);
}

}  // namespace

// ======================================================================================== C-ABI
extern "C" size_t slotattn_pages_workspace(int64_t N, int64_t R, int64_t M, int64_t page, int64_t Hq, int64_t Hk, int64_t D, int64_t most,
                                           int64_t window, int has_prefix) {
    if (N < 1 || R < 1 || M < 1 || page < 1 || Hk < 1 || Hq < Hk || Hq % Hk || N > SLOTATTN_MAX_T || most < 1 || window < 1) return 0;
    return plan(N, R, M, page, Hq, Hk, D, std::min(most, N), window, has_prefix).all;
}

extern "C" int slotattn_pages(const void* q, int64_t q_sh, int64_t q_st, const void* k, int64_t k_sp, int64_t k_sh, int64_t k_st,
                              const void* v, int64_t v_sp, int64_t v_sh, int64_t v_st, int dtype, const int32_t* table, int64_t t_sr,
                              const int32_t* starts, const int32_t* ends, int64_t N, int64_t R, int64_t M, int64_t P, int64_t page,
                              int64_t Hq, int64_t Hk, int64_t D, int64_t most, float scale, int64_t window, float cap, const float* slopes,
                              const int32_t* prefix, void* workspace, void* out, void* stream) {
    if (N < 1 || R < 1 || M < 1 || P < 1) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_pages: N, R, M and P must be >= 1");
    if (page < SLOTPAGE_MIN || (page & (page - 1)) || page > SLOTPAGE_MAX) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_pages: page must be a power of two in [16, 4096]");
    if (M * page > SLOTATTN_MAX_T || P > SLOTATTN_MAX_T || R > 1 << 24 || t_sr < 0 || most < 1)
        return fail(SLOTSCAN_ERR_SHAPE, "slotattn_pages: shape too large");
    if (int r = slotattn_host::check(q, 0, q_sh, q_st, k, k_sp, k_sh, k_st, v, v_sp, v_sh, v_st, dtype, 1, N, page, Hq, Hk, D, scale, window, cap)) return r;
    if (!table || !starts || !ends || !out) return fail(SLOTSCAN_ERR_NULL, "slotattn_pages: a required pointer is NULL");
    if (!al16(out) || !al16(workspace)) return fail(SLOTSCAN_ERR_ALIGN, "slotattn_pages: out and workspace must be 16-byte aligned");
    const Plan x = plan(N, R, M, page, Hq, Hk, D, std::min(most, N), window, prefix != nullptr);
    if (x.all && !workspace) return fail(SLOTSCAN_ERR_NULL, "slotattn_pages: workspace is NULL");
    // running costs are 32-bit: tiles of all units of one head
    if (x.kind == MANY && (x.units + 1) * ((M * page + KT - 1) / KT) > 0x3fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_pages: shape too large");
    PagedArgs a{};
    a.s = slotattn_host::args(q, 0, q_sh, q_st, k, k_sp, k_sh, k_st, v, v_sp, v_sh, v_st, 1, N, page, Hq, Hk, scale, 1, window, cap, slopes, nullptr, prefix);
    a.q = q; a.k = k; a.v = v;
    a.q_sh = q_sh; a.q_st = q_st; a.k_sp = k_sp; a.k_sh = k_sh; a.k_st = k_st; a.v_sp = v_sp; a.v_sh = v_sh; a.v_st = v_st;
    a.table = table; a.t_sr = t_sr; a.starts = starts; a.ends = ends; a.prefix = prefix; a.slopes = slopes;
    a.N = (int)N; a.R = (int)R; a.M = (int)M; a.P = (int)P; a.Hq = (int)Hq; a.Hk = (int)Hk; a.rep = (int)(Hq / Hk);
    a.W = a.s.W; a.shift = __builtin_ctzll((unsigned long long)page); a.units = (int)x.units;
    char* ws = (char*)workspace;
    a.plan = (int*)ws; a.join = (Unit*)(ws + x.join); a.pm = (float2*)(ws + x.pm); a.po = (float*)(ws + x.po);
    a.out = out;
    hipStream_t st = (hipStream_t)stream;
    const bool cp = cap > 0.f;
    const int tiles = (int)((std::min(most, N) * a.rep + 31) / 32), rows = (int)std::min<int64_t>(32, std::min(most, N) * a.rep);
    hipError_t e;
    if (x.kind == MANY) {
        slothost::Scope sc(SLOTSCAN_K_ATTN_PLAN, st);
        slothost::launch(pages_plan, dim3(1), dim3(LT), 0, st, a);
        e = hipGetLastError();
        if (e != hipSuccess) return hip_fail(e, "pages_plan launch");
    }
    {
        slothost::Scope sc(SLOTSCAN_K_ATTN, st);
        if (dtype == SLOTSCAN_BF16) D == 128 ? launch_attn<bf16_t, 128>(a, cp, x, tiles, st) : launch_attn<bf16_t, 64>(a, cp, x, tiles, st);
        else D == 128 ? launch_attn<f16_t, 128>(a, cp, x, tiles, st) : launch_attn<f16_t, 64>(a, cp, x, tiles, st);
        e = hipGetLastError();
    }
    if (e != hipSuccess) return hip_fail(e, "pages_many or pages_few launch");
    if (x.kind == SINGLE) return 0;
    {
        slothost::Scope sc(SLOTSCAN_K_ATTN_JOIN, st);
        if (dtype == SLOTSCAN_BF16) D == 128 ? launch_join<bf16_t, 128>(a, x, rows, st) : launch_join<bf16_t, 64>(a, x, rows, st);
        else D == 128 ? launch_join<f16_t, 128>(a, x, rows, st) : launch_join<f16_t, 64>(a, x, rows, st);
        e = hipGetLastError();
    }
    return e == hipSuccess ? 0 : hip_fail(e, "pages_join launch");
}
