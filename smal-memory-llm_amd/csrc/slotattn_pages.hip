// Attention of the newest tokens of many sequences over a cache in pages, for MI355X (gfx950); semantics: include/slotattn.h, the sharing out of
// the work: slot_attn_pages.h.
//
//   pages_many   128 rows a workgroup, 32 per wave, 64-key tiles; pages_plan before it: the units' costs and their running sums
//   pages_few    16 or 32 rows, 32-key tiles (slotattn_few.hip)
//   pages_join   pieces of one unit
#include "slot_attn_few.h"
#include "slotscan.h"
#include "slotattn.h"
#include "slotpage.h"

using namespace slotattn;
using slothost::fail;
using slothost::hip_fail;
using slothost::al16;

#define MW 4                                         // waves of a workgroup of pages_many
#define MT (64 * MW)
#define MQ (32 * MW)                                 // its query rows
#define MG 512                                       // workgroups: two a CU
#define ML 2                                         // what a unit costs beside its tiles, in tiles: its search, first loads and end take about 5 us
#define MA 9                                         // shares of a CU's first and second workgroup
#define MB 7
// Units run whole, one a workgroup, if none costs more than LW tiles beside LP % of an equal share.  Plan, attention and join of whole units / of shares, 12
// heads of 128 on 4: 8 x 1,024 tokens (the longest 1.1 times a share) 60 / 71 us, 2 x 4,096 (1.27) 157 / 171, 1 x 8,192 (1.3) 280 / 278, 1 x 6,000
// (1.8) 187 / 157.  At D = 64, where pieces are half as large, never: 6 heads, 8 x 1,024 40 / 38, 200 x 33 37 / 35.
#define LW 4
#define LP 120
#define LG 65536                                     // of them at most
#define LT 1024                                      // threads of pages_plan
// The waves of a workgroup of pages_few share one unit up to this many keys and units (a round of workgroups); SINGLE / SHARED with its join, D = 128:
// 32 units of 512 keys 11 / 18 us, 16 of 2,048 24 / 18, 1,024 of 512 54 / 51.
#define UNIT_KEYS 1024
#define UNIT_MOST 256

namespace {

// ------------------------------------------------------------------------------------------- plan
// One workgroup: the rows' tiles of MQ query rows in a row (units), then their key tiles.  Latency: two running sums (4.5 us
// for 8,192 tokens of two prompts, 6 with the list of whole units); without it each of 512 workers would form both.
// (neither past `most`, under 2^30: rows that share tokens may add up to anything)
__device__ __forceinline__ int before_sum(int x, int most, int* s, int& all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int v = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(v, d);
        if (lane >= d) v = min(v + y, most);
    }
    int ex = __shfl_up(v, 1);
    if (lane == 0) ex = 0;
    __syncthreads();
    if (lane == 63) s[w] = v;
    __syncthreads();
    int base = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < LT / 64; i++) {
        if (i == w) base = sum;
        sum = min(sum + s[i], most);
    }
    all = sum;
    return min(base + ex, most);
}

__global__ __launch_bounds__(LT) void pages_plan(PagedArgs a) {
    __shared__ int s_sum[LT / 64], s_most, s_count[LT];
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
        const int u = min(u0 + before_sum(min(tiles, a.units), a.units, s_sum, all), a.units);
        if (r < a.R) first[r] = u;
        u0 = min(u0 + all, a.units);
    }
    if (tid == 0) first[a.R] = u0, s_most = 0;
    s_count[tid] = 0;
    __syncthreads();
    auto row_of = [&](int i) -> int {                 // the last row whose first unit is at or before i
        int lo = 0, hi = a.R;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (first[mid] <= i) lo = mid; else hi = mid;
        }
        return lo;
    };
    int shift = 0;                                    // for the lists of units of about one cost, the longest ones first
    while ((ML + (((a.M << a.shift) + KT - 1) / KT)) >> shift >= LT) shift++;
    int c0 = 0, c1 = 0, lo1 = 0;                      // c1, lo1: of the thread's first unit
    for (int i0 = 0; i0 < u0; i0 += LT) {
        const int i = i0 + tid;
        int c = 0, lo = 0;
        if (i < u0) {
            lo = row_of(i);
            const Seq x = seq_of(a, lo);
            const int t = i - first[lo], off = x.end - x.n, last = min(MQ * (t + 1), x.n * a.rep) - 1;
            c = ML + max(1, Reach<KT>(a, x, MQ * t / a.rep + off, last / a.rep + off).tiles());
            atomicAdd(&s_count[LT - 1 - (c >> shift)], 1);
        }
        int most = c;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) most = max(most, __shfl_xor(most, d));
        if ((tid & 63) == 0) atomicMax(&s_most, most);
        const int at = c0 + before_sum(c, 0x3fffffff, s_sum, all);
        if (i < u0) {
            cost[i] = at;
            if (i == first[lo]) cost_r[lo] = at;
        }
        if (i0 == 0) c1 = c, lo1 = lo;
        c0 += all;
    }
    if (tid == 0) cost[u0] = c0;
    __syncthreads();
    // Whole units, one a workgroup, the longest first, where none is much longer than an equal share: no pieces, nothing to join
    int* list = cost + a.units + 1;
    const int64_t shares = min(a.G, max(c0 * a.Hk / 4, 1)), longest = LW + (int64_t)c0 * a.Hk * LP / (100 * shares);
    const bool whole = s_most <= longest && (int64_t)u0 * a.Hk <= a.whole;
    if (tid == 0) list[0] = whole ? u0 : 0;
    if (whole) {
        const int at = before_sum(s_count[tid], 0x3fffffff, s_sum, all);
        s_count[tid] = at;
        __syncthreads();
        for (int i = tid; i < u0; i += LT) {          // (units of one list in any order: each is computed by itself)
            const int c = i < LT ? c1 : cost[i + 1] - cost[i], lo = i < LT ? lo1 : row_of(i);
            const int k = atomicAdd(&s_count[LT - 1 - (c >> shift)], 1);
            list[1 + 2 * k] = lo;
            list[2 + 2 * k] = i - first[lo];
        }
        // (the row's costs are not read)
    } else {
        // rows without units stand where the next row stands
        for (int r = tid; r < a.R; r += LT)
            if (first[r] == first[r + 1]) cost_r[r] = cost[first[r]];
    }
    if (tid == 0) cost_r[a.R] = c0;
}

// the last i of [lo, hi) with mul x[i] <= y (x ascending, x[lo] does), by all lanes
__device__ __forceinline__ int find(const int* x, int lo, int hi, int mul, int y, int lane) {
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
// Shares of pages_many's workers where two workgroups share each CU: a SIMD issues its older wave first, so the workgroups of the first half of
// the grid have 1.83 us a tile and those of the second 2.35 (8,192 tokens of first prompts); with equal shares the second half ended 30 us later.
// Worker w of an XCD's G / 8: the first half of them are of the grid's first half.
struct PairShares {
    int total, G, h;                                  // h: half of an XCD's workers; 0: equal shares
    __device__ __forceinline__ PairShares(int t, int workers) : total(t), G(workers), h(workers == MG ? workers / 16 : 0) {}
    __device__ __forceinline__ int begin(int w) const {
        if (!h) return (int)((int64_t)total * w / G);
        const int e = w / (2 * h), k = w - 2 * h * e, c = e * h * (MA + MB) + min(k, h) * MA + max(k - h, 0) * MB;
        return (int)((int64_t)total * c / (8 * h * (MA + MB)));
    }
    __device__ __forceinline__ int owner(int x) const {               // of tile x
        if (!h) return (int)(((int64_t)(x + 1) * G - 1) / total);
        const int c = (int)(((int64_t)(x + 1) * (8 * h * (MA + MB)) - 1) / total), e = c / (h * (MA + MB)), k = c - e * h * (MA + MB);
        return 2 * h * e + (k < h * MA ? k / MA : h + (k - h * MA) / MB);
    }
};

// As attn_fwd's: the score tile is K Qt, so that a lane has one query, and its probabilities, rounded to 16 bits, are the next product's operand where
// they are; 64-key tiles by direct loads into two buffers, one barrier a tile.  What differs is where keys lie (a group of 16 keys is of one
// page: its address is scalar) and who does what: a workgroup a whole unit, or 512 workers with equal shares of all key tiles, in which a unit may begin and
// end anywhere; pages_plan chooses.
// Bound by issue beside the matrix products where rows are many, by memory where a unit has a token alone (three waves of four then only load; the unit's tiles
// count as any other's).  Two prompts of 4,096 tokens, 12 heads of 128 on 4: 120 us call after call, 860 TFLOP/s (attn_fwd without pages, in the same process,
// 113); 151 in the first calls of a process, under the profiler.  Of its cycles the matrix units are busy 41 %, vector instructions are issued in 44 % and scalar
// ones in 21 %.  Some of both are the register allocator's: 141 to 196 scalar registers are kept in lanes of vector registers (attn_fwd: 37 to 109), and read
// back in every tile.  56 tokens and 4 prompts of 300 to 1,200 with 200 to 4,000 keys before them, pages of 16: 89 us in such first calls; measured apart
// before, the prompts took 61 and the tokens 28 (140 MB) of 85.  With 8
// waves a workgroup (256 rows, halves of it half a tile apart) 153 where shares took 150, and 127 instead of 79 for the mixture, whose units are small.
template <typename T, int D, bool CAP, bool BIAS>
__global__ __launch_bounds__(MT, 2) void pages_many(PagedArgs a) {
    constexpr int KK = D / 16, DT = D / 32, STAGE = KT * 2 * D;
    constexpr int VA = CAP ? 2 : 4;                   // value operands read ahead: beside a cap's four of them registers would spill
                                                     // in the loop (56 tokens and 4 prompts with a cap: 112 us, with two 108; what spills then is set up
                                                     // once a unit)
    typedef PageLoad<D, KT, MW> Load;
    __shared__ __align__(1024) unsigned char smem[2][2][STAGE];      // [buffer][keys, values]
    const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    fill_rest<D>(a, (int64_t)blockIdx.x * MT + tid, (int64_t)gridDim.x * MT);
    const int* cost_r = a.plan;
    const int* first = a.plan + a.R + 1;
    const int* cost = first + a.R + 1;
    const int total = ld_uni(cost_r, a.R) * a.Hk;
    const int* list = cost + a.units + 1;
    const int units = D == 128 ? ld_uni(list, 0) : 0, G = units ? units * a.Hk : min(a.G, max((total + 3) / 4, 1));
    int me = blockIdx.x;
    if (me >= G) {
        if (tid == 0 && me < a.G) a.join[me].parts = 0;
        return;
    }
    const PairShares sh(total, G);
    int x = 0, end = 1, r = 0;
    if (!units) {
        // workers that follow each other run on one XCD (workgroup i on XCD i % 8): they share keys
        if (G % 8 == 0) me = (me & 7) * (G / 8) + (me >> 3);
        x = sh.begin(me);
        end = sh.begin(me + 1);
        r = uni(find(cost_r, 0, a.R, a.Hk, x, lane));
    }
    Unit left{0, 0, 0, 0, 0};
    const unsigned lds = lds_addr(smem);
    const Load lk(a.k_sp, a.k_st, a.shift, w, lane), lv(a.v_sp, a.v_st, a.shift, w, lane);
    const Ops<D> ops(lane);
    const float f2 = fabsf(a.s.f);
    RowSums<T, D, BIAS> sum(f2);
    while (x < end) {
        // the unit of x, and this worker's key tiles [ka, kb) of its c
        int hk, t, ka = 0, kb = 0xffffff, c = kb;        // (all of them)
        if (units) {
            const int i = me / a.Hk;
            hk = me - i * a.Hk;
            r = ld_uni(list, 1 + 2 * i);
            t = ld_uni(list, 2 + 2 * i);
            x = end;
        } else {
            const int cr = ld_uni(cost_r, r), per = ld_uni(cost_r, r + 1) - cr, y = x - cr * a.Hk;
            if (y >= per * a.Hk) { r++; continue; }
            hk = y / per;
            const int z = y - hk * per + cr, u0 = ld_uni(first, r), u = uni(find(cost, u0, ld_uni(first, r + 1), 1, z, lane));
            const int cu = ld_uni(cost, u), y0 = z - cu;
            c = ld_uni(cost, u + 1) - cu - ML;
            const int y1 = min(c + ML, y0 + end - x);
            ka = max(0, y0 - ML);
            kb = max(0, y1 - ML);
            x += y1 - y0;
            if (kb <= ka) continue;                   // of this unit the worker's share is its beginning alone
            t = u - u0;
        }
        const Seq sq = seq_uni(a, r);
        const int rows = sq.n * a.rep, off = sq.end - sq.n, row0 = MQ * t + 32 * w, row = min(row0 + (lane & 31), rows - 1);
        const int tok = row / a.rep, hq = hk * a.rep + row - tok * a.rep, p = tok + off;
        const Mask mk{1, a.W, sq.pre, sq.klen};
        const int p0 = MQ * t / a.rep + off, p1 = (min(MQ * (t + 1), rows) - 1) / a.rep + off;
        Sight sight(a, sq, row0 / a.rep + off, (min(row0 + 32, rows) - 1) / a.rep + off);
        if (row0 >= rows) sight.s1 = -1, sight.s2 = 0;               // a wave without rows
        Reach<KT> reach(a, sq, p0, p1);
        reach.upto(kb);
        const T* kbase = (const T*)a.k + hk * a.k_sh;
        const T* vbase = (const T*)a.v + hk * a.v_sh;
        const int64_t tab = r * a.t_sr;
        const int last = sq.klen - 1;
        Steps<KT, 1> f;                               // the tile that is fetched
        f.enter(reach, ka);
        Pages<KT / 16> pg;
        auto load = [&](int buf) {
            pg.check(a);
            lk.issue(kbase, pg, f.j, last, lds + (2 * buf) * STAGE);
            lv.issue(vbase, pg, f.j, last, lds + (2 * buf + 1) * STAGE);
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
        bool now = f.next(), more = false;            // a tile is on its way; the pages of the next one are known
        int j0 = f.j, j1 = 0;
        uint32_t lost = 0, lost1 = 0;
        __syncthreads();                              // the last unit's tiles are read
        if (now) {
            pg.fetch(a, tab, f.j, last);
            load(0);
            lost = pg.lost;
            more = f.next();
            if (more) pg.fetch(a, tab, f.j, last);
        }
        // one barrier a tile: behind it the tile is there for every wave and the other buffer is read, so the next one's loads
        // run during this one's products
        for (int buf = 0; now; buf ^= 1) {
            wait_vm<0>();
            tile_barrier();
            now = more;
            if (more) {
                load(buf ^ 1);
                j1 = f.j;
                lost1 = pg.lost;
                more = f.next();
                if (more) pg.fetch(a, tab, f.j, last);
            }
            if (sight.some(j0, j0 + KT - 1)) {
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
                uint4 vr[VA + 1];                     // operand i: column block i % DT of 16 keys i / DT
                auto colop = [&](int i) {
                    vr[i % (VA + 1)] = Ops<D>::at_col(Ops<D>::block(cc, i % DT), Ops<D>::block(c8, i % DT), STAGE + 16 * (i / DT) * Tile<D>::ROWB);
                };
#pragma unroll
                for (int i = 0; i < VA; i++) colop(i);
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    scores<CAP>(s[i], a.s);
                    if constexpr (BIAS) bias(s[i], f2, slope, p, j0 + 32 * i, h);
                }
                if (lost || !sight.all(j0, j0 + KT - 1)) {
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
                    sum.o[i % DT] = mfma32<T>(vr[i % (VA + 1)], pf[i / DT >> 1][i / DT & 1], sum.o[i % DT]);
                    if (i + VA < 4 * DT) colop(i + VA);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            j0 = j1;
            lost = lost1;
        }
        // (a lane's row is found again rather than kept: the loop needs every register)
        int ln = lane;
        asm volatile("" : "+v"(ln));
        const int row1 = min(row0 + (ln & 31), rows - 1), tok1 = row1 / a.rep;
        const Rows rw{sq.s, tok1, hk * a.rep + row1 - tok1 * a.rep, tok1 + off, min(32, rows - row0), see, slope};
        finish<T, D, CAP, BIAS>(a, sum, rw, kbase, vbase, a.table + r * a.t_sr, reach.key(ka), reach.hi, sq.klen, ka == 0 && kb == c,
                                ((int64_t)(2 * me + (ka == 0)) * MW + w) * 32, lane, [&](int j) { return sight.some(j & -KT, j | (KT - 1)); });
        if (ka == 0 && kb < c) left = {r, hk, t, sq.n, sh.owner(end + c - kb - 1) - me + 1};        // its other pieces: up to the worker of its last tile
    }
    if (tid == 0 && me < a.G) a.join[me] = left;
}

// ------------------------------------------------------------------------------------------- join
// A group of D / 4 lanes has 4 columns each of one row: pieces [0, parts) at rows row(s) of the workspace, every `step`-th from `s0` on, as maximum M, sum L and
// weighted values.  Pieces are read four at a time: a row of many is a few round trips to memory.  (A piece in which nothing is visible has l = 0.)
template <int D, class ROW> __device__ __forceinline__ void join_pieces(const PagedArgs& a, int s0, int step, int parts, int c, ROW row, float& M, float& L, float4& acc) {
    M = -INFINITY;
    L = 0.f;
    acc = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int s = s0; s < parts; s += 4 * step) {
        float2 x[4];
        float4 o[4];
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const int64_t at = row(min(s + k * step, parts - 1));
            x[k] = a.pm[at];
            o[k] = *reinterpret_cast<const float4*>(a.po + at * D + 4 * c);
            if (s + k * step >= parts) x[k] = make_float2(-INFINITY, 0.f);
        }
        const float mn = fmaxf(fmaxf(fmaxf(M, x[0].x), fmaxf(x[1].x, x[2].x)), x[3].x), mu = mn == -INFINITY ? 0.f : mn, f0 = exp2_(M - mu);
        L *= f0;
        acc.x *= f0; acc.y *= f0; acc.z *= f0; acc.w *= f0;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool any = x[k].y != 0.f;
            const float f = any ? exp2_(x[k].x - mu) : 0.f;
            if (!any) o[k] = make_float4(0.f, 0.f, 0.f, 0.f);
            L = fmaf(x[k].y, f, L);
            acc.x = fmaf(o[k].x, f, acc.x);
            acc.y = fmaf(o[k].y, f, acc.y);
            acc.z = fmaf(o[k].z, f, acc.z);
            acc.w = fmaf(o[k].w, f, acc.w);
        }
        M = mn;
    }
}
// Row `row` of sequence r's packed rows of head hk, columns 4 c ..
template <typename T, int D> __device__ __forceinline__ void put_joined(const PagedArgs& a, int s, int hk, int row, int c, float L, const float4& o) {
    const float inv = L > 0.f || L != L ? 1.f / L : 0.f;
    const int tok = row / a.rep, hq = hk * a.rep + row - tok * a.rep;
    put4<T>(a.out, nullptr, ((int64_t)(s + tok) * a.Hq + hq) * D + 4 * c, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
}

// Pieces of pages_many: a worker whose last unit goes on in the next ones; a group of lanes a row.  Memory: 512 workers' pieces, 67 MB, 13 us.
template <typename T, int D>
__global__ __launch_bounds__(256) void pages_join(PagedArgs a) {
    constexpr int LN = D / 4, RW = 256 / LN;
    const int me = blockIdx.x;
    const Unit u = a.join[me];
    const int i = blockIdx.y * RW + threadIdx.x / LN, c = threadIdx.x % LN, row = MQ * u.t + i;
    if (u.parts < 2 || row >= u.n * a.rep) return;
    float M, L;
    float4 acc;
    join_pieces<D>(a, 0, 1, u.parts, c, [&](int s) { return (int64_t)(s ? 2 * (me + s) : 2 * me + 1) * MQ + i; }, M, L, acc);
    put_joined<T, D>(a, min(max(a.starts[u.r], 0), a.N), u.hk, row, c, L, acc);
}

// Pieces of pages_few: a row may have hundreds.  A workgroup has `per` of the (row of the batch, head) pairs, and of their units every gridDim.y-th query
// row, one at a time; its NG groups of lanes take every NG-th piece and meet in LDS in order.  Latency: 4 us for 32 sequences, 5.5 for the 1,024
// pieces of one.
template <typename T, int D, int NT>
__global__ __launch_bounds__(NT) void pages_join_few(PagedArgs a, int per, int QR) {
    constexpr int LN = D / 4, NG = NT / LN;
    __shared__ __align__(16) float s_o[NG][D];
    __shared__ float2 s_m[NG];
    const int lane = threadIdx.x & 63, c = threadIdx.x % LN, g = threadIdx.x / LN;
    const int u0 = blockIdx.x * per, u1 = min(a.R * a.Hk, u0 + per);
    for (int b0 = u0; b0 < u1; b0 += 64) {
        const int u = b0 + lane, r = min(u, u1 - 1) / a.Hk, hk = min(u, u1 - 1) - r * a.Hk;
        const Seq x = seq_of(a, r);
        const int rows = x.n * a.rep, at = x.s * a.rep / QR + r;
        Piece p{0, 0};
        if (rows && u < u1) p = a.pieces[at * a.Hk + hk];
        p.parts = p.there(a.G);
        for (uint64_t b = __ballot(u < u1 && (p.parts > 1 || rows > QR)); b; b &= b - 1) {
            const int k = __builtin_ctzll(b), n = lane_of(rows, k), hd = lane_of(hk, k), s = lane_of(x.s, k), at0 = lane_of(at, k);
            Piece q{lane_of(p.me, k), lane_of(p.parts, k)};
            for (int t = 0; QR * t < n; t++) {
                if (t) q = a.pieces[(at0 + t) * a.Hk + hd], q.parts = q.there(a.G);
                if (q.parts < 2) continue;
                for (int i = blockIdx.y; i < min(QR, n - QR * t); i += gridDim.y) {
                    float M, L;
                    float4 acc;
                    join_pieces<D>(a, g, NG, q.parts, c, [&](int z) { return (int64_t)(z ? 2 * (q.me + z) : 2 * q.me + 1) * QR + i; }, M, L, acc);
                    __syncthreads();                  // the last row's sums are read
                    *reinterpret_cast<float4*>(&s_o[g][4 * c]) = acc;
                    if (c == 0) s_m[g] = make_float2(M, L);
                    __syncthreads();
                    if (g == 0) {
                        M = -INFINITY;
#pragma unroll 8
                        for (int z = 0; z < NG; z++) M = fmaxf(M, s_m[z].x);
                        const float Mu = M == -INFINITY ? 0.f : M;
                        L = 0.f;
                        acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
                        for (int z = 0; z < NG; z++) {
                            const float f = exp2_(s_m[z].x - Mu);
                            const float4 o = *reinterpret_cast<const float4*>(&s_o[z][4 * c]);
                            L = fmaf(s_m[z].y, f, L);
                            acc.x = fmaf(o.x, f, acc.x);
                            acc.y = fmaf(o.y, f, acc.y);
                            acc.z = fmaf(o.z, f, acc.z);
                            acc.w = fmaf(o.w, f, acc.w);
                        }
                        put_joined<T, D>(a, s, hd, QR * t + i, c, L, acc);
                    }
                }
            }
        }
    }
}

// How a call runs.
//   MANY    tiles of 128 query rows
//   SHARED  one tile of at most 32 rows a key/value head (one or a few tokens of each sequence): equal shares of all keys, and a join
//   SINGLE  the same where no row has many keys: a workgroup a unit, no join
// Calls of SHARED run as MANY, too; SHARED / MANY with plan and join, D = 128, three query heads a group: a token each of 32 sequences (cap) 58 / 74 us,
// of 256 with a window of 1,024 80 / 79, 2 to 8 tokens of 16 sequences 52 / 52: as fast from two tiles of 16 rows on, and a launch less up to there.
enum { MANY, SHARED, SINGLE };
struct Plan { int kind, QR, G, wgs; int64_t units; size_t join, pm, po, all; };
Plan plan(int64_t N, int64_t R, int64_t M, int64_t page, int64_t Hq, int64_t Hk, int64_t D, int64_t most, int64_t W, bool prefix) {
    Plan x{};
    const int64_t rep = Hq / Hk, rows = std::min(N, R);
    const int64_t keys = prefix ? M * page : std::min(M * page, W + most + 32);
    auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
    x.kind = most * rep > 32 ? MANY : keys <= UNIT_KEYS && rows * Hk <= UNIT_MOST ? SINGLE : SHARED;
    if (x.kind == SINGLE && (R > 65535 || Hk > 65535)) x.kind = SHARED;
    // (its sums of tiles and its numbers of pieces are 32-bit ones)
    if (x.kind == SHARED && ((N * rep / 16 + rows) * Hk * ((M * page + 31) / 32) > 0x3fffffffLL || (N * rep / 16 + R) * Hk > 0x3fffffffLL)) x.kind = MANY;
    x.QR = x.kind == MANY ? MQ : most * rep > 16 ? 32 : 16;
    const int64_t Q = x.QR, K = x.kind == MANY ? KT : 32;
    x.units = N * rep / Q + rows;
    if (x.kind == SINGLE) return x;
    const int64_t tiles = x.units * Hk * ((M * page + K - 1) / K + ML);
    x.G = x.kind == MANY ? (int)std::min<int64_t>(MG, (tiles + 3) / 4) : (int)std::min<int64_t>(FG * 128 / D, std::max<int64_t>(tiles / FS, 1));
    x.join = x.kind == MANY ? up((size_t)(2 * (R + 1) + 3 * x.units + 2) * 4) : 0;
    x.wgs = D == 128 ? (int)std::max<int64_t>(x.G, std::min<int64_t>(x.units * Hk, LG)) : x.G;
    x.pm = x.join + up(x.kind == MANY ? (size_t)x.G * sizeof(Unit) : (size_t)(N * rep / Q + R) * Hk * sizeof(Piece));
    x.po = x.pm + up((size_t)x.G * 2 * Q * sizeof(float2));
    x.all = x.po + up((size_t)x.G * 2 * Q * D * sizeof(float));
    return x;
}

template <typename T, int D, bool CAP, bool BIAS>
void launch_one(const PagedArgs& a, int G, hipStream_t st) {
    slothost::launch(pages_many<T, D, CAP, BIAS>, dim3((unsigned)G), dim3(MT), 0, st, a);
}
template <typename T, int D>
void launch_attn(const PagedArgs& a, bool cap, int G, hipStream_t st) {
    if (cap) a.slopes ? launch_one<T, D, true, true>(a, G, st) : launch_one<T, D, true, false>(a, G, st);
    else a.slopes ? launch_one<T, D, false, true>(a, G, st) : launch_one<T, D, false, false>(a, G, st);
}
template <typename T, int D>
void launch_join(const PagedArgs& a, const Plan& x, int rows, hipStream_t st) {
    if (x.kind == MANY) {
        slothost::launch(pages_join<T, D>, dim3((unsigned)x.G, (unsigned)(MQ * (D / 4) / 256)), dim3(256), 0, st, a);
        return;
    }
    // few units have many pieces each
    const int pairs = a.R * a.Hk, per = (pairs + 2047) / 2048, grid = (pairs + per - 1) / per;
    const dim3 blocks((unsigned)grid, (unsigned)std::max(1, std::min(rows, 4096 / grid)));
    if (pairs <= 32) slothost::launch(pages_join_few<T, D, 1024>, blocks, dim3(1024), 0, st, a, per, x.QR);
    else slothost::launch(pages_join_few<T, D, 256>, blocks, dim3(256), 0, st, a, per, x.QR);
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
    if (k_sp < 0 || v_sp < 0 || k_sp >> 31 || v_sp >> 31) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_pages: pages must be fewer than 2^31 elements apart");
    if (M * page > SLOTATTN_MAX_T || P > SLOTATTN_MAX_T || R > 1 << 24 || t_sr < 0 || most < 1)
        return fail(SLOTSCAN_ERR_SHAPE, "slotattn_pages: shape too large");
    if (int r = slotattn_host::check(q, 0, q_sh, q_st, k, k_sp, k_sh, k_st, v, v_sp, v_sh, v_st, dtype, 1, N, page, Hq, Hk, D, scale, window, cap)) return r;
    if (!table || !starts || !ends || !out) return fail(SLOTSCAN_ERR_NULL, "slotattn_pages: a required pointer is NULL");
    if (!al16(out) || !al16(workspace)) return fail(SLOTSCAN_ERR_ALIGN, "slotattn_pages: out and workspace must be 16-byte aligned");
    const Plan x = plan(N, R, M, page, Hq, Hk, D, std::min(most, N), window, prefix != nullptr);
    if (x.all && !workspace) return fail(SLOTSCAN_ERR_NULL, "slotattn_pages: workspace is NULL");
    // (the sums of all units' tiles are 32-bit ones)
    if (x.kind == MANY && (x.units + 1) * Hk * ((M * page + KT - 1) / KT + ML) > 0x3fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotattn_pages: shape too large");
    PagedArgs a{};
    a.s = slotattn_host::args(q, 0, q_sh, q_st, k, k_sp, k_sh, k_st, v, v_sp, v_sh, v_st, 1, N, page, Hq, Hk, scale, 1, window, cap, slopes, nullptr, prefix);
    a.q = q; a.k = k; a.v = v;
    a.q_sh = q_sh; a.q_st = q_st; a.k_sp = k_sp; a.k_sh = k_sh; a.k_st = k_st; a.v_sp = v_sp; a.v_sh = v_sh; a.v_st = v_st;
    a.table = table; a.t_sr = t_sr; a.starts = starts; a.ends = ends; a.prefix = prefix; a.slopes = slopes;
    a.N = (int)N; a.R = (int)R; a.M = (int)M; a.P = (int)P; a.Hq = (int)Hq; a.Hk = (int)Hk; a.rep = (int)(Hq / Hk);
    a.W = a.s.W; a.shift = __builtin_ctzll((unsigned long long)page); a.units = (int)x.units; a.G = x.G; a.whole = D == 128 ? x.wgs : 0;
    char* ws = (char*)workspace;
    a.plan = (int*)ws; a.join = (Unit*)(ws + x.join); a.pieces = (Piece*)(ws + x.join); a.pm = (float2*)(ws + x.pm); a.po = (float*)(ws + x.po);
    a.out = out;
    hipStream_t st = (hipStream_t)stream;
    const bool cp = cap > 0.f;
    const int tiles = (int)((std::min(most, N) * a.rep + x.QR - 1) / x.QR), rows = (int)std::min<int64_t>(x.QR, std::min(most, N) * a.rep);
    hipError_t e;
    if (x.kind == MANY) {
        slothost::Scope sc(SLOTSCAN_K_ATTN_PLAN, st);
        slothost::launch(pages_plan, dim3(1), dim3(LT), 0, st, a);
        e = hipGetLastError();
        if (e != hipSuccess) return hip_fail(e, "pages_plan launch");
    }
    {
        slothost::Scope sc(SLOTSCAN_K_ATTN, st);
        if (x.kind != MANY) slotattn_few::launch(a, dtype, (int)D, cp, x.QR, x.G, tiles, st);
        else if (dtype == SLOTSCAN_BF16) D == 128 ? launch_attn<bf16_t, 128>(a, cp, x.wgs, st) : launch_attn<bf16_t, 64>(a, cp, x.wgs, st);
        else D == 128 ? launch_attn<f16_t, 128>(a, cp, x.wgs, st) : launch_attn<f16_t, 64>(a, cp, x.wgs, st);
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
