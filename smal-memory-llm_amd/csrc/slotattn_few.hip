// Attention over a cache in pages where a sequence has few query rows: a generated token, a few guessed ones (slot_attn_pages.h).
//
// A unit is one tile of 16 NQ query rows of a key/value head, against 32-key tiles; each wave goes through a ring of its own of two tiles without a
// barrier in the loop.
//   SHARED  every wave is a worker with an equal share of all units' tiles; keys are fetched across the units' borders
//   SINGLE  a workgroup's NW waves share one unit, every NW-th tile each, and meet in LDS: no join behind it
//
// Operands of v_mfma_f32_16x16x32 (16-bit inputs): lane l holds 8 consecutive k values 8 (l >> 4) .. + 7 of row (A) or column (B) l & 15; register r of
// the result holds row 4 (l >> 4) + r of column l & 15.  With the keys as rows a lane's scores are one query's, and those of two blocks of 16 keys
// are the B operand of the next product over 32 keys in the order that two transposing LDS reads give its A operand.  The keys of a block go to rows in the
// order of key_row: a transposing read then meets every bank once (its lanes 0 .. 31 have rows 0 .. 3 and 8 .. 11).
// 16 query rows a product, not 32: of a group's 3 or 4 query heads and one token, tiles of 32 x 32 would be nearly empty, at twice the vector work.
//
// Bound by memory: a step reads each sequence's keys and values once (running maxima and sums, nothing stored between the products).  One sequence of 131,072,
// 262,144 and 524,288 keys takes 52, 96 and 184 us: 8 us, in which the first keys are found (the rows' costs, a search, page numbers) and arrive, and its
// bytes at 6.1 TB/s (a large read alone: 5.8 with its start).  32 sequences of 1,024 to 8,191 keys, 12 heads of 128 on 4, cap 50 (260 MB): 55 us, 4.8
// TB/s; one of 131,072 keys (268 MB) 53; 256 with a window of 1,024 (315 MB) 74, where a unit is hardly longer than a share, so most are cut in two; 2 to 8
// tokens of 16 sequences of up to 16,000 (195 MB) 46: two tiles of rows, both computed also where a sequence's rows fit into one.  1,024 waves, one a SIMD,
// each with a ring of two tiles (32 KB at D = 128); with 1,280 no change.
// Each wave goes through the rows' lengths by itself, 64 at a time.  Rows of 512 keys: 256 46 us, 1,024 197, 8,192 1,535 (5.6 TB/s); on pages_many with its
// plan 53, 202 and 1,541.
#include "slot_attn_pages.h"
#include "slotscan.h"
#include "slot_attn_few.h"

using namespace slotattn;

namespace {

template <typename T> __device__ __forceinline__ f32x4 mfma16(const uint4& a, const uint4& b, f32x4 c);
template <> __device__ __forceinline__ f32x4 mfma16<bf16_t>(const uint4& a, const uint4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4 mfma16<f16_t>(const uint4& a, const uint4& b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ int swap12(int x) { return ((x & 1) << 1) | (x >> 1); }        // 0, 2, 1, 3
__device__ __forceinline__ int key_row(int m) { return 4 * swap12(m >> 2) + (m & 3); }    // the key of row m of a block
// over the four lanes of a query, l, l ^ 16, l ^ 32, l ^ 48
__device__ __forceinline__ float quad_max(float v) {
    auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return half_max(fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1])));
}

// The scores' forms (slot_attn.h), for N values
template <bool CAP, int N> __device__ __forceinline__ void scores_n(float (&s)[N], const AttnArgs& a) {
    if constexpr (CAP) {
        float m = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) m = fmaxf(m, fabsf(s[i]));
        if (__all(m <= a.lim)) {
#pragma unroll
            for (int i = 0; i < N; i++) s[i] = tanh_poly(s[i], a);
        } else if (a.mix) {
#pragma unroll
            for (int i = 0; i < N; i++) s[i] = tanh_mix(s[i], a);
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) s[i] = tanh_exp(s[i], a);
        }
    }
}

// A tile's rows: 16 query rows, one a lane and group of 16 lanes
template <typename T, int D, bool BIAS> struct Rows16 {
    static constexpr int DB = D / 16, KS = D / 32;
    f32x4 o[DB];
    float m, mu, l;                                   // a row's reference, the same in base 2, its sum
    bool far;
    uint4 q[KS];
    int tok, hq, p;
    Sees see;
    float slope;
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < DB; i++) o[i] = {0.f, 0.f, 0.f, 0.f};
        m = -INFINITY;
        mu = l = 0.f;
        far = false;
    }
    // 8 scores a lane become probabilities as an operand (slot_attn_rows.h), in bf16 as two of them, whose sum has 16 bits: one alone would be off by as
    // much as the result's own rounding, and the products wait for memory anyway
    static constexpr int PARTS = sizeof(T) == 2 && HEAD<T> == 0.f ? 2 : 1;
    __device__ __forceinline__ void weigh(float (&s)[8], float F, float lazy, float head, uint4 (&pf)[PARTS]) {
        float mx = s[0];
#pragma unroll
        for (int i = 1; i < 8; i++) mx = fmaxf(mx, s[i]);
        mx = quad_max(mx) - head;
        if (__any(mx > m + lazy)) {
            const float mn = fmaxf(m, mx), f = m == -INFINITY ? 0.f : exp2_((m - mn) * F);
            m = mn;
            mu = m == -INFINITY ? 0.f : m * F;
            far = __any(fabsf(mu) > FAR);
            l *= f;
#pragma unroll
            for (int i = 0; i < DB; i++) o[i] *= f;
        }
        if (far) {
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] = (s[i] - (m == -INFINITY ? 0.f : m)) * F;
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] = fmaf(s[i], F, -mu);
        }
#pragma unroll
        for (int i = 0; i < 8; i++) {
            s[i] = exp2_(s[i]);
            l += s[i];
        }
        pf[0] = make_uint4(pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3]), pack2<T>(s[4], s[5]), pack2<T>(s[6], s[7]));
        if constexpr (PARTS == 2) {
            const uint32_t x[4] = {pf[0].x, pf[0].y, pf[0].z, pf[0].w};
#pragma unroll
            for (int i = 0; i < 8; i++) s[i] -= unpack<T>(x[i / 2], i & 1);
            pf[1] = make_uint4(pack2<T>(s[0], s[1]), pack2<T>(s[2], s[3]), pack2<T>(s[4], s[5]), pack2<T>(s[6], s[7]));
        }
    }
    __device__ __forceinline__ void close() {
        auto p2 = __builtin_amdgcn_permlane16_swap(__float_as_uint(l), __float_as_uint(l), false, false);
        l = half_sum(__uint_as_float(p2[0]) + __uint_as_float(p2[1]));
        m = m == -INFINITY ? m : mu;
    }
    __device__ __forceinline__ bool ill() const {     // a value that is not finite
        float t = l * 0.f;
#pragma unroll
        for (int i = 0; i < DB; i++)
#pragma unroll
            for (int r = 0; r < 4; r++) t = fmaf(o[i][r], 0.f, t);
        return t != 0.f;
    }
};
__device__ __forceinline__ uint32_t bits16(bool x) {                  // rows (lanes l, l ^ 16, l ^ 32, l ^ 48) for which x holds
    uint64_t b = __ballot(x);
    b |= b >> 32;
    return (uint32_t)(b | b >> 16) & 0xffffu;
}

// Sum over the lanes up to this one, `most` at most (under 2^30).  (Rows that share tokens may add up to anything: the tiles behind `most` are nobody's.)
__device__ __forceinline__ int scan_up(int x, int lane, int most) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if (lane >= d) x = min(x + y, most);
    }
    return x;
}
// Tiles of QR rows of a sequence, and 32-key tiles of each: as many as its tokens see together, so that no table of them is needed
template <int QR> __device__ __forceinline__ int few_tiles(const PagedArgs& a, const Seq& x, int& per) {
    per = max(1, Reach<32>(a, x, x.end - x.n, x.end - 1).tiles());
    return (x.n * a.rep + QR - 1) / QR;
}
template <int QR> __device__ __forceinline__ int few_cost(const PagedArgs& a, int r) {
    if (r >= a.R) return 0;
    int per;
    const int t = few_tiles<QR>(a, seq_of(a, r), per);
    return t * per;
}

// A place in the worker's share: row, tiles of one head in front of it, the next tile and the share's end
struct Place { int r, base, x, end; };
// A unit: its sequence and head, tile of rows, and of its key tiles [ka, kb); positions of its rows; its keys up to the last of those tiles
struct FewUnit {
    Seq sq;
    int r, hk, t, per, ka, kb, p0, p1;
    Reach<32> reach;
    template <int QR> __device__ __forceinline__ void rows(const PagedArgs& a) {
        const int n = sq.n * a.rep, off = sq.end - sq.n;
        p0 = QR * t / a.rep + off;
        p1 = (min(QR * (t + 1), n) - 1) / a.rep + off;
        reach = Reach<32>(a, sq, p0, p1);
        reach.upto(kb);
    }
    // the next unit of a share
    template <int QR> __device__ __forceinline__ bool next(const PagedArgs& a, Place& at) {
        while (at.x < at.end) {
            sq = seq_uni(a, at.r);
            const int cost = few_tiles<QR>(a, sq, per) * per, y = at.x - at.base * a.Hk;
            if (y >= cost * a.Hk) {                   // the next row
                if (++at.r >= a.R) return false;
                at.base += cost;
                continue;
            }
            r = at.r;
            hk = y / cost;
            const int z = y - hk * cost;
            t = z / per;
            ka = z - t * per;
            kb = min(per, ka + at.end - at.x);
            at.x += kb - ka;
            rows<QR>(a);
            return true;
        }
        return false;
    }
};
template <typename T, int D, bool CAP, bool BIAS, int NQ, int NW, bool SHARED>
__global__ __launch_bounds__(64 * NW) void pages_few(PagedArgs a) {
    constexpr int KS = D / 32, DB = D / 16, ST = 32 * 2 * D, QR = 16 * NQ;
    typedef PageLoad<D, 32, 1> Load;
    typedef Tile<D> Ti;
    __shared__ __align__(1024) unsigned char smem[NW][2][2][ST];     // [wave][buffer][keys, values]
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int w = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
    Place at{0, 0, 0, 0};                             // what is computed next
    FewUnit u;
    int me = 0, total = 0, G = 1;
    if constexpr (SHARED) {
        const int C = (a.R + 63) / 64, most = 0x3fffffff / a.Hk;
        int mine = 0;
        for (int i = 0; i < C; i++) mine = min(mine + few_cost<QR>(a, lane * C + i), most);
        const int upto = scan_up(mine, lane, most);
        total = lane_of(upto, 63) * a.Hk;
        G = min((int)gridDim.x, max(total / FS, 1));
        me = blockIdx.x;
        if (me < G) {
            if (G % 8 == 0) me = (me & 7) * (G / 8) + (me >> 3);     // workers that follow each other run on one XCD
            const Shares sh(total, G);
            at.x = sh.begin(me);
            at.end = sh.begin(me + 1);
            const int y = at.x / a.Hk, up = __shfl_up(upto, 1), ahead0 = lane ? up : 0, L = 63 - __builtin_clzll(__ballot(ahead0 <= y) | 1);
            at.base = lane_of(ahead0, L);
            at.r = L * C;
            for (int i0 = 0; C > 1 && i0 < C; i0 += 64) {            // the row within the lane's rows
                const int cost = i0 + lane < C ? few_cost<QR>(a, at.r + i0 + lane) : 0, v = scan_up(cost, lane, most), all = lane_of(v, 63);
                if (at.base + all <= y) { at.base += all; continue; }
                const int vp = __shfl_up(v, 1), v0 = lane ? vp : 0, k = 63 - __builtin_clzll(__ballot(at.base + v0 <= y) | 1);
                at.base += lane_of(v0, k);
                at.r += i0 + k;
                break;
            }
        }
    } else {
        u.r = blockIdx.z;
        u.hk = blockIdx.y;
        u.t = blockIdx.x;
    }
    const unsigned lds = lds_addr(smem[w]);
    const Load lk(a.k_sp, a.k_st, a.shift, 0, lane), lv(a.v_sp, a.v_st, a.shift, 0, lane);
    // a lane's operand addresses: chunk 4 ks + g of key row l & 15, and of a transposing read 4 columns of one of 4 keys
    const int kr = key_row(lane & 15), vr = 4 * swap12(g) + ((lane & 15) >> 2);
    const unsigned krow = kr * Ti::ROWB + 16 * Ti::pos(kr, g), vcol = vr * Ti::ROWB + 16 * Ti::pos(vr, (lane & 3) >> 1) + 8 * (lane & 1);
    const int key0 = 4 * swap12(g);                   // the lane's keys of a block: key0 .. + 3
    const float f2 = fabsf(a.s.f), F = BIAS ? 1.f : f2, lazy = LAZY / F, head = HEAD<T> / F;
    Rows16<T, D, BIAS> row[NQ];
    // what is fetched, two tiles ahead
    Place ahead{0, 0, 0, 0};
    Steps<32, NW> f;
    Pages<2> pg;
    int64_t ftab = 0;
    int flast = 0;
    const T* fk = nullptr;
    const T* fv = nullptr;
    bool open = false;                                // f is in a unit
    auto enter = [&](const FewUnit& n) {
        f.enter(n.reach, n.ka + w);
        ftab = n.r * a.t_sr;
        flast = n.sq.klen - 1;
        fk = (const T*)a.k + n.hk * a.k_sh;
        fv = (const T*)a.v + n.hk * a.v_sh;
        open = true;
    };
    auto fetch = [&]() -> bool {
        for (;;) {
            if (open && f.next()) break;
            open = false;
            FewUnit n;
            if (!SHARED || !n.next<QR>(a, ahead)) return false;
            enter(n);
        }
        pg.fetch(a, ftab, f.j, flast);
        return true;
    };
    auto keys = [&](int buf) {
        pg.check(a);
        lk.issue(fk, pg, f.j, flast, lds + (2 * buf) * ST);
    };
    auto values = [&](int buf) { lv.issue(fv, pg, f.j, flast, lds + (2 * buf + 1) * ST); };
    bool e1 = false, e2 = false;                      // the next tile is on its way, the one after it is known
    uint32_t lost0 = 0, lost1 = 0;
    auto begin = [&]() {
        e1 = e2 = false;
        if (!fetch()) return;
        keys(0);
        values(0);
        lost0 = pg.lost;
        e1 = fetch();
        if (!e1) return;
        keys(1);
        values(1);
        lost1 = pg.lost;
        e2 = fetch();
    };
    int buf = 0;
    if constexpr (SHARED) {
        ahead = at;
        begin();
    }
    for (;;) {
        if constexpr (SHARED) {
            if (!u.next<QR>(a, at)) break;
        } else {
            u.sq = seq_uni(a, u.r);
            if (u.t >= few_tiles<QR>(a, u.sq, u.per)) break;
            u.ka = 0;
            u.kb = u.per;
            u.rows<QR>(a);
            enter(u);
            buf = 0;
            begin();
        }
        const int rows = u.sq.n * a.rep, off = u.sq.end - u.sq.n, r0 = QR * u.t;
        const Mask mk{1, a.W, u.sq.pre, u.sq.klen};
#pragma unroll
        for (int n = 0; n < NQ; n++) {
            Rows16<T, D, BIAS>& x = row[n];
            const int i = min(r0 + 16 * n + (lane & 15), rows - 1);
            x.tok = i / a.rep;
            x.hq = u.hk * a.rep + i - x.tok * a.rep;
            x.p = x.tok + off;
            const T* q = (const T*)a.q + x.hq * a.q_sh + (int64_t)(u.sq.s + x.tok) * a.q_st + 8 * g;
#pragma unroll
            for (int ks = 0; ks < KS; ks++) x.q[ks] = ld16(q + 32 * ks);
            if (a.s.f < 0.f)                          // a negative scale: of the queries' sign, so that larger products are larger scores
#pragma unroll
                for (int ks = 0; ks < KS; ks++) { x.q[ks].x ^= 0x80008000u; x.q[ks].y ^= 0x80008000u; x.q[ks].z ^= 0x80008000u; x.q[ks].w ^= 0x80008000u; }
            x.slope = BIAS ? a.slopes[x.hq] * LOG2E : 0.f;
            x.see = Sees::query(mk, x.p);
            x.clear();
        }
        const Sight sight(a, u.sq, u.p0, u.p1);
        Steps<32, NW> c;
        c.enter(u.reach, u.ka + w);
        // Keys and values are fetched two tiles ahead, each into the place that it has just been read from.  With slopes the counted waits are the loop's only
        // ones, and a wave has one and a half to two tiles on their way while it computes.  Without them it has less: the compiler does not know that the counted
        // waits cover the query rows' loads and waits for these where they are first used, in the loop, which in every tile is a wait for all that is
        // outstanding.  This tile's values and the whole next tile are there before its first product, and only the tile after that comes in beside the rest.
        for (; c.next(); buf ^= 1) {
            const int j0 = c.j;
            if (e1) wait_vm<3 * Load::N>();           // behind this tile's keys: its values, the next keys and values
            else wait_vm<Load::N>();
            asm volatile("" ::: "memory");
            const unsigned bk = lds + (2 * buf) * ST + krow, bv = lds + (2 * buf + 1) * ST + vcol;
            f32x4 s[NQ][2];
#pragma unroll
            for (int n = 0; n < NQ; n++) s[n][0] = s[n][1] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ks++)
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const uint4 k = lds16((bk ^ (64 * ks)) + 16 * b * Ti::ROWB);
#pragma unroll
                    for (int n = 0; n < NQ; n++) s[n][b] = mfma16<T>(k, row[n].q[ks], s[n][b]);
                }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the keys are read before their place is filled again
            if (e2) keys(buf);
            const bool all = lost0 == 0 && sight.all(j0, j0 + 31);
            uint4 pf[NQ][Rows16<T, D, BIAS>::PARTS];
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                Rows16<T, D, BIAS>& x = row[n];
                float v[8];
#pragma unroll
                for (int i = 0; i < 8; i++) v[i] = s[n][i >> 2][i & 3];
                scores_n<CAP>(v, a.s);
                if constexpr (BIAS) {
                    const float d = (float)(x.p - j0 - key0);
#pragma unroll
                    for (int i = 0; i < 8; i++) v[i] = fmaf(-x.slope, fabsf(d - (float)(16 * (i >> 2) + (i & 3))), v[i] * f2);
                }
                if (!all) {
                    const unsigned y = (unsigned)(j0 + key0), z = y - x.see.first;
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const unsigned at8 = 16 * (i >> 2) + (i & 3);
                        const bool ok = (z + at8 <= x.see.count || y + at8 < x.see.below) && !bit(lost0, i >> 2);
                        v[i] = ok ? v[i] : -INFINITY;
                    }
                }
                x.weigh(v, F, lazy, head, pf[n]);
            }
            if (e2) wait_vm<3 * Load::N>();           // behind the values: the next tile, the keys after it
            else if (e1) wait_vm<2 * Load::N>();
            else wait_vm<0>();
            asm volatile("" ::: "memory");
#pragma unroll
            for (int d = 0; d < DB; d++) {
                const unsigned v = bv ^ (32 * d);
                const uint2 lo = lds_tr(v), hi = lds_tr(v + 16 * Ti::ROWB);
                const uint4 vt = make_uint4(lo.x, lo.y, hi.x, hi.y);
#pragma unroll
                for (int n = 0; n < NQ; n++)
#pragma unroll
                    for (int i = 0; i < Rows16<T, D, BIAS>::PARTS; i++) row[n].o[d] = mfma16<T>(vt, pf[n][i], row[n].o[d]);
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");        // the values, too
            lost0 = lost1;
            e1 = e2;
            if (e2) {
                values(buf);
                lost1 = pg.lost;
                e2 = fetch();
            }
        }
        const T* kb = (const T*)a.k + u.hk * a.k_sh;
        const T* vb = (const T*)a.v + u.hk * a.v_sh;
        const int32_t* tab = a.table + u.r * a.t_sr;
        const int first = u.reach.key(u.ka);
        auto keeps = [&](const Rows16<T, D, BIAS>& x) {
            return keeps_paged<T, D>(a, kb, vb, tab, x.see, first, u.reach.hi, u.sq.klen, 32, Rows16<T, D, BIAS>::PARTS == 2, lane,
                                     [&](int j) { return (j & ~31) < u.reach.at || (j & ~31) >= u.reach.at + u.reach.gap; });
        };
        auto exact = [&](const Rows16<T, D, BIAS>& x, int i, float& m1, float& l1, float (&o1)[D / 64]) {
            exact_paged<T, D, CAP, BIAS>(a, (const T*)a.q + lane_of(x.hq, i) * a.q_sh + (int64_t)(u.sq.s + lane_of(x.tok, i)) * a.q_st, kb, vb, tab,
                                         lane_of(x.see, i), lane_of(x.slope, i), lane_of(x.p, i), first, u.reach.hi, lane, m1, l1, o1);
        };
        if constexpr (SHARED) {
            const bool whole = u.ka == 0 && u.kb == u.per;
            const int64_t part = (int64_t)(2 * me + (u.ka == 0)) * QR;
            if (u.ka == 0 && lane == 0)
                a.pieces[(u.sq.s * a.rep / QR + u.r + u.t) * a.Hk + u.hk] = {me, whole ? 1 : Shares(total, G).owner(at.end + u.per - u.kb - 1) - me + 1};
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                Rows16<T, D, BIAS>& x = row[n];
                const int used = rows - r0 - 16 * n;
                const bool in = (lane & 15) < used;
                x.close();
                uint32_t odd = bits16(x.ill() && x.l == x.l && in);
                if (odd) odd &= ~bits16(keeps(x));
                for (uint32_t b = odd; b; b &= b - 1) {               // rows next to infinities and NaN, from their visible pairs alone
                    const int i = __builtin_ctz(b);
                    float m1, l1, o1[D / 64];
                    exact(x, i, m1, l1, o1);
                    if (whole) {
                        const float inv1 = l1 > 0.f || l1 != l1 ? 1.f / l1 : 0.f;
                        for (int e = 0; e < D / 64; e++) o1[e] *= inv1;
                        put_row<T, D>((T*)a.out + ((int64_t)(u.sq.s + lane_of(x.tok, i)) * a.Hq + lane_of(x.hq, i)) * D, lane, o1);
                    } else {
                        for (int e = 0; e < D / 64; e++) a.po[(part + 16 * n + i) * D + lane * (D / 64) + e] = o1[e];
                        if (lane == 0) a.pm[part + 16 * n + i] = make_float2(m1, l1);
                    }
                }
                if (!in || bit(odd, lane & 15)) continue;
                if (whole) {
                    const int64_t o = ((int64_t)(u.sq.s + x.tok) * a.Hq + x.hq) * D + 4 * g;
                    const float inv = x.l > 0.f || x.l != x.l ? 1.f / x.l : 0.f;
#pragma unroll
                    for (int d = 0; d < DB; d++) put4<T>(a.out, nullptr, o + 16 * d, x.o[d][0] * inv, x.o[d][1] * inv, x.o[d][2] * inv, x.o[d][3] * inv);
                } else {
                    const int64_t o = part + 16 * n + (lane & 15);
#pragma unroll
                    for (int d = 0; d < DB; d++) *reinterpret_cast<f32x4*>(a.po + o * D + 16 * d + 4 * g) = x.o[d];
                    if (g == 0) a.pm[o] = make_float2(x.m, x.l);
                }
            }
        } else {
            // the waves' parts: (m, l) of every row to all, then the weighted sums through LDS (its tiles are read)
            __shared__ float s_m[NW][QR], s_l[NW][QR], s_L[QR];      // the waves' maxima and sums of every row, the workgroup's sums
            __shared__ uint32_t s_bad[NW];
            float* so = reinterpret_cast<float*>(smem);               // [wave][row][D + 4]
            constexpr int SO = D + 4;
            static_assert(NW * QR * SO * 4 <= (int)sizeof(smem), "the waves' sums fit");
            const int used = min(QR, rows - r0);
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                row[n].close();
                if (g == 0) { s_m[w][16 * n + lane] = row[n].m; s_l[w][16 * n + lane] = row[n].l; }
            }
            __syncthreads();
            uint32_t odd = 0;
#pragma unroll
            for (int n = 0; n < NQ; n++) {
                Rows16<T, D, BIAS>& x = row[n];
                const int i = 16 * n + (lane & 15);
                float M = -INFINITY, Ls = 0.f;
#pragma unroll
                for (int k = 0; k < NW; k++) M = fmaxf(M, s_m[k][i]);
                const float Mu = M == -INFINITY ? 0.f : M;
#pragma unroll
                for (int k = 0; k < NW; k++) Ls += s_l[k][i] * exp2_(s_m[k][i] - Mu);
                const float fm = exp2_(x.m - Mu);
                odd |= bits16(x.ill() && Ls == Ls && i < used) << (16 * n);
                if (i < used)
#pragma unroll
                    for (int d = 0; d < DB; d++) *reinterpret_cast<f32x4*>(so + (w * QR + i) * SO + 16 * d + 4 * g) = x.o[d] * fm;
                if (w == 0 && g == 0) s_L[i] = Ls;    // not over s_l, which the other waves may still read
            }
            if (lane == 0) s_bad[w] = odd;
            __syncthreads();
            uint32_t bad = 0;
#pragma unroll
            for (int k = 0; k < NW; k++) bad |= s_bad[k];
            if (bad) {                                // rows next to infinities and NaN, from their visible pairs alone; the same in every wave
                uint32_t kept = 0;
#pragma unroll
                for (int n = 0; n < NQ; n++) kept |= bits16(keeps(row[n])) << (16 * n);
                bad &= ~kept;
                for (; bad; bad &= bad - 1) {
                    const int i = __builtin_ctz(bad);
                    if (i % NW != w) continue;
                    float m1, l1, o1[D / 64];
                    exact(NQ == 2 && i >= 16 ? row[NQ - 1] : row[0], i & 15, m1, l1, o1);
                    for (int k = 0; k < NW; k++)
                        for (int e = 0; e < D / 64; e++) so[(k * QR + i) * SO + lane * (D / 64) + e] = k ? 0.f : o1[e];
                    if (lane == 0) s_L[i] = l1;
                }
                __syncthreads();
            }
            // used rows x D values: 8 lanes a row
            for (int i = tid >> 3; i < used; i += 8 * NW) {
                const int c4 = 4 * (tid & 7), k = r0 + i;
                const float lr = s_L[i], inv = lr > 0.f || lr != lr ? 1.f / lr : 0.f;
                const int kt = k / a.rep, kh = u.hk * a.rep + k - kt * a.rep;
                const int64_t o = ((int64_t)(u.sq.s + kt) * a.Hq + kh) * D;
#pragma unroll
                for (int e = 0; e < D / 32; e++) {
                    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int z = 0; z < NW; z++) v += *reinterpret_cast<const f32x4*>(so + (z * QR + i) * SO + c4 + 32 * e);
                    put4<T>(a.out, nullptr, o + c4 + 32 * e, v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
                }
            }
            u.t += gridDim.x;
            __syncthreads();                          // the sums are read before the next unit's tiles take their place
        }
    }
    fill_rest<D>(a, ((int64_t)(blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * 64 * NW + tid, (int64_t)gridDim.x * gridDim.y * gridDim.z * 64 * NW);
}

template <typename T, int D, bool CAP, bool BIAS, int NQ>
void launch_rows(const PagedArgs& a, int G, int tiles, hipStream_t st) {
    if (G) slothost::launch(pages_few<T, D, CAP, BIAS, NQ, 1, true>, dim3((unsigned)G), dim3(64), 0, st, a);
    else slothost::launch(pages_few<T, D, CAP, BIAS, NQ, FW, false>, dim3((unsigned)tiles, (unsigned)a.Hk, (unsigned)a.R), dim3(64 * FW), 0, st, a);
}
template <typename T, int D, bool CAP, bool BIAS>
void launch_one(const PagedArgs& a, int QR, int G, int tiles, hipStream_t st) {
    QR == 16 ? launch_rows<T, D, CAP, BIAS, 1>(a, G, tiles, st) : launch_rows<T, D, CAP, BIAS, 2>(a, G, tiles, st);
}
template <typename T, int D>
void launch_attn(const PagedArgs& a, bool cap, int QR, int G, int tiles, hipStream_t st) {
    if (cap) a.slopes ? launch_one<T, D, true, true>(a, QR, G, tiles, st) : launch_one<T, D, true, false>(a, QR, G, tiles, st);
    else a.slopes ? launch_one<T, D, false, true>(a, QR, G, tiles, st) : launch_one<T, D, false, false>(a, QR, G, tiles, st);
}

}  // namespace

void slotattn_few::launch(const PagedArgs& a, int dtype, int D, bool cap, int QR, int G, int tiles, hipStream_t st) {
    if (dtype == SLOTSCAN_BF16) D == 128 ? launch_attn<bf16_t, 128>(a, cap, QR, G, tiles, st) : launch_attn<bf16_t, 64>(a, cap, QR, G, tiles, st);
    else D == 128 ? launch_attn<f16_t, 128>(a, cap, QR, G, tiles, st) : launch_attn<f16_t, 64>(a, cap, QR, G, tiles, st);
}
