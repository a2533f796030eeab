// What the kernels of the attention over pages share (slotattn_pages.hip, slotattn_few.hip).
//
// The query rows of a key/value head -- the tokens of a sequence times the query heads of the group -- are cut into tiles; a tile against the keys
// that it sees is a unit, and all units' key tiles in a row are shared out to the workers in equal contiguous pieces, so that neither
// ragged lengths nor causality leave a worker more than another.  A piece that is not a whole unit leaves its rows' maxima, sums and
// weighted values in the workspace, two such pieces a worker at most, and pages_join combines a unit's pieces in order.
// (pages_many takes whole units, a workgroup each, where they are much alike.)
#pragma once
#include "slot_attn_rows.h"
#include "slot_attn_host.h"

namespace slotattn {

// What is left for the join.  pages_many: of each worker, the unit that begins in it and goes on in the next (row, head, tile, tokens, pieces; 0: none).
// pages_few: of each unit, the worker in which it begins and its pieces, at ((s rep) / QR + row + tile) Hk + head, s its sequence's first token:
// a place of its own for every tile of QR rows of the batch.
struct Unit { int r, hk, t, n, parts; };
struct Piece {
    int me, parts;
    // Pieces to read of those of `workers` workers.  Rows that share tokens can ask for more tiles than are handed out; units behind those leave nothing
    // here, and what the workspace held before counts only where it names workers: the join then reads pieces of other units, but none outside.
    __host__ __device__ __forceinline__ int there(int workers) const { return me >= 0 && parts <= workers - me ? parts : 0; }
};

struct PagedArgs {
    AttnArgs s;                                       // the scores' constants
    const void* q; const void* k; const void* v;
    int64_t q_sh, q_st, k_sp, k_sh, k_st, v_sp, v_sh, v_st;
    const int32_t* table; int64_t t_sr;
    const int32_t* starts; const int32_t* ends; const int32_t* prefix; const float* slopes;
    int N, R, M, P, Hq, Hk, rep, W, shift, units, G, whole;   // units: room for them in the plan; pages_many's workers; whole units at most
    // running costs of the rows (R + 1), first units of the rows (R + 1), running costs (units + 1); then 0, or the number of units
    // and (row, tile of rows) of each, the longest first
    int* plan;
    Unit* join; Piece* pieces;
    float* po; float2* pm;                            // (worker, piece that it begins or goes on with, row of the tile)
    void* out;
};

// Whole numbers that no kernel of this library writes while they are read, at addresses that are the same for the wave: loaded through the
// scalar cache, so that a wait for them is none for the direct loads on their way
typedef __attribute__((address_space(4))) const int32_t const_i32;
__device__ __forceinline__ int ld_uni(const int32_t* p, int64_t i) { return ((const_i32*)(uintptr_t)p)[i]; }

// A sequence's part of the batch, whatever the tensors hold: tokens s .. s + n - 1 of [0, N), the first at position end - n
struct Seq { int s, n, end, klen, pre; };
__host__ __device__ __forceinline__ Seq make_seq(const PagedArgs& a, int s0, int s1, int end, int pre) {
    Seq x;
    x.s = min(max(s0, 0), a.N);
    x.n = min(max(s1, x.s), a.N) - x.s;
    x.end = min(max(end, 0), (1 << 30) - 1);
    x.klen = min(x.end, a.M << a.shift);
    x.pre = max(0, min(pre, x.klen));                 // (any number: sums and differences with it stay in range)
    return x;
}
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int r) {                       // a row of the lane's
    return make_seq(a, a.starts[r], a.starts[r + 1], a.ends[r], a.prefix ? a.prefix[r] : 0);
}
__device__ __forceinline__ Seq seq_uni(const PagedArgs& a, int r) {                      // a row of the wave's
    return make_seq(a, ld_uni(a.starts, r), ld_uni(a.starts, r + 1), ld_uni(a.ends, r), a.prefix ? ld_uni(a.prefix, r) : 0);
}
// The tiles of STEP keys that positions [p0, p1] see: [lo, hi) from a multiple of STEP on, without the `gap` keys from `at` on that may lie between
// a prefix and the band.  Tiles are numbered, counted and shared out without the gap.
template <int STEP> struct Reach {
    int lo, hi, at, gap;
    Reach() = default;
    __host__ __device__ __forceinline__ Reach(const PagedArgs& a, const Seq& x, int p0, int p1) {
        const int band = max(0, max(p0, 0) - a.W + 1) & ~(STEP - 1);
        lo = x.pre > 0 ? 0 : band;
        hi = p1 < 0 ? lo : min(x.klen, max(p1 + 1, x.pre));
        at = (x.pre + STEP - 1) & ~(STEP - 1);
        gap = x.pre > 0 ? max(0, band - at) : 0;
    }
    __host__ __device__ __forceinline__ int key(int i) const {        // the i-th tile's first
        const int y = lo + STEP * i;
        return y + (y >= at ? gap : 0);
    }
    __host__ __device__ __forceinline__ int tiles() const {
        const int n = (hi - lo + STEP - 1) / STEP;
        return max(0, n - max(0, min(gap, lo + STEP * n - at)) / STEP);
    }
    __host__ __device__ __forceinline__ void upto(int n) { hi = min(hi, key(n - 1) + STEP); }      // the first n tiles alone (n >= 1)
};

// Equal shares of `total` tiles for G workers: worker w has those from begin(w) on.
struct Shares {
    int G, q, rem;
    __host__ __device__ __forceinline__ Shares(int total, int workers) : G(workers), q(total / workers), rem(total - q * workers) {}
    __host__ __device__ __forceinline__ int begin(int w) const { return w * q + min(w, rem); }
    __host__ __device__ __forceinline__ int owner(int x) const {      // of tile x
        const int big = rem * (q + 1);
        return x < big ? x / (q + 1) : rem + (x - big) / q;
    }
};

// The pages of a tile's groups of 16 keys from j0 on.  fetch() asks for their numbers and check() looks at them, a tile later: a number outside of the
// pool stands for page 0, and its group's bit says that its keys are not seen.  A group behind the sequence's last key has that key's page.
template <int GROUPS> struct Pages {
    int id[GROUPS];
    uint32_t lost;
    __device__ __forceinline__ void fetch(const PagedArgs& a, int64_t row, int j0, int last) {
        id[0] = ld_uni(a.table, row + (j0 >> a.shift));
        if (16 * GROUPS >> a.shift > 1) {
#pragma unroll
            for (int g = 1; g < GROUPS; g++) id[g] = ld_uni(a.table, row + (min(j0 + 16 * g, last) >> a.shift));
        }
    }
    __device__ __forceinline__ void check(const PagedArgs& a) {
        if (16 * GROUPS >> a.shift <= 1) {            // one page
            const bool bad = (unsigned)id[0] >= (unsigned)a.P;
            id[0] = bad ? 0 : id[0];
            lost = bad ? (1u << GROUPS) - 1 : 0u;
            return;
        }
        lost = 0;
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            const bool bad = (unsigned)id[g] >= (unsigned)a.P;
            id[g] = bad ? 0 : id[g];
            lost |= bad ? 1u << g : 0u;
        }
    }
};

// One direct load as dma16s's, whose base is in scalar registers already
__device__ __forceinline__ void dma16b(uint64_t base, unsigned off, unsigned lds) {
    // five wait states for a base that the vector unit has just written
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "{m0}"(lds), "v"(off), "s"(base) : "memory");
}
// Direct loads of a tile of ROWS keys by wave w of NW, laid out as TileLoad's.  A group of 16 keys is of one page: its address is formed once, by
// the scalar unit, and a lane's offsets within a group are held in registers.  (With 64-bit products for every load they were half of a wave's instructions.)
template <int D, int ROWS, int NW> struct PageLoad {
    static constexpr int N = ROWS * 2 * D / 1024 / NW, RPL = 512 / D;  // loads per wave, rows per load
    static constexpr int VAR = RPL * NW >= 16 ? 1 : 16 / (RPL * NW);  // loads of one group
    static constexpr int GROUPS = ROWS / 16, GPL = RPL * NW > 16 ? 2 : 1;                // groups of one load of all waves
    static_assert(NW == 1 || VAR == 1, "one load a group, or all of them");
    unsigned off[VAR], sp, st;                        // sp, st: bytes between pages and between rows
    int w, lane, shift;
    __device__ __forceinline__ PageLoad(int64_t page_stride, int64_t stride, int shift_, int wave, int l)
        : sp((unsigned)(2 * page_stride)), st((unsigned)(2 * stride)), w(wave), lane(l), shift(shift_) {
#pragma unroll
        for (int i = 0; i < VAR; i++) off[i] = (unsigned)((RPL * (NW * i + w) & 15) + lane / Tile<D>::CH) * st + 16 * chunk(i);
    }
    __device__ __forceinline__ int row(int i) const { return RPL * (NW * i + w) + lane / Tile<D>::CH; }
    __device__ __forceinline__ int chunk(int i) const { return Tile<D>::pos(row(i), lane % Tile<D>::CH); }
    // keys j0 .. (a multiple of ROWS), `last` the sequence's last (>= j0), which stands for those behind it
    template <typename T> __device__ __forceinline__ void issue(const T* base, const Pages<GROUPS>& pg, int j0, int last, unsigned lds) const {
        const uint64_t p = (uint64_t)base;
        const int in = (1 << shift) - 1;
        uint64_t b[GROUPS];
        b[0] = p + (uint64_t)(unsigned)pg.id[0] * sp + (uint64_t)(unsigned)(j0 & in) * st;
        if (in >= ROWS - 1) {                         // the tile is of one page
#pragma unroll
            for (int g = 1; g < GROUPS; g++) b[g] = b[g - 1] + 16 * (uint64_t)st;
        } else {                                      // it begins with a page
#pragma unroll
            for (int g = 1; g < GROUPS; g++) b[g] = p + (uint64_t)(unsigned)pg.id[g] * sp + (16 * g & in ? 16 * (uint64_t)st : 0);
        }
        if (last - j0 >= ROWS - 1) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                constexpr int S = RPL * NW / 16;
                uint64_t x = b[RPL * NW * i / 16];
                if constexpr (GPL == 2) x = w >= NW / 2 ? b[(S * i + 1) % GROUPS] : x;
                dma16b(x, off[i % VAR], lds + 1024u * (NW * i + w));
            }
        } else {
            const int gl = (last - j0) >> 4;          // the last key's group
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int gi = min(RPL * (NW * i + w) / 16, gl);
                uint64_t x = b[0];
#pragma unroll
                for (int g = 1; g < GROUPS; g++) x = gi == g ? b[g] : x;
                dma16b(x, (unsigned)(min(row(i), last - j0) - 16 * gi) * st + 16 * chunk(i), lds + 1024u * (NW * i + w));
            }
        }
    }
};

// The way through a unit's tiles from the first-th one on, NW tiles at a time
template <int STEP, int NW> struct Steps {
    int y, j, hi, at, gap;                            // y: j without the gap
    __host__ __device__ __forceinline__ void enter(const Reach<STEP>& x, int first) {
        y = x.lo + STEP * (first - NW);
        hi = x.hi;
        at = x.at;
        gap = x.gap;
    }
    __host__ __device__ __forceinline__ bool next() {
        y += STEP * NW;
        j = y + (y >= at ? gap : 0);
        return j < hi;
    }
};
// Keys of which rows at positions [p0, p1] see all: [f0, f1], and those up to f2.  Of any others they see some: [s0, s1], and those below s2.
struct Sight {
    int f0, f1, f2, s0, s1, s2;
    __device__ __forceinline__ Sight(const PagedArgs& a, const Seq& x, int p0, int p1) {
        f0 = max(0, p1 - a.W + 1);
        f1 = min(p0, x.klen - 1);
        f2 = p0 >= 0 ? min(x.pre, x.klen) - 1 : -1;
        s0 = max(0, p0 - a.W + 1);
        s1 = min(p1, x.klen - 1);
        s2 = p1 >= 0 ? min(x.pre, x.klen) : 0;
    }
    __device__ __forceinline__ bool all(int j0, int j1) const { return (j0 >= f0 && j1 <= f1) || j1 <= f2; }
    __device__ __forceinline__ bool some(int j0, int j1) const { return (j1 >= s0 && j0 <= s1) || j0 < s2; }
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
        for (int k0 = 0; k0 < 64; k0 += 16) {         // 16 loads on their way
            if (!(b >> k0 & 0xffff)) continue;
            T z[16][N];
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const T* r = vb + lane_of(ok ? id : 0, k0 + k) * a.v_sp + ((j0 + k0 + k) & in) * a.v_st + lane * N;
#pragma unroll
                for (int i = 0; i < N; i++) z[k][i] = r[i];
            }
#pragma unroll
            for (int k = 0; k < 16; k++) {
                const float y = lane_of(e, k0 + k);
#pragma unroll
                for (int i = 0; i < N; i++) o[i] = fmaf(y, b >> (k0 + k) & 1 ? widen1(z[k][i]) : 0.f, o[i]);
            }
        }
    }
}

// Whether the lane's row keeps its sums although they are not finite (slot_attn.h's keeps, the rows found through the table): it sees a value that is
// not, and no column holds one in a masked place only.  Keys [lo, hi); met(j): the wave multiplied key j; step: keys of a tile, whose last one may stand for
// those behind it; parts: probabilities in two parts make a NaN of an infinity that is seen, so that such a row is formed again.
template <typename T, int D, class MET>
__device__ __forceinline__ bool keeps_paged(const PagedArgs& a, const T* kb, const T* vb, const int32_t* tab, const Sees& see, int lo, int hi, int klen, int step, bool parts,
                                            int lane, MET met) {
    Ill<T, D> ill;
    const int in = (1 << a.shift) - 1, end = min(klen, lo + (hi - lo + step - 1) / step * step), last = klen % step ? klen - 1 : -1;
    for (int j0 = lo; j0 < end; j0 += 64) {
        const int j = j0 + lane, id = j < end ? tab[j >> a.shift] : -1;
        const bool there = (unsigned)id < (unsigned)a.P;
        const int64_t row = there ? id : 0;           // (a page that is not there: page 0 was multiplied in its place)
        const bool odd = j < end && !(finite_row<T, D>(kb + row * a.k_sp + (j & in) * a.k_st) && finite_row<T, D>(vb + row * a.v_sp + (j & in) * a.v_st));
        for (uint64_t b = __ballot(odd); b; b &= b - 1) {
            const int k = __builtin_ctzll(b), i = j0 + k;
            const T* z = vb + lane_of((int)row, k) * a.v_sp + (i & in) * a.v_st;
            const bool sees = i < hi && lane_of((int)there, k) && sees1(see, i, nullptr, 0);
            ill.add(z, sees, met(i), i == last, lane);
            if (parts)
#pragma unroll
                for (int e = 0; e < D / 64; e++) {
                    const uint64_t inf = __ballot(fabsf(widen1(z[lane * (D / 64) + e])) == INFINITY);
                    if (sees) ill.odd[e] |= inf;
                }
        }
    }
    return ill.kept();
}

// The end of a piece: a wave's 32 rows, a row a lane and half.  Whole units are normalised and written, others leave their sums at row
// `part` of the workspace.  Rows next to infinities and NaN are formed again, from their visible pairs among keys [lo, hi) alone.
struct Rows {
    int s, tok, hq, p, used;                          // the sequence's first token; the lane's token, query head and position; rows of the wave
    Sees see;
    float slope;
};
template <typename T, int D, bool CAP, bool BIAS, class MET>
__device__ __forceinline__ void finish(const PagedArgs& a, RowSums<T, D, BIAS>& sum, const Rows& w, const T* kb, const T* vb, const int32_t* tab, int lo, int hi,
                                       int klen, bool whole, int64_t part, int lane, MET met) {
    constexpr int DT = D / 32;
    const int h = lane >> 5;
    const bool in = (lane & 31) < w.used;
    sum.close();
    float nf = sum.l * 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) nf = nonfinite(sum.o[dt], nf);
    uint32_t odd = row_bits(nf != 0.f && sum.l == sum.l && in);      // (a NaN in its sum makes all of a row NaN)
    if (odd) odd &= ~row_bits(keeps_paged<T, D>(a, kb, vb, tab, w.see, lo, hi, klen, KT, false, lane, met));
    for (uint32_t b = odd; b; b &= b - 1) {
        const int i = __builtin_ctz(b);
        float m1, l1, o1[D / 64];
        exact_paged<T, D, CAP, BIAS>(a, (const T*)a.q + lane_of(w.hq, i) * a.q_sh + (int64_t)(w.s + lane_of(w.tok, i)) * a.q_st, kb, vb, tab,
                                     lane_of(w.see, i), lane_of(w.slope, i), lane_of(w.p, i), lo, hi, lane, m1, l1, o1);
        if (whole) {
            const float inv1 = l1 > 0.f || l1 != l1 ? 1.f / l1 : 0.f;
            for (int e = 0; e < D / 64; e++) o1[e] *= inv1;
            put_row<T, D>((T*)a.out + ((int64_t)(w.s + lane_of(w.tok, i)) * a.Hq + lane_of(w.hq, i)) * D, lane, o1);
        } else {
            for (int e = 0; e < D / 64; e++) a.po[(part + i) * D + lane * (D / 64) + e] = o1[e];
            if (lane == 0) a.pm[part + i] = make_float2(m1, l1);
        }
    }
    if (!in || bit(odd, lane & 31)) return;
    if (whole) {
        const int64_t at = ((int64_t)(w.s + w.tok) * a.Hq + w.hq) * D + 4 * h;
        const float inv = sum.l > 0.f || sum.l != sum.l ? 1.f / sum.l : 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                put4<T>(a.out, nullptr, at + 32 * dt + 8 * g, sum.o[dt][4 * g] * inv, sum.o[dt][4 * g + 1] * inv, sum.o[dt][4 * g + 2] * inv,
                        sum.o[dt][4 * g + 3] * inv);
    } else {
        float* po = a.po + (part + (lane & 31)) * D + 4 * h;
#pragma unroll
        for (int dt = 0; dt < DT; dt++)
#pragma unroll
            for (int g = 0; g < 4; g++)
                *reinterpret_cast<float4*>(po + 32 * dt + 8 * g) = make_float4(sum.o[dt][4 * g], sum.o[dt][4 * g + 1], sum.o[dt][4 * g + 2], sum.o[dt][4 * g + 3]);
        if (h == 0) a.pm[part + lane] = make_float2(sum.m, sum.l);
    }
}

// Zeros for the tokens of no row, by thread `i0` of `all`
template <int D> __device__ __forceinline__ void fill_rest(const PagedArgs& a, int64_t i0, int64_t all) {
    const int s0 = min(max(ld_uni(a.starts, 0), 0), a.N), s1 = min(max(ld_uni(a.starts, a.R), s0), a.N);
    const int64_t n = (int64_t)a.Hq * D / 8, n0 = s0 * n, n1 = n0 + (a.N - s1) * n;
    for (int64_t i = i0; i < n1; i += all) reinterpret_cast<uint4*>(a.out)[i < n0 ? i : i - n0 + s1 * n] = make_uint4(0, 0, 0, 0);
}

}  // namespace slotattn
