// What the kernels of the attention over pages share (slotattn_pages.hip, slotattn_few.hip).
//
// The query rows of a key/value head -- the tokens of a sequence times the query heads of the group -- are cut into tiles; a tile against the keys
// that it sees is a unit, and all units' key tiles in a row are shared out to the workers in equal contiguous pieces, so that neither
// ragged lengths nor causality leave a worker more than another.  A piece that is not a whole unit leaves its rows' maxima, sums and
// weighted values in the workspace, two such pieces a worker at most, and pages_join combines a unit's pieces in order.
#pragma once
#include "slot_attn_rows.h"
#include "slot_attn_host.h"

namespace slotattn {

// What is left for the join.  pages_many: of each worker, the unit that begins in it and goes on in the next (row, head, tile, tokens, pieces; 0: none).
// pages_few: of each unit, the worker in which it begins and its pieces, at ((s rep) / 32 + row + tile) Hk + head, s its sequence's first token:
// a place of its own for every tile of the batch.
struct Unit { int r, hk, t, n, parts; };
struct Piece { int me, parts; };

struct PagedArgs {
    AttnArgs s;                                       // the scores' constants
    const void* q; const void* k; const void* v;
    int64_t q_sh, q_st, k_sp, k_sh, k_st, v_sp, v_sh, v_st;
    const int32_t* table; int64_t t_sr;
    const int32_t* starts; const int32_t* ends; const int32_t* prefix; const float* slopes;
    int N, R, M, P, Hq, Hk, rep, W, shift, units;     // units: room for them in the plan
    int* plan;                                        // running costs of the rows (R + 1), first units of the rows (R + 1), running costs (units + 1)
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
__device__ __forceinline__ Seq make_seq(const PagedArgs& a, int s0, int s1, int end, int pre) {
    Seq x;
    x.s = min(max(s0, 0), a.N);
    x.n = min(max(s1, x.s), a.N) - x.s;
    x.end = min(max(end, 0), (1 << 30) - 1);
    x.klen = min(x.end, a.M << a.shift);
    x.pre = pre;
    return x;
}
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int r) {                       // a row of the lane's
    return make_seq(a, a.starts[r], a.starts[r + 1], a.ends[r], a.prefix ? a.prefix[r] : 0);
}
__device__ __forceinline__ Seq seq_uni(const PagedArgs& a, int r) {                      // a row of the wave's
    return make_seq(a, ld_uni(a.starts, r), ld_uni(a.starts, r + 1), ld_uni(a.ends, r), a.prefix ? ld_uni(a.prefix, r) : 0);
}
// Keys that positions [p0, p1] see lie in [lo, hi), lo a multiple of STEP
template <int STEP> __device__ __forceinline__ void keys_of(const PagedArgs& a, const Seq& x, int p0, int p1, int& lo, int& hi) {
    lo = x.pre > 0 ? 0 : max(0, max(p0, 0) - a.W + 1) & ~(STEP - 1);
    hi = p1 < 0 ? lo : min(x.klen, max(p1 + 1, x.pre));
}

// Equal shares of `total` tiles for G workers: worker w has those from begin(w) on.
struct Shares {
    int G, q, rem;
    __device__ __forceinline__ Shares(int total, int workers) : G(workers), q(total / workers), rem(total - q * workers) {}
    __device__ __forceinline__ int begin(int w) const { return w * q + min(w, rem); }
    __device__ __forceinline__ int owner(int x) const {               // of tile x
        const int big = rem * (q + 1);
        return x < big ? x / (q + 1) : rem + (x - big) / q;
    }
};

// The pages of a tile's groups of 16 keys from j0 on.  A number outside of the pool stands for page 0, and its group's bit says that its keys are
// not seen; a group behind the sequence's last key has that key's page.
template <int GROUPS> struct Pages {
    int id[GROUPS];
    uint32_t lost;
    __device__ __forceinline__ void fetch(const PagedArgs& a, int64_t row, int j0, int klen) {
        lost = 0;
#pragma unroll
        for (int g = 0; g < GROUPS; g++) {
            id[g] = ld_uni(a.table, row + (min(j0 + 16 * g, klen - 1) >> a.shift));
            if ((unsigned)id[g] >= (unsigned)a.P) {
                id[g] = 0;
                lost |= 1u << g;
            }
        }
    }
};

// One direct load as dma16s's, whose base is in scalar registers already
template <typename T> __device__ __forceinline__ const T* scalar_ptr(const T* x) {
    const uint64_t p = (uint64_t)x;
    return (const T*)(((uint64_t)(unsigned)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)p));
}
__device__ __forceinline__ void dma16b(const void* base, unsigned off, unsigned lds) {
    // five wait states for a base that the vector unit has just written
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "{m0}"(lds), "v"(off), "s"(base) : "memory");
}
// Direct loads of a tile of ROWS keys by wave w of NW, laid out as TileLoad's.  A group of 16 keys is of one page: its base is formed once, and a
// lane's offsets within a group are held in registers.
template <int D, int ROWS, int NW> struct PageLoad {
    static constexpr int N = ROWS * 2 * D / 1024 / NW, RPL = 512 / D;  // loads per wave, rows per load
    static constexpr int VAR = RPL * NW >= 16 ? 1 : 16 / (RPL * NW);  // loads of one group
    static_assert(NW == 1 || VAR == 1, "one load a group, or all of them");
    unsigned off[VAR];
    int64_t sp, st;
    int w, lane, in;                                  // in: rows of a page, less one
    __device__ __forceinline__ PageLoad(int64_t page_stride, int64_t stride, int shift, int wave, int l)
        : sp(page_stride), st(stride), w(wave), lane(l), in((1 << shift) - 1) {
#pragma unroll
        for (int i = 0; i < VAR; i++) off[i] = (unsigned)((RPL * (NW * i + w) & 15) + lane / Tile<D>::CH) * (unsigned)(2 * st) + 16 * chunk(i);
    }
    __device__ __forceinline__ int row(int i) const { return RPL * (NW * i + w) + lane / Tile<D>::CH; }
    __device__ __forceinline__ int chunk(int i) const { return Tile<D>::pos(row(i), lane % Tile<D>::CH); }
    // keys j0 .. (a multiple of 32), `last` the sequence's last (>= j0), which stands for those behind it
    template <typename T> __device__ __forceinline__ void issue(const T* base, const Pages<ROWS / 16>& pg, int j0, int last, unsigned lds) const {
        if (last - j0 >= ROWS - 1) {
            const T* p = nullptr;
#pragma unroll
            for (int i = 0; i < N; i++) {
                if (i % VAR == 0) {
                    const int g = RPL * (NW * i + w) / 16;
                    int id = pg.id[RPL * NW * i / 16];
                    if constexpr (RPL * NW > 16) id = g & 1 ? pg.id[(RPL * NW * i / 16 + 1) % (ROWS / 16)] : id;     // (a load a wave over two groups)
                    p = scalar_ptr(base + id * sp + ((j0 + 16 * g) & in) * st);
                }
                dma16b(p, off[i % VAR], lds + 1024u * (NW * i + w));
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const int g = RPL * (NW * i + w) / 16;
                int id = pg.id[RPL * NW * i / 16];
                if constexpr (RPL * NW > 16) id = g & 1 ? pg.id[(RPL * NW * i / 16 + 1) % (ROWS / 16)] : id;
                const int j = min(j0 + row(i), last);
                dma16(base + id * sp + (j & in) * st + 8 * chunk(i), lds + 1024u * (NW * i + w));
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

// The end of a piece: a wave's 32 rows, a row a lane and half.  Whole units are normalised and written, others leave their sums at row
// `part` of the workspace.  Rows next to infinities and NaN are formed again, from their visible pairs among keys [lo, hi) alone.
struct Rows {
    int s, tok, hq, p, used;                          // the sequence's first token; the lane's token, query head and position; rows of the wave
    Sees see;
    float slope;
};
template <typename T, int D, bool CAP, bool BIAS>
__device__ __forceinline__ void finish(const PagedArgs& a, RowSums<T, D, BIAS>& sum, const Rows& w, const T* kb, const T* vb, const int32_t* tab, int lo, int hi,
                                       bool whole, int64_t part, int lane) {
    constexpr int DT = D / 32;
    const int h = lane >> 5;
    const bool in = (lane & 31) < w.used;
    sum.close();
    float nf = sum.l * 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; dt++) nf = nonfinite(sum.o[dt], nf);
    const uint32_t odd = row_bits(nf != 0.f && sum.l == sum.l && in);
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
