// Device helpers shared by the attention kernels, forward (slotattn.hip) and backward (slotattn_bwd.hip).
//
// Operands of v_mfma_f32_32x32x16 (16-bit inputs): lane l holds 8 consecutive k values 8 (l >> 5) .. + 7 of row (A) or
// column (B) l & 31; register r of the result holds row 8 (r >> 2) + 4 (l >> 5) + (r & 3) of column l & 31.  So a score
// tile with the keys as rows has one query per lane, and its registers 8 m .. 8 m + 7, rounded to 16 bits, are the B
// operand of the next product over the same 16 keys -- in the order 16 m + 4 h + {0..3}, 16 m + 8 + 4 h + {0..3} for
// the lane half h -- when the A operand names its keys in that order too: two transposing LDS reads of 4 keys each.
#pragma once
#include "slot_common.h"

namespace slotattn {

using namespace slot;

typedef _Float16 f16_t;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;

#define LOG2E 1.4426950408889634f
// tanh(x) / x on [0, 3/4] as a polynomial in x^2, fitted for the smallest largest relative error
#define TANH0 0.99999943f
#define TANH1 -0.33328252f
#define TANH2 0.13258983f
#define TANH3 -0.05005631f
#define TANH4 0.01292964f
#define KT 64                                        // keys (or query rows) of a staged tile

template <typename T> __device__ __forceinline__ f32x16 mfma32(const uint4& a, const uint4& b, f32x16 c);
template <> __device__ __forceinline__ f32x16 mfma32<bf16_t>(const uint4& a, const uint4& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x16 mfma32<f16_t>(const uint4& a, const uint4& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
template <typename T> __device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack2<bf16_t>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <> __device__ __forceinline__ uint32_t pack2<f16_t>(float lo, float hi) {
    const f16x2 x = {(f16_t)lo, (f16_t)hi};          // round to nearest even
    return __builtin_bit_cast(uint32_t, x);
}
// a result tile's registers 8 m .. 8 m + 7 as one operand
template <typename T> __device__ __forceinline__ uint4 pack8(const f32x16& s, int m) {
    return make_uint4(pack2<T>(s[8 * m], s[8 * m + 1]), pack2<T>(s[8 * m + 2], s[8 * m + 3]), pack2<T>(s[8 * m + 4], s[8 * m + 5]),
                      pack2<T>(s[8 * m + 6], s[8 * m + 7]));
}
__device__ __forceinline__ uint4 ld16(const void* p) { return *reinterpret_cast<const uint4*>(p); }
__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int r = 0; r < 16; r++) z[r] = 0.f;
    return z;
}
// the other half's value (lanes l and l ^ 32), combined
__device__ __forceinline__ float half_max(float v) {
    auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float half_sum(float v) {
    auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// wait until at most n of this wave's vector-memory operations are outstanding.  The direct loads into LDS are not
// tracked by the compiler; every other vector-memory operation of a wave is younger or tracked, so it can only make
// these waits longer, never shorter.
template <int n> __device__ __forceinline__ void wait_vm() {
    static_assert(n >= 0 && n < 64, "vmcnt is 6 bits");
    __builtin_amdgcn_s_waitcnt(0x0F70 | (n & 15) | ((n >> 4) << 14));
}
// workgroup barrier behind this wave's LDS accesses; it adds no wait for direct loads in flight
__device__ __forceinline__ void tile_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// A staged tile: rows of D 16-bit values, the 16-byte chunk c of row r at chunk c ^ swz(r).  The 64 banks are 256 bytes wide,
// a row operand read serves 16 consecutive rows at one chunk at a time, a transposing read 4 rows (4 a .. 4 a + 3) at 4
// chunks: swz gives the first 16 different places in the banks and the second 4 different groups of 4 (row bits 0, 1 --
// those that the banks do not see already -- are its high bits, the next two its low ones).  With the row number itself in the place of swz
// every read took twice its cycles.
template <int D> struct Tile {
    static constexpr int CH = D / 8, ROWB = 2 * D;
    static __device__ __forceinline__ int swz(int r) { return D == 128 ? ((r & 3) << 2) | ((r >> 2) & 3) : ((r & 2) << 1) | ((r >> 2) & 3); }
    static __device__ __forceinline__ int pos(int r, int c) { return c ^ swz(r); }
};

// A lane's operand addresses in a staged tile, as LDS byte addresses: every k step or column block is the same address with
// a few bits flipped, every 16 rows a constant further, so a lane holds three of them.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) const u32x4 lds_u4;
typedef __attribute__((address_space(3))) const f32x4 lds_f4;
__device__ __forceinline__ uint4 lds16(unsigned a) { return __builtin_bit_cast(uint4, *(lds_u4*)(uintptr_t)a); }
__device__ __forceinline__ f32x4 lds4f(unsigned a) { return *(lds_f4*)(uintptr_t)a; }
__device__ __forceinline__ uint2 lds_tr(unsigned a) {
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)(uintptr_t)a));
}
template <int D> struct Ops {
    typedef Tile<D> Ti;
    unsigned row, col, col8;                         // relative to a tile's start (1 KB aligned); col8: 8 rows further
    __device__ __forceinline__ Ops(int lane) {
        const int l = lane & 31, h = lane >> 5, i = lane & 15, cr = 4 * h + (i >> 2);
        row = l * Ti::ROWB + 16 * Ti::pos(l, h);
        const int c = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), by = 8 * (lane & 1);
        col = cr * Ti::ROWB + 16 * Ti::pos(cr, c) + by;
        col8 = (cr + 8) * Ti::ROWB + 16 * Ti::pos(cr + 8, c) + by;
    }
    // A tile's operands, from a lane's address of one of the three kinds plus the tile's start (1 KB aligned): tiles a
    // constant apart share the flipped address, the rest is the instruction's offset.
    // row operand of k step kk: values 16 kk + 8 h .. + 7 of row l & 31, `at` bytes further
    static __device__ __forceinline__ unsigned k_step(unsigned row, int kk) { return row ^ (32 * kk); }
    static __device__ __forceinline__ unsigned block(unsigned col, int dt) { return col ^ (64 * dt); }
    // operand over rows r + 16 m + 4 h .. + 3 and + 8 (a result tile's order) of a column block: block() of col and col8
    static __device__ __forceinline__ uint4 at_col(unsigned c, unsigned c8, int at) {
        const uint2 lo = lds_tr(c + at), hi = lds_tr(c8 + at);
        return make_uint4(lo.x, lo.y, hi.x, hi.y);
    }
};

// One direct global -> LDS load as dma16's, the address a wave-uniform base plus a lane's 32-bit offset in bytes.
__device__ __forceinline__ void dma16s(const void* base, unsigned off, unsigned lds) {
    const uint64_t p = (uint64_t)base;               // the compiler does not always see that it is one value for the wave
    base = (const void*)(((uint64_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)p));
    // five wait states: readfirstlane writes the base from the vector unit, and the hazard before a memory instruction that
    // reads it is not the compiler's inside of an asm block
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %1, %2" : : "{m0}"(lds), "v"(off), "s"(base) : "memory");
}
// One direct global -> LDS load of 4 bytes per lane from g into LDS at lds + 4 * lane.
__device__ __forceinline__ void dma4(const void* g, unsigned lds) {
    asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" : : "{m0}"(lds), "v"(g) : "memory");
}
// Direct loads of a tile of ROWS rows by wave w of NW.  Load i fills 1 KB: RPL rows from row RPL (NW i + w) on.  A lane's offset
// is formed once (the swizzle repeats every 16 rows: VAR of them), the loads' bases are scalars: with an address per
// lane and load the multiplications took 500 of a tile's 3,500 cycles.  Rows past the tensor's last repeat it: what they hold
// never counts (their scores are masked), and nothing outside the tensor is read.
template <int D, int ROWS, int NW> struct TileLoad {
    static constexpr int N = ROWS * 2 * D / 1024 / NW, RPL = 512 / D;  // loads per wave, rows per load
    static constexpr int VAR = RPL * NW >= 16 ? 1 : 16 / (RPL * NW);
    static_assert(ROWS * 2 * D % (1024 * NW) == 0, "whole loads");
    unsigned off[VAR];
    int64_t st;
    int w, lane;
    __device__ __forceinline__ TileLoad(int64_t stride, int wave, int l) : st(stride), w(wave), lane(l) {
#pragma unroll
        for (int i = 0; i < VAR; i++) off[i] = (unsigned)(RPL * w + lane / Tile<D>::CH) * (unsigned)(2 * st) + 16 * chunk(i);
    }
    __device__ __forceinline__ int row(int i) const { return RPL * (NW * i + w) + lane / Tile<D>::CH; }
    __device__ __forceinline__ int chunk(int i) const { return Tile<D>::pos(row(i), lane % Tile<D>::CH); }
    // rows r0 .. of `base`, `last` the tensor's last row (>= r0)
    template <typename T> __device__ __forceinline__ void issue(const T* base, int r0, int last, unsigned lds) const {
        base += r0 * st;
        if (last - r0 >= ROWS - 1) {
#pragma unroll
            for (int i = 0; i < N; i++) dma16s(base + i * (RPL * NW) * st, off[i % VAR], lds + 1024u * (NW * i + w));
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) dma16(base + min(row(i), last - r0) * st + 8 * chunk(i), lds + 1024u * (NW * i + w));
        }
    }
};

// The keys of a tile [j0, j1] that queries of positions [p0, p1] see: none, some or all of the pairs.
struct Span { int p0, p1, lo, hi; bool one; };       // positions; documents: range of ids, all of one document
struct Mask {
    int causal, W, prefix, klen;
    __device__ __forceinline__ bool some(const Span& s, int j0, int j1) const {
        // the closest pair's distance, p - j
        const bool b = causal ? (j0 <= s.p1 && s.p0 - j1 < W) : (s.p0 - j1 < W && j0 - s.p1 < W);
        return (b || j0 < prefix) && j0 < klen;
    }
    __device__ __forceinline__ bool all(const Span& s, int j0, int j1) const {
        const bool b = causal ? (j1 <= s.p0 && s.p1 - j0 < W) : (s.p1 - j0 < W && j1 - s.p0 < W);
        return (b || (j1 < prefix && s.p0 >= 0)) && j1 < klen;
    }
};

struct AttnArgs {
    const void* q; const void* k; const void* v;
    int64_t q_sb, q_sh, q_st, k_sb, k_sh, k_st, v_sb, v_sh, v_st;
    int B, Tq, Tk, Hq, Hk, R;                        // R = Hq / Hk
    int causal, W;
    const float* slopes;
    const int32_t* ids; const int2* range; int ntd;  // documents: padded ids (B, 64 ntd), ranges (B, ntd)
    const int32_t* prefix; const int32_t* lens;
    float f;                                         // what makes scores() base 2: scale log2(e), or cap log2(e)
    float kc, ct;                                    // capped: scale / cap, and 2 log2(e) of it
    int mix;                                         // a cap so far above that small scores need a form of their own
    float lim, t0, t1, t2, t3, t4;                   // the polynomial's limit and coefficients, for products <q, k>
    void* out; void* res; float* lse;                // res: what rounding took from out, for the backward's delta
    // split rows
    float* po; float* pm; int chunk, nsplit, tiles, groups;
    // backward
    const void* dout; int64_t do_sb, do_sh, do_st;
    float* delta; void* dq; void* dk; void* dv;
    float* part; int units; float scale;             // split keys of attn_dkv: partial sums, query tiles per workgroup
};

// a float4 of results and what rounding takes from it
template <typename T> __device__ __forceinline__ float unpack(uint32_t x, int i);
template <> __device__ __forceinline__ float unpack<bf16_t>(uint32_t x, int i) { return __uint_as_float(i ? x & 0xffff0000u : x << 16); }
template <> __device__ __forceinline__ float unpack<f16_t>(uint32_t x, int i) { return (float)__builtin_bit_cast(f16x2, x)[i]; }
template <typename T> __device__ __forceinline__ void put4(void* out, void* res, int64_t at, float x, float y, float z, float w) {
    const uint2 o = make_uint2(pack2<T>(x, y), pack2<T>(z, w));
    *reinterpret_cast<uint2*>((T*)out + at) = o;
    if (res) *reinterpret_cast<uint2*>((T*)res + at) =
        make_uint2(pack2<T>(x - unpack<T>(o.x, 0), y - unpack<T>(o.x, 1)), pack2<T>(z - unpack<T>(o.y, 0), w - unpack<T>(o.y, 1)));
}

// key of register r of a score tile's lane half h, from the tile's first key
__device__ __forceinline__ constexpr int key_of(int r, int h) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// The products s of a 32 x 32 tile become scores up to the factor() that makes them base 2: as they are, or tanh(x), x = kc s, where
// they are capped.  tanh(x) is x times a polynomial in x^2 while |x| <= 3/4 (relative error 7e-7; 6 instructions, none of them a
// transcendental one), which the scores of a whole tile usually are, else 1 - 2 / (1 + e^2x).  That is off by a few 2^-24 of 1, not
// of itself, and a score is cap tanh(x): up to a cap of 64 less than 2^-16, but 0.1 at 1e6.  Above 64 each x takes the form that is exact for it
// (8,192 tokens, forward, tiles that all hold scores past the cap: 371 us against 281 by the exponential form alone); the polynomial
// with x formed first, as the powers of a small kc in the shorter one's coefficients would leave 32 bits.
__device__ __forceinline__ float tanh_poly(float s, const AttnArgs& a) {
    const float y = s * s;
    return s * fmaf(fmaf(fmaf(fmaf(a.t4, y, a.t3), y, a.t2), y, a.t1), y, a.t0);
}
__device__ __forceinline__ float tanh_exp(float s, const AttnArgs& a) { return fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + exp2_(s * a.ct)), 1.f); }
__device__ __forceinline__ float tanh_mix(float s, const AttnArgs& a) {
    const float x = s * a.kc, y = x * x, t = fmaf(-2.f, __builtin_amdgcn_rcpf(1.f + exp2_(x * (2.f * LOG2E))), 1.f);
    return fabsf(x) <= 0.75f ? x * fmaf(fmaf(fmaf(fmaf(TANH4, y, TANH3), y, TANH2), y, TANH1), y, TANH0) : t;
}
__device__ __forceinline__ bool poly_holds(const f32x16& s, const AttnArgs& a) {
    float m = 0.f;
#pragma unroll
    for (int r = 0; r < 16; r++) m = fmaxf(m, fabsf(s[r]));
    return __all(m <= a.lim);
}
template <bool CAP> __device__ __forceinline__ void scores(f32x16& s, const AttnArgs& a) {
    if constexpr (CAP) {
        if (poly_holds(s, a)) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = tanh_poly(s[r], a);
        } else if (a.mix) {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = tanh_mix(s[r], a);
        } else {
#pragma unroll
            for (int r = 0; r < 16; r++) s[r] = tanh_exp(s[r], a);
        }
    }
}
// Scores in base 2, less slope (in base 2) x distance: the lane's own position p against rows j0 + key_of(r, h); their
// factor is 1 from here on
__device__ __forceinline__ void bias(f32x16& s, float f, float slope, int p, int j0, int h) {
    const float d = (float)(p - j0 - 4 * h);
#pragma unroll
    for (int r = 0; r < 16; r++) s[r] = fmaf(-slope, fabsf(d - (float)key_of(r, 0)), s[r] * f);
}

// A value that is the same in every lane, in a scalar register.  (Loads behind the asm blocks' memory clobbers go through
// vector registers, and what is computed from them -- a tile's base address -- would stay there.)
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
// Tokens of sequence b that count, and its length that positions are taken from (a length past the keys keeps its positions).
__device__ __forceinline__ int length_of(const AttnArgs& a, int b) { return uni(a.lens ? min(max(a.lens[b], 0), (1 << 30) - 1) : a.Tk); }
__device__ __forceinline__ int prefix_of(const AttnArgs& a, int b) { return uni(a.prefix ? a.prefix[b] : 0); }

// range of the ids of a document tile as slotattn_docs leaves it: x = smallest (bit 31: some are padding), y = largest
__device__ __forceinline__ int range_lo(int2 r) { return r.x & 0x7fffffff; }
__device__ __forceinline__ bool range_one(int2 r) { return r.x == r.y; }
// The ids of positions [s.p0, s.p1] (at most 128 of them), from the ranges of the 64-id tiles that they touch: wider than
// they are where they fill no whole tile.
__device__ __forceinline__ void doc_span(const int2* range, Span& s) {
    const int x0 = uni(s.p0 / KT), x1 = uni(max(s.p0, s.p1) / KT);
    int lo = 0x7fffffff, hi = -2;
    bool one = true;
#pragma unroll
    for (int i = 0; i < 3; i++) {
        const int2 r = range[min(x0 + i, x1)];
        lo = min(lo, range_lo(r));
        hi = max(hi, r.y);
        one = one && range_one(r);
    }
    s.lo = uni(lo);
    s.hi = uni(hi);
    s.one = uni((int)(one && lo == hi));
}
// What one lane sees of the other side's rows: those with i - first <= count (unsigned), first + count inclusive; and, for a
// query that a prefix reaches behind the band, those below `below`.
struct Sees {
    unsigned first, count, below;
    // a query at position p (negative: sees nothing), against keys
    static __device__ __forceinline__ Sees query(const Mask& m, int p) {
        int lo = p - m.W + 1, hi = min(m.causal ? p : p + m.W - 1, m.klen - 1);
        int b = p >= 0 ? min(m.prefix, m.klen) : 0;
        if (lo <= b && b > 0) {                       // one interval
            lo = 0;
            hi = max(hi, b - 1);
            b = 0;
        }
        lo = max(lo, 0);
        if (hi < lo || p < 0) { lo = 0x7fffffff; hi = lo; }
        return {(unsigned)lo, (unsigned)(hi - lo), (unsigned)max(b, 0)};
    }
    // a key at position j, against queries of positions up to `last`
    static __device__ __forceinline__ Sees key(const Mask& m, int j, int last) {
        int lo = m.causal ? j : j - m.W + 1, hi = min(j + m.W - 1, last);
        if (j < m.prefix) { lo = 0; hi = last; }
        lo = max(lo, 0);
        if (hi < lo) { lo = 0x7fffffff; hi = lo; }
        return {(unsigned)lo, (unsigned)(hi - lo), 0u};
    }
};
// The 16 rows of a result tile from row j0 on (rows j0 + key_of(r, h)) that a lane sees, as bits: by its interval, by the prefix
// where a lane's does not join it (pre), by the document ids (at ids + 8 g + 4 h; null: none)
__device__ __forceinline__ uint32_t seen16(const Sees& v, int j0, int h, bool pre, const int* ids, int id) {
    unsigned x = (unsigned)(j0 + 4 * h) - v.first;
    const unsigned y = (unsigned)(j0 + 4 * h);
    asm volatile("" : "+v"(x));                       // only where it is asked for: not computed ahead of the branch around it
    uint32_t m = 0;
#pragma unroll
    for (int r = 0; r < 16; r++) m |= (x + key_of(r, 0) <= v.count ? 1u : 0u) << r;
    if (pre) {
#pragma unroll
        for (int r = 0; r < 16; r++) m |= (y + key_of(r, 0) < v.below ? 1u : 0u) << r;
    }
    if (ids) {
#pragma unroll
        for (int g = 0; g < 4; g++) {
            const int4 d = *reinterpret_cast<const int4*>(ids + 8 * g + 4 * h);
            m &= ~(((d.x != id ? 1u : 0u) | (d.y != id ? 2u : 0u) | (d.z != id ? 4u : 0u) | (d.w != id ? 8u : 0u)) << (4 * g));
        }
    }
    return m;
}
__device__ __forceinline__ bool bit(uint32_t m, int r) { return (m >> r & 1) != 0; }

// ---- rows next to infinities and NaN -----------------------------------------------------------------------
// A masked pair has the weight 0 in its product, and 0 times an infinity or a NaN of the other operand is a NaN.  So a row whose
// sums come out so is formed again by its wave, one row at a time, from its visible pairs alone, unless it sees a value that is not
// finite and the sums are what that makes of them: no column holds such a value in a masked place only (Ill).  Where all is finite that
// costs the tests, about 1 instruction per value of the accumulators.  8,192 tokens, 12 heads, forward (0.23 ms): a value that every row
// sees costs each wave one pass over the keys, 2.0 ms, and 6.5 ms where every value is NaN; one next to a tile's finite rows costs
// these rows one by one (the last token's value: 127 rows a head, 28 ms).
__device__ __forceinline__ float nonfinite(const f32x16& x, float t) {            // t + 0 if all of x is finite, else NaN
#pragma unroll
    for (int r = 0; r < 16; r++) t = fmaf(x[r], 0.f, t);
    return t;
}
__device__ __forceinline__ int lane_of(int x, int i) { return __builtin_amdgcn_readlane(x, i); }
__device__ __forceinline__ float lane_of(float x, int i) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), i)); }
__device__ __forceinline__ Sees lane_of(const Sees& v, int i) {
    return {(unsigned)lane_of((int)v.first, i), (unsigned)lane_of((int)v.count, i), (unsigned)lane_of((int)v.below, i)};
}
__device__ __forceinline__ float widen1(bf16_t x) { return bf2f(x); }
__device__ __forceinline__ float widen1(f16_t x) { return (float)x; }
template <typename T, int D> __device__ __forceinline__ float dot_row(const T* x, const T* y) {
    float s = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; c++) {
        const uint4 u = ld16(x + 8 * c), v = ld16(y + 8 * c);
        const uint32_t us[4] = {u.x, u.y, u.z, u.w}, vs[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 8; i++) s = fmaf(unpack<T>(us[i / 2], i & 1), unpack<T>(vs[i / 2], i & 1), s);
    }
    return s;
}
template <typename T, int D> __device__ __forceinline__ bool finite_row(const T* x) {
    float t = 0.f;
#pragma unroll 4
    for (int c = 0; c < D / 8; c++) {
        const uint4 u = ld16(x + 8 * c);
        const uint32_t us[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 8; i++) t = fmaf(unpack<T>(us[i / 2], i & 1), 0.f, t);
    }
    return t == 0.f;
}
// o += sum over the rows k of m, at most n of them, of lane k's w times the row; values D / 64 lane .. of it per lane
template <typename T, int D> __device__ __forceinline__ void add_rows(float (&o)[D / 64], float w, uint64_t m, const T* rows, int64_t st, int n, int lane) {
    constexpr int N = D / 64;
    for (int k0 = 0; k0 < 64; k0 += 16) {             // 16 loads on their way
        T x[16][N];
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const T* r = rows + min(k0 + k, n - 1) * st + lane * N;
#pragma unroll
            for (int i = 0; i < N; i++) x[k][i] = r[i];
        }
#pragma unroll
        for (int k = 0; k < 16; k++) {
            const float y = lane_of(w, k0 + k);
#pragma unroll
            for (int i = 0; i < N; i++) o[i] = fmaf(y, m >> (k0 + k) & 1 ? widen1(x[k][i]) : 0.f, o[i]);
        }
    }
}
// the score of one pair in base 2, and the slope of the cap
template <bool CAP, bool BIAS> __device__ __forceinline__ float score1(float x, const AttnArgs& a, float slope, int dist, float& tang) {
    tang = 1.f;
    if constexpr (CAP) {
        x = fabsf(x) <= a.lim ? tanh_poly(x, a) : a.mix ? tanh_mix(x, a) : tanh_exp(x, a);
        tang = fmaf(-x, x, 1.f);
    }
    x *= a.f;
    if constexpr (BIAS) x = fmaf(-slope, fabsf((float)dist), x);
    return x;
}
__device__ __forceinline__ bool sees1(const Sees& v, int j, const int* ids, int id) {
    return ((unsigned)j - v.first <= v.count || (unsigned)j < v.below) && (!ids || ids[j] == id);
}
// What became of the lane's row where rows of the other side are not finite: whether it sees one, and, as bits over the columns that
// are summed (lane D / 64 .. of them per lane), where one that it sees holds a NaN and where one met under a mask alone holds anything not finite.
template <typename T, int D> struct Ill {
    static constexpr int N = D / 64;
    bool hit = false, lost = false;                   // lost: every column is NaN by what the row sees
    uint64_t nan[N] = {}, odd[N] = {};
    // row z (of the wave) of the summed operand.  met: its tile was multiplied; copies: and holds it again behind the last row
    __device__ __forceinline__ void add(const T* z, bool sees, bool met, bool copies, int lane) {
        hit = hit || sees;
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float x = widen1(z[lane * N + i]);
            const uint64_t n = __ballot(x != x), o = __ballot(!(fabsf(x) < INFINITY));
            if (sees) nan[i] |= n;
            if (met && (copies || !sees)) odd[i] |= o;
        }
    }
    // the sums are those of the visible pairs as they are
    __device__ __forceinline__ bool kept() const {
        uint64_t x = 0;
#pragma unroll
        for (int i = 0; i < N; i++) x |= odd[i] & ~nan[i];
        return lost || (hit && x == 0);
    }
};
// The same for keys [lo, hi), whose two rows both count, in steps of 64: sees(j) for the lane's row, met(j) for the wave, j a key of the step.
template <typename T, int D, class SEES, class MET>
__device__ __forceinline__ bool keeps(const T* kb, int64_t k_st, const T* vb, int64_t v_st, const T* zb, int64_t z_st, int lo, int hi, int last, int lane,
                                      SEES sees, MET met) {
    Ill<T, D> ill;
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        for (uint64_t b = __ballot(j < hi && !(finite_row<T, D>(kb + j * k_st) && finite_row<T, D>(vb + j * v_st))); b; b &= b - 1) {
            const int i = j0 + __builtin_ctzll(b);
            ill.add(zb + i * z_st, sees(i), met(i), i == last, lane);
        }
    }
    return ill.kept();
}
// rows of the wave (lanes l and l + 32 have row l) for which x holds, as bits
__device__ __forceinline__ uint32_t row_bits(bool x) {
    const uint64_t b = __ballot(x);
    return (uint32_t)(b | b >> 32);
}
// One query's softmax over keys [lo, hi): maximum, sum and unnormalised output, values lane D / 64 .. of it per lane
template <typename T, int D, bool CAP, bool BIAS>
__device__ __forceinline__ void exact_row(const AttnArgs& a, const T* q, const T* kb, const T* vb, const Sees& v, const int* ids, int id, float slope,
                                          int p, int lo, int hi, int lane, float& m, float& l, float (&o)[D / 64]) {
    m = -INFINITY;
    l = 0.f;
    for (int i = 0; i < D / 64; i++) o[i] = 0.f;
    for (int j0 = lo; j0 < hi; j0 += 64) {
        const int j = j0 + lane;
        const bool ok = j < hi && sees1(v, j, ids, id);
        const uint64_t b = __ballot(ok);
        if (!b) continue;
        float x = -INFINITY, tang;
        if (ok) x = score1<CAP, BIAS>(dot_row<T, D>(q, kb + j * a.k_st), a, slope, p - j, tang);
        float mx = x;
        for (int i = 1; i < 64; i <<= 1) mx = fmaxf(mx, __shfl_xor(mx, i));
        const float mn = fmaxf(m, mx), mu = mn == -INFINITY ? 0.f : mn, f = m == -INFINITY ? 0.f : exp2_(m - mn);
        const float e = ok ? exp2_(x - mu) : 0.f;
        m = mn;
        l = l * f + wavesum(e);
        for (int i = 0; i < D / 64; i++) o[i] *= f;
        if (l != l) {                                 // its own query, or an overflow
            for (int i = 0; i < D / 64; i++) o[i] = NAN;
            return;
        }
        add_rows<T, D>(o, e, b, vb + j0 * a.v_st, a.v_st, hi - j0, lane);
    }
}
template <typename T, int D> __device__ __forceinline__ void put_row(T* out, int lane, const float (&o)[D / 64]) {
    if constexpr (D == 128) *reinterpret_cast<uint32_t*>(out + 2 * lane) = pack2<T>(o[0], o[1]);
    else *reinterpret_cast<uint16_t*>(out + lane) = (uint16_t)pack2<T>(o[0], 0.f);
}

// The walk over the 64-key tiles that a workgroup's queries see.  Each lane tests one of 64 tiles at a time; what a
// workgroup visits, a wave computes and a wave computes without masks are three ballots.
struct Walk {
    const Mask& mk;
    const Span& sw; const Span& sv;                  // positions of the workgroup's queries and of the wave's
    const int2* range;                               // documents of this sequence, or null
    int nt, base, lane;
    uint64_t act = 0, mine = 0, full = 0;
    __device__ __forceinline__ Walk(const Mask& m, const Span& w, const Span& v, const int2* r, int l) : mk(m), sw(w), sv(v), range(r), lane(l) {
        // up to the band's or the prefix' end, from the band's start where there is no prefix
        const int end = mk.causal ? min(mk.klen, max(sw.p1 + 1, mk.prefix)) : mk.klen;
        nt = (end + KT - 1) / KT;
        base = (mk.prefix > 0 ? 0 : (max(0, max(sw.p0, 0) - mk.W + 1) / KT) & ~63) - 64;
    }
    // whether the wave computes tile x (of the wave)
    __device__ __forceinline__ bool computes(int x) const {
        const int j0 = x * KT;
        if (!(sv.p0 <= sv.p1 && mk.some(sv, j0, j0 + KT - 1))) return false;
        return !range || (range_lo(range[x]) <= sv.hi && sv.lo <= range[x].y);
    }
    // the next visible tile (-1: none), whether this wave's rows see any of it and whether they see all of it
    __device__ __forceinline__ void next(int& jt, bool& some, bool& all) {
        while (!act) {
            base += 64;
            if (base >= nt) { jt = -1; return; }
            const int x = base + lane, j0 = x * KT, j1 = j0 + KT - 1;
            const bool in = x < nt;
            int2 r = make_int2(0, 0);
            if (range && in) r = range[x];
            act = __ballot(in && mk.some(sw, j0, j1) && (!range || (range_lo(r) <= sw.hi && sw.lo <= r.y)));
            mine = __ballot(in && sv.p0 <= sv.p1 && mk.some(sv, j0, j1) && (!range || (range_lo(r) <= sv.hi && sv.lo <= r.y)));
            full = __ballot(in && mk.all(sv, j0, j1) && (!range || (sv.one && range_one(r) && r.y == sv.lo)));
        }
        const int i = __builtin_ctzll(act);
        act &= act - 1;
        jt = base + i;
        some = mine >> i & 1;
        all = full >> i & 1;
    }
};

}  // namespace slotattn
