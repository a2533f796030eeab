// Pages of a cache handed out to growing sequences and taken back, for MI355X (gfx950): include/slotpage.h.
//
// One workgroup walks the rows, a row a thread: running sums over the rows (DPP-free shuffles within a wave, then the waves' sums in LDS) give
// each row its place in the packed batch and in the stack of free pages, so nothing depends on the order in which threads run.  All
// of it is latency: a few dependent reads and five barriers per 1,024 rows.  The tokens' positions and slots follow from the rows' starts alone: the
// same workgroup writes those of a small batch, a second kernel those of a large one.  256 rows of one token 4.8 us and 3.9 to trim
// them, 23,000 tokens of 64 rows 5.2 to 5.7 and 3.5 (their positions and slots), 4 to 4.5 to trim them.
#include "slot_common.h"
#include "slotscan.h"
#include "slotpage.h"
#include "slot_host.h"

using namespace slot;
using slothost::fail;
using slothost::hip_fail;

#define PT 1024                                      // threads of the workgroup that walks the rows
#define PW (PT / 64)
#define PL 8192                                      // tokens that it writes itself
#define PR 4096                                      // rows whose starts it keeps in LDS for that

namespace {

struct PageArgs {
    const int32_t* new_; int32_t* lens; int32_t* table; int64_t t_sr; int32_t* free_; const int32_t* keep;
    int R, M, P, N, shift;
    int32_t* starts; int32_t* ends; int64_t* slots; int32_t* pos;
};

__device__ __forceinline__ int up(int n, int shift) { return (int)(((int64_t)n + (1 << shift) - 1) >> shift); }
__device__ __forceinline__ uint32_t satsum(uint32_t a, uint32_t b, uint32_t top) { return min(a + b, top); }   // a, b <= top < 2^31

// Sum of the x of the threads before this one and of all threads, neither past top.  s: PW + 1 words of LDS.
__device__ __forceinline__ uint32_t before(uint32_t x, uint32_t top, uint32_t* s, uint32_t& all) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    uint32_t v = x;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t y = __shfl_up(v, d);
        if (lane >= d) v = satsum(v, y, top);
    }
    uint32_t ex = __shfl_up(v, 1);
    if (lane == 0) ex = 0;
    __syncthreads();                                  // the last call's sums are read
    if (lane == 63) s[w] = v;
    __syncthreads();
    uint32_t base = 0, sum = 0;
#pragma unroll
    for (int i = 0; i < PW; i++) {
        if (i == w) base = sum;
        sum = satsum(sum, s[i], top);
    }
    all = sum;
    return satsum(base, ex, top);
}

// Page p of a round of rows, which begin at pages off[0 .. rows) (ascending): the last row that begins at or before it.
__device__ __forceinline__ int row_of(const uint32_t* off, int rows, uint32_t p) {
    int lo = 0, hi = rows;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (off[mid] <= p) lo = mid; else hi = mid;
    }
    return lo;
}

// Token i of the packed batch: its row is the last one that starts at or before it.
__device__ __forceinline__ void put_token(const PageArgs& a, const int32_t* starts, int i) {
    int lo = 0, hi = a.R;                             // starts[lo] <= i < starts[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (starts[mid] <= i) lo = mid; else hi = mid;
    }
    const int s0 = starts[lo], s1 = starts[lo + 1], end = a.ends[lo];
    int p = -1;
    int64_t slot = -1;
    if (i < s1 && end > 0) {
        p = end - (s1 - s0) + (i - s0);
        const int id = a.table[lo * a.t_sr + (p >> a.shift)];
        if ((unsigned)id < (unsigned)a.P) slot = ((int64_t)id << a.shift) + (p & ((1 << a.shift) - 1));
    }
    a.pos[i] = p;
    a.slots[i] = slot;
}

__global__ __launch_bounds__(PT) void page_extend(PageArgs a) {
    __shared__ uint32_t s_sum[PW + 1];
    __shared__ int32_t s_start[PR + 1], s_first[PT];  // rows' first tokens; of a round's rows the number of the first new page, -1: none
    __shared__ uint32_t s_off[PT];                    // and the pages asked for before them
    __shared__ uint32_t s_taken;                      // pages handed out: those up to the last row that got any
    const int tid = threadIdx.x;
    const int n = min(max(a.free_[0], 0), a.P);
    const uint32_t topN = (uint32_t)a.N + 1, topP = (uint32_t)n + 1;
    uint32_t at = 0, off = 0;                         // of the rows of earlier rounds: tokens, pages asked for
    const bool here = a.R <= PR && a.N <= PL;
    if (tid == 0) {
        a.starts[0] = 0;
        s_start[0] = 0;
        s_taken = 0;
    }
    for (int r0 = 0; r0 < a.R; r0 += PT) {
        const int r = r0 + tid;
        const bool in = r < a.R;
        const int want = in ? max(a.new_[r], 0) : 0, have = in ? a.lens[r] : 0;
        uint32_t all;
        const uint32_t x = min((uint32_t)want, topN);
        const uint32_t s0 = satsum(at, before(x, topN, s_sum, all), topN), s1 = satsum(s0, x, topN);
        at = satsum(at, all, topN);
        const bool fits = want > 0 && s1 <= (uint32_t)a.N && have >= 0 && (int64_t)have + want <= (int64_t)a.M << a.shift;
        const int first = up(max(have, 0), a.shift), need = fits ? up(have + want, a.shift) - first : 0;
        const uint32_t y = min((uint32_t)need, topP);
        const uint32_t o0 = satsum(off, before(y, topP, s_sum, all), topP), begin = off;
        off = satsum(off, all, topP);
        const bool got = fits && (need == 0 || satsum(o0, y, topP) <= (uint32_t)n);
        if (got && need) atomicMax(&s_taken, o0 + y);
        if (in) {
            const int start = min((int)s1, a.N);
            a.starts[r + 1] = start;
            if (here) s_start[r + 1] = start;
            a.ends[r] = got ? have + want : 0;
            if (got) a.lens[r] = have + want;
        }
        // The round's new pages, from the top of the stack down: a thread each (58 rows of 400 tokens: 5.2 us, row after row by a wave 7.2), or
        // each by its row's thread where no row has two (256 rows of a token: 4.8, else 5.1)
        s_off[tid] = o0;
        s_first[tid] = got ? first : -1;
        if (!__syncthreads_or(got && need > 1)) {
            if (got && need) a.table[r * a.t_sr + first] = a.free_[n - (int)o0];
            continue;
        }
        for (uint32_t p = begin + tid; p < min(off, (uint32_t)n); p += PT) {
            const int k = row_of(s_off, min(PT, a.R - r0), p);
            if (s_first[k] >= 0) a.table[(r0 + k) * a.t_sr + s_first[k] + (int)(p - s_off[k])] = a.free_[n - (int)p];
        }
    }
    __syncthreads();                                  // the table, the ends and the starts are written
    if (tid == 0) a.free_[0] = n - (int)s_taken;
    if (!here) return;
    for (int i = tid; i < a.N; i += PT) put_token(a, s_start, i);
}

__global__ __launch_bounds__(256) void page_tokens(PageArgs a) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < a.N) put_token(a, a.starts, i);
}

__global__ __launch_bounds__(PT) void page_trim(PageArgs a) {
    __shared__ uint32_t s_sum[PW + 1], s_off[PT];     // pages that come back from the rows before a round's
    __shared__ int32_t s_first[PT];                   // the number of a row's first page that does
    const int tid = threadIdx.x;
    const int n = min(max(a.free_[0], 0), a.P);
    const uint32_t top = 0x7ffffffe;
    auto row = [&](int r, int& first, int& keep) -> int {             // pages that row r gives back, from its page `first` on
        first = 0;
        keep = 0;
        if (r >= a.R) return 0;
        const int have = (int)min((int64_t)max(a.lens[r], 0), (int64_t)a.M << a.shift);
        keep = min(max(a.keep[r], 0), have);
        first = up(keep, a.shift);
        return up(have, a.shift) - first;
    };
    // how many in all: the stack's new top is the first row's first page
    uint32_t total = 0;
    for (int r0 = 0; r0 < a.R; r0 += PT) {
        int f, k;
        uint32_t all;
        before((uint32_t)row(r0 + tid, f, k), top, s_sum, all);
        total = satsum(total, all, top);
    }
    const int end = (int)min((int64_t)n + total, (int64_t)0x7ffffffe);
    uint32_t off = 0;
    for (int r0 = 0; r0 < a.R; r0 += PT) {
        const int r = r0 + tid;
        int first, keep;
        uint32_t all;
        const int c = row(r, first, keep);
        const uint32_t o0 = satsum(off, before((uint32_t)c, top, s_sum, all), top), begin = off;
        off = satsum(off, all, top);
        if (r < a.R) a.lens[r] = keep;
        s_off[tid] = o0;
        s_first[tid] = first;
        auto give = [&](int32_t* t, int to) {         // to in [1, P] unless pages come back that were never handed out
            if (to >= 1 && to <= a.P) a.free_[to] = *t;
            *t = -1;
        };
        if (!__syncthreads_or(c > 1)) {
            if (c) give(a.table + r * a.t_sr + first, end - (int)o0);
            continue;
        }
        for (uint32_t p = begin + tid; p < off; p += PT) {
            const int k = row_of(s_off, min(PT, a.R - r0), p);
            give(a.table + (r0 + k) * a.t_sr + s_first[k] + (int)(p - s_off[k]), end - (int)p);
        }
    }
    __syncthreads();
    if (tid == 0) a.free_[0] = min(end, a.P);
}

int check_pages(int64_t R, int64_t M, int64_t t_sr, int64_t P, int64_t page, const void* lens, const void* table, const void* free_) {
    if (R < 1 || M < 1 || P < 0) return fail(SLOTSCAN_ERR_SHAPE, "slotpage: R and M must be >= 1, P >= 0");
    if (page < SLOTPAGE_MIN || (page & (page - 1)) || page > SLOTPAGE_MAX) return fail(SLOTSCAN_ERR_SHAPE, "slotpage: page must be a power of two in [16, 4096]");
    if (R > 1 << 24 || P > 0x3fffffffLL || M * page > 0x3fffffffLL || t_sr < M) return fail(SLOTSCAN_ERR_SHAPE, "slotpage: shape too large, or table rows that overlap");
    if (!lens || !table || !free_) return fail(SLOTSCAN_ERR_NULL, "slotpage: a required pointer is NULL");
    return 0;
}

PageArgs base_args(int64_t R, int64_t M, int64_t t_sr, int64_t P, int64_t page, int32_t* lens, int32_t* table, int32_t* free_) {
    PageArgs a{};
    a.lens = lens; a.table = table; a.t_sr = t_sr; a.free_ = free_;
    a.R = (int)R; a.M = (int)M; a.P = (int)P; a.shift = __builtin_ctzll((unsigned long long)page);
    return a;
}

}  // namespace

extern "C" int slotpage_extend(const int32_t* new_, int32_t* lens, int32_t* table, int64_t t_sr, int32_t* free_, int64_t R, int64_t M,
                               int64_t P, int64_t page, int64_t N, int32_t* starts, int32_t* ends, int64_t* slots, int32_t* pos,
                               void* stream) {
    if (int r = check_pages(R, M, t_sr, P, page, lens, table, free_)) return r;
    if (N < 0 || N > 0x3fffffffLL) return fail(SLOTSCAN_ERR_SHAPE, "slotpage_extend: N must be in [0, 2^30)");
    if (!new_ || !starts || !ends || (N && (!slots || !pos))) return fail(SLOTSCAN_ERR_NULL, "slotpage_extend: a required pointer is NULL");
    PageArgs a = base_args(R, M, t_sr, P, page, lens, table, free_);
    a.new_ = new_; a.N = (int)N;
    a.starts = starts; a.ends = ends; a.slots = slots; a.pos = pos;
    hipStream_t st = (hipStream_t)stream;
    slothost::Scope sc(SLOTSCAN_K_PAGES, st);
    slothost::launch(page_extend, dim3(1), dim3(PT), 0, st, a);
    if (N > PL || (R > PR && N)) slothost::launch(page_tokens, dim3((unsigned)((N + 255) / 256)), dim3(256), 0, st, a);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "page_extend launch");
}

extern "C" int slotpage_trim(const int32_t* keep, int32_t* lens, int32_t* table, int64_t t_sr, int32_t* free_, int64_t R, int64_t M,
                             int64_t P, int64_t page, void* stream) {
    if (int r = check_pages(R, M, t_sr, P, page, lens, table, free_)) return r;
    if (!keep) return fail(SLOTSCAN_ERR_NULL, "slotpage_trim: a required pointer is NULL");
    PageArgs a = base_args(R, M, t_sr, P, page, lens, table, free_);
    a.keep = keep;
    hipStream_t st = (hipStream_t)stream;
    slothost::Scope sc(SLOTSCAN_K_PAGES, st);
    slothost::launch(page_trim, dim3(1), dim3(PT), 0, st, a);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : hip_fail(e, "page_trim launch");
}
