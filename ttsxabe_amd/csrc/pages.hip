// The paged cache's small operators: the plan of a step's attention, the bounds
// of a page's keys, and the selection of pages from them.
//
//   bounds:  mx[d] = max, mn[d] = min over the live keys k of a page, dim by dim
//   score of a page for a kv head = max over the heads of its group of
//            sum_d max(q_d, 0) mx_d + min(q_d, 0) mn_d   >=   any q.k of the page
#include <algorithm>

#include "common.h"
#include "kvlayout.h"
#include "paged.h"

namespace llmtie {

// --------------------------------------------------------------------- plan

constexpr int PG_SPAN = 4;  // blocks of an item at least: one a wave

// What row r sees: the first f positions and those from lo to tk (f = lo = 0: all); its table row, or -1.
__device__ __forceinline__ int4 row_sees(const PagePlanArgs& a, int r) {
    const int tk = max(0, min(a.tk[r], a.cols << a.shift));
    int table = a.row ? a.row[r] : r, lo = a.lo ? a.lo[r] : 0;
    if (table < 0 || table >= a.rows) table = -1;
    if (a.window) lo = max(lo, tk - a.window);
    lo = max(0, min(lo, tk));
    int f = min(a.shared, tk);
    if (f >= lo) f = lo = 0;
    return make_int4(f, lo, tk, table);
}

// The blocks of 32 positions that a row's own item walks, or those of a tile of
// rows: [0, na), [b0, c0) and [d0, e), where the blocks from c0 to d0 are its group's.
struct OwnBlocks {
    int na = 0, b0 = 0x7fffffff, e = 0, c0, d0, n;
    __device__ __forceinline__ void add(const int4& s) {
        if (s.w < 0) return;
        na = max(na, (s.x + 31) >> 5);
        if (s.y < s.z) b0 = min(b0, s.y >> 5), e = max(e, (s.z + 31) >> 5);
    }
    __device__ __forceinline__ void close(int glo, int ghi) {
        b0 = max(na, min(b0, e));
        c0 = max(b0, ghi > glo ? glo : e);
        d0 = ghi > glo ? ghi : c0;
        n = na + (e ? c0 - b0 + max(0, e - d0) : 0);
    }
};

// The sums of `v` over the threads before this one, and of all in `total`.
template <int PP>
__device__ __forceinline__ int2 scan_before(int2 v, int2* waves, int tid, int2& total) {
    int2 x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x.x, d), z = __shfl_up(x.y, d);
        if ((tid & 63) >= d) x.x += y, x.y += z;
    }
    if ((tid & 63) == 63) waves[tid >> 6] = x;
    __syncthreads();
    int2 before = make_int2(x.x - v.x, x.y - v.y);
    total = make_int2(0, 0);
#pragma unroll
    for (int w = 0; w < PP / 64; ++w) {
        const int2 y = waves[w];
        if (w < (tid >> 6)) before.x += y.x, before.y += y.y;
        total.x += y.x, total.y += y.y;
    }
    __syncthreads();
    return before;
}

// One workgroup. Tiles are up to PG_COLS columns (rows times a kv head's query
// heads): a group's rows over the blocks that all of them see whole and hold in the
// same pages, and rows of one sequence that follow one another (within an aligned
// tile of rows) over what else they see, each key masked by row; what a row alone sees is its own
// item's. All are cut into items of about the same cost, `target` of them a kv head in
// all. Bound by its chain of loads and barriers: a row a thread, few waves where there
// are few rows (ONE: what they see is held in LDS, else in the plan itself). 40 rows in
// five groups 6.4 us, 244 rows of four prompts 10.2.
template <int PP, bool ONE>
__global__ __launch_bounds__(PP) void page_plan_kernel(PagePlanArgs a) {
    __shared__ int gst[PG_GROUPS + 1], glo[PG_GROUPS], ghi[PG_GROUPS], gat[PG_GROUPS], gruns[PG_GROUPS];
    __shared__ int4 held[ONE ? PP : 1];
    __shared__ int2 waves[PP / 64];
    __shared__ uint64_t links[PP / 64 + 1];
    __shared__ unsigned long long work, tiled;
    const int tid = threadIdx.x;
    const int tile_rows = PG_TILE_ROWS(a.group);
    const int per = ONE ? 1 : (a.nseq + PP - 1) / PP;
    const int r0 = min(a.nseq, tid * per), r1 = min(a.nseq, r0 + per);
    int groups = a.starts ? a.groups : 0;
    int4* rows = reinterpret_cast<int4*>(a.plan + PG_HEAD);
    int4* items = reinterpret_cast<int4*>(a.plan + plan_items_at(a.nseq));
    auto sees = [&](int r) {
        if constexpr (ONE) return held[r];
        else return rows[PG_ROW / 4 * (size_t)r + 2];
    };
    // (The groups' loads before the first row's are waited for.)
    int falls = 0;
    for (int g = tid; g < groups; g += PP) {
        const int x = max(0, min(a.starts[g], a.nseq)), y = max(0, min(a.starts[g + 1], a.nseq)), p = a.prefix[g];
        gst[g] = x, ghi[g] = p, glo[g] = 0;
        if (g == groups - 1) gst[groups] = y;
        falls |= x > y;
    }
    for (int r = r0; r < r1; ++r) {
        const int4 s = row_sees(a, r);
        rows[PG_ROW / 4 * (size_t)r + 2] = s;
        if constexpr (ONE) held[r] = s;
    }
    if (tid == 0) work = tiled = 0;
    // Starts that decrease: no groups (tiles would lie over one another, more than there is room for).
    if (__syncthreads_or(falls)) groups = 0;
    auto group_of = [&](int r) {
        int lo = -1, hi = groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (gst[mid] <= r) lo = mid;
            else hi = mid;
        }
        return lo >= 0 && r < gst[lo + 1] ? lo : -1;
    };
    auto wide_cost = [&](int n) { return min(n, tile_rows) * a.group > 16 ? 7 : 4; };
    if (groups) {
        for (int r = r0; r < r1; ++r) {
            const int g = group_of(r);
            if (g < 0) continue;
            const int4 s = sees(r);
            atomicMin(&ghi[g], s.w < 0 ? 0 : s.z);
            atomicMax(&glo[g], s.y);
        }
        __syncthreads();
        for (int g = tid; g < groups; g += PP) {
            const int n = gst[g + 1] - gst[g];
            const int lo = (glo[g] + 31) >> 5, hi = max(0, ghi[g]) >> 5;
            const bool share = !a.whole && n >= 2 && hi > lo;
            glo[g] = share ? lo : 0;
            ghi[g] = share ? hi : 0;
            if (share)
                atomicAdd(&tiled, (unsigned long long)((n + tile_rows - 1) / tile_rows) * (unsigned)(hi - lo) * wide_cost(n));
        }
        __syncthreads();
    }
    // A row's own part: with those of the rows of its aligned tile that follow one another
    // and are of one sequence and group.
    struct Own {
        OwnBlocks o;
        int g, first, rows;
    };
    // Whether row r goes on with the sequence and the group of the one before.
    auto goes_on = [&](int r) {
        if (!a.together || r <= 0 || r >= a.nseq) return false;
        const int t = sees(r).w;
        return t >= 0 && t == sees(r - 1).w && (!groups || group_of(r) == group_of(r - 1));
    };
    if constexpr (ONE) {
        const uint64_t on = __ballot(goes_on(tid));
        if ((tid & 63) == 0) links[tid >> 6] = on;
        if (tid == 0) links[PP / 64] = 0;
        __syncthreads();
    }
    auto own_of = [&](int r) {
        Own x;
        x.g = groups ? group_of(r) : -1;
        const int t0 = r / tile_rows * tile_rows, to = min(t0 + tile_rows, a.nseq);
        x.first = r;
        int end = r + 1;
        if constexpr (ONE) {
            // The links of rows t0 up to t0 + 63: bits up to r back to the last that is not set, and on from there.
            const int w = t0 >> 6, sh = t0 & 63;
            const uint64_t on = (links[w] >> sh | (sh ? links[w + 1] << (64 - sh) : 0)) & ~1ull;
            const int at = r - t0;
            const uint64_t begins = ~on & ((2ull << at) - 1);  // (bit 0 is one)
            x.first = t0 + 63 - __clzll((long long)begins);
            const uint64_t breaks = ~on >> (at + 1);
            end = breaks ? min(to, r + __ffsll((long long)breaks)) : to;
        } else if (a.together) {
            while (x.first > t0 && goes_on(x.first)) --x.first;
            while (end < to && goes_on(end)) ++end;
        }
        x.rows = end - x.first;
        if (x.rows < PG_RUN_ROWS(a.group)) x.first = r, x.rows = 1;  // (so many tiles there is room for)
        for (int i = 0; i < x.rows; ++i) x.o.add(sees(x.first + i));
        x.o.close(x.g >= 0 ? glo[x.g] : 0, x.g >= 0 ? ghi[x.g] : 0);
        return x;
    };
    Own mine;
    if constexpr (ONE) {
        mine = own_of(min(tid, a.nseq - 1));
    } else {  // kept where the row's words will be
        for (int r = r0; r < r1; ++r) {
            const Own x = own_of(r);
            rows[PG_ROW / 4 * (size_t)r] = make_int4(x.o.na, x.o.b0, x.o.c0, x.o.d0);
            rows[PG_ROW / 4 * (size_t)r + 1] = make_int4(x.o.n, x.g, x.first, x.rows);
        }
    }
    auto own = [&](int r) {
        if constexpr (ONE) {
            return mine;
        } else {
            const int4 d = rows[PG_ROW / 4 * (size_t)r], e = rows[PG_ROW / 4 * (size_t)r + 1];
            Own x;
            x.o.na = d.x, x.o.b0 = d.y, x.o.c0 = d.z, x.o.d0 = d.w, x.o.n = e.x;
            x.g = e.y, x.first = e.z, x.rows = e.w;
            return x;
        }
    };
    unsigned long long cost = 0;
    for (int r = r0; r < r1; ++r) {
        const Own x = own(r);
        if (x.rows == 1) cost += (unsigned long long)x.o.n * 4;
        else if (x.first == r) atomicAdd(&tiled, (unsigned long long)x.o.n * wide_cost(x.rows));
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) cost += __shfl_xor(cost, d);
    if ((tid & 63) == 0) atomicAdd(&work, cost);
    __syncthreads();
    // Cost of an item, four a block (seven of two column tiles). (A sequence costs up to
    // 7 * 2^25: 32 bits, as divisions of 64 take half a microsecond each.)
    const unsigned target = (unsigned)(tiled > work ? a.tile_target : a.target);
    const unsigned long long each = (work + tiled + target - 1) / target;
    const unsigned c = (unsigned)max(min(each, 0x7fffffffull), (unsigned long long)(4 * PG_SPAN));
    auto cut = [&](int blocks, int cost) { return a.whole ? 1 : (int)(((unsigned)blocks * cost + c - 1) / c); };

    // Shared tiles, a group's runs of blocks outermost, so that its tiles read a run at one time.
    int ns = 0;
    auto runs_of = [&](int g) { return gruns[g]; };
    auto tiles_of = [&](int g) { return (gst[g + 1] - gst[g] + tile_rows - 1) / tile_rows; };
    if (groups) {
        const int each = (groups + PP - 1) / PP, g0 = min(groups, tid * each), g1 = min(groups, g0 + each);
        int2 n = make_int2(0, 0), total;
        for (int g = g0; g < g1; ++g) {
            gruns[g] = ghi[g] > glo[g] ? cut(ghi[g] - glo[g], wide_cost(gst[g + 1] - gst[g])) : 0;
            n.x += tiles_of(g) * gruns[g];
        }
        int at = scan_before<PP>(n, waves, tid, total).x;
        for (int g = g0; g < g1; ++g) gat[g] = at, at += tiles_of(g) * gruns[g];
        __syncthreads();
        ns = min(total.x, a.max_wide);
        for (int i = tid; i < ns; i += PP) {
            // Its group: the last one that begins at or before it and has items.
            int lo = 0, hi = groups;
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (gat[mid] <= i) lo = mid;
                else hi = mid;
            }
            const int g = lo, tiles = tiles_of(g), nb = ghi[g] - glo[g], share = (nb + gruns[g] - 1) / gruns[g];
            const int in = i - gat[g], t = in % tiles, b = in / tiles * share, first = gst[g] + t * tile_rows;
            int4* d = items + PG_ITEM / 4 * (size_t)i;
            d[0] = make_int4(first, min(tile_rows, gst[g + 1] - first), sees(first).w, PG_SHARED);
            d[1] = make_int4(0, glo[g], ghi[g], ghi[g]);
            d[2] = make_int4(b, min(nb, b + share), 0, 0);
        }
    }
    // Tiles of one sequence's rows (x), and rows by themselves (y).
    auto items_of = [&](const Own& x) {
        const bool shares = x.g >= 0 && ghi[x.g] > glo[x.g];
        return x.o.n ? cut(x.o.n, x.rows > 1 ? wide_cost(x.rows) : 4) : shares ? 0 : 1;
    };
    int2 n = make_int2(0, 0), total;
    for (int r = r0; r < r1; ++r) {
        const Own x = own(r);
        if (x.rows == 1) n.y += items_of(x);
        else if (x.first == r) n.x += items_of(x);
    }
    const int2 before = scan_before<PP>(n, waves, tid, total);
    int wide = ns + before.x, alone = before.y;
    const int nw = min(ns + total.x, a.max_wide);
    for (int r = r0; r < r1; ++r) {
        const Own x = own(r);
        const bool shares = x.g >= 0 && ghi[x.g] > glo[x.g];
        const int runs = items_of(x), share = runs ? (x.o.n + runs - 1) / runs : 0;
        int4 d = make_int4(alone, runs, 0, 0), e = make_int4(0, 0, -1, 0);
        if (shares) {
            const int in = r - gst[x.g];
            d.z = gat[x.g] + in / tile_rows;
            d.w = runs_of(x.g);
            e.x = tiles_of(x.g);
            e.y = in % tile_rows * a.group;
        }
        if (x.rows > 1) {
            // `wide` counts the items of the tiles that begin before this row: its own tile's are the last, but for its first row.
            d.x = x.first == r ? wide : wide - runs;
            e.z = (r - x.first) * a.group;
        }
        rows[PG_ROW / 4 * (size_t)r] = d;
        rows[PG_ROW / 4 * (size_t)r + 1] = e;
        if (x.first != r) continue;
        const int at = x.rows > 1 ? wide : nw + alone, end = x.rows > 1 ? nw : nw + a.max_own;
        for (int i = 0; i < runs; ++i) {
            if (at + i >= end) break;
            int4* t = items + PG_ITEM / 4 * (size_t)(at + i);
            t[0] = make_int4(r, x.rows, sees(r).w, runs == 1 && !shares ? PG_WHOLE : 0);
            t[1] = make_int4(x.o.na, x.o.b0, x.o.c0, x.o.d0);
            t[2] = make_int4(i * share, min(x.o.n, (i + 1) * share), 0, 0);
        }
        if (x.rows > 1) wide += runs;
        else alone += runs;
    }
    if (tid == 0) {
        int4* h = reinterpret_cast<int4*>(a.plan);
        h[0] = make_int4(nw + min(total.y, a.max_own), nw, a.nseq, a.group);
        h[1] = make_int4(a.kv_heads, a.shift, a.cols, a.rows);
        h[2] = make_int4(a.max_wide, a.max_own, a.whole, 0);
    }
}

hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t st) {
    if (a.nseq <= 256) hipLaunchKernelGGL((page_plan_kernel<256, true>), dim3(1), dim3(256), 0, st, a);
    else if (a.nseq <= 1024) hipLaunchKernelGGL((page_plan_kernel<1024, true>), dim3(1), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((page_plan_kernel<1024, false>), dim3(1), dim3(1024), 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------- bounds

// A wave takes 32 dims of a (page, kv head): lane (col, grp) reads keys 8 (col /
// 4) + 4 T + col % 4 of its eight dims, 1 KB a load, and the sixteen lanes of a
// row are then joined. Bound by reading the keys.
template <int HD>
__global__ __launch_bounds__(256) void page_bounds_kernel(PageBoundsArgs a) {
    constexpr int NS = HD / 32;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const long w = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
    const int s = (int)(w % NS), kh = (int)(w / NS % a.kv_heads);
    const long rest = w / NS / a.kv_heads;
    const int slot = (int)(rest % a.per), r = (int)(rest / a.per);
    if (r >= a.nseq) return;
    const int t = a.row ? a.row[r] : r;
    if (t < 0 || t >= a.p.rows) return;
    const int page = 1 << a.p.shift;
    const int tk = min(a.tk[r], a.p.cols << a.p.shift);
    if (tk <= 0) return;
    const int low = a.low ? max(0, a.low[r]) : 0;
    if (low >= tk) return;
    const int end = (tk - 1) / page + 1;
    for (int i = low / page + slot; i < end; i += a.per) {
        const int id = a.p.table[(size_t)t * a.p.cols + i];
        if (id < 0 || id >= a.p.pages) continue;
        const half_t* k = reinterpret_cast<const half_t*>(a.p.cache) +
                          ((size_t)id * a.kv_heads + kh) * ((size_t)(page / 32) * 64 * HD) + s * 512 + lane * 8;
        const int live = min(page, tk - i * page);
        half8 up, dn;
#pragma unroll
        for (int j = 0; j < 8; ++j) up[j] = (half_t)-__builtin_inff(), dn[j] = (half_t)__builtin_inff();
        for (int b = 0; b < (live + 31) / 32; ++b) {
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                if (32 * b + 8 * (col >> 2) + 4 * T + (col & 3) >= live) continue;
                const half8 x = ld_h8(k + (size_t)b * 64 * HD + T * NS * 512);
                up = __builtin_elementwise_maximum(up, x);
                dn = __builtin_elementwise_minimum(dn, x);
            }
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            uint4 u = __builtin_bit_cast(uint4, up), v = __builtin_bit_cast(uint4, dn);
            u = make_uint4(__shfl_xor(u.x, d), __shfl_xor(u.y, d), __shfl_xor(u.z, d), __shfl_xor(u.w, d));
            v = make_uint4(__shfl_xor(v.x, d), __shfl_xor(v.y, d), __shfl_xor(v.z, d), __shfl_xor(v.w, d));
            up = __builtin_elementwise_maximum(up, __builtin_bit_cast(half8, u));
            dn = __builtin_elementwise_minimum(dn, __builtin_bit_cast(half8, v));
        }
        half_t* out = reinterpret_cast<half_t*>(a.bounds) + ((size_t)id * a.kv_heads + kh) * 2 * HD + 32 * s + 8 * grp;
        if (col == 0) *reinterpret_cast<half8*>(out) = up;
        if (col == 1) *reinterpret_cast<half8*>(out + HD) = dn;
    }
}

hipError_t launch_page_bounds(int hd, const PageBoundsArgs& a, hipStream_t st) {
    const size_t waves = (size_t)a.nseq * a.per * a.kv_heads * (hd / 32);
    const dim3 grid((unsigned)((waves + 3) / 4));
    if (hd == 128) hipLaunchKernelGGL((page_bounds_kernel<128>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((page_bounds_kernel<64>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
}

// ---------------------------------------------------------------- selection
//
// A selection is whole numbers, and two pages' scores lie within an f32 sum's
// rounding of each other in one selection of ten thousand: the definition's sums
// are f64's. But f64 decides at the border only. All scores s are formed by the
// matrix units as s' from q as the sum of two f16 (scaled by a power of two so
// that the largest |q| is in 2^14 to 2^15; the bounds are f16), with
//   |s' - s| <= E = 1.05 (4 HD + 2) 2^-23 A + 1,   A = sum_d |q_d b_d| over the products of the sum:
// q's two halves are 2^-22 of it off and 2^-25 more (256 times 65504 of these are
// 0.5), the products are exact, and 4 HD additions to f32 lose at most 2^-23 of A
// each, whatever order and rounding the matrix unit has. A itself is formed from
// the upper halves, 2^-11 and its own additions off: within the 1.05, as the
// roundings of t +- 2 E are.
// With t the count-th largest s' (a bin of a histogram that it lies in) and E the largest
// one, pages with s' > t + 2 E are selected, those with s' < t - 2 E are not, and the few
// between (1 to 5 of 500 random ones) are ranked by sums in f64. (All sums in f64, 32 sequences of 2000-32768
// positions, pages of 64: 59.5 us.)

constexpr int SE = 1024;         // threads of a selection
constexpr int SC = 256;          // and of a part of its scores
constexpr int DIGIT = 12;
constexpr int PS_LDS = 8192;     // pages whose scores a workgroup holds
constexpr int PS_NEAR = 256;     // pages near the border that it ranks
constexpr int PS_BINS = 1024;

struct SelectUnit {
    int r, kh, table, live;
    const float* q;
    __device__ __forceinline__ SelectUnit(const SelectArgs& a, int unit) {
        r = unit / a.kv_heads, kh = unit % a.kv_heads;
        table = a.row ? a.row[r] : r;
        const int tk = max(0, min(a.tk[r], a.wide << a.shift));
        live = table < 0 || table >= a.rows ? 0 : (tk + (1 << a.shift) - 1) >> a.shift;
        q = a.q + (size_t)r * a.q_stride;
    }
};

// A kv head's queries as the matrix unit's operands: the upper and lower halves of
// their positive and of their negative part, [4][HD / 32][64 lanes] of eight.
template <int HD>
struct QueryLds {
    half_t part[4 * HD / 32 * 64 * 8];
    float size[16];
};

// Scores s' of pages p0 .. p1 - 1 by W waves, 16 pages a step: q's heads are
// the rows of the tile, pages its columns. Returns this lane's largest E (infinite where a
// page is not there or something is not finite), and its largest and least s' of pages from k0 up to k1. Bound by reading the bounds: 16
// waves a workgroup, each with a step's 8 KB on their way. (The operands formed by
// each wave for itself took 16 waves 4.5 us, and eight waves were slower for it.)
template <int HD, int W>
__device__ __forceinline__ float score_pages(const SelectArgs& a, const SelectUnit& x, int p0, int p1, float* out,
                                             QueryLds<HD>& ql, int tid, int k0, int k1, float& top, float& least) {
    constexpr int NS = HD / 32;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), col = lane & 15, grp = lane >> 4;
    const int* ids = a.table + (size_t)x.table * a.cols;
    auto id_of = [&](int t) { return ids[min(p0 + 16 * t + col, p1 - 1)]; };
    struct Step {
        half8 mx[NS], mn[NS];
        bool gone;
    };
    auto load = [&](Step& y, int id) __attribute__((always_inline)) {
        y.gone = id < 0 || id >= a.pages;
        const half_t* b = reinterpret_cast<const half_t*>(a.bounds) +
                          ((size_t)(y.gone ? 0 : id) * a.kv_heads + x.kh) * 2 * HD + 8 * grp;
#pragma unroll
        for (int s = 0; s < NS; ++s) y.mx[s] = ld_h8(b + 32 * s), y.mn[s] = ld_h8(b + HD + 32 * s);
    };
    const int steps = (p1 - p0 + 15) / 16;
    const int first = id_of(wave);
    int ahead = id_of(wave + W);
    constexpr int N = 16 * HD / (64 * W);  // values of a thread: heads past the group's are 0
    const float* q = x.q + (size_t)x.kh * a.group * HD;
    float v[N], size = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = tid + 64 * W * i;
        v[i] = e < a.group * HD ? q[e] : 0.0f;
        size = fmaxf(size, fabsf(v[i]));
    }
    Step cur;
    load(cur, first);
    size = wave_max(size);
    if (lane == 0) ql.size[wave] = size;
    lds_barrier();
#pragma unroll
    for (int k = 0; k < W; ++k) size = fmaxf(size, ql.size[k]);
    int e2 = 0;
    (void)frexpf(size, &e2);  // in 2^(e2 - 1) to 2^e2
    const int up = size > 0.0f && size < __builtin_inff() ? 15 - e2 : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const int e = tid + 64 * W * i, h = e / HD, d = e % HD;
        half_t* at = ql.part + (d / 32 * 64 + h + 16 * (d / 8 % 4)) * 8 + d % 8;
        half_t hi, lo;
        const float y = ldexpf(v[i], up);
        split_h(y < 0.0f ? 0.0f : y, hi, lo);  // (a NaN stays one)
        at[0] = hi, at[NS * 512] = lo;
        split_h(y > 0.0f ? 0.0f : y, hi, lo);
        at[2 * NS * 512] = hi, at[3 * NS * 512] = lo;
    }
    lds_barrier();
    half8 ph[NS], pl[NS], nh[NS], nl[NS];
    const half8* part = reinterpret_cast<const half8*>(ql.part);
#pragma unroll
    for (int s = 0; s < NS; ++s) {
        ph[s] = part[s * 64 + lane], pl[s] = part[(NS + s) * 64 + lane];
        nh[s] = part[(2 * NS + s) * 64 + lane], nl[s] = part[(3 * NS + s) * 64 + lane];
    }
    float worst = 0.0f;
    for (int t = wave; t < steps; t += W) {
        floatx4 sc = zero_f4(), ab = zero_f4();
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            typedef uint32_t u4 __attribute__((ext_vector_type(4)));
            const half8 amx = __builtin_bit_cast(half8, __builtin_bit_cast(u4, cur.mx[s]) & 0x7fff7fffu);
            const half8 amn = __builtin_bit_cast(half8, __builtin_bit_cast(u4, cur.mn[s]) | 0x80008000u);
            ab = mfma16(ph[s], amx, ab);
            ab = mfma16(nh[s], amn, ab);
            sc = mfma16(pl[s], cur.mx[s], sc);
            sc = mfma16(nl[s], cur.mn[s], sc);
            sc = mfma16(ph[s], cur.mx[s], sc);
            sc = mfma16(nh[s], cur.mn[s], sc);
        }
        const bool gone = cur.gone;
        load(cur, ahead);
        ahead = id_of(t + 2 * W);
        float best = ninf(), most = 0.0f;
        bool odd = gone;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (4 * grp + r < a.group) {
                best = fmaxf(best, sc[r]);
                most = fmaxf(most, ab[r]);
                odd = odd || !(ab[r] < 0x1p40f);  // (the most of finite ones is 2^39)
            }
        }
        best = max4grp(best);
        worst = fmaxf(worst, odd ? __builtin_inff() : most);
        const int p = p0 + 16 * t + col;
        if (grp == 0 && p < p1) out[p] = best;
        if (p >= k0 && p < min(p1, k1)) top = fmaxf(top, best), least = fminf(least, best);
    }
    return worst < __builtin_inff() ? __builtin_fmaf(worst, 1.05f * (4 * HD + 2) * 0x1p-23f, 1.0f) : worst;
}

// The definition: one page's score by a wave, in f64.
template <int HD>
__device__ __forceinline__ double score_exact(const SelectArgs& a, const SelectUnit& x, int p, int lane) {
    constexpr int D = HD / 64;
    const int id = a.table[(size_t)x.table * a.cols + p];
    if (id < 0 || id >= a.pages) return __builtin_inf();  // as its keys make the row NaN
    const half_t* b = reinterpret_cast<const half_t*>(a.bounds) + ((size_t)id * a.kv_heads + x.kh) * 2 * HD + D * lane;
    double best = -__builtin_inf();
    constexpr int U = 4;  // heads side by side
    for (int g0 = 0; g0 < a.group; g0 += U) {
        double s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* q = x.q + (size_t)(x.kh * a.group + min(g0 + u, a.group - 1)) * HD + D * lane;
            s[u] = 0.0;
#pragma unroll
            for (int j = 0; j < D; ++j) {
                const double y = (double)q[j];
                s[u] = __builtin_fma(y < 0.0 ? 0.0 : y, (double)(float)b[j], s[u]);
                s[u] = __builtin_fma(y > 0.0 ? 0.0 : y, (double)(float)b[HD + j], s[u]);
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1)
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] += __shfl_xor(s[u], d);
#pragma unroll
        for (int u = 0; u < U; ++u) best = fmax(best, s[u] == s[u] ? s[u] : __builtin_inf());
    }
    return best + 0.0;  // -0: 0
}

// Bits that order as the numbers do.
__device__ __forceinline__ uint64_t order(double s) {
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

struct SelectLds {
    int hist[1 << DIGIT];
    int waves[SE / 64], above[SE / 64], at[SE / 64];
    int found[3];
    int near, sure;
    float worst[SE / 64], top[SE / 64], least[SE / 64];
    int page[PS_NEAR];
    double score[PS_NEAR];
};

// The digits, from the top, of the count-th largest of key(0 .. n - 1): each a
// histogram of those that agree above it. `mask` holds the digits found when the
// border's bin is taken whole, `need` how many of the border's are taken.
template <typename K, typename Key>
__device__ __forceinline__ void border_of(SelectLds& w, int n, int count, int tid, Key&& key, K& border, K& mask, int& need) {
    constexpr int B = (1 << DIGIT) / SE;
    const int lane = tid & 63, wave = tid >> 6;
    border = mask = 0, need = count;
    for (int top = 8 * (int)sizeof(K); top > 0;) {
        const int bits = min(DIGIT, top), low = top - bits;
        int4* h = reinterpret_cast<int4*>(w.hist);
#pragma unroll
        for (int i = 0; i < B / 4; ++i) h[tid + SE * i] = make_int4(0, 0, 0, 0);
        __syncthreads();
        for (int p = tid; p < n; p += SE) {
            const K k = key(p);
            if ((k & mask) == border) atomicAdd(&w.hist[(int)(k >> low) & ((1 << bits) - 1)], 1);
        }
        __syncthreads();
        // From the top bin down, B bins a thread.
        int bin[B], sum = 0;
        const int first = (1 << DIGIT) - B * (tid + 1);
#pragma unroll
        for (int i = 0; i < B / 4; ++i) {
            const int4 y = h[first / 4 + i];
            bin[4 * i] = y.x, bin[4 * i + 1] = y.y, bin[4 * i + 2] = y.z, bin[4 * i + 3] = y.w;
        }
#pragma unroll
        for (int i = 0; i < B; ++i) sum += bin[i];
        int upto = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(upto, d);
            if (lane >= d) upto += y;
        }
        if (lane == 63) w.waves[wave] = upto;
        __syncthreads();
        for (int k = 0; k < wave; ++k) upto += w.waves[k];
        if (upto >= need && upto - sum < need) {
            int left = need - (upto - sum);
            bool done = false;
#pragma unroll
            for (int i = B - 1; i >= 0; --i) {
                if (!done && bin[i] >= left) {
                    w.found[0] = first + i, w.found[1] = left, w.found[2] = bin[i];
                    done = true;
                }
                if (!done) left -= bin[i];
            }
        }
        __syncthreads();
        border |= (K)w.found[0] << low;
        mask |= (K)((1 << bits) - 1) << low;
        need = w.found[1];
        top = low;
        if (w.found[2] == need) break;
    }
}

// Pages with above(p), and the first `need` with at(p), in order: a thread's pages lie together.
template <typename Above, typename At>
__device__ __forceinline__ void emit(SelectLds& w, int n, int need, int* out, int tid, Above&& above, At&& at) {
    const int lane = tid & 63, wave = tid >> 6, per = (n + SE - 1) / SE, p0 = min(n, tid * per), p1 = min(n, p0 + per);
    int ng = 0, ne = 0;
    for (int p = p0; p < p1; ++p) {
        const bool gt = above(p);
        ng += gt, ne += !gt && at(p);
    }
    int g = ng, e = ne;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(g, d), z = __shfl_up(e, d);
        if (lane >= d) g += y, e += z;
    }
    if (lane == 63) w.above[wave] = g, w.at[wave] = e;
    __syncthreads();
    for (int k = 0; k < wave; ++k) g += w.above[k], e += w.at[k];
    g -= ng, e -= ne;
    for (int p = p0; p < p1; ++p) {
        const bool gt = above(p), eq = !gt && at(p);
        if (gt || (eq && e < need)) out[g + min(e, need)] = p;
        g += gt, e += eq;
    }
}

// All sums in f64: pages past those that a workgroup holds, or something not finite.
template <int HD>
__device__ void select_exact(SelectLds& w, const SelectArgs& a, const SelectUnit& x, int unit, int* out, int tid) {
    double* score = a.exact + (size_t)unit * a.wide;
    for (int p = tid >> 6; p < x.live; p += SE / 64) {
        const double s = score_exact<HD>(a, x, p, tid & 63);
        if ((tid & 63) == 0) score[p] = s;
    }
    __syncthreads();
    auto key = [&](int p) { return p < a.first || p >= x.live - a.last ? ~0ull : order(score[p]); };
    uint64_t border, mask;
    int need;
    border_of<uint64_t>(w, x.live, a.count, tid, key, border, mask, need);
    emit(w, x.live, need, out, tid, [&](int p) { return (key(p) & mask) > border; },
         [&](int p) { return (key(p) & mask) == border; });
}

// A workgroup a (row, kv head). SCORED: its pages' scores are in the workspace.
template <int HD, bool SCORED>
__global__ __launch_bounds__(SE) void page_select_kernel(SelectArgs a) {
    extern __shared__ float sc[];
    __shared__ SelectLds w;
    __shared__ __attribute__((aligned(16))) QueryLds<HD> ql;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, unit = (int)blockIdx.x;
    const SelectUnit x(a, unit);
    int* out = a.chosen + (size_t)unit * a.count;
    if (x.live <= a.count) {
        for (int i = tid; i < a.count; i += SE) out[i] = i < x.live ? i : -1;
        return;
    }
    if (a.wide > PS_LDS) {
        select_exact<HD>(w, a, x, unit, out, tid);
        return;
    }
    auto kept = [&](int p) { return p < a.first || p >= x.live - a.last; };
    const int keep = a.first + a.last;
    if (keep == a.count) {
        emit(w, x.live, 0, out, tid, kept, [](int) { return false; });
        return;
    }
    for (int i = tid; i < PS_BINS; i += SE) w.hist[i] = 0;
    if (tid == 0) w.near = 0, w.sure = 0;
    float worst = 0.0f, top = ninf(), least = -ninf();
    if constexpr (SCORED) {
        const float* from = a.score + (size_t)unit * a.wide;
        for (int p = tid; p < x.live; p += SE) {
            const float s = from[p];
            sc[p] = s;
            if (!kept(p)) top = fmaxf(top, s), least = fminf(least, s);
        }
        for (int i = tid; i < a.chunks; i += SE) worst = fmaxf(worst, a.worst[(size_t)unit * a.chunks + i]);
    } else {
        worst = score_pages<HD, SE / 64>(a, x, 0, x.live, sc, ql, tid, a.first, x.live - a.last, top, least);
    }
    worst = wave_max(worst), top = wave_max(top), least = -wave_max(-least);
    if (lane == 0) w.worst[wave] = worst, w.top[wave] = top, w.least[wave] = least;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < SE / 64; ++k)
        worst = fmaxf(worst, w.worst[k]), top = fmaxf(top, w.top[k]), least = fminf(least, w.least[k]);
    const float e2 = 2.0f * worst;
    if (!(e2 < 0x1p40f)) {
        select_exact<HD>(w, a, x, unit, out, tid);
        return;
    }
    // The bin of the border, of even ones between the least and the largest. (By
    // digits as border_of has them, nearly all fall into a few bins of the first: 2048
    // pages 20 us, so 10.)
    const float wide = (top - least) / PS_BINS, mul = top > least ? PS_BINS / (top - least) : 0.0f;
    for (int p = tid; p < x.live; p += SE)
        if (!kept(p)) atomicAdd(&w.hist[min((int)((sc[p] - least) * mul), PS_BINS - 1)], 1);
    __syncthreads();
    if (wave == 0) {
        constexpr int B = PS_BINS / 64;
        const int4* h = reinterpret_cast<const int4*>(w.hist);
        int bin[B], sum = 0;
        const int first = PS_BINS - B * (lane + 1), need = a.count - keep;
#pragma unroll
        for (int i = 0; i < B / 4; ++i) {
            const int4 y = h[first / 4 + i];
            bin[4 * i] = y.x, bin[4 * i + 1] = y.y, bin[4 * i + 2] = y.z, bin[4 * i + 3] = y.w;
        }
#pragma unroll
        for (int i = 0; i < B; ++i) sum += bin[i];
        int upto = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(upto, d);
            if (lane >= d) upto += y;
        }
        if (upto >= need && upto - sum < need) {
            int left = need - (upto - sum), at = first + B - 1;
#pragma unroll
            for (int i = B - 1; i > 0; --i)
                if (at == first + i && bin[i] < left) left -= bin[i], --at;
            w.found[0] = at;
        }
    }
    __syncthreads();
    // (The roundings of a bin's ends are a few 2^-24 of the largest score: within E's 1.05.)
    const float low = least + (float)w.found[0] * wide - e2, high = least + (float)(w.found[0] + 1) * wide + e2;
    int sure = 0;
    for (int p = tid; p < x.live; p += SE) {
        if (kept(p) || sc[p] > high) {
            ++sure;
        } else if (sc[p] >= low) {
            const int i = atomicAdd(&w.near, 1);
            if (i < PS_NEAR) w.page[i] = p;
        }
    }
    const uint64_t any = __ballot(sure != 0);
    if (any) {
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) sure += __shfl_xor(sure, d);
        if (lane == 0) atomicAdd(&w.sure, sure);
    }
    __syncthreads();
    const int near = w.near, left = a.count - w.sure;
    if (near > PS_NEAR) {
        select_exact<HD>(w, a, x, unit, out, tid);
        return;
    }
    if (near > left) {
        for (int i = wave; i < near; i += SE / 64) {
            const double s = score_exact<HD>(a, x, w.page[i], lane);
            if (lane == 0) w.score[i] = s;
        }
        __syncthreads();
        if (tid < near) {
            int rank = 0;
            for (int i = 0; i < near; ++i)
                rank += w.score[i] > w.score[tid] || (w.score[i] == w.score[tid] && w.page[i] < w.page[tid]);
            if (rank >= left) sc[w.page[tid]] = ninf();
        }
        __syncthreads();
    }
    emit(w, x.live, 0, out, tid, [&](int p) { return kept(p) || sc[p] >= low; }, [](int) { return false; });
}

// Few (row, kv head)s of many pages: their scores by `chunks` workgroups each.
template <int HD>
__global__ __launch_bounds__(SC) void page_score_kernel(SelectArgs a) {
    __shared__ float top[SC / 64];
    __shared__ __attribute__((aligned(16))) QueryLds<HD> ql;
    const int tid = threadIdx.x, unit = (int)(blockIdx.x / (unsigned)a.chunks), chunk = (int)(blockIdx.x % (unsigned)a.chunks);
    const SelectUnit x(a, unit);
    const int share = (((x.live + 15) / 16 + a.chunks - 1) / a.chunks) * 16;
    const int p0 = chunk * share, p1 = min(x.live, p0 + share);
    float worst = 0.0f;
    float most = 0.0f, least = 0.0f;
    if (p0 < p1) worst = score_pages<HD, SC / 64>(a, x, p0, p1, a.score + (size_t)unit * a.wide, ql, tid, 0, 0, most, least);
    worst = wave_max(worst);
    if ((tid & 63) == 0) top[tid >> 6] = worst;
    __syncthreads();
    if (tid == 0) a.worst[(size_t)unit * a.chunks + chunk] = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
}

hipError_t launch_select(int hd, const SelectArgs& a, hipStream_t st) {
    const unsigned units = (unsigned)a.nseq * (unsigned)a.kv_heads;
    const size_t lds = a.wide <= PS_LDS ? (size_t)a.wide * sizeof(float) : 0;
    const bool scored = a.chunks > 1 && a.wide <= PS_LDS && a.wide > a.count;
#define SL(HD)                                                                                                  \
    if (hd == HD) {                                                                                             \
        if (scored) {                                                                                           \
            hipLaunchKernelGGL((page_score_kernel<HD>), dim3(units * (unsigned)a.chunks), dim3(SC), 0, st, a);  \
            hipLaunchKernelGGL((page_select_kernel<HD, true>), dim3(units), dim3(SE), lds, st, a);              \
        } else hipLaunchKernelGGL((page_select_kernel<HD, false>), dim3(units), dim3(SE), lds, st, a);          \
    }
    SL(64) SL(128)
#undef SL
    return hipGetLastError();
}

}  // namespace llmtie
