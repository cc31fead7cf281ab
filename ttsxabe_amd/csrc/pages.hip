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

// What row r sees: the first f positions and those from lo to tk (f = lo = 0: all).
struct RowSeen {
    int tk, lo, f, table;
    __device__ __forceinline__ RowSeen(const PagePlanArgs& a, int r) {
        table = a.row ? a.row[r] : r;
        tk = max(0, min(a.tk[r], a.cols << a.shift));
        if (table < 0 || table >= a.rows) table = -1;
        lo = a.lo ? a.lo[r] : 0;
        if (a.window) lo = max(lo, tk - a.window);
        lo = max(0, min(lo, tk));
        f = min(a.shared, tk);
        if (f >= lo) f = lo = 0;
    }
};

// The blocks of 32 positions that a row's own item walks: [0, na), [b0, c0) and
// [d0, e), where the blocks from c0 to d0 are its group's.
struct OwnBlocks {
    int na, b0, c0, d0, n;
    __device__ __forceinline__ OwnBlocks(const RowSeen& s, int glo, int ghi) {
        const int e = (s.tk + 31) >> 5;
        na = (s.f + 31) >> 5;
        b0 = max(na, s.lo >> 5);
        c0 = ghi > glo ? glo : e;
        d0 = ghi > glo ? ghi : e;
        c0 = max(b0, c0);
        n = na + (s.lo < s.tk ? c0 - b0 + max(0, e - d0) : 0);
        if (s.table < 0) n = 0;
    }
};

// The sum of `v` over the threads before this one, and of all in `total`.
template <int PP>
__device__ __forceinline__ int scan_before(int v, int* waves, int tid, int& total) {
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(x, d);
        if ((tid & 63) >= d) x += y;
    }
    if ((tid & 63) == 63) waves[tid >> 6] = x;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PP / 64; ++w) {
        if (w < (tid >> 6)) before += waves[w];
        total += waves[w];
    }
    __syncthreads();
    return before + x - v;
}

// A row's group (-1: none), what it sees and its own blocks.
struct PlanRow {
    RowSeen s;
    int g;
};

// One workgroup. A shared tile is up to PG_COLS columns (rows of a group times a
// kv head's query heads) over the blocks that all the group's rows see whole and
// hold in the same pages; what else a row sees is its own tile's. Each tile is
// cut into items of about the same cost, `target` of them a kv head in all.
// Bound by its chain of loads and barriers: a row a thread, whose lengths are
// read once, and few waves where there are few rows.
template <int PP, bool ONE>
__global__ __launch_bounds__(PP) void page_plan_kernel(PagePlanArgs a) {
    __shared__ int gst[PG_GROUPS + 1], glo[PG_GROUPS], ghi[PG_GROUPS], gat[PG_GROUPS];
    __shared__ int waves[PP / 64];
    __shared__ unsigned long long work;
    const int tid = threadIdx.x;
    const int tile_rows = PG_TILE_ROWS(a.group);
    const int per = ONE ? 1 : (a.nseq + PP - 1) / PP;
    const int r0 = min(a.nseq, tid * per), r1 = min(a.nseq, r0 + per);
    int groups = a.starts ? a.groups : 0;
    PlanRow held{RowSeen(a, min(tid, a.nseq - 1)), -1};
    for (int g = tid; g <= groups && groups; g += PP) gst[g] = max(0, min(a.starts[g], a.nseq));
    for (int g = tid; g < groups; g += PP) ghi[g] = a.prefix[g], glo[g] = 0;
    if (tid == 0) work = 0;
    __syncthreads();
    // Starts that decrease: no groups (tiles would lie over one another, more than there is room for).
    int falls = 0;
    for (int g = tid; g < groups; g += PP) falls |= gst[g] > gst[g + 1];
    if (groups && __syncthreads_or(falls)) groups = 0;
    auto group_of = [&](int r) {
        int lo = -1, hi = groups;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (gst[mid] <= r) lo = mid;
            else hi = mid;
        }
        return lo >= 0 && r < gst[lo + 1] ? lo : -1;
    };
    if constexpr (ONE) held.g = groups && tid < a.nseq ? group_of(tid) : -1;
    auto row_of = [&](int r) {
        if constexpr (ONE) return held;
        return PlanRow{RowSeen(a, r), groups ? group_of(r) : -1};
    };
    if (groups) {
        for (int r = r0; r < r1; ++r) {
            const PlanRow x = row_of(r);
            if (x.g < 0) continue;
            atomicMin(&ghi[x.g], x.s.table < 0 ? 0 : x.s.tk);
            atomicMax(&glo[x.g], x.s.lo);
        }
        __syncthreads();
        for (int g = tid; g < groups; g += PP) {
            const int n = gst[g + 1] - gst[g];
            const int lo = (glo[g] + 31) >> 5, hi = max(0, ghi[g]) >> 5;
            const bool share = !a.whole && n >= 2 && hi > lo;
            glo[g] = share ? lo : 0;
            ghi[g] = share ? hi : 0;
            if (share)
                atomicAdd(&work, (unsigned long long)((n + tile_rows - 1) / tile_rows) * (unsigned)(hi - lo) *
                                     (min(n, tile_rows) * a.group > 16 ? 7u : 4u));
        }
        __syncthreads();
    }
    auto own_of = [&](const PlanRow& x) { return OwnBlocks(x.s, x.g >= 0 ? glo[x.g] : 0, x.g >= 0 ? ghi[x.g] : 0); };
    unsigned long long mine = 0;
    for (int r = r0; r < r1; ++r) mine += 4ull * (unsigned)own_of(row_of(r)).n;
    if (mine) atomicAdd(&work, mine);
    __syncthreads();
    // Cost of an item, four a block (seven of two column tiles).
    const unsigned long long c = max((work + a.target - 1) / a.target, (unsigned long long)(4 * PG_SPAN));
    auto cut = [&](int blocks, int cost) {
        return a.whole ? 1 : (int)(((unsigned long long)blocks * cost + c - 1) / c);
    };
    int4* rows = reinterpret_cast<int4*>(a.plan + PG_HEAD);
    int4* items = rows + (PG_ROW * (size_t)a.nseq + PG_ROW * (size_t)a.nseq % 16) / 4;

    // Shared tiles, a group's runs of blocks outermost, so that its tiles read a run at one time.
    int ns = 0;
    auto runs_of = [&](int g) {
        return cut(ghi[g] - glo[g], min(gst[g + 1] - gst[g], tile_rows) * a.group > 16 ? 7 : 4);
    };
    auto tiles_of = [&](int g) { return (gst[g + 1] - gst[g] + tile_rows - 1) / tile_rows; };
    if (groups) {
        const int each = (groups + PP - 1) / PP, g0 = min(groups, tid * each), g1 = min(groups, g0 + each);
        auto items_of = [&](int g) { return ghi[g] > glo[g] ? tiles_of(g) * runs_of(g) : 0; };
        int n = 0;
        for (int g = g0; g < g1; ++g) n += items_of(g);
        int at = scan_before<PP>(n, waves, tid, ns);
        for (int g = g0; g < g1; ++g) gat[g] = at, at += items_of(g);
        __syncthreads();
        ns = min(ns, a.max_shared);
        for (int g = 0; g < groups; ++g) {
            if (ghi[g] <= glo[g]) continue;
            const int tiles = tiles_of(g), runs = runs_of(g), nb = ghi[g] - glo[g], share = (nb + runs - 1) / runs;
            for (int i = tid; i < tiles * runs; i += PP) {
                if (gat[g] + i >= ns) break;
                const int t = i % tiles, b = i / tiles * share, first = gst[g] + t * tile_rows;
                const int row = a.row ? a.row[first] : first;
                int4* d = items + PG_ITEM / 4 * (size_t)(gat[g] + i);
                d[0] = make_int4(first, min(tile_rows, gst[g + 1] - first), row, 0);
                d[1] = make_int4(0, glo[g], ghi[g], ghi[g]);
                d[2] = make_int4(b, min(nb, b + share), 0, 0);
            }
        }
    }
    // Rows and their own items.
    auto own_items = [&](const PlanRow& x, int n) {
        const bool shares = x.g >= 0 && ghi[x.g] > glo[x.g];
        return n ? cut(n, 4) : shares ? 0 : 1;
    };
    int n = 0, no = 0;
    for (int r = r0; r < r1; ++r) {
        const PlanRow x = row_of(r);
        n += own_items(x, own_of(x).n);
    }
    int at = scan_before<PP>(n, waves, tid, no);
    for (int r = r0; r < r1; ++r) {
        const PlanRow x = row_of(r);
        const OwnBlocks o = own_of(x);
        const bool shares = x.g >= 0 && ghi[x.g] > glo[x.g];
        const int runs = own_items(x, o.n), share = runs ? (o.n + runs - 1) / runs : 0;
        int4 d = make_int4(at, runs, 0, 0), e = make_int4(0, 0, 0, 0);
        if (shares) {
            const int in = r - gst[x.g];
            d.z = gat[x.g] + in / tile_rows;
            d.w = runs_of(x.g);
            e.x = tiles_of(x.g);
            e.y = in % tile_rows * a.group;
        }
        rows[PG_ROW / 4 * (size_t)r] = d;
        rows[PG_ROW / 4 * (size_t)r + 1] = e;
        for (int i = 0; i < runs; ++i) {
            if (at + i >= a.max_own) break;
            int4* t = items + PG_ITEM / 4 * (size_t)(ns + at + i);
            t[0] = make_int4(r, 1, x.s.table, runs == 1 && !shares);
            t[1] = make_int4(o.na, o.b0, o.c0, o.d0);
            t[2] = make_int4(i * share, min(o.n, (i + 1) * share), x.s.f, x.s.lo);
            t[3] = make_int4(x.s.tk, 0, 0, 0);
        }
        at += runs;
    }
    if (tid == 0) {
        no = min(no, a.max_own);
        int4* h = reinterpret_cast<int4*>(a.plan);
        h[0] = make_int4(ns + no, ns, a.nseq, a.group);
        h[1] = make_int4(a.kv_heads, a.shift, a.cols, a.rows);
        h[2] = make_int4(a.max_shared, a.max_own, a.whole, 0);
    }
}

hipError_t launch_page_plan(const PagePlanArgs& a, hipStream_t st) {
    if (a.nseq <= 256) hipLaunchKernelGGL((page_plan_kernel<256, true>), dim3(1), dim3(256), 0, st, a);
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
// Scores are formed in f64: a selection is whole numbers, and two pages' scores
// differ by less than an f32 sum's rounding often enough (one selection in ten
// thousand) that f32 would choose another page there than the definition does.

constexpr int SC = 256;

// Sixteen lanes a page, eight dims each (of HD 64: eight lanes).
template <int HD>
__global__ __launch_bounds__(SC) void page_score_kernel(SelectArgs a, int chunks) {
    constexpr int LP = HD / 8, PPW = SC / LP;  // lanes of a page; pages of a workgroup's step
    extern __shared__ double qs[];             // [group][2][HD]
    const int tid = threadIdx.x;
    const int unit = (int)(blockIdx.x / (unsigned)chunks), chunk = (int)(blockIdx.x % (unsigned)chunks);
    const int r = unit / a.kv_heads, kh = unit % a.kv_heads;
    const int t = a.row ? a.row[r] : r;
    if (t < 0 || t >= a.rows) return;
    const int tk = max(0, min(a.tk[r], a.wide << a.shift));
    const int live = (tk + (1 << a.shift) - 1) >> a.shift;
    const int share = (live + chunks - 1) / chunks, p0 = chunk * share, p1 = min(live, p0 + share);
    if (p0 >= p1) return;
    const float* q = a.q + (size_t)r * a.q_stride + (size_t)kh * a.group * HD;
    for (int e = tid; e < a.group * HD; e += SC) {
        const double x = (double)q[e];
        qs[e / HD * 2 * HD + e % HD] = x < 0.0 ? 0.0 : x;  // (a NaN stays one)
        qs[e / HD * 2 * HD + HD + e % HD] = x > 0.0 ? 0.0 : x;
    }
    __syncthreads();
    const int l = tid % LP;
    for (int p = p0 + tid / LP; p < p1; p += PPW) {
        const int id = a.table[(size_t)t * a.cols + p];
        const bool good = id >= 0 && id < a.pages;
        const half_t* b = reinterpret_cast<const half_t*>(a.bounds) + ((size_t)(good ? id : 0) * a.kv_heads + kh) * 2 * HD + 8 * l;
        const half8 mx = ld_h8(b), mn = ld_h8(b + HD);
        double best = -__builtin_inf();
        for (int g = 0; g < a.group; ++g) {
            const double* w = qs + g * 2 * HD + 8 * l;
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                s = __builtin_fma(w[j], (double)(float)mx[j], s);
                s = __builtin_fma(w[HD + j], (double)(float)mn[j], s);
            }
#pragma unroll
            for (int d = 1; d < LP; d <<= 1) s += __shfl_xor(s, d);
            best = fmax(best, s == s ? s : __builtin_inf());
        }
        // A page that the cache does not have: its keys make the row NaN, as they would be attended.
        if (!good) best = __builtin_inf();
        if (l == 0) a.score[(size_t)unit * a.wide + p] = best;
    }
}

// A score as bits that order as it does.
__device__ __forceinline__ uint64_t order(double s) {
    const uint64_t u = __builtin_bit_cast(uint64_t, s + 0.0);  // -0: 0
    return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

constexpr int SE = 256, DIGIT = 11;

// The `count` best pages of a (row, kv head): the border score by its digits
// from the top, each a histogram of the pages that agree above it, until the
// border's bin is taken whole; then the pages in order.
__global__ __launch_bounds__(SE) void page_select_kernel(SelectArgs a) {
    __shared__ int hist[1 << DIGIT];
    __shared__ int waves[2][SE / 64];
    __shared__ int found[3];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, unit = (int)blockIdx.x;
    const int r = unit / a.kv_heads;
    const int t = a.row ? a.row[r] : r;
    int* out = a.chosen + (size_t)unit * a.count;
    const int tk = max(0, min(a.tk[r], a.wide << a.shift));
    const int live = t < 0 || t >= a.rows ? 0 : (tk + (1 << a.shift) - 1) >> a.shift;
    if (live <= a.count) {
        for (int i = tid; i < a.count; i += SE) out[i] = i < live ? i : -1;
        return;
    }
    const double* score = a.score + (size_t)unit * a.wide;
    auto key = [&](int p) {
        return p < a.first || p >= live - a.last ? ~0ull : order(score[p]);
    };
    uint64_t border = 0, mask = 0;
    int need = a.count;  // of those that agree with the border above its digits so far
    for (int top = 64; top > 0;) {
        const int bits = min(DIGIT, top), low = top - bits;
        for (int i = tid; i < 1 << DIGIT; i += SE) hist[i] = 0;
        __syncthreads();
        for (int p = tid; p < live; p += SE) {
            const uint64_t k = key(p);
            if ((k & mask) == border) atomicAdd(&hist[(int)(k >> low) & ((1 << bits) - 1)], 1);
        }
        __syncthreads();
        if (wave == 0) {
            // From the top bin down: 64 lanes of 32 bins each.
            constexpr int B = (1 << DIGIT) / 64;
            int sum = 0;
            for (int i = 0; i < B; ++i) sum += hist[(63 - lane) * B + i];
            int upto = sum;
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const int y = __shfl_up(upto, d);
                if (lane >= d) upto += y;
            }
            if (upto >= need && upto - sum < need) {
                int left = need - (upto - sum), i = (63 - lane) * B + B - 1;
                while (hist[i] < left) left -= hist[i--];
                found[0] = i, found[1] = left, found[2] = hist[i];
            }
        }
        __syncthreads();
        border |= (uint64_t)found[0] << low;
        mask |= (uint64_t)((1 << bits) - 1) << low;
        need = found[1];
        top = low;
        const bool whole = found[2] == need;
        __syncthreads();
        if (whole) break;
    }
    // Pages above the border, and the first `need` at it.
    int above = 0, at = 0;
    for (int p0 = 0; p0 < live; p0 += SE) {
        const int p = p0 + tid;
        const uint64_t k = p < live ? key(p) & mask : 0;
        const bool gt = p < live && k > border, eq = p < live && k == border;
        const uint64_t mg = __ballot(gt), me = __ballot(eq), before = (1ull << lane) - 1;
        if (lane == 0) waves[0][wave] = __popcll(mg), waves[1][wave] = __popcll(me);
        __syncthreads();
        int g = above + __popcll(mg & before), e = at + __popcll(me & before);
        for (int w = 0; w < SE / 64; ++w) {
            if (w < wave) g += waves[0][w], e += waves[1][w];
            above += waves[0][w], at += waves[1][w];
        }
        if (gt || (eq && e < need)) out[g + min(e, need)] = p;
        __syncthreads();
    }
}

hipError_t launch_select(int hd, const SelectArgs& a, hipStream_t st) {
    const int units = a.nseq * a.kv_heads;
    if (a.wide > a.count) {
        // Workgroups of a (row, kv head) so that two a compute unit work, of 32 pages or more.
        const int chunks = std::max(1, std::min((a.wide + 31) / 32, (512 + units - 1) / units));
        const dim3 grid((unsigned)units * (unsigned)chunks);
        const size_t lds = (size_t)a.group * 2 * hd * sizeof(double);
        if (hd == 128) hipLaunchKernelGGL((page_score_kernel<128>), grid, dim3(SC), lds, st, a, chunks);
        else hipLaunchKernelGGL((page_score_kernel<64>), grid, dim3(SC), lds, st, a, chunks);
    }
    hipLaunchKernelGGL(page_select_kernel, dim3((unsigned)units), dim3(SE), 0, st, a);
    return hipGetLastError();
}

}  // namespace llmtie
