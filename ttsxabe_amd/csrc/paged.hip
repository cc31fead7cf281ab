// Attention of query rows over the pages of their sequences: a token of each of
// a batch, or rows of prompts. Row r sees positions of table row t of its own,
//
//   s_j = c tanh(scale q.k_j / c) - slope_h (tk - 1 - j),  out = sum_j p_j v_j,  p = softmax of s,
//
// the first `shared` ones and those from lo to tk (pages.hip's plan), or those of
// the pages that were selected for it. The plan's shared tiles attend what the
// rows of a group hold in the same pages once for up to 32 columns, a column
// being a row and one of a kv head's query heads; (m, l, O) of the parts are
// joined by a second launch.
//
// Products are S^T = K Q^T and O^T = V^T P^T with q and P as the sums of two f16
// (22 bits of each), so the context carries f32's precision off the f16 cache.
#include <algorithm>

#include "common.h"
#include "kvlayout.h"
#include "paged.h"
#include "scores.h"

namespace llmtie {

constexpr int PW = 4, PT = PW * LLMTIE_WAVE;

// What a wave does with 32 keys for NQT * 16 columns.
template <int HD, int MODE, int NQT>
struct Columns {
    static constexpr int NS = HD / 32, NT = HD / 16;
    half8 qh[NQT][NS], ql[NQT][NS];
    floatx4 o[NT][NQT];
    float m[NQT], l[NQT];
    float slope2[NQT];
    int at[NQT];  // SM_BIAS: the column's own position
    floatx4 sc[NQT][2];
    half8 ph[NQT], pl[NQT];
    float sl2, c1, c2;
    int grp;

    // Columns of `rows` rows from r0 on, `group` heads of kv head kh each.
    __device__ __forceinline__ void start(const PagedArgs& a, int r0, int rows, int kh, int lane, int tk) {
        const int col = lane & 15, n = rows * a.group;
        grp = lane >> 4;
        sl2 = a.scale * LLMTIE_LOG2E;
        c1 = (MODE & SM_CAP) != 0 ? a.scale / a.softcap : 0.0f;
        c2 = a.softcap * LLMTIE_LOG2E;
#pragma unroll
        for (int u = 0; u < NQT; ++u) {
            const int c = min(16 * u + col, n - 1), row = c / a.group, g = c % a.group;
            const bool has = 16 * u + col < n;
            const float* q = a.q + (size_t)(r0 + row) * a.q_stride + (size_t)(kh * a.group + g) * HD + 8 * grp;
#pragma unroll
            for (int s = 0; s < NS; ++s)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    half_t x, y;
                    split_h(has ? q[32 * s + j] : 0.0f, x, y);
                    qh[u][s][j] = x;
                    ql[u][s][j] = y;
                }
            if constexpr ((MODE & SM_BIAS) != 0) {
                slope2[u] = a.slopes[kh * a.group + g] * LLMTIE_LOG2E;
                at[u] = (tk >= 0 ? tk : min(a.tk[r0 + row], a.p.cols << a.p.shift)) - 1;
            }
            m[u] = RG_NOREF;
            l[u] = 0.0f;
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < NQT; ++u) o[t][u] = zero_f4();
    }
    __device__ __forceinline__ void scores(const half8 (&k)[2 * NS]) {
#pragma unroll
        for (int u = 0; u < NQT; ++u) sc[u][0] = sc[u][1] = zero_f4();
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int u = 0; u < NQT; ++u) {
                    sc[u][T] = mfma16(k[T * NS + s], ql[u][s], sc[u][T]);
                    sc[u][T] = mfma16(k[T * NS + s], qh[u][s], sc[u][T]);
                }
    }
    // Keys k0 ..; see(key): whether they are seen, where not all are.
    template <typename See>
    __device__ __forceinline__ void softmax(int k0, bool part, See&& see) {
#pragma unroll
        for (int u = 0; u < NQT; ++u) {
            if constexpr ((MODE & SM_CAP) != 0) cap_scores(sc[u], c1, sl2, c2);
            float mx = ninf();
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = k0 + 8 * grp + 4 * T + r;
                    float s = (MODE & SM_CAP) != 0 ? sc[u][T][r] : sc[u][T][r] * sl2;
                    if constexpr ((MODE & SM_BIAS) != 0) s = __builtin_fmaf(-slope2[u], (float)(at[u] - key), s);
                    if (part) s = see(key) ? s : ninf();
                    sc[u][T][r] = s;
                    mx = fmaxf(mx, s);
                }
            mx = max4grp(mx);
            if (__any(mx > m[u])) {
                const float mn = fmaxf(m[u], mx), fac = ex2(m[u] - mn);
                m[u] = mn;
                l[u] *= fac;
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t][u] *= fac;
            }
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // (The difference first: the key m is has 0, however large m is.)
                    const float p = ex2((sc[u][T][r] - m[u]) + RD_LIFT);
                    l[u] += p;
                    half_t x, y;
                    split_h(p, x, y);
                    ph[u][4 * T + r] = x;
                    pl[u][4 * T + r] = y;
                }
        }
    }
    __device__ __forceinline__ void values(const half8 (&v)[NT]) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < NQT; ++u) {
                o[t][u] = mfma16(v[t], pl[u], o[t][u]);
                o[t][u] = mfma16(v[t], ph[u], o[t][u]);
            }
    }
};

// LDS of a workgroup: the four waves' O rows, padded, and their (m, l).
template <int HD>
struct WaveParts {
    static constexpr int OP = HD + 4;
    float o[PW * PG_COLS * OP];
    float m[PW][PG_COLS], l[PW][PG_COLS];
};

// Where a tile's columns go: the context itself, or partials.
struct Sink {
    float* o;     // [columns][HD]
    float2* ml;   // null: the context
};

// The four waves' columns joined.
template <int HD, int MODE, int NQT>
__device__ __forceinline__ void join(WaveParts<HD>& w, Columns<HD, MODE, NQT>& c, int cols, const Sink& to, int tid) {
    constexpr int NT = HD / 16, OP = WaveParts<HD>::OP;
    const int lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int u = 0; u < NQT; ++u) {
        const float l = sum4grp(c.l[u]);
        if (16 * u + col >= cols) continue;
        const int at = wave * PG_COLS + 16 * u + col;
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<floatx4*>(&w.o[at * OP + 16 * t + 4 * grp]) = c.o[t][u];
        if (grp == 0) w.m[wave][16 * u + col] = c.m[u], w.l[wave][16 * u + col] = l;
    }
    __syncthreads();
    for (int e4 = tid; e4 < cols * (HD / 4); e4 += PT) {
        const int g = e4 / (HD / 4), d = 4 * (e4 % (HD / 4));
        float M = w.m[0][g], L = 0.0f;
#pragma unroll
        for (int k = 1; k < PW; ++k) M = fmaxf(M, w.m[k][g]);
        floatx4 y = zero_f4();
#pragma unroll
        for (int k = 0; k < PW; ++k) {
            const float f = ex2(w.m[k][g] - M);
            L += w.l[k][g] * f;
            y += *reinterpret_cast<const floatx4*>(&w.o[(k * PG_COLS + g) * OP + d]) * f;
        }
        if (!to.ml) y *= L > 0.0f || L != L ? 1.0f / L : 0.0f;
        *reinterpret_cast<floatx4*>(to.o + 4 * (size_t)e4) = y;
        if (to.ml && d == 0) to.ml[g] = make_float2(M, L);
    }
}

template <int HD, int AUX>
__device__ __forceinline__ void load_k(half8 (&k)[2 * (HD / 32)], const Region& r, int lane) {
#pragma unroll
    for (int j = 0; j < 2 * (HD / 32); ++j)
        k[j] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(r.r, 16 * lane + 1024 * j, 0, AUX));
}
template <int HD, int AUX>
__device__ __forceinline__ void load_v(half8 (&v)[HD / 16], const Region& r, int lane) {
#pragma unroll
    for (int j = 0; j < HD / 16; ++j)
        v[j] = __builtin_bit_cast(
            half8, __builtin_amdgcn_raw_buffer_load_b128(r.r, 16 * lane + 1024 * (2 * (HD / 32) + j), 0, AUX));
}

// One row's columns (a kv head's query heads), the waves taking every fourth
// block of positions begin to end of its list; place(i) is block i's first
// position, or -1. Bound by reading K and V: the next block's 16 loads a lane
// are in flight while one is computed.
template <int HD, int MODE, int AUX, typename Place>
__device__ __forceinline__ void one_row(const PagedArgs& a, WaveParts<HD>& w, int row, int table, int kh, int begin, int end,
                                        int f, int lo, int tk, const Sink& to, Place&& place) {
    constexpr int NS = HD / 32, NT = HD / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t stride = (size_t)a.kv_heads << (a.p.shift - 5);  // blocks of a page
    const int per = 1 << (a.p.shift - 5);
    Columns<HD, MODE, 1> c;
    int id = -1, pos = 0;
    bool bad = false;
    auto look = [&](int base) {
        const int i = base + wave + PW * lane;
        id = -1, pos = 0;
        if (i < end) {
            pos = place(i);
            if (pos >= 0) {
                const int at = pos >> a.p.shift;
                id = at < a.p.cols ? a.p.table[(size_t)table * a.p.cols + at] : -1;
                if (id < 0 || id >= a.p.pages) id = -1, bad = true;
            }
        }
    };
    struct Block {
        half8 k[2 * NS], v[NT];
    };
    auto load = [&](Block& x, int k) __attribute__((always_inline)) {
        const int i = __builtin_amdgcn_readlane(id, k), p = __builtin_amdgcn_readlane(pos, k);
        const Region r = region(reinterpret_cast<const char*>(a.p.cache) +
                                    ((size_t)max(i, 0) * stride + (size_t)kh * per + ((p >> 5) & (per - 1))) * (128 * HD),
                                i < 0 ? 0 : 128 * HD);
        load_k<HD, AUX>(x.k, r, lane);
        load_v<HD, AUX>(x.v, r, lane);
    };
    auto fold = [&](Block& x, int k) __attribute__((always_inline)) {
        if (__builtin_amdgcn_readlane(id, k) < 0) return;
        const int k0 = __builtin_amdgcn_readlane(pos, k);
        auto see = [&](int key) { return key < f || (key >= lo && key < tk); };
        const bool part = !(k0 + 32 <= f || (k0 >= lo && k0 + 32 <= tk));
        c.scores(x.k);
        c.softmax(k0, part, see);
        if (part) {
            // Values of keys not seen may be anything; 0 * NaN is NaN.
            const int grp = lane >> 4;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool on = see(k0 + 8 * grp + j);
#pragma unroll
                for (int t = 0; t < NT; ++t) x.v[t][j] = on ? x.v[t][j] : (half_t)0.0f;
            }
        }
        c.values(x.v);
    };
    bool any = false;
    Block x0, x1;
    for (int base = begin; base < end; base += PW * 64) {
        look(base);
        any = any || __any(bad);
        const int n = min(64, (end - base - wave + PW - 1) / PW);  // the wave's blocks
        if (n <= 0) break;
        load(x0, 0);
        load(x1, min(1, 63));
        if (base == begin) c.start(a, row, 1, kh, lane, tk);
        for (int k = 0; k < n; k += 2) {
            fold(x0, k);
            load(x0, min(k + 2, 63));
            if (k + 1 < n) fold(x1, k + 1);
            load(x1, min(k + 3, 63));
        }
    }
    if (begin + wave >= end) c.start(a, row, 1, kh, lane, tk);
    if (any) c.l[0] = __builtin_nanf("");
    join<HD, MODE, 1>(w, c, a.group, to, tid);
}

// A shared tile: up to 32 columns of `rows` rows from r0 on, every key of its
// blocks seen by all of them. The next block's keys are loaded once the scores
// have this one's, and its values once the products have them.
template <int HD, int MODE, int NQT>
__device__ __forceinline__ void shared_tile(const PagedArgs& a, WaveParts<HD>& w, int r0, int rows, int table, int kh,
                                            int first, int begin, int end, const Sink& to) {
    constexpr int NS = HD / 32, NT = HD / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const size_t stride = (size_t)a.kv_heads << (a.p.shift - 5);
    const int per = 1 << (a.p.shift - 5);
    Columns<HD, MODE, NQT> c;
    int id = -1;
    bool any = false;
    half8 k[2 * NS], v[NT];
    auto at = [&](int base, int i) __attribute__((always_inline)) {
        const int p = __builtin_amdgcn_readlane(id, i), b = first + base + wave + PW * i;
        return region(reinterpret_cast<const char*>(a.p.cache) +
                          ((size_t)max(p, 0) * stride + (size_t)kh * per + (b & (per - 1))) * (128 * HD),
                      p < 0 ? 0 : 128 * HD);
    };
    c.start(a, r0, rows, kh, lane, -1);
    for (int base = begin; base < end; base += PW * 64) {
        const int i = base + wave + PW * lane;
        id = -1;
        if (i < end) {
            const int p = (first + i) >> (a.p.shift - 5);
            id = p < a.p.cols ? a.p.table[(size_t)table * a.p.cols + p] : -1;
            if (id < 0 || id >= a.p.pages) id = -1, any = true;
        }
        const int n = min(64, (end - base - wave + PW - 1) / PW);
        if (n <= 0) break;
        Region r = at(base, 0);
        load_k<HD, 0>(k, r, lane);
        load_v<HD, 0>(v, r, lane);
        for (int j = 0; j < n; ++j) {
            const int k0 = 32 * (first + base + wave + PW * j);
            const Region next = at(base, min(j + 1, 63));
            c.scores(k);
            load_k<HD, 0>(k, next, lane);
            c.softmax(k0, false, [](int) { return true; });
            c.values(v);
            load_v<HD, 0>(v, next, lane);
        }
    }
    if (__any(any)) {
#pragma unroll
        for (int u = 0; u < NQT; ++u) c.l[u] = __builtin_nanf("");
    }
    join<HD, MODE, NQT>(w, c, rows * a.group, to, tid);
}

// Partials: own items' O, [item][kv head][group][HD]; shared ones', [item][kv
// head][PG_COLS][HD]; then (m, l) of both in the same order.
__device__ __forceinline__ Sink own_part(const PagedArgs& a, int hd, int item, int kh) {
    const size_t at = ((size_t)item * a.kv_heads + kh) * a.group;
    const size_t all = ((size_t)a.max_own * a.group + (size_t)a.max_shared * PG_COLS) * a.kv_heads;
    return Sink{a.part + at * hd, reinterpret_cast<float2*>(a.part + all * hd) + at};
}
__device__ __forceinline__ Sink shared_part(const PagedArgs& a, int hd, int item, int kh) {
    const size_t at = (size_t)a.max_own * a.group * a.kv_heads + ((size_t)item * a.kv_heads + kh) * PG_COLS;
    const size_t all = ((size_t)a.max_own * a.group + (size_t)a.max_shared * PG_COLS) * a.kv_heads;
    return Sink{a.part + at * hd, reinterpret_cast<float2*>(a.part + all * hd) + at};
}

__device__ __forceinline__ const int* plan_items(const PagedArgs& a) {
    return a.plan + PG_HEAD + (size_t)PG_ROW * a.nseq + (PG_ROW * (size_t)a.nseq % 16);
}
// Whether the plan is one of this call's sizes (a step's own is).
__device__ __forceinline__ bool plan_fits(const PagedArgs& a) {
    const int* h = a.plan;
    return h[2] == a.nseq && h[3] == a.group && h[4] == a.kv_heads && h[5] == a.p.shift && h[6] == a.p.cols &&
           h[7] == a.p.rows && h[8] == a.max_shared && h[9] == a.max_own && h[10] == !a.merge;
}

// Every element of a row's kv head.
__device__ __forceinline__ void fill(float* out, int n, float v) {
    for (int e = threadIdx.x; e < n; e += PT) out[e] = v;
}

template <int HD, int MODE, int AUX>
__global__ __launch_bounds__(PT, 2) void paged_kernel(PagedArgs a) {
    __shared__ __attribute__((aligned(16))) WaveParts<HD> w;
    const int kh = (int)(blockIdx.x % (unsigned)a.kv_heads), item = (int)(blockIdx.x / (unsigned)a.kv_heads);
    const int n = a.group * HD;
    const int* d = plan_items(a) + (size_t)PG_ITEM * item;
    if (!plan_fits(a)) {
        for (int r = item; r < a.nseq; r += a.items)
            fill(a.out + ((size_t)r * a.kv_heads + kh) * n, n, __builtin_nanf(""));
        return;
    }
    if (item >= a.plan[0]) return;
    const int row = d[0], rows = d[1], table = d[2], begin = d[8], end = d[9], ns = a.plan[1];
    if (item < ns) {
        const Sink to = shared_part(a, HD, item, kh);
        if (rows * a.group > 16) shared_tile<HD, MODE, 2>(a, w, row, rows, table, kh, d[5], begin, end, to);
        else shared_tile<HD, MODE, 1>(a, w, row, rows, table, kh, d[5], begin, end, to);
        return;
    }
    float* out = a.out + ((size_t)row * a.kv_heads + kh) * n;
    const Sink to = d[3] ? Sink{out, nullptr} : own_part(a, HD, item - ns, kh);
    if (table < 0) {
        fill(out, n, __builtin_nanf(""));
        return;
    }
    const int na = d[4], b0 = d[5], c0 = d[6], d0 = d[7];
    one_row<HD, MODE, AUX>(a, w, row, table, kh, begin, end, d[10], d[11], d[12], to, [&](int i) {
        const int j = i - na, x = c0 - b0;
        return 32 * (i < na ? i : j < x ? b0 + j : d0 + j - x);
    });
}

// Over selected pages: workgroup (row, kv head, run) takes its share of `count` pages' blocks.
template <int HD, int MODE, int AUX>
__global__ __launch_bounds__(PT, 2) void selected_kernel(PagedArgs a) {
    __shared__ __attribute__((aligned(16))) WaveParts<HD> w;
    const int kh = (int)(blockIdx.x % (unsigned)a.kv_heads), item = (int)(blockIdx.x / (unsigned)a.kv_heads);
    const int run = item % a.runs, row = item / a.runs, n = a.group * HD;
    const int table = a.row ? a.row[row] : row;
    const int tk = max(0, min(a.tk[row], a.p.cols << a.p.shift));
    float* out = a.out + ((size_t)row * a.kv_heads + kh) * n;
    const Sink to = a.runs == 1 ? Sink{out, nullptr} : own_part(a, HD, item, kh);
    const bool live = table >= 0 && table < a.p.rows;
    if (a.runs == 1 && !live) {
        fill(out, n, __builtin_nanf(""));
        return;
    }
    const int s = a.p.shift - 5, blocks = a.count << s;
    const int share = (blocks + a.runs - 1) / a.runs, begin = run * share, end = live ? min(blocks, begin + share) : 0;
    const int* chosen = a.chosen + ((size_t)row * a.kv_heads + kh) * a.count;
    one_row<HD, MODE, AUX>(a, w, row, table, kh, begin, end, 0, 0, tk, to, [&](int i) {
        const int p = chosen[i >> s];
        if (p < 0 || p >= a.p.cols) return -1;
        const int first = (p << a.p.shift) + 32 * (i & ((1 << s) - 1));
        return first < tk ? first : -1;
    });
}

// The parts of a row's columns of kv head kh: `on` of its own, then `sn` of its
// group's. None (n = 0): its item wrote the context.
template <int HD, bool PLAN>
struct Parts {
    int o0, on, s0 = 0, n, step = 0, col = 0;
    bool bad = false;  // no such table row
    __device__ __forceinline__ Parts(const PagedArgs& a, int row) {
        if constexpr (PLAN) {
            const int* d = a.plan + PG_HEAD + (size_t)PG_ROW * row;
            o0 = d[0], on = d[1], s0 = d[2], step = d[4], col = d[5];
            n = on == 1 && d[3] == 0 ? 0 : on + d[3];
        } else {
            const int table = a.row ? a.row[row] : row;
            bad = table < 0 || table >= a.p.rows;
            o0 = row * a.runs, on = n = a.runs;
        }
    }
    // The i-th part's O and (m, l) of query head g.
    __device__ __forceinline__ Sink of(const PagedArgs& a, int i, int kh, int g) const {
        Sink p = i < on ? own_part(a, HD, o0 + i, kh) : shared_part(a, HD, s0 + (i - on) * step, kh);
        const int at = g + (i < on ? 0 : col);
        p.o += (size_t)at * HD, p.ml += at;
        return p;
    }
};

// The context from its parts, in their order: M = max m, O = sum 2^(m - M) O / sum
// 2^(m - M) l. A part in which a row sees no key has m = RG_NOREF and l = 0.
//
// Many rows, of few parts each: a thread takes four dims of a (row, head) (244
// rows of 20 heads of 64, by a workgroup a (row, head) as below 13.8 us, so 7.3).
template <int HD, bool PLAN>
__global__ __launch_bounds__(PT) void paged_merge_rows_kernel(PagedArgs a) {
    constexpr int C = HD / 4, U = 4;
    const long i = (long)blockIdx.x * PT + threadIdx.x;
    const int heads = a.kv_heads * a.group, c = (int)(i % C), h = (int)(i / C % heads);
    const long row = i / C / heads;
    if (row >= a.nseq || (PLAN && !plan_fits(a))) return;
    const Parts<HD, PLAN> p(a, (int)row);
    float* out = a.out + 4 * i;
    const int kh = h / a.group, g = h % a.group;
    if (p.bad) {
        *reinterpret_cast<floatx4*>(out) = zero_f4() + __builtin_nanf("");
        return;
    }
    if (p.n == 0) return;
    float M = RG_NOREF, L = 0.0f;
    floatx4 y = zero_f4();
    for (int s0 = 0; s0 < p.n; s0 += U) {
        float2 ml[U];
        floatx4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const Sink s = p.of(a, min(s0 + u, p.n - 1), kh, g);
            ml[u] = *s.ml;
            x[u] = *reinterpret_cast<const floatx4*>(s.o + 4 * c);
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < U; ++u) mn = fmaxf(mn, ml[u].x);
        const float f = ex2(M - mn);
        M = mn;
        L *= f;
        y *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= p.n) break;
            const float w = ex2(ml[u].x - M);
            L += ml[u].y * w;
            y += x[u] * w;
        }
    }
    *reinterpret_cast<floatx4*>(out) = y * (L > 0.0f || L != L ? 1.0f / L : 0.0f);
}

// Few rows: a workgroup a (row, query head), the threads HD / 4 columns of four
// dims by phases of the parts, whose loads go out together (one sequence of 32
// parts, all four heads by one thread a column: 12.4 us, so 3.9).
constexpr int PM_PARTS = 1088;  // parts of a row at most: each side's target and one

template <int HD, bool PLAN>
__global__ __launch_bounds__(PT) void paged_merge_kernel(PagedArgs a) {
    constexpr int C = HD / 4, R = PT / C, U = 4;
    __shared__ float wt[PM_PARTS];
    __shared__ floatx4 red[PT];
    const int heads = a.kv_heads * a.group, h = (int)(blockIdx.x % (unsigned)heads);
    const int row = (int)(blockIdx.x / (unsigned)heads), kh = h / a.group;
    const int tid = threadIdx.x, c = tid % C, phase = tid / C, lane = tid & 63;
    if (PLAN && !plan_fits(a)) return;
    const Parts<HD, PLAN> p(a, row);
    float* out = a.out + (size_t)blockIdx.x * HD;
    if (p.bad) {
        fill(out, HD, __builtin_nanf(""));
        return;
    }
    const int n = min(p.n, PM_PARTS);
    if (n == 0) return;
    auto part = [&](int i) { return p.of(a, i, kh, h % a.group); };
    // The first parts' columns are on their way while the weights are formed.
    floatx4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
        x[u] = *reinterpret_cast<const floatx4*>(part(min(phase + u * R, n - 1)).o + 4 * c);
    float M = RG_NOREF, L = 0.0f;
    for (int i = lane; i < n; i += 64) M = fmaxf(M, part(i).ml->x);
    M = wave_max(M);
    for (int i = lane; i < n; i += 64) {
        const float2 ml = *part(i).ml;
        const float f = ex2(ml.x - M);
        L += ml.y * f;
        if (tid < 64) wt[i] = f;
    }
    L = wave_sum(L);
    __syncthreads();
    floatx4 y = zero_f4();
    for (int i = phase; i < n; i += U * R) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (i + u * R < n) y += x[u] * wt[i + u * R];
            x[u] = *reinterpret_cast<const floatx4*>(part(min(i + (U + u) * R, n - 1)).o + 4 * c);
        }
    }
    red[tid] = y;
    __syncthreads();
    if (phase == 0) {
        for (int k = 1; k < R; ++k) y += red[tid + k * C];
        *reinterpret_cast<floatx4*>(out + 4 * c) = y * (L > 0.0f || L != L ? 1.0f / L : 0.0f);
    }
}

hipError_t launch_paged(int hd, const PagedArgs& a, hipStream_t st) {
    const int mode = (a.softcap > 0.0f ? SM_CAP : 0) | (a.slopes ? SM_BIAS : 0);
    const dim3 grid((unsigned)((a.plan ? (size_t)a.items : (size_t)a.nseq * a.runs) * a.kv_heads));
    bool done = false;
#define PK(HD, M, AUX)                                                                           \
    if (!done && hd == HD && mode == M && (a.stream ? AUX_STREAM : 0) == AUX) {                  \
        if (a.plan) hipLaunchKernelGGL((paged_kernel<HD, M, AUX>), grid, dim3(PT), 0, st, a);    \
        else hipLaunchKernelGGL((selected_kernel<HD, M, AUX>), grid, dim3(PT), 0, st, a);        \
        done = true;                                                                             \
    }
#define PM(HD, M) PK(HD, M, 0) PK(HD, M, AUX_STREAM)
    PM(64, 0) PM(64, 1) PM(64, 2) PM(64, 3) PM(128, 0) PM(128, 1) PM(128, 2) PM(128, 3)
#undef PM
#undef PK
    if (!done) return hipErrorInvalidValue;
    if (a.merge) {
        const size_t rows = (size_t)a.nseq * a.kv_heads * a.group;
#define MK(HD, P)                                                                                              \
    if (hd == HD && (a.plan != nullptr) == P) {                                                                \
        if (rows >= 2048)                                                                                      \
            hipLaunchKernelGGL((paged_merge_rows_kernel<HD, P>), dim3((unsigned)((rows * (HD / 4) + PT - 1) / PT)), \
                               dim3(PT), 0, st, a);                                                            \
        else hipLaunchKernelGGL((paged_merge_kernel<HD, P>), dim3((unsigned)rows), dim3(PT), 0, st, a);        \
    }
        MK(64, false) MK(64, true) MK(128, false) MK(128, true)
#undef MK
    }
    return hipGetLastError();
}

}  // namespace llmtie
