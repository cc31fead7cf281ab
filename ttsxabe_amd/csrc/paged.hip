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

typedef float floatx2 __attribute__((ext_vector_type(2)));
typedef _Float16 halfx2 __attribute__((ext_vector_type(2)));

// What a wave does with 32 keys for NQT * 16 columns.
template <int HD, int MODE, int NQT>
struct Columns {
    static constexpr int NS = HD / 32, NT = HD / 16;
    // q goes through LDS, as the four waves' columns are the same. Its lower halves, of two
    // tiles, stay there (in registers too, 210 of them spilled at HD 128).
    static constexpr bool LOW_LDS = NQT > 1;
    half8 qh[NQT][NS], ql[LOW_LDS ? 1 : NQT][LOW_LDS ? 1 : NS];
    const half8* low;
    floatx4 o[NT][NQT];
    // Weights are 2^(s - m), up to 2^RD_LIFT, and l their sum. The reference m is the
    // largest score less RD_LIFT, or as it is past 2^23, where that is not exact.
    float m[NQT], l[NQT];
    float slope2[NQT];
    int at[NQT];  // SM_BIAS: the column's own position
    floatx4 sc[NQT][2];
    half8 ph[NQT], pl[NQT];
    float sl2, c1, c2;
    int grp;

    // Columns of `rows` rows from r0 on, `group` heads of kv head kh each (past the last
    // one: that one again, which nobody keeps): their queries on the way, a quarter a
    // wave. A row's position is that of its length, also where it is alone in a shared tile
    // (whose ColumnSees has no end).
    static constexpr int QP = (NQT * NS + PW - 1) / PW;  // (tile, 32 dims) pairs of a wave
    floatx4 raw[QP][2];
    __device__ __forceinline__ void fetch(const PagedArgs& a, int r0, int rows, int kh, int lane, int wave) {
        const int col = lane & 15, n = rows * a.group;
        grp = lane >> 4;
        auto column = [&](int u, int& row, int& g) {
            const int c = min(16 * u + col, n - 1);
            row = rows == 1 ? 0 : c / a.group, g = c - row * a.group;
        };
#pragma unroll
        for (int i = 0; i < QP; ++i) {
            const int p = min(wave + PW * i, NQT * NS - 1);
            int row, g;
            column(p / NS, row, g);
            const float* q = a.q + (size_t)(r0 + row) * a.q_stride + (size_t)(kh * a.group + g) * HD + 8 * grp + 32 * (p % NS);
            __builtin_memcpy(&raw[i][0], q, 16);  // (4-byte aligned)
            __builtin_memcpy(&raw[i][1], q + 4, 16);
        }
        if constexpr ((MODE & SM_BIAS) != 0) {
#pragma unroll
            for (int u = 0; u < NQT; ++u) {
                int row, g;
                column(u, row, g);
                slope2[u] = a.slopes[kh * a.group + g] * LLMTIE_LOG2E;
                at[u] = min(a.tk[r0 + row], a.p.cols << a.p.shift) - 1;
            }
        }
    }
    // (With a barrier.)
    __device__ __forceinline__ void start(const PagedArgs& a, int lane, int wave, half8* mem) {
        sl2 = a.scale * LLMTIE_LOG2E;
        c1 = (MODE & SM_CAP) != 0 ? a.scale / a.softcap : 0.0f;
        c2 = a.softcap * LLMTIE_LOG2E;
        low = mem + NQT * NS * 64;
#pragma unroll
        for (int i = 0; i < QP; ++i) {
            const int p = min(wave + PW * i, NQT * NS - 1);
            half8 hi, lo;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                half_t x, y;
                split_h(raw[i][j / 4][j % 4], x, y);
                hi[j] = x, lo[j] = y;
            }
            mem[p * 64 + lane] = hi, mem[(NQT * NS + p) * 64 + lane] = lo;
        }
#pragma unroll
        for (int u = 0; u < NQT; ++u) m[u] = RG_NOREF, l[u] = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < NQT; ++u) o[t][u] = zero_f4();
        lds_barrier();
#pragma unroll
        for (int u = 0; u < NQT; ++u)
#pragma unroll
            for (int s = 0; s < NS; ++s) {
                qh[u][s] = mem[(u * NS + s) * 64 + lane];
                if constexpr (!LOW_LDS) ql[u][s] = low[(u * NS + s) * 64 + lane];
            }
    }
    __device__ __forceinline__ half8 lower(int u, int s, int lane) const {
        if constexpr (LOW_LDS) return low[(u * NS + s) * 64 + lane];
        else return ql[u][s];
    }
    __device__ __forceinline__ void scores(const half8 (&k)[2 * NS]) {
#pragma unroll
        for (int u = 0; u < NQT; ++u) sc[u][0] = sc[u][1] = zero_f4();
        int lane = threadIdx.x & 63;
        if constexpr (LOW_LDS) asm volatile("" : "+v"(lane));  // read each time, not held over the blocks
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int u = 0; u < NQT; ++u) {
                const half8 lo = lower(u, s, lane);
#pragma unroll
                for (int T = 0; T < 2; ++T) {
                    sc[u][T] = mfma16(k[T * NS + s], lo, sc[u][T]);
                    sc[u][T] = mfma16(k[T * NS + s], qh[u][s], sc[u][T]);
                }
            }
    }
    // Keys k0 ..; see(u, key): whether this lane's column of sixteen u sees them, where not all are.
    template <typename See>
    __device__ __forceinline__ void softmax(int k0, bool part, See&& see) {
#pragma unroll
        for (int u = 0; u < NQT; ++u) {
            if constexpr ((MODE & SM_CAP) != 0) cap_scores(sc[u], c1, sl2, c2);
            float mx = ninf();
            // The distance of the lane's first key (below 2^24 exact, as those of its others are).
            const float far = (MODE & SM_BIAS) != 0 ? (float)(at[u] - k0 - 8 * grp) : 0.0f;
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int key = k0 + 8 * grp + 4 * T + r;
                    float s = (MODE & SM_CAP) != 0 ? sc[u][T][r] : sc[u][T][r] * sl2;
                    if constexpr ((MODE & SM_BIAS) != 0) s = __builtin_fmaf(-slope2[u], far - (float)(4 * T + r), s);
                    if (part) s = see(u, key) ? s : ninf();
                    sc[u][T][r] = s;
                    mx = fmaxf(mx, s);
                }
            mx = max4grp(mx);
            const bool more = mx - m[u] > RD_LIFT;
            if (__any(more)) {
                const float to = !more ? m[u] : fabsf(mx) < 0x1p23f ? mx - RD_LIFT : mx, fac = ex2(m[u] - to);
                m[u] = to;
                l[u] *= fac;
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t][u] *= fac;
            }
            // Upper halves two at a time, and what is left of each in one instruction.
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int r = 0; r < 4; r += 2) {
                    floatx2 p = {ex2(sc[u][T][r] - m[u]), ex2(sc[u][T][r + 1] - m[u])};
                    l[u] += p[0];
                    l[u] += p[1];
                    const halfx2 x = __builtin_convertvector(p, halfx2);
                    p[0] = __builtin_fmaf(-(float)x[0], 1.0f, p[0]);
                    p[1] = __builtin_fmaf(-(float)x[1], 1.0f, p[1]);
                    const halfx2 y = __builtin_convertvector(p, halfx2);
                    ph[u][4 * T + r] = x[0], ph[u][4 * T + r + 1] = x[1];
                    pl[u][4 * T + r] = y[0], pl[u][4 * T + r + 1] = y[1];
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

// LDS of a workgroup: sixteen of the four waves' O rows, padded, and their (m, l).
template <int HD>
struct WaveParts {
    static constexpr int OP = HD + 4;
    float o[PW * 16 * OP];
    float m[PW][16], l[PW][16];
    half8 q[2 * 2 * (HD / 32) * 64];  // Columns::start
};

// Where a tile's columns go: the context itself (a row's heads together, rows
// `stride` apart), or partials.
struct Sink {
    float* o;
    float2* ml;   // null: the context
    long stride;  // elements from a row's columns to the next one's
};

// The four waves' columns joined, sixteen at a time. CHECK: false, with nothing
// written, where something is not finite.
template <int HD, int MODE, int NQT, bool CHECK>
__device__ __forceinline__ bool join(WaveParts<HD>& w, Columns<HD, MODE, NQT>& c, int group, int cols, const Sink& to,
                                     int tid) {
    constexpr int NT = HD / 16, OP = WaveParts<HD>::OP;
    const int lane = tid & 63, wave = tid >> 6, col = lane & 15, grp = lane >> 4;
    bool odd = false;
    if constexpr (CHECK) {
        float x = 0.0f;
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < NQT; ++u) x += (c.o[t][u][0] + c.o[t][u][1]) + (c.o[t][u][2] + c.o[t][u][3]);
        odd = !(x - x == 0.0f);
    }
#pragma unroll
    for (int u = 0; u < NQT; ++u) {
        if (16 * u >= cols) break;
        const int n = min(16, cols - 16 * u);
        const float l = sum4grp(c.l[u]);
        if (u) __syncthreads();
        if (col < n) {
#pragma unroll
            for (int t = 0; t < NT; ++t)
                *reinterpret_cast<floatx4*>(&w.o[(wave * 16 + col) * OP + 16 * t + 4 * grp]) = c.o[t][u];
            if (grp == 0) w.m[wave][col] = c.m[u], w.l[wave][col] = l;
        }
        if (CHECK && u == 0) {
            if (__syncthreads_or(odd)) return false;
        } else {
            __syncthreads();
        }
        for (int e4 = tid; e4 < n * (HD / 4); e4 += PT) {
            const int g = e4 / (HD / 4), d = 4 * (e4 % (HD / 4)), at = 16 * u + g;
            float M = w.m[0][g], L = 0.0f;
#pragma unroll
            for (int k = 1; k < PW; ++k) M = fmaxf(M, w.m[k][g]);
            floatx4 y = zero_f4();
#pragma unroll
            for (int k = 0; k < PW; ++k) {
                const float f = ex2(w.m[k][g] - M);
                L += w.l[k][g] * f;
                y += *reinterpret_cast<const floatx4*>(&w.o[(k * 16 + g) * OP + d]) * f;
            }
            if (!to.ml) y *= L > 0.0f || L != L ? 1.0f / L : 0.0f;
            *reinterpret_cast<floatx4*>(to.o + (size_t)(at / group) * to.stride + (at % group) * HD + d) = y;
            if (to.ml && d == 0) to.ml[at] = make_float2(M, L);
        }
    }
    return true;
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

// A wave's blocks of an item, every fourth from `base` on: lane k holds the
// k-th's first position, its page (-1: nothing to read) and which of a tile's rows
// see it, 64 looked up at a time.
struct Blocks {
    int pos, id;
    uint32_t rows;
    // place(i, rows): block i's first position, or -1. Returns whether a page that is needed is not there.
    template <typename Place>
    __device__ __forceinline__ bool look(const PagedArgs& a, int table, int i, int end, Place&& place) {
        id = -1, pos = 0, rows = 0;
        if (i >= end) return false;
        pos = place(i, rows);
        if (pos < 0) return false;
        const int at = pos >> a.p.shift;
        id = at < a.p.cols ? a.p.table[(size_t)table * a.p.cols + at] : -1;
        if (id >= 0 && id < a.p.pages) return false;
        id = -1;
        return true;
    }
    template <int HD>
    __device__ __forceinline__ Region block(const PagedArgs& a, int kh, int k) const {
        const int i = __builtin_amdgcn_readlane(id, k), p = __builtin_amdgcn_readlane(pos, k), s = a.p.shift - 5;
        const size_t b = (((size_t)max(i, 0) * a.kv_heads + kh) << s) + ((p >> 5) & ((1 << s) - 1));
        return region(reinterpret_cast<const char*>(a.p.cache) + b * (128 * HD), i < 0 ? 0 : 128 * HD);
    }
    __device__ __forceinline__ bool has(int k) const { return __builtin_amdgcn_readlane(id, k) >= 0; }
    __device__ __forceinline__ int key0(int k) const { return __builtin_amdgcn_readlane(pos, k); }
};

// One row's columns (a kv head's query heads), the waves taking every fourth
// of blocks begin to end. Bound by reading K and V: the next block's 16 loads a lane
// are in flight while one is computed. Returns false, with nothing written, where
// something is not finite (see tile).
template <int HD, int MODE, int AUX, typename Place>
__device__ __forceinline__ bool one_row(const PagedArgs& a, WaveParts<HD>& w, int row, int table, int kh, int begin, int end,
                                        int f, int lo, int tk, const Sink& to, Place&& place) {
    constexpr int NS = HD / 32, NT = HD / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Columns<HD, MODE, 1> c;
    Blocks at;
    struct Block {
        half8 k[2 * NS], v[NT];
    };
    auto load = [&](Block& x, int k) __attribute__((always_inline)) {
        const Region r = at.block<HD>(a, kh, k);
        load_k<HD, AUX>(x.k, r, lane);
        load_v<HD, AUX>(x.v, r, lane);
    };
    auto fold = [&](Block& x, int k) __attribute__((always_inline)) {
        if (!at.has(k)) return;
        const int k0 = at.key0(k);
        auto see = [&](int, int key) { return key < f || (key >= lo && key < tk); };
        const bool part = !(k0 + 32 <= f || (k0 >= lo && k0 + 32 <= tk));
        c.scores(x.k);
        c.softmax(k0, part, see);
        if (part) {
            // Values of keys not seen may be anything; 0 * NaN is NaN.
            const int grp = lane >> 4;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool on = see(0, k0 + 8 * grp + j);
#pragma unroll
                for (int t = 0; t < NT; ++t) x.v[t][j] = on ? x.v[t][j] : (half_t)0.0f;
            }
        }
        c.values(x.v);
    };
    Block x0, x1;
    c.fetch(a, row, 1, kh, lane, wave);
    bool none = at.look(a, table, begin + wave + PW * lane, end, place), gone = __any(none);
    load(x0, 0);
    c.start(a, lane, wave, w.q);
    load(x1, 1);
    for (int base = begin; base < end; base += PW * 64) {
        const int n = min(64, (end - base - wave + PW - 1) / PW);  // the wave's blocks
        if (n <= 0) break;
        if (base != begin) {
            none = at.look(a, table, base + wave + PW * lane, end, place);
            gone = gone || __any(none);
            load(x0, 0);
            load(x1, 1);
        }
        for (int k = 0; k < n; k += 2) {
            fold(x0, k);
            load(x0, min(k + 2, 63));
            if (k + 1 < n) fold(x1, k + 1);
            load(x1, min(k + 3, 63));
        }
    }
    if (gone) c.l[0] = __builtin_nanf("");
    return join<HD, MODE, 1, true>(w, c, a.group, a.group, to, tid);
}

// What a column of a tile sees: the first f positions and those from lo to tk.
struct ColumnSees {
    int f, lo, tk;
};

// A tile: up to 32 columns of `rows` rows of one sequence or of one shared prefix, from r0
// on. The next block's keys are loaded once the scores have this one's, and its
// values once the products have them. Each row sees keys of its own, sees(i) of the
// tile's i-th one (of a shared prefix, all; one function for both, whose pieces the compiler
// else merges at the price of 100 spilled registers).
//
// Returns false, with nothing written, where something is not finite. A value that a row
// does not see, or whose weight's lower half is 0 or below, may then have made a NaN of an
// infinity or of nothing; the rows are taken again one by one (ONE): values that
// the row does not see are cleared, and those that are not finite are added as they are.
template <int HD, int MODE, int NQT, bool ONE, typename Place, typename Sees>
__device__ __forceinline__ bool tile(const PagedArgs& a, WaveParts<HD>& w, int r0, int rows, int table, int kh, int begin,
                                     int end, const Sink& to, Place&& place, Sees&& sees) {
    constexpr int NS = HD / 32, NT = HD / 16;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Columns<HD, MODE, NQT> c;
    Blocks at;
    half8 k[2 * NS], v[NT];
    ColumnSees own[NQT];
    int bit[NQT];
    c.fetch(a, r0, rows, kh, lane, wave);
#pragma unroll
    for (int u = 0; u < NQT; ++u) {
        bit[u] = rows == 1 ? 0 : min(16 * u + (lane & 15), rows * a.group - 1) / a.group;
        own[u] = sees(bit[u]);
    }
    bool none = at.look(a, table, begin + wave + PW * lane, end, place), gone = __any(none);
    Region r = at.block<HD>(a, kh, 0);
    load_k<HD, 0>(k, r, lane);
    load_v<HD, 0>(v, r, lane);
    c.start(a, lane, wave, w.q);
    for (int base = begin; base < end; base += PW * 64) {
        const int n = min(64, (end - base - wave + PW - 1) / PW);
        if (n <= 0) break;
        if (base != begin) {
            none = at.look(a, table, base + wave + PW * lane, end, place);
            gone = gone || __any(none);
            r = at.block<HD>(a, kh, 0);
            load_k<HD, 0>(k, r, lane);
            load_v<HD, 0>(v, r, lane);
        }
        for (int j = 0; j < n; ++j) {
            const int k0 = at.key0(j);
            const Region next = at.block<HD>(a, kh, min(j + 1, 63));
            if (ONE && !at.has(j)) {  // not this row's
                load_k<HD, 0>(k, next, lane);
                load_v<HD, 0>(v, next, lane);
                continue;
            }
            ColumnSees now[NQT];
            const uint32_t on = ONE ? 1u : (uint32_t)__builtin_amdgcn_readlane((int)at.rows, j);
            bool some = false;
#pragma unroll
            for (int u = 0; u < NQT; ++u) {
                now[u] = on >> bit[u] & 1 ? own[u] : ColumnSees{0, 0, 0};
                some = some || !(k0 + 32 <= now[u].f || (k0 >= now[u].lo && k0 + 32 <= now[u].tk));
            }
            c.scores(k);
            load_k<HD, 0>(k, next, lane);
            c.softmax(k0, __any(some),
                      [&](int u, int key) { return key < now[u].f || (key >= now[u].lo && key < now[u].tk); });
            if constexpr (ONE) {
                half8 one;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int key = k0 + 8 * (lane >> 4) + i;
                    one[i] = key < now[0].f || (key >= now[0].lo && key < now[0].tk) ? (half_t)1.0f : (half_t)0.0f;
                }
#pragma unroll
                for (int t = 0; t < NT; ++t) {
                    half8 odd;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const half_t x = one[i] != (half_t)0.0f ? v[t][i] : (half_t)0.0f;
                        const bool fine = x - x == (half_t)0.0f;
                        v[t][i] = fine ? x : (half_t)0.0f;
                        odd[i] = fine ? (half_t)0.0f : x;
                    }
                    c.o[t][0] = mfma16(odd, one, c.o[t][0]);
                }
            }
            c.values(v);
            load_v<HD, 0>(v, next, lane);
        }
    }
    // (Of a tile, not finite: other rows may do without that page.)
    if (gone) {
        if constexpr (ONE) c.l[0] = __builtin_nanf("");
        else c.o[0][0][0] = __builtin_nanf("");
    }
    return join<HD, MODE, NQT, !ONE>(w, c, a.group, rows * a.group, to, tid);
}

// Partials: own items' O, [item][kv head][group][HD]; wide ones' (tiles'), [item][kv
// head][PG_COLS][HD]; then (m, l) of both in the same order.
__device__ __forceinline__ Sink part_at(const PagedArgs& a, int hd, size_t at) {
    const size_t all = ((size_t)a.max_own * a.group + (size_t)a.max_wide * PG_COLS) * a.kv_heads;
    return Sink{a.part + at * hd, reinterpret_cast<float2*>(a.part + all * hd) + at, (long)a.group * hd};
}
__device__ __forceinline__ Sink own_part(const PagedArgs& a, int hd, int item, int kh) {
    return part_at(a, hd, ((size_t)item * a.kv_heads + kh) * a.group);
}
__device__ __forceinline__ Sink wide_part(const PagedArgs& a, int hd, int item, int kh) {
    return part_at(a, hd, (size_t)a.max_own * a.group * a.kv_heads + ((size_t)item * a.kv_heads + kh) * PG_COLS);
}
__device__ __forceinline__ Sink context(const PagedArgs& a, int hd, int row, int kh) {
    return Sink{a.out + ((size_t)row * a.kv_heads + kh) * a.group * hd, nullptr, (long)a.kv_heads * a.group * hd};
}
// The columns of a tile's row.
__device__ __forceinline__ Sink row_of(const PagedArgs& a, int hd, const Sink& tile, int row) {
    return Sink{tile.o + row * tile.stride, tile.ml ? tile.ml + row * a.group : nullptr, tile.stride};
}

__device__ __forceinline__ const int* plan_row(const PagedArgs& a, int row) {
    return a.plan + PG_HEAD + (size_t)PG_ROW * row;
}
__device__ __forceinline__ const int* plan_item(const PagedArgs& a, int item) {
    return a.plan + plan_items_at(a.nseq) + (size_t)PG_ITEM * item;
}
// Whether the plan is one of this call's sizes (a step's own is).
__device__ __forceinline__ bool plan_fits(const PagedArgs& a) {
    const int* h = a.plan;
    return h[2] == a.nseq && h[3] == a.group && h[4] == a.kv_heads && h[5] == a.p.shift && h[6] == a.p.cols &&
           h[7] == a.p.rows && h[8] == a.max_wide && h[9] == a.max_own && h[10] == !a.merge;
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
    const int* d = plan_item(a, item);
    if (!plan_fits(a)) {
        for (int r = item; r < a.nseq; r += a.items) fill(context(a, HD, r, kh).o, n, __builtin_nanf(""));
        return;
    }
    if (item >= a.plan[0]) return;
    const int row = d[0], table = d[2], flags = d[3], begin = d[8], end = d[9], wide = a.plan[1];
    int rows = d[1];
    const int na = d[4], b0 = d[5], c0 = d[6], d0 = d[7];
    Sink to = flags & PG_WHOLE ? context(a, HD, row, kh)
              : item < wide    ? wide_part(a, HD, item, kh)
                               : own_part(a, HD, item - wide, kh);
    if (table < 0) {
        fill(to.o, n, __builtin_nanf(""));
        return;
    }
    auto place = [&](int i, uint32_t& on) {
        const int j = i - na, x = c0 - b0;
        on = ~0u;
        return 32 * (i < na ? i : j < x ? b0 + j : d0 + j - x);
    };
    const bool two = rows * a.group > 16, shared = (flags & PG_SHARED) != 0;
    auto sees = [&](int i) {
        const int* p = plan_row(a, row + i) + 8;
        return shared ? ColumnSees{0, 0, 0x7fffffff} : ColumnSees{p[0], p[1], p[2]};
    };
    if (rows == 1) {
        const ColumnSees s = sees(0);
        if (one_row<HD, MODE, AUX>(a, w, row, table, kh, begin, end, s.f, s.lo, s.tk, to, place)) return;
    } else if (two ? tile<HD, MODE, 2, false>(a, w, row, rows, table, kh, begin, end, to, place, sees)
                   : tile<HD, MODE, 1, false>(a, w, row, rows, table, kh, begin, end, to, place, sees)) {
        return;
    }
    for (int i = 0; i < rows; ++i) {
        const ColumnSees of = sees(i);
        auto of_row = [&](int b, uint32_t& on) {
            const int p = place(b, on);
            return p < of.f || (p + 32 > of.lo && p < of.tk) ? p : -1;
        };
        tile<HD, MODE, 1, true>(a, w, row + i, 1, table, kh, begin, end, row_of(a, HD, to, i), of_row,
                                [&](int) { return of; });
        __syncthreads();  // the join's arrays
    }
}

// The rows of a selection that are attended together: those of an aligned tile of
// rows that follow one another and whose sequence is one. (By a whole wave.)
struct Together {
    int tile, r0, rows, table;  // rows: 1 where they are taken one by one
    __device__ __forceinline__ Together(const PagedArgs& a, int row) {
        const int per = PG_TILE_ROWS(a.group), lane = threadIdx.x & 63;
        tile = row / per, r0 = tile * per;
        if (!a.together) {
            r0 = row, rows = 1, table = a.row ? a.row[row] : row;
            return;
        }
        const int n = min(per, a.nseq - r0), at = row - r0;
        const int t = a.row ? a.row[r0 + min(lane, n - 1)] : r0 + lane;
        table = __builtin_amdgcn_readlane(t, at);
        // Bits of the rows that differ: the nearest on each side of this one.
        const uint64_t other = ~__ballot(lane < n && t == table);
        const uint64_t below = other & ((1ull << at) - 1), above = other >> at;
        const int first = below ? 64 - __clzll(below) : 0, last = at + __ffsll((long long)above) - 1;
        r0 += first, rows = last - first;
        if (a.p.cols > PG_UNION || table < 0 || table >= a.p.rows) r0 = row, rows = 1;
    }
    __device__ __forceinline__ int runs(const PagedArgs& a) const {
        return rows == 1 ? a.runs : min(a.tile_runs, rows * a.runs);
    }
};
// What the join has to know of a row: its place in its tile's rows and their count;
// whether its table row is missing.
__device__ __forceinline__ int* row_note(const PagedArgs& a, int hd, int row) {
    const size_t all = ((size_t)a.max_own * a.group + (size_t)a.max_wide * PG_COLS) * a.kv_heads;
    return reinterpret_cast<int*>(a.part + all * (hd + 2)) + row;
}

// Over selected pages: workgroup (row, kv head, run) takes its share of `count`
// pages' blocks. Rows of one sequence mostly select the same pages (neighbours of a
// prompt), so a tile of them walks the pages that any of them selected, each read once,
// its workgroups being those of its rows (127 rows over 24 pages each of 32/8/128,
// row by row 42.5 us, so 34.5).
template <int HD, int MODE>
__global__ __launch_bounds__(PT, 2) void selected_kernel(PagedArgs a) {
    __shared__ __attribute__((aligned(16))) WaveParts<HD> w;
    __shared__ uint32_t mask[PG_UNION];   // rows that selected a page, a bit each
    __shared__ uint16_t list[PG_UNION];   // the pages that some row selected
    __shared__ int waves[PW];
    const int kh = (int)(blockIdx.x % (unsigned)a.kv_heads), item = (int)(blockIdx.x / (unsigned)a.kv_heads);
    const int run = item % a.runs, row = item / a.runs, tid = threadIdx.x, lane = tid & 63;
    const int s = a.p.shift - 5;
    auto length = [&](int r) { return max(0, min(a.tk[r], a.p.cols << a.p.shift)); };
    const Together t(a, row);
    const int runs = t.runs(a);
    const bool live = t.table >= 0 && t.table < a.p.rows;
    if (a.merge && run == 0 && kh == 0 && tid == 0) *row_note(a, HD, row) = (row - t.r0) | t.rows << 8 | (live ? 0 : 1 << 16);
    if (t.rows > 1) {
        const int sub = (row - t.r0) * a.runs + run;
        if (sub >= runs) return;
        int top = 0;
        for (int i = 0; i < t.rows; ++i) top = max(top, length(t.r0 + i));
        const int live = (top + (1 << a.p.shift) - 1) >> a.p.shift;
        for (int p = tid; p < live; p += PT) mask[p] = 0;
        __syncthreads();
        for (int e = tid; e < t.rows * a.count; e += PT) {
            const int i = e / a.count, r = t.r0 + i;
            const int p = a.chosen[((size_t)r * a.kv_heads + kh) * a.count + e % a.count];
            if (p >= 0 && p < a.p.cols && p << a.p.shift < length(r)) atomicOr(&mask[p], 1u << i);
        }
        __syncthreads();
        int n = 0;
        for (int p0 = 0; p0 < live; p0 += PT) {
            const int p = p0 + tid;
            const bool on = p < live && mask[p] != 0;
            const uint64_t m = __ballot(on);
            if (lane == 0) waves[tid >> 6] = __popcll(m);
            __syncthreads();
            int at = n + __popcll(m & ((1ull << lane) - 1));
            for (int k = 0; k < PW; ++k) {
                if (k < tid >> 6) at += waves[k];
                n += waves[k];
            }
            if (on) list[at] = (uint16_t)p;
            __syncthreads();
        }
        const int blocks = n << s, share = (blocks + runs - 1) / runs, begin = sub * share, end = min(blocks, begin + share);
        const Sink to = runs == 1 ? context(a, HD, t.r0, kh)
                                  : row_of(a, HD, wide_part(a, HD, t.tile * a.tile_runs + sub, kh),
                                           t.r0 - t.tile * PG_TILE_ROWS(a.group));
        auto place = [&](int i, uint32_t& on) {
            const int p = list[i >> s];
            on = mask[p];
            return (p << a.p.shift) + 32 * (i & ((1 << s) - 1));
        };
        auto sees = [&](int i) { return ColumnSees{0, 0, length(t.r0 + i)}; };
        if (t.rows * a.group > 16
                ? tile<HD, MODE, 2, false>(a, w, t.r0, t.rows, t.table, kh, begin, end, to, place, sees)
                : tile<HD, MODE, 1, false>(a, w, t.r0, t.rows, t.table, kh, begin, end, to, place, sees))
            return;
        for (int i = 0; i < t.rows; ++i) {
            auto of_row = [&](int b, uint32_t& on) {
                const int at = place(b, on);
                return (on >> i & 1) && at < length(t.r0 + i) ? at : -1;
            };
            tile<HD, MODE, 1, true>(a, w, t.r0 + i, 1, t.table, kh, begin, end, row_of(a, HD, to, i), of_row,
                                        [&](int) { return sees(i); });
            __syncthreads();  // the join's arrays
        }
        return;
    }
    const int n = a.group * HD, tk = length(row);
    const Sink to = runs == 1 ? context(a, HD, row, kh) : own_part(a, HD, item, kh);
    if (runs == 1 && !live) {
        fill(to.o, n, __builtin_nanf(""));
        return;
    }
    const int blocks = a.count << s, share = (blocks + runs - 1) / runs, begin = run * share;
    const int end = live ? min(blocks, begin + share) : 0;
    const int* chosen = a.chosen + ((size_t)row * a.kv_heads + kh) * a.count;
    auto place = [&](int i, uint32_t&) {
        const int p = chosen[i >> s];
        if (p < 0 || p >= a.p.cols) return -1;
        const int first = (p << a.p.shift) + 32 * (i & ((1 << s) - 1));
        return first < tk ? first : -1;
    };
    if (one_row<HD, MODE, 0>(a, w, row, t.table, kh, begin, end, 0, 0, tk, to, place)) return;
    tile<HD, MODE, 1, true>(a, w, row, 1, t.table, kh, begin, end, to, place, [&](int) { return ColumnSees{0, 0, tk}; });
}

// The parts of a row's columns of kv head kh: `on` of its own, then its group's.
// None (n = 0): its item wrote the context.
template <int HD, bool PLAN>
struct Parts {
    int o0, on, s0 = 0, n, step = 0, col = 0, own_col = -1;  // own_col: its own parts are a tile's
    bool bad = false;  // no such table row
    __device__ __forceinline__ Parts(const PagedArgs& a, int row) {
        if constexpr (PLAN) {
            const int* d = plan_row(a, row);
            o0 = d[0], on = d[1], s0 = d[2], step = d[4], col = d[5], own_col = d[6];
            n = on == 1 && d[3] == 0 ? 0 : on + d[3];
        } else {
            const int note = *row_note(a, HD, row), rows = note >> 8 & 255, per = PG_TILE_ROWS(a.group);
            bad = note >> 16 != 0;
            on = rows == 1 ? a.runs : min(a.tile_runs, rows * a.runs);
            n = on == 1 ? 0 : on;
            o0 = row * a.runs;
            if (rows > 1) o0 = row / per * a.tile_runs, own_col = row % per * a.group;
        }
    }
    // The i-th part's O and (m, l) of query head g.
    __device__ __forceinline__ Sink of(const PagedArgs& a, int i, int kh, int g) const {
        Sink p = i >= on        ? wide_part(a, HD, s0 + (i - on) * step, kh)
                 : own_col >= 0 ? wide_part(a, HD, o0 + i, kh)
                                : own_part(a, HD, o0 + i, kh);
        const int at = g + (i >= on ? col : own_col >= 0 ? own_col : 0);
        p.o += (size_t)at * HD, p.ml += at;
        return p;
    }
};

// The context from its parts, in their order: M = max m, O = sum 2^(m - M) O / sum
// 2^(m - M) l. A part in which a row sees no key has m = RG_NOREF and l = 0.
//
// Many rows, of few parts each: a thread takes four dims of a (row, head) (244
// rows of 20 heads of 64, by a workgroup a (row, head) as below 12.4 us, so 5.2; 127
// of 32 of 128 10.6, so 4.8).
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
// parts, all four heads by one thread a column: 12.4 us, so 4.0).
template <int HD, bool PLAN>
__global__ __launch_bounds__(PT) void paged_merge_kernel(PagedArgs a) {
    constexpr int C = HD / 4, R = PT / C, U = 4;
    __shared__ float wt[PG_PARTS];
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
    const int n = min(p.n, PG_PARTS);  // (all of them: paged_sizes, selected_sizes)
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
#define PM(HD, M)                                                                                       \
    if (!done && hd == HD && mode == M) {                                                               \
        if (!a.plan) hipLaunchKernelGGL((selected_kernel<HD, M>), grid, dim3(PT), 0, st, a);            \
        else if (a.stream) hipLaunchKernelGGL((paged_kernel<HD, M, AUX_STREAM>), grid, dim3(PT), 0, st, a); \
        else hipLaunchKernelGGL((paged_kernel<HD, M, 0>), grid, dim3(PT), 0, st, a);                    \
        done = true;                                                                                    \
    }
    PM(64, 0) PM(64, 1) PM(64, 2) PM(64, 3) PM(128, 0) PM(128, 1) PM(128, 2) PM(128, 3)
#undef PM
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
