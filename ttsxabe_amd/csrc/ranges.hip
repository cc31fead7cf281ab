// Attention in which every query row sees its own keys: the first `first[r]`
// of the cache and those from lo[r] up to hi[r]. Causal and full prompts,
// packed documents, a window behind shared leading positions and a prefix that
// a document's rows all see are such ranges. Scores may be capped by a tanh and
// biased by distance:
//
//   s_j = c tanh(scale q.k_j / c) - slope_h |i - j|,   i = past + r,
//   out = sum_j p_j v_j,  p = softmax of s over the keys the row sees.
//
// A row that sees no key is zeros. Keys a row does not see contribute nothing,
// whatever they hold. The cache is the tiled f16 one (kvlayout.h).
#include <algorithm>
#include <type_traits>

#include "common.h"
#include "decode.h"
#include "kvlayout.h"
#include "ranges.h"
#include "scores.h"

namespace llmtie {

// ---------------------------------------------------------------- row table

constexpr int KR = 256;
constexpr int KR_LDS = 2048;  // starts held in LDS

// One thread a row: its document by bisection of the starts, held in LDS up to
// KR_LDS of them (the search is a chain of loads, 100 clocks each there).
__global__ __launch_bounds__(KR) void key_ranges_kernel(KeyRangeArgs a) {
    __shared__ int held[KR_LDS];
    const bool lds = a.starts && a.docs + 1 <= KR_LDS;
    if (lds) {
        for (int i = threadIdx.x; i <= a.docs; i += KR) held[i] = a.starts[i];
        __syncthreads();
    }
    const int r = (int)blockIdx.x * KR + (int)threadIdx.x;
    if (r >= a.rows) return;
    const long i = (long)a.past + r, n = (long)a.past + a.rows;
    long s = 0, e = n;
    int d = 0;
    bool inside = true;
    if (a.starts) {
        // The last start at or before r; -1 or docs: in no document.
        int lo = -1, hi = a.docs + 1;
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if ((lds ? held[mid] : a.starts[mid]) <= r) lo = mid;
            else hi = mid;
        }
        d = lo;
        inside = d >= 0 && d < a.docs;
        if (inside) {
            s = (long)a.past + (lds ? held[d] : a.starts[d]);
            e = min(n, (long)a.past + (lds ? held[d + 1] : a.starts[d + 1]));
        }
    }
    long lo = 0, hi = 0, first = 0, pos = 0;
    if (inside) {
        lo = s;
        hi = a.causal ? i + 1 : e;
        if (a.window) {
            lo = max(lo, i - a.window + 1);
            if (!a.causal) hi = min(hi, i + a.window);
        }
        if (a.prefix) hi = max(hi, min(s + a.prefix[d], e));
        first = min((long)a.shared, a.causal ? i + 1 : n);
        pos = i - s;
    }
    a.table[r] = (int)first;
    a.table[(size_t)a.rows + r] = (int)lo;
    a.table[2 * (size_t)a.rows + r] = (int)hi;
    if (a.pos) a.pos[r] = (int)pos;
}

hipError_t launch_key_ranges(const KeyRangeArgs& a, hipStream_t st) {
    if (a.rows == 0) return hipSuccess;
    hipLaunchKernelGGL(key_ranges_kernel, dim3((unsigned)((a.rows + (long)KR - 1) / KR)), dim3(KR), 0, st, a);
    return hipGetLastError();
}

// ------------------------------------------------------------------- scores

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));

// ------------------------------------------------------------------ prompts

constexpr int RW = 4, RT = RW * LLMTIE_WAVE;
constexpr int KT = 64;  // keys of a tile

// Minimum over the 16 lanes of a row of lanes (every lane gets it).
__device__ __forceinline__ int row_min(int v) {
    v = min(v, __builtin_amdgcn_update_dpp(0, v, 0xb1, 0xf, 0xf, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x4e, 0xf, 0xf, false));
    v = min(v, __builtin_amdgcn_update_dpp(0, v, 0x141, 0xf, 0xf, false));
    return min(v, __builtin_amdgcn_update_dpp(0, v, 0x140, 0xf, 0xf, false));
}
__device__ __forceinline__ int row_max(int v) { return -row_min(-v); }

// What a set of rows sees, as bounds: [0, f1) and [l0, h1) hold every key some
// row sees; every row sees those below f0 and those in [l1, h0).
struct Bounds {
    int f0, f1, l0, l1, h0, h1;
    __device__ __forceinline__ bool touches(int kv0) const { return kv0 < f1 || (kv0 + KT > l0 && kv0 < h1); }
    __device__ __forceinline__ bool whole(int kv0) const {
        return kv0 + KT <= f0 || (kv0 >= l1 && kv0 + KT <= h0);
    }
};

// Two halves a word: bit 15 of each set where the half is not finite.
__device__ __forceinline__ uint32_t not_finite(uint32_t w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; }

// One 64-key tile's products for the NQT * 16 rows of a wave. LDS tile: the
// keys' K fragments then V fragments, each 64 lanes x 16 bytes in the order of
// the MFMA A operands (two blocks of the tiled cache, copied verbatim): K
// fragment (half, T, s) holds in lane (col, grp) key 32 half + 8 (col / 4) + 4 T
// + col % 4, dims 32 s + 8 grp ..; V fragment (half, t) dim 16 t + col, keys 32
// half + 8 grp ... S^T = K Q^T then leaves lane (col, grp) the scores of row
// col's keys 32 half + 8 grp + 4 T + r: the B operand of O^T = V^T P^T, so P
// never leaves registers.
template <int HD, int MODE, int NQT>
struct RangeTile {
    static constexpr int NS = HD / 32, NT = HD / 16, KF = 4 * NS, VF = 2 * NT, FH = 64 * 8, QPW = 16 * NQT;
    half8 qb[NQT][NS];
    floatx4 o[NT][NQT];
    floatx4 l[NQT];  // the sum of the weights, in each element
    float m[NQT];
    const int* rg;   // the wave's rows' ranges in LDS: first, lo, hi, QPW each
    int pos0, last;  // SM_BIAS: the wave's first row's position, and the prompt's last
    floatx4 sc[2][2][NQT];
    half8 pb[2][NQT];
    float mul, add;  // a logit (log2 units) is mul * (what logits() leaves) + add + the bias
    float kc;        // SM_CAP: 2 log2(e) scale / c
    float lift;      // a row's reference is set so far below its largest score
    float slope2;    // SM_BIAS: slope * log2(e)
    int grp, lane;

    uint32_t up[NQT], dn[NQT];  // values that are not finite (specials)
    uint32_t seen[NQT];  // the masked tile's keys that row col sees, of this lane's: bit 8 half + e

    // Bits 0 .. n - 1 of 64.
    __device__ __forceinline__ static uint64_t below(int n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
    // Which of the tile's keys the rows see, one bit a key (a compare a score
    // kept 175 scalar registers of masks, and spilled).
    __device__ __forceinline__ uint64_t tile_of(int u, int kv0) const {
        const int* p = rg + 16 * u + (lane & 15);
        return below(p[0] - kv0) | (below(p[2 * QPW] - kv0) & ~below(p[QPW] - kv0));
    }
    __device__ __forceinline__ void look(int kv0) {
#pragma unroll
        for (int u = 0; u < NQT; ++u) {
            const uint64_t b = tile_of(u, kv0);
            seen[u] = (uint32_t)(b >> (8 * grp)) & 0xffu;
            seen[u] |= ((uint32_t)(b >> 32 >> (8 * grp)) & 0xffu) << 8;
        }
    }
    // All ones where this lane's key 32 half + 8 grp + e of the tile is seen.
    __device__ __forceinline__ uint32_t sees(int u, int hf, int e) const {
        return (uint32_t)__builtin_amdgcn_sbfe((int)seen[u], 8 * hf + e, 1);
    }

    // The queries and ranges of the wave's rows from p0 on; the bounds of what
    // they see. `mem`: 3 * QPW ints of LDS.
    __device__ __forceinline__ Bounds start(const RangesArgs& a, int p0, int h, int lane_, int* mem) {
        lane = lane_;
        grp = lane >> 4;
        rg = mem;
        const int col = lane & 15, ktot = a.past + a.tq;
        pos0 = a.past + p0;
        last = ktot - 1;
        mul = a.scale * LLMTIE_LOG2E;
        add = 0.0f;
        lift = a.lift;
        if constexpr ((MODE & SM_CAP) != 0) {
            kc = 2.0f * LLMTIE_LOG2E * (a.scale / a.softcap);
            add = a.softcap * LLMTIE_LOG2E;
            mul = -2.0f * add;
        }
        if constexpr ((MODE & SM_BIAS) != 0) slope2 = a.slopes[h] * LLMTIE_LOG2E;
        Bounds b{0x7fffffff, 0, 0x7fffffff, 0, 0x7fffffff, 0};
#pragma unroll
        for (int u = 0; u < NQT; ++u) {
            const int r = min(p0 + 16 * u + col, a.tq - 1);
            // Clamped to the keys the cache holds; a range that holds none is
            // moved past every key, so that bounds over rows pass it by.
            const int f = max(0, min(a.first[r], ktot));
            int lo = max(0, a.lo[r]), hi = min(a.hi[r], ktot);
            if (lo >= hi) lo = 0x7fffffff, hi = 0;
            if (grp == 0) {
                int* p = mem + 16 * u + col;
                p[0] = f, p[QPW] = lo, p[2 * QPW] = hi;
            }
            b.f0 = min(b.f0, f), b.f1 = max(b.f1, f);
            b.l0 = min(b.l0, lo), b.l1 = max(b.l1, lo);
            b.h0 = min(b.h0, hi), b.h1 = max(b.h1, hi);
            m[u] = RG_NOREF;
            l[u] = zero_f4();
            up[u] = dn[u] = 0;
            const uint16_t* q = a.q + (size_t)r * a.q_stride + (size_t)h * HD + 8 * grp;
            if (a.qal) {
#pragma unroll
                for (int s = 0; s < NS; ++s) qb[u][s] = ld_h8(q + 32 * s);
            } else {
#pragma unroll
                for (int s = 0; s < NS; ++s)
#pragma unroll
                    for (int j = 0; j < 8; ++j) qb[u][s][j] = __builtin_bit_cast(half_t, q[32 * s + j]);
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int u = 0; u < NQT; ++u) o[t][u] = zero_f4();
        b.f0 = __builtin_amdgcn_readfirstlane(row_min(b.f0));
        b.f1 = __builtin_amdgcn_readfirstlane(row_max(b.f1));
        b.l0 = __builtin_amdgcn_readfirstlane(row_min(b.l0));
        b.l1 = __builtin_amdgcn_readfirstlane(row_max(b.l1));
        b.h0 = __builtin_amdgcn_readfirstlane(row_min(b.h0));
        b.h1 = __builtin_amdgcn_readfirstlane(row_max(b.h1));
        return b;
    }

    // Fragment reads kept in flight ahead of the MFMAs that use them.
    template <int NR>
    __device__ __forceinline__ static void pipeline() {
        constexpr int PD = NR < 10 ? NR : 10;
        __builtin_amdgcn_sched_group_barrier(0x100, PD, 0);
#pragma unroll
        for (int i = 0; i < NR - PD; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, NQT, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, NQT * PD, 0);
        __builtin_amdgcn_sched_barrier(0);
    }

    __device__ __forceinline__ void scores(const half_t* tb) {
        const half8* kf = reinterpret_cast<const half8*>(tb);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int T = 0; T < 2; ++T)
#pragma unroll
                for (int u = 0; u < NQT; ++u) sc[hf][T][u] = zero_f4();
        // Dims outermost: independent accumulators between two products into one.
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                for (int T = 0; T < 2; ++T) {
                    const half8 af = kf[((hf * 2 + T) * NS + s) * 64 + lane];
#pragma unroll
                    for (int u = 0; u < NQT; ++u) sc[hf][T][u] = mfma16(af, qb[u][s], sc[hf][T][u]);
                }
        pipeline<4 * NS>();
    }

    // The scores in place as what a multiply-add makes a logit of: as they are,
    // or with a cap 1 / (1 + 2^(kc s)), of which the tanh is 1 less twice:
    //   c tanh(x) = c - 2 c / (1 + e^2x),   x = scale s / c;
    // and an infinity for a key not seen. A wave issues an instruction in 4 to 7
    // clocks, whatever it is: four a score here and three in softmax(), which
    // the cap needs instead of three, set the time of a capped prompt. (A
    // cubic in x^2 for scores under half the cap, no transcendentals but 9.5
    // instructions, was no faster.)
    __device__ __forceinline__ void logits(int kv0, bool whole) {
        if constexpr ((MODE & SM_CAP) != 0) {
#pragma unroll
            for (int u = 0; u < NQT; ++u)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int T = 0; T < 2; ++T)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            sc[hf][T][u][r] = __builtin_amdgcn_rcpf(ex2(kc * sc[hf][T][u][r]) + 1.0f);
        }
        if constexpr ((MODE & SM_BIAS) != 0) {
            if (mixed(kv0)) {
                // softmax() takes the keys as behind their rows: for those
                // ahead of them, twice their distance.
                const float k2 = 2.0f * slope2 / mul;
#pragma unroll
                for (int u = 0; u < NQT; ++u) {
                    const float d0 = (float)(min(pos0 + 16 * u + (lane & 15), last) - kv0 - 8 * grp);
#pragma unroll
                    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                        for (int T = 0; T < 2; ++T)
#pragma unroll
                            for (int r = 0; r < 4; ++r)
                                sc[hf][T][u][r] = __builtin_fmaf(k2, fminf(d0 - (float)(32 * hf + 4 * T + r), 0.0f),
                                                                 sc[hf][T][u][r]);
                }
            }
        }
        if (!whole) {
            constexpr uint32_t OUT = (MODE & SM_CAP) != 0 ? 0x7f800000u : 0xff800000u;  // mul times it: -inf
            look(kv0);
#pragma unroll
            for (int u = 0; u < NQT; ++u)
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int T = 0; T < 2; ++T)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const uint32_t on = sees(u, hf, 4 * T + r);
                            sc[hf][T][u][r] = __uint_as_float((__float_as_uint(sc[hf][T][u][r]) & on) | (OUT & ~on));
                        }
        }
    }
    // SM_BIAS: whether the tile has keys behind some rows and ahead of others,
    // and on which side of the rows its keys lie if not (those of a mixed tile: behind).
    __device__ __forceinline__ bool mixed(int kv0) const { return kv0 + KT - 1 > pos0 && kv0 < pos0 + QPW - 1; }
    __device__ __forceinline__ float side(int kv0) const { return kv0 >= pos0 + QPW - 1 ? -slope2 : slope2; }

    // The online softmax of the tile in log2 units. P = 2^(s - m) is formed
    // against the row's reference m, which moves only when a weight passes 2^15
    // (a key 15 above m, or the first one seen), to `lift` below the row's
    // largest score: O and l carry the same factor, so O / l does not depend on
    // where m sits, P stays inside f16, and the tile's max is taken on the rare
    // tiles that move m. P is rounded to f16 for the product (2^-11 of each
    // weight, as the f16 context's own rounding, and at most 2^-25 where it is
    // small: 2^(-25 - lift) of the largest, which over all keys is 2^-12 of it);
    // l is the sum of the rounded weights at f32, by the matrix unit (a product
    // with ones in values()): 16 additions a row and lane less, beside a
    // packed maximum that watches for 2^15.
    // (One copy of it: a masked and an unmasked one spilled 320 registers.)
    __device__ __forceinline__ void softmax(int kv0, bool whole) {
        logits(kv0, whole);
#pragma unroll
        for (int u = 0; u < NQT; ++u) {
            float sl = 0.0f, at = add;
            if constexpr ((MODE & SM_BIAS) != 0) {
                sl = side(kv0);
                at += sl * (float)(kv0 + 8 * grp - min(pos0 + 16 * u + (lane & 15), last));
            }
            // The logit of the lane's key c of the tile, with `off` for what the keys share.
            auto logit = [&](float s, int c, float off) __attribute__((always_inline)) {
                if constexpr ((MODE & SM_BIAS) != 0) off = __builtin_fmaf(sl, (float)c, off);
                return __builtin_fmaf(s, mul, off);
            };
            auto form = [&](auto moved) __attribute__((always_inline)) {
                // Less m in the offset; behind a move in a step of its own, so
                // that the key m was taken from has a weight of exactly 1 (of
                // logits past 2^24 the offset's rounding is more than a weight).
                constexpr bool M = decltype(moved)::value;
                const float off = M ? at : at - m[u], ref = M ? m[u] : 0.0f;
                auto weight = [&](float s, int c) __attribute__((always_inline)) {
                    const float x = logit(s, c, off);
                    return to_h(ex2(M ? x - ref : x));
                };
                half2_t top;
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int T = 0; T < 2; ++T)
#pragma unroll
                        for (int r = 0; r < 4; r += 2) {
                            half2_t p;
                            p[0] = weight(sc[hf][T][u][r], 32 * hf + 4 * T + r);
                            p[1] = weight(sc[hf][T][u][r + 1], 32 * hf + 4 * T + r + 1);
                            pb[hf][u][4 * T + r] = p[0];
                            pb[hf][u][4 * T + r + 1] = p[1];
                            top = hf | T | r ? __builtin_elementwise_max(top, p) : p;
                        }
                return fmaxf((float)top[0], (float)top[1]);
            };
            if (__any(!(form(std::false_type{}) <= 32768.0f))) {
                float mx = ninf();
#pragma unroll
                for (int hf = 0; hf < 2; ++hf)
#pragma unroll
                    for (int T = 0; T < 2; ++T)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            mx = fmaxf(mx, logit(sc[hf][T][u][r], 32 * hf + 4 * T + r, at));
                mx = max4grp(mx);
                const float mn = fmaxf(m[u], fabsf(mx) < 0x1p23f ? mx - lift : mx);
                const float fac = ex2(m[u] - mn);
                m[u] = mn;
                l[u] *= fac;
#pragma unroll
                for (int t = 0; t < NT; ++t) o[t][u] *= fac;
                form(std::true_type{});
            }
        }
    }

    __device__ __forceinline__ void values(const half_t* tb) {
        const half8* vf = reinterpret_cast<const half8*>(tb + KF * FH);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                const half8 af = vf[(hf * NT + t) * 64 + lane];
#pragma unroll
                for (int u = 0; u < NQT; ++u) o[t][u] = mfma16(af, pb[hf][u], o[t][u]);
            }
        half8 ones;
#pragma unroll
        for (int j = 0; j < 8; ++j) ones[j] = (half_t)1.0f;
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
            for (int u = 0; u < NQT; ++u) l[u] = mfma16(ones, pb[hf][u], l[u]);
        pipeline<2 * NT>();
    }

    // The values that screen() took out of the tile: whether a key that a row
    // sees held one, a bit a dim of this lane's (4 t + i), for +inf or NaN and
    // for -inf or NaN. (Adding them to O here had the loop keep it in two places.)
    __device__ __forceinline__ void specials(const uint4* sp, int kv0) {
        uint64_t b[NQT];
#pragma unroll
        for (int u = 0; u < NQT; ++u) b[u] = tile_of(u, kv0);
#pragma nounroll
        for (int d = 0; d < 4 * NT; ++d) {
            const uint4 w = sp[16 * (d >> 2) + 4 * grp + (d & 3)];
#pragma unroll
            for (int u = 0; u < NQT; ++u) {
                const uint32_t b0 = (uint32_t)b[u], b1 = (uint32_t)(b[u] >> 32);
                up[u] |= min((w.x & b0) | (w.y & b1), 1u) << d;
                dn[u] |= min((w.z & b0) | (w.w & b1), 1u) << d;
            }
        }
    }
    // What a sum with them is: +inf, -inf, or NaN with both.
    __device__ __forceinline__ void close() {
        uint32_t any = 0;
#pragma unroll
        for (int u = 0; u < NQT; ++u) any |= up[u] | dn[u];
        if (!__any(any != 0)) return;
#pragma unroll
        for (int u = 0; u < NQT; ++u)
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    o[t][u][i] += __uint_as_float((up[u] >> (4 * t + i) & 1u) * 0x7f800000u);
                    o[t][u][i] -= __uint_as_float((dn[u] >> (4 * t + i) & 1u) * 0x7f800000u);
                }
    }
};

// Whether some value of a tile is not finite, as this wave's share of a look by
// all waves of the workgroup shows.
template <int HD>
__device__ __forceinline__ bool odd_values(const half_t* vt, int tid) {
    const uint4* v = reinterpret_cast<const uint4*>(vt);
    uint32_t x = 0;
#pragma unroll
    for (int k = 0; k < 2 * (HD / 16) / RW; ++k) {
        const uint4 y = v[tid + RT * k];
        x |= not_finite(y.x) | not_finite(y.y) | not_finite(y.z) | not_finite(y.w);
    }
    return __any(x != 0);
}

// The bounds of all waves' rows (a barrier).
__device__ __forceinline__ Bounds together(const Bounds& mine, int (*wb)[6], int wave, int lane) {
    if (lane == 0) {
        wb[wave][0] = mine.f0, wb[wave][1] = mine.f1, wb[wave][2] = mine.l0;
        wb[wave][3] = mine.l1, wb[wave][4] = mine.h0, wb[wave][5] = mine.h1;
    }
    __syncthreads();
    Bounds b = mine;
#pragma unroll
    for (int w = 0; w < RW; ++w) {
        b.f0 = min(b.f0, wb[w][0]), b.f1 = max(b.f1, wb[w][1]), b.l0 = min(b.l0, wb[w][2]);
        b.l1 = max(b.l1, wb[w][3]), b.h0 = min(b.h0, wb[w][4]), b.h1 = max(b.h1, wb[w][5]);
    }
    b.f0 = __builtin_amdgcn_readfirstlane(b.f0), b.f1 = __builtin_amdgcn_readfirstlane(b.f1);
    b.l0 = __builtin_amdgcn_readfirstlane(b.l0), b.l1 = __builtin_amdgcn_readfirstlane(b.l1);
    b.h0 = __builtin_amdgcn_readfirstlane(b.h0), b.h1 = __builtin_amdgcn_readfirstlane(b.h1);
    return b;
}

// The 64-key tiles that hold a key some row sees: na of the leading keys, then
// those from tb on; walked from the last to the first. (With a bias by distance
// the near keys weigh most: from the first to the last, nearly every tile of a
// steep head raised the row's max and was formed twice.)
struct Tiles {
    int na, tb, n;
    __device__ __forceinline__ explicit Tiles(const Bounds& b) {
        na = (b.f1 + KT - 1) / KT;
        tb = max(na, b.l0 / KT);
        n = na + max(0, (b.h1 + KT - 1) / KT - tb);
    }
    __device__ __forceinline__ int key0(int i) const {
        const int j = n - 1 - i;
        return __builtin_amdgcn_readfirstlane(KT * (j < na ? j : tb + j - na));
    }
};

// Takes the values that are not finite out of a tile in LDS (a weight of 0 must
// not meet them: a row may not see their keys), by all threads of a
// workgroup: they become 0, and sp[dim] holds which of the 64 keys had +inf or
// NaN there (x, y) and -inf or NaN (z, w). Barriers before and after are the
// caller's.
template <int HD>
__device__ __forceinline__ void screen_clear(uint4* sp, int tid) {
    if (tid < HD) sp[tid] = make_uint4(0, 0, 0, 0);
}
template <int HD>
__device__ __forceinline__ void screen(half_t* vt, uint4* sp, int tid) {
    constexpr int NT = HD / 16;
    uint4* v = reinterpret_cast<uint4*>(vt);
    for (int c = tid; c < 2 * NT * 64; c += RT) {
        const int hf = c / (NT * 64), dim = 16 * (c / 64 % NT) + (c & 15), key = 8 * (c >> 4 & 3);
        uint4 y = v[c];
        uint32_t* w = &y.x;
        uint32_t* at = reinterpret_cast<uint32_t*>(sp + dim) + hf;
        bool any = false;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t nf = not_finite(w[e]);
            if (!nf) continue;
            any = true;
            const uint32_t nan = nf & ((w[e] & 0x03ff03ffu) + 0x7fff7fffu);
            const uint32_t up = nan | (nf & ~w[e]), dn = nan | (nf & w[e]);
            const int k = key + 2 * e;
            atomicOr(at, ((up >> 15 & 1u) | (up >> 30 & 2u)) << k);
            atomicOr(at + 2, ((dn >> 15 & 1u) | (dn >> 30 & 2u)) << k);
            w[e] &= ~((nf >> 15) * 0xffffu);
        }
        if (any) v[c] = y;
    }
}

// Fragments of one tile into LDS by direct loads, its waves taking every fourth:
// per-lane offsets fixed for the launch, a scalar one a load. Where the tile's
// second block lies past the last one that holds keys, both halves come from
// the first, so every address lies in a live block.
template <int HD>
struct RangeLoad {
    static constexpr int NS = HD / 32, NT = HD / 16, KF = 4 * NS, VF = 2 * NT, FH = 64 * 8;
    static constexpr int KI = KF / RW, VI = VF / RW, KFB = KF / 2;
    static constexpr uint32_t BLK = 128 * HD;  // bytes of a block
    static_assert(KFB % RW == 0, "a load takes the same block for every wave");
    const uint16_t* head;
    int w0, lastb;
    uint32_t off;
    __device__ __forceinline__ RangeLoad(const RangesArgs& a, int kh, int lane, int wave)
        : head(a.cache + (size_t)kh * tiled_nblk(a.cap) * (BLK / 2)),
          w0(__builtin_amdgcn_readfirstlane(wave)),
          lastb((a.past + a.tq - 1) >> 5),
          off(16u * lane + 1024u * wave) {}
    __device__ __forceinline__ void operator()(int kv0, half_t* dst) const {
        half_t* l = dst + w0 * FH;
        const int b = kv0 >> 5;
        const uint32_t second = b + 1 <= lastb ? BLK : 0;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint16_t*>(head) + (size_t)b * (BLK / 2), 0, 2 * (int)BLK, 0x00020000);
#pragma unroll
        for (int i = 0; i < KI + VI; ++i) {
            const int f = RW * (i < KI ? i : i - KI);  // of its area, for wave 0
            const uint32_t in = (i < KI ? 0u : 64u * HD) + 1024u * (f % KFB);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, l + RW * i * FH, 16, (int)off, f / KFB * second + in, 0, 0);
        }
    }
};

// Sixteen context rows of a wave as f16 in line order through its own LDS
// region R (16 x HD halves): a row's 16-byte chunk c at c ^ (row % chunks).
template <int HD, int NQT>
__device__ __forceinline__ void store_rows(half_t* R, const floatx4 (&o)[HD / 16][NQT], int u, float inv, int lane,
                                           const RangesArgs& a, int row0, int h) {
    constexpr int NT = HD / 16, LPR = HD / 8, RPI = 64 / LPR;
    const int col = lane & 15, grp = lane >> 4;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        half4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = to_h(o[t][u][i] * inv);
        *reinterpret_cast<half4*>(R + col * HD + 8 * ((2 * t + (grp >> 1)) ^ (col % LPR)) + 4 * (grp & 1)) = y;
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
        const int row = i * RPI + lane / LPR, c = lane % LPR;
        const half8 x = *reinterpret_cast<const half8*>(R + row * HD + 8 * (c ^ (row % LPR)));
        if (row0 + row < a.tq)
            *reinterpret_cast<half8*>(a.out + ((size_t)(row0 + row) * a.heads + h) * HD + 8 * c) = x;
    }
    __builtin_amdgcn_wave_barrier();
}

// The rows of sixteen queries' run as f32 partials and their (m, l).
template <int HD, int NQT>
__device__ __forceinline__ void store_part(const floatx4 (&o)[HD / 16][NQT], int u, float m, float l, int lane,
                                           const RangesArgs& a, int sp, int row0, int h) {
    const int col = lane & 15, grp = lane >> 4, r = row0 + col;
    if (r >= a.tq) return;
    const size_t rows = (size_t)a.tq * a.heads, at = ((size_t)sp * a.tq + r) * a.heads + h;
#pragma unroll
    for (int t = 0; t < HD / 16; ++t) *reinterpret_cast<floatx4*>(a.ws + at * HD + 16 * t + 4 * grp) = o[t][u];
    if (grp == 0) reinterpret_cast<float2*>(a.ws + (size_t)a.splits * rows * HD)[at] = make_float2(m, l);
}

// A workgroup is four waves: `gb` heads of one GQA group (one K/V tile in LDS
// serves them) times 4 / gb blocks of 16 * NQT rows. It walks the 64-key tiles
// that hold a key some of its rows sees, double-buffered, one barrier a tile.
template <int HD, int MODE, int NQT, bool SPLIT>
__global__ __launch_bounds__(RT, 2) void ranges_kernel(RangesArgs a) {
    using Tile = RangeTile<HD, MODE, NQT>;
    constexpr int FH = Tile::FH, KF = Tile::KF, VF = Tile::VF, QPW = 16 * NQT;
    // Two arrays, each step's its own: reads of one array's halves are taken for
    // reads of the loads in flight into the other and wait for them, each tile
    // (8192 rows of 32/8/128, capped, 664 -> 606 us, as 1500 of 20/20/64 25.8 -> 22.5;
    // with lds_barrier() 588 and 21.5).
    __shared__ __attribute__((aligned(16))) half_t even[(KF + VF) * FH], odd[(KF + VF) * FH];
    __shared__ int wrg[RW][3 * QPW];
    __shared__ int wb[RW][6];
    __shared__ int wbad[RW];
    __shared__ uint4 sp_[HD];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int gb = a.gb, pb = QPW * (RW / gb), group = a.heads / a.kv_heads;
    const int item = a.xcd ? (int)(blockIdx.x % 8) * a.grid8 + (int)(blockIdx.x / 8) : (int)blockIdx.x;
    int gy = item / a.nrb, sp = 0;
    const int bx = a.nrb - 1 - item % a.nrb;  // causal rows see most keys last: heaviest first
    if constexpr (SPLIT) {
        sp = gy % a.splits;
        gy /= a.splits;
    }
    const int h = gy * gb + wave % gb, kh = gy * gb / group;
    const int p0 = bx * pb + (wave / gb) * QPW;
    const RangeLoad<HD> issue(a, kh, lane, wave);

    Tile t;
    const Bounds mine = t.start(a, p0, h, lane, wrg[wave]);
    const Bounds all = together(mine, wb, wave, lane);
    const Tiles tiles(all);
    int i0 = 0, i1 = tiles.n;
    if constexpr (SPLIT) {
        i0 = __builtin_amdgcn_readfirstlane((int)((long)tiles.n * sp / a.splits));
        i1 = __builtin_amdgcn_readfirstlane((int)((long)tiles.n * (sp + 1) / a.splits));
    }
    auto key0 = [&](int i) { return tiles.key0(i); };

    if (i0 < i1) issue(key0(i0), even);
    int i = i0;
    auto step = [&](half_t* cur, half_t* next) __attribute__((always_inline)) {
        const int kv0 = key0(i);
        __builtin_amdgcn_s_waitcnt(0);  // this wave's loads of `cur` have landed
        __syncthreads();                 // every wave's; the other buffer is free
        if (i + 1 < i1) issue(key0(i + 1), next);
        ++i;
        bool bad = false;
        if (!all.whole(kv0)) {
            // Some row does not see some key: are all its values finite?
            const bool any = odd_values<HD>(cur + KF * FH, tid);
            if (lane == 0) wbad[wave] = any;
            lds_barrier();
            bad = (wbad[0] | wbad[1] | wbad[2] | wbad[3]) != 0;
            if (bad) {
                screen_clear<HD>(sp_, tid);
                lds_barrier();
                screen<HD>(cur + KF * FH, sp_, tid);
                lds_barrier();
            }
        }
        if (!mine.touches(kv0)) return;
        t.scores(cur);
        t.softmax(kv0, mine.whole(kv0));
        t.values(cur);
        if (bad) t.specials(sp_, kv0);
    };
    while (i < i1) {
        step(even, odd);
        if (i < i1) step(odd, even);
    }
    // The context through the buffer that does not hold the last tile: every
    // wave left it before the last tile's barrier.
    half_t* R = ((i1 - i0) & 1 ? odd : even) + wave * 16 * HD;
    t.close();
#pragma unroll
    for (int u = 0; u < NQT; ++u) {
        const float lt = t.l[u][0];
        if constexpr (SPLIT) store_part<HD, NQT>(t.o, u, t.m[u], lt, lane, a, sp, p0 + 16 * u, h);
        else store_rows<HD, NQT>(R, t.o, u, lt > 0.0f || lt != lt ? 1.0f / lt : 0.0f, lane, a, p0 + 16 * u, h);
    }
}

// The context of a split prompt from its runs' (m, l, O), in run order: M = max
// m, O = sum 2^(m - M) O / sum 2^(m - M) l. A run in which a row sees no key
// has m = RG_NOREF and l = 0. One thread takes eight dims of one (row, head).
template <int HD>
__global__ __launch_bounds__(RT) void ranges_merge_kernel(const float* ws, uint16_t* out, long rows, int splits) {
    constexpr int LPR = HD / 8;
    const long i = (long)blockIdx.x * RT + threadIdx.x;
    const long row = i / LPR;
    if (row >= rows) return;
    const float4* o = reinterpret_cast<const float4*>(ws) + 2 * i;
    const float2* ml = reinterpret_cast<const float2*>(ws + (size_t)splits * rows * HD) + row;
    constexpr int U = 8;  // runs in flight together (four: a turn of 173 rows 26.5 -> 25.5 us)
    float M = RG_NOREF, l = 0.0f;
    float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += U) {
        float2 c[U];
        float4 x[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = min(s0 + u, splits - 1);
            c[u] = ml[(size_t)s * rows];
            x[u][0] = o[(size_t)s * rows * (2 * LPR)];
            x[u][1] = o[(size_t)s * rows * (2 * LPR) + 1];
        }
        float mn = M;
#pragma unroll
        for (int u = 0; u < U; ++u) mn = fmaxf(mn, c[u].x);
        const float f = ex2(M - mn);
        M = mn;
        l *= f;
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[k] *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (s0 + u >= splits) break;
            const float w = ex2(c[u].x - M);
            l += w * c[u].y;
            acc[0] += w * x[u][0].x, acc[1] += w * x[u][0].y, acc[2] += w * x[u][0].z, acc[3] += w * x[u][0].w;
            acc[4] += w * x[u][1].x, acc[5] += w * x[u][1].y, acc[6] += w * x[u][1].z, acc[7] += w * x[u][1].w;
        }
    }
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    half8 y;
#pragma unroll
    for (int k = 0; k < 8; ++k) y[k] = to_h(acc[k] * inv);
    *reinterpret_cast<half8*>(out + 8 * i) = y;
}

hipError_t launch_ranges(int hd, int nqt, const RangesArgs& a, hipStream_t st) {
    RangesArgs b = a;
    const int pb = 16 * nqt * (RW / a.gb);
    b.nrb = (a.tq + pb - 1) / pb;
    const unsigned items = (unsigned)b.nrb * (unsigned)(a.heads / a.gb) * (unsigned)a.splits;
    b.xcd = items % 8 == 0;
    b.grid8 = (int)(items / 8);
    const int mode = (a.softcap > 0.0f ? SM_CAP : 0) | (a.slopes ? SM_BIAS : 0);
    const long rows = (long)a.tq * a.heads;
#define RL(HD, M, N)                                                                                             \
    if (hd == HD && mode == M && nqt == N && a.splits == 1) {                                                    \
        hipLaunchKernelGGL((ranges_kernel<HD, M, N, false>), dim3(items), dim3(RT), 0, st, b);                   \
        return hipGetLastError();                                                                                \
    }
#define RS(HD, M)                                                                                                \
    if (hd == HD && mode == M && nqt == 1 && a.splits > 1) {                                                     \
        hipLaunchKernelGGL((ranges_kernel<HD, M, 1, true>), dim3(items), dim3(RT), 0, st, b);                    \
        hipLaunchKernelGGL((ranges_merge_kernel<HD>), dim3((unsigned)((rows * (HD / 8) + RT - 1) / RT)),         \
                           dim3(RT), 0, st, a.ws, a.out, rows, a.splits);                                        \
        return hipGetLastError();                                                                                \
    }
#define RM(HD, M) RL(HD, M, 1) RL(HD, M, 2) RS(HD, M)
    RM(64, 0) RM(64, 1) RM(64, 2) RM(64, 3) RM(128, 0) RM(128, 1) RM(128, 2) RM(128, 3)
#undef RM
#undef RS
#undef RL
    return hipErrorInvalidValue;
}

// ------------------------------------------------------------ single tokens

// One query row of each of nseq sequences over its slot of the cache. A
// workgroup is four waves on one (sequence, kv head, run of 32-key blocks), the
// waves taking every fourth block; the <= 16 query heads of the group are the
// 16 columns of the MFMA tile, so a key and value is read once for all of them.
// The products are S^T = K Q^T and O^T = V^T P^T as in the prompts' kernel, with
// q and P as the sums of two f16 (22 bits of each, P's down to 2^-17 of the
// largest and 2^-40 of it below that), so the context carries f32's precision
// off the f16 cache. What bounds it is reading K and V: the next
// block's 16 loads a lane are in flight while one is computed.
//
// The lengths are on the device, so the launch has `splits` runs a head for any
// of them; a head is cut into even ones, of `span` blocks or more, and those
// past them end at once. A head of several runs leaves (m, l, O) of each with
// coherent stores, counts its arrivals, and the last one merges them in order
// (the results do not depend on which that is).
constexpr int RD_MAX_ROWS = 1024;  // splits * group at most

template <int HD, int MODE, int AUX>
__global__ __launch_bounds__(RT, 2) void ranges_decode_kernel(RangesDecodeArgs a) {
    constexpr int NS = HD / 32, NT = HD / 16, OP = HD + 4;  // a wave's O rows in LDS, padded
    struct Block {
        half8 k[2 * NS], v[NT];
    };
    __shared__ __attribute__((aligned(16))) float lds[RW * 16 * OP];
    __shared__ float wm[RW][16], wl[RW][16];
    __shared__ int last;
    static_assert(RW * 16 * OP >= 2 * RD_MAX_ROWS + 16 + RT * 4, "the merge's arrays fit");
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int group = a.group, n = group * HD;
    const int sp = (int)(blockIdx.x % (unsigned)a.splits);
    const unsigned head = blockIdx.x / (unsigned)a.splits;  // sequence * kv_heads + kv head
    const int kh = (int)(head % (unsigned)a.kv_heads), seq = (int)(head / (unsigned)a.kv_heads);
    const int slot = a.slot ? a.slot[seq] : seq;
    const int tk = max(0, min(a.tk[seq], a.cap));
    int lo = a.lo ? a.lo[seq] : 0;
    if (a.window) lo = max(lo, tk - a.window);
    lo = max(0, min(lo, tk));
    int f = min(a.shared, tk);
    if (f >= lo) f = lo = 0;  // no key left out
    float* out = a.out + (size_t)head * n;
    // Blocks: na of the shared keys, then those from b0 on.
    const int na = (f + 31) >> 5, b0 = max(na, lo >> 5);
    const int nb = na + (lo < tk ? max(0, ((tk + 31) >> 5) - b0) : 0);
    const bool live = slot >= 0 && slot < a.slots;
    if (!live || nb == 0) {
        // No such slot: NaN. No key: zeros.
        if (sp == 0)
            for (int e = tid; e < n; e += RT) out[e] = live ? 0.0f : __builtin_nanf("");
        return;
    }
    // Its head in even runs.
    const int runs = nb <= a.whole ? 1 : min(a.splits, (nb + a.span - 1) / a.span);
    if (sp >= runs) return;
    const int share = (nb + runs - 1) / runs, begin = sp * share, end = min(nb, begin + share);

    const char* base = reinterpret_cast<const char*>(a.cache) +
                       ((size_t)slot * a.kv_heads + kh) * tiled_nblk(a.cap) * (128 * HD);
    auto block = [&](int i) { return i < na ? i : b0 + i - na; };
    // Unconditional, so that each wait counts its own loads; past the run's end
    // the resource holds no bytes and nothing is read.
    auto load = [&](Block& x, int i) __attribute__((always_inline)) {
        const Region r = region(base + (size_t)block(i) * (128 * HD), i < end ? 128 * HD : 0);
#pragma unroll
        for (int j = 0; j < 2 * NS; ++j)
            x.k[j] = __builtin_bit_cast(half8, __builtin_amdgcn_raw_buffer_load_b128(r.r, 16 * lane + 1024 * j, 0, AUX));
#pragma unroll
        for (int j = 0; j < NT; ++j)
            x.v[j] = __builtin_bit_cast(
                half8, __builtin_amdgcn_raw_buffer_load_b128(r.r, 16 * lane + 1024 * (2 * NS + j), 0, AUX));
    };
    int i = begin + wave;
    Block x0, x1;
    load(x0, i);
    load(x1, i + RW);
    half8 qh[NS], ql[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) qh[s] = ql[s] = zero_h8();
    if (col < group) {
        const float* q = a.q + (size_t)seq * a.q_stride + (size_t)(kh * group + col) * HD + 8 * grp;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                half_t hi_, lo_;
                split_h(q[32 * s + j], hi_, lo_);
                qh[s][j] = hi_;
                ql[s][j] = lo_;
            }
    }
    const float sl2 = a.scale * LLMTIE_LOG2E;
    const float c1 = (MODE & SM_CAP) != 0 ? a.scale / a.softcap : 0.0f, c2 = a.softcap * LLMTIE_LOG2E;
    const float slope2 = (MODE & SM_BIAS) != 0 ? a.slopes[kh * group + min(col, group - 1)] * LLMTIE_LOG2E : 0.0f;
    floatx4 o[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) o[t] = zero_f4();
    float m = RG_NOREF, l = 0.0f;

    auto fold = [&](Block& x, int b) __attribute__((always_inline)) {
        const int k0 = 32 * b;
        floatx4 sc[2] = {zero_f4(), zero_f4()};
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int T = 0; T < 2; ++T) {
                sc[T] = mfma16(x.k[T * NS + s], ql[s], sc[T]);
                sc[T] = mfma16(x.k[T * NS + s], qh[s], sc[T]);
            }
        const bool part = !(k0 + 32 <= f || (k0 >= lo && k0 + 32 <= tk));
        if constexpr ((MODE & SM_CAP) != 0) cap_scores(sc, c1, sl2, c2);
        float mx = ninf();
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int key = k0 + 8 * grp + 4 * T + r;
                float s = (MODE & SM_CAP) != 0 ? sc[T][r] : sc[T][r] * sl2;
                if constexpr ((MODE & SM_BIAS) != 0) s = __builtin_fmaf(-slope2, (float)(tk - 1 - key), s);
                if (part) s = key < f || (key >= lo && key < tk) ? s : ninf();
                sc[T][r] = s;
                mx = fmaxf(mx, s);
            }
        mx = max4grp(mx);
        if (__any(mx > m)) {
            const float mn = fmaxf(m, mx), fac = ex2(m - mn);
            m = mn;
            l *= fac;
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t] *= fac;
        }
        half8 ph, pl;
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                // (The difference first: the key m is has 0, however large m is.)
                const float p = ex2((sc[T][r] - m) + RD_LIFT);
                l += p;
                half_t hi_, lo_;
                split_h(p, hi_, lo_);
                ph[4 * T + r] = hi_;
                pl[4 * T + r] = lo_;
            }
        if (part) {
            // Values of keys not seen may be anything; 0 * NaN is NaN.
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int key = k0 + 8 * grp + j;
                const bool see = key < f || (key >= lo && key < tk);
#pragma unroll
                for (int t = 0; t < NT; ++t) x.v[t][j] = see ? x.v[t][j] : (half_t)0.0f;
            }
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
            o[t] = mfma16(x.v[t], pl, o[t]);
            o[t] = mfma16(x.v[t], ph, o[t]);
        }
    };
    while (i < end) {
        fold(x0, block(i));
        load(x0, i + 2 * RW);
        i += RW;
        if (i >= end) break;
        fold(x1, block(i));
        load(x1, i + 2 * RW);
        i += RW;
    }

    // The four waves' O, (m, l) through LDS.
    l = sum4grp(l);
    if (col < group) {
#pragma unroll
        for (int t = 0; t < NT; ++t) *reinterpret_cast<floatx4*>(&lds[(wave * 16 + col) * OP + 16 * t + 4 * grp]) = o[t];
        if (grp == 0) wm[wave][col] = m, wl[wave][col] = l;
    }
    __syncthreads();
    auto weights = [&](int g, float (&w)[RW]) __attribute__((always_inline)) {
        float M = wm[0][g];
#pragma unroll
        for (int k = 1; k < RW; ++k) M = fmaxf(M, wm[k][g]);
#pragma unroll
        for (int k = 0; k < RW; ++k) w[k] = ex2(wm[k][g] - M);
        return M;
    };
    auto total = [&](int g, const float (&w)[RW]) __attribute__((always_inline)) {
        float L = 0.0f;
#pragma unroll
        for (int k = 0; k < RW; ++k) L += wl[k][g] * w[k];
        return L;
    };
    auto column = [&](int e4, const float (&w)[RW]) __attribute__((always_inline)) {
        const int g = 4 * e4 / HD, d = 4 * e4 % HD;
        floatx4 y = zero_f4();
#pragma unroll
        for (int k = 0; k < RW; ++k) y += *reinterpret_cast<const floatx4*>(&lds[(k * 16 + g) * OP + d]) * w[k];
        return y;
    };
    float w[RW];
    if (runs == 1) {
        for (int e4 = tid; e4 < n / 4; e4 += RT) {
            const int g = 4 * e4 / HD;
            weights(g, w);
            const float L = total(g, w);
            *reinterpret_cast<floatx4*>(out + 4 * e4) = column(e4, w) * (L > 0.0f || L != L ? 1.0f / L : 0.0f);
        }
        return;
    }
    // The run's partials, coherent past the XCDs' separate L2s; the stores are
    // waited for before the arrival is counted.
    float* po = a.part + (size_t)head * a.splits * n;
    float* pml = a.part + a.ml_off + (size_t)head * a.splits * group * 2;
    {
        const __amdgpu_buffer_rsrc_t rp = __builtin_amdgcn_make_buffer_rsrc(po + (size_t)sp * n, 0, n * 4, 0x00020000);
        typedef float v4 __attribute__((ext_vector_type(4)));
        for (int e4 = tid; e4 < n / 4; e4 += RT) {
            weights(4 * e4 / HD, w);
            const floatx4 y = column(e4, w);
            const v4 z = {y[0], y[1], y[2], y[3]};
            __builtin_amdgcn_raw_buffer_store_b128(z, rp, e4 * 16, 0, AUX_AGENT);
        }
    }
    if (tid < group) {
        const float M = weights(tid, w);
        st_coherent(pml + ((size_t)sp * group + tid) * 2, M);
        st_coherent(pml + ((size_t)sp * group + tid) * 2 + 1, total(tid, w));
    }
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    unsigned* ctr = a.ctr + (size_t)head * CTR_STRIDE;
    if (tid == 0)
        last = __hip_atomic_fetch_add(ctr, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)(runs - 1);
    __syncthreads();
    if (!last) return;
    __atomic_signal_fence(__ATOMIC_SEQ_CST);

    // The merge, runs in order: their (m, l) and the first columns in flight together.
    float* wt = lds;                        // [runs][group]
    float* gl = lds + 2 * RD_MAX_ROWS;      // [group]
    floatx4* red = reinterpret_cast<floatx4*>(lds + 2 * RD_MAX_ROWS + 16);  // [RT]
    const Region ro = region(po, (uint32_t)((size_t)runs * n * 4));
    const Region rml = region(pml, (uint32_t)((size_t)runs * group * 8));
    constexpr uint32_t OUT = 0x80000000u;  // past any region
    for (int g = wave; g < group; g += RW) {
        float mx = ninf(), L = 0.0f;
        float2 c[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = lane + 64 * k;
            c[k] = ld_region2<AUX_AGENT>(rml, s < runs ? (uint32_t)((s * group + g) * 8) : OUT);
            if (s < runs) mx = fmaxf(mx, c[k].x);
        }
        mx = wave_max(mx);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int s = lane + 64 * k;
            if (s < runs) {
                const float x = ex2(c[k].x - mx);
                wt[s * group + g] = x;
                L += c[k].y * x;
            }
        }
        L = wave_sum(L);
        if (lane == 0) gl[g] = L;
    }
    __syncthreads();
    const int C = n / 4, R = C >= RT ? 1 : RT / C;  // columns; phases of the runs
    for (int cb = 0; cb < C; cb += RT) {
        const int c4 = cb + (R > 1 ? tid % C : tid), phase = R > 1 ? tid / C : 0;
        const bool has = c4 < C && phase < R;
        const int g = min(4 * c4 / HD, group - 1);
        floatx4 acc = zero_f4();
        constexpr int U = 8;
        for (int s0 = phase; has && s0 < runs; s0 += U * R) {
            float4 y[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * R;
                y[u] = ld_region4<AUX_AGENT>(ro, s < runs ? (uint32_t)(((size_t)s * n + 4 * c4) * 4) : OUT);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int s = s0 + u * R;
                const float x = s < runs ? wt[s * group + g] : 0.0f;
                acc += floatx4{y[u].x, y[u].y, y[u].z, y[u].w} * x;
            }
        }
        red[tid] = acc;
        __syncthreads();
        if (has && phase == 0) {
            for (int k = 1; k < R; ++k) acc += red[tid + k * C];
            const float L = gl[g];
            *reinterpret_cast<floatx4*>(out + 4 * c4) = acc * (L > 0.0f || L != L ? 1.0f / L : 0.0f);
        }
        __syncthreads();
    }
    if (tid == 0) __hip_atomic_store(ctr, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

hipError_t launch_ranges_decode(int hd, const RangesDecodeArgs& a, hipStream_t st) {
    const dim3 grid((unsigned)((size_t)a.nseq * a.kv_heads * a.splits));
    const int mode = (a.softcap > 0.0f ? SM_CAP : 0) | (a.slopes ? SM_BIAS : 0);
#define RD(HD, M)                                                                         \
    if (hd == HD && mode == M) {                                                          \
        if (a.stream)                                                                     \
            hipLaunchKernelGGL((ranges_decode_kernel<HD, M, AUX_STREAM>), grid, dim3(RT), 0, st, a); \
        else hipLaunchKernelGGL((ranges_decode_kernel<HD, M, 0>), grid, dim3(RT), 0, st, a); \
        return hipGetLastError();                                                         \
    }
    RD(64, 0) RD(64, 1) RD(64, 2) RD(64, 3) RD(128, 0) RD(128, 1) RD(128, 2) RD(128, 3)
#undef RD
    return hipErrorInvalidValue;
}

}  // namespace llmtie
