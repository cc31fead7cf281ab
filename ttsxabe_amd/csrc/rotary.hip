// Rotary positions by row: each row at a position of its own, pairs of halves
// (i, i + rot / 2) or interleaved (2i, 2i + 1), over the first `rot` dims of a
// head, frequencies theta^(-2i / rot) / div_i, the rotated values times mscale;
// and the same with the store of k and v into the slots of a tiled f16 cache.
//
// Positions of extended contexts are large: an angle of 131072 radians has an
// ulp of 1/128 in f32. The angle is therefore formed in f64 as turns and
// reduced to a half before its sine and cosine are taken in f32.
#include <algorithm>

#include "common.h"
#include "kvlayout.h"
#include "rotary.h"

namespace llmtie {

constexpr int RO = 256;
constexpr int GR = 64;  // rows from which a store takes k and v eight rows at a time

// V values of a pair's side, as loaded and stored.
template <int V>
struct Vec {
    float x[V];
};
template <int V>
__device__ __forceinline__ Vec<V> ld_vec(const float* p) {
    Vec<V> r;
    if constexpr (V == 4) {
        const float4 y = *reinterpret_cast<const float4*>(p);
        r.x[0] = y.x, r.x[1] = y.y, r.x[2] = y.z, r.x[3] = y.w;
    } else {
        r.x[0] = *p;
    }
    return r;
}
template <int V>
__device__ __forceinline__ void st_vec(float* p, const float* x) {
    if constexpr (V == 4) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else *p = x[0];
}
template <int V>
__device__ __forceinline__ void st_vec(half_t* p, const float* x) {
    if constexpr (V == 4) {
        half4 y;
        y[0] = to_h(x[0]), y[1] = to_h(x[1]), y[2] = to_h(x[2]), y[3] = to_h(x[3]);
        *reinterpret_cast<half4*>(p) = y;
    } else {
        *p = to_h(x[0]);
    }
}

// The angles of PN rows from r0 on: (cos, sin) * mscale of pair j of row r0 + p
// at cs[p * rot / 2 + j].
template <int PN>
__device__ __forceinline__ void angles(const RotaryArgs& a, int r0, float2* cs, int tid) {
    const int half = a.rot / 2;
    for (int e = tid; e < PN * half; e += RO) {
        const int p = PN == 1 ? 0 : e / half, j = PN == 1 ? e : e % half, r = r0 + p;
        if (r < 0 || r >= a.rows) continue;
        double f = exp2(-2.0 * j / a.rot * a.log2_theta) * 0.15915494309189535;  // turns a position
        if (a.div) f /= (double)a.div[j];
        const double t = f * (double)(a.pos ? a.pos[r] : a.first + r);
        float s, c;
        sincospif((float)(2.0 * (t - rint(t))), &s, &c);
        cs[e] = make_float2(c * a.mscale, s * a.mscale);
    }
}

// A head is rot / 2 V units of V dims and their V partners, then (hd - rot) / 2 V
// units of 2 V dims that are not rotated. d0 and d1 are where a unit's two
// halves lie.
template <int V>
struct Unit {
    Vec<V> x, y;
    int d0, d1;
    __device__ __forceinline__ Unit(const RotaryArgs& a, const float* head, int u) {
        const bool halves = !a.interleaved && u < a.rot / 2 / V;
        d0 = halves ? V * u : 2 * V * u;
        d1 = halves ? d0 + a.rot / 2 : d0 + V;
        x = ld_vec<V>(head + d0);
        y = ld_vec<V>(head + d1);
    }
    __device__ __forceinline__ void turn(const RotaryArgs& a, const float2* cs, int u) {
        if (u >= a.rot / 2 / V) return;
        if (!a.interleaved) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 w = cs[V * u + i];
                const float re = x.x[i] * w.x - y.x[i] * w.y;
                y.x[i] = x.x[i] * w.y + y.x[i] * w.x;
                x.x[i] = re;
            }
        } else {
            float z[2 * V];
#pragma unroll
            for (int i = 0; i < V; ++i) z[i] = x.x[i], z[V + i] = y.x[i];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 w = cs[V * u + i];
                const float re = z[2 * i] * w.x - z[2 * i + 1] * w.y;
                z[2 * i + 1] = z[2 * i] * w.y + z[2 * i + 1] * w.x;
                z[2 * i] = re;
            }
#pragma unroll
            for (int i = 0; i < V; ++i) x.x[i] = z[i], y.x[i] = z[V + i];
        }
    }
};

// Block of row r's place for kv head kh, its position in it in kk; null for a
// padding row.
__device__ __forceinline__ half_t* home(const RotaryArgs& a, int r, int kh, int& kk) {
    const int s = a.slot[r], i = a.index[r];
    kk = i & 31;
    if (s < 0 || s >= a.slots || i < 0 || i >= a.cap) return nullptr;
    return reinterpret_cast<half_t*>(a.cache) +
           (((size_t)s * a.kv + kh) * tiled_nblk(a.cap) + (i >> 5)) * (64 * (size_t)a.hd);
}

template <int V>
__device__ __forceinline__ void put_q(const RotaryArgs& a, int r, int h, const Unit<V>& x) {
    const size_t at = (size_t)r * a.qo_stride + (size_t)h * a.hd;
    if (a.qo_f16) {
        st_vec<V>(static_cast<half_t*>(a.qo) + at + x.d0, x.x.x);
        st_vec<V>(static_cast<half_t*>(a.qo) + at + x.d1, x.y.x);
    } else {
        st_vec<V>(static_cast<float*>(a.qo) + at + x.d0, x.x.x);
        st_vec<V>(static_cast<float*>(a.qo) + at + x.d1, x.y.x);
    }
}
template <int V>
__device__ __forceinline__ void put_k(const RotaryArgs& a, int r, int h, const Unit<V>& x) {
    int kk;
    half_t* b = home(a, r, h, kk);
    if (!b) return;
    st_vec<V>(b + t16_k_off(a.hd, kk, x.d0), x.x.x);
    st_vec<V>(b + t16_k_off(a.hd, kk, x.d1), x.y.x);
}

// One row a workgroup, heads h0 .. h1 - 1 of q's, k's and v's. (Eight rows a
// workgroup, which form 512 angles before their first load: 8192 rows of 32
// heads of 128 46.9 -> 42.5 us, 6.3 TB/s of reads and writes; with 96 of 128
// dims rotated 54 -> 43; a turn of 127 4.9 -> 4.2. Loading two units a thread
// before the angles took 30 registers more and was no faster: 45, 45.9, 4.6.)
template <int V, bool STORE>
__device__ __forceinline__ void row(const RotaryArgs& a, int r, int h0, int h1, float2* cs, int tid) {
    const int units = a.hd / (2 * V), nh = a.q ? a.heads : 0;
    const int t1 = min(h1, nh + (STORE ? a.kv : 0)), n = max(0, t1 - h0) * units;  // units to rotate
    auto head = [&](int h) {
        return h < nh ? a.q + (size_t)r * a.q_stride + (size_t)h * a.hd
                      : a.k + (size_t)r * a.k_stride + (size_t)(h - nh) * a.hd;
    };
    auto put = [&](int h, const Unit<V>& x) __attribute__((always_inline)) {
        if (!STORE || h < nh) put_q<V>(a, r, h, x);
        else put_k<V>(a, r, h - nh, x);
    };
    if (n > 0) {
        angles<1>(a, r, cs, tid);
        __syncthreads();
        for (int e = tid; e < n; e += RO) {
            Unit<V> x(a, head(h0 + e / units), e % units);
            x.turn(a, cs, e % units);
            put(h0 + e / units, x);
        }
    }
    if constexpr (STORE) {
        // v: four dims a thread, one key of a chunk of eight (2-byte stores).
        const int v0 = max(h0, nh + a.kv), quads = a.hd / 4;
        for (int e = tid; e < (h1 - v0) * quads; e += RO) {
            const int h = v0 - nh - a.kv + e / quads, d = 4 * (e % quads);
            float x[4];
            const float* src = a.v + (size_t)r * a.v_stride + (size_t)h * a.hd + d;
#pragma unroll
            for (int i = 0; i < 4; i += V) {
                const Vec<V> y = ld_vec<V>(src + i);
#pragma unroll
                for (int c = 0; c < V; ++c) x[i + c] = y.x[c];
            }
            int kk;
            half_t* b = home(a, r, h, kk);
            if (!b) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) b[32 * a.hd + t16_v_off(kk, d + i)] = to_h(x[i]);
        }
    }
}

// Eight rows a workgroup, heads h0 .. h1 - 1 of k's and v's, for prompts: rows
// that fill a run of eight cache positions store v in whole 16-byte chunks, and
// k's 16-byte chunks of the rows lie together. r0 is a multiple of eight behind
// the first row's cache position, so a run's rows do. Us, with k and v by row /
// so: 4000 rows of 32/8/128 50.6 / 31.5 (147 MB; a copy of them 28.6), 1999 24.6 /
// 16.0, 500 10.2 / 7.3, 100 5.0 / 5.1, 64 4.9 / 4.8; rows of a place each 32 4.5 / 6.5.
template <int V>
__device__ __forceinline__ void rows8(const RotaryArgs& a, int r0, int h0, int h1, float2* cs, int tid) {
    const int units = a.hd / (2 * V), half = a.rot / 2, k1 = min(h1, a.kv);
    if (h0 < k1) {
        angles<8>(a, r0, cs, tid);
        __syncthreads();
        const int n = (k1 - h0) * units;
        for (int e = tid; e < 8 * n; e += RO) {
            const int p = e / n, u = e % n % units, h = h0 + e % n / units, r = r0 + p;
            if (r < 0 || r >= a.rows) continue;
            Unit<V> x(a, a.k + (size_t)r * a.k_stride + (size_t)h * a.hd, u);
            x.turn(a, cs + p * half, u);
            put_k<V>(a, r, h, x);
        }
    }
    const int v0 = max(h0, a.kv);
    if (v0 >= h1) return;
    bool run = r0 >= 0 && r0 + 8 <= a.rows;
    if (run) {
        const int s = a.slot[r0], i = a.index[r0];
        run = (i & 7) == 0 && s >= 0 && s < a.slots && i >= 0 && i < a.cap - 7;
        for (int p = 1; p < 8 && run; ++p) run = a.slot[r0 + p] == s && a.index[r0 + p] == i + p;
    }
    const int quads = a.hd / 4;
    for (int e = tid; e < (h1 - v0) * quads; e += RO) {
        const int h = v0 - a.kv + e / quads, d = 4 * (e % quads);
        float x[8][4];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int r = max(0, min(r0 + p, a.rows - 1));
            const float* src = a.v + (size_t)r * a.v_stride + (size_t)h * a.hd + d;
#pragma unroll
            for (int i = 0; i < 4; i += V) {
                const Vec<V> y = ld_vec<V>(src + i);
#pragma unroll
                for (int c = 0; c < V; ++c) x[p][i + c] = y.x[c];
            }
        }
        int kk;
        if (run) {
            half_t* b = home(a, r0, h, kk) + 32 * a.hd;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                half8 y;
#pragma unroll
                for (int p = 0; p < 8; ++p) y[p] = to_h(x[p][i]);
                *reinterpret_cast<half8*>(b + t16_v_off(kk, d + i)) = y;
            }
            continue;
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
            const int r = r0 + p;
            if (r < 0 || r >= a.rows) continue;
            half_t* b = home(a, r, h, kk);
            if (!b) continue;
#pragma unroll
            for (int i = 0; i < 4; ++i) b[32 * a.hd + t16_v_off(kk, d + i)] = to_h(x[p][i]);
        }
    }
}

// GROUPS: the first `g8` workgroups take k and v eight rows at a time, the
// others q by row; else all by row. Rows past a launch's workgroups follow at
// its stride.
template <int V, bool STORE, bool GROUPS>
__global__ __launch_bounds__(RO) void rotary_kernel(RotaryArgs a, int g8, int hpb8, int groups, int hpb, int heads) {
    extern __shared__ float2 cs[];
    const int tid = threadIdx.x;
    if constexpr (GROUPS) {
        if ((int)blockIdx.x < g8) {
            const int per = (2 * a.kv + hpb8 - 1) / hpb8, g = (int)blockIdx.x / per, h0 = (int)blockIdx.x % per * hpb8;
            const int shift = a.index[0] & 7;
            rows8<V>(a, 8 * g - shift, h0, min(2 * a.kv, h0 + hpb8), cs, tid);
            return;
        }
    }
    const int per = (heads + hpb - 1) / hpb, b = (int)blockIdx.x - (GROUPS ? g8 : 0);
    const int h0 = b % per * hpb, stride = ((int)gridDim.x - (GROUPS ? g8 : 0)) / per;
    for (int r = b / per; r < groups; r += stride) {
        row<V, STORE && !GROUPS>(a, r, h0, min(heads, h0 + hpb), cs, tid);
        __syncthreads();  // the angles are read
    }
}

static inline bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

hipError_t launch_rotary(const RotaryArgs& a, bool store, hipStream_t st) {
    const int nq = a.q ? a.heads : 0;
    if (a.rows == 0 || nq + (store ? a.kv : 0) == 0) return hipSuccess;
    bool vec = a.rot % 8 == 0 && a.hd % 8 == 0;
    if (a.q)
        vec = vec && at16(a.q) && a.q_stride % 4 == 0 && a.qo_stride % 4 == 0 &&
              (reinterpret_cast<uintptr_t>(a.qo) & (a.qo_f16 ? 7 : 15)) == 0;
    if (store) vec = vec && at16(a.k) && at16(a.v) && a.k_stride % 4 == 0 && a.v_stride % 4 == 0;
    const bool groups = store && a.rows >= GR;
    // Heads of a row are split over workgroups as far as the rows leave the chip
    // short of two a compute unit (each forms the angles again): four, 500 rows
    // 9.0 us against 7.3, 30 rows of q alone 4.1 / 3.7.
    auto split = [](int heads, long n) { return std::max(1, (int)std::min<long>(heads, (512 + n - 1) / n)); };
    const int heads = groups ? nq : nq + (store ? 2 * a.kv : 0);
    const int hpb = heads ? (heads + split(heads, a.rows) - 1) / split(heads, a.rows) : 1;
    const int per = heads ? (heads + hpb - 1) / hpb : 0;
    const long n8 = groups ? ((long)a.rows + 14) / 8 : 0;
    const int hpb8 = groups ? (2 * a.kv + split(2 * a.kv, n8) - 1) / split(2 * a.kv, n8) : 1;
    const int g8 = groups ? (int)(n8 * ((2 * a.kv + hpb8 - 1) / hpb8)) : 0;
    const int rows = std::min(a.rows, 1 << 16);
    const dim3 grid((unsigned)(g8 + rows * per));
    const size_t lds = (size_t)(groups ? 8 : 1) * (a.rot / 2) * sizeof(float2);
#define RO_(V, S, G)                                                                                              \
    if ((vec ? 4 : 1) == V && store == S && groups == G) {                                                        \
        hipLaunchKernelGGL((rotary_kernel<V, S, G>), grid, dim3(RO), lds, st, a, g8, hpb8, a.rows, hpb, heads);   \
        return hipGetLastError();                                                                                 \
    }
    RO_(4, false, false) RO_(4, true, false) RO_(4, true, true) RO_(1, false, false) RO_(1, true, false) RO_(1, true, true)
#undef RO_
    return hipErrorInvalidValue;
}

}  // namespace llmtie
