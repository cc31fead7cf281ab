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

// A workgroup takes PN rows and a run of the heads (q's, then k's, then v's):
// the rows' angles once into LDS, then its heads' units of 2 V dims. PN = 8
// (prompts) lies on multiples of eight of the first row's cache position, so
// that eight rows of v fill whole 16-byte runs of the cache.
template <int V, int PN, bool STORE>
__global__ __launch_bounds__(RO) void rotary_kernel(RotaryArgs a, int groups, int hpb) {
    extern __shared__ float2 cs[];  // [PN][rot / 2] (cos, sin) * mscale
    const int tid = threadIdx.x, half = a.rot / 2, hd = a.hd;
    const int nh = a.q ? a.heads : 0, all = nh + (STORE ? 2 * a.kv : 0);
    const int h0 = (int)blockIdx.y * hpb, h1 = min(all, h0 + hpb);
    const int shift = STORE && PN == 8 ? a.index[0] & 7 : 0;
    const int units = hd / (2 * V), turned = half / V;  // units of a head; of them rotated
    const int nblk = STORE ? tiled_nblk(a.cap) : 0;
    for (int g = blockIdx.x; g < groups; g += gridDim.x) {
        const int r0 = PN * g - shift;
        if (h0 < nh + (STORE ? a.kv : 0)) {
            for (int e = tid; e < PN * half; e += RO) {
                const int p = e / half, j = e % half, r = r0 + p;
                if (r < 0 || r >= a.rows) continue;
                double f = exp2(-2.0 * j / a.rot * a.log2_theta) * 0.15915494309189535;
                if (a.div) f /= (double)a.div[j];
                const double t = f * (double)(a.pos ? a.pos[r] : a.first + r);
                float s, c;
                sincospif((float)(2.0 * (t - rint(t))), &s, &c);
                cs[e] = make_float2(c * a.mscale, s * a.mscale);
            }
        }
        __syncthreads();
        // The rotated heads: q's and k's.
        auto rotate = [&](const float* src, int p, int u, float (&lo)[V], float (&hi)[V], int& d0, int& d1)
            __attribute__((always_inline)) {
            if (u < turned) {
                if (a.interleaved) {
                    d0 = 2 * V * u;
                    d1 = d0 + V;
                    const Vec<V> x = ld_vec<V>(src + d0), y = ld_vec<V>(src + d1);
                    float z[2 * V];
#pragma unroll
                    for (int i = 0; i < V; ++i) z[i] = x.x[i], z[V + i] = y.x[i];
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float2 w = cs[p * half + V * u + i];
                        const float re = z[2 * i] * w.x - z[2 * i + 1] * w.y, im = z[2 * i] * w.y + z[2 * i + 1] * w.x;
                        z[2 * i] = re;
                        z[2 * i + 1] = im;
                    }
#pragma unroll
                    for (int i = 0; i < V; ++i) lo[i] = z[i], hi[i] = z[V + i];
                } else {
                    d0 = V * u;
                    d1 = d0 + half;
                    const Vec<V> x = ld_vec<V>(src + d0), y = ld_vec<V>(src + d1);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        const float2 w = cs[p * half + V * u + i];
                        lo[i] = x.x[i] * w.x - y.x[i] * w.y;
                        hi[i] = x.x[i] * w.y + y.x[i] * w.x;
                    }
                }
            } else {
                d0 = 2 * V * u;
                d1 = d0 + V;
                const Vec<V> x = ld_vec<V>(src + d0), y = ld_vec<V>(src + d1);
#pragma unroll
                for (int i = 0; i < V; ++i) lo[i] = x.x[i], hi[i] = y.x[i];
            }
        };
        const int q1 = min(h1, nh);
        if (h0 < q1) {
            const int n = (q1 - h0) * units;
            for (int e = tid; e < PN * n; e += RO) {
                const int p = e / n, u = e % n % units, h = h0 + e % n / units, r = r0 + p;
                if (r < 0 || r >= a.rows) continue;
                float lo[V], hi[V];
                int d0, d1;
                rotate(a.q + (size_t)r * a.q_stride + (size_t)h * hd, p, u, lo, hi, d0, d1);
                const size_t at = (size_t)r * a.qo_stride + (size_t)h * hd;
                if (a.qo_f16) {
                    st_vec<V>(static_cast<half_t*>(a.qo) + at + d0, lo);
                    st_vec<V>(static_cast<half_t*>(a.qo) + at + d1, hi);
                } else {
                    st_vec<V>(static_cast<float*>(a.qo) + at + d0, lo);
                    st_vec<V>(static_cast<float*>(a.qo) + at + d1, hi);
                }
            }
        }
        if constexpr (STORE) {
            auto home = [&](int r, int kh, int& kk) -> half_t* {
                const int s = a.slot[r], i = a.index[r];
                kk = i & 31;
                if (s < 0 || s >= a.slots || i < 0 || i >= a.cap) return nullptr;  // a padding row
                return reinterpret_cast<half_t*>(a.cache) + (((size_t)s * a.kv + kh) * nblk + (i >> 5)) * (64 * (size_t)hd);
            };
            const int k0 = max(h0, nh), k1 = min(h1, nh + a.kv);
            if (k0 < k1) {
                const int n = (k1 - k0) * units;
                for (int e = tid; e < PN * n; e += RO) {
                    const int p = e / n, u = e % n % units, h = k0 - nh + e % n / units, r = r0 + p;
                    if (r < 0 || r >= a.rows) continue;
                    int kk;
                    half_t* b = home(r, h, kk);
                    if (!b) continue;
                    float lo[V], hi[V];
                    int d0, d1;
                    rotate(a.k + (size_t)r * a.k_stride + (size_t)h * hd, p, u, lo, hi, d0, d1);
                    st_vec<V>(b + t16_k_off(hd, kk, d0), lo);
                    st_vec<V>(b + t16_k_off(hd, kk, d1), hi);
                }
            }
            const int v0 = max(h0, nh + a.kv), v1 = h1;
            if (v0 < v1) {
                // Four dims of PN rows a thread.
                const int quads = hd / 4, n = (v1 - v0) * quads;
                bool run = PN == 8;
                if constexpr (PN == 8) {
                    const int r = max(0, min(r0, a.rows - 1)), s = a.slot[r], i = a.index[r];
                    run = r0 >= 0 && r0 + 8 <= a.rows && (i & 7) == 0 && s >= 0 && s < a.slots && i >= 0 && i < a.cap - 7;
                    for (int p = 1; p < 8 && run; ++p) run = a.slot[r0 + p] == s && a.index[r0 + p] == i + p;
                }
                for (int e = tid; e < n; e += RO) {
                    const int h = v0 - nh - a.kv + e / quads, d = 4 * (e % quads);
                    float x[PN][4];
#pragma unroll
                    for (int p = 0; p < PN; ++p) {
                        const int r = max(0, min(r0 + p, a.rows - 1));
                        const float* src = a.v + (size_t)r * a.v_stride + (size_t)h * hd + d;
#pragma unroll
                        for (int i = 0; i < 4; i += V) {
                            const Vec<V> y = ld_vec<V>(src + i);
#pragma unroll
                            for (int c = 0; c < V; ++c) x[p][i + c] = y.x[c];
                        }
                    }
                    if (run) {
                        int kk;
                        half_t* b = home(r0, h, kk) + 32 * hd;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            half8 y;
#pragma unroll
                            for (int p = 0; p < 8; ++p) y[p] = to_h(x[p % PN][i]);
                            *reinterpret_cast<half8*>(b + t16_v_off(kk, d + i)) = y;
                        }
                        continue;
                    }
#pragma unroll
                    for (int p = 0; p < PN; ++p) {
                        const int r = r0 + p;
                        if (r < 0 || r >= a.rows) continue;
                        int kk;
                        half_t* b = home(r, h, kk);
                        if (!b) continue;
#pragma unroll
                        for (int i = 0; i < 4; ++i) b[32 * hd + t16_v_off(kk, d + i)] = to_h(x[p][i]);
                    }
                }
            }
        }
        __syncthreads();  // the angles are read
    }
}

static inline bool at16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

hipError_t launch_rotary(const RotaryArgs& a, bool store, hipStream_t st) {
    const int all = (a.q ? a.heads : 0) + (store ? 2 * a.kv : 0);
    if (a.rows == 0 || all == 0) return hipSuccess;
    bool vec = a.rot % 8 == 0 && a.hd % 8 == 0;
    if (a.q)
        vec = vec && at16(a.q) && a.q_stride % 4 == 0 && a.qo_stride % 4 == 0 &&
              (reinterpret_cast<uintptr_t>(a.qo) & (a.qo_f16 ? 7 : 15)) == 0;
    if (store) vec = vec && at16(a.k) && at16(a.v) && a.k_stride % 4 == 0 && a.v_stride % 4 == 0;
    const bool many = a.rows >= 64;
    const int pn = many ? 8 : 1;
    const int groups = many ? (int)(((long)a.rows + 14) / 8) : a.rows;
    const int ny = std::max(1, std::min(all, (1024 + groups - 1) / groups));
    const int hpb = (all + ny - 1) / ny;
    const dim3 grid((unsigned)std::min(groups, 1 << 16), (unsigned)((all + hpb - 1) / hpb));
    const size_t lds = (size_t)pn * (a.rot / 2) * sizeof(float2);
#define RO_(V, PN, S)                                                                                     \
    if ((vec ? 4 : 1) == V && pn == PN && store == S) {                                                   \
        hipLaunchKernelGGL((rotary_kernel<V, PN, S>), grid, dim3(RO), lds, st, a, groups, hpb);           \
        return hipGetLastError();                                                                         \
    }
    RO_(4, 8, false) RO_(4, 1, false) RO_(1, 8, false) RO_(1, 1, false)
    RO_(4, 8, true) RO_(4, 1, true) RO_(1, 8, true) RO_(1, 1, true)
#undef RO_
    return hipErrorInvalidValue;
}

}  // namespace llmtie
