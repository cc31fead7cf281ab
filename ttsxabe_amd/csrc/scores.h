// What the attention kernels over key ranges and over pages do to their scores.
#pragma once
#include "common.h"

namespace llmtie {

// What a launch does to its scores.
constexpr int SM_CAP = 1, SM_BIAS = 2;

// A reference max before a row has one: finite, so that 2^(s - m) of any seen
// key overflows (and moves m) while an unseen one's, s = -inf, is 0.
constexpr float RG_NOREF = -1e30f;

// A weight is formed as 2^(s - m + RD_LIFT), m the largest score: what f16's
// smallest half step, 2^-25, takes from it is then 2^-40 of the largest weight
// (unlifted, keys 25 below a dominant one were in l and not in O). O and l
// carry the same factor, and 2^15 is within f16. Its addition is not seen in
// the time (32 sequences of 256-8192 96.2 us with and without it, one of 4001 9.6).
// The kernels over pages have it in the reference, a weight's one subtraction.
constexpr float RD_LIFT = 15.0f;

// c2 tanh(c1 s) of a lane's eight scores, c1 c2 = sl2. For |x| up to 0.45 the
// series of tanh x / x to x^12, 2^-25.6 off there; where a lane's score is
// larger the library's, which branches for each (one sequence of 500 positions
// of 32/8/128 8.56 -> 7.82 us, of 40/40/128 10.4 -> 9.6; without a cap 7.2, 9.1).
// (1 - 2 / (1 + e^2x), as the prompts have it, is off by a half step of c, not of
// the score.)
__device__ __forceinline__ void cap_scores(floatx4 (&sc)[2], float c1, float sl2, float c2) {
    float top = 0.0f;
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, fabsf(sc[T][r]));
    if (__any(top * c1 > 0.45f)) {
#pragma unroll
        for (int T = 0; T < 2; ++T)
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[T][r] = c2 * tanhf(sc[T][r] * c1);
        return;
    }
#pragma unroll
    for (int T = 0; T < 2; ++T)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float x = sc[T][r] * c1, t = x * x, z = sc[T][r] * sl2;
            float p = __builtin_fmaf(t, 21844.0f / 6081075.0f, -1382.0f / 155925.0f);
            p = __builtin_fmaf(p, t, 62.0f / 2835.0f);
            p = __builtin_fmaf(p, t, -17.0f / 315.0f);
            p = __builtin_fmaf(p, t, 2.0f / 15.0f);
            p = __builtin_fmaf(p, t, -1.0f / 3.0f);
            sc[T][r] = __builtin_fmaf(z * t, p, z);
        }
}

}  // namespace llmtie
