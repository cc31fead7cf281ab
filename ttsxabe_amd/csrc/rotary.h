// Launch interface of the rotary positions by row (rotary.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llmtie {

struct RotaryArgs {
    const float* q;    // rows of `heads` heads, q_stride apart; null: none
    void* qo;          // the rotated rows: f32, or f16 where qo_f16 (may be q itself)
    const float* k;    // store only: rows of `kv` heads to rotate and store ..
    const float* v;    // .. and to store
    const int* pos;    // [rows] rotary positions, or null: first + row
    const int* slot;   // store only: [rows] cache slot and position
    const int* index;
    const int* table;  // paged store: [trows][tcols] slots (pages of 2^shift positions); slot is then a row of it
    const float* div;  // [rot / 2] divisors of the frequencies, or null
    uint16_t* cache;   // [slots][kv][blocks of 32 positions]
    long q_stride, qo_stride, k_stride, v_stride;
    int rows, heads, kv, hd, rot, first, interleaved, qo_f16, slots, cap;
    int trows, tcols, shift;
    float mscale;
    double log2_theta;
};
// store: k and v go to the cache too, where the table has their pages if there is one.
hipError_t launch_rotary(const RotaryArgs& a, bool store, hipStream_t st);

}  // namespace llmtie
