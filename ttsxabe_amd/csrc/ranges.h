// Launch interface of the attention over key ranges (ranges.hip): prompts and
// batched single tokens over a tiled f16 cache, scores capped or biased.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace llmtie {

// Which keys the rows of a packed prompt see (llmtie_key_ranges).
struct KeyRangeArgs {
    const int* starts;  // [docs + 1] first rows of the documents, or null: one document from cache position 0
    const int* prefix;  // [docs] leading rows that a document's rows all see, or null
    int* table;         // first, lo, hi, `rows` each
    int* pos;           // rotary positions, or null
    int docs, rows, past, causal, window, shared;
};
hipError_t launch_key_ranges(const KeyRangeArgs& a, hipStream_t st);

struct RangesArgs {
    const uint16_t* q;      // f16 query rows, q_stride apart
    const uint16_t* cache;  // the slot's blocks: [kv_heads][blocks of 32 positions]
    uint16_t* out;          // f16 [tq, heads * hd]
    const int* first;       // [tq] each: row r sees keys j < first[r] and lo[r] <= j < hi[r]
    const int* lo;
    const int* hi;
    const float* slopes;    // [heads] distance bias, or null
    long q_stride;
    int tq, past, heads, kv_heads, cap;
    float scale, softcap;   // softcap 0: none
    float lift;             // binades that a row's largest weight is formed above 1 (0 to 10)
    int gb;                 // query heads of a workgroup (1, 2 or 4)
    int splits;             // runs of a row block's tiles (1: whole)
    float* ws;              // splits > 1: splits * tq * heads * (hd + 2) floats
    // Set by launch_ranges: workgroup L runs item (L % 8) * grid8 + L / 8 of
    // the (head group, run, row block) list, so that each XCD, dealt every
    // eighth workgroup, takes whole head groups and keeps their K and V in its L2.
    int nrb, grid8, xcd;
    int qal;                // query rows are 16-byte aligned
};
// nqt: 16-row query tiles a wave (1 or 2).
hipError_t launch_ranges(int hd, int nqt, const RangesArgs& a, hipStream_t st);

struct RangesDecodeArgs {
    const float* q;         // sequence s's heads at s * q_stride
    const uint16_t* cache;  // [slots][kv_heads][blocks]
    float* out;             // [nseq, heads * hd]
    const int* tk;          // [nseq] live lengths
    const int* slot;        // [nseq], or null: slot s for sequence s
    const int* lo;          // [nseq] first key behind the shared ones, or null
    const float* slopes;
    float* part;            // [nseq * kv_heads][splits][group * hd], then (m, l) at ml_off
    long ml_off;
    unsigned* ctr;          // arrivals, one every CTR_STRIDE words, zero between calls
    long q_stride;
    int nseq, slots, cap, kv_heads, group, window, shared;
    int splits, span;       // workgroups of a head at most; blocks of 32 keys each takes at least
    int whole;              // a head of up to so many blocks is one workgroup's
    int stream;             // more bytes than are worth keeping in the Infinity Cache
    float scale, softcap;
};
hipError_t launch_ranges_decode(int hd, const RangesDecodeArgs& a, hipStream_t st);

}  // namespace llmtie
