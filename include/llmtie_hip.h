/*
 * llmtie_hip.h - C ABI of the MI355X (gfx950) fused-attention library.
 *
 * A drop-in replacement for the attention operators of the reference's
 * `llmtie_cuda::Gpu` (crates/llmtie-cuda/src/device.rs) and for the KV-cache
 * producers they read from. Every entry point takes plain device pointers with
 * element counts (so every bounds check the reference makes can still be made),
 * a hipStream_t passed as `void*` (NULL = the default stream), and returns a
 * status code named after the reference's `CudaError` variant
 * (crates/llmtie-cuda/src/error.rs:148-282). Shapes are refused before any
 * launch; a refused call touches no memory. Outputs are caller-owned.
 *
 * Calls are asynchronous on `stream` exactly like the reference's (one stream
 * per Gpu, device.rs:740-755). A decode scratch must not be shared by calls
 * that can run concurrently (device.rs:166-180).
 *
 * Layouts (as in the reference unless noted):
 *   q           [rows, heads * head_dim] f32, the heads of one GQA group adjacent
 *   K cache     [kv_heads, cap, head_dim]   (f32 or f16 bits)
 *   V cache     [kv_heads, head_dim, cap]   (transposed, f32 or f16 bits)
 *   tiled f16   (new) one buffer per layer, [kv_heads][blocks of 32 positions],
 *               each block K then V in MFMA fragment order (kvlayout.h); with
 *               slots, one such cache after the other
 *   Q8_0 cache  (new; no reference counterpart) for `slots` sequences, tiled the
 *               same way: [slots][kv_heads][blocks], each block K codes, V
 *               codes, K scales, V scales; element = f16 scale * int8 code, one
 *               scale per 32 dims of one position (the GGUF Q8_0 block,
 *               crates/llmtie-gguf/src/dequant.rs:180-185); 272 bytes per
 *               position and kv head at head_dim 128.
 *   int8 twin   `n` int8 codes then `n / 32` f32 scales in one buffer (the
 *               reference's `Q8` buffer, device.rs:498-520)
 */
#ifndef LLMTIE_HIP_H
#define LLMTIE_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes: one per `CudaError` variant the attention path can raise. */
typedef enum llmtie_status {
    LLMTIE_OK = 0,
    LLMTIE_UNSUPPORTED_ATTENTION = 1, /* UnsupportedAttention{head_dim, heads, kv_heads} error.rs:270 */
    LLMTIE_ODD_CACHE_CAPACITY = 2,    /* OddCacheCapacity{cap}            error.rs:178 */
    LLMTIE_CACHE_OVERRUN = 3,         /* CacheOverrun{at, cap}            error.rs:162 */
    LLMTIE_SLICE_OVERRUN = 4,         /* SliceOverrun{at, len}            error.rs:149 */
    LLMTIE_RAGGED_BLOCK = 5,          /* RaggedBlock{k, block}            error.rs:63 */
    LLMTIE_MISMATCHED_Q8 = 6,         /* MismatchedQ8{rows, k, want_rows, want_k} error.rs:129 */
    LLMTIE_ODD_HEAD_DIM = 7,          /* OddHeadDim{head_dim}             error.rs:210 */
    LLMTIE_DRIVER = 8,                /* Driver{what, source}             error.rs:281 */
    LLMTIE_NO_DEVICE = 9,             /* NoDevice(String)                 error.rs:242 */
    LLMTIE_INVALID_ARGUMENT = 10,     /* a null pointer where a buffer is required, or a prefill
                                        * workspace off 16 bytes (no reference twin) */
    LLMTIE_SCRATCH_GROWTH_IN_CAPTURE = 11, /* a decode scratch would have to grow while its stream captures a
                                            * graph (no reference twin: the reference does not capture);
                                            * fields: partial floats needed, held, counters needed, held */
    LLMTIE_SCRATCH_LIMIT = 12,             /* the fixed scratch of llmtie_attn_decode_f16_noalloc is too small
                                            * for the call (no reference twin); fields as above */
    LLMTIE_SPLIT_HEAD_LOST = 13            /* an earlier decode through this scratch wrote NaN for a head whose
                                            * split workgroups did not share an XCD (no reference twin; see
                                            * llmtie_decode_scratch_status); no fields */
} llmtie_status;

/* The last error raised on the calling thread: the status, up to four numeric
 * fields of the variant in its declaration order, and a rendered message. */
typedef struct llmtie_error {
    int status;
    size_t field[4];
    char message[240];
} llmtie_error;

/* Copies the calling thread's last error into *out; returns its status. */
int llmtie_last_error(llmtie_error* out);

/* Library version, "major.minor.patch". */
const char* llmtie_version(void);

/* Opaque decode scratch: split partials and arrival counters, grown on demand
 * and owned by the caller. Replaces `DecodeScratch::new()` (device.rs:219).
 * Its counters start at zero and every call leaves them at zero.
 * Graphs: a call captured into a HIP graph records the scratch's buffers.
 * Growth never frees a buffer: every replaced one stays allocated until
 * llmtie_decode_scratch_free, so an earlier graph keeps replaying correctly.
 * Growth is refused while the stream is capturing
 * (LLMTIE_SCRATCH_GROWTH_IN_CAPTURE): make one eager call of the largest shape
 * first. Freeing the scratch invalidates every graph that used it. */
typedef struct llmtie_decode_scratch llmtie_decode_scratch;
llmtie_decode_scratch* llmtie_decode_scratch_new(void);
void llmtie_decode_scratch_free(llmtie_decode_scratch* s);

/* The XCD-local split hand-off (no reference twin). When every XCD's run of a
 * launch's workgroups holds whole heads, a head's split partials pass
 * through that XCD's L2 instead of memory. The kernel checks that each head's
 * workgroups really shared an XCD; a head whose did not is written as NaN
 * (its int8 twin with NaN scales), never as a silently wrong context, and the
 * scratch records it in a host-visible word. The next decode call through the
 * scratch then returns LLMTIE_SPLIT_HEAD_LOST without launching, and
 * llmtie_decode_scratch_status returns (and clears) the same status after a
 * stream synchronisation; LLMTIE_OK otherwise. No failure has been seen on
 * gfx950, whose dispatcher deals workgroups L and L + 8k to one XCD; the
 * environment variable LLMTIE_DECODE_XCD=0 selects the coherent hand-off
 * everywhere (about 2 % slower at C2). The no-allocation entry point always
 * uses the coherent hand-off. */
int llmtie_decode_scratch_status(llmtie_decode_scratch* s);

/* Test hook (no reference twin; never needed in use): nonzero makes every
 * later decode report fake XCC ids (workgroup L as (L / 8) % 8) to the
 * XCD-local check, so a test can drive the check's failure path. */
void llmtie_debug_fake_xcc(int on);

/* ---------------------------------------------------------------- prefill */

/* Gpu::supports_flash (device.rs:5697): head_dim 64 or 128, heads a multiple
 * of kv_heads. */
int llmtie_supports_flash(size_t head_dim, size_t heads, size_t kv_heads);

/* Gpu::flash_attn (device.rs:5702): causal or full attention of tq query rows
 * (positions past .. past+tq-1) against an f32 cache holding past+tq keys.
 * out = [tq, heads*head_dim] f32.
 * The kernel rounds the f32 keys and values to f16 on their way into its
 * LDS tiles (the reference's arithmetic); nothing is allocated. */
int llmtie_flash_attn(void* stream, const float* q, size_t q_len, const float* k, size_t k_len,
                      const float* v, size_t v_len, float* out, size_t out_len, size_t tq, size_t past,
                      size_t heads, size_t kv_heads, size_t head_dim, size_t cap, float scale, int causal);

/* Gpu::flash_attn_f16 (device.rs:5754): the same against an f16 cache (cap even). */
int llmtie_flash_attn_f16(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                          const uint16_t* v, size_t v_len, float* out, size_t out_len, size_t tq, size_t past,
                          size_t heads, size_t kv_heads, size_t head_dim, size_t cap, float scale, int causal);

/* No counterpart in the reference: the f16 prefills with a workspace, for
 * launches of few rows over many keys (a turn of a long conversation), whose
 * keys are then cut into runs attended by workgroups of their own and merged
 * in a second launch. llmtie_flash_attn_workspace gives the floats such a call
 * needs (0: the shape is not split, and no workspace is needed; never more than
 * 64 * 16 * (head_dim + 2) a compute unit, 136 MB at head_dim 128). The workspace
 * is written and read on `stream` by this call alone and may be reused or
 * freed in stream order after it; concurrent calls need one each. Split, the
 * context is the plain call's to rounding. `ws` NULL is the plain call. A
 * workspace shorter than needed is refused as LLMTIE_SLICE_OVERRUN, one that is
 * not 16-byte aligned as LLMTIE_INVALID_ARGUMENT. */
size_t llmtie_flash_attn_workspace(size_t tq, size_t past, size_t heads, size_t kv_heads, size_t head_dim);
int llmtie_flash_attn_f16_ws(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                             const uint16_t* v, size_t v_len, float* out, size_t out_len, size_t tq, size_t past,
                             size_t heads, size_t kv_heads, size_t head_dim, size_t cap, float scale, int causal,
                             float* ws, size_t ws_len);
int llmtie_flash_attn_t16_ws(void* stream, const float* q, size_t q_len, const uint16_t* cache, size_t cache_len,
                             float* out, size_t out_len, size_t tq, size_t past, size_t heads, size_t kv_heads,
                             size_t head_dim, size_t cap, float scale, int causal, float* ws, size_t ws_len);

/* Gpu::flash_attn_rows (device.rs:5812): non-causal attention over a stacked
 * [t, 3*heads*head_dim] q/k/v product, scale on q, context as f16 bits
 * [t, heads*head_dim]. head_dim 64. The rows are read where they lie and
 * rounded to f16 inside the kernel; nothing is allocated. */
int llmtie_flash_attn_rows(void* stream, const float* qkv, size_t qkv_len, uint16_t* out, size_t out_len,
                           size_t t, size_t heads, size_t head_dim, float scale);

/* ----------------------------------------------------------------- decode */

/* Gpu::attn_decode_f16 (device.rs:5949): one query row [heads*head_dim] over
 * tk live positions of an f16 cache; scale on q (scale_q) or on the scores.
 * Every decode entry accepts head_dim 64 and 128 and GQA groups up to 16: a
 * superset of the reference's refusals (it refuses groups over 4, 8 for its
 * head_dim-64 g8 kernel, device.rs:6245-6251, and an f32 cache at head_dim
 * 128, device.rs:6146). A binding that relies on those refusals to choose a
 * fallback refuses such shapes itself. */
int llmtie_attn_decode_f16(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                           const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads, size_t head_dim,
                           size_t tk, size_t cap, float scale, int scale_q, llmtie_decode_scratch* scratch,
                           float* out, size_t out_len);

/* No counterpart in the reference: llmtie_attn_decode_f16 for callers that
 * cannot allocate (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). Same arguments and result bits, no
 * scratch argument: the split partials and arrival counters live in a fixed
 * 4.25 MiB device array the library holds on each device (1M partial floats,
 * 256 kv heads' counters); a call that needs more is refused with
 * LLMTIE_SCRATCH_LIMIT before any launch. It calls no allocator. Every call
 * on one device shares that array, so calls that can overlap on one GPU (two
 * streams, two threads) race and must not be made. */
int llmtie_attn_decode_f16_noalloc(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                                   const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads, size_t head_dim,
                                   size_t tk, size_t cap, float scale, int scale_q, float* out, size_t out_len);

/* Gpu::attn_decode_f16_q (device.rs:5973): plus the context's int8 twin
 * (twin_len >= n + 4*(n/32) bytes, n = heads*head_dim). */
int llmtie_attn_decode_f16_q(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                             const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads, size_t head_dim,
                             size_t tk, size_t cap, float scale, int scale_q, llmtie_decode_scratch* scratch,
                             float* out, size_t out_len, int8_t* twin, size_t twin_len);

/* Gpu::attn_decode_f16_q_row (device.rs:6001): query from element q_off of q;
 * context into row `row` of out [rows, n] and of the twin [twin_rows, twin_k]. */
int llmtie_attn_decode_f16_q_row(void* stream, const float* q, size_t q_len, size_t q_off, const uint16_t* k,
                                 size_t k_len, const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads,
                                 size_t head_dim, size_t tk, size_t cap, float scale, int scale_q,
                                 llmtie_decode_scratch* scratch, float* out, size_t out_len, int8_t* twin,
                                 size_t twin_rows, size_t twin_k, size_t row);

/* Gpu::attn_decode (device.rs:6132): the same off an f32 cache (head_dim 128
 * accepted as well as the reference's 64). */
int llmtie_attn_decode(void* stream, const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                       size_t v_len, size_t heads, size_t kv_heads, size_t head_dim, size_t tk, size_t cap,
                       float scale, int scale_q, llmtie_decode_scratch* scratch, float* out, size_t out_len);

/* Batched decode over a tiled GGUF Q8_0 cache (new; the reference's nearest
 * caller is Translator::step_rows, crates/llmtie-translate/src/model.rs:764,
 * which launches one f16 decode per row). nseq sequences in one launch:
 * sequence s attends its tk_dev[s] live positions of cache slot slot_dev[s];
 * q and out are [nseq, heads*head_dim]. tk_dev and slot_dev are device int32
 * arrays; max_tk bounds every tk_dev[s] (the kernel clamps to it, never
 * reading past it) and must be <= cap. A sequence whose slot is out of range
 * or whose length is 0 gets a NaN row. cache_len is in bytes
 * (llmtie_q8_cache_bytes). Up to 64 sequences max_tk also decides how the keys
 * are divided over the chip: results under two bounds agree to rounding. */
int llmtie_attn_decode_q8_batch(void* stream, const float* q, size_t q_len, const int8_t* cache, size_t cache_len,
                                size_t slots, const int32_t* tk_dev, const int32_t* slot_dev, size_t nseq,
                                size_t max_tk, size_t heads, size_t kv_heads, size_t head_dim, size_t cap,
                                float scale, int scale_q, llmtie_decode_scratch* scratch, float* out,
                                size_t out_len);

/* ------------------------------------------- tiled f16 cache (new layout)
 *
 * One buffer per layer holds K and V in fragment order, 32 positions a block
 * (see ttsxabe_amd/csrc/kvlayout.h): every load the decode and prefill kernels
 * make of it is a contiguous 1 KB wave-wide read. These mirror the reference
 * operators they are named after, with the two cache slices replaced by the
 * one tiled buffer; cap may be any positive count (rounded up to whole blocks
 * internally). */

/* Halves a tiled f16 cache of this shape holds. */
size_t llmtie_t16_cache_len(size_t kv_heads, size_t head_dim, size_t cap);

/* cache_append_f16 (device.rs:2849) into the tiled cache; value selects V. */
int llmtie_t16_append(void* stream, const float* src, size_t src_len, size_t src_off, uint16_t* cache,
                      size_t cache_len, size_t n, size_t kv_heads, size_t head_dim, size_t cap, size_t past,
                      int value);

/* rope_cache_f16 (device.rs:2915) into the tiled cache. */
int llmtie_t16_rope_cache(void* stream, float* q, size_t q_len, size_t q_off, const float* k, size_t k_len,
                          size_t k_off, const float* v, size_t v_len, size_t v_off, const float* freq_div,
                          size_t heads, size_t kv_heads, size_t head_dim, float theta, size_t pos, uint16_t* cache,
                          size_t cache_len, size_t cap);

/* cache_grow_f16 (device.rs:3152) for the tiled cache. */
int llmtie_t16_grow(void* stream, const uint16_t* src, size_t src_len, uint16_t* dst, size_t dst_len,
                    size_t kv_heads, size_t head_dim, size_t cap, size_t new_cap, size_t live);

/* Repack reference-layout f16 caches (positions 0..live-1) into a tiled one. */
int llmtie_t16_from_ref(void* stream, const uint16_t* k, size_t k_len, const uint16_t* v, size_t v_len,
                        size_t kv_heads, size_t head_dim, size_t cap, size_t live, uint16_t* cache,
                        size_t cache_len);

/* attn_decode_f16 (device.rs:5949) off the tiled cache. */
int llmtie_attn_decode_t16(void* stream, const float* q, size_t q_len, const uint16_t* cache, size_t cache_len,
                           size_t heads, size_t kv_heads, size_t head_dim, size_t tk, size_t cap, float scale,
                           int scale_q, llmtie_decode_scratch* scratch, float* out, size_t out_len);

/* attn_decode_f16_q_row (device.rs:6001) off the tiled cache; twin may be NULL. */
int llmtie_attn_decode_t16_q_row(void* stream, const float* q, size_t q_len, size_t q_off, const uint16_t* cache,
                                 size_t cache_len, size_t heads, size_t kv_heads, size_t head_dim, size_t tk,
                                 size_t cap, float scale, int scale_q, llmtie_decode_scratch* scratch, float* out,
                                 size_t out_len, int8_t* twin, size_t twin_rows, size_t twin_k, size_t row);

/* flash_attn_f16 (device.rs:5754) off the tiled cache. */
int llmtie_flash_attn_t16(void* stream, const float* q, size_t q_len, const uint16_t* cache, size_t cache_len,
                          float* out, size_t out_len, size_t tq, size_t past, size_t heads, size_t kv_heads,
                          size_t head_dim, size_t cap, float scale, int causal);

/* --------------------------------------------------------- KV producers */

/* Gpu::rope / rope_scaled (device.rs:5410, :5430; kernel kernels.rs:4915): in place over x[off ..] of
 * [t, heads*head_dim]; freq_div (head_dim/2 floats, device) may be NULL. */
int llmtie_rope(void* stream, float* x, size_t x_len, size_t off, const float* freq_div, size_t t, size_t heads,
                size_t head_dim, float theta, size_t first);

/* Gpu::cache_append / cache_append_f16 (device.rs:3013 / :2849): n rows of
 * src[src_off ..] ([n, kv_heads*head_dim]) into positions past.. of a cache;
 * transposed selects the V layout. */
int llmtie_cache_append(void* stream, const float* src, size_t src_len, size_t src_off, float* dst, size_t dst_len,
                        size_t n, size_t kv_heads, size_t head_dim, size_t cap, size_t past, int transposed);
int llmtie_cache_append_f16(void* stream, const float* src, size_t src_len, size_t src_off, uint16_t* dst,
                            size_t dst_len, size_t n, size_t kv_heads, size_t head_dim, size_t cap, size_t past,
                            int transposed);

/* Gpu::rope_cache_f16 (device.rs:2915): q rotated in place, k rotated and v
 * stored into the f16 caches at `pos`. */
int llmtie_rope_cache_f16(void* stream, float* q, size_t q_len, size_t q_off, const float* k, size_t k_len,
                          size_t k_off, const float* v, size_t v_len, size_t v_off, const float* freq_div,
                          size_t heads, size_t kv_heads, size_t head_dim, float theta, size_t pos, uint16_t* kc,
                          uint16_t* vc, size_t cache_len, size_t cap);

/* Gpu::cache_grow / cache_grow_f16 (device.rs:3086, :3152): re-stride the first
 * `live` positions of every head from capacity cap to new_cap. */
int llmtie_cache_grow(void* stream, const float* src, size_t src_len, float* dst, size_t dst_len, size_t kv_heads,
                      size_t head_dim, size_t cap, size_t new_cap, size_t live, int transposed);
int llmtie_cache_grow_f16(void* stream, const uint16_t* src, size_t src_len, uint16_t* dst, size_t dst_len,
                          size_t kv_heads, size_t head_dim, size_t cap, size_t new_cap, size_t live,
                          int transposed);

/* Bytes a tiled Q8_0 cache of this shape holds (layout at the top). */
size_t llmtie_q8_cache_bytes(size_t slots, size_t kv_heads, size_t head_dim, size_t cap);

/* Q8_0 cache append (new): n rows of k[k_off..] and v[v_off..] ([n,
 * kv_heads*head_dim], k already rotated) quantized into slot `slot` at
 * positions past.. . Quantization is ggml's quantize_row_q8_0_ref. */
int llmtie_kv_q8_append(void* stream, const float* k, size_t k_len, size_t k_off, const float* v, size_t v_len,
                        size_t v_off, int8_t* cache, size_t cache_len, size_t slots, size_t slot, size_t n,
                        size_t kv_heads, size_t head_dim, size_t cap, size_t past);

/* The Q8_0 twin of llmtie_rope_cache_f16 (new): q rotated in place, k rotated
 * and quantized, v quantized, into slot `slot` at `pos`. */
int llmtie_rope_cache_q8(void* stream, float* q, size_t q_len, size_t q_off, const float* k, size_t k_len,
                         size_t k_off, const float* v, size_t v_len, size_t v_off, const float* freq_div,
                         size_t heads, size_t kv_heads, size_t head_dim, float theta, size_t pos, int8_t* cache,
                         size_t cache_len, size_t slots, size_t slot, size_t cap);

/* ------------------------------------------- attention over key ranges (new)
 *
 * No counterpart in the reference. Prompts and batched single tokens over a
 * tiled f16 cache of `slots` sequences ([slots][kv_heads][blocks of 32
 * positions]: llmtie_t16_cache_len halves each, one after the other), in which
 * every query row sees keys of its own, with
 *
 *   score of key j = c * tanh(scale * q.k_j / c) - slope[head] * |i - j|
 *
 * where softcap c = 0 stands for no cap, slopes NULL (else [heads] f32, device)
 * for no bias, and i and j are cache positions: a row's own and the key's. The
 * scale is 1e-15 to 1e15, the cap 0 or 0.001 to 1000, a slope 0 to 1e15. A row that sees no
 * key gets zeros. Keys that a row does not see contribute nothing to it, whatever they hold. */

/* Which keys the rows of a packed prompt see: made once for all layers. Row r
 * (of `rows`) is at cache position i = past + r. starts (device, starts_len =
 * documents + 1, never decreasing) holds each document's first row and the row
 * behind the last; row r of document d, which covers positions s = past +
 * starts[d] up to e = past + starts[d + 1] (at most past + rows), sees
 *   j < table[r]                                      and
 *   table[rows + r] <= j < table[2 * rows + r]:
 *   table[r]            = min(shared, causal ? i + 1 : past + rows): leading positions that every row
 *                         sees (a shared prompt, what a sliding window leaves behind)
 *   table[rows + r]     = s, or i - window + 1 where a window is given (nonzero) and that is more
 *   table[2 * rows + r] = causal ? i + 1 : e (at most i + window), and at least min(s + prefix[d], e) where
 *                         prefix is given (device, one a document): rows that their document's all see.
 * starts NULL is one document from cache position 0 (s = 0, e = past + rows;
 * prefix then has one entry). Rows of no document see nothing (zeros). pos, if not NULL, gets the
 * rows' rotary positions i - s. Attention clamps the ranges to the keys the cache holds. */
int llmtie_key_ranges(void* stream, const int32_t* starts, size_t starts_len, const int32_t* prefix, size_t prefix_len,
                      size_t rows, size_t past, int causal, size_t window, size_t shared, int32_t* table,
                      size_t table_len, int32_t* pos, size_t pos_len);

/* Attention of tq query rows (f16, row r at q[q_off + r * q_stride ..], as
 * llmtie_rope_rows and llmtie_t16_rope_store leave them) over slot `slot`, which
 * holds past + tq keys; table as above, of exactly these rows. out = [tq,
 * heads*head_dim] f16. max_keys bounds the keys a row sees and is used for the
 * plan alone (0: past + tq). ws: a workspace of
 * llmtie_flash_attn_ranges_workspace floats, 16-byte aligned, for launches of
 * few rows over many keys, which are then cut into runs of keys and merged by a
 * second launch (0 floats, or NULL: not cut). Its size is asked for with the
 * call's own max_keys, past + tq in place of 0. It is written and read on
 * `stream` by this call alone; concurrent calls need one each. cache and out
 * are 16-byte aligned. */
size_t llmtie_flash_attn_ranges_workspace(size_t tq, size_t max_keys, size_t heads, size_t kv_heads, size_t head_dim);
int llmtie_flash_attn_ranges_t16(void* stream, const uint16_t* q, size_t q_len, size_t q_off, size_t q_stride,
                                 const uint16_t* cache, size_t cache_len, size_t slots, size_t slot,
                                 const int32_t* table, size_t table_len, size_t max_keys, uint16_t* out,
                                 size_t out_len, size_t tq, size_t past, size_t heads, size_t kv_heads,
                                 size_t head_dim, size_t cap, float scale, float softcap, const float* slopes,
                                 size_t slopes_len, float* ws, size_t ws_len);

/* One token of each of nseq sequences: sequence s attends with row q[q_off + s *
 * q_stride ..] (f32, magnitudes up to 65504: it is read as the sum of two f16) the
 * first tk_dev[s] positions of slot slot_dev[s] (slot_dev NULL: slot s), of
 * those the first `shared` ones and the ones from max(lo_dev[s], tk_dev[s] -
 * window) on (lo_dev NULL: 0; window 0: none). Its own position is tk_dev[s] -
 * 1. The three arrays are on the device and may change between replays of a
 * captured call. Lengths are clamped to cap; max_tk plans the launch for the
 * lengths to come (longer ones are attended too, less evenly spread) and decides
 * with it how keys are divided: results under two bounds agree to rounding. (An
 * eager call of the most sequences and the largest max_tk sizes the scratch for
 * every smaller one that is captured.) A
 * sequence whose slot is out of range gets a NaN row, one that sees no key
 * zeros. GQA groups up to 16. out = [nseq, heads*head_dim] f32, 16-byte aligned
 * as the cache is. */
int llmtie_attn_decode_ranges_t16(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride,
                                  const uint16_t* cache, size_t cache_len, size_t slots, const int32_t* tk_dev,
                                  const int32_t* slot_dev, const int32_t* lo_dev, size_t nseq, size_t max_tk,
                                  size_t window, size_t shared, size_t heads, size_t kv_heads, size_t head_dim,
                                  size_t cap, float scale, float softcap, const float* slopes, size_t slopes_len,
                                  llmtie_decode_scratch* scratch, float* out, size_t out_len);

/* --------------------------------------- rotary positions by row (new)
 *
 * Row r at position pos[r] (device int32), the first rot_dim dims of each head
 * (even, 0 to head_dim; the others are copied) rotated in pairs of halves (d, d
 * + rot_dim / 2) or, `interleaved`, (2d, 2d + 1), by the angle pos * theta^(-2d /
 * rot_dim) / freq_div[d] (freq_div NULL: 1; rot_dim / 2 floats, device), the
 * rotated values times mscale. Angles are formed in f64 (llmtie_rope's are the
 * reference's f32 ones). At most 2^26 rows a call, of fewer than 2^29 values each. */

/* t rows of `heads` heads from x[off + r * stride ..] into out[out_off + r *
 * out_stride ..], f32 or (out_f16) f16. out may be x itself (the same rows, f32)
 * or apart from them. pos NULL: positions first + r. head_dim even, at most 1024. */
int llmtie_rope_rows(void* stream, const float* x, size_t x_len, size_t off, size_t stride, void* out, size_t out_len,
                     size_t out_off, size_t out_stride, int out_f16, const int32_t* pos, size_t pos_len, size_t first,
                     const float* freq_div, size_t div_len, size_t t, size_t heads, size_t head_dim, size_t rot_dim,
                     float theta, float mscale, int interleaved);

/* q rotated into q_out (as llmtie_rope_rows; q NULL: none), k rotated and v
 * stored as f16 at position index[r] of slot slot[r] of a tiled f16 cache of
 * `slots` slots: the tokens of a batch of sequences, or a prompt's rows, in one
 * launch. pos, slot and index are device arrays of index_len >= rows entries. A
 * row whose slot or index is out of range stores nothing (its q is rotated);
 * no two rows of a call may name the same place. The projections may be one
 * stacked buffer: q rotated in place then lies beside k and v at the one stride of all
 * three, and another q_out lies apart from them. */
int llmtie_t16_rope_store(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride, void* q_out,
                          size_t q_out_len, size_t q_out_off, size_t q_out_stride, int q_out_f16, const float* k,
                          size_t k_len, size_t k_off, size_t k_stride, const float* v, size_t v_len, size_t v_off,
                          size_t v_stride, const int32_t* pos, const int32_t* slot, const int32_t* index,
                          size_t index_len, const float* freq_div, size_t div_len, size_t rows, size_t heads,
                          size_t kv_heads, size_t head_dim, size_t rot_dim, float theta, float mscale,
                          int interleaved, uint16_t* cache, size_t cache_len, size_t slots, size_t cap);

/* ------------------------------------------------ a cache in pages (new)
 *
 * No counterpart in the reference. The tiled f16 cache with its slots taken as
 * pages of `page` positions (a power of two from 32 to 4096; llmtie_t16_cache_len(..,
 * page) halves each): a sequence lies where row t of a table says, table[t *
 * table_cols + p] being the page of its positions p * page .. (device int32, of
 * table_rows rows; entries behind a sequence's last page are not read). At most
 * 2^30 positions a sequence. Query rows are a token of each sequence, or rows of
 * prompts: row r is at position tk_dev[r] - 1 of table row row_dev[r] (row_dev NULL:
 * row r) and sees some of the tk_dev[r] first positions. A row that sees no key gets
 * zeros; one whose table row does not exist, or that needs a page the cache does not
 * have, NaN. Keys that a row does not see contribute nothing, whatever they hold;
 * a value that it does see and that is not finite leaves that element of its context
 * not finite (an infinity or NaN), whatever its weight. Lengths, tables and rows
 * may change between replays of captured calls. Scores are those of the key ranges
 * above, with the same bounds of their arguments. */

/* llmtie_t16_rope_store into pages: row r to position index[r] of table row
 * seq[r]. Rows whose table row, position or page does not exist store nothing; no two
 * rows of a call may name the same place, nor one by two sequences that share a page. */
int llmtie_paged_rope_store(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride, void* q_out,
                            size_t q_out_len, size_t q_out_off, size_t q_out_stride, int q_out_f16, const float* k,
                            size_t k_len, size_t k_off, size_t k_stride, const float* v, size_t v_len, size_t v_off,
                            size_t v_stride, const int32_t* pos, const int32_t* seq, const int32_t* index,
                            size_t index_len, const int32_t* table, size_t table_len, size_t table_rows,
                            size_t table_cols, const float* freq_div, size_t div_len, size_t rows, size_t heads,
                            size_t kv_heads, size_t head_dim, size_t rot_dim, float theta, float mscale,
                            int interleaved, uint16_t* cache, size_t cache_len, size_t pages, size_t page);

/* The plan of a step's attention, made once for all its layers (plan: device
 * int32, llmtie_page_plan_len of them, written on `stream`; read by the calls it
 * is for). Row r of nseq sees of its first tk_dev[r] positions the first `shared`
 * ones and those from max(lo_dev[r], tk_dev[r] - window) on (lo_dev NULL: 0; window
 * 0: none). Rows starts[g] up to starts[g + 1] (device, groups + 1 entries, never
 * decreasing; groups 0: none) promise that their tables' rows name the same pages
 * for positions below prefix[g]: what all of them see of these is then read and
 * attended once for up to 32 / (heads / kv_heads) rows together. A prefix counts in
 * whole blocks of 32 positions and no further than the shortest row's length. max_tk is the
 * longest length or near it (it says which launch is made; longer rows are attended too).
 * Rows of one sequence that follow one another in row_dev, as a prompt's do, are attended together,
 * their keys read once, where nseq > table_rows; in a table of as many rows or more each
 * reads its own, and only prefixes are shared. GQA groups up to 16, at most 1024 groups and 2^20 rows. */
size_t llmtie_page_plan_len(size_t nseq, size_t groups, size_t max_tk, size_t table_rows, size_t heads,
                            size_t kv_heads);
int llmtie_page_plan(void* stream, const int32_t* tk_dev, const int32_t* row_dev, const int32_t* lo_dev, size_t nseq,
                     const int32_t* starts, const int32_t* prefix, size_t groups, size_t max_tk, size_t window,
                     size_t shared, size_t table_rows, size_t table_cols, size_t page, size_t heads, size_t kv_heads,
                     size_t head_dim, int32_t* plan, size_t plan_len);

/* Attention of nseq query rows (f32, row r at q[q_off + r * q_stride ..], magnitudes
 * up to 65504) over what the plan says; plan, tk_dev and the sizes are those that
 * it was made with (rows are NaN under a plan of other sizes). ws: a workspace of
 * llmtie_attn_paged_workspace floats, 16-byte aligned, written and read on `stream` by this
 * call alone. out = [nseq, heads*head_dim] f32, 16-byte aligned as the cache is. */
size_t llmtie_attn_paged_workspace(size_t nseq, size_t groups, size_t max_tk, size_t table_rows, size_t heads,
                                   size_t kv_heads, size_t head_dim);
int llmtie_attn_decode_paged(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride,
                             const uint16_t* cache, size_t cache_len, size_t pages, size_t page, const int32_t* table,
                             size_t table_len, size_t table_rows, size_t table_cols, const int32_t* tk_dev,
                             const int32_t* plan, size_t plan_len, size_t nseq, size_t groups, size_t max_tk,
                             size_t heads, size_t kv_heads, size_t head_dim, float scale, float softcap,
                             const float* slopes, size_t slopes_len, float* ws, size_t ws_len, float* out,
                             size_t out_len);

/* The same over `count` pages of each (row, kv head): chosen[(r * kv_heads + h) *
 * count ..] are numbers of pages within the sequence (device int32, as
 * llmtie_select_pages leaves them, in any order; none may be there twice, it would count
 * once or twice; ones below 0 or with no position that the row has name nothing). Row r
 * sees those of their positions that are below tk_dev[r]. Rows of one sequence that follow one another, as a prompt's do,
 * are attended together, each page read once for those that selected it, where there are more
 * rows than the table has. */
size_t llmtie_attn_selected_workspace(size_t nseq, size_t count, size_t page, size_t table_rows, size_t heads,
                                      size_t kv_heads, size_t head_dim);
int llmtie_attn_decode_selected(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride,
                                const uint16_t* cache, size_t cache_len, size_t pages, size_t page,
                                const int32_t* table, size_t table_len, size_t table_rows, size_t table_cols,
                                const int32_t* tk_dev, const int32_t* row_dev, const int32_t* chosen, size_t chosen_len,
                                size_t count, size_t nseq, size_t heads, size_t kv_heads, size_t head_dim, float scale,
                                float softcap, const float* slopes, size_t slopes_len, float* ws, size_t ws_len,
                                float* out, size_t out_len);

/* The greatest and the least key of pages, dim by dim: bounds[((page * kv_heads +
 * h) * 2 + 0) * head_dim ..] and [.. + 1 ..] (f16; NaN where a key is) over the positions below tk_dev[r] of
 * every page of row r's sequence that holds one from low_dev[r] (NULL: 0) up to
 * tk_dev[r]. Pages without one, and those the cache does not have, are left as they
 * are. max_new is how many positions that is at most, or near it. No two rows of a
 * call may give one page different lengths. cache and bounds are 16-byte aligned. */
int llmtie_page_bounds(void* stream, const uint16_t* cache, size_t cache_len, size_t pages, size_t page,
                       const int32_t* table, size_t table_len, size_t table_rows, size_t table_cols,
                       const int32_t* row_dev, const int32_t* low_dev, const int32_t* tk_dev, size_t nseq,
                       size_t max_new, size_t kv_heads, size_t head_dim, uint16_t* bounds, size_t bounds_len);

/* The `count` pages of its sequence that each (row, kv head) attends: the first
 * `first` and the last `last` ones, and of the others those with the largest
 *   max over the heads of the kv head of  sum_d max(q_d, 0) greatest_d + min(q_d, 0) least_d,
 * which no product of those heads with a key of the page exceeds; formed in f64, a NaN
 * as +inf (and a page that the cache does not have), ties to the lowest number.
 * chosen [nseq, kv_heads, count] in rising order, -1 behind the last where the
 * sequence has fewer. Lengths are clamped to the pages of max_tk. ws:
 * llmtie_select_pages_workspace doubles, 16-byte aligned, as the attention's. */
size_t llmtie_select_pages_workspace(size_t nseq, size_t max_tk, size_t page, size_t count, size_t kv_heads);
int llmtie_select_pages(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride,
                        const uint16_t* bounds, size_t bounds_len, size_t pages, size_t page, const int32_t* table,
                        size_t table_len, size_t table_rows, size_t table_cols, const int32_t* tk_dev,
                        const int32_t* row_dev, size_t nseq, size_t max_tk, size_t heads, size_t kv_heads,
                        size_t head_dim, size_t count, size_t first, size_t last, double* ws, size_t ws_len,
                        int32_t* chosen, size_t chosen_len);

#ifdef __cplusplus
}
#endif

#endif /* LLMTIE_HIP_H */
