// The C ABI (include/llmtie_hip.h): argument checks in the reference's order
// and with its error variants, then one launch. Mirrors the `impl Gpu`
// attention methods of crates/llmtie-cuda/src/device.rs:5697-6410 and the
// cache producers at :2849-3190, :5410-5470.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <atomic>
#include <mutex>
#include <vector>

#include "../../include/llmtie_hip.h"
#include "decode.h"
#include "kvlayout.h"
#include "kvcache.h"
#include "prefill.h"
#include "ranges.h"
#include "rotary.h"

using namespace llmtie;

namespace {

thread_local llmtie_error g_err = {0, {0, 0, 0, 0}, {0}};
// llmtie_debug_fake_xcc: the test hook for the XCD-local check.
std::atomic<bool> g_fake_xcc{false};

int fail(int status, size_t f0, size_t f1, size_t f2, size_t f3, const char* fmt, ...) {
    g_err.status = status;
    g_err.field[0] = f0;
    g_err.field[1] = f1;
    g_err.field[2] = f2;
    g_err.field[3] = f3;
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err.message, sizeof g_err.message, fmt, ap);
    va_end(ap);
    return status;
}

int ok() {
    g_err.status = LLMTIE_OK;
    g_err.message[0] = 0;
    return LLMTIE_OK;
}

int unsupported(size_t hd, size_t heads, size_t kv) {
    return fail(LLMTIE_UNSUPPORTED_ATTENTION, hd, heads, kv, 0,
                "fused attention wants head_dim 64 or 128 and heads a multiple of kv_heads, got head_dim %zu, "
                "%zu heads over %zu",
                hd, heads, kv);
}
int overrun_slice(size_t at, size_t len) {
    return fail(LLMTIE_SLICE_OVERRUN, at, len, 0, 0, "reading to %zu in a buffer of %zu", at, len);
}
int overrun_cache(size_t at, size_t cap) {
    return fail(LLMTIE_CACHE_OVERRUN, at, cap, 0, 0, "appending at %zu to a cache with room for %zu", at, cap);
}
int odd_cap(size_t cap) {
    return fail(LLMTIE_ODD_CACHE_CAPACITY, cap, 0, 0, 0, "an f16 cache with an odd capacity of %zu", cap);
}
int invalid(const char* what) { return fail(LLMTIE_INVALID_ARGUMENT, 0, 0, 0, 0, "%s is null", what); }
int driver(const char* what, hipError_t e) {
    if (e == hipErrorNoDevice || e == hipErrorInsufficientDriver)
        return fail(LLMTIE_NO_DEVICE, 0, 0, 0, 0, "no usable HIP device: %s", hipGetErrorString(e));
    return fail(LLMTIE_DRIVER, (size_t)e, 0, 0, 0, "%s: %s", what, hipGetErrorString(e));
}
int launched(const char* what, hipError_t e) { return e == hipSuccess ? ok() : driver(what, e); }

hipStream_t S(void* s) { return reinterpret_cast<hipStream_t>(s); }

// Every kernel takes int extents; anything that does not fit is refused as
// an overrun of the int range rather than silently wrapped.
constexpr size_t IMAX = 0x7fffffff;

// Sizes computed from caller arguments saturate at SIZE_MAX instead of
// wrapping, so a length check on a sum or product never passes on overflow.
size_t smul(size_t a, size_t b) {
    size_t r;
    return __builtin_mul_overflow(a, b, &r) ? SIZE_MAX : r;
}
size_t smul(size_t a, size_t b, size_t c) { return smul(smul(a, b), c); }
size_t sadd(size_t a, size_t b) {
    size_t r;
    return __builtin_add_overflow(a, b, &r) ? SIZE_MAX : r;
}
// The first of up to four counts that does not fit an int, refused as an
// overrun of the int range (0 when all fit).
int over_int(size_t a, size_t b = 0, size_t c = 0, size_t d = 0) {
    const size_t m = std::max(std::max(a, b), std::max(c, d));
    return m > IMAX ? overrun_slice(m, IMAX) : 0;
}

}  // namespace

struct llmtie_decode_scratch {
    float* part = nullptr;
    size_t part_cap = 0;  // floats
    unsigned* ctr = nullptr;
    size_t ctr_cap = 0;   // counters
    int device = -1;
    // Buffers replaced by growth. A HIP graph captured with the scratch keeps
    // their addresses, so they stay allocated until the scratch is freed.
    std::vector<void*> retired;
    // Host-visible word (pinned host memory) the decode kernel sets when an
    // XCD-local head's split workgroups turn out not to share an XCD.
    unsigned* lost = nullptr;
};

extern "C" {

int llmtie_last_error(llmtie_error* out) {
    if (out) *out = g_err;
    return g_err.status;
}

const char* llmtie_version(void) { return "0.1.0"; }

llmtie_decode_scratch* llmtie_decode_scratch_new(void) { return new llmtie_decode_scratch(); }

void llmtie_decode_scratch_free(llmtie_decode_scratch* s) {
    if (!s) return;
    if (s->part) (void)hipFree(s->part);
    if (s->ctr) (void)hipFree(s->ctr);
    for (void* p : s->retired) (void)hipFree(p);
    if (s->lost) (void)hipHostFree(s->lost);
    delete s;
}

int llmtie_decode_scratch_status(llmtie_decode_scratch* s) {
    if (!s || !s->lost || !__atomic_load_n(s->lost, __ATOMIC_ACQUIRE)) return LLMTIE_OK;
    __atomic_store_n(s->lost, 0u, __ATOMIC_RELEASE);
    return fail(LLMTIE_SPLIT_HEAD_LOST, 0, 0, 0, 0,
                "an earlier decode through this scratch wrote NaN for a head whose split workgroups did not "
                "share an XCD; LLMTIE_DECODE_XCD=0 selects the coherent hand-off");
}

void llmtie_debug_fake_xcc(int on) { g_fake_xcc.store(on != 0); }

int llmtie_supports_flash(size_t head_dim, size_t heads, size_t kv_heads) {
    return (head_dim == 64 || head_dim == 128) && kv_heads > 0 && heads % kv_heads == 0 && heads > 0;
}

}  // extern "C"

namespace {

int compute_units();

// 16-query tiles per wave: the most that still leaves about two workgroups
// per CU (256 CUs), so short prefills spread over the whole chip.
int pick_nqt(size_t tq, size_t heads, int gb, bool staged = false) {
    if (const char* e = getenv("LLMTIE_PREFILL_NQT")) {
        const int v = atoi(e);
        if (v == 1 || v == 2 || v == 4) return v;
    }
    // Measured on MI355X (C3 shapes, 512 to 8192 rows): two 16-row query
    // tiles per wave (each K/V fragment read from LDS feeds two MFMAs) win
    // once the launch still has >= 512 workgroups; below that, one tile per
    // wave, for the parallelism.
    const size_t pb2 = 32 * (4 / gb);
    const size_t wg2 = ((tq + pb2 - 1) / pb2) * (heads / gb);
    if (wg2 >= 512) return 2;
    // f32 sources staged through registers: two tiles per wave halve the
    // staging per query row, which wins down to about one workgroup per CU
    // (the encoder rows at 240 workgroups: 38.7 vs 40.1 us, before their
    // eight-wave kernel).
    if (staged && wg2 >= 192) return 2;
    return 1;
}

// Runs the tiles of each position block of a prefill off an f16 cache are cut
// into (1: not split), one workgroup each: the cheapest under a model of the
// launch in microseconds, fitted on MI355X to 2700 causal shapes of nine head
// counts of 64 and 128, half of them timed at up to eleven run counts. A
// workgroup's 64-key tile takes 0.86 on an empty chip and 0.24 more for each
// workgroup a compute unit holds, up to two; further ones wait. Counts that do
// not deal whole eighths to the XCDs' L2s cost 13 % a tile; a whole launch of
// head_dim 64 that fills half the units saves 10 %.
// Splitting adds the merge's launch and the partials' traffic, so few rows over
// many keys split far and many rows or few keys not at all. Four of those
// shapes are slower than whole by more than 1 %, the worst 6.2 % (17 rows after
// 513 of 40/40/128, 13.55 / 12.76); of 500 others two, 1.8 %, the mean 0.47 of
// the whole one's time. Measured, split / not: 173 rows after
// 3011 positions of 32/8/128, 28-31 / 45-47 us; 16 after 3000, 14.6 / 44; 100
// after 7000, 28 / 95; 40 after 1000, 13.1 / 19.5; at head_dim 64, 173 after
// 3011, 19.4 / 40.7; 40 after 1000, 10.9 / 18; 16 after 3000, 12.2 / 39.4. Where
// it keeps one run, two or three measured slower: 206 rows after 691, 19.4 /
// 16.9; 125 after 622, 16.0 / 14.3; 300 after 700, 24 / 20; 400 after 1500 of
// 40/40/128, 49 / 42; 2000 first rows of 8/2/128, 33-35 / 34.
// The partials are bounded by the workgroups: 64 (row, head)s each, at most 16 a
// compute unit, 136 MB at head_dim 128 on 256 units, which only turns past
// 30000 positions come near (526 rows after 129000 of 32/8/128, 22 runs 1344 us,
// whole 1887).
constexpr size_t PREFILL_MAX_SPLITS = 32, PREFILL_MAX_SPLIT_WGS = 16;  // the latter a compute unit
size_t plan_prefill_splits(size_t tq, size_t past, size_t heads, size_t kv_heads, size_t hd) {
    if (getenv("LLMTIE_PREFILL_NQT")) return 1;
    const size_t group = heads / kv_heads;
    const size_t gb = group % 4 == 0 ? 4 : (group % 2 == 0 ? 2 : 1);
    const size_t pb = 16 * (4 / gb);
    const double cus = compute_units();
    const double items = (double)((tq + pb - 1) / pb) * (double)(heads / gb);
    if (items > 2 * cus) return 1;
    const size_t tiles = (past + tq + 63) / 64;
    if (tiles <= 8) return 1;  // no shape measured gains; the Python binding does not ask either
    // One run's partials written and read, and its share of the merge's chain.
    const double run_us = (double)(tq * heads * hd) * 8.0 / 3.1e6 + 0.11;
    size_t best = 1;
    double least = 0.0, whole = 0.0;
    for (size_t n = 1; n <= PREFILL_MAX_SPLITS && n <= tiles; ++n) {
        const double load = items * (double)n / cus;
        if (n > 1 && load > (double)PREFILL_MAX_SPLIT_WGS) break;
        double period = load <= 2.0 ? 0.86 + 0.24 * load : 0.67 * std::ceil(load);
        if ((size_t)items * n % 8 != 0) period *= 1.13;
        if (n == 1 && hd == 64 && 2 * items > cus) period *= 0.9;
        const double merge_us = n == 1 ? 0.0 : (load <= 1.0 ? 3.4 : 5.4) + (double)n * run_us;
        const double us = (double)((tiles + n - 1) / n) * period + merge_us;
        if (n == 1) whole = least = us;
        if (us < least) {
            best = n;
            least = us;
        }
    }
    // Within 5 % of the whole one the two measured either way.
    return least < 0.95 * whole ? best : 1;
}

int prefill_common(void* stream, int kind, const float* q, size_t q_len, const void* k, size_t k_len, const void* v,
                   size_t v_len, float* out, size_t out_len, size_t tq, size_t past, size_t heads, size_t kv_heads,
                   size_t hd, size_t cap, float scale, int causal, float* ws = nullptr, size_t ws_len = 0) {
    if (!(hd == 64 || hd == 128) || kv_heads == 0 || heads % kv_heads != 0) return unsupported(hd, heads, kv_heads);
    if (sadd(past, tq) > cap) return overrun_cache(sadd(past, tq), cap);
    if (int r = over_int(smul(heads, hd), cap)) return r;
    const size_t nq = smul(tq, heads, hd);
    if (nq > (size_t)1 << 40) return overrun_slice(nq, (size_t)1 << 40);
    if (q_len < nq) return overrun_slice(nq, q_len);
    const size_t need = smul(kv_heads, cap, hd);
    if (k_len < need || v_len < need) return overrun_slice(need, std::min(k_len, v_len));
    if (out_len < nq) return overrun_slice(nq, out_len);
    if (tq == 0) return ok();
    if (!q || !k || !v || !out) return invalid("a buffer");
    const size_t group = heads / kv_heads;
    const int gb = group % 4 == 0 ? 4 : (group % 2 == 0 ? 2 : 1);
    PrefillArgs a{};
    a.cus = compute_units();
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.tq = (int)tq;
    a.past = (int)past;
    a.heads = (int)heads;
    a.kv_heads = (int)kv_heads;
    a.cap = (int)cap;
    a.scale = scale;
    a.causal = causal ? 1 : 0;
    a.gb = gb;
    a.qs = (int)(heads * hd);
    a.kvs = 0;
    a.os = (int)(heads * hd);
    a.scale_q = 0;
    a.v_bytes = v_len * (kind == PF_F32 ? 4 : 2);
    int nqt = pick_nqt(tq, heads, gb, kind == PF_F32);
    const size_t splits = ws ? plan_prefill_splits(tq, past, heads, kv_heads, hd) : 1;
    if (splits > 1) {
        const size_t need = smul(smul(splits, tq, heads), hd + 2);
        if (ws_len < need) return overrun_slice(need, ws_len);
        if (reinterpret_cast<uintptr_t>(ws) % 16 != 0)
            return fail(LLMTIE_INVALID_ARGUMENT, 0, 0, 0, 0, "a workspace off 16 bytes");
        a.splits = (int)splits;
        a.ws = ws;
        nqt = 1;
    }
    return launched("flash_attn", launch_prefill((int)hd, kind, nqt, a, S(stream)));
}

// Compute units of the current device (cached per device).
int compute_units() {
    static int cus[64] = {0};
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    if (!cus[dev]) {
        int n = 0;
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) n = 256;
        cus[dev] = n;
    }
    return cus[dev];
}

// Floats of the (m, l) area per (sequence, kv head): whole 256-byte lines,
// so no line is shared by two heads' partials.
size_t ml_stride(int splits, size_t group) { return ((size_t)splits * group * 2 + 63) / 64 * 64; }

// Sizes of the no-allocation decode's fixed scratch: split partials, then
// arrival counters (CTR_STRIDE words per kv head).
constexpr size_t NOALLOC_PART_FLOATS = (size_t)1 << 20;
constexpr size_t NOALLOC_CTR_WORDS = (size_t)256 * CTR_STRIDE;

// The longest context, in 32-key blocks, that a single-sequence decode keeps
// in one split, and the waves its workgroups have then. The cross-workgroup
// merge (three memory round trips, ~3 us) costs more than the parallelism
// saves on short contexts. Eight waves (from five blocks on) against four, and
// against splits, in us: 32/8/128 reference layout, 211 keys 8.0 / 8.35, 256
// keys 8.5 / 8.8; tiled, 300 keys 6.85 / 8.0 / 8.3, 384 keys 7.15 / 7.8 / 7.9,
// 420 keys 9.0 / - / 8.35; 20/20/64 f32, 224 keys 4.25 / 4.61, 448 keys 5.68 /
// - / 7.04; f16, 400 keys 6.59 / - / 7.20, 512 keys 7.07 / - / 7.34; 32/8/64,
// 384 keys 6.7 / 7.7, 500 keys 8.2 / - / 7.46.
// The reference layout at head_dim 128 splits from ten blocks on (its line
// requests set one compute unit's pace): 300 / 320 / 352 / 384 keys, three
// splits against one: 32/8, 9.36 9.31 9.35 9.18 / 9.88 9.80 10.2 10.5; 16/8,
// 9.23 9.20 9.20 9.24 / 9.70 9.63 10.2 10.8; 8/2, 8.96 8.72 8.78 8.57 / 9.50
// 8.89 9.39 9.97; 40/40, 8.68 8.68 8.69 8.70 / 8.61 8.39 8.68 9.11. The line
// lies by the shape alone, so that a call has one result whatever scratch it
// is given: not where three splits' partials pass the fixed scratch, and every
// growing scratch has room for them (ensure_scratch).
size_t one_split_blocks(int kind, size_t kv_heads, size_t group, size_t hd) {
    if (kind == KV_F16 && hd == 128 && kv_heads * (3 * group * hd + ml_stride(3, group)) <= NOALLOC_PART_FLOATS)
        return 9;
    return hd == 64 && group == 1 ? 16 : 12;
}
int one_split_waves(size_t tk, int kind, size_t group, size_t hd) {
    if (getenv("LLMTIE_DECODE_WGS") || getenv("LLMTIE_DECODE_NIT")) return 4;
    // An f32 cache's hi + lo fragments need four waves' registers (the MFMA
    // fold at head_dim 64 spilled 85 of them at eight).
    if (kind == KV_F32 && (hd != 64 || group != 1 || getenv("LLMTIE_DECODE_G1_MFMA"))) return 4;
    return tk > 128 ? 8 : 4;
}

// Splits of one head: about `target` workgroups over the whole launch, each
// wave taking whole 32-key blocks, and never more than the merge can hold; one
// split up to `one_split` blocks.
void plan_decode(size_t tk_max, size_t units, size_t group, int& nit, int& splits, size_t one_split = 12) {
    const size_t max_splits = std::min<size_t>(DECODE_MAX_SPLITS, DECODE_MAX_SPLIT_ROWS / std::max<size_t>(1, group));
    // Measured on MI355X: a lone sequence decodes fastest over ~256
    // workgroups (C2: 10.99 us at 128, 10.69 at 256, flat beyond; with the
    // arrival counters on separate lines the in-launch merge no longer grows
    // costlier with the split count); a batch wants about three splits per
    // (sequence, kv head) at its longest context so the long sequences do not
    // set the time alone.
    size_t target = std::max<size_t>(256, 3 * units);
    if (const char* e = getenv("LLMTIE_DECODE_WGS")) target = std::max(1, atoi(e));
    const size_t blocks = (tk_max + 31) / 32;
    size_t want = std::max<size_t>(1, target / std::max<size_t>(1, units));
    size_t per_wg = (blocks + want - 1) / want;           // 32-key blocks per workgroup
    size_t n = std::max<size_t>(1, (per_wg + 3) / 4);     // per wave
    if (const char* e = getenv("LLMTIE_DECODE_NIT")) n = std::max(1, atoi(e));
    if (blocks <= one_split && !getenv("LLMTIE_DECODE_WGS") && !getenv("LLMTIE_DECODE_NIT")) n = (blocks + 3) / 4;
    size_t span = 4 * n * 32;
    while ((tk_max + span - 1) / span > max_splits) {
        ++n;
        span = 4 * n * 32;
    }
    nit = (int)n;
    splits = (int)((tk_max + span - 1) / span);
}

// Whether a batched Q8_0 decode runs stream-K (one workgroup per compute unit,
// each wave an equal share of the batch's blocks) rather than on the
// host-planned grid (splits of the longest sequence), whose plan it may widen.
// Stream-K balances ragged lengths, but each wave holds a head's pieces, so a
// batch of few blocks pays for merging hundreds of them: the host only knows
// the lengths' bound, so the line is drawn at the bytes that it allows. Host
// plan / stream-K, us, at 8 kv heads of 128: 1 sequence of 4000, 8.6 / 42.6; 4 of
// 500-2000, 9.8 / 22.1; 8 of 256-4096 (bound 71 MB), 15.2 / 23.0; 8 of
// 6000-8000 (139 MB), 25.9 / 34.1; 32 of 100-1000 (70 MB), 12.4 / 16.7; 12 of
// 20-8000 (209 MB), 45 / 35; 16 of 500-4000 (139 MB), 28 / 23; 32 of 256-8192
// (570 MB), 68 / 54.6. More than 64 sequences always take the plan.
bool plan_q8_batch(size_t nseq, size_t kv_heads, size_t hd, size_t max_tk, int& nit, int& splits) {
    const char* e = getenv("LLMTIE_DECODE_STATIC");
    if (nseq > 64 || (e && atoi(e))) return false;
    if (e) return true;
    const size_t units = nseq * kv_heads;
    const double mb = (double)units * (double)max_tk * (double)(2 * hd + hd / 8) * 1e-6;
    if (mb > (units <= 64 ? 150.0 : 75.0)) return true;
    // Beyond one round of workgroups, even spans of up to 1024 keys (eight blocks
    // a wave): 12 sequences of 100-1000, 11.0 us against 14.0 in three splits
    // each; 20, 12.2 / 14.4; 32, 12.4 / 17.2.
    if (units > 64 && units * (size_t)splits > 256 && nit < 8 && !getenv("LLMTIE_DECODE_NIT") &&
        !getenv("LLMTIE_DECODE_WGS")) {
        const size_t spans = (max_tk + 1023) / 1024;
        nit = (int)(((max_tk + 31) / 32 + 4 * spans - 1) / (4 * spans));
        splits = (int)((max_tk + 128 * (size_t)nit - 1) / (128 * (size_t)nit));
    }
    // Split heads past one workgroup a compute unit (three at head_dim 64, which
    // fit side by side) lose to stream-K. Over 8 kv heads of 128: 17 sequences of
    // up to 1646, 23.8 / 20.5 us; 18 of 283-1135, 17.8 / 16.2; 17 of 924-1027, 18.2
    // / 17.1; but 16 of 529-1059 (256 workgroups), 14.0 / 16.6. Of 64: 60 of
    // 274-1096, 21.7 / 19.7; 53 of 263-1054 (848 workgroups), 19.0 / 17.9; but 47 of
    // 1136-1263 (752), 16.7 / 22.0.
    return splits > 1 && units * (size_t)splits > (hd == 64 ? 768 : 256);
}

// Whether the split partials are merged by a second launch rather than by
// the last-arriving workgroup of each head.
int two_phase_merge(int splits, size_t units) {
    if (const char* e = getenv("LLMTIE_DECODE_TWO_PHASE")) return atoi(e) ? 1 : 0;
    // The in-launch hand-off (coherent stores, a wait, an atomic per
    // workgroup, each counter on its own line) measured faster than a second
    // launch up to 512 workgroups (C2 at 256: 10.69 vs 12.12 us); a second
    // launch merges beyond 1024.
    return (size_t)splits * units > 1024 ? 1 : 0;
}

// Whether a host-planned in-launch merge keeps every head on one XCD: the
// dispatcher deals a launch's workgroups to the eight XCDs of gfx950 in
// turn, so workgroups L and L + 8k share an XCD (which XCD a launch starts on
// varies with what ran before; a partitioned device with fewer XCDs still
// groups them). The plan runs workgroup L on item (L % 8) * (launch / 8) +
// L / 8, so each XCD's run of items must hold whole heads. The kernel checks
// the grouping itself (the arrival counter sums the XCC ids).
int xcd_local(int splits, size_t units, int two_phase) {
    if (const char* e = getenv("LLMTIE_DECODE_XCD")) {
        if (!atoi(e)) return 0;
    }
    const size_t total = (size_t)splits * units;
    if (two_phase || splits <= 1 || total % 8 != 0) return 0;
    return (total / 8) % (size_t)splits == 0 ? 1 : 0;
}

// A buffer the scratch no longer uses. It is kept allocated until the
// scratch is freed: a graph captured earlier may still read it. (Growth is by
// powers of two, so a scratch retires a few dozen buffers at most.)
int retire(llmtie_decode_scratch* s, void* p) {
    if (p) s->retired.push_back(p);
    return LLMTIE_OK;
}

// `room`: partial floats an eager call makes room for beyond its own, so that
// a longer context may be captured after it; a capture goes without.
int ensure_scratch(llmtie_decode_scratch* s, size_t part_floats, size_t ctrs, hipStream_t st, size_t room = 0) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return driver("hipGetDevice", e);
    const bool swap = s->device != dev;
    const bool fits = !swap && s->part_cap >= part_floats && s->ctr_cap >= ctrs;
    if (fits && s->part_cap >= room) return LLMTIE_OK;
    // Allocating inside a stream capture would put the allocation into the
    // graph (or fail); the caller makes one eager call first instead.
    hipStreamCaptureStatus cs = hipStreamCaptureStatusNone;
    e = hipStreamIsCapturing(st, &cs);
    if (e != hipSuccess) return driver("hipStreamIsCapturing", e);
    if (cs != hipStreamCaptureStatusNone && fits) return LLMTIE_OK;
    if (cs != hipStreamCaptureStatusNone)
        return fail(LLMTIE_SCRATCH_GROWTH_IN_CAPTURE, part_floats, s->part_cap, ctrs, s->ctr_cap,
                    "the decode scratch must grow to %zu partial floats and %zu counters while the stream is "
                    "capturing a graph; make one call of this shape before capturing",
                    part_floats, ctrs);
    part_floats = std::max(part_floats, room);
    int r;
    if (swap) {
        // A scratch follows the device it is used on; switching starts over.
        if ((r = retire(s, s->part)) != LLMTIE_OK || (r = retire(s, s->ctr)) != LLMTIE_OK) return r;
        s->part = nullptr;
        s->ctr = nullptr;
        s->part_cap = s->ctr_cap = 0;
        s->device = dev;
    }
    if (!s->lost) {
        void* w = nullptr;
        e = hipHostMalloc(&w, sizeof(unsigned), hipHostMallocMapped | hipHostMallocCoherent);
        if (e != hipSuccess) return driver("allocating the scratch's status word", e);
        s->lost = static_cast<unsigned*>(w);
        *s->lost = 0;
    }
    if (s->part_cap < part_floats) {
        size_t want = 1024;
        while (want < part_floats) want <<= 1;
        // Room for three splits' partials of any decode whose one split fits:
        // a context of ten to twelve blocks may be captured after a shorter
        // one sized the scratch (one_split_blocks).
        want = std::max(want, std::min(4 * want, NOALLOC_PART_FLOATS));
        float* p = nullptr;
        e = hipMalloc(&p, want * sizeof(float));
        if (e != hipSuccess) return driver("allocating", e);
        if ((r = retire(s, s->part)) != LLMTIE_OK) {
            (void)hipFree(p);
            return r;
        }
        s->part = p;
        s->part_cap = want;
    }
    if (s->ctr_cap < ctrs) {
        size_t want = 64;
        while (want < ctrs) want <<= 1;
        unsigned* c = nullptr;
        e = hipMalloc(&c, want * sizeof(unsigned));
        if (e != hipSuccess) return driver("allocating", e);
        // Zeroed by a kernel on the caller's stream (a memset node inside a
        // captured graph is not to be relied on).
        e = launch_fill_u32(c, want, 0u, st);
        if (e != hipSuccess) {
            (void)hipFree(c);
            return driver("zeroing", e);
        }
        if ((r = retire(s, s->ctr)) != LLMTIE_OK) return r;
        s->ctr = c;
        s->ctr_cap = want;
    }
    return LLMTIE_OK;
}

// Partials and counters of the no-allocation decode (device addresses).
struct FixedScratch {
    float* part;
    size_t part_cap;  // floats
    unsigned* ctr;
    size_t ctr_cap;   // words
};

int noalloc_scratch(hipStream_t st, FixedScratch& f);

// The checks and the launch behind every single-sequence decode
// (device.rs:6224-6410).
int decode_common(void* stream, int kind, const float* q, size_t q_len, size_t q_off, const void* k, size_t k_len,
                  const void* v, size_t v_len, size_t heads, size_t kv_heads, size_t hd, size_t tk, size_t cap,
                  float scale, int scale_q, llmtie_decode_scratch* scratch, float* out, size_t out_len,
                  size_t out_off, int8_t* twin, size_t twin_rows, size_t twin_k, bool has_twin,
                  bool noalloc = false) {
    const bool tiled = kind == KV_T16;
    if (!(hd == 64 || hd == 128)) return unsupported(hd, heads, kv_heads);
    if (kv_heads == 0 || heads % kv_heads != 0 || heads / kv_heads > 16) return unsupported(hd, heads, kv_heads);
    if (tk == 0 || tk > cap) return overrun_cache(tk, cap);
    const size_t esz = kind == KV_F32 ? 4 : 2;
    if (!tiled && (cap * esz) % 8 != 0) return odd_cap(cap);
    if (int r = over_int(cap, heads)) return r;
    if (smul(kv_heads, cap, hd) > ((size_t)1 << 40)) return overrun_slice(smul(kv_heads, cap, hd), (size_t)1 << 40);
    if (tiled) {
        const size_t need = kv_heads * (size_t)tiled_nblk((int)cap) * 64 * hd;
        if (k_len < need) return overrun_slice(need, k_len);
        v = k;
    } else {
        const size_t need = kv_heads * cap * hd;
        if (k_len < need || v_len < need) return overrun_slice(need, std::min(k_len, v_len));
    }
    const size_t n = heads * hd;
    if (q_len < sadd(q_off, n)) return overrun_slice(sadd(q_off, n), q_len);
    if (out_len < sadd(out_off, n)) return overrun_slice(sadd(out_off, n), out_len);
    if (out_off % 32 != 0) return fail(LLMTIE_RAGGED_BLOCK, out_off, 32, 0, 0, "a row of %zu in blocks of 32", out_off);
    if (has_twin) {
        // The scales follow the codes at twin + twin_rows * twin_k.
        if (int r = over_int(twin_rows)) return r;
        if (twin_k != n || smul(twin_rows, twin_k) < out_off + n)
            return fail(LLMTIE_MISMATCHED_Q8, twin_rows, twin_k, out_off / n + 1, n,
                        "an int8 twin of %zu rows by %zu where %zu by %zu is needed", twin_rows, twin_k,
                        out_off / n + 1, n);
        if (!twin) return invalid("twin");
    }
    if (!q || !k || !v || !out) return invalid("a buffer");
    if (!scratch && !noalloc) return invalid("scratch");
    // A head lost by an earlier call through this scratch (see
    // llmtie_decode_scratch_status) is reported before anything is launched.
    if (!noalloc) {
        if (int r = llmtie_decode_scratch_status(scratch)) return r;
    }
    const size_t group = heads / kv_heads;
    int nit, splits;
    const size_t one_split = one_split_blocks(kind, kv_heads, group, hd);
    plan_decode(tk, kv_heads, group, nit, splits, one_split);
    const bool one = splits == 1 && (tk + 31) / 32 <= one_split;
    const int waves = one ? one_split_waves(tk, kind, group, hd) : 4;
    if (waves == 8) nit = (int)((tk + 255) / 256);
    const size_t mls = ml_stride(splits, group);
    const size_t part = kv_heads * ((size_t)splits * group * hd + mls);
    const long ml_off = (long)(kv_heads * (size_t)splits * group * hd);
    float* part_p;
    unsigned* ctr_p;
    if (noalloc) {
        // Refused before the device is touched.
        if (part > NOALLOC_PART_FLOATS || kv_heads * CTR_STRIDE > NOALLOC_CTR_WORDS)
            return fail(LLMTIE_SCRATCH_LIMIT, part, NOALLOC_PART_FLOATS, kv_heads * CTR_STRIDE, NOALLOC_CTR_WORDS,
                        "the call needs %zu partial floats and %zu counter words; the fixed scratch holds %zu and "
                        "%zu",
                        part, kv_heads * CTR_STRIDE, NOALLOC_PART_FLOATS, NOALLOC_CTR_WORDS);
        FixedScratch f;
        int r = noalloc_scratch(S(stream), f);
        if (r != LLMTIE_OK) return r;
        part_p = f.part;
        ctr_p = f.ctr;
    } else {
        // A context that the rule keeps whole makes room for the splits it
        // would take past twelve blocks, as its neighbours past the line do.
        size_t room = 0;
        if (one && (tk + 31) / 32 > 12) {
            int nit2, splits2;
            plan_decode(tk, kv_heads, group, nit2, splits2);
            room = kv_heads * ((size_t)splits2 * group * hd + ml_stride(splits2, group));
        }
        int r = ensure_scratch(scratch, part, kv_heads * CTR_STRIDE, S(stream), room);
        if (r != LLMTIE_OK) return r;
        part_p = scratch->part;
        ctr_p = scratch->ctr;
    }
    DecodeArgs a;
    memset(&a, 0, sizeof a);
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    if (has_twin) {
        a.twin_codes = twin;
        a.twin_scales = reinterpret_cast<float*>(twin + twin_rows * twin_k);
    }
    a.part = part_p;
    a.ml_off = ml_off;
    a.ctr = ctr_p;
    a.q_off = (long)q_off;
    a.out_off = (long)out_off;
    a.tk = (int)tk;
    a.cap = (int)cap;
    a.kv_heads = (int)kv_heads;
    a.group = (int)group;
    a.score_l2 = (scale_q ? 1.0f : scale) * 1.4426950408889634f;
    a.qscale = scale_q ? scale : 1.0f;
    a.nit = nit;
    a.waves = waves;
    a.splits = splits;
    a.ml_stride = (long)mls;
    a.two_phase = two_phase_merge(splits, kv_heads);
    // The no-allocation path has no status word to report a lost head to,
    // so it always hands partials over coherently.
    a.xcd = noalloc ? 0 : xcd_local(splits, kv_heads, a.two_phase);
    a.xcd_fake = g_fake_xcc.load() ? 1 : 0;
    a.lost = noalloc ? nullptr : scratch->lost;
    return launched("attn_decode", launch_decode((int)hd, kind, a, (int)kv_heads, 1, S(stream)));
}

}  // namespace

extern "C" {

int llmtie_flash_attn(void* stream, const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                      size_t v_len, float* out, size_t out_len, size_t tq, size_t past, size_t heads,
                      size_t kv_heads, size_t head_dim, size_t cap, float scale, int causal) {
    return prefill_common(stream, PF_F32, q, q_len, k, k_len, v, v_len, out, out_len, tq, past, heads, kv_heads,
                          head_dim, cap, scale, causal);
}

int llmtie_flash_attn_f16(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                          const uint16_t* v, size_t v_len, float* out, size_t out_len, size_t tq, size_t past,
                          size_t heads, size_t kv_heads, size_t head_dim, size_t cap, float scale, int causal) {
    if (!(head_dim == 64 || head_dim == 128)) return unsupported(head_dim, heads, kv_heads);
    if (cap % 2 != 0) return odd_cap(cap);
    return prefill_common(stream, PF_F16, q, q_len, k, k_len, v, v_len, out, out_len, tq, past, heads, kv_heads,
                          head_dim, cap, scale, causal);
}

size_t llmtie_flash_attn_workspace(size_t tq, size_t past, size_t heads, size_t kv_heads, size_t head_dim) {
    // Shapes the prefill itself refuses need none.
    if (!llmtie_supports_flash(head_dim, heads, kv_heads) || tq == 0 || sadd(past, tq) > IMAX ||
        smul(heads, head_dim) > IMAX || smul(tq, heads, head_dim) > (size_t)1 << 40)
        return 0;
    const size_t n = plan_prefill_splits(tq, past, heads, kv_heads, head_dim);
    return n > 1 ? smul(smul(n, tq, heads), head_dim + 2) : 0;
}

int llmtie_flash_attn_f16_ws(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                             const uint16_t* v, size_t v_len, float* out, size_t out_len, size_t tq, size_t past,
                             size_t heads, size_t kv_heads, size_t head_dim, size_t cap, float scale, int causal,
                             float* ws, size_t ws_len) {
    if (!(head_dim == 64 || head_dim == 128)) return unsupported(head_dim, heads, kv_heads);
    if (cap % 2 != 0) return odd_cap(cap);
    return prefill_common(stream, PF_F16, q, q_len, k, k_len, v, v_len, out, out_len, tq, past, heads, kv_heads,
                          head_dim, cap, scale, causal, ws, ws_len);
}

int llmtie_flash_attn_rows(void* stream, const float* qkv, size_t qkv_len, uint16_t* out, size_t out_len, size_t t,
                           size_t heads, size_t head_dim, float scale) {
    if (head_dim != 64 || heads == 0) return unsupported(head_dim, heads, heads);
    if (int r = over_int(smul(heads, head_dim, 3), t)) return r;
    const size_t d = heads * head_dim;
    if (qkv_len < smul(t, 3 * d)) return overrun_slice(smul(t, 3 * d), qkv_len);
    if (out_len < smul(t, d)) return overrun_slice(smul(t, d), out_len);
    if (t == 0) return ok();
    if (!qkv || !out) return invalid("a buffer");
    PrefillArgs a{};
    a.cus = compute_units();
    a.q = qkv;
    a.k = qkv + d;
    a.v = qkv + 2 * d;
    a.out = out;
    a.tq = (int)t;
    a.past = 0;
    a.heads = (int)heads;
    a.kv_heads = (int)heads;
    a.cap = (int)t;
    a.scale = scale;
    a.causal = 0;
    a.gb = 1;
    a.qs = (int)(3 * d);
    a.kvs = (int)(3 * d);
    a.os = (int)d;
    a.scale_q = 1;
    a.out_f16 = 1;
    // The stacked f32 rows are read in place: the attention kernel stages
    // them through registers into its f16 LDS tiles (no copy, no workspace).
    // Eight-wave workgroups of one query tile per wave: the staging per row
    // of two tiles per wave, at two waves per SIMD (C4 encoder 38.2 -> 35.8
    // us). LLMTIE_ROWS_W8=0 selects the four-wave kernel.
    const char* w8 = getenv("LLMTIE_ROWS_W8");
    if (!(w8 && !atoi(w8))) return launched("flash_attn_rows", launch_prefill(64, PF_ROWS, 1, a, S(stream), 8));
    return launched("flash_attn_rows", launch_prefill(64, PF_ROWS, pick_nqt(t, heads, 1, true), a, S(stream)));
}

int llmtie_attn_decode_f16(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                           const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads, size_t head_dim,
                           size_t tk, size_t cap, float scale, int scale_q, llmtie_decode_scratch* scratch,
                           float* out, size_t out_len) {
    return decode_common(stream, KV_F16, q, q_len, 0, k, k_len, v, v_len, heads, kv_heads, head_dim, tk, cap, scale,
                         scale_q, scratch, out, out_len, 0, nullptr, 0, 0, false);
}

}  // extern "C"

// ------------------------------------------------ decode without allocation
//
// `scratch`: the split partials (NOALLOC_PART_FLOATS floats) then the arrival
// counters (NOALLOC_CTR_WORDS words, CTR_STRIDE per kv head) of
// llmtie_attn_decode_f16_noalloc, 4.25 MiB held on every device the library
// runs on until the process ends. Host code never passes the array's name
// (a host-side stand-in, not a device address) to the device: it uses the
// address hipGetSymbolAddress gives for the current device, obtained once per
// device.
static __device__ __align__(256) float scratch[NOALLOC_PART_FLOATS + NOALLOC_CTR_WORDS];

namespace {

std::mutex noalloc_mu;
float* noalloc_ptr[64];

// This device's copy of `scratch` (zero at load; every call leaves its
// counters at zero).
int noalloc_scratch(hipStream_t st, FixedScratch& f) {
    (void)st;
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return driver("hipGetDevice", e);
    if (dev < 0 || dev >= 64) return driver("device index", hipErrorInvalidDevice);
    std::lock_guard<std::mutex> lock(noalloc_mu);
    if (!noalloc_ptr[dev]) {
        float* p = nullptr;
        e = hipGetSymbolAddress(reinterpret_cast<void**>(&p), HIP_SYMBOL(scratch));
        if (e != hipSuccess) return driver("hipGetSymbolAddress(scratch)", e);
        // No clearing launch: the array has no initialiser, so it is zero
        // when the code object is loaded (a zero-filled segment), and every
        // call leaves its counters at zero. A fill here would be recorded
        // into a graph if this first call were made under stream capture.
        noalloc_ptr[dev] = p;
    }
    f.part = noalloc_ptr[dev];
    f.part_cap = NOALLOC_PART_FLOATS;
    f.ctr = reinterpret_cast<unsigned*>(noalloc_ptr[dev] + NOALLOC_PART_FLOATS);
    f.ctr_cap = NOALLOC_CTR_WORDS;
    return LLMTIE_OK;
}

}  // namespace

extern "C" {

int llmtie_attn_decode_f16_noalloc(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                                   const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads, size_t head_dim,
                                   size_t tk, size_t cap, float scale, int scale_q, float* out, size_t out_len) {
    return decode_common(stream, KV_F16, q, q_len, 0, k, k_len, v, v_len, heads, kv_heads, head_dim, tk, cap, scale,
                         scale_q, nullptr, out, out_len, 0, nullptr, 0, 0, false, true);
}

int llmtie_attn_decode_f16_q(void* stream, const float* q, size_t q_len, const uint16_t* k, size_t k_len,
                             const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads, size_t head_dim,
                             size_t tk, size_t cap, float scale, int scale_q, llmtie_decode_scratch* scratch,
                             float* out, size_t out_len, int8_t* twin, size_t twin_len) {
    const size_t n = smul(heads, head_dim);
    if (twin_len < sadd(n, (n / 32) * 4)) return overrun_slice(sadd(n, (n / 32) * 4), twin_len);
    if (n % 32 != 0) return fail(LLMTIE_RAGGED_BLOCK, n, 32, 0, 0, "a row of %zu in blocks of 32", n);
    return decode_common(stream, KV_F16, q, q_len, 0, k, k_len, v, v_len, heads, kv_heads, head_dim, tk, cap, scale,
                         scale_q, scratch, out, out_len, 0, twin, 1, n, true);
}

int llmtie_attn_decode_f16_q_row(void* stream, const float* q, size_t q_len, size_t q_off, const uint16_t* k,
                                 size_t k_len, const uint16_t* v, size_t v_len, size_t heads, size_t kv_heads,
                                 size_t head_dim, size_t tk, size_t cap, float scale, int scale_q,
                                 llmtie_decode_scratch* scratch, float* out, size_t out_len, int8_t* twin,
                                 size_t twin_rows, size_t twin_k, size_t row) {
    return decode_common(stream, KV_F16, q, q_len, q_off, k, k_len, v, v_len, heads, kv_heads, head_dim, tk, cap,
                         scale, scale_q, scratch, out, out_len, smul(row, heads, head_dim), twin, twin_rows, twin_k,
                         true);
}

int llmtie_attn_decode(void* stream, const float* q, size_t q_len, const float* k, size_t k_len, const float* v,
                       size_t v_len, size_t heads, size_t kv_heads, size_t head_dim, size_t tk, size_t cap,
                       float scale, int scale_q, llmtie_decode_scratch* scratch, float* out, size_t out_len) {
    return decode_common(stream, KV_F32, q, q_len, 0, k, k_len, v, v_len, heads, kv_heads, head_dim, tk, cap, scale,
                         scale_q, scratch, out, out_len, 0, nullptr, 0, 0, false);
}

int llmtie_attn_decode_q8_batch(void* stream, const float* q, size_t q_len, const int8_t* cache, size_t cache_len,
                                size_t slots, const int32_t* tk_dev, const int32_t* slot_dev, size_t nseq,
                                size_t max_tk, size_t heads, size_t kv_heads, size_t head_dim, size_t cap,
                                float scale, int scale_q, llmtie_decode_scratch* scratch, float* out,
                                size_t out_len) {
    if (!(head_dim == 64 || head_dim == 128)) return unsupported(head_dim, heads, kv_heads);
    // Groups are bounded by the stream-K kernel's LDS (sk_group_max: 16 at
    // head_dim 64 and 128).
    if (kv_heads == 0 || heads % kv_heads != 0 || heads / kv_heads > (size_t)sk_group_max((int)head_dim))
        return unsupported(head_dim, heads, kv_heads);
    if (max_tk == 0 || max_tk > cap) return overrun_cache(max_tk, cap);
    if (nseq > 65535) return overrun_slice(nseq, 65535);
    // The stream-K kernel addresses one (slot, kv head)'s blocks through a
    // 32-bit buffer range.
    if (smul((cap + 31) / 32, sk_block_bytes((int)head_dim)) > 0x7fffffffu) return overrun_cache(cap, 0x7fffffffu / sk_block_bytes((int)head_dim) * 32);
    if (int r = over_int(cap, slots, heads)) return r;
    const size_t need = llmtie_q8_cache_bytes(slots, kv_heads, head_dim, cap);
    if (cache_len < need) return overrun_slice(need, cache_len);
    const size_t n = heads * head_dim;
    if (q_len < nseq * n) return overrun_slice(nseq * n, q_len);
    if (out_len < nseq * n) return overrun_slice(nseq * n, out_len);
    if (nseq == 0) return ok();
    if (!q || !cache || !tk_dev || !slot_dev || !out) return invalid("a buffer");
    if (!scratch) return invalid("scratch");
    if (int r = llmtie_decode_scratch_status(scratch)) return r;
    const size_t group = heads / kv_heads;
    int nit, splits;
    plan_decode(max_tk, kv_heads * nseq, group, nit, splits);
    bool sk = plan_q8_batch(nseq, kv_heads, head_dim, max_tk, nit, splits);
    const size_t mls = ml_stride(splits, group);
    size_t part = nseq * kv_heads * ((size_t)splits * group * head_dim + mls);
    long ml_off = (long)(nseq * kv_heads * (size_t)splits * group * head_dim);
    const size_t slots2 = (size_t)compute_units() * SK_WAVES * 2;
    const size_t sk_part = slots2 * (16 * head_dim + 32);
    // Every batch of up to 64 sequences takes the partials of the stream-K
    // slots, whichever grid it runs on, so that a scratch which served one of
    // them serves the next under capture, whatever its lengths' bound.
    if (nseq <= 64 && !getenv("LLMTIE_DECODE_STATIC")) {
        sk = sk || part > sk_part;
        part = sk_part;
    }
    const int items = sk ? compute_units() : 0;
    if (sk) {
        ml_off = (long)(slots2 * 16 * head_dim);
        part = sk_part;
    }
    int r = ensure_scratch(scratch, part, nseq * kv_heads * CTR_STRIDE, S(stream));
    if (r != LLMTIE_OK) return r;
    DecodeArgs a;
    memset(&a, 0, sizeof a);
    a.q = q;
    a.k = cache;
    a.out = out;
    a.part = scratch->part;
    a.ml_off = ml_off;
    a.ctr = scratch->ctr;
    a.tk_arr = tk_dev;
    a.slot_arr = slot_dev;
    a.q_stride = (long)n;
    a.out_stride = (long)n;
    a.tk = (int)max_tk;
    a.slots = (int)slots;
    a.cap = (int)cap;
    a.kv_heads = (int)kv_heads;
    a.group = (int)group;
    a.score_l2 = (scale_q ? 1.0f : scale) * 1.4426950408889634f;
    a.qscale = scale_q ? scale : 1.0f;
    a.nit = nit;
    a.splits = splits;
    a.ml_stride = (long)mls;
    a.two_phase = sk ? 0 : two_phase_merge(splits, kv_heads * nseq);
    // Up to 64 sequences the hand-off is coherent on either grid: no head of
    // such a batch can be lost. XCD-local / coherent on the planned grid: 8
    // sequences of 256-4096 at 32/8/128, a step of 8 layers 290 / 297 us; 20 of
    // 386-1042 at 32/8/64, four layers 47.2 / 42.9; nine other batches within 2 %.
    a.xcd = sk || nseq <= 64 ? 0 : xcd_local(splits, kv_heads * nseq, a.two_phase);
    a.xcd_fake = g_fake_xcc.load() ? 1 : 0;
    a.lost = scratch->lost;
    a.sk = sk ? 1 : 0;
    a.nseq = (int)nseq;
    a.items = items;
    return launched("attn_decode_q8_batch", launch_decode((int)head_dim, KV_TQ8, a, (int)kv_heads, (int)nseq, S(stream)));
}

int llmtie_rope(void* stream, float* x, size_t x_len, size_t off, const float* freq_div, size_t t, size_t heads,
                size_t head_dim, float theta, size_t first) {
    if (int r = over_int(t, heads, head_dim, first)) return r;
    const size_t nx = smul(t, heads, head_dim);
    if (sadd(off, nx) > x_len) return overrun_slice(sadd(off, nx), x_len);
    if (head_dim % 2 != 0) return fail(LLMTIE_ODD_HEAD_DIM, head_dim, 0, 0, 0, "a rotary head of odd width %zu", head_dim);
    if (nx == 0) return ok();
    if (!x) return invalid("x");
    return launched("rope", launch_rope(x, (long)off, freq_div, (int)t, (int)heads, (int)head_dim, theta, (int)first,
                                        S(stream)));
}

static int append_common(void* stream, const float* src, size_t src_len, size_t src_off, void* dst, size_t dst_len,
                         int f16, size_t n, size_t kv, size_t hd, size_t cap, size_t past, int tr) {
    if (sadd(past, n) > cap) return overrun_cache(sadd(past, n), cap);
    if (f16 && cap % 2 != 0) return odd_cap(cap);
    if (int r = over_int(cap, kv, hd)) return r;
    const size_t total = smul(n, kv, hd);
    if (sadd(src_off, total) > src_len) return overrun_slice(sadd(src_off, total), src_len);
    if (smul(kv, cap, hd) > dst_len) return overrun_slice(smul(kv, cap, hd), dst_len);
    if (total == 0) return ok();
    if (!src || !dst) return invalid("a buffer");
    return launched("cache_append", launch_append(src, (long)src_off, dst, f16, tr, (int)n, (int)kv, (int)hd,
                                                  (int)cap, (int)past, S(stream)));
}

int llmtie_cache_append(void* stream, const float* src, size_t src_len, size_t src_off, float* dst, size_t dst_len,
                        size_t n, size_t kv_heads, size_t head_dim, size_t cap, size_t past, int transposed) {
    return append_common(stream, src, src_len, src_off, dst, dst_len, 0, n, kv_heads, head_dim, cap, past, transposed);
}

int llmtie_cache_append_f16(void* stream, const float* src, size_t src_len, size_t src_off, uint16_t* dst,
                            size_t dst_len, size_t n, size_t kv_heads, size_t head_dim, size_t cap, size_t past,
                            int transposed) {
    return append_common(stream, src, src_len, src_off, dst, dst_len, 1, n, kv_heads, head_dim, cap, past, transposed);
}

int llmtie_rope_cache_f16(void* stream, float* q, size_t q_len, size_t q_off, const float* k, size_t k_len,
                          size_t k_off, const float* v, size_t v_len, size_t v_off, const float* freq_div,
                          size_t heads, size_t kv_heads, size_t head_dim, float theta, size_t pos, uint16_t* kc,
                          uint16_t* vc, size_t cache_len, size_t cap) {
    if (pos >= cap) return overrun_cache(sadd(pos, 1), cap);
    if (cap % 2 != 0) return odd_cap(cap);
    if (head_dim % 2 != 0) return fail(LLMTIE_ODD_HEAD_DIM, head_dim, 0, 0, 0, "a rotary head of odd width %zu", head_dim);
    if (int r2 = over_int(cap, heads, head_dim)) return r2;
    if (sadd(q_off, heads * head_dim) > q_len) return overrun_slice(sadd(q_off, heads * head_dim), q_len);
    if (sadd(k_off, kv_heads * head_dim) > k_len) return overrun_slice(sadd(k_off, kv_heads * head_dim), k_len);
    if (sadd(v_off, kv_heads * head_dim) > v_len) return overrun_slice(sadd(v_off, kv_heads * head_dim), v_len);
    if (cache_len < smul(cap, kv_heads, head_dim)) return overrun_slice(smul(cap, kv_heads, head_dim), cache_len);
    if (!q || !k || !v || !kc || !vc) return invalid("a buffer");
    return launched("rope_cache_f16",
                    launch_rope_cache_f16(q, (long)q_off, k, (long)k_off, v, (long)v_off, freq_div, (int)heads,
                                          (int)kv_heads, (int)head_dim, theta, (int)pos, kc, vc, (int)cap, S(stream)));
}

static int grow_common(void* stream, const void* src, size_t src_len, void* dst, size_t dst_len, int esz, size_t kv,
                       size_t hd, size_t cap, size_t new_cap, size_t live, int tr) {
    if (live > cap || new_cap < cap) return overrun_cache(std::max(live, cap), std::min(new_cap, cap));
    size_t rows, len, ss, ds;
    if (!tr) {
        rows = kv;
        len = live * hd;
        ss = cap * hd;
        ds = new_cap * hd;
    } else {
        rows = kv * hd;
        len = live;
        ss = cap;
        ds = new_cap;
    }
    if (int r = over_int(rows, ss, ds)) return r;
    if (smul(rows, ss) > src_len) return overrun_slice(smul(rows, ss), src_len);
    if (smul(rows, ds) > dst_len) return overrun_slice(smul(rows, ds), dst_len);
    if (rows * len == 0) return ok();
    if (!src || !dst) return invalid("a buffer");
    return launched("cache_grow", launch_grow(src, dst, esz, (int)rows, (int)len, (int)ss, (int)ds, S(stream)));
}

int llmtie_cache_grow(void* stream, const float* src, size_t src_len, float* dst, size_t dst_len, size_t kv_heads,
                      size_t head_dim, size_t cap, size_t new_cap, size_t live, int transposed) {
    return grow_common(stream, src, src_len, dst, dst_len, 4, kv_heads, head_dim, cap, new_cap, live, transposed);
}

int llmtie_cache_grow_f16(void* stream, const uint16_t* src, size_t src_len, uint16_t* dst, size_t dst_len,
                          size_t kv_heads, size_t head_dim, size_t cap, size_t new_cap, size_t live,
                          int transposed) {
    return grow_common(stream, src, src_len, dst, dst_len, 2, kv_heads, head_dim, cap, new_cap, live, transposed);
}

static int q8_cache_checks(size_t hd, size_t heads, size_t kv, size_t cap, size_t slots, size_t slot,
                           size_t cache_len) {
    if (!(hd == 64 || hd == 128)) return unsupported(hd, heads, kv);
    if (slot >= slots) return overrun_slice(sadd(slot, 1), slots);
    if (int r = over_int(cap, slots, kv)) return r;
    const size_t need = llmtie_q8_cache_bytes(slots, kv, hd, cap);
    if (cache_len < need) return overrun_slice(need, cache_len);
    return LLMTIE_OK;
}

size_t llmtie_q8_cache_bytes(size_t slots, size_t kv_heads, size_t head_dim, size_t cap) {
    if (cap > IMAX) return SIZE_MAX;
    return smul(smul(slots, kv_heads), (size_t)tiled_nblk((int)cap), (size_t)tq8_block_bytes((int)head_dim));
}

size_t llmtie_t16_cache_len(size_t kv_heads, size_t head_dim, size_t cap) {
    if (cap > IMAX) return SIZE_MAX;
    return smul(smul(kv_heads, (size_t)tiled_nblk((int)cap)), 64, head_dim);
}

int llmtie_kv_q8_append(void* stream, const float* k, size_t k_len, size_t k_off, const float* v, size_t v_len,
                        size_t v_off, int8_t* cache, size_t cache_len, size_t slots, size_t slot, size_t n,
                        size_t kv_heads, size_t head_dim, size_t cap, size_t past) {
    int r = q8_cache_checks(head_dim, kv_heads, kv_heads, cap, slots, slot, cache_len);
    if (r != LLMTIE_OK) return r;
    if (sadd(past, n) > cap) return overrun_cache(sadd(past, n), cap);
    const size_t total = smul(n, kv_heads, head_dim);
    if (sadd(k_off, total) > k_len) return overrun_slice(sadd(k_off, total), k_len);
    if (sadd(v_off, total) > v_len) return overrun_slice(sadd(v_off, total), v_len);
    if (total == 0) return ok();
    if (!k || !v || !cache) return invalid("a buffer");
    return launched("kv_q8_append", launch_append_q8(k, (long)k_off, v, (long)v_off, reinterpret_cast<char*>(cache),
                                                     (int)slot, (int)n, (int)kv_heads, (int)head_dim, (int)cap,
                                                     (int)past, S(stream)));
}

int llmtie_rope_cache_q8(void* stream, float* q, size_t q_len, size_t q_off, const float* k, size_t k_len,
                         size_t k_off, const float* v, size_t v_len, size_t v_off, const float* freq_div,
                         size_t heads, size_t kv_heads, size_t head_dim, float theta, size_t pos, int8_t* cache,
                         size_t cache_len, size_t slots, size_t slot, size_t cap) {
    int r = q8_cache_checks(head_dim, heads, kv_heads, cap, slots, slot, cache_len);
    if (r != LLMTIE_OK) return r;
    if (pos >= cap) return overrun_cache(sadd(pos, 1), cap);
    if (int r2 = over_int(cap, heads, head_dim)) return r2;
    if (sadd(q_off, heads * head_dim) > q_len) return overrun_slice(sadd(q_off, heads * head_dim), q_len);
    if (sadd(k_off, kv_heads * head_dim) > k_len) return overrun_slice(sadd(k_off, kv_heads * head_dim), k_len);
    if (sadd(v_off, kv_heads * head_dim) > v_len) return overrun_slice(sadd(v_off, kv_heads * head_dim), v_len);
    if (!q || !k || !v || !cache) return invalid("a buffer");
    return launched("rope_cache_q8", launch_rope_cache_q8(q, (long)q_off, k, (long)k_off, v, (long)v_off, freq_div,
                                                          (int)heads, (int)kv_heads, (int)head_dim, theta, (int)pos,
                                                          reinterpret_cast<char*>(cache), (int)slot, (int)cap,
                                                          S(stream)));
}

// ------------------------------------------------------------ tiled f16

static int t16_checks(size_t hd, size_t heads, size_t kv, size_t cap, size_t cache_len) {
    if (!(hd == 64 || hd == 128) || kv == 0) return unsupported(hd, heads, kv);
    if (int r = over_int(cap, heads, kv)) return r;
    const size_t need = llmtie_t16_cache_len(kv, hd, cap);
    if (cache_len < need) return overrun_slice(need, cache_len);
    return LLMTIE_OK;
}

int llmtie_t16_append(void* stream, const float* src, size_t src_len, size_t src_off, uint16_t* cache,
                      size_t cache_len, size_t n, size_t kv_heads, size_t head_dim, size_t cap, size_t past,
                      int value) {
    int r = t16_checks(head_dim, kv_heads, kv_heads, cap, cache_len);
    if (r != LLMTIE_OK) return r;
    if (sadd(past, n) > cap) return overrun_cache(sadd(past, n), cap);
    const size_t total = smul(n, kv_heads, head_dim);
    if (sadd(src_off, total) > src_len) return overrun_slice(sadd(src_off, total), src_len);
    if (total == 0) return ok();
    if (!src || !cache) return invalid("a buffer");
    return launched("t16_append", launch_append_t16(src, (long)src_off, cache, (int)n, (int)kv_heads, (int)head_dim,
                                                    (int)cap, (int)past, value ? 1 : 0, S(stream)));
}

int llmtie_t16_rope_cache(void* stream, float* q, size_t q_len, size_t q_off, const float* k, size_t k_len,
                          size_t k_off, const float* v, size_t v_len, size_t v_off, const float* freq_div,
                          size_t heads, size_t kv_heads, size_t head_dim, float theta, size_t pos, uint16_t* cache,
                          size_t cache_len, size_t cap) {
    int r = t16_checks(head_dim, heads, kv_heads, cap, cache_len);
    if (r != LLMTIE_OK) return r;
    if (pos >= cap) return overrun_cache(sadd(pos, 1), cap);
    if (int r2 = over_int(cap, heads, head_dim)) return r2;
    if (sadd(q_off, heads * head_dim) > q_len) return overrun_slice(sadd(q_off, heads * head_dim), q_len);
    if (sadd(k_off, kv_heads * head_dim) > k_len) return overrun_slice(sadd(k_off, kv_heads * head_dim), k_len);
    if (sadd(v_off, kv_heads * head_dim) > v_len) return overrun_slice(sadd(v_off, kv_heads * head_dim), v_len);
    if (!q || !k || !v || !cache) return invalid("a buffer");
    return launched("t16_rope_cache",
                    launch_rope_cache_t16(q, (long)q_off, k, (long)k_off, v, (long)v_off, freq_div, (int)heads,
                                          (int)kv_heads, (int)head_dim, theta, (int)pos, cache, (int)cap, S(stream)));
}

int llmtie_t16_grow(void* stream, const uint16_t* src, size_t src_len, uint16_t* dst, size_t dst_len,
                    size_t kv_heads, size_t head_dim, size_t cap, size_t new_cap, size_t live) {
    if (live > cap || new_cap < cap) return overrun_cache(std::max(live, cap), std::min(new_cap, cap));
    int r = t16_checks(head_dim, kv_heads, kv_heads, cap, src_len);
    if (r != LLMTIE_OK) return r;
    r = t16_checks(head_dim, kv_heads, kv_heads, new_cap, dst_len);
    if (r != LLMTIE_OK) return r;
    const size_t bl = 64 * head_dim;  // halves per block
    const size_t rows = kv_heads, len = (size_t)tiled_nblk((int)live) * bl;
    if (rows * len == 0) return ok();
    if (!src || !dst) return invalid("a buffer");
    return launched("t16_grow", launch_grow(src, dst, 2, (int)rows, (int)len, (int)(tiled_nblk((int)cap) * bl),
                                            (int)(tiled_nblk((int)new_cap) * bl), S(stream)));
}

int llmtie_t16_from_ref(void* stream, const uint16_t* k, size_t k_len, const uint16_t* v, size_t v_len,
                        size_t kv_heads, size_t head_dim, size_t cap, size_t live, uint16_t* cache,
                        size_t cache_len) {
    int r = t16_checks(head_dim, kv_heads, kv_heads, cap, cache_len);
    if (r != LLMTIE_OK) return r;
    if (live > cap) return overrun_cache(live, cap);
    const size_t need = smul(kv_heads, cap, head_dim);
    if (k_len < need || v_len < need) return overrun_slice(need, std::min(k_len, v_len));
    if (live == 0) return ok();
    if (!k || !v || !cache) return invalid("a buffer");
    return launched("t16_from_ref", launch_ref_to_t16(k, v, cache, (int)kv_heads, (int)head_dim, (int)cap, (int)live,
                                                      (int)cap, S(stream)));
}

int llmtie_attn_decode_t16(void* stream, const float* q, size_t q_len, const uint16_t* cache, size_t cache_len,
                           size_t heads, size_t kv_heads, size_t head_dim, size_t tk, size_t cap, float scale,
                           int scale_q, llmtie_decode_scratch* scratch, float* out, size_t out_len) {
    return decode_common(stream, KV_T16, q, q_len, 0, cache, cache_len, nullptr, 0, heads, kv_heads, head_dim, tk,
                         cap, scale, scale_q, scratch, out, out_len, 0, nullptr, 0, 0, false);
}

int llmtie_attn_decode_t16_q_row(void* stream, const float* q, size_t q_len, size_t q_off, const uint16_t* cache,
                                 size_t cache_len, size_t heads, size_t kv_heads, size_t head_dim, size_t tk,
                                 size_t cap, float scale, int scale_q, llmtie_decode_scratch* scratch, float* out,
                                 size_t out_len, int8_t* twin, size_t twin_rows, size_t twin_k, size_t row) {
    return decode_common(stream, KV_T16, q, q_len, q_off, cache, cache_len, nullptr, 0, heads, kv_heads, head_dim,
                         tk, cap, scale, scale_q, scratch, out, out_len, smul(row, heads, head_dim), twin, twin_rows,
                         twin_k, twin != nullptr);
}

int llmtie_flash_attn_t16_ws(void* stream, const float* q, size_t q_len, const uint16_t* cache, size_t cache_len,
                             float* out, size_t out_len, size_t tq, size_t past, size_t heads, size_t kv_heads,
                             size_t head_dim, size_t cap, float scale, int causal, float* ws, size_t ws_len) {
    int r = t16_checks(head_dim, heads, kv_heads, cap, cache_len);
    if (r != LLMTIE_OK) return r;
    // The tiled cache holds both areas in one buffer; the length checks of the
    // shared path are satisfied by passing the whole-cache extent for both.
    const size_t ext = smul(kv_heads, cap, head_dim);
    return prefill_common(stream, PF_T16, q, q_len, cache, ext, cache, ext, out, out_len, tq, past, heads, kv_heads,
                          head_dim, cap, scale, causal, ws, ws_len);
}

int llmtie_flash_attn_t16(void* stream, const float* q, size_t q_len, const uint16_t* cache, size_t cache_len,
                          float* out, size_t out_len, size_t tq, size_t past, size_t heads, size_t kv_heads,
                          size_t head_dim, size_t cap, float scale, int causal) {
    return llmtie_flash_attn_t16_ws(stream, q, q_len, cache, cache_len, out, out_len, tq, past, heads, kv_heads,
                                    head_dim, cap, scale, causal, nullptr, 0);
}

}  // extern "C"

// ------------------------------------- key ranges and rotary positions by row

namespace {

int refuse(const char* what) { return fail(LLMTIE_INVALID_ARGUMENT, 0, 0, 0, 0, "%s", what); }
bool off16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) != 0; }
// Elements that `rows` rows of `n`, `stride` apart, reach from `off`.
size_t reach(size_t off, size_t rows, size_t stride, size_t n) {
    return rows == 0 ? off : sadd(off, sadd(smul(rows - 1, stride), n));
}
// Workgroups of 256 threads that a launch (fewer than 2^32 threads) holds.
constexpr size_t MAX_WGS = ((size_t)1 << 24) - 1;

// Batched decode over key ranges: blocks of a head kept in one workgroup, and the
// bytes (half of the 256 MB Infinity Cache) past which a launch streams.
constexpr int RD_WHOLE = 20;
constexpr size_t RD_LONG = 192;  // blocks of a bound under which lengths may differ much
constexpr size_t RD_TWO = 64;    // and from which heads past a round are two runs
constexpr size_t RD_STREAM_BYTES = (size_t)128 << 20;

// What the score arguments must be: every logit of finite queries and keys is
// then above the reference maximum that a row starts from, -1e30, and twice a
// slope over the scale is finite.
int score_checks(float scale, float softcap, const float* slopes, size_t slopes_len, size_t heads) {
    if (!(scale >= 1e-15f) || !(scale <= 1e15f)) return refuse("a score scale that is not in 1e-15 to 1e15");
    if (softcap != 0.0f && !(softcap >= 1e-3f && softcap <= 1e3f))
        return refuse("a score cap that is neither 0 nor in 0.001 to 1000");
    if (slopes && slopes_len < heads) return overrun_slice(heads, slopes_len);
    return LLMTIE_OK;
}

// Runs that a prompt's row blocks are cut into (1: whole) when they are few and
// their keys many: two workgroups a compute unit, of four tiles or more. Us, as
// planned / whole: 173 rows after 3011 of 32/8/128 26.9 / 44.7 (5 runs; 4 28.8, 8
// 29.0), 16 after 3000 15.6 / 42.1 (11; 8 15.5, 16 16.2), 100 after 7000 28.8 / 91
// (9; 4 32.5), 40 after 1000 12.2 / 17.8, 400 after 1500 30.7 / 30.0 (2; 4 34.3); 40 after
// 2000 of 20/20/64 11.1 / 21.0; 1000 rows of 32/8/128 (504 blocks, whole) in 2 33.4 / 21.8.
size_t plan_range_splits(size_t tq, size_t keys, size_t heads, size_t kv_heads) {
    const size_t group = heads / kv_heads;
    const size_t gb = group % 4 == 0 ? 4 : (group % 2 == 0 ? 2 : 1);
    const size_t pb = 16 * (4 / gb), items = (tq + pb - 1) / pb * (heads / gb);
    const size_t cus = (size_t)compute_units(), tiles = (keys + 63) / 64;
    if (items >= cus || tiles <= 8) return 1;
    return std::max<size_t>(1, std::min<size_t>(std::min<size_t>(32, tiles / 4), 2 * cus / items));
}

// 16-row query tiles a wave (each K and V fragment read from LDS serves both of
// two). Two where the launch then still has workgroups enough: two a compute unit, fewer
// where the rows are alike (no fewer positions before them than there are rows,
// so that none ends early), more where a score takes longer than its reads (head_dim 64).
// Us, one / two; workgroups at two: 304 (1200 rows of 32/8/128) 26.7 / 33.3, after
// 4000 134 / 126; 440, after 4000 169 / 151; 504 47.0 / 54.0, capped 53 / 67, after 186 / 165;
// 656 75.6 / 72.1, capped 87.4 / 86.9; 1000 156 / 126. head_dim 64: 440 (1750 of 32/8) after
// 4000 96 / 100; 640 (4000 of 20/20) 102 / 92, after 305 / 183, capped 119 / 156; 656 (2600 of
// 32/8) 44.5 / 51.3, after 150 / 137; 1000 88 / 85, capped 116 / 115.
int range_tiles(size_t tq, size_t past, size_t heads, size_t hd, int gb, bool capped) {
    if (getenv("LLMTIE_PREFILL_NQT")) return std::min(2, pick_nqt(tq, heads, gb));
    const size_t rows = 32 * (4 / gb), wgs = (tq + rows - 1) / rows * (heads / gb);
    const size_t cus = (size_t)compute_units();
    if (past >= tq) return wgs >= (hd == 128 ? cus + cus / 8 : 2 * cus) ? 2 : 1;
    return wgs >= (hd == 128 ? 2 * cus : capped ? 4 * cus - cus / 8 : 5 * cus / 2) ? 2 : 1;
}

// Workgroups that a decode cuts each (sequence, kv head) into: those that fill the
// compute units once without a second round, or twice where the launch streams; a
// launch just past a round waits for it. Us at runs (workgroups): 40 heads of 3000
// keys of 128 dims 6 (240) 16.5, 7 (280) 18.2, 12 (480) 17.6; 80 of 3000 3 (240) 26.3,
// 4 (320) 29.4, 6 (480) 26.4; streamed, 40 of 8000 5 (200) 32.7, 6 31.7, 12 (480) 31.1,
// 13 (520) 36.4; 96 of 8000 2 67.7, 3 81.7, 5 (480) 66.2, 6 73.6; 160 of 500-5000 1 59.9,
// 2 50.2, 3 (480) 49.1, 4 50.2. (Very uneven ones can gain by more: 96 of 20-8000 5
// 45.1, 6 37.9; of 256-8192 47.7, 45.5.)
// Heads that fill the compute units by themselves are whole, unless the bound is so
// long that lengths under it differ much: then four runs. Means of eight batches of
// 32/8/128 under 8192, capped, whole / in two / in four: of 256-8192 224 heads 93.7 /
// 93.6 / 89.9, 240 96.8 / 96.9 / 95.4, 256 100.6 / 101.0 / 100.0; of 64-8192 over their
// logarithm 70.2 / 48.5 / 45.0, 70.7 / 49.3 / 47.9, 71.3 / 50.3 / 49.9; but of 4096-8192 113.6 /
// 115.4 / 118.2, 120.3 / 123.2 / 124.4, 126.9 / 130.2 / 132.4. Means of three batches of 256-8192:
// 264 heads 126 / 108 / 108, 288 160 / 117 / 118, 384 176 / 159 / 151; 448 184 / - / 167, 640 of 64
// dims 135 / - / 119. (Under 192 blocks whole: 224 of 1000-4000 53.6 / - / 59.1, 256 of 2500
// 53.0 / - / 62.5.)
// Some more than one a compute unit are two runs: 288 of 1000-4000 78.0 / 73.5, 320 of
// 2500 79.4 / 73.4, 448 90.3 / 98.6; behind a window of 1024 34.8 / 37.1.
size_t range_runs(size_t units, size_t blocks, bool streams) {
    const size_t cus = (size_t)compute_units(), one = std::max<size_t>(1, cus / units), two = 2 * cus / units;
    if (!streams) return one;
    if (two >= 3) return two;
    if (units <= 3 * cus && blocks >= RD_LONG) return 4;
    return units > cus && units <= cus + cus / 2 && blocks >= RD_TWO ? 2 : 1;
}
// The most partials (a workgroup's each) that range_runs leaves to any batch, of
// bounds up to `blocks`: four runs of three heads a compute unit, two of one and a
// half, or twice the compute units.
size_t range_room(size_t blocks) {
    return (size_t)compute_units() * (blocks >= RD_LONG ? 12 : blocks >= RD_TWO ? 3 : 2);
}

// Binades that a prompt's row forms its largest weight above 1. A weight's
// rounding to f16 is at most 2^-25 where it is small, 2^(-25 - lift) of the
// largest: over 2^13 keys 2^-12 of it, half of a weight's own rounding, and each
// doubling of the keys wants one more. (At 0, a key 25 binades above 2^17 others,
// with its tile the first, rounded all of them away, 0.4 % of the context.) Not seen
// in the time where it is wanted, us at 0 / so: 1000 rows of 32/8/128 behind 31000 593 / 593
// (2), behind 130000 2444 / 2437 (4), capped 2982 / 2985. More than that costs: lifted
// rows leave f16's range sooner, and a tile that moves the reference is formed twice
// (8192 rows at 0 / 5 / 8 / 11 490 / 496 / 507 / 517, capped 585 / 590 / 595 / 613).
float range_lift(size_t keys) {
    int lift = 0;
    while (lift < 10 && keys > (size_t)1 << (13 + lift)) ++lift;
    return (float)lift;
}

int rotary_checks(size_t hd, size_t rot, float theta, float mscale, size_t rows, size_t heads, size_t pos_len,
                  bool has_pos, size_t first, bool has_div, size_t div_len) {
    if (hd % 2 != 0 || hd == 0) return fail(LLMTIE_ODD_HEAD_DIM, hd, 0, 0, 0, "a rotary head of odd width %zu", hd);
    if (rot % 2 != 0) return fail(LLMTIE_ODD_HEAD_DIM, rot, 0, 0, 0, "a rotary head of odd width %zu", rot);
    if (rot > hd) return overrun_slice(rot, hd);
    if (hd > 1024) return refuse("a rotary head wider than 1024");
    if (!(theta > 0.0f) || !std::isfinite(theta) || !std::isfinite(mscale))
        return refuse("a rotary base that is not positive, or a multiplier that is not finite");
    // Workgroups of a launch, and its rows and threads' items, are ints.
    if (rows > (size_t)1 << 26) return overrun_slice(rows, (size_t)1 << 26);
    if (int r = over_int(smul(heads, hd, 4), sadd(first, rows))) return r;
    if (has_pos && pos_len < rows) return overrun_slice(rows, pos_len);
    if (has_div && div_len < rot / 2) return overrun_slice(rot / 2, div_len);
    return LLMTIE_OK;
}

// Whether the rotated rows may be written: over the source itself, or apart from it.
bool overlap(const void* a, size_t an, const void* b, size_t bn) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + bn && y < x + an;
}
// Whether some of `rows` rows of an floats from a on, sa apart, shares a byte with
// one of bn from b on, sb apart. (Two strides through the same memory: taken for it.)
bool rows_overlap(const float* a, size_t an, size_t sa, const float* b, size_t bn, size_t sb, size_t rows) {
    if (!overlap(a, reach(0, rows, sa, an) * 4, b, reach(0, rows, sb, bn) * 4)) return false;
    if (rows == 1 || sa != sb) return true;
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b), s = sa * 4;
    const uintptr_t d = x <= y ? (y - x) % s : (s - (x - y) % s) % s;  // where b's row begins in a's stride
    return d < an * 4 || d + bn * 4 > s;
}

}  // namespace

extern "C" {

int llmtie_key_ranges(void* stream, const int32_t* starts, size_t starts_len, const int32_t* prefix, size_t prefix_len,
                      size_t rows, size_t past, int causal, size_t window, size_t shared, int32_t* table,
                      size_t table_len, int32_t* pos, size_t pos_len) {
    if (int r = over_int(sadd(past, rows), starts_len)) return r;
    if (starts && starts_len == 0) return overrun_slice(1, 0);
    const size_t docs = starts ? starts_len - 1 : 1;
    if (prefix && prefix_len < docs) return overrun_slice(docs, prefix_len);
    if (smul(rows, 3) > table_len) return overrun_slice(smul(rows, 3), table_len);
    if (pos && pos_len < rows) return overrun_slice(rows, pos_len);
    if (rows == 0) return ok();
    if (!table) return invalid("a buffer");
    KeyRangeArgs a{};
    a.starts = starts;
    a.prefix = prefix;
    a.table = table;
    a.pos = pos;
    a.docs = (int)docs;
    a.rows = (int)rows;
    a.past = (int)past;
    a.causal = causal ? 1 : 0;
    a.window = (int)std::min(window, IMAX);  // wider than any position: no window's effect
    a.shared = (int)std::min(shared, IMAX);
    return launched("key_ranges", launch_key_ranges(a, S(stream)));
}

int llmtie_rope_rows(void* stream, const float* x, size_t x_len, size_t off, size_t stride, void* out, size_t out_len,
                     size_t out_off, size_t out_stride, int out_f16, const int32_t* pos, size_t pos_len, size_t first,
                     const float* freq_div, size_t div_len, size_t t, size_t heads, size_t head_dim, size_t rot_dim,
                     float theta, float mscale, int interleaved) {
    if (int r = rotary_checks(head_dim, rot_dim, theta, mscale, t, heads, pos_len, pos != nullptr, first,
                              freq_div != nullptr, div_len))
        return r;
    const size_t n = smul(heads, head_dim);
    if (t > 1 && (stride < n || out_stride < n)) return overrun_slice(n, std::min(stride, out_stride));
    if (reach(off, t, stride, n) > x_len) return overrun_slice(reach(off, t, stride, n), x_len);
    if (reach(out_off, t, out_stride, n) > out_len) return overrun_slice(reach(out_off, t, out_stride, n), out_len);
    if (t == 0 || n == 0) return ok();
    if (!x || !out) return invalid("a buffer");
    const size_t es = out_f16 ? 2 : 4;
    const char* o = static_cast<char*>(out) + out_off * es;
    const bool same = !out_f16 && o == reinterpret_cast<const char*>(x + off) && (stride == out_stride || t == 1);
    if (!same && overlap(x + off, reach(0, t, stride, n) * 4, o, reach(0, t, out_stride, n) * es))
        return refuse("rotated rows that overlap their source but are not its own");
    RotaryArgs a{};
    a.q = x + off;
    a.qo = const_cast<char*>(o);
    a.pos = pos;
    a.first = (int)first;
    a.div = freq_div;
    a.q_stride = t > 1 ? (long)stride : 0;
    a.qo_stride = t > 1 ? (long)out_stride : 0;
    a.rows = (int)t;
    a.heads = (int)heads;
    a.hd = (int)head_dim;
    a.rot = (int)rot_dim;
    a.interleaved = interleaved ? 1 : 0;
    a.qo_f16 = out_f16 ? 1 : 0;
    a.mscale = mscale;
    a.log2_theta = std::log2((double)theta);
    return launched("rope_rows", launch_rotary(a, false, S(stream)));
}

int llmtie_t16_rope_store(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride, void* q_out,
                          size_t q_out_len, size_t q_out_off, size_t q_out_stride, int q_out_f16, const float* k,
                          size_t k_len, size_t k_off, size_t k_stride, const float* v, size_t v_len, size_t v_off,
                          size_t v_stride, const int32_t* pos, const int32_t* slot, const int32_t* index,
                          size_t index_len, const float* freq_div, size_t div_len, size_t rows, size_t heads,
                          size_t kv_heads, size_t head_dim, size_t rot_dim, float theta, float mscale,
                          int interleaved, uint16_t* cache, size_t cache_len, size_t slots, size_t cap) {
    if (!(head_dim == 64 || head_dim == 128) || kv_heads == 0) return unsupported(head_dim, heads, kv_heads);
    if (int r = rotary_checks(head_dim, rot_dim, theta, mscale, rows, std::max(heads, kv_heads), index_len, true, 0,
                              freq_div != nullptr, div_len))
        return r;
    if (int r = over_int(cap, slots, kv_heads)) return r;
    const size_t need = smul(slots, llmtie_t16_cache_len(kv_heads, head_dim, cap));
    if (cache_len < need) return overrun_slice(need, cache_len);
    const size_t n = smul(heads, head_dim), nk = smul(kv_heads, head_dim);
    const size_t es = q_out_f16 ? 2 : 4;
    if (q) {
        if (rows > 1 && (q_stride < n || q_out_stride < n)) return overrun_slice(n, std::min(q_stride, q_out_stride));
        if (reach(q_off, rows, q_stride, n) > q_len) return overrun_slice(reach(q_off, rows, q_stride, n), q_len);
        if (reach(q_out_off, rows, q_out_stride, n) > q_out_len)
            return overrun_slice(reach(q_out_off, rows, q_out_stride, n), q_out_len);
    }
    if (rows > 1 && (k_stride < nk || v_stride < nk)) return overrun_slice(nk, std::min(k_stride, v_stride));
    if (reach(k_off, rows, k_stride, nk) > k_len) return overrun_slice(reach(k_off, rows, k_stride, nk), k_len);
    if (reach(v_off, rows, v_stride, nk) > v_len) return overrun_slice(reach(v_off, rows, v_stride, nk), v_len);
    if (rows == 0) return ok();
    if (!k || !v || !pos || !slot || !index || !cache || (q && !q_out)) return invalid("a buffer");
    if (off16(cache)) return refuse("a cache off 16 bytes");
    RotaryArgs a{};
    if (q && heads) {
        const char* o = static_cast<char*>(q_out) + q_out_off * es;
        const size_t on = reach(0, rows, q_out_stride, n) * es;
        const bool same =
            !q_out_f16 && o == reinterpret_cast<const char*>(q + q_off) && (q_stride == q_out_stride || rows == 1);
        if (!same && (overlap(q + q_off, reach(0, rows, q_stride, n) * 4, o, on) ||
                      overlap(k + k_off, reach(0, rows, k_stride, nk) * 4, o, on) ||
                      overlap(v + v_off, reach(0, rows, v_stride, nk) * 4, o, on)))
            return refuse("rotated queries that overlap a source but are not their own");
        if (same && (rows_overlap(q + q_off, n, q_stride, k + k_off, nk, k_stride, rows) ||
                     rows_overlap(q + q_off, n, q_stride, v + v_off, nk, v_stride, rows)))
            return refuse("queries rotated in place that lie over k's or v's rows");
        a.q = q + q_off;
        a.qo = const_cast<char*>(o);
    }
    a.k = k + k_off;
    a.v = v + v_off;
    a.pos = pos;
    a.slot = slot;
    a.index = index;
    a.div = freq_div;
    a.cache = cache;
    a.q_stride = rows > 1 ? (long)q_stride : 0;
    a.qo_stride = rows > 1 ? (long)q_out_stride : 0;
    a.k_stride = rows > 1 ? (long)k_stride : 0;
    a.v_stride = rows > 1 ? (long)v_stride : 0;
    a.rows = (int)rows;
    a.heads = (int)heads;
    a.kv = (int)kv_heads;
    a.hd = (int)head_dim;
    a.rot = (int)rot_dim;
    a.interleaved = interleaved ? 1 : 0;
    a.qo_f16 = q_out_f16 ? 1 : 0;
    a.slots = (int)slots;
    a.cap = (int)cap;
    a.mscale = mscale;
    a.log2_theta = std::log2((double)theta);
    return launched("t16_rope_store", launch_rotary(a, true, S(stream)));
}

size_t llmtie_flash_attn_ranges_workspace(size_t tq, size_t max_keys, size_t heads, size_t kv_heads, size_t head_dim) {
    if (!llmtie_supports_flash(head_dim, heads, kv_heads) || tq == 0 || tq > IMAX || max_keys > IMAX) return 0;
    const size_t splits = plan_range_splits(tq, max_keys, heads, kv_heads);
    return splits > 1 ? smul(smul(splits, tq, heads), head_dim + 2) : 0;
}

int llmtie_flash_attn_ranges_t16(void* stream, const uint16_t* q, size_t q_len, size_t q_off, size_t q_stride,
                                 const uint16_t* cache, size_t cache_len, size_t slots, size_t slot,
                                 const int32_t* table, size_t table_len, size_t max_keys, uint16_t* out,
                                 size_t out_len, size_t tq, size_t past, size_t heads, size_t kv_heads,
                                 size_t head_dim, size_t cap, float scale, float softcap, const float* slopes,
                                 size_t slopes_len, float* ws, size_t ws_len) {
    if (!llmtie_supports_flash(head_dim, heads, kv_heads)) return unsupported(head_dim, heads, kv_heads);
    if (int r = score_checks(scale, softcap, slopes, slopes_len, heads)) return r;
    if (sadd(past, tq) > cap) return overrun_cache(sadd(past, tq), cap);
    if (int r = over_int(smul(heads, head_dim), sadd(cap, 128), slots)) return r;
    if (slot >= slots) return overrun_slice(sadd(slot, 1), slots);
    const size_t one = llmtie_t16_cache_len(kv_heads, head_dim, cap);
    if (cache_len < smul(slots, one)) return overrun_slice(smul(slots, one), cache_len);
    const size_t n = smul(heads, head_dim), nq = smul(tq, n);
    if (nq > (size_t)1 << 40) return overrun_slice(nq, (size_t)1 << 40);
    if (tq > 1 && q_stride < n) return overrun_slice(n, q_stride);
    if (reach(q_off, tq, q_stride, n) > q_len) return overrun_slice(reach(q_off, tq, q_stride, n), q_len);
    if (out_len < nq) return overrun_slice(nq, out_len);
    if (table_len < smul(tq, 3)) return overrun_slice(smul(tq, 3), table_len);
    if (table_len != smul(tq, 3)) return refuse("a row table of another row count");
    if (tq == 0) return ok();
    if (!q || !cache || !table || !out) return invalid("a buffer");
    if (off16(cache) || off16(out)) return refuse("a cache or a context off 16 bytes");
    const size_t group = heads / kv_heads;
    const int gb = group % 4 == 0 ? 4 : (group % 2 == 0 ? 2 : 1);
    const size_t keys = std::min(max_keys ? max_keys : IMAX, past + tq);
    const size_t splits = ws && ws_len ? plan_range_splits(tq, keys, heads, kv_heads) : 1;
    if (splits > 1) {
        const size_t need = smul(smul(splits, tq, heads), head_dim + 2);
        if (ws_len < need) return overrun_slice(need, ws_len);
        if (off16(ws)) return refuse("a workspace off 16 bytes");
    }
    const int nqt = splits > 1 ? 1 : range_tiles(tq, past, heads, head_dim, gb, softcap != 0.0f);
    const size_t items = smul((tq + 16 * nqt * (4 / gb) - 1) / (16 * nqt * (4 / gb)), heads / gb, splits);
    if (items > MAX_WGS) return overrun_slice(items, MAX_WGS);
    RangesArgs a{};
    a.q = q + q_off;
    a.cache = cache + slot * one;
    a.out = out;
    a.first = table;
    a.lo = table + tq;
    a.hi = table + 2 * tq;
    a.slopes = slopes;
    a.q_stride = tq > 1 ? (long)q_stride : 0;
    a.tq = (int)tq;
    a.past = (int)past;
    a.heads = (int)heads;
    a.kv_heads = (int)kv_heads;
    a.cap = (int)cap;
    a.scale = scale;
    a.softcap = softcap;
    a.lift = range_lift(past + tq);
    a.gb = gb;
    a.splits = (int)splits;
    a.ws = ws;
    a.qal = !off16(a.q) && a.q_stride % 8 == 0;
    return launched("flash_attn_ranges", launch_ranges((int)head_dim, nqt, a, S(stream)));
}

int llmtie_attn_decode_ranges_t16(void* stream, const float* q, size_t q_len, size_t q_off, size_t q_stride,
                                  const uint16_t* cache, size_t cache_len, size_t slots, const int32_t* tk_dev,
                                  const int32_t* slot_dev, const int32_t* lo_dev, size_t nseq, size_t max_tk,
                                  size_t window, size_t shared, size_t heads, size_t kv_heads, size_t head_dim,
                                  size_t cap, float scale, float softcap, const float* slopes, size_t slopes_len,
                                  llmtie_decode_scratch* scratch, float* out, size_t out_len) {
    if (!llmtie_supports_flash(head_dim, heads, kv_heads) || heads / kv_heads > 16)
        return unsupported(head_dim, heads, kv_heads);
    if (int r = score_checks(scale, softcap, slopes, slopes_len, heads)) return r;
    if (max_tk == 0 || max_tk > cap) return overrun_cache(max_tk, cap);
    if (int r = over_int(smul(heads, head_dim), sadd(cap, 128), slots, nseq)) return r;
    const size_t need = smul(slots, llmtie_t16_cache_len(kv_heads, head_dim, cap));
    if (cache_len < need) return overrun_slice(need, cache_len);
    const size_t n = smul(heads, head_dim);
    if (nseq > 1 && q_stride < n) return overrun_slice(n, q_stride);
    if (reach(q_off, nseq, q_stride, n) > q_len) return overrun_slice(reach(q_off, nseq, q_stride, n), q_len);
    if (out_len < smul(nseq, n)) return overrun_slice(smul(nseq, n), out_len);
    if (!slot_dev && nseq > slots) return overrun_slice(nseq, slots);
    if (nseq == 0) return ok();
    if (!q || !cache || !tk_dev || !out) return invalid("a buffer");
    if (!scratch) return invalid("scratch");
    if (off16(cache) || off16(out)) return refuse("a cache or a context off 16 bytes");
    if (int r = llmtie_decode_scratch_status(scratch)) return r;
    const size_t group = heads / kv_heads, units = smul(nseq, kv_heads);
    const size_t keys = window ? std::min(max_tk, sadd(window, shared)) : max_tk;
    const size_t blocks = (keys + 31) / 32;
    // Runs of a head, of four blocks (one a wave) or more; a head of up to RD_WHOLE
    // blocks is one run (a merge costs ~3 us). Us, whole / cut: 1 sequence of 32/8/128, 14
    // blocks 6.8 / 7.5, 18 7.5 / 7.5, 28 8.9 / 7.5; of 20/20/64, 18 5.9 / 7.2, 28
    // 7.0 / 7.3; 16 sequences of 32/8/128, 18 blocks 12.2 / 12.9, 28 16.0 / 15.7.
    const size_t span = 4;
    const size_t most = std::min<size_t>(DECODE_MAX_SPLITS, DECODE_MAX_SPLIT_ROWS / group);
    // Past half the Infinity Cache a launch streams: what it reads cannot be
    // kept until it is read again, and loads that do not try read faster (32
    // sequences of 256-8192, 113 / 101 us; 4 of 200-6000, which fit, 15.2 / 16.6).
    const bool streams = smul(smul(units, blocks), 128, head_dim) > RD_STREAM_BYTES;
    const size_t runs = range_runs(units, blocks, streams);
    const size_t splits = std::max<size_t>(1, std::min(std::min((blocks + span - 1) / span, most), runs));
    if (smul(units, splits) > MAX_WGS) return overrun_slice(smul(units, splits), MAX_WGS);
    const size_t parts = smul(units, splits, n / kv_heads);
    // An eager call makes room for the runs of any smaller batch under its bound too
    // (they can be more): one of the largest sizes a scratch for captured ones.
    const size_t row = smul(group, head_dim + 2);
    if (int r = ensure_scratch(scratch, smul(units, splits, row), smul(units, CTR_STRIDE), S(stream),
                               smul(range_room(blocks), row)))
        return r;
    RangesDecodeArgs a{};
    a.q = q + q_off;
    a.cache = cache;
    a.out = out;
    a.tk = tk_dev;
    a.slot = slot_dev;
    a.lo = lo_dev;
    a.slopes = slopes;
    a.part = scratch->part;
    a.ml_off = (long)parts;
    a.ctr = scratch->ctr;
    a.q_stride = nseq > 1 ? (long)q_stride : 0;
    a.nseq = (int)nseq;
    a.slots = (int)slots;
    a.cap = (int)cap;
    a.kv_heads = (int)kv_heads;
    a.group = (int)group;
    a.window = (int)std::min(window, IMAX);
    a.shared = (int)std::min(shared, IMAX);
    a.splits = (int)splits;
    a.span = (int)span;
    a.whole = RD_WHOLE;
    a.stream = streams ? 1 : 0;
    a.scale = scale;
    a.softcap = softcap;
    return launched("attn_decode_ranges", launch_ranges_decode((int)head_dim, a, S(stream)));
}

}  // extern "C"
