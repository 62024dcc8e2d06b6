// swiftkv_internal.hpp -- the library's objects and the helpers that its host
// files (swiftkv_capi.cpp, swiftkv_block_capi.cpp) share: errors, the context,
// its children's life time.
#pragma once

#include "../../include/swiftkv.h"

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "swiftkv_common.hpp"

namespace swiftkv {

constexpr int kTimerSlots = 64;

// A fixed buffer, so that reporting an error never allocates.
inline thread_local char g_last_error[512];

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    std::vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
    va_end(ap);
    return code;
}

inline int ok() {
    g_last_error[0] = '\0';
    return SWIFTKV_OK;
}

#define SKV_HIP(expr)                                                                          \
    do {                                                                                       \
        hipError_t e_ = (expr);                                                                \
        if (e_ != hipSuccess)                                                                  \
            return fail(SWIFTKV_EHIP, "%s: %s (%s:%d)", #expr, hipGetErrorString(e_), __FILE__, \
                        __LINE__);                                                             \
    } while (0)

// Device memory; where there is none, no error stays behind for the next launch's
// check to report.
inline bool device_malloc(void** p, size_t bytes) {
    if (hipMalloc(p, bytes) == hipSuccess) return true;
    (void)hipGetLastError();
    return false;
}

struct ProfilePair {
    hipEvent_t begin;
    hipEvent_t end;
    int kind;
};

}  // namespace swiftkv

struct swiftkv_context {
    int device = 0;
    int cus = 256;              // compute units of the device
    int step_per_cu = 3;        // 4-wave step workgroups one CU holds at once
    hipStream_t stream = nullptr;
    int32_t split_tokens = 0;   // 0: heuristic
    swiftkv::StepShape forced_shape{0, 0};   // testing aid: waves 0 = the launch plan's shape
    // split-context workspace: [partial_rows][32] arrival words (kArrivalStride
    // apart), then [partial_rows][32][partial_slots][kSlotWords] tagged words,
    // zero-filled when allocated (generation 0; tag 0 is never current)
    uint64_t* partials = nullptr;
    int32_t partial_rows = 0;
    int32_t partial_slots = 0;
    // Graphs record the workspace pointer in their kernel nodes.  Each graph
    // names the buffer it recorded (if any), with a count of live graphs per
    // buffer here; a buffer the workspace outgrows is freed at once unless a
    // live graph recorded it, and is then kept in `retired` until the last
    // such graph is destroyed.
    std::unordered_map<void*, int64_t> graph_refs;
    std::vector<void*> retired;
    bool capture_uses_workspace = false;   // a split launch of the capture in progress used `partials`
    // [kMaxBatchPerLaunch][32] arrival words (kArrivalStride apart), zero, for
    // launches that split no head: the step reads its arrival word on every
    // path but only a split head's merge writes one
    uint64_t* arrivals = nullptr;
    // workspace of the integer-compatibility step: the exp2 table, then the
    // split exchange (kExactWorkspaceWords; fixed, so a graph may record it at
    // any time)
    uint64_t* exact_workspace = nullptr;
    uint8_t* scratch = nullptr;     // this device's allocation-free workspace (arrival words, then partials)
    // Fault word of the split merges: pinned host memory that a step kernel
    // writes (system scope) when a merge gives up on a partial, read without
    // a device round trip by swiftkv_synchronize, the step entries and graph
    // launches, which report it once and clear it.
    uint32_t* fault_host = nullptr;
    uint32_t* fault_dev = nullptr;
    bool merge_fault_test = false;  // testing aid: merges wait for a tag no word carries
    // timing
    hipEvent_t timers[swiftkv::kTimerSlots] = {};
    bool profiling = false;
    std::vector<swiftkv::ProfilePair> profile_pool;
    size_t profile_used = 0;
    bool capturing = false;     // the stream is being recorded into a graph
    // host-memory I/O mode: step inputs/outputs are host pointers staged here
    bool host_io = false;
    uint8_t* io_stage = nullptr;
    size_t io_bytes = 0;
    // Objects created from the context (caches, tables, graphs, device
    // buffers) may outlive swiftkv_context_destroy: the context is only
    // marked released then, and freed when the last of them is destroyed.
    int64_t children = 0;
    bool released = false;
    std::unordered_set<void*> buffers;   // swiftkv_device_alloc allocations not yet freed
    // Arrival counts and split partials of the block cache's attention, of a
    // fixed size (a graph may record them at any time): allocated with the first
    // block cache.
    uint32_t* block_workspace = nullptr;
    // The same of the paged cache's attention, allocated with the first paged cache.
    uint32_t* paged_workspace = nullptr;
    int32_t paged_rows = 0;     // testing aid: rows of a paged attention workgroup, 0 = the plan's
};

struct swiftkv_graph {
    swiftkv_context* ctx = nullptr;
    hipGraph_t graph = nullptr;
    hipGraphExec_t exec = nullptr;
    void* workspace = nullptr;   // the split workspace buffer its launches recorded, if any
};

struct swiftkv_rope_lut {
    swiftkv_context* ctx = nullptr;
    int32_t positions = 0;
    int2* table = nullptr;              // device [positions][64] (cos, sin)
    std::vector<int2> host;             // host copy for export
};

struct swiftkv_kv_cache {
    swiftkv_context* ctx = nullptr;
    int32_t layers = 0;
    int32_t max_batch = 0;
    int32_t seq_cap = 0;
    int64_t page_bytes = 0;
    size_t bytes = 0;
    int8_t* base = nullptr;
};

namespace swiftkv {

inline int set_device(const swiftkv_context* ctx) {
    if (ctx->released) return fail(SWIFTKV_ESTATE, "the context has been destroyed");
    SKV_HIP(hipSetDevice(ctx->device));
    return SWIFTKV_OK;
}

// Releases everything the context owns (swiftkv_capi.cpp).
void free_context(swiftkv_context* ctx);

// One object created from `ctx` has been destroyed.
inline void release_child(swiftkv_context* ctx) {
    if (--ctx->children == 0 && ctx->released) free_context(ctx);
}

// Entry points that synchronize, copy, allocate or memset cannot be recorded.
inline int not_capturing(const swiftkv_context* ctx, const char* what) {
    if (ctx && ctx->capturing) return fail(SWIFTKV_ESTATE, "%s is not allowed during graph capture", what);
    return SWIFTKV_OK;
}

// The rotary frequencies of `dim` channels in 64 bits, and what multiplies cos
// and sin (see swiftkv_rope_scaling).  `f` has dim / 2 places.
inline int rope_frequencies(int32_t dim, double theta, const swiftkv_rope_scaling* scaling, double* f,
                            double* magnitude) {
    if (!(theta > 1.0) || !std::isfinite(theta)) return fail(SWIFTKV_EINVAL, "theta must be finite and > 1");
    const swiftkv_rope_scaling none{};
    const swiftkv_rope_scaling& sc = scaling ? *scaling : none;
    if (sc.kind < 0 || sc.kind > SWIFTKV_ROPE_BANDS) return fail(SWIFTKV_EINVAL, "unknown RoPE scaling %d", sc.kind);
    if (sc.kind != 0 && (!(sc.factor >= 1.0) || !std::isfinite(sc.factor)))
        return fail(SWIFTKV_EINVAL, "RoPE scaling: factor must be finite and >= 1");
    if (sc.kind == SWIFTKV_ROPE_THETA && dim < 4)
        return fail(SWIFTKV_EINVAL, "RoPE scaling by theta needs at least 4 rotary channels");
    if (sc.kind == SWIFTKV_ROPE_BANDS &&
        (sc.original_positions < 1 || !(sc.low > 0.0) || !(sc.high > sc.low) || !std::isfinite(sc.high)))
        return fail(SWIFTKV_EINVAL, "RoPE scaling by bands: original_positions >= 1 and 0 < low < high");
    if (!std::isfinite(sc.magnitude)) return fail(SWIFTKV_EINVAL, "RoPE scaling: magnitude must be finite");
    *magnitude = sc.magnitude == 0.0 ? 1.0 : sc.magnitude;
    const int32_t half = dim / 2;
    const double base =
        sc.kind == SWIFTKV_ROPE_THETA ? theta * std::pow(sc.factor, static_cast<double>(dim) / (dim - 2)) : theta;
    if (!std::isfinite(base)) return fail(SWIFTKV_EINVAL, "RoPE scaling: the stretched theta overflows");
    for (int32_t j = 0; j < half; ++j) {
        f[j] = 1.0 / std::pow(base, static_cast<double>(j) / half);
        if (sc.kind == SWIFTKV_ROPE_LINEAR) f[j] /= sc.factor;
        if (sc.kind == SWIFTKV_ROPE_BANDS) {
            const double turns = sc.original_positions * f[j] / (2.0 * 3.14159265358979323846);
            double keep = (turns - sc.low) / (sc.high - sc.low);
            keep = keep < 0.0 ? 0.0 : keep > 1.0 ? 1.0 : keep;
            f[j] = (1.0 - keep) * f[j] / sc.factor + keep * f[j];
        }
    }
    return SWIFTKV_OK;
}

}  // namespace swiftkv
