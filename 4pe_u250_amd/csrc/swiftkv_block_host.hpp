// swiftkv_block_host.hpp -- what the host files of the rotary positions, the block
// cache and the paged cache share: the rotary table, checks of arguments.
#pragma once

#include "swiftkv_internal.hpp"

#include "swiftkv_block.hpp"

struct swiftkv_rotary_table {
    swiftkv_context* ctx = nullptr;
    int32_t rotary_dim = 0;
    int32_t positions = 0;
    float2* table = nullptr;   // device [positions][rotary_dim / 2] (cos, sin)
};

namespace swiftkv {

inline int check_tensor(const char* name, const void* p, int64_t stride, int64_t row, int32_t dtype) {
    if (!p) return fail(SWIFTKV_EINVAL, "null %s", name);
    if (reinterpret_cast<uintptr_t>(p) & 15u) return fail(SWIFTKV_EINVAL, "%s must be 16-byte aligned", name);
    if (stride < row || stride > (int64_t(1) << 40))
        return fail(SWIFTKV_EINVAL, "%s stride %lld outside [%lld, 2^40]", name, static_cast<long long>(stride),
                    static_cast<long long>(row));
    if (stride * static_cast<int64_t>(element_bytes(dtype)) % 16 != 0)
        return fail(SWIFTKV_EINVAL, "%s stride %lld is not a multiple of 16 bytes", name,
                    static_cast<long long>(stride));
    return SWIFTKV_OK;
}

inline int check_idle_io(const swiftkv_context* ctx) {
    if (!ctx) return fail(SWIFTKV_EINVAL, "null context");
    if (ctx->released) return fail(SWIFTKV_ESTATE, "the context has been destroyed");
    if (ctx->host_io) return fail(SWIFTKV_ESTATE, "this entry takes device pointers: switch host-memory I/O mode off");
    return SWIFTKV_OK;
}

}  // namespace swiftkv
