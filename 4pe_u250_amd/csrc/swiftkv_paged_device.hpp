// swiftkv_paged_device.hpp -- device code that the paged cache's kernel files share.
#pragma once

#include "swiftkv_block_device.hpp"
#include "swiftkv_paged.hpp"

namespace swiftkv {
namespace dev {

template <typename T>
using Half8 = T __attribute__((ext_vector_type(8)));

// Bytes of a step's cells from its start (the layout above).
__device__ __forceinline__ int k_cell(int token, int chunk) {
    return ((((chunk >> 2) * 2 + ((token >> 2) & 1)) * 4 + (chunk & 3)) * 16 + ((token >> 3) * 4 + (token & 3))) * 16;
}
__device__ __forceinline__ int v_cell(int octet, int channel, int head_dim) {
    return kStepTokens * head_dim * 2 + (((channel >> 4) * 4 + octet) * 16 + (channel & 15)) * 16;
}

// What a token of a call sees of it, and how deep it stands.  One wave, a token in
// each lane (n <= 64): bit j of the mask is token j, itself among them.  Each turn
// joins the mask of the token that a chain of ancestors has reached and doubles
// the chain.
struct TreePlace {
    uint64_t mask;
    bool live;
};
__device__ __forceinline__ uint64_t from_lane(uint64_t x, int lane) {
    return static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(x), lane))) |
           static_cast<uint64_t>(static_cast<uint32_t>(__shfl(static_cast<int>(x >> 32), lane))) << 32;
}
__device__ __forceinline__ TreePlace tree_place(const uint8_t* parents, int n, int lane) {
    const uint8_t parent = lane < n ? parents[lane] : kTreeNone;
    TreePlace t{uint64_t(1) << lane, parent != kTreeNone};
    int up = parent < kTreeTokens ? parent : lane;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        t.mask |= from_lane(t.mask, up);
        up = __shfl(up, up);
    }
    return t;
}

// A pair (a, b) turned by (cos, sin), in FP32 and one order of operations in every
// kernel, so that a key's row does not depend on which of them appends it.  (The
// empty asm keeps the compiler from one instruction that multiplies, adds and rounds
// to float16 at once, which it took in some places.)
__device__ __forceinline__ float in_fp32(float x) {
    asm("" : "+v"(x));
    return x;
}
__device__ __forceinline__ float turn_first(float a, float b, float2 f) { return in_fp32(__builtin_fmaf(a, f.x, -(b * f.y))); }
__device__ __forceinline__ float turn_second(float a, float b, float2 f) { return in_fp32(__builtin_fmaf(a, f.y, b * f.x)); }

// 8 channels, 8 * chunk .., of a head's row turned by the angles of `cs`, rounded
// once.  Both pairings; a pair's other half is read from the row again.
template <typename T>
__device__ __forceinline__ Half8<T> turned(const T* row, int chunk, const PagedRotation& r, const float2* cs) {
    const Half8<T> own = *reinterpret_cast<const Half8<T>*>(row + 8 * chunk);
    if (r.table == nullptr) return own;
    const int half = r.rotary_dim / 2, c0 = 8 * chunk;
    Half8<T> out = own;
    if (!r.halves) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool turns = c0 + 2 * i < r.rotary_dim;
            const float2 f = cs[turns ? 4 * chunk + i : 0];
            const float a = static_cast<float>(own[2 * i]), b = static_cast<float>(own[2 * i + 1]);
            if (turns) {
                out[2 * i] = static_cast<T>(turn_first(a, b, f));
                out[2 * i + 1] = static_cast<T>(turn_second(a, b, f));
            }
        }
    } else if ((half & 7) == 0) {
        const bool turns = c0 < r.rotary_dim, second = c0 >= half;
        const int other = !turns ? c0 : second ? c0 - half : c0 + half, j = !turns ? 0 : second ? c0 - half : c0;
        const Half8<T> pair = *reinterpret_cast<const Half8<T>*>(row + other);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float2 f = cs[j + i];
            const float x = static_cast<float>(own[i]), y = static_cast<float>(pair[i]);
            const float z = second ? turn_second(y, x, f) : turn_first(x, y, f);
            if (turns) out[i] = static_cast<T>(z);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = c0 + i;
            if (c >= r.rotary_dim) continue;
            const bool second = c >= half;
            const float2 f = cs[second ? c - half : c];
            const float x = static_cast<float>(own[i]), y = static_cast<float>(row[second ? c - half : c + half]);
            out[i] = static_cast<T>(second ? turn_second(y, x, f) : turn_first(x, y, f));
        }
    }
    return out;
}
// The angles of a position.
__device__ __forceinline__ const float2* angles(const PagedRotation& r, int position) {
    return r.table + static_cast<int64_t>(r.table == nullptr ? 0 : position) * (r.rotary_dim / 2);
}

}  // namespace dev
}  // namespace swiftkv
