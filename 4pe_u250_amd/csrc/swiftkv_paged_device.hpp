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
// Byte i (below 64) of a sequence's; `sequence` and n are uniform.
__device__ __forceinline__ uint32_t tree_byte(const TreeBytes& bytes, int sequence, int n, int i) {
    typedef uint32_t Words __attribute__((ext_vector_type(kTreeTokens / 4), aligned(4)));
    Words words = *reinterpret_cast<const Words*>(bytes.words + sequence * (tree_pitch(n) / 4));
    asm("" : "+s"(words));               // one load of all, not each under the condition below
    uint32_t mine = 0;
#pragma unroll
    for (int w = 0; w < kTreeTokens / 4; ++w)
        if (i >> 2 == w) mine = words[w];
    return mine >> (8 * (i & 3)) & 0xffu;
}
__device__ __forceinline__ TreePlace tree_place(const TreeBytes& parents, int sequence, int n, int lane) {
    const uint32_t parent = lane < n ? tree_byte(parents, sequence, n, lane) : kTreeNone;
    TreePlace t{uint64_t(1) << lane, parent != kTreeNone};
    int up = parent < kTreeTokens ? static_cast<int>(parent) : lane;
#pragma unroll
    for (int i = 0; i < 6; ++i) {
        t.mask |= from_lane(t.mask, up);
        up = __shfl(up, up);
    }
    return t;
}

// x cos + y sin (the sine's sign is the caller's), in FP32 and one order of operations
// in every kernel, so that a key's row does not depend on which of them appends it.  (The
// empty asm keeps the compiler from one instruction that multiplies, adds and rounds to
// float16 at once, which it took in some places.)
__device__ __forceinline__ float turn(float x, float y, float c, float s) {
    float z = __builtin_fmaf(x, c, y * s);
    asm("" : "+v"(z));
    return z;
}

// 8 channels, 8 * chunk .., of a head's row, and what turns them: a channel's partner is
// its neighbour, or with `halves` a channel half the rotary channels away, which is read
// from the row again.  Loads and arithmetic apart, so that several chunks' loads can be on
// their way; small code, since a workgroup runs it once, and fetches it for that.
template <typename T>
struct Chunk {
    Half8<T> own, other;
    v4f angle[4];

    // ok: aligned_rotation(r)
    __device__ __forceinline__ void load(const T* row, int chunk, const PagedRotation& r, const float2* cs) {
        const int half = r.rotary_dim / 2, c0 = 8 * chunk;
        const bool turns = c0 < r.rotary_dim, upper = c0 >= half;
        own = *reinterpret_cast<const Half8<T>*>(row + c0);
        const int partner = upper ? c0 - half : c0 + half, at = r.halves ? (upper ? c0 - half : c0) : c0 / 2;
        other = *reinterpret_cast<const Half8<T>*>(row + (turns && r.halves ? partner : c0));
        const v4f* const angles = reinterpret_cast<const v4f*>(cs + (turns ? at : 0));
#pragma unroll
        for (int i = 0; i < 4; ++i) angle[i] = angles[r.halves ? i : i & 1];
    }
    __device__ __forceinline__ Half8<T> turned(int chunk, const PagedRotation& r) const {
        const int c0 = 8 * chunk;
        Half8<T> out;
        if (r.halves) {
            const uint32_t sign = c0 >= r.rotary_dim / 2 ? 0u : 0x80000000u;
#pragma unroll
            for (int j = 0; j < 8; ++j)
                out[j] = static_cast<T>(turn(static_cast<float>(own[j]), static_cast<float>(other[j]), angle[j >> 1][2 * (j & 1)],
                                             __uint_as_float(__float_as_uint(angle[j >> 1][2 * (j & 1) + 1]) ^ sign)));
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float s = angle[j >> 2][2 * (j >> 1 & 1) + 1];
                out[j] = static_cast<T>(turn(static_cast<float>(own[j]), static_cast<float>(own[j ^ 1]), angle[j >> 2][2 * (j >> 1 & 1)], j & 1 ? s : -s));
            }
        }
        return c0 < r.rotary_dim ? out : own;
    }
};
// Whether whole chunks turn and their partners and angles are whole 16-byte pieces.
__device__ __forceinline__ bool aligned_rotation(const PagedRotation& r) {
    return r.table != nullptr && (r.halves ? (r.rotary_dim & 15) == 0 : (r.rotary_dim & 7) == 0);
}
// One chunk, by any rotation or none.
template <typename T>
__device__ __forceinline__ Half8<T> turned(const T* row, int chunk, const PagedRotation& r, const float2* cs) {
    if (aligned_rotation(r)) {
        Chunk<T> x;
        x.load(row, chunk, r, cs);
        return x.turned(chunk, r);
    }
    const int half = r.rotary_dim / 2, c0 = 8 * chunk;
    Half8<T> out = *reinterpret_cast<const Half8<T>*>(row + c0);
#pragma unroll 1
    for (int c = c0; c < min(c0 + 8, r.rotary_dim); ++c) {
        const bool second = r.halves ? c >= half : c & 1;
        const int other = r.halves ? (second ? c - half : c + half) : c ^ 1, j = r.halves ? (second ? c - half : c) : c >> 1;
        const T z = static_cast<T>(turn(static_cast<float>(row[c]), static_cast<float>(row[other]), cs[j].x, second ? cs[j].y : -cs[j].y));
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c - c0 == k) out[k] = z;
    }
    return out;
}
// The angles of a position.
__device__ __forceinline__ const float2* angles(const PagedRotation& r, int position) {
    return r.table + static_cast<int64_t>(r.table == nullptr ? 0 : position) * (r.rotary_dim / 2);
}

}  // namespace dev
}  // namespace swiftkv
