// swiftkv_block_device.hpp -- device code that the block cache's kernel files
// share.
#pragma once

#include <type_traits>

#include "swiftkv_block.hpp"
#include "swiftkv_device.hpp"

namespace swiftkv {
namespace dev {

constexpr float kFloatMax = 3.402823466e+38f;

template <typename T>
struct alignas(16) Vec8 {
    T v[8];
};

template <typename F>
void with_type(ElementType t, F&& f) {
    if (t == kF32) f(float{});
    else if (t == kBF16) f(__bf16{});
    else f(_Float16{});
}

// 1 / s of a power of two within 2^-126 .. 2^126, exactly.
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float((254u << 23) - __float_as_uint(s)); }

// r / group and the query token of a row, without a division.
__device__ __forceinline__ int row_token(const BlockAttendArgs& a, int r) {
    return a.group_magic == 0 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), a.group_magic));
}

// Tiles of each split but the last of a sequence that has `splits`: even shares,
// in whole turns of four waves (so that none is longer than the launch's
// split_tiles, a multiple of four, and none is empty).
__device__ __forceinline__ int split_length(int tiles, int splits) { return ((tiles + splits - 1) / splits + 3) & ~3; }

// What one workgroup tells another: write-through stores, loads past the caches.
__device__ __forceinline__ void publish(float* p, float v) {
    __hip_atomic_store(reinterpret_cast<uint32_t*>(p), __float_as_uint(v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float fetch(const float* p) {
    return __uint_as_float(__hip_atomic_load(const_cast<uint32_t*>(reinterpret_cast<const uint32_t*>(p)),
                                             __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// x 2^d of a whole d <= 0, also where 2^d leaves FP32's range and the product does not:
// with a reference value that follows weights times V scales, sums of weights go up to 2^100.
__device__ __forceinline__ float scaled(float x, float d) { return ldexpf(x, static_cast<int>(fmaxf(d, -400.0f))); }

// One output channel d of a row from its splits' (m, l, acc), `step` floats apart,
// in split order.  Eight splits' loads go out together.  WHOLE: the m are whole
// numbers and go by weights times V scales.
template <bool WHOLE>
__device__ __forceinline__ void join_splits(const float* src, int step, int splits, int d, float& m, float& l, float& o) {
    m = -INFINITY;
    l = o = 0.0f;
    for (int j0 = 0; j0 < splits; j0 += 8) {
        float mj[8], lj[8], oj[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float* at = src + static_cast<int64_t>(min(j0 + j, splits - 1)) * step;
            mj[j] = fetch(at);
            lj[j] = fetch(at + 1);
            oj[j] = fetch(at + 2 + d);
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (j0 + j >= splits) mj[j] = -INFINITY, lj[j] = oj[j] = 0.0f;
            top = fmaxf(top, mj[j]);
        }
        const float safe = top == -INFINITY ? 0.0f : top;
        auto add = [&](float mi, float li, float oi) {
            if (WHOLE) {
                l += scaled(li, mi - safe);
                o += scaled(oi, mi - safe);
            } else {
                const float f = fast_exp2(mi - safe);
                l = __builtin_fmaf(li, f, l);
                o = __builtin_fmaf(oi, f, o);
            }
        };
        const float l0 = l, o0 = o;
        l = o = 0.0f;
        add(m, l0, o0);
#pragma unroll
        for (int j = 0; j < 8; ++j) add(mj[j], lj[j], oj[j]);
        m = top;
    }
}

// A tile's scales, uniform over the wave.
struct TileHead {
    float ks[kTileBlocks], vs[kTileBlocks];
};

// The table entries and scales of 64 of a wave's tiles, a tile in each lane,
// so that the scan's loads wait for no other: read one tile at a time (scalar
// loads, which share a counter with LDS accesses) they took two trips to memory
// a tile, and 64 sequences of 4096 tokens 128 us.
struct TileHeads {
    uint64_t entry;
    uint64_t scale[kTileBlocks];

    __device__ __forceinline__ void load_entries(const uint64_t* table, int tile, int last) {
        entry = table[min(tile, last)];
    }
    __device__ __forceinline__ void load_scales(const int8_t* scales) {
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j)
            scale[j] = *reinterpret_cast<const uint64_t*>(scales + 8 * ((entry >> (16 * j)) & 0xffffu));
    }
    // Waits for the scales here, and not in each turn of the loop that uses them.
    __device__ __forceinline__ void arrive() const {
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) asm volatile("" ::"v"(scale[j]));
    }
    // Records 0 and 1 of a tile, then 2 and 3.
    __device__ __forceinline__ uint32_t low(int lane) const {
        return __builtin_amdgcn_readlane(static_cast<uint32_t>(entry), lane);
    }
    __device__ __forceinline__ uint32_t high(int lane) const {
        return __builtin_amdgcn_readlane(static_cast<uint32_t>(entry >> 32), lane);
    }
    __device__ __forceinline__ void scales_of(int lane, TileHead& h) const {
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            h.ks[j] = __uint_as_float(__builtin_amdgcn_readlane(static_cast<uint32_t>(scale[j]), lane));
            h.vs[j] = __uint_as_float(__builtin_amdgcn_readlane(static_cast<uint32_t>(scale[j] >> 32), lane));
        }
    }
};

}  // namespace dev
}  // namespace swiftkv
