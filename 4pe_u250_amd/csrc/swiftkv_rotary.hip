// swiftkv_rotary.hip -- rotation of query and key heads by their positions.
//
// Reading x and writing out bound it (3 operations a channel).  Vector form: a
// thread turns 8 pairs of one head, 16 channels, as two 8-channel loads and
// stores.  Scalar form, for sizes, strides or addresses that 8-element
// vectors do not divide: a thread turns one pair.
#include <type_traits>

#include "swiftkv_block.hpp"

namespace swiftkv {
namespace {

constexpr int kRotaryThreads = 256;

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};

// grid (token of the sequence, part of the token's units, sequence); a unit is 2 V channels
// of one head: V pairs, or where they do not turn, a copy.
template <typename T, int V, bool HALVES, bool INVERSE>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(const RotaryArgs a) {
    const int turning = a.rotary_dim / (2 * V);
    const int units = turning + (a.head_dim - a.rotary_dim + 2 * V - 1) / (2 * V);
    const int id = blockIdx.y * kRotaryThreads + threadIdx.x;
    if (id >= units * a.heads) return;
    const int head = id / units, unit = id % units;
    const int64_t token = static_cast<int64_t>(blockIdx.z) * a.n + blockIdx.x;
    const T* x = static_cast<const T*>(a.x) + token * a.x_stride + static_cast<int64_t>(head) * a.head_dim;
    T* out = static_cast<T*>(a.out) + token * a.out_stride + static_cast<int64_t>(head) * a.head_dim;
    using P = Pack<T, V>;
    if (unit >= turning) {
        const int c = a.rotary_dim + (unit - turning) * 2 * V;
        *reinterpret_cast<P*>(out + c) = *reinterpret_cast<const P*>(x + c);
        if (c + V < a.head_dim) *reinterpret_cast<P*>(out + c + V) = *reinterpret_cast<const P*>(x + c + V);
        return;
    }
    const int half = a.rotary_dim / 2, j = unit * V;
    const int first = HALVES ? j : 2 * j, second = HALVES ? half + j : 2 * j + V;
    const P p0 = *reinterpret_cast<const P*>(x + first), p1 = *reinterpret_cast<const P*>(x + second);
    const float2* cs = a.table + static_cast<int64_t>(a.positions[blockIdx.z] + static_cast<int>(blockIdx.x)) * half + j;
    P r0, r1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float2 f = cs[i];
        const float s = INVERSE ? -f.y : f.y;
        // adjacent pairs: pair i of the 2 V channels that p0 and p1 hold in order
        const float u = static_cast<float>(HALVES ? p0.v[i] : (2 * i < V ? p0.v[(2 * i) % V] : p1.v[(2 * i) % V]));
        const float w = static_cast<float>(HALVES ? p1.v[i] : (2 * i + 1 < V ? p0.v[(2 * i + 1) % V] : p1.v[(2 * i + 1) % V]));
        const T t0 = static_cast<T>(u * f.x - w * s), t1 = static_cast<T>(u * s + w * f.x);
        if (HALVES) {
            r0.v[i] = t0;
            r1.v[i] = t1;
        } else {
            (2 * i < V ? r0 : r1).v[(2 * i) % V] = t0;
            (2 * i + 1 < V ? r0 : r1).v[(2 * i + 1) % V] = t1;
        }
    }
    *reinterpret_cast<P*>(out + first) = r0;
    *reinterpret_cast<P*>(out + second) = r1;
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, int batch, ElementType t, bool halves, bool inverse, hipStream_t s) {
    const bool vectors = a.head_dim % 8 == 0 && a.rotary_dim % 16 == 0 && a.x_stride % 8 == 0 && a.out_stride % 8 == 0 &&
                         reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
    auto go = [&](auto tag, auto v) {
        using T = decltype(tag);
        constexpr int V = decltype(v)::value;
        const int units = a.rotary_dim / (2 * V) + (a.head_dim - a.rotary_dim + 2 * V - 1) / (2 * V);
        const dim3 grid(a.n, (units * a.heads + kRotaryThreads - 1) / kRotaryThreads, batch);
        if (halves && inverse) rotary_kernel<T, V, true, true><<<grid, kRotaryThreads, 0, s>>>(a);
        else if (halves) rotary_kernel<T, V, true, false><<<grid, kRotaryThreads, 0, s>>>(a);
        else if (inverse) rotary_kernel<T, V, false, true><<<grid, kRotaryThreads, 0, s>>>(a);
        else rotary_kernel<T, V, false, false><<<grid, kRotaryThreads, 0, s>>>(a);
    };
    auto typed = [&](auto tag) {
        if (vectors) go(tag, std::integral_constant<int, 8>{});
        else go(tag, std::integral_constant<int, 1>{});
    };
    if (t == kF32) typed(float{});
    else if (t == kBF16) typed(__bf16{});
    else typed(_Float16{});
    return hipGetLastError();
}

}  // namespace swiftkv
