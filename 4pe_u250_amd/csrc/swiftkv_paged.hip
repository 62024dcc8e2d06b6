// swiftkv_paged.hip -- rows of the paged cache: append, values, keep, copy, and
// its table.  Layout: swiftkv_paged.hpp.
#include "swiftkv_paged_device.hpp"

namespace swiftkv {
namespace {

using namespace dev;

constexpr int kRowThreads = 256;

__global__ __launch_bounds__(kMapEntries) void paged_map_kernel(const PagedMapArgs a) {
    const int i = threadIdx.x;
    if (i < a.n) a.entries[i] = a.pages[i];
}

// The step's cells of one head, or null where its tokens have no page.
__device__ __forceinline__ uint8_t* step_cells(const PagedView& v, int slot, int layer, int kh, int step) {
    const int page = v.table[static_cast<int64_t>(slot) * v.entries + step / kPageSteps];
    if (page < 0) return nullptr;
    return v.base + paged_record(v, layer, page, kh) + (step % kPageSteps) * paged_step_bytes(v.head_dim);
}

// Workgroup (key/value head, step of 32 tokens, sequence).  Reading the rows and
// writing the cells bound it: a wave turns and writes four tokens' K cells, 64
// consecutive bytes of each chunk, and V goes through LDS into whole cells; where
// a cell's octet holds other tokens too, only the new ones' bytes are written.
template <typename T, int HD, typename Tree>
__global__ __launch_bounds__(kRowThreads) void paged_append_kernel(const PagedRowsArgs a, const Tree tree) {
    constexpr bool kTree = std::is_same<Tree, PagedTree>::value;
    constexpr int kChunks = HD / 8, kItems = kStepTokens * kChunks / kRowThreads;
    constexpr int kPitch = HD + 8;
    __shared__ __align__(16) T rows[kStepTokens * kPitch];
    const int kh = blockIdx.x, b = blockIdx.z, lane = threadIdx.x & 63;
    const int p = a.positions[b];
    if (p < 0) return;
    const int step = p / kStepTokens + static_cast<int>(blockIdx.y), tok0 = step * kStepTokens;
    TreePlace place{};
    int end = p + a.n;
    if constexpr (kTree) {
        place = tree_place(tree.parents + b * a.n, a.n, lane);
        end = p + __popcll(__ballot(place.live));
    }
    if (tok0 >= end) return;
    uint8_t* const cells = step_cells(a.view, a.slot0 + b, a.layer, kh, step);
    if (cells == nullptr) return;
    const int64_t row0 = static_cast<int64_t>(b) * a.n;
    const T* const k = static_cast<const T*>(a.k) + kh * HD;
    const T* const v = static_cast<const T*>(a.v) + kh * HD;
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int item = it * kRowThreads + threadIdx.x, t = item / kChunks, chunk = item % kChunks;
        const int tok = tok0 + t;
        const bool fresh = tok >= p && tok < end;
        const int i = min(max(tok, p), end - 1) - p;         // (lanes without a row of their own take the nearest)
        int position = p + i;
        if constexpr (kTree) position = p + __popcll(from_lane(place.mask, i)) - 1;
        const Half8<T> kk = turned(k + (row0 + i) * a.k_stride, chunk, a.rotation, angles(a.rotation, position));
        const Half8<T> vv = *reinterpret_cast<const Half8<T>*>(v + (row0 + i) * a.v_stride + 8 * chunk);
        if (fresh) *reinterpret_cast<Half8<T>*>(cells + k_cell(t, chunk)) = kk;
        *reinterpret_cast<Half8<T>*>(rows + t * kPitch + 8 * chunk) = vv;
    }
    __syncthreads();
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int item = it * kRowThreads + threadIdx.x, octet = item / HD, channel = item % HD;
        const int first = tok0 + octet * 8;
        Half8<T> w;
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = rows[(octet * 8 + j) * kPitch + channel];
        uint8_t* const cell = cells + v_cell(octet, channel, HD);
        if (first >= p && first + 8 <= end) {
            *reinterpret_cast<Half8<T>*>(cell) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (first + j >= p && first + j < end) reinterpret_cast<T*>(cell)[j] = w[j];
        }
    }
}

// The reverse, with the same lanes (16-bit patterns of either type): workgroup
// (key/value head, step, layer and sequence).
template <int HD>
__global__ __launch_bounds__(kRowThreads) void paged_values_kernel(const PagedRowsArgs a, int batch) {
    using T = uint16_t;
    constexpr int kChunks = HD / 8, kItems = kStepTokens * kChunks / kRowThreads;
    constexpr int kPitch = HD + 8;
    __shared__ __align__(16) T rows[kStepTokens * kPitch];
    const int kh = blockIdx.x, b = blockIdx.z % batch, layer = blockIdx.z / batch;
    const int p = a.positions[b], end = p + a.n;
    if (p < 0) return;
    const int step = p / kStepTokens + static_cast<int>(blockIdx.y), tok0 = step * kStepTokens;
    if (tok0 >= end) return;
    const uint8_t* const cells = step_cells(a.view, a.slot0 + b, a.layer + layer, kh, step);
    if (cells == nullptr) return;
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int item = it * kRowThreads + threadIdx.x, octet = item / HD, channel = item % HD;
        const Vec8<T> w = *reinterpret_cast<const Vec8<T>*>(cells + v_cell(octet, channel, HD));
#pragma unroll
        for (int j = 0; j < 8; ++j) rows[(octet * 8 + j) * kPitch + channel] = w.v[j];
    }
    __syncthreads();
    const int64_t stride = static_cast<int64_t>(a.view.kv_heads) * HD;
    const int64_t row0 = layer * a.layer_rows + static_cast<int64_t>(b) * a.n - p;
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int item = it * kRowThreads + threadIdx.x, t = item / kChunks, chunk = item % kChunks;
        const int tok = tok0 + t;
        if (tok < p || tok >= end) continue;
        const int64_t at = (row0 + tok) * stride + kh * HD + 8 * chunk;
        *reinterpret_cast<Vec8<T>*>(static_cast<T*>(a.k_out) + at) = *reinterpret_cast<const Vec8<T>*>(cells + k_cell(t, chunk));
        *reinterpret_cast<Vec8<T>*>(static_cast<T*>(a.v_out) + at) = *reinterpret_cast<const Vec8<T>*>(rows + t * kPitch + 8 * chunk);
    }
}

// Workgroup (layer and key/value head, sequence): row accepted[j] goes to row j.  A
// row may be a source and a target, so all are read before any is written.
template <int HD, int ROWS>
__global__ __launch_bounds__(kRowThreads) void paged_keep_kernel(const PagedKeepArgs a) {
    constexpr int kChunks = HD / 8;
    constexpr int kCells = (ROWS * kChunks + kRowThreads - 1) / kRowThreads, kValues = ROWS * HD / kRowThreads;
    const int layer = a.layer0 + static_cast<int>(blockIdx.x) / a.view.kv_heads, kh = blockIdx.x % a.view.kv_heads;
    const int b = blockIdx.y, p = a.positions[b];
    if (p < 0) return;
    const uint8_t* const accepted = a.accepted + b * a.m;
    const int32_t* const table = a.view.table + static_cast<int64_t>(a.slot0 + b) * a.view.entries;
    // Cells of a token's step; its place in the step.
    auto cells_of = [&](int tok) -> uint8_t* {
        const int page = table[tok / kPageTokens];
        if (page < 0) return nullptr;
        return a.view.base + paged_record(a.view, layer, page, kh) + (tok / kStepTokens % kPageSteps) * paged_step_bytes(HD);
    };
    Vec8<uint16_t> k[kCells];
    uint16_t v[kValues];
    auto source = [&](int j) {       // of row j, or -1 where it stays
        const int from = j < a.m ? accepted[j] : 255;
        return from < kTreeTokens && from != j ? from : -1;
    };
    auto k_at = [&](uint8_t* cells, int tok, int chunk) {
        return reinterpret_cast<Vec8<uint16_t>*>(cells + k_cell(tok % kStepTokens, chunk));
    };
    auto v_at = [&](uint8_t* cells, int tok, int channel) {
        const int t = tok % kStepTokens;
        return reinterpret_cast<uint16_t*>(cells + v_cell(t / 8, channel, HD)) + t % 8;
    };
#pragma unroll
    for (int it = 0; it < kCells; ++it) {
        const int item = it * kRowThreads + threadIdx.x, j = item / kChunks, from = j < ROWS ? source(j) : -1;
        uint8_t* const cells = from < 0 ? nullptr : cells_of(p + from);
        if (cells != nullptr) k[it] = *k_at(cells, p + from, item % kChunks);
    }
#pragma unroll
    for (int it = 0; it < kValues; ++it) {
        const int item = it * kRowThreads + threadIdx.x, from = source(item / HD);
        uint8_t* const cells = from < 0 ? nullptr : cells_of(p + from);
        if (cells != nullptr) v[it] = *v_at(cells, p + from, item % HD);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // read, and not only asked for
    __syncthreads();
#pragma unroll
    for (int it = 0; it < kCells; ++it) {
        const int item = it * kRowThreads + threadIdx.x, j = item / kChunks;
        uint8_t* const cells = j < ROWS && source(j) >= 0 && cells_of(p + source(j)) != nullptr ? cells_of(p + j) : nullptr;
        if (cells != nullptr) *k_at(cells, p + j, item % kChunks) = k[it];
    }
#pragma unroll
    for (int it = 0; it < kValues; ++it) {
        const int item = it * kRowThreads + threadIdx.x, j = item / HD;
        uint8_t* const cells = source(j) >= 0 && cells_of(p + source(j)) != nullptr ? cells_of(p + j) : nullptr;
        if (cells != nullptr) *v_at(cells, p + j, item % HD) = v[it];
    }
}

// Every layer's records of one page: workgroups (layer, part).
constexpr int kCopyParts = 16;
__global__ __launch_bounds__(kRowThreads) void paged_copy_kernel(const PagedView v, int64_t from, int64_t to) {
    const int64_t bytes = v.kv_heads * paged_record_bytes(v.head_dim);
    const v4i* src = reinterpret_cast<const v4i*>(v.base + paged_record(v, blockIdx.x, from, 0));
    v4i* dst = reinterpret_cast<v4i*>(v.base + paged_record(v, blockIdx.x, to, 0));
    for (int64_t i = blockIdx.y * kRowThreads + threadIdx.x; i < bytes / 16; i += kCopyParts * kRowThreads) dst[i] = src[i];
}

template <typename F>
void with_half(ElementType t, F&& f) {
    if (t == kBF16) f(__bf16{});
    else f(_Float16{});
}

int touched_steps(int n) { return (n + 2 * kStepTokens - 2) / kStepTokens; }

}  // namespace

hipError_t launch_paged_map(const PagedMapArgs& a, hipStream_t s) {
    paged_map_kernel<<<1, kMapEntries, 0, s>>>(a);
    return hipGetLastError();
}

hipError_t launch_paged_append(const PagedRowsArgs& a, const PagedTree* tree, int batch, ElementType t, hipStream_t s) {
    const dim3 grid(a.view.kv_heads, touched_steps(a.n), batch);
    with_half(t, [&](auto tag) {
        using T = decltype(tag);
        if (tree && a.view.head_dim == 64) paged_append_kernel<T, 64><<<grid, kRowThreads, 0, s>>>(a, *tree);
        else if (tree) paged_append_kernel<T, 128><<<grid, kRowThreads, 0, s>>>(a, *tree);
        else if (a.view.head_dim == 64) paged_append_kernel<T, 64><<<grid, kRowThreads, 0, s>>>(a, PagedChain{});
        else paged_append_kernel<T, 128><<<grid, kRowThreads, 0, s>>>(a, PagedChain{});
    });
    return hipGetLastError();
}

hipError_t launch_paged_values(const PagedRowsArgs& a, int layers, int batch, hipStream_t s) {
    const dim3 grid(a.view.kv_heads, touched_steps(a.n), layers * batch);
    if (a.view.head_dim == 64) paged_values_kernel<64><<<grid, kRowThreads, 0, s>>>(a, batch);
    else paged_values_kernel<128><<<grid, kRowThreads, 0, s>>>(a, batch);
    return hipGetLastError();
}

hipError_t launch_paged_keep(const PagedKeepArgs& a, int layers, int batch, hipStream_t s) {
    const dim3 grid(layers * a.view.kv_heads, batch);
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (a.m <= 8) paged_keep_kernel<HD, 8><<<grid, kRowThreads, 0, s>>>(a);
        else paged_keep_kernel<HD, kTreeTokens><<<grid, kRowThreads, 0, s>>>(a);
    };
    if (a.view.head_dim == 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, 128>{});
    return hipGetLastError();
}

hipError_t launch_paged_copy(const PagedView& v, int64_t from, int64_t to, hipStream_t s) {
    paged_copy_kernel<<<dim3(v.layers, kCopyParts), kRowThreads, 0, s>>>(v, from, to);
    return hipGetLastError();
}

}  // namespace swiftkv
