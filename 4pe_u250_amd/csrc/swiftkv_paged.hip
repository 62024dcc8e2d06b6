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
        place = tree_place(tree.parents, b, a.n, lane);
        end = p + __popcll(__ballot(place.live));
    }
    if (!step_has_new(tok0, p, end)) return;
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
        const int i = nearest_row(tok, p, end);
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

// The reverse (16-bit patterns of either type): workgroup (HEADS key/value heads of a
// layer, window of OCTETS octets of tokens, sequence).  All loads of a thread go out
// before the first is waited for, and of few tokens a workgroup takes four heads' where
// that leaves enough of them: 8 tokens of 64 sequences, 32 layers and 8 heads 37 us a
// launch (49 with one head and step a workgroup and K's loads behind V's transposition),
// for which the cells' lines bound it: a token's K is 16 bytes of 16 lines, an octet's V
// 2 KiB.  A prompt of 4095 tokens and 32 heads 21 us, 6.3 TB/s read and written.
template <int HD, int OCTETS, int HEADS>
__global__ __launch_bounds__(kRowThreads) void paged_values_kernel(const PagedRowsArgs a, int batch) {
    using T = uint16_t;
    typedef T Eight __attribute__((ext_vector_type(8)));
    constexpr int kChunks = HD / 8, kTokens = 8 * OCTETS, kItems = HEADS * OCTETS * HD / kRowThreads;
    constexpr int kPitch = HD + 8;
    static_assert(HEADS * OCTETS * HD % kRowThreads == 0 && HD % 64 == 0 && 8 % (64 / kChunks) == 0, "a wave's items are of one octet");
    __shared__ __align__(16) T rows[HEADS * kTokens * kPitch];
    const int kh0 = blockIdx.x * HEADS, b = blockIdx.z % static_cast<uint32_t>(batch), layer = blockIdx.z / static_cast<uint32_t>(batch);
    const int p = a.positions[b], end = p + a.n;
    if (p < 0) return;
    const int octet0 = p / 8 + static_cast<int>(blockIdx.y) * OCTETS;
    if (octet0 * 8 >= end) return;
    // Item it * kRowThreads + thread: head, octet, and a channel of V or a token and chunk of
    // K.  (What lies behind the last token takes that one's place, and is not written.)
    const uint32_t wave0 = __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u), lane = threadIdx.x & 63, chunk = lane % kChunks;
    const int32_t* const table = a.view.table + static_cast<int64_t>(a.slot0 + b) * a.view.entries;
    const int64_t page_bytes = a.view.kv_heads * paged_record_bytes(HD);
    const uint8_t* const head0 = a.view.base + paged_record(a.view, a.layer + layer, 0, kh0);
    auto token_of = [&](int it) { return octet0 * 8 + static_cast<int>((it * kRowThreads + wave0 + lane) / kChunks % kTokens); };
    Eight kk[kItems], vv[kItems];
    int page[kItems];
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const uint32_t first = it * kRowThreads + wave0, head = first / (OCTETS * HD);
        const int octet = min(octet0 + static_cast<int>(first / HD % OCTETS), (end - 1) / 8);
        page[it] = table[octet * 8 / kPageTokens];
        const uint8_t* const cells = head0 + head * paged_record_bytes(HD) + max(page[it], 0) * page_bytes + octet * 8 / kStepTokens % kPageSteps * paged_step_bytes(HD);
        kk[it] = *reinterpret_cast<const Eight*>(cells + k_cell(min(max(token_of(it), p), end - 1) % kStepTokens, chunk));
        vv[it] = *reinterpret_cast<const Eight*>(cells + v_cell(octet % 4, first % HD + lane, HD));
    }
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const uint32_t item = it * kRowThreads + threadIdx.x;
#pragma unroll
        for (int j = 0; j < 8; ++j) rows[(item / HD * 8 + j) * kPitch + item % HD] = vv[it][j];
    }
    __syncthreads();
    const int64_t stride = static_cast<int64_t>(a.view.kv_heads) * HD;
    const int64_t row0 = layer * a.layer_rows + static_cast<int64_t>(b) * a.n - p;
#pragma unroll
    for (int it = 0; it < kItems; ++it) {
        const int tok = token_of(it), head = (it * kRowThreads + wave0) / (OCTETS * HD);
        if (page[it] < 0 || tok < p || tok >= end) continue;
        const int64_t at = (row0 + tok) * stride + (kh0 + head) * HD + 8 * chunk;
        *reinterpret_cast<Eight*>(static_cast<T*>(a.k_out) + at) = kk[it];
        *reinterpret_cast<Eight*>(static_cast<T*>(a.v_out) + at) =
            *reinterpret_cast<const Eight*>(rows + (head * kTokens + tok - octet0 * 8) * kPitch + 8 * chunk);
    }
}

// Workgroup (layer and `heads` key/value heads, sequence): row accepted[j] goes to row j.
// A row may be a source and a target, so all are read, into LDS, before any is written.  K
// moves by its cells, V by whole target cells, each of whose 8 tokens comes from its source
// or from where it is.  Few instructions count here more than few loads: a workgroup runs
// each once, and unrolled forms of this spent 13 us a launch on fetching them.
template <int HD, int ROWS>
__global__ __launch_bounds__(kRowThreads) void paged_keep_kernel(const PagedKeepArgs a, int heads) {
    constexpr int kChunks = HD / 8, kOctets = (ROWS + 14) / 8, kHeads = ROWS <= 8 ? 4 : 1;
    constexpr int64_t kRecord = 2 * kStepTokens * 2 * 2 * HD;        // between two heads
    __shared__ __align__(16) Vec8<uint16_t> held[kHeads * (ROWS * kChunks + kOctets * HD)];
    // Of token 8 (p / 8) + s: the K cells and V values that go there, from the layer's first
    // head on, and its own; whether a row comes to its octet.
    __shared__ int64_t k_from[kOctets * 8], k_to[kOctets * 8], v_from[kOctets * 8], v_to[kOctets * 8];
    __shared__ int comes[kOctets];
    const int parts = a.view.kv_heads / heads, layer = a.layer0 + static_cast<int>(blockIdx.x) / parts;
    const int kh0 = static_cast<int>(blockIdx.x) % parts * heads, b = blockIdx.y, p = a.positions[b], tid = threadIdx.x;
    if (p < 0) return;
    const int tok0 = p & ~7, octets = (p - tok0 + a.m + 7) / 8;
    if (tid < kOctets) comes[tid] = 0;
    const uint32_t accepted = tree_byte(a.accepted, b, a.m, (tok0 + tid - p) & (kTreeTokens - 1));
    __syncthreads();
    if (tid < octets * 8) {
        const int32_t* const table = a.view.table + static_cast<int64_t>(a.slot0 + b) * a.view.entries;
        const int64_t page_bytes = a.view.kv_heads * paged_record_bytes(HD);
        const int to = tok0 + tid, j = to - p, from = j >= 0 && j < a.m && accepted < kTreeTokens ? p + static_cast<int>(accepted) : to;
        const int page = table[min(from / kPageTokens, a.view.entries - 1)], to_page = table[min(to / kPageTokens, a.view.entries - 1)];
        const bool moves = from != to && page >= 0 && to_page >= 0;
        auto step_of = [&](int64_t on, int tok) { return on * page_bytes + tok / kStepTokens % kPageSteps * paged_step_bytes(HD); };
        auto key = [&](int tok) { return k_cell(tok % kStepTokens, 0); };
        auto value = [&](int tok) { return v_cell(tok % kStepTokens / 8, 0, HD); };
        k_from[tid] = moves ? step_of(page, from) + key(from) : -1;
        k_to[tid] = step_of(max(to_page, 0), to) + key(to);
        v_from[tid] = moves ? step_of(page, from) + value(from) + 2 * (from % 8) : step_of(max(to_page, 0), to) + value(to) + 2 * (to % 8);
        v_to[tid] = step_of(max(to_page, 0), to) + value(to);
        if (moves) comes[tid / 8] = 1;
    }
    __syncthreads();
    uint8_t* const base = a.view.base + paged_record(a.view, layer, 0, kh0);
    const int keys = a.m * kChunks, cells = octets * HD;
    Vec8<uint16_t>* const held_v = held + kHeads * ROWS * kChunks;
    auto key_at = [&](int item) { return item / keys * kRecord + k_cell(0, item % kChunks); };
    auto value_at = [&](int item) { return item / cells * kRecord + (item % HD >> 4) * 1024 + (item % HD & 15) * 16; };
    const int skip = p - tok0;
#pragma unroll 1
    for (int item = tid; item < heads * keys; item += kRowThreads) {
        const int64_t from = k_from[skip + item % keys / kChunks];
        if (from >= 0) held[item] = *reinterpret_cast<const Vec8<uint16_t>*>(base + from + key_at(item));
    }
#pragma unroll 1
    for (int item = tid; item < heads * cells; item += kRowThreads) {
        const int octet = item % cells / HD;
        if (!comes[octet]) continue;
        Vec8<uint16_t> w;
#pragma unroll
        for (int e = 0; e < 8; ++e) w.v[e] = *reinterpret_cast<const uint16_t*>(base + v_from[octet * 8 + e] + value_at(item));
        held_v[item] = w;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // read, and not only asked for
    __syncthreads();
#pragma unroll 1
    for (int item = tid; item < heads * keys; item += kRowThreads) {
        const int s = skip + item % keys / kChunks;
        if (k_from[s] >= 0) *reinterpret_cast<Vec8<uint16_t>*>(base + k_to[s] + key_at(item)) = held[item];
    }
#pragma unroll 1
    for (int item = tid; item < heads * cells; item += kRowThreads) {
        const int octet = item % cells / HD;
        if (comes[octet]) *reinterpret_cast<Vec8<uint16_t>*>(base + v_to[octet * 8] + value_at(item)) = held_v[item];
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

// (layer, key/value head, sequence) triples from which a workgroup takes four heads' few rows.
constexpr int kManyHeads = 4096;
int heads_of(const PagedView& v, int layers, int batch) {
    return v.kv_heads % 4 == 0 && layers * v.kv_heads * batch >= kManyHeads ? 4 : 1;
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
    auto go = [&](auto octets, auto heads) {
        constexpr int OCTETS = decltype(octets)::value, HEADS = decltype(heads)::value;
        const dim3 grid(a.view.kv_heads / HEADS, (a.n + 6 + 8 * OCTETS) / (8 * OCTETS), layers * batch);
        if (a.view.head_dim == 64) paged_values_kernel<64, OCTETS, HEADS><<<grid, kRowThreads, 0, s>>>(a, batch);
        else paged_values_kernel<128, OCTETS, HEADS><<<grid, kRowThreads, 0, s>>>(a, batch);
    };
    using std::integral_constant;
    if (a.n <= 9 && heads_of(a.view, layers, batch) == 4) go(integral_constant<int, 2>{}, integral_constant<int, 4>{});
    else go(integral_constant<int, 4>{}, integral_constant<int, 1>{});
    return hipGetLastError();
}

hipError_t launch_paged_keep(const PagedKeepArgs& a, int layers, int batch, hipStream_t s) {
    const int heads = a.m <= 8 ? heads_of(a.view, layers, batch) : 1;
    const dim3 grid(layers * (a.view.kv_heads / heads), batch);
    auto go = [&](auto hd) {
        constexpr int HD = decltype(hd)::value;
        if (a.m <= 8) paged_keep_kernel<HD, 8><<<grid, kRowThreads, 0, s>>>(a, heads);
        else paged_keep_kernel<HD, kTreeTokens><<<grid, kRowThreads, 0, s>>>(a, heads);
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
