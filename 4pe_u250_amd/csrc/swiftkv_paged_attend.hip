// swiftkv_paged_attend.hip -- attention over the paged cache where a (sequence,
// key/value head) has few rows, and the join of splits.
#include "swiftkv_paged_attend_device.hpp"

namespace swiftkv {
namespace {

using namespace dev;

constexpr int kAttendThreads = 256;
constexpr int kWaves = 4;
static_assert(kSplitQuantumSteps % kWaves == 0, "a split is whole turns of the waves");

// What one workgroup tells another, 8 bytes at a time: write-through stores, loads
// past the caches.
__device__ __forceinline__ void publish2(float* p, float x, float y) {
    __hip_atomic_store(reinterpret_cast<uint64_t*>(p), static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ v2f fetch2(const float* p) {
    const uint64_t w = __hip_atomic_load(const_cast<uint64_t*>(reinterpret_cast<const uint64_t*>(p)), __ATOMIC_RELAXED,
                                         __HIP_MEMORY_SCOPE_AGENT);
    return v2f{__uint_as_float(static_cast<uint32_t>(w)), __uint_as_float(static_cast<uint32_t>(w >> 32))};
}

// ROWS = R * RT rows of a (sequence, key/value head) over the steps of one split.  Reading
// the cells bounds it: each wave takes steps w, w + 4, ... and loads their cells as
// operands, 1 KiB of consecutive bytes an instruction, K of the next step during the softmax
// and V after the products, as registers fall free; with RT > 1 each serves RT tiles of
// rows.  The waves meet in LDS.  One token of 64 sequences at 4096 170 us, 6.3 TB/s of
// K and V; 64 rows of each 195 us, 5.5 TB/s.  Where chunks share the cells, what a CU's loads
// deliver bounds it: 512 tokens onto 4095 54 us and 0.68 PFLOP/s with 64 rows, 59 with 32.
//
// ONCE: no other workgroup reads the cells, and they pass the caches (one token of 64
// sequences 170 us, 16 tokens 194; kept in the caches 185 and 204); if others do they stay (512
// tokens 53.7 us, passing the caches 54.5; 64 tokens of 8 sequences 56.6 and 70).
//
// 16 rows: a sequence's splits publish (m, l, sums), wait until that has arrived, and
// count themselves; the last to arrive joins all in split order, so the result does not
// depend on who that is.  The partial results of more rows are joined by a launch of
// paged_join_kernel, whose workgroups share the rows out (26 tokens onto 4095: 4.0 us of 15.8).
template <typename T, int HD, int R, int RT, bool ONCE, typename Tree>
__global__ __launch_bounds__(kAttendThreads, 2) void paged_attend_kernel(const PagedAttendArgs a, const Tree tree) {
    using Tile = RowTile<T, HD, R, R * RT == 16>;
    constexpr int ROWS = R * RT, THREADS = kAttendThreads;
    using S = Share<ROWS, Tree>;
    constexpr int NL = Tile::NL, CG = HD / 4, kPitch = HD + 8;
    constexpr int kPolicy = ONCE ? 2 : 0;        // 2: nontemporal
    constexpr int kStepBytes = 2 * kStepTokens * HD * 2;
    __shared__ __align__(16) v4f lds[kWaves * CG * (ROWS + 1)];     // queries, then the waves' sums
    __shared__ float stats[kWaves][ROWS][2];
    __shared__ uint32_t arrived;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane / R, place = lane % R;
    S share;
    share.start(a, tree, lane);
    if (share.split >= share.my_splits) return;
    const int b = share.b, kh = share.kh, p = share.p, step_begin = share.step_begin, step_end = share.step_end;

    // The pages of 64 of the wave's steps, one in each lane (a lane past its last step
    // asks for that one's).
    const int32_t* const table = a.view.table + static_cast<int64_t>(a.slot0 + b) * a.view.entries;
    int pages = 0;
    auto load_pages = [&](int step) { pages = table[max(0, min(step + lane * kWaves, step_end - 1)) / kPageSteps]; };
    load_pages(step_begin + wave);
    uint8_t* const layer_head = a.view.base + paged_record(a.view, a.layer, 0, kh);
    const int64_t page_bytes = a.view.kv_heads * paged_record_bytes(HD);

    // The call's rows are appended by every workgroup that scans them, with the same bytes:
    // its own writes are what it finds then.
    if (a.k != nullptr) share.template append<T, HD, THREADS>(a, table, layer_head, page_bytes, wave, lane);

    T* const staged = reinterpret_cast<T*>(lds);
    share.template stage_queries<T, HD, THREADS>(a, staged);
    __syncthreads();
    Tile tiles[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        tiles[rt].clear();
        share.sees(a, tiles[rt], rt * R + place);
#pragma unroll
        for (int s = 0; s < Tile::NS; ++s)
            tiles[rt].q[s] = *reinterpret_cast<const Half8<T>*>(staged + (rt * R + place) * kPitch + (s * Tile::G + g) * 8);
    }

    const int k_lane = R == 16 ? lane * 16 : (((place >> 3) & 1) * 64 + g * 16 + (place >> 4) * 8 + ((place >> 2) & 1) * 4 + (place & 3)) * 16;
    const int v_lane = R == 16 ? lane * 16 : ((place >> 4) * 64 + g * 16 + (place & 15)) * 16;
    auto cell_at = [](int l) { return R == 16 ? l * 1024 : ((l >> 1) * 128 + (l & 1) * 32) * 16; };
    Half8<T> kb[NL], vb[NL];
    auto cells_of = [&](int step, int at) {
        return step_resource(layer_head, page_bytes, __builtin_amdgcn_readlane(pages, at), step, step_end, kStepBytes);
    };
    // (offsets up to 4095 travel in the instruction)
    auto load = [&](__amdgpu_buffer_rsrc_t cells, int lane_at, int at) {
        return __builtin_bit_cast(Half8<T>, __builtin_amdgcn_raw_buffer_load_b128(cells, lane_at + (at & 4095), at & ~4095, kPolicy));
    };
    auto load_k = [&](__amdgpu_buffer_rsrc_t cells) {
#pragma unroll
        for (int i = 0; i < NL; ++i) kb[i] = load(cells, k_lane, cell_at(i));
    };
    auto load_v = [&](__amdgpu_buffer_rsrc_t cells) {
#pragma unroll
        for (int i = 0; i < NL; ++i) vb[i] = load(cells, v_lane, kStepBytes / 2 + cell_at(i));
    };
    // The scores of a step are formed while the weights of the one before are.
    int step = step_begin + wave, at = 0, again = step_end;     // the step from which V has to be looked at again
    float s[RT][Tile::NV];
    __amdgpu_buffer_rsrc_t next = cells_of(step, 0);
    auto seen = [&](const Tile& tile, int st) { return st < step_end ? tile.seen(st, g) : 0u; };
    auto turn_pages = [&]() {
        if (__builtin_expect(++at == 64, 0)) {
            load_pages(step + 2 * kWaves);
            at = 0;
        }
    };
    if (step < step_end) {
        load_k(next);
        load_v(next);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            const uint32_t bits = seen(tiles[rt], step);
            tiles[rt].scores(kb, s[rt]);
            tiles[rt].hide(bits, s[rt]);
            tiles[rt].rise(s[rt], a);
        }
        next = cells_of(step + kWaves, ++at);
        load_k(next);
    }
    auto run = [&](auto masked, int end) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        for (; step < end; step += kWaves) {
            turn_pages();
            const __amdgpu_buffer_rsrc_t after = cells_of(step + 2 * kWaves, at);
            float sn[RT][Tile::NV];
            Half8<T> w[RT][Tile::TERMS][Tile::NP];
            uint32_t bits[RT];
            if constexpr (kMasked)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) bits[rt] = seen(tiles[rt], step + kWaves);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) tiles[rt].scores(kb, sn[rt]);
            load_k(after);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) tiles[rt].weights(s[rt], a.scale, w[rt]);
            if constexpr (kMasked)
                if (__builtin_expect(Tile::no_numbers(vb), 0)) {
                    again = min(again, step);
                    Tile::clean(vb);
                }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) tiles[rt].add(vb, w[rt]);
            load_v(next);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if constexpr (kMasked) tiles[rt].hide(bits[rt], sn[rt]);
                tiles[rt].rise(sn[rt], a);
            }
            next = after;
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int i = 0; i < Tile::NV; ++i) s[rt][i] = sn[rt][i];
        }
    };
    run(std::false_type{}, share.plain_end - kWaves);
    run(std::true_type{}, step_end);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
        if (tiles[rt].no_number_sums()) again = step_begin + wave;
    if (__builtin_expect(again < step_end, 0))
        look_again<kWaves>(tiles, vb, again, step_end, g, [&](int st, Half8<T> (&x)[NL]) __attribute__((always_inline)) {
            const int page = __builtin_amdgcn_readfirstlane(table[st / kPageSteps]);
            const __amdgpu_buffer_rsrc_t cells = step_resource(layer_head, page_bytes, page, st, step_end, kStepBytes);
#pragma unroll
            for (int i = 0; i < NL; ++i) x[i] = load(cells, v_lane, kStepBytes / 2 + cell_at(i));
        });

    __syncthreads();                             // everyone has its queries
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = Tile::groups_sum(tiles[rt].l);
        if (g == 0) {
            stats[wave][rt * R + place][0] = tiles[rt].reference();
            stats[wave][rt * R + place][1] = sum;
        }
        tiles[rt].leave(lds + wave * CG * (ROWS + 1), ROWS + 1, rt * R + place, g);
    }
    __syncthreads();
    constexpr int kItems = ROWS * CG / THREADS;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int item = threadIdx.x + k * THREADS, row = item / CG, quad = item % CG;
        v2f ml[kWaves];
        v4f sums[kWaves];
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            ml[w] = v2f{stats[w][row][0], stats[w][row][1]};
            sums[w] = lds[(w * CG + quad) * (ROWS + 1) + row];
        }
        Joined all;
        all.add(ml, sums, a.scale);
        float* const dst = share.template partial<HD>(a, share.split);
        if (share.my_splits == 1) {
            share.template finish<T, HD>(a, row, quad, all.l, all.o);
        } else if (ROWS == 16) {
            if (quad == 0) publish2(dst + row * 2, all.m, all.l);
            publish2(dst + ROWS * 2 + row * HD + quad * 4, all.o[0], all.o[1]);
            publish2(dst + ROWS * 2 + row * HD + quad * 4 + 2, all.o[2], all.o[3]);
        } else {
            if (quad == 0) *reinterpret_cast<v2f*>(dst + row * 2) = v2f{all.m, all.l};
            *reinterpret_cast<v4f*>(dst + ROWS * 2 + row * HD + quad * 4) = all.o;
        }
    }
    if constexpr (ROWS == 16) {
        if (share.my_splits == 1) return;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // what was published has arrived
        __syncthreads();
        uint32_t* const counter = a.counters + (static_cast<int64_t>(b) * a.view.kv_heads + kh) * kCounterStride;
        if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (static_cast<int>(arrived) != share.my_splits - 1) return;
        // The last split joins everybody's, eight of all items' loads at a time; the counter
        // is zero again.
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        constexpr int kAtOnce = 8;
        Joined all[kItems];
        for (int j0 = 0; j0 < share.my_splits; j0 += kAtOnce) {
            v2f ml[kItems][kAtOnce];
            v4f sums[kItems][kAtOnce];
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
                const int item = threadIdx.x + k * kAttendThreads, row = min(item / CG, share.rows - 1), quad = item % CG;
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const float* src = share.template partial<HD>(a, min(j0 + j, share.my_splits - 1));
                    ml[k][j] = fetch2(src + row * 2);
                    const v2f low = fetch2(src + ROWS * 2 + row * HD + quad * 4), high = fetch2(src + ROWS * 2 + row * HD + quad * 4 + 2);
                    sums[k][j] = v4f{low[0], low[1], high[0], high[1]};
                }
            }
#pragma unroll
            for (int k = 0; k < kItems; ++k) {
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j)
                    if (j0 + j >= share.my_splits) ml[k][j] = v2f{-INFINITY, 0.0f}, sums[k][j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
                all[k].add(ml[k], sums[k], a.scale);
            }
        }
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int item = threadIdx.x + k * kAttendThreads;
            share.template finish<T, HD>(a, item / CG, item % CG, all[k].l, all[k].o);
        }
    }
}

// Splits of chunks of ROWS rows joined in split order: workgroup (a few rows, chunk and
// key/value head; sequence), a quad of channels a thread, four or eight splits' loads at a time.
template <typename T, int HD, int ROWS, typename Tree>
__global__ __launch_bounds__(kAttendThreads) void paged_join_kernel(const PagedAttendArgs a, const Tree tree) {
    constexpr int CG = HD / 4, kRows = kAttendThreads / CG, kAtOnce = ROWS < 64 ? 8 : 4;
    Share<ROWS, Tree> share;
    // (heads fastest, as the workgroups that left the partial results)
    const int kh = blockIdx.x % a.view.kv_heads, id = blockIdx.x / a.view.kv_heads, part = id % (ROWS / kRows);
    share.start(a, tree, blockIdx.y, kh + id / (ROWS / kRows) * a.view.kv_heads * a.splits, a.splits, threadIdx.x & 63);
    const int row = part * kRows + threadIdx.x / CG, quad = threadIdx.x % CG;
    if (share.my_splits == 1 || row >= share.rows) return;
    Joined all;
    for (int j0 = 0; j0 < share.my_splits; j0 += kAtOnce) {
        v2f ml[kAtOnce];
        v4f sums[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
            const float* src = share.template partial<HD>(a, min(j0 + j, share.my_splits - 1));
            ml[j] = *reinterpret_cast<const v2f*>(src + row * 2);
            sums[j] = *reinterpret_cast<const v4f*>(src + ROWS * 2 + row * HD + quad * 4);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (j0 + j >= share.my_splits) ml[j] = v2f{-INFINITY, 0.0f}, sums[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        all.add(ml, sums, a.scale);
    }
    share.template finish<T, HD>(a, row, quad, all.l, all.o);
}

template <typename F>
void with_shape(const PagedAttendArgs& a, ElementType t, F&& f) {
    using std::integral_constant;
    auto sized = [&](auto tag) {
        if (a.view.head_dim == 64) f(tag, integral_constant<int, 64>{});
        else f(tag, integral_constant<int, 128>{});
    };
    if (t == kBF16) sized(__bf16{});
    else sized(_Float16{});
}

}  // namespace

hipError_t launch_paged_attend(const PagedAttendArgs& a, const PagedTree* tree, int batch, int rows, ElementType t, hipStream_t s) {
    const dim3 grid = a.all_splits ? dim3(a.view.kv_heads * a.chunks * a.all_splits) : dim3(a.view.kv_heads * a.chunks * a.splits, batch);
    with_shape(a, t, [&](auto tag, auto hd) {
        using T = decltype(tag);
        constexpr int HD = decltype(hd)::value;
        auto go = [&](auto r, auto rt, auto once) {
            constexpr int R = decltype(r)::value, RT = decltype(rt)::value;
            constexpr bool ONCE = decltype(once)::value;
            if (tree) paged_attend_kernel<T, HD, R, RT, ONCE><<<grid, kAttendThreads, 0, s>>>(a, *tree);
            else paged_attend_kernel<T, HD, R, RT, ONCE><<<grid, kAttendThreads, 0, s>>>(a, PagedChain{});
        };
        using std::integral_constant;
        using std::true_type;
        using std::false_type;
        constexpr integral_constant<int, 1> one{};
        constexpr integral_constant<int, 2> two{};
        constexpr integral_constant<int, 3> three{};
        constexpr integral_constant<int, 16> narrow{};
        constexpr integral_constant<int, 32> wide{};
        if (rows == 16) go(narrow, one, true_type{});
        else if (rows == 48) go(narrow, three, true_type{});
        else if (rows == 32 && a.chunks == 1) go(wide, one, true_type{});
        else if (rows == 32) go(wide, one, false_type{});
        else if (a.chunks == 1) go(wide, two, true_type{});
        else go(wide, two, false_type{});
    });
    return hipGetLastError();
}

hipError_t launch_paged_join(const PagedAttendArgs& a, const PagedTree* tree, int batch, int rows, ElementType t, hipStream_t s) {
    with_shape(a, t, [&](auto tag, auto hd) {
        using T = decltype(tag);
        constexpr int HD = decltype(hd)::value;
        const dim3 grid(a.view.kv_heads * a.chunks * (rows / (kAttendThreads / (HD / 4))), batch);
        auto go = [&](auto r) {
            constexpr int ROWS = decltype(r)::value;
            if (tree) paged_join_kernel<T, HD, ROWS><<<grid, kAttendThreads, 0, s>>>(a, *tree);
            else paged_join_kernel<T, HD, ROWS><<<grid, kAttendThreads, 0, s>>>(a, PagedChain{});
        };
        if (rows == 32) go(std::integral_constant<int, 32>{});
        else if (rows == 48) go(std::integral_constant<int, 48>{});
        else if (rows == 64) go(std::integral_constant<int, 64>{});
        else if (rows == 128) go(std::integral_constant<int, 128>{});
        else go(std::integral_constant<int, 256>{});
    });
    return hipGetLastError();
}

}  // namespace swiftkv
