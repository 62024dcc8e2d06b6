// swiftkv_paged_many.hip -- attention over the paged cache where a (sequence,
// key/value head) has many rows: large trees, chunks of prompts.
#include "swiftkv_paged_attend_device.hpp"

namespace swiftkv {
namespace {

using namespace dev;

constexpr int kManyThreads = 512;
constexpr int kManyWaves = 8;

// A workgroup of eight waves: RW of them take 32 rows each, of the same steps, and
// TEAMS = 8 / RW such teams take steps of the split in turn.  Vector instructions and
// matrix products bound it, so a step's cells come from memory once for all rows of a
// team (as operands straight from memory they are bound by what a CU's loads deliver,
// 64 bytes a clock), straight into LDS, in the order in which the lanes of the
// 32x32x16 form read them.  A turn, one step of each team, forms the scores of the next
// step while it forms the weights of this one, so K lies one turn ahead of V.  Each has
// SLOTS slots: a turn asks for cells SLOTS - 1 turns ahead, into the slots that nobody
// reads in it, waits for those that it asked for SLOTS - 2 turns before, and ends with a
// barrier.  4096 tokens onto 4095 434 us, 0.95 PFLOP/s with 256 rows.
template <int HD, int RW>
struct ManyShape {
    static constexpr int TEAMS = kManyWaves / RW, ROWS = 32 * RW;
    static constexpr int kHalfBytes = kStepTokens * HD * 2;  // K or V of a step
    static constexpr int SLOTS = 3;
    static constexpr int kRing = 2 * SLOTS * TEAMS * kHalfBytes;
    static constexpr int kMerge = TEAMS * (HD / 4) * (ROWS + 1) * 16;
    static constexpr int kQueries = ROWS * (HD + 8) * 2;
    static constexpr int kBytes = kRing + kQueries > kMerge ? kRing + kQueries : kMerge;
};

template <typename T, int HD, int RW, typename Tree>
__global__ __launch_bounds__(kManyThreads, 2) void paged_many_kernel(const PagedAttendArgs a, const Tree tree) {
    using M = ManyShape<HD, RW>;
    using Tile = RowTile<T, HD, 32>;
    constexpr int TEAMS = M::TEAMS, ROWS = M::ROWS, kHalfBytes = M::kHalfBytes, kStepBytes = 2 * kHalfBytes;
    constexpr int NL = Tile::NL, CG = HD / 4, kPitch = HD + 8;
    constexpr int SLOTS = M::SLOTS, NH = TEAMS * 2 * NL / kManyWaves;    // a wave's loads of a turn
    static_assert(NH >= 1 && TEAMS * 2 * NL % kManyWaves == 0, "a turn's loads are shared evenly");
    __shared__ __align__(16) uint8_t lds[M::kBytes];
    __shared__ float stats[TEAMS][ROWS][2];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane / 32, place = lane % 32, row = wave % RW * 32 + place, team = wave / RW;
    Share<ROWS, Tree> share;
    share.start(a, tree, lane);
    if (share.split >= share.my_splits) return;
    const int step_begin = share.step_begin, step_end = share.step_end;

    // The pages of 64 steps from `window` on, one in each lane, and of the 64 after them.
    const int32_t* const table = a.view.table + static_cast<int64_t>(a.slot0 + share.b) * a.view.entries;
    auto pages_from = [&](int step) { return table[max(0, min(step + lane, step_end - 1)) / kPageSteps]; };
    int window = step_begin, pages = pages_from(step_begin), pages_next = pages_from(step_begin + 64);
    uint8_t* const layer_head = a.view.base + paged_record(a.view, a.layer, 0, share.kh);
    const int64_t page_bytes = a.view.kv_heads * paged_record_bytes(HD);

    // A wave's loads of a turn: NH of its 1 KiB blocks, first the teams' K, then their V.
    // Product x of K reads, with lane (g', 16 m' + 8 h + m''), cell [x / 2][h][2 (x & 1) + g'][8 m' + m''];
    // product (c / 2, x & 1) of V, with lane (g', 16 (c & 1) + m), cell [c][2 (x & 1) + g'][m].
    const int k_lane = (((place >> 3) & 1) * 64 + g * 16 + (place >> 4) * 8 + (place & 7)) * 16;
    const int v_lane = ((place >> 4) * 64 + g * 16 + (place & 15)) * 16;
    auto load_turn = [&](int k_step, int v_step, int k_slot, int v_slot) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            const int block = i * kManyWaves + wave, of_kind = block % (TEAMS * NL), of_step = of_kind % NL;
            const bool is_v = block >= TEAMS * NL;
            const int step = (is_v ? v_step : k_step) + of_kind / NL, at = step - window;    // below 128: the window follows K
            const int page = at < 64 ? __builtin_amdgcn_readlane(pages, max(at, 0)) : __builtin_amdgcn_readlane(pages_next, min(at - 64, 63));
            uint8_t* const to = lds + ((is_v ? SLOTS + v_slot : k_slot) * TEAMS * NL + of_kind) * 1024;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(step_resource(layer_head, page_bytes, page, step, step_end, kStepBytes),
                                                     reinterpret_cast<__attribute__((address_space(3))) void*>(reinterpret_cast<uintptr_t>(to)), 16,
                                                     is_v ? v_lane : k_lane, (is_v ? kHalfBytes : 0) + (of_step >> 1) * 2048 + (of_step & 1) * 512, 0, 0);
        }
    };
    auto k_cells = [&](int slot) { return lds + (slot * TEAMS + team) * kHalfBytes + lane * 16; };
    auto v_cells = [&](int slot) { return lds + ((SLOTS + slot) * TEAMS + team) * kHalfBytes + lane * 16; };

    // K lies one turn ahead of V.
    auto load_first = [&]() __attribute__((always_inline)) {
#pragma unroll
        for (int t = 0; t < SLOTS; ++t)
            load_turn(step_begin + t * TEAMS, t == 0 ? step_end : step_begin + (t - 1) * TEAMS, t, t == 0 ? SLOTS - 1 : t - 1);
    };
    // A tree's rows (a few steps) are appended by every workgroup that reads them, with the
    // same bytes: its own writes are what it finds then.
    const bool late = a.k != nullptr && share.p >= 0 && (step_begin + SLOTS * TEAMS) * kStepTokens > share.p;
    if (!late) load_first();
    if (a.k != nullptr) share.template append<T, HD, kManyThreads>(a, table, layer_head, page_bytes, wave, lane);
    T* const staged = reinterpret_cast<T*>(lds + M::kRing);
    share.template stage_queries<T, HD, kManyThreads>(a, staged);
    __syncthreads();
    Tile tiles[1];
    Tile& tile = tiles[0];
    tile.clear();
    share.sees(a, tile, row);
#pragma unroll
    for (int s = 0; s < Tile::NS; ++s) tile.q[s] = *reinterpret_cast<const Half8<T>*>(staged + row * kPitch + (s * 2 + g) * 8);
    if (late) load_first();
    // All but the last `left` turns' loads are there, for everyone.
    auto arrive = [&](auto left) __attribute__((always_inline)) {
        constexpr int N = decltype(left)::value * NH;
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    using std::integral_constant;
    auto operands = [&](Half8<T> (&x)[NL], const uint8_t* cells) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < NL; ++i) x[i] = *reinterpret_cast<const Half8<T>*>(cells + i * 1024);
    };
    auto seen = [&](int st) { return st < step_end ? tile.seen(st, g) : 0u; };
    float s[Tile::NV], s1[Tile::NV];
    arrive(integral_constant<int, SLOTS - 1>{});
    {
        const uint32_t bits = seen(step_begin + team);
        Half8<T> kb[NL];
        operands(kb, k_cells(0));
        tile.scores(kb, s);
        tile.hide(bits, s);
        tile.rise(s, a);
    }
    arrive(integral_constant<int, SLOTS - 2>{});

    // Slots of this turn's V and the next turn's K, and of what this turn asks for.
    int step0 = step_begin, v_slot = 0, k_slot = 1;
    int again = step_end;                        // the step from which V has to be looked at again
    // One turn: weights and sums of the scores `now`, scores `then` of the next.
    auto turn = [&](auto masked, const float (&now)[Tile::NV], float (&then)[Tile::NV]) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        const int step = step0 + team;
        const int k_free = k_slot == 0 ? SLOTS - 1 : k_slot - 1, v_free = v_slot == 0 ? SLOTS - 1 : v_slot - 1;
        load_turn(step0 + SLOTS * TEAMS, step0 + (SLOTS - 1) * TEAMS, k_free, v_free);
        if (!kMasked || step < step_end) {
            const uint32_t bits = kMasked ? seen(step + TEAMS) : 0u;
            Half8<T> kb[NL], vb[NL], w[Tile::TERMS][Tile::NP];
            operands(kb, k_cells(k_slot));
            operands(vb, v_cells(v_slot));
            tile.scores(kb, then);
            tile.weights(now, a.scale, w);
            if constexpr (kMasked)
                if (step >= share.plain_end && __builtin_expect(Tile::no_numbers(vb), 0)) {
                    again = min(again, step);
                    Tile::clean(vb);
                }
            tile.add(vb, w);
            if constexpr (kMasked) tile.hide(bits, then);
            tile.rise(then, a);
        }
        if (__builtin_expect(step0 + (SLOTS + 2) * TEAMS > window + 128, 0)) {
            window += 64;
            pages = pages_next;
            pages_next = pages_from(window + 64);
        }
        step0 += TEAMS;
        k_slot = k_slot == SLOTS - 1 ? 0 : k_slot + 1;
        v_slot = v_slot == SLOTS - 1 ? 0 : v_slot + 1;
        arrive(integral_constant<int, SLOTS - 2>{});
    };
    auto run = [&](auto masked, int end) __attribute__((always_inline)) {
        while (step0 < end) {                    // an even number of turns: a turn past the last does nothing
            turn(masked, s, s1);
            turn(masked, s1, s);
        }
    };
    run(std::false_type{}, share.plain_end - 3 * TEAMS + 1);
    run(std::true_type{}, step_end);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // nothing is on its way to LDS any more
    if (tile.no_number_sums()) again = step_begin + team;
    if (__builtin_expect(again < step_end, 0)) {
        Half8<T> vb[NL];
        look_again<TEAMS>(tiles, vb, again, step_end, g, [&](int st, Half8<T> (&x)[NL]) __attribute__((always_inline)) {
            const int page = __builtin_amdgcn_readfirstlane(table[st / kPageSteps]);
            const __amdgpu_buffer_rsrc_t cells = step_resource(layer_head, page_bytes, page, st, step_end, kStepBytes);
#pragma unroll
            for (int i = 0; i < NL; ++i) {
                const int at = kHalfBytes + (i >> 1) * 2048 + (i & 1) * 512;
                x[i] = __builtin_bit_cast(Half8<T>, __builtin_amdgcn_raw_buffer_load_b128(cells, v_lane + (at & 4095), at & ~4095, 0));
            }
        });
    }
    __syncthreads();

    // The teams' sums meet in LDS, quads of channels of a row together.
    v4f* const quads = reinterpret_cast<v4f*>(lds);
    const float sum = Tile::groups_sum(tile.l);
    if (g == 0) {
        stats[team][row][0] = tile.reference();
        stats[team][row][1] = sum;
    }
    tile.leave(quads + team * CG * (ROWS + 1), ROWS + 1, row, g);
    __syncthreads();
    // A thread's quad of channels, of every kRows-th row.
    constexpr int kRows = kManyThreads / CG;
    const int quad = threadIdx.x % CG, row0 = threadIdx.x / CG;
    float* const dst = share.template partial<HD>(a, share.split);
    v4f* const sums_out = reinterpret_cast<v4f*>(dst + ROWS * 2 + row0 * HD + quad * 4);
#pragma unroll 2
    for (int k = 0; k < ROWS / kRows; ++k) {
        const int r = row0 + k * kRows;
        v2f ml[TEAMS];
        v4f sums[TEAMS];
#pragma unroll
        for (int w = 0; w < TEAMS; ++w) {
            ml[w] = v2f{stats[w][r][0], stats[w][r][1]};
            sums[w] = quads[(w * CG + quad) * (ROWS + 1) + r];
        }
        Joined all;
        if constexpr (TEAMS == 1) {
            all.m = ml[0][0];
            all.l = ml[0][1];
            all.o = sums[0];
        } else {
            all.add(ml, sums, a.scale);
        }
        if (share.my_splits == 1) {
            share.template finish<T, HD>(a, r, quad, all.l, all.o);
        } else if (r < share.rows) {
            if (quad == 0) *reinterpret_cast<v2f*>(dst + r * 2) = v2f{all.m, all.l};
            sums_out[k * (kRows * HD / 4)] = all.o;
        }
    }
}

}  // namespace

hipError_t launch_paged_many(const PagedAttendArgs& a, const PagedTree* tree, int batch, int rows, ElementType t, hipStream_t s) {
    using std::integral_constant;
    const dim3 grid = a.all_splits ? dim3(a.view.kv_heads * a.chunks * a.all_splits) : dim3(a.view.kv_heads * a.chunks * a.splits, batch);
    auto go = [&](auto tag, auto hd, auto rw) {
        using T = decltype(tag);
        constexpr int HD = decltype(hd)::value, RW = decltype(rw)::value;
        if (tree) paged_many_kernel<T, HD, RW><<<grid, kManyThreads, 0, s>>>(a, *tree);
        else paged_many_kernel<T, HD, RW><<<grid, kManyThreads, 0, s>>>(a, PagedChain{});
    };
    auto shaped = [&](auto tag, auto hd) {
        if (rows == 128) go(tag, hd, integral_constant<int, 4>{});
        else go(tag, hd, integral_constant<int, 8>{});
    };
    auto typed = [&](auto tag) {
        if (a.view.head_dim == 64) shaped(tag, integral_constant<int, 64>{});
        else shaped(tag, integral_constant<int, 128>{});
    };
    if (t == kBF16) typed(__bf16{});
    else typed(_Float16{});
    return hipGetLastError();
}

}  // namespace swiftkv
