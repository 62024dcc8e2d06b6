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
// 64 bytes a clock), through registers into LDS, in the order in which the lanes of the
// 32x32x16 form read them.  A turn, one step of each team, forms the scores of the next
// step while it forms the weights of this one, so K lies one turn ahead of V, each in
// two slots: what a turn reads nobody writes in it, and one barrier ends it.
template <int HD, int RW>
struct ManyShape {
    static constexpr int TEAMS = kManyWaves / RW, ROWS = 32 * RW;
    static constexpr int kHalfBytes = kStepTokens * HD * 2;  // K or V of a step
    static constexpr int kRing = 4 * TEAMS * kHalfBytes;
    static constexpr int kMerge = TEAMS * (HD / 4) * (ROWS + 1) * 16;
    static constexpr int kQueries = ROWS * (HD + 8) * 2;
    static constexpr int kMost = kRing > kMerge ? kRing : kMerge;
    static constexpr int kBytes = kMost > kQueries ? kMost : kQueries;
};

template <typename T, int HD, int RW, typename Tree>
__global__ __launch_bounds__(kManyThreads, 2) void paged_many_kernel(const PagedAttendArgs a, const Tree tree) {
    using M = ManyShape<HD, RW>;
    using Tile = RowTile<T, HD, 32>;
    constexpr int TEAMS = M::TEAMS, ROWS = M::ROWS, kHalfBytes = M::kHalfBytes, kStepBytes = 2 * kHalfBytes;
    constexpr int NL = Tile::NL, CG = HD / 4, kPitch = HD + 8;
    constexpr int kCells = HD * 4;               // of K, and of V, in a step
    constexpr int NH = TEAMS * 2 * kCells / kManyThreads;    // a thread's cells of a turn
    static_assert(NH >= 1 && kCells % 64 == 0, "a wave's cells are of one step");
    __shared__ __align__(16) uint8_t lds[M::kBytes];
    __shared__ float stats[TEAMS][ROWS][2];
    __shared__ int no_numbers[2][TEAMS];         // of a V slot: 1 + the step whose values are not all numbers
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane / 32, place = lane % 32, row = wave % RW * 32 + place, team = wave / RW;
    Share<ROWS, Tree> share;
    share.start(a, tree, blockIdx.x, lane);
    if (share.split >= share.my_splits) return;
    const int step_begin = share.step_begin, step_end = share.step_end;

    // The pages of 64 steps from `window` on, one in each lane, and of the 64 after them.
    const int32_t* const table = a.view.table + static_cast<int64_t>(a.slot0 + share.b) * a.view.entries;
    auto pages_from = [&](int step) { return table[max(0, min(step + lane, step_end - 1)) / kPageSteps]; };
    int window = step_begin, pages = pages_from(step_begin), pages_next = pages_from(step_begin + 64);
    uint8_t* const layer_head = a.view.base + paged_record(a.view, a.layer, 0, share.kh);
    const int64_t page_bytes = a.view.kv_heads * paged_record_bytes(HD);

    // A tree's rows (a few steps) are appended by every workgroup that reads them, with the
    // same bytes: its own writes are what it finds then.
    if (a.k != nullptr && share.template append<T, HD, kManyThreads>(a, table, layer_head, page_bytes, threadIdx.x, 1, 0)) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    }

    // Cell i * kManyThreads + thread of a turn: first the teams' K cells, then their V
    // cells.  A K cell [c][h][g'][m] is read by product 2 c + (g' >> 1)'s lane (g' & 1, 16 (m >> 3) +
    // 8 h + (m & 7)), a V cell [c][g'][m] by product (c >> 1, g' >> 1)'s lane (g' & 1, 16 (c & 1) + m).
    const int first_cell = wave * 64;            // of the wave, in a turn's first kManyThreads
    auto cell_of = [&](int i) { return i * kManyThreads + first_cell; };
    auto reader = [&](int cell, bool is_v) {
        const int m = cell & 15, gg = (cell >> 4) & 3, c = is_v ? cell >> 6 : cell >> 7, h = (cell >> 6) & 1;
        const int product = (is_v ? c >> 1 : c) * 2 + (gg >> 1);
        return product * 1024 + ((gg & 1) * 32 + (is_v ? (c & 1) * 16 + m : (m >> 3) * 16 + h * 8 + (m & 7))) * 16;
    };
    // K of turn `k_step`, V of turn `v_step` (first steps of their turns).
    auto load_turn = [&](v4i (&held)[NH], int k_step, int v_step) {
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            const bool is_v = cell_of(i) >= TEAMS * kCells;
            const int in_kind = cell_of(i) - (is_v ? TEAMS * kCells : 0), step = (is_v ? v_step : k_step) + in_kind / kCells;
            const int at = step - window;        // below 128: the window follows K
            const int page = at < 64 ? __builtin_amdgcn_readlane(pages, max(at, 0)) : __builtin_amdgcn_readlane(pages_next, min(at - 64, 63));
            held[i] = __builtin_amdgcn_raw_buffer_load_b128(step_resource(layer_head, page_bytes, page, step, step_end, kStepBytes), lane * 16,
                                                            (is_v ? kHalfBytes : 0) + in_kind % kCells * 16, 0);
        }
    };
    // CHECK: of V cells (turn v_step) that a turn of the tail reads.
    auto store_turn = [&](auto check, const v4i (&held)[NH], int k_slot, int v_slot, int v_step) {
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            const bool is_v = cell_of(i) >= TEAMS * kCells;
            const int in_kind = cell_of(i) - (is_v ? TEAMS * kCells : 0);
            uint8_t* const slot = lds + (((is_v ? 2 + v_slot : k_slot) * TEAMS) + in_kind / kCells) * kHalfBytes;
            *reinterpret_cast<v4i*>(slot + reader(in_kind % kCells + lane, is_v)) = held[i];
            if (decltype(check)::value && is_v && Tile::no_numbers(__builtin_bit_cast(typename Tile::Pairs, held[i])) != 0)
                no_numbers[v_slot][in_kind / kCells] = v_step + in_kind / kCells + 1;
        }
    };
    auto k_cells = [&](int slot) { return lds + (slot * TEAMS + team) * kHalfBytes + lane * 16; };
    auto v_cells = [&](int slot) { return lds + ((2 + slot) * TEAMS + team) * kHalfBytes + lane * 16; };
    if (threadIdx.x < 2 * TEAMS) no_numbers[threadIdx.x / TEAMS][threadIdx.x % TEAMS] = 0;
    v4i held[NH], held_first[NH];
    load_turn(held_first, step_begin, step_begin);
    load_turn(held, step_begin + TEAMS, step_end);

    T* const staged = reinterpret_cast<T*>(lds);
    share.template stage_queries<T, HD, kManyThreads>(a, staged);
    __syncthreads();
    Tile tile;
    tile.clear();
    share.sees(a, tile, row);
#pragma unroll
    for (int s = 0; s < Tile::NS; ++s) tile.q[s] = *reinterpret_cast<const Half8<T>*>(staged + row * kPitch + (s * 2 + g) * 8);
    __syncthreads();
    store_turn(std::true_type{}, held_first, 0, 0, step_begin);
    __syncthreads();
    float s[Tile::NV];
    auto seen = [&](int st) { return st < step_end ? tile.seen(st, g) : 0u; };
    auto operands = [&](Half8<T> (&x)[NL], const uint8_t* cells) {
#pragma unroll
        for (int i = 0; i < NL; ++i) x[i] = *reinterpret_cast<const Half8<T>*>(cells + i * 1024);
    };
    {
        Half8<T> kb[NL];
        operands(kb, k_cells(0));
        tile.scores(kb, s);
        tile.hide(seen(step_begin + team), s);
        tile.rise(s, a.scale);
    }
    store_turn(std::false_type{}, held, 1, 1, 0);
    load_turn(held, step_begin + 2 * TEAMS, step_begin + TEAMS);
    __syncthreads();

    int step0 = step_begin, odd = 0;
    // One turn: weights and sums of the scores `now`, scores `then` of the next.
    auto turn = [&](auto masked, const float (&now)[Tile::NV], float (&then)[Tile::NV]) __attribute__((always_inline)) {
        constexpr bool kMasked = decltype(masked)::value;
        const int step = step0 + team;
        if (!kMasked || step < step_end) {
            Half8<T> kb[NL], vb[NL], w[Tile::TERMS][Tile::NP];
            operands(kb, k_cells(odd ^ 1));
            operands(vb, v_cells(odd));
            __builtin_amdgcn_sched_barrier(0);   // all asked for before the first is waited for
            tile.scores(kb, then);
            tile.weights(now, a.scale, w);
            if constexpr (kMasked)
                if (__builtin_expect(no_numbers[odd][team] == step + 1, 0)) tile.part_with_no_numbers(vb, seen(step));
            tile.add(vb, w);
            if constexpr (kMasked) tile.hide(seen(step + TEAMS), then);
            tile.rise(then, a.scale);
        }
        store_turn(masked, held, odd, odd ^ 1, step0 + TEAMS);
        if (__builtin_expect(step0 + 3 * TEAMS + TEAMS > window + 128, 0)) {
            window += 64;
            pages = pages_next;
            pages_next = pages_from(window + 64);
        }
        load_turn(held, step0 + 3 * TEAMS, step0 + 2 * TEAMS);
        odd ^= 1;
        step0 += TEAMS;
        __syncthreads();
    };
    float s1[Tile::NV];
    auto run = [&](auto masked, int end) __attribute__((always_inline)) {
        while (step0 < end) {                    // an even number of turns: a turn past the last does nothing
            turn(masked, s, s1);
            turn(masked, s1, s);
        }
    };
    run(std::false_type{}, share.plain_end - 4 * TEAMS + 1);   // (the tail's V cells are checked a turn ahead)
    run(std::true_type{}, step_end);

    // The teams' sums meet in LDS, quads of channels of a row together.
    v4f* const quads = reinterpret_cast<v4f*>(lds);
    const float sum = Tile::groups_sum(tile.l);
    if (g == 0) {
        stats[team][row][0] = tile.m;
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
            all.add(ml, sums);
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
    const dim3 grid(a.view.kv_heads * a.splits * a.chunks, batch);
    auto go = [&](auto tag, auto hd, auto rw) {
        using T = decltype(tag);
        constexpr int HD = decltype(hd)::value, RW = decltype(rw)::value;
        if (tree) paged_many_kernel<T, HD, RW><<<grid, kManyThreads, 0, s>>>(a, *tree);
        else paged_many_kernel<T, HD, RW><<<grid, kManyThreads, 0, s>>>(a, PagedChain{});
    };
    auto shaped = [&](auto tag, auto hd) {
        if (rows == 64) go(tag, hd, integral_constant<int, 2>{});
        else if (rows == 128) go(tag, hd, integral_constant<int, 4>{});
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
