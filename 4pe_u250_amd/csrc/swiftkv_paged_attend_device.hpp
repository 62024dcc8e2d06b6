// swiftkv_paged_attend_device.hpp -- what the paged attention's kernels share: the
// products on 16-bit matrix instructions, the softmax of one step of 32 cached
// tokens, a workgroup's share of a call, and how partial results are joined.
#pragma once

#include "swiftkv_paged_device.hpp"

namespace swiftkv {
namespace dev {

typedef float v16f __attribute__((ext_vector_type(16)));

// D[R][R] += A B.  Lane = (group g, place m): A has row m and contraction places
// 8 g .., B column m and the same places; D column m, rows 4 g .. of every
// 4 * 64 / R.
template <typename T, int R>
struct Product;
template <>
struct Product<__bf16, 16> {
    using Sum = v4f;
    static __device__ __forceinline__ Sum add(Half8<__bf16> a, Half8<__bf16> b, Sum c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Product<_Float16, 16> {
    using Sum = v4f;
    static __device__ __forceinline__ Sum add(Half8<_Float16> a, Half8<_Float16> b, Sum c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
};
template <>
struct Product<__bf16, 32> {
    using Sum = v16f;
    static __device__ __forceinline__ Sum add(Half8<__bf16> a, Half8<__bf16> b, Sum c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
};
template <>
struct Product<_Float16, 32> {
    using Sum = v16f;
    static __device__ __forceinline__ Sum add(Half8<_Float16> a, Half8<_Float16> b, Sum c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
};

__device__ __forceinline__ int row_token(uint32_t group_magic, int r) {
    return group_magic == 0 ? r : static_cast<int>(__umulhi(static_cast<uint32_t>(r), group_magic));
}

// The bits of tokens tok0 .. tok0 + 31 that a row sees: all before `first`, and
// those of `mask` from there on.  Without a branch, and the kernels ask for them before
// they form the scores: where a branch lay between matrix products and the reading of
// their results, hipcc 7.2 left the waits for them out on one of its paths.
__device__ __forceinline__ uint32_t seen_bits(int tok0, int first, uint64_t mask) {
    const int d = tok0 - first, below = min(max(-d, 0), 63), past = min(max(d, 0), 63);
    const uint32_t bits = static_cast<uint32_t>(((mask << below) | ((1ull << below) - 1ull)) >> past);
    return d < 64 ? bits : 0u;
}

// R rows of a wave: their queries as B operands, and softmax(scale q k^T) v over the
// steps that the wave takes, 32 cached tokens each:
//
//   scores  S^T[token][row] = K Q^T: a lane ends with one row and, of the step's
//           four octets of tokens, whole ones;
//   output  O^T[channel][row] = V^T P^T, with P straight from those registers,
//           rounded to the cache's type.
//
// Both A operands are the cache's cells as they lie (swiftkv_paged.hpp).  Nothing
// moves between lanes but, now and then, a row's maximum: the reference score that
// weights are taken over follows it only when a score is above its limit, with p <=
// 2^kScoreSlack until then.  (That branch is marked unlikely, which also keeps the sums'
// registers where the products want them.)  A score's difference to the reference is
// formed before it is scaled, and is 0 for equal scores.  (A multiply-add with the scaled
// reference is an instruction less, 420 us against 429 for 4096 tokens onto 4095, and leaves
// the product's rounding, more than all of a weight where scaled scores reach 2^24.  Loops of
// both kinds: 64 tokens of 8 sequences 56 us against 57, 26 tokens 15.4 against 15.3.)
//
// 16 rows leave the matrix instructions idle, so a bfloat16 weight is two terms there
// (2^-16 of it); with more rows it is one, 2^-8, as much as the output's own rounding (two
// terms: 64 tokens of 8 sequences 69 us against 60, 512 onto 4095 70 against 55, 4096 onto 4095
// 606 against 441).  A float16 weight is 2^(kShift + kScoreSlack) at most and is good to
// 2^-11, or to 2^-36 of the row's largest.  A bfloat16 weight is 2^-18 at most, so that
// kPagedMaxSeq of them times the largest values stay in FP32's range, 2^127 together, here
// and where waves and splits are joined; what that takes from the other end is below 2^-104
// of the row's largest weight.  (Up to 2^0.5 more where the limit was rounded up.)
template <typename T, int HD, int R, bool FINE = false>
struct RowTile {
    using P = Product<T, R>;
    using Sum = typename P::Sum;
    static constexpr bool kHalf = std::is_same<T, _Float16>::value;
    static constexpr int G = 64 / R;             // lane groups
    static constexpr int NV = kStepTokens / G;   // scores of a lane
    static constexpr int NP = NV / 8;            // octets of a lane
    static constexpr int NL = HD / 16;           // operands of K, and of V, a step
    static constexpr int NS = HD / (8 * G);      // products of a score
    static constexpr int ND = HD / R;            // output tiles
    static constexpr int NE = R * R / 64;        // sums of a lane in one
    static constexpr int TERMS = FINE && !kHalf ? 2 : 1;
    static constexpr float kShift = kHalf ? 11.0f : -22.0f;
    static_assert(kHalf || (1 << static_cast<int>(-kShift - kScoreSlack)) > kPagedMaxSeq, "sums of weights times values");
    typedef uint32_t Pairs __attribute__((ext_vector_type(4)));

    Half8<T> q[NS];
    Sum acc[ND];
    float t, limit, l;                           // reference score (0 before the first), where it follows, sum of weights
    uint64_t mask;
    int first;                                   // what the row sees: seen_bits' arguments

    __device__ __forceinline__ void clear() {
        t = l = 0.0f;
        limit = -INFINITY;
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[i] = Sum{};
    }
    // The reference score as others see it: -inf without one.
    __device__ __forceinline__ float reference() const { return limit == -INFINITY ? -INFINITY : t; }

    __device__ __forceinline__ void scores(const Half8<T> (&kb)[NL], float (&s)[NV]) const {
        if constexpr (R == 16) {
            Sum c[2] = {Sum{}, Sum{}};
#pragma unroll
            for (int i = 0; i < NL; ++i) c[i & 1] = P::add(kb[i], q[i >> 1], c[i & 1]);
#pragma unroll
            for (int i = 0; i < NV; ++i) s[i] = c[i >> 2][i & 3];
        } else {
            Sum c = Sum{};
#pragma unroll
            for (int i = 0; i < NL; ++i) c = P::add(kb[i], q[i], c);
#pragma unroll
            for (int i = 0; i < NV; ++i) s[i] = c[i];
        }
    }

    // The lane's part of what the row sees of the step: its octet o at bit 8 o G.
    __device__ __forceinline__ uint32_t seen(int step, int g) const { return seen_bits(step * kStepTokens, first, mask) >> (8 * g); }
    static __device__ __forceinline__ void hide(uint32_t bits, float (&s)[NV]) {
#pragma unroll
        for (int o = 0; o < NP; ++o)
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (!(bits >> (8 * o * G + j) & 1u)) s[8 * o + j] = -INFINITY;
    }

    static __device__ __forceinline__ float groups_max(float x) {
        if (R == 16) x = fmaxf(x, __shfl_xor(x, 16));
        return fmaxf(x, __shfl_xor(x, 32));
    }
    static __device__ __forceinline__ float groups_sum(float x) {
        if (R == 16) x += __shfl_xor(x, 16);
        return x + __shfl_xor(x, 32);
    }

    // The reference score follows scores above its limit: `slack` above it, or at it where
    // FP32 has none within an eighth of that.
    __device__ __forceinline__ void rise(const float (&s)[NV], const PagedAttendArgs& a) {
        float top = s[0];
#pragma unroll
        for (int i = 1; i < NV; ++i) top = fmaxf(top, s[i]);
        if (__builtin_expect(__any(top > limit), 0)) {
            top = groups_max(top);
            const bool follows = top > limit;
            const float fall = follows && limit != -INFINITY ? fast_exp2((t - top) * a.scale) : 1.0f;
            float above = top + a.slack;
            if (above - top > 1.125f * a.slack) above = top;
            t = follows ? top : t;
            limit = follows ? above : limit;
            l *= fall;
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= fall;
        }
    }
    // Scores to weights, as B operands.
    __device__ __forceinline__ void weights(const float (&s)[NV], float scale, Half8<T> (&w)[TERMS][NP]) {
#pragma unroll
        for (int o = 0; o < NP; ++o) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = fast_exp2(__builtin_fmaf(s[8 * o + j] - t, scale, kShift));
                w[0][o][j] = static_cast<T>(x[j]);
                if constexpr (TERMS == 2) w[TERMS - 1][o][j] = static_cast<T>(x[j] - static_cast<float>(w[0][o][j]));
            }
            l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        }
    }

    static constexpr uint32_t kInf = kHalf ? 0x7c00 : 0x7f80, kOne = kHalf ? 0x3c00 : 0x3f80;
    // Not zero where one of a cell's values is no number: a half of `rest` is 0 where its
    // exponent is all ones.
    static __device__ __forceinline__ uint32_t no_numbers(Pairs cell) {
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint32_t rest = ~cell[j] & (kInf << 16 | kInf);
            bad |= (rest - 0x00010001u) & ~rest & 0x80008000u;
        }
        return bad;
    }
    static __device__ __forceinline__ bool no_numbers(const Half8<T> (&vb)[NL]) {
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < NL; ++i) bad |= no_numbers(__builtin_bit_cast(Pairs, vb[i]));
        return __any(bad != 0);
    }

    // A weight that rounds to 0 times an infinity is a NaN, a second term may have the other
    // sign, and rows of a masked step do not all see its values.  So what is no number takes
    // no part in sums: where it made them none, they start again from 0 (drop), where rows
    // see different tokens it leaves V first (clean), and the steps are gone through once
    // more for it alone (look_again).  It then reaches the rows that see it, whatever their
    // weights: products of ones count such values.
    __device__ __forceinline__ bool no_number_sums() const {
        float x[4] = {};                         // (a sum that leaves the range is looked at for nothing)
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < NE; ++e) x[e & 3] += acc[d][e];
        const float sum = (x[0] + x[1]) + (x[2] + x[3]);
        return __any(!(fabsf(sum) < INFINITY));
    }
    __device__ __forceinline__ void drop() {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < NE; ++e) acc[d][e] = fabsf(acc[d][e]) < INFINITY ? acc[d][e] : 0.0f;
    }
    __device__ __forceinline__ void part_with_no_numbers(const Half8<T> (&vb)[NL], uint32_t bits) {
#pragma unroll 1
        for (int kind = 0; kind < 3; ++kind) {   // NaN, inf, -inf: from `low` on, `span` patterns
            const float value = kind == 0 ? __builtin_nanf("") : kind == 1 ? INFINITY : -INFINITY;
            const uint32_t sign = kind == 0 ? 0x7fffu : 0xffffu, low = kind == 0 ? kInf + 1 : kind == 1 ? kInf : kInf | 0x8000u;
            const uint32_t span = kind == 0 ? 0x8000u - low : 1u;
            auto count_of = [&](uint32_t u) { return ((u & sign) - low) < span ? kOne : 0u; };
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                Sum n = Sum{};
#pragma unroll
                for (int o = 0; o < NP; ++o) {
                    Pairs u = __builtin_bit_cast(Pairs, vb[d * NP + o]), sees;
                    asm volatile("" : "+v"(u), "+v"(bits));      // nothing of this is worth a register outside the loop
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        u[j] = count_of(u[j] >> 16) << 16 | count_of(u[j] & 0xffffu);
                        const uint32_t two = bits >> (8 * o * G + 2 * j);
                        sees[j] = (two & 1u) * kOne | (two & 2u) * (kOne << 15);
                    }
                    n = P::add(__builtin_bit_cast(Half8<T>, u), __builtin_bit_cast(Half8<T>, sees), n);
                }
#pragma unroll
                for (int e = 0; e < NE; ++e) acc[d][e] += n[e] > 0.0f ? value : 0.0f;
            }
        }
    }
    static __device__ __forceinline__ void clean(Half8<T> (&vb)[NL]) {
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            Pairs u = __builtin_bit_cast(Pairs, vb[i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t high = u[j] >> 16, lower = u[j] & 0xffffu;
                u[j] = ((high & kInf) == kInf ? 0u : high << 16) | ((lower & kInf) == kInf ? 0u : lower);
            }
            vb[i] = __builtin_bit_cast(Half8<T>, u);
        }
    }

    __device__ __forceinline__ void add(const Half8<T> (&vb)[NL], const Half8<T> (&w)[TERMS][NP]) {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int o = 0; o < NP; ++o)
#pragma unroll
                for (int t = 0; t < TERMS; ++t) acc[d] = P::add(vb[d * NP + o], w[t][o], acc[d]);
    }

    // The sums as quads of channels: quads[quad * pitch + row].
    __device__ __forceinline__ void leave(v4f* quads, int pitch, int row, int g) const {
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < NE / 4; ++e)
                quads[(d * (R / 4) + e * G + g) * pitch + row] = v4f{acc[d][4 * e], acc[d][4 * e + 1], acc[d][4 * e + 2], acc[d][4 * e + 3]};
    }
};

// What is no number to the sums of a wave's rows: its steps first, first + STRIDE, ... below
// `end` again.  load(step, vb): V of a step as operands.
template <int STRIDE, typename Tile, int RT, typename Operands, typename Load>
__device__ __forceinline__ void look_again(Tile (&tiles)[RT], Operands& vb, int first, int end, int g, Load&& load) {
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) tiles[rt].drop();
#pragma unroll 1
    for (int step = first; step < end; step += STRIDE) {
        load(step, vb);
        if (!Tile::no_numbers(vb)) continue;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) tiles[rt].part_with_no_numbers(vb, tiles[rt].seen(step, g));
    }
}

// A workgroup's share of a call: ROWS rows of a chunk, the steps of a split.
template <int ROWS, typename Tree>
struct Share {
    static constexpr bool kTree = std::is_same<Tree, PagedTree>::value;
    int b, kh, split, chunk;
    int row_first, rows;
    int p, count;                                // cached tokens before the call (negative: none), tokens of the call
    int my_splits, step_begin, step_end;
    int plain_end;                               // up to here every row sees whole steps
    TreePlace place;
    uint64_t live;                               // tokens of the tree

    // The workgroup's share.  Consecutive workgroups go to XCDs in turn; if the splits that a
    // short sequence does not have lay among them, some XCDs would get more than their CUs
    // hold.  The grid is one row of the splits that there are then (trees of 16 sequences of up
    // to 32511, 20 heads over 4: 99 us against 125).
    __device__ __forceinline__ void start(const PagedAttendArgs& a, const Tree& tree, int lane) {
        if (a.all_splits == 0) return start(a, tree, blockIdx.y, blockIdx.x, a.splits, lane);
        typedef uint32_t Words __attribute__((ext_vector_type(kPagedBatch / 4), aligned(4)));
        Words low = *reinterpret_cast<const Words*>(a.first_split), high = *reinterpret_cast<const Words*>(a.first_split + kPagedBatch / 4);
        asm("" : "+s"(low), "+s"(high));
        uint32_t mine = ~0u;
#pragma unroll
        for (int w = 0; w < kPagedBatch / 4; ++w) {
            if (lane == w) mine = low[w];
            if (lane == w + kPagedBatch / 4) mine = high[w];
        }
        const int unit = a.view.kv_heads * a.chunks, at = blockIdx.x / static_cast<uint32_t>(unit);
        const int y = __popcll(__ballot(static_cast<int>(mine & 0xffffu) <= at)) + __popcll(__ballot(static_cast<int>(mine >> 16) <= at)) - 1;
        auto first = [&](int i) { return static_cast<int>(static_cast<uint32_t>(__builtin_amdgcn_readlane(mine, i >> 1)) >> (i & 1) * 16 & 0xffffu); };
        const int before = first(y), next = y + 1 < a.batch ? first(y + 1) : a.all_splits;
        start(a, tree, y, blockIdx.x - before * unit, next - before, lane);
    }
    // `id`: the (split, chunk, head) of grid row y, heads fastest, so that a head's
    // workgroups share an XCD's L2.
    __device__ __forceinline__ void start(const PagedAttendArgs& a, const Tree& tree, int y, int id, int splits, int lane) {
        const PagedRow of_grid = a.order[y];
        b = of_grid.sequence;
        p = of_grid.position;
        kh = id % a.view.kv_heads;
        id /= a.view.kv_heads;
        split = id % splits;
        chunk = a.chunks - 1 - id / splits;      // the longest first
        row_first = chunk * ROWS;
        rows = min(ROWS, a.group * a.n - row_first);
        count = a.n;
        live = 0;
        if constexpr (kTree) {
            place = tree_place(tree.parents, b, a.n, lane);
            live = __ballot(place.live);
            count = __popcll(live);
        }
        // Tokens that some row sees, and those that all do.
        int most = 0, all_see = 0;
        if (p >= 0) {
            most = kTree ? p + count : p + row_token(a.group_magic, row_first + rows - 1) + 1;
            all_see = kTree ? p : p + row_token(a.group_magic, row_first) + 1;
        }
        const int steps = (most + kStepTokens - 1) / kStepTokens;
        my_splits = max(1, (steps + a.split_steps - 1) / a.split_steps);
        const int per = split_length(steps, my_splits);
        step_begin = split * per;
        step_end = min(steps, step_begin + per);
        plain_end = min(step_end, all_see / kStepTokens);
    }
    // The query token of a row, clamped to the chunk's.
    __device__ __forceinline__ int token(const PagedAttendArgs& a, int row) const {
        return row_token(a.group_magic, row_first + min(row, rows - 1));
    }
    __device__ __forceinline__ int position(int i) const {
        if constexpr (kTree) return turn_position(p, __popcll(from_lane(place.mask, i)) - 1, live >> i & 1);
        else return turn_position(p, i, true);
    }
    template <typename Tile>
    __device__ __forceinline__ void sees(const PagedAttendArgs& a, Tile& tile, int row) const {
        const int i = token(a, row);
        tile.mask = kTree ? from_lane(place.mask, i) : 0;
        tile.first = kTree ? p : p + i + 1;
    }
    // All rows' queries, turned, to LDS with a pitch of HD + 8.
    template <typename T, int HD, int THREADS>
    __device__ __forceinline__ void stage_queries(const PagedAttendArgs& a, T* staged) const {
        constexpr int kChunks = HD / 8, kItems = (ROWS * kChunks + THREADS - 1) / THREADS, kAtOnce = kItems < 4 ? kItems : 4;
        static_assert(kItems % kAtOnce == 0 && THREADS % kChunks == 0, "whole batches");
        const int c = threadIdx.x % kChunks;
        // (threads past the last row take that one again)
        auto row_of = [&](int it) { return min(it * (THREADS / kChunks) + static_cast<int>(threadIdx.x) / kChunks, ROWS - 1); };
        auto source = [&](int i, int row) {
            const int r = row_first + min(row, rows - 1);
            return static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.n + i) * a.q_stride + (kh * a.group + r - i * a.group) * HD;
        };
        auto leave = [&](int row, Half8<T> x) {
            if (a.negative) x = -x;
            *reinterpret_cast<Half8<T>*>(staged + row * (HD + 8) + 8 * c) = x;
        };
        if (aligned_rotation(a.rotation)) {
#pragma unroll 1
            for (int it0 = 0; it0 < kItems; it0 += kAtOnce) {
                Chunk<T> x[kAtOnce];
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) {
                    const int row = row_of(it0 + k), i = token(a, row);
                    x[k].load(source(i, row), c, a.rotation, angles(a.rotation, position(i)));
                }
#pragma unroll
                for (int k = 0; k < kAtOnce; ++k) leave(row_of(it0 + k), x[k].turned(c, a.rotation));
            }
        } else {
#pragma unroll 1
            for (int it = 0; it < kItems; ++it) {
                const int row = row_of(it), i = token(a, row);
                leave(row, turned(source(i, row), c, a.rotation, angles(a.rotation, position(i))));
            }
        }
    }
    // The call's rows that fall into the split's steps to the cache, by the whole workgroup, N
    // chunks' loads of a thread at a time (two are quicker where it has several, and slower
    // code where it has one: us of a step, 26 tokens 15.2 and 15.6, one token 10.8 and 10.6).
    // What it writes has arrived when it returns; everyone's has behind the next barrier.
    template <typename T, int HD, int THREADS>
    __device__ __forceinline__ void append(const PagedAttendArgs& a, const int32_t* table, uint8_t* layer_head, int64_t page_bytes, int wave,
                                           int lane) const {
        constexpr int kChunks = HD / 8, N = ROWS == 32 || ROWS == 48 || ROWS == 64 ? 2 : 1;
        static_assert(64 % kChunks == 0, "a thread's chunk stays");
        const int t0 = max(p, step_begin * kStepTokens), t1 = min(p + count, step_end * kStepTokens);
        if (p < 0 || t0 >= t1) return;
        const bool fast = aligned_rotation(a.rotation);
        const int items = (t1 - t0) * kChunks, c = lane % kChunks;
#pragma unroll 1
        for (int base = wave * 64; base < items; base += N * THREADS) {
            Chunk<T> k[N];
            Half8<T> v[N];
            int page[N];
            auto token_of = [&](int x) { return t0 + min(base + x * THREADS + lane, items - 1) / kChunks; };
#pragma unroll
            for (int x = 0; x < N; ++x) {
                const int tok = token_of(x), i = tok - p;
                const int64_t at = static_cast<int64_t>(b) * a.n + i;
                const T* const row = static_cast<const T*>(a.k) + at * a.k_stride + kh * HD;
                const float2* const cs = angles(a.rotation, position(i));
                page[x] = table[tok / kPageTokens];
                v[x] = *reinterpret_cast<const Half8<T>*>(static_cast<const T*>(a.v) + at * a.v_stride + kh * HD + 8 * c);
                if (fast) k[x].load(row, c, a.rotation, cs);
                else k[x].own = turned(row, c, a.rotation, cs);
            }
#pragma unroll
            for (int x = 0; x < N; ++x) {
                const int tok = token_of(x), step = tok / kStepTokens, t = tok % kStepTokens;
                if (base + x * THREADS + lane >= items || page[x] < 0) continue;
                uint8_t* const cells = layer_head + page[x] * page_bytes + (step % kPageSteps) * paged_step_bytes(HD);
                *reinterpret_cast<Half8<T>*>(cells + k_cell(t, c)) = fast ? k[x].turned(c, a.rotation) : k[x].own;
                T* const dst = reinterpret_cast<T*>(cells + v_cell(t / 8, 8 * c, HD)) + t % 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) dst[8 * j] = v[x][j];
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    // A row's values, sums over the sum of weights: zero for rows without a token.
    template <typename T, int HD>
    __device__ __forceinline__ void finish(const PagedAttendArgs& a, int row, int quad, float l, v4f o) const {
        if (row >= rows) return;
        const int r = row_first + row, i = row_token(a.group_magic, r);
        bool is_live = p >= 0;
        if constexpr (kTree) is_live &= (live >> i & 1) != 0;
        struct alignas(sizeof(T) * 4) Four { T v[4]; } t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t.v[e] = static_cast<T>(is_live ? o[e] / l : 0.0f);
        *reinterpret_cast<Four*>(static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.n + i) * a.out_stride +
                                 (kh * a.group + r - i * a.group) * HD + 4 * quad) = t;
    }
    // Where split j leaves (m, l) of a row, and a row's quads behind them.
    template <int HD>
    __device__ __forceinline__ float* partial(const PagedAttendArgs& a, int j) const {
        return a.partials + (((static_cast<int64_t>(b) * a.view.kv_heads + kh) * a.chunks + chunk) * a.splits + j) * (ROWS * (HD + 2));
    }
};

// Partial results (reference score, sum of weights, sums) joined one after another.
struct Joined {
    float m = -INFINITY, l = 0.0f;
    v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
    // N of them at once.
    template <int N>
    __device__ __forceinline__ void add(const v2f (&ml)[N], const v4f (&sums)[N], float scale) {
        float top = m;
#pragma unroll
        for (int j = 0; j < N; ++j) top = fmaxf(top, ml[j][0]);
        const float safe = top == -INFINITY ? 0.0f : top, f0 = fast_exp2((m - safe) * scale);
        const v4f before = o;
        l *= f0;
        o *= f0;
        float f[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            f[j] = fast_exp2((ml[j][0] - safe) * scale);
            l += ml[j][1] * f[j];
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(sums[j][e], f[j], o[e]);
        }
        // An infinity stays one where its factor is 0.
        const float all = (o[0] + o[1]) + (o[2] + o[3]);
        if (__builtin_expect(__any(all != all), 0)) {
            auto finite = [](float x) { return fabsf(x) < INFINITY; };
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                o[e] = finite(before[e]) ? before[e] * f0 : before[e];
#pragma unroll
                for (int j = 0; j < N; ++j) o[e] = finite(sums[j][e]) ? __builtin_fmaf(sums[j][e], f[j], o[e]) : o[e] + sums[j][e];
            }
        }
        m = top;
    }
};

// The page of `step` and on it its cells as a resource; past `end` an empty one, from
// which nothing is fetched.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t step_resource(uint8_t* layer_head, int64_t page_bytes, int page, int step, int end,
                                                                int step_bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(layer_head + max(page, 0) * page_bytes + (step % kPageSteps) * step_bytes,
                                             static_cast<short>(0), step < end ? step_bytes : 0, kBufferWord3);
}

}  // namespace dev
}  // namespace swiftkv
