// swiftkv_paged_attend.hip -- attention over the paged cache: one token, a chunk
// of a prompt or a tree of drafted tokens of each sequence.
#include "swiftkv_paged_device.hpp"

namespace swiftkv {
namespace {

using namespace dev;

constexpr int kAttendThreads = 256;
constexpr int kWaves = 4;
static_assert(kSplitQuantumSteps % kWaves == 0, "a split is whole turns of the waves");

typedef float v16f __attribute__((ext_vector_type(16)));

// D[R][R] += A B on 16-bit matrix instructions.  Lane = (group g, place m): A has
// row m and contraction places 8 g .., B column m and the same places; D column m,
// rows 4 g .. of every 4 * 64 / R.
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

// Over the lanes that share a place.
template <int R>
__device__ __forceinline__ float groups_max(float x) {
    if (R == 16) x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
template <int R>
__device__ __forceinline__ float groups_sum(float x) {
    if (R == 16) x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

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

// The bits of tokens tok0 .. tok0 + 31 that a row sees: all before `first`, and
// those of `mask` from there on.
__device__ __forceinline__ uint32_t seen_bits(int tok0, int first, uint64_t mask) {
    const int d = tok0 - first;
    if (d >= 0) return d < 64 ? static_cast<uint32_t>(mask >> d) : 0u;
    if (d <= -kStepTokens) return ~0u;
    return ((1u << -d) - 1u) | static_cast<uint32_t>(mask << -d);
}

// softmax(scale q k^T) v of the rows of one chunk -- query tokens times the
// query heads that share a key/value head, ROWS = R * RT of them -- over the steps
// of one split, 32 cached tokens each:
//
//   scores  S^T[token][row] = K Q^T: a lane ends with one row and, of the step's
//           four octets of tokens, whole ones;
//   output  O^T[channel][row] = V^T P^T, with P straight from those registers,
//           rounded to the cache's type.
//
// Both A operands are the cache's cells as they lie (swiftkv_paged.hpp), so a step
// is HD / 8 loads of 1 KiB a wave and nothing moves between lanes but, now and then,
// a row's maximum: the reference value that weights are taken over follows it only
// when a score is more than 2^kSlack above, with p <= 2^kSlack until then.
//
// Rows of few queries leave the matrix instructions idle, so a bfloat16 weight is
// two terms there (2^-16 of it); with more rows it is one, 2^-8.  A float16 weight
// is 2^(kShift + kSlack) at most and is good to 2^-11, or to 2^-36 of the row's largest.
//
// Wave w takes steps w, w + 4, ... of the split; the waves meet in LDS.  A
// sequence's splits publish (m, l, sums), wait until that has arrived, and count
// themselves; the last to arrive joins all in split order, so the result does not
// depend on who that is.
template <typename T, int HD, int R, int RT, typename Tree>
__global__ __launch_bounds__(kAttendThreads, R == 16 ? 3 : RT == 1 ? 2 : 1) void paged_attend_kernel(const PagedAttendArgs a,
                                                                                                 const Tree tree) {
    using P = Product<T, R>;
    using Sum = typename P::Sum;
    constexpr bool kTree = std::is_same<Tree, PagedTree>::value, kHalf = std::is_same<T, _Float16>::value;
    constexpr int ROWS = R * RT, G = 64 / R;     // lane groups
    constexpr int NV = kStepTokens / G;          // scores of a lane
    constexpr int NP = NV / 8;                   // octets of a lane
    constexpr int NL = HD / 16;                  // loads of K, and of V
    constexpr int NS = HD / (8 * G);             // products of a score
    constexpr int ND = HD / R;                   // output tiles
    constexpr int TERMS = R == 16 && !kHalf ? 2 : 1;
    constexpr float kSlack = 4.0f, kShift = kHalf ? 11.0f : 0.0f;
    constexpr int kPolicy = ROWS < 64 ? 2 : 0;   // nontemporal where a page is read once
    constexpr int kStepBytes = 2 * kStepTokens * HD * 2, kChunks = HD / 8;
    constexpr int CG = HD / 4;                   // quads of output channels
    __shared__ __align__(16) v4f lds[kWaves * CG * (ROWS + 1)];  // queries, then the waves' sums
    __shared__ float stats[kWaves][ROWS][2];
    __shared__ uint32_t arrived;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane / R, place = lane % R;
    const int b = a.order[blockIdx.y];
    int id = blockIdx.x;
    const int kh = id % a.view.kv_heads;         // heads fastest: a head's workgroups share an XCD's L2
    id /= a.view.kv_heads;
    const int split = id % a.splits, chunk = a.chunks - 1 - id / a.splits;    // the longest first
    const int all_rows = a.group * a.n;
    const int row_first = chunk * ROWS, rows = min(ROWS, all_rows - row_first);
    const int p = a.positions[b];
    TreePlace at_place{};
    uint64_t live_nodes = 0;
    int count = a.n;
    if constexpr (kTree) {
        at_place = tree_place(tree.parents + b * a.n, a.n, lane);
        live_nodes = __ballot(at_place.live);
        count = __popcll(live_nodes);
    }
    // Tokens that some row sees, and those that all do.
    int most = 0, all_see = 0;
    if (p >= 0) {
        most = kTree ? p + count : p + row_token(a.group_magic, row_first + rows - 1) + 1;
        all_see = kTree ? p : p + row_token(a.group_magic, row_first) + 1;
    }
    const int steps = (most + kStepTokens - 1) / kStepTokens;
    const int my_splits = max(1, (steps + a.split_steps - 1) / a.split_steps);
    if (split >= my_splits) return;
    const int per = split_length(steps, my_splits), step_begin = split * per, step_end = min(steps, step_begin + per);

    // The pages of 64 of the wave's steps, one in each lane (a lane past its last step
    // asks for that one's).
    const int32_t* const table = a.view.table + static_cast<int64_t>(a.slot0 + b) * a.view.entries;
    int pages = 0;
    auto load_pages = [&](int step) {
        pages = table[max(0, min(step + lane * kWaves, step_end - 1)) / kPageSteps];
    };
    load_pages(step_begin + wave);
    uint8_t* const layer_base = a.view.base + paged_record(a.view, a.layer, 0, kh);
    const int64_t page_bytes = a.view.kv_heads * paged_record_bytes(HD);
    auto step_cells = [&](int page, int step) { return layer_base + page * page_bytes + (step % kPageSteps) * kStepBytes; };

    // A wave appends the call's rows to the steps that it will scan; nobody else reads
    // those (one chunk).
    if (a.k != nullptr && p >= 0) {
        const int last = min(step_end, (p + count - 1) / kStepTokens + 1);
        int step = max(step_begin, p / kStepTokens);
        step += (wave - (step - step_begin)) & (kWaves - 1);
        bool wrote = false;
        for (; step < last; step += kWaves) {
            const int page = table[step / kPageSteps];
            const int t0 = max(p, step * kStepTokens), t1 = min(p + count, (step + 1) * kStepTokens);
            if (page < 0) continue;
            uint8_t* const cells = step_cells(page, step);
            const int items = (t1 - t0) * kChunks;
            for (int base = 0; base < items; base += 64) {
                const int item = min(base + lane, items - 1), tok = t0 + item / kChunks, c = item % kChunks, i = tok - p;
                const int64_t row = static_cast<int64_t>(b) * a.n + i;
                int position = tok;
                if constexpr (kTree) position = p + __popcll(from_lane(at_place.mask, i)) - 1;
                const Half8<T> kk = turned(static_cast<const T*>(a.k) + row * a.k_stride + kh * HD, c, a.rotation, angles(a.rotation, position));
                const Half8<T> vv = *reinterpret_cast<const Half8<T>*>(static_cast<const T*>(a.v) + row * a.v_stride + kh * HD + 8 * c);
                const int t = tok % kStepTokens;
                *reinterpret_cast<Half8<T>*>(cells + k_cell(t, c)) = kk;
                T* const dst = reinterpret_cast<T*>(cells + v_cell(t / 8, 8 * c, HD)) + t % 8;
#pragma unroll
                for (int j = 0; j < 8; ++j) dst[8 * j] = vv[j];
            }
            wrote = true;
        }
        if (wrote) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the scan's loads find them
    }

    // The chunk's queries, turned once for the workgroup and read as B operands.
    constexpr int kPitch = HD + 8;
    T* const staged = reinterpret_cast<T*>(lds);
#pragma unroll
    for (int it = 0; it < (ROWS * kChunks + kAttendThreads - 1) / kAttendThreads; ++it) {
        const int item = min(it * kAttendThreads + static_cast<int>(threadIdx.x), ROWS * kChunks - 1), row = item / kChunks, c = item % kChunks;
        const int r = row_first + min(row, rows - 1), i = row_token(a.group_magic, r);
        int position = p + i;
        if constexpr (kTree) position = p + __popcll(from_lane(at_place.mask, i)) - 1;
        Half8<T> x = turned(static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.n + i) * a.q_stride + (kh * a.group + r - i * a.group) * HD,
                            c, a.rotation, angles(a.rotation, max(position, 0)));
        if (a.negative) x = -x;
        *reinterpret_cast<Half8<T>*>(staged + row * kPitch + 8 * c) = x;
    }
    // What the lane's rows see past all_see.
    uint64_t mask[RT];
    int first[RT];                               // seen_bits' argument
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int i = row_token(a.group_magic, row_first + min(rt * R + place, rows - 1));
        mask[rt] = kTree ? from_lane(at_place.mask, i) : 0;
        first[rt] = kTree ? p : p + i + 1;
    }
    __syncthreads();
    Half8<T> q[RT][NS];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int s = 0; s < NS; ++s)
            q[rt][s] = *reinterpret_cast<const Half8<T>*>(staged + (rt * R + place) * kPitch + (s * G + g) * 8);

    const int k_lane = R == 16 ? lane * 16 : (((place >> 3) & 1) * 64 + g * 16 + (place >> 4) * 8 + ((place >> 2) & 1) * 4 + (place & 3)) * 16;
    const int v_lane = R == 16 ? lane * 16 : ((place >> 4) * 64 + g * 16 + (place & 15)) * 16;
    auto cell_at = [](int l) { return R == 16 ? l * 1024 : ((l >> 1) * 128 + (l & 1) * 32) * 16; };

    Sum acc[RT][ND];
    float m[RT], l[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY;
        l[rt] = 0.0f;
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[rt][i] = Sum{};
    }

    // A step's K and V are asked for as soon as the registers of the one before are
    // free, K during its softmax and V after its products; past the wave's last step
    // the resource is empty, and nothing is fetched.
    Half8<T> kb[NL], vb[NL];
    auto cells_of = [&](int step, int at) {
        const int page = __builtin_amdgcn_readlane(pages, at);
        return __builtin_amdgcn_make_buffer_rsrc(step_cells(max(page, 0), step), static_cast<short>(0),
                                                 step < step_end ? kStepBytes : 0, kBufferWord3);
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

    // One step, and the loads of the next; MASKED: rows see different tokens of it.
    auto scan = [&](auto masked, int step, __amdgpu_buffer_rsrc_t next) {
        constexpr bool kMasked = decltype(masked)::value;
        uint32_t bits[RT];
        Half8<T> w[RT][TERMS][NP];
        float s[RT][NV];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if constexpr (R == 16) {
                Sum c[2] = {Sum{}, Sum{}};
#pragma unroll
                for (int i = 0; i < NL; ++i) c[i & 1] = P::add(kb[i], q[rt][i >> 1], c[i & 1]);
#pragma unroll
                for (int i = 0; i < NV; ++i) s[rt][i] = c[i >> 2][i & 3];
            } else {
                Sum c = Sum{};
#pragma unroll
                for (int i = 0; i < NL; ++i) c = P::add(kb[i], q[rt][i], c);
#pragma unroll
                for (int i = 0; i < NV; ++i) s[rt][i] = c[i];
            }
        }
        __builtin_amdgcn_sched_barrier(0);
        load_k(next);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if constexpr (kMasked) {
                bits[rt] = seen_bits(step * kStepTokens, first[rt], mask[rt]) >> (8 * g);
#pragma unroll
                for (int o = 0; o < NP; ++o)
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        if (!(bits[rt] >> (8 * o * G + j) & 1u)) s[rt][8 * o + j] = -INFINITY;
            }
            float top = s[rt][0];
#pragma unroll
            for (int i = 1; i < NV; ++i) top = fmaxf(top, s[rt][i]);
            top *= a.scale;
            if (__any(top > m[rt] + kSlack)) {
                top = groups_max<R>(top);
                const float next = top > m[rt] + kSlack ? top : m[rt];
                const float fall = next == -INFINITY ? 1.0f : fast_exp2(m[rt] - next);
                m[rt] = next;
                l[rt] *= fall;
#pragma unroll
                for (int i = 0; i < ND; ++i) acc[rt][i] *= fall;
            }
            const float c = kShift - (m[rt] == -INFINITY ? 0.0f : m[rt]);
#pragma unroll
            for (int o = 0; o < NP; ++o)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float x = fast_exp2(__builtin_fmaf(s[rt][8 * o + j], a.scale, c));
                    l[rt] += x;
                    w[rt][0][o][j] = static_cast<T>(x);
                    if constexpr (TERMS == 2) w[rt][TERMS - 1][o][j] = static_cast<T>(x - static_cast<float>(w[rt][0][o][j]));
                }
        }
        if constexpr (kMasked) {
            // 0 times an infinity or a NaN is a NaN, so what is no number leaves V here and
            // reaches the rows that see it by itself: products of ones count such values.
            typedef uint32_t Pairs __attribute__((ext_vector_type(4)));
            constexpr uint32_t kInf = kHalf ? 0x7c00 : 0x7f80, kInfs = kInf << 16 | kInf, kOne = kHalf ? 0x3c00 : 0x3f80;
            uint32_t bad = 0;                    // a half of `rest` is 0 where its exponent is all ones
#pragma unroll
            for (int i = 0; i < NL; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t rest = ~__builtin_bit_cast(Pairs, vb[i])[j] & kInfs;
                    bad |= (rest - 0x00010001u) & ~rest & 0x80008000u;
                }
            if (__any(bad != 0)) {
#pragma unroll 1
                for (int kind = 0; kind < 3; ++kind) {       // NaN, inf, -inf: from `low` on, `span` patterns
                    const float value = kind == 0 ? __builtin_nanf("") : kind == 1 ? INFINITY : -INFINITY;
                    const uint32_t sign = kind == 0 ? 0x7fffu : 0xffffu, low = kind == 0 ? kInf + 1 : kind == 1 ? kInf : kInf | 0x8000u;
                    const uint32_t span = kind == 0 ? 0x8000u - low : 1u;
                    auto count_of = [&](uint32_t u) { return ((u & sign) - low) < span ? kOne : 0u; };
#pragma unroll
                    for (int d = 0; d < ND; ++d) {
                        Half8<T> is[NP];
#pragma unroll
                        for (int o = 0; o < NP; ++o) {
                            Pairs u = __builtin_bit_cast(Pairs, vb[d * NP + o]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) u[j] = count_of(u[j] >> 16) << 16 | count_of(u[j] & 0xffffu);
                            is[o] = __builtin_bit_cast(Half8<T>, u);
                        }
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt) {
                            Sum n = Sum{};
#pragma unroll
                            for (int o = 0; o < NP; ++o) {
                                Pairs sees;
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    const uint32_t two = bits[rt] >> (8 * o * G + 2 * j);
                                    sees[j] = (two & 1u) * kOne | (two & 2u) * (kOne << 15);
                                }
                                n = P::add(is[o], __builtin_bit_cast(Half8<T>, sees), n);
                            }
#pragma unroll
                            for (int e = 0; e < R * R / 64; ++e) acc[rt][d][e] += n[e] > 0.0f ? value : 0.0f;
                        }
                    }
                }
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
        }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int o = 0; o < NP; ++o)
#pragma unroll
                    for (int t = 0; t < TERMS; ++t) acc[rt][d] = P::add(vb[d * NP + o], w[rt][t][o], acc[rt][d]);
    };
    const int plain_end = min(step_end, all_see / kStepTokens);
    int step = step_begin + wave, at = 0;
    if (step < step_end) {
        const __amdgpu_buffer_rsrc_t cells = cells_of(step, 0);
        load_k(cells);
        load_v(cells);
    }
    auto run = [&](auto masked, int end) {
        for (; step < end; step += kWaves) {
            if (++at == 64) {
                load_pages(step + kWaves);
                at = 0;
            }
            const __amdgpu_buffer_rsrc_t next = cells_of(step + kWaves, at);
            scan(masked, step, next);
            __builtin_amdgcn_sched_barrier(0);
            load_v(next);
        }
    };
    run(std::false_type{}, plain_end);
    run(std::true_type{}, step_end);

    __syncthreads();                             // everyone has its queries
    // The waves' sums meet in LDS, quads of channels of a row together.
    const int row_of = place;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const float sum = groups_sum<R>(l[rt]);
        if (g == 0) {
            stats[wave][rt * R + row_of][0] = m[rt];
            stats[wave][rt * R + row_of][1] = sum;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int e = 0; e < R * R / 256; ++e) {
                const int quad = d * (R / 4) + e * G + g;
                lds[(wave * CG + quad) * (ROWS + 1) + rt * R + row_of] =
                    v4f{acc[rt][d][4 * e], acc[rt][d][4 * e + 1], acc[rt][d][4 * e + 2], acc[rt][d][4 * e + 3]};
            }
    }
    __syncthreads();
    constexpr int kItems = ROWS * CG / kAttendThreads;
    const int64_t pair = (static_cast<int64_t>(b) * a.view.kv_heads + kh) * a.chunks + chunk;
    constexpr int kPartial = ROWS * (HD + 2);
    float* const partials = a.partials + pair * a.splits * kPartial;
    // A row's place in `out`, and its values: sums over the sum of weights, zero for rows
    // without a token.
    auto finish = [&](int row, int quad, float l_all, v4f o) {
        if (row >= rows) return;
        const int r = row_first + row, i = row_token(a.group_magic, r);
        bool live = p >= 0;
        if constexpr (kTree) live &= (live_nodes >> i & 1) != 0;
        struct alignas(sizeof(T) * 4) Four { T v[4]; } t;
#pragma unroll
        for (int e = 0; e < 4; ++e) t.v[e] = static_cast<T>(live ? o[e] / l_all : 0.0f);
        *reinterpret_cast<Four*>(static_cast<T*>(a.out) + (static_cast<int64_t>(b) * a.n + i) * a.out_stride +
                                 (kh * a.group + r - i * a.group) * HD + 4 * quad) = t;
    };
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int item = threadIdx.x + k * kAttendThreads, row = item / CG, quad = item % CG;
        float m_all = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) m_all = fmaxf(m_all, stats[w][row][0]);
        const float safe = m_all == -INFINITY ? 0.0f : m_all;
        float l_all = 0.0f;
        v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = fast_exp2(stats[w][row][0] - safe);
            l_all += stats[w][row][1] * f;
            o += lds[(w * CG + quad) * (ROWS + 1) + row] * f;
        }
        if (my_splits == 1) {
            finish(row, quad, l_all, o);
        } else {
            float* const dst = partials + static_cast<int64_t>(split) * kPartial;
            if (quad == 0) publish2(dst + row * 2, m_all, l_all);
            float* const sums = dst + ROWS * 2 + row * HD + quad * 4;
            publish2(sums, o[0], o[1]);
            publish2(sums + 2, o[2], o[3]);
        }
    }
    if (my_splits == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // what was published has arrived
    __syncthreads();
    uint32_t* const counter = a.counters + pair * kCounterStride;
    if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (static_cast<int>(arrived) != my_splits - 1) return;
    // The last split joins everybody's, four at a time; the counter is zero again.
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int item = threadIdx.x + k * kAttendThreads, row = item / CG, quad = item % CG;
        if (row >= rows) continue;
        float m_all = -INFINITY, l_all = 0.0f;
        v4f o = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int j0 = 0; j0 < my_splits; j0 += 4) {
            v2f ml[4], lo[4], hi[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float* src = partials + static_cast<int64_t>(min(j0 + j, my_splits - 1)) * kPartial;
                ml[j] = fetch2(src + row * 2);
                lo[j] = fetch2(src + ROWS * 2 + row * HD + quad * 4);
                hi[j] = fetch2(src + ROWS * 2 + row * HD + quad * 4 + 2);
            }
            float top = m_all;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j0 + j >= my_splits) ml[j] = v2f{-INFINITY, 0.0f}, lo[j] = hi[j] = v2f{0.0f, 0.0f};
                top = fmaxf(top, ml[j][0]);
            }
            const float safe = top == -INFINITY ? 0.0f : top, f0 = fast_exp2(m_all - safe);
            l_all *= f0;
            o *= f0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float f = fast_exp2(ml[j][0] - safe);
                l_all += ml[j][1] * f;
                o += v4f{lo[j][0], lo[j][1], hi[j][0], hi[j][1]} * f;
            }
            m_all = top;
        }
        finish(row, quad, l_all, o);
    }
}

}  // namespace

hipError_t launch_paged_attend(const PagedAttendArgs& a, const PagedTree* tree, int batch, int rows, ElementType t, hipStream_t s) {
    const dim3 grid(a.view.kv_heads * a.splits * a.chunks, batch);
    auto go = [&](auto tag, auto hd, auto r, auto rt) {
        using T = decltype(tag);
        constexpr int HD = decltype(hd)::value, R = decltype(r)::value, RT = decltype(rt)::value;
        if (tree) paged_attend_kernel<T, HD, R, RT><<<grid, kAttendThreads, 0, s>>>(a, *tree);
        else paged_attend_kernel<T, HD, R, RT><<<grid, kAttendThreads, 0, s>>>(a, PagedChain{});
    };
    auto shaped = [&](auto tag, auto hd) {
        using std::integral_constant;
        if (rows == 16) go(tag, hd, integral_constant<int, 16>{}, integral_constant<int, 1>{});
        else if (rows == 32) go(tag, hd, integral_constant<int, 32>{}, integral_constant<int, 1>{});
        else go(tag, hd, integral_constant<int, 32>{}, integral_constant<int, 2>{});
    };
    auto typed = [&](auto tag) {
        if (a.view.head_dim == 64) shaped(tag, std::integral_constant<int, 64>{});
        else shaped(tag, std::integral_constant<int, 128>{});
    };
    if (t == kBF16) typed(__bf16{});
    else typed(_Float16{});
    return hipGetLastError();
}

}  // namespace swiftkv
