// swiftkv_block_prompt.hip -- attention of a prompt's chunk over the block cache:
// calls with more rows (query tokens times the query heads that share a
// key/value head) than one matrix instruction's digits hold.
#include "swiftkv_block_device.hpp"

namespace swiftkv {
namespace {

using namespace dev;

// Workgroup (key/value head, 64 rows, split): TEAMS teams of four waves take
// every TEAMS-th tile of the split; a wave has 16 rows.  Matrix products and the
// work around them bound it, so they run on 16-bit floats, which hold a code
// exactly, and not on the digits of swiftkv_block.hip, which would take four times
// the rows (512 tokens onto 4096, 32 heads over 8, in the first form: 84 us against 161;
// two teams 101, two row tiles a wave 94, two buffers and two teams 88; now 66).  Each team turns a
// tile's codes into half floats in LDS, once for its 64 rows
// (0x6400 + byte is 1024 + byte, so a byte permute and a packed subtraction), in
// the order in which the instruction reads them:
//
//   scores  S^T[token][row] = K Q^T: a lane ends with one row, its four tokens of
//           each block.  The query is scaled by a power of two to below 2^15 and
//           rounded to a half float; FP32 queries are two of them, 22 bits.
//   output  O^T[channel][row] = V^T P^T, with P straight from those registers:
//           which token stands in which place of the product does not matter as
//           long as V's layout agrees, so nothing moves between lanes but a row's
//           maximum.  A weight counts times its block's V scale, P = 2^11 p v over a
//           power of two that follows the largest p v which the row has seen (not the
//           largest p times the largest v: a block that the row does not see, or hardly
//           weighs, would take bits from the rest), rounded to a half float: 2^-11 of
//           each, below the output's own rounding in bfloat16 and at it in float16, or
//           2^-35 of the row's largest where that is more; FP32 outputs take two, 22 bits
//           of 2^15 p v, or 2^-39.  The sum of weights is that of P / v, in FP32.
constexpr int kTeamWaves = 4;                     // 16 rows each
constexpr int kTeamThreads = kTeamWaves * 64;

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v2h pack_halves(float a, float b) {
    return v2h{static_cast<_Float16>(a), static_cast<_Float16>(b)};
}

// Four codes as half floats.
__device__ __forceinline__ v2u code_halves(uint32_t w) {
    w ^= 0x80808080u;                            // byte + 128
    const v2h off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    const uint32_t low = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u);
    const uint32_t high = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
    return v2u{__builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, low) + off),
               __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, high) + off)};
}

// N products with operands from LDS, at(i) after the lane's first, each read
// kAhead products before it is used.  (Left to itself the compiler saves registers
// and waits for each read: 74 us against 66 for 512 tokens onto 4096.)
template <int N, typename At, typename Multiply>
__device__ __forceinline__ void products(const uint8_t* first, At at, Multiply multiply) {
    constexpr int kAhead = 4;
    v8h ring[kAhead];
#pragma unroll
    for (int i = 0; i < kAhead; ++i) ring[i] = *reinterpret_cast<const v8h*>(first + at(i));
#pragma unroll
    for (int i = 0; i < N; ++i) {
        __builtin_amdgcn_sched_barrier(0);
        multiply(i, ring[i % kAhead]);
        __builtin_amdgcn_sched_barrier(0);
        if (i + kAhead < N) ring[i % kAhead] = *reinterpret_cast<const v8h*>(first + at(i + kAhead));
    }
}

// a * b rounded, not part of a fused operation.
__device__ __forceinline__ float rounded_product(float a, float b) {
#pragma clang fp contract(off)
    return a * b;
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = max(x, dpp_u<kDppQuadXor1>(x));
    x = max(x, dpp_u<kDppQuadXor2>(x));
    x = max(x, dpp_u<kDppHalfMirror>(x));
    x = max(x, dpp_u<kDppRowRor8>(x));
    const uint32_t a = __builtin_amdgcn_readlane(x, 0), b = __builtin_amdgcn_readlane(x, 16),
                   c = __builtin_amdgcn_readlane(x, 32), d = __builtin_amdgcn_readlane(x, 48);
    return max(max(a, b), max(c, d));
}

__device__ __forceinline__ float across_groups_max(float x) {
    x = fmaxf(x, __shfl_xor(x, 16));
    return fmaxf(x, __shfl_xor(x, 32));
}
__device__ __forceinline__ float across_groups_sum(float x) {
    x += __shfl_xor(x, 16);
    return x + __shfl_xor(x, 32);
}

template <typename T, int HD, int TEAMS>
__global__ __launch_bounds__(TEAMS * kTeamThreads) void block_prompt_kernel(const BlockAttendArgs a) {
    constexpr int TERMS = sizeof(T) == 4 ? 2 : 1;    // half floats of a query value, and of a weight
    // A row's reference value, a whole number, follows the largest score + log2 of the
    // V scale only when that is more than kSlack above it, so that most tiles neither exchange
    // maxima nor scale what is there.
    constexpr int kSlackExp = TERMS == 1 ? 4 : 0, kWeightExp = 15 - kSlackExp;
    constexpr float kSlack = kSlackExp, kFloatMin = 0x1p-126f;
    // Sums of weights count in 2^-kSumExp of them, which keeps them and 1 / v in FP32's range.
    constexpr int kSumExp = 6;
    constexpr uint32_t kScaleMin = 127 - 100;    // exponent bits of the smallest scale
    // Between V scales further apart a weight may vanish beside p v that counts in the sum.
    constexpr uint32_t kWide = 96;
    // Beyond this a score has no room for log2 of a V scale beside it.
    constexpr float kFar = 0x1p22f;
    constexpr int NS = HD / 32, ND = HD / 16, kRecord = 2 * kBlockRows * HD;
    constexpr int kTileBytes = kTileTokens * HD * 2;         // of K, and of V
    constexpr int NL = kTileBlocks * kRecord / 16 / kTeamThreads;    // a thread's 16-byte pieces of a tile
    constexpr int kPieces = kRecord / 16;
    constexpr int kMergeFloats = kPromptRows * (HD + 2);
    constexpr int kLdsBytes = TEAMS * 2 * kTileBytes > (TEAMS - 1) * kMergeFloats * 4 ? TEAMS * 2 * kTileBytes : (TEAMS - 1) * kMergeFloats * 4;
    __shared__ __align__(16) uint8_t lds[kLdsBytes];
    __shared__ uint32_t arrived;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n16 = lane & 15;
    const int team = wave / kTeamWaves, part = wave % kTeamWaves;
    const int tid = threadIdx.x % kTeamThreads;
    const int b = a.order[blockIdx.y];
    int id = blockIdx.x;
    const int kh = id % a.view.kv_heads;         // heads fastest: a head's workgroups share an XCD's L2
    id /= a.view.kv_heads;
    const int split = id % a.splits, chunk = a.chunks - 1 - id / a.splits;    // the longest first
    const int all_rows = a.group * a.n;
    const int row_first = chunk * kPromptRows, rows = min(kPromptRows, all_rows - row_first);
    const int p = a.positions[b];
    const int most = p < 0 ? 0 : p + row_token(a, row_first + rows - 1) + 1;
    const int tiles = (most + kTileTokens - 1) / kTileTokens;
    const int my_splits = max(1, (tiles + a.split_tiles - 1) / a.split_tiles);
    if (split >= my_splits) return;
    const int per = split_length(tiles, my_splits), tile_begin = split * per, tile_end = min(tiles, tile_begin + per);

    const int64_t page = block_page(a.view, a.slot0 + b, a.layer, kh);
    int8_t* const base = a.view.base + page * a.view.page_bytes;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
        base, static_cast<short>(0), static_cast<int32_t>(a.view.page_bytes), kBufferWord3);
    const uint64_t* table = reinterpret_cast<const uint64_t*>(a.view.table + page * a.view.blocks);
    const int8_t* const scale_base = base + static_cast<int64_t>(a.view.blocks) * kRecord;

    // The row of this lane: its query as B operands, channels 32 s + 8 g ..
    const int row = part * 16 + n16;
    const int r = row_first + min(row, rows - 1), i_q = row_token(a, r);
    const int limit = row < rows && p >= 0 ? p + i_q + 1 : 0;
    const bool any_row = part * 16 < rows;
    const int wave_limit = p + row_token(a, row_first + min(part * 16 + 15, rows - 1)) + 1;      // of its last row
    v8h q[TERMS][NS];
    float qs;
    {
        const T* src = static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.n + i_q) * a.q_stride +
                       (kh * a.group + r - i_q * a.group) * HD + g * 8;
        Vec8<T> w[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) w[s] = *reinterpret_cast<const Vec8<T>*>(src + 32 * s);
        uint32_t amax = 0;                       // of the magnitudes' bits: what is no number is above infinity
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) amax = max(amax, __float_as_uint(static_cast<float>(w[s].v[j])) & 0x7fffffffu);
        amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 16)));
        amax = max(amax, static_cast<uint32_t>(__shfl_xor(static_cast<int>(amax), 32)));
        const bool poison = amax >= 0x7f800000u;
        const int e = poison ? 0 : max(static_cast<int>(amax >> 23) - 126, -90);     // magnitudes < 2^e
        qs = poison ? __builtin_nanf("") : ldexpf(fabsf(a.scale), e - 15);
        const float to_half = (a.scale < 0.0f ? -1.0f : 1.0f) * ldexpf(1.0f, 15 - e);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                const float x = static_cast<float>(w[s].v[j]) * to_half, y = static_cast<float>(w[s].v[j + 1]) * to_half;
                const v2h h = pack_halves(x, y);
                q[0][s][j] = h[0];
                q[0][s][j + 1] = h[1];
                if (TERMS == 2) {
                    const v2h rest = pack_halves(x - static_cast<float>(h[0]), y - static_cast<float>(h[1]));
                    q[TERMS - 1][s][j] = rest[0];
                    q[TERMS - 1][s][j + 1] = rest[1];
                }
            }
    }

    uint8_t* const k_lds = lds + team * 2 * kTileBytes;      // [block][32-channel step][lane][16 bytes]
    uint8_t* const v_lds = k_lds + kTileBytes;               // [16 channels][32 tokens][lane][16 bytes]
    TileHeads heads;
    uint32_t scale_pair[kTileBlocks];            // upper halves (all of a power of two) of a tile's K and V scales
    v4i piece[NL];
    // Piece i of the thread: unit `unit` of block blk(i), so that two pieces are the
    // same unit of a pair of blocks.
    const int unit = tid % kPieces;
    auto blk = [&](int i) { return NL == kTileBlocks ? i : part / (kPieces / 64) * NL + i; };
    auto load_tile = [&](int at) {
        const uint32_t low = heads.low(at), high = heads.high(at);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            const int j = blk(i);
            const uint32_t rec = ((j & 2 ? high : low) >> (16 * (j & 1))) & 0xffffu;
            piece[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, unit * 16, static_cast<int>(rec) * kRecord, 0);
        }
    };
    auto store_tile = [&]() {
#pragma unroll
        for (int i = 0; i < NL; i += 2) {
            const int j = blk(i);
            v2u h[2][4];
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int k = 0; k < 4; ++k) h[o][k] = code_halves(static_cast<uint32_t>(piece[i + o][k]));
            if (unit < HD) {     // K: 16 channels (chunk c) of token t
                const int c = unit >> 4, t = unit & 15;
#pragma unroll
                for (int o = 0; o < 2; ++o) {
                    v4u* dst = reinterpret_cast<v4u*>(k_lds) + ((j + o) * NS + (c >> 1)) * 64 + (c & 1) * 32 + t;
                    dst[0] = v4u{h[o][0].x, h[o][0].y, h[o][1].x, h[o][1].y};
                    dst[16] = v4u{h[o][2].x, h[o][2].y, h[o][3].x, h[o][3].y};
                }
            } else {             // V: 16 tokens of channel d of both; tokens 4 g' .. go to lane group g'
                const int d = unit - HD;
                v4u* dst = reinterpret_cast<v4u*>(v_lds) + ((d >> 4) * 2 + (j >> 1)) * 64 + (d & 15);
#pragma unroll
                for (int k = 0; k < 4; ++k) dst[k * 16] = v4u{h[0][k].x, h[0][k].y, h[1][k].x, h[1][k].y};
            }
        }
    };

    v4f acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_run = 0.0f;       // m_run: kWeightExp above the reference value
    float shift = 0.0f;                          // of the row's scores, a whole number; 0 unless one was far
    bool far = false;                            // some row's was
    uint32_t scale_low = 255, scale_high = 0;    // exponent bits of the V scales that the wave's rows see until the window's end
    bool wide = false, bad = false;
    bool poison = false;
    const int my_first = tile_begin + team;
    const int turns = (tile_end - tile_begin + TEAMS - 1) / TEAMS;   // every team's
    const int last_tile = max(tile_begin, tile_end - 1);
    for (int turn = 0; turn < turns; ++turn) {
        const int at = turn & 63, tile = my_first + turn * TEAMS;
        if (at == 0) {
            heads.load_entries(table, tile + lane * TEAMS, last_tile);
            heads.load_scales(scale_base);
            load_tile(0);
            // V scales are powers of two: exponents will do, 255 for one that is not a number.
            const int first = min(tile + lane * TEAMS, last_tile) * kTileTokens;
            uint32_t low = 255, high = 0;
            bool nan = false;
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
                const uint32_t e = max(static_cast<uint32_t>(heads.scale[j] >> 55) & 255u, kScaleMin);
                scale_pair[j] = static_cast<uint32_t>(heads.scale[j]) >> 16 | e << 23;
                nan |= e == 255;
                if (e < 255 && first + kBlockRows * j < wave_limit) {
                    low = min(low, e);
                    high = max(high, e);
                }
            }
            bad = __any(nan);
            scale_low = min(scale_low, ~wave_max(~low));
            scale_high = max(scale_high, wave_max(high));
            wide = scale_high > scale_low + kWide;
        }
        __syncthreads();                         // everyone is done with the tile before
        store_tile();
        __syncthreads();
        if (tile >= tile_end || !any_row) {
            load_tile((at + 1) & 63);
            continue;
        }
        float ks[kTileBlocks];
        uint32_t ev[kTileBlocks];                // exponent bits of the V scales
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            const uint32_t both = __builtin_amdgcn_readlane(scale_pair[j], at);
            ks[j] = __uint_as_float(both << 16);
            ev[j] = both >> 23;
        }
        const int tok0 = tile * kTileTokens;
        v4f s[kTileBlocks];
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) s[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        products<NS * kTileBlocks>(
            k_lds + lane * 16, [](int i) { return (i % kTileBlocks * NS + i / kTileBlocks) * 1024; },
            [&](int i, v8h kk) {
#pragma unroll
                for (int t = 0; t < TERMS; ++t)
                    s[i % kTileBlocks] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[t][i / kTileBlocks], s[i % kTileBlocks], 0, 0, 0);
            });
        // The next tile's codes: after the scores, which need the registers, and
        // without a condition, which would keep the last ones (a tile too many is read).
        load_tile((at + 1) & 63);
        // Scores are s * f, f > 0.
        float f[kTileBlocks];
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) f[j] = qs * ks[j];
        if (__any(tok0 + kTileTokens > limit)) {
            asm volatile("");                    // a branch, not selects in every tile
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
                // a factor that leaves -inf as it is
                if (tok0 + kBlockRows * j >= limit || f[j] < kFloatMin) f[j] = kFloatMin;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tok0 + kBlockRows * j + 4 * g + i >= limit) s[j][i] = -INFINITY;
            }
        }
        // Where scores are far, what follows sees them less the row's shift, which is the
        // largest at the time it was far.
        auto shift_scores = [&]() {
            float largest = -INFINITY;
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    s[j][i] = rounded_product(s[j][i], f[j]);
                    largest = fmaxf(largest, s[j][i]);
                }
                f[j] = 1.0f;
            }
            largest = across_groups_max(largest);
            if (fabsf(largest) < INFINITY && (m_run == -INFINITY ? fabsf(largest) > kFar : largest - shift > kFar)) {
                const float next = rintf(largest);
                m_run -= next - shift;
                shift = next;
            }
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) s[j] -= shift;
        };
        if (far) shift_scores();
        if (bad) {
            // A V scale that is not a number poisons the rows that see its block.
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j)
                if (ev[j] == 255) {
                    ev[j] = kScaleMin;
                    if (tok0 + kBlockRows * j < limit) poison = true;
                }
        }
        float vk[kTileBlocks];
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) vk[j] = static_cast<float>(static_cast<int>(ev[j]) - 127 + kWeightExp);
        auto largest_weight = [&]() {
            float top = -INFINITY;
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j)
                top = fmaxf(top, __builtin_fmaf(f[j], fmaxf(fmaxf(s[j][0], s[j][1]), fmaxf(s[j][2], s[j][3])), vk[j]));
            return top;
        };
        float top = largest_weight();
        if (__any(top > m_run + kSlack)) {
            top = across_groups_max(top);
            if (!far && __any(fabsf(top) > kFar && fabsf(top) < INFINITY)) {
                far = true;
                shift_scores();
                top = across_groups_max(largest_weight());
            }
            const float m_new = top > m_run + kSlack ? ceilf(top) : m_run;
            const float alpha = m_new == -INFINITY ? 0.0f : fast_exp2(m_run - m_new);
            if (m_new > -INFINITY) l_run = scaled(l_run, m_run - m_new);
            m_run = m_new;
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= alpha;
        }
        const float base_exp = (m_run == -INFINITY ? 0.0f : m_run) - kWeightExp;
        if (wide) {
            const float c = (kWeightExp - kSumExp) - base_exp;
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) l_run += fast_exp2(__builtin_fmaf(s[j][i], f[j], c));
        }
        v8h w[TERMS][2];
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            const float c = vk[j] - base_exp;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = fast_exp2(__builtin_fmaf(s[j][i], f[j], c));
            const float per_scale = wide ? 0.0f : __uint_as_float((254u - kSumExp - ev[j]) << 23);
            l_run = __builtin_fmaf((x[0] + x[1]) + (x[2] + x[3]), per_scale, l_run);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const v2h h = pack_halves(x[i], x[i + 1]);
                w[0][j >> 1][(j & 1) * 4 + i] = h[0];
                w[0][j >> 1][(j & 1) * 4 + i + 1] = h[1];
                if (TERMS == 2) {
                    const v2h rest = pack_halves(x[i] - static_cast<float>(h[0]), x[i + 1] - static_cast<float>(h[1]));
                    w[TERMS - 1][j >> 1][(j & 1) * 4 + i] = rest[0];
                    w[TERMS - 1][j >> 1][(j & 1) * 4 + i + 1] = rest[1];
                }
            }
        }
        products<2 * ND>(
            v_lds + lane * 16, [](int i) { return (i % ND * 2 + i / ND) * 1024; },
            [&](int i, v8h vv) {
#pragma unroll
                for (int t = 0; t < TERMS; ++t)
                    acc[i % ND] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, w[t][i / ND], acc[i % ND], 0, 0, 0);
            });
    }

    // Join the teams in LDS: (m, l, acc) per row of all but the first.
    float l = across_groups_sum(l_run);
    if (poison) l = __builtin_nanf("");
    if (far) {
        // The reference value of the scores themselves, as near as FP32 has it.
        const float all = m_run + shift;
        const int rest = static_cast<int>(fminf(fmaxf(m_run - (all - shift), -60.0f), 60.0f));
        m_run = all;
        l = ldexpf(l, rest);
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int k = 0; k < 4; ++k) acc[i][k] = ldexpf(acc[i][k], rest);
    }
    constexpr float kToValues = 1.0f / (1 << kSumExp);
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] *= kToValues;
    __syncthreads();
    float* const merge = reinterpret_cast<float*>(lds);
    if (team > 0) {
        float* const mine = merge + (team - 1) * kMergeFloats + row * (HD + 2);
        if (g == 0) {
            mine[0] = m_run;
            mine[1] = l;
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) *reinterpret_cast<v2f*>(mine + 2 + i * 16 + g * 4) = v2f{acc[i][0], acc[i][1]},
            *reinterpret_cast<v2f*>(mine + 4 + i * 16 + g * 4) = v2f{acc[i][2], acc[i][3]};
    }
    __syncthreads();
    const int64_t pair = (static_cast<int64_t>(b) * a.view.kv_heads + kh) * a.chunks + chunk;
    float* const partial = a.partials + pair * a.splits * kMergeFloats;
    const int64_t token = static_cast<int64_t>(b) * a.n + i_q;
    T* const out = static_cast<T*>(a.out) + token * a.out_stride + (kh * a.group + r - i_q * a.group) * HD;
    if (team == 0) {
        const float* const others = merge + row * (HD + 2);
        float m = m_run;
#pragma unroll
        for (int t = 0; t < TEAMS - 1; ++t) m = fmaxf(m, others[t * kMergeFloats]);
        const float m_safe = m == -INFINITY ? 0.0f : m;
        const float f1 = fast_exp2(m_run - m_safe);
        float f2[TEAMS - 1];
        l = scaled(l, m_run - m_safe);
#pragma unroll
        for (int t = 0; t < TEAMS - 1; ++t) {
            f2[t] = fast_exp2(others[t * kMergeFloats] - m_safe);
            l += scaled(others[t * kMergeFloats + 1], others[t * kMergeFloats] - m_safe);
        }
        float* const dst = partial + static_cast<int64_t>(split) * kMergeFloats + row * (HD + 2);
        if (my_splits > 1 && g == 0) {
            publish(dst, m);
            publish(dst + 1, l);
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) {
            struct alignas(sizeof(T) * 4) Four { T v[4]; } t;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float o = acc[i][k] * f1;
#pragma unroll
                for (int u = 0; u < TEAMS - 1; ++u) o += others[u * kMergeFloats + 2 + i * 16 + g * 4 + k] * f2[u];
                if (my_splits > 1) publish(dst + 2 + i * 16 + g * 4 + k, o);
                else t.v[k] = static_cast<T>(l == 0.0f ? 0.0f : o / l);
            }
            if (my_splits == 1 && row < rows) *reinterpret_cast<Four*>(out + i * 16 + g * 4) = t;
        }
    }
    if (my_splits == 1) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // what was published has arrived
    __syncthreads();
    uint32_t* const counter = a.counters + pair * kCounterStride;
    if (threadIdx.x == 0) arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (static_cast<int>(arrived) != my_splits - 1) return;
    // The last split joins everybody's, in split order; the counter is zero again.
    if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int i = threadIdx.x; i < rows * HD; i += TEAMS * kTeamThreads) {
        const int jr = i / HD, d = i % HD, rr = row_first + jr, ii = row_token(a, rr);
        float m, ls, o;
        join_splits<true>(partial + jr * (HD + 2), kMergeFloats, my_splits, d, m, ls, o);
        static_cast<T*>(a.out)[(static_cast<int64_t>(b) * a.n + ii) * a.out_stride +
                               (kh * a.group + rr - ii * a.group) * HD + d] = static_cast<T>(ls == 0.0f ? 0.0f : o / ls);
    }
}

}  // namespace

hipError_t launch_block_prompt(const BlockAttendArgs& a, int batch, ElementType t, hipStream_t s) {
    const dim3 grid(a.view.kv_heads * a.splits * a.chunks, batch);
    with_type(t, [&](auto tag) {
        using T = decltype(tag);
        constexpr int TEAMS = sizeof(T) == 4 ? 2 : 4;
        if (a.view.head_dim == 64) block_prompt_kernel<T, 64, TEAMS><<<grid, TEAMS * kTeamThreads, 0, s>>>(a);
        else block_prompt_kernel<T, 128, TEAMS><<<grid, TEAMS * kTeamThreads, 0, s>>>(a);
    });
    return hipGetLastError();
}

}  // namespace swiftkv
