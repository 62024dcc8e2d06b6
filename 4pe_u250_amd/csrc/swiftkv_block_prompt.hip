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
// the rows (512 tokens onto 4096, 32 heads over 8: 84 us against 161; two teams
// 101, two row tiles a wave 94, two buffers and two teams 88).  Each team turns a
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
//           maximum.  P = 2^15 p (scale over the largest seen), rounded to a half
//           float: 2^-12 of each weight, below the output's own rounding in
//           bfloat16 and at it in float16; FP32 outputs take two, 22 bits.
constexpr int kTeamWaves = 4;                     // 16 rows each
constexpr int kTeamThreads = kTeamWaves * 64;

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

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
    v8h q[TERMS][NS];
    float qs;
    {
        const T* src = static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.n + i_q) * a.q_stride +
                       (kh * a.group + r - i_q * a.group) * HD + g * 8;
        Vec8<T> w[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) w[s] = *reinterpret_cast<const Vec8<T>*>(src + 32 * s);
        float amax = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = fabsf(static_cast<float>(w[s].v[j]));
                amax = fmaxf(amax, x <= kFloatMax ? x : INFINITY);
            }
        amax = across_groups_max(amax);
        const bool poison = amax == INFINITY;
        const int e = poison ? 0 : max(static_cast<int>(__float_as_uint(amax) >> 23) - 126, -90);   // amax < 2^e
        qs = poison ? __builtin_nanf("") : ldexpf(a.scale, e - 15);
#pragma unroll
        for (int s = 0; s < NS; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = poison ? 0.0f : ldexpf(static_cast<float>(w[s].v[j]), 15 - e);
                const _Float16 h = static_cast<_Float16>(x);
                q[0][s][j] = h;
                if (TERMS == 2) q[TERMS - 1][s][j] = static_cast<_Float16>(x - static_cast<float>(h));
            }
    }

    uint8_t* const k_lds = lds + team * 2 * kTileBytes;      // [block][32-channel step][lane][16 bytes]
    uint8_t* const v_lds = k_lds + kTileBytes;               // [16 channels][32 tokens][lane][16 bytes]
    TileHeads heads;
    v4i piece[NL];
    // Piece i of the thread: unit `unit` of block blk(i).
    const int unit = tid % kPieces;
    auto blk = [&](int i) { return (i * kTeamThreads + part * 64) / kPieces; };
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
        for (int i = 0; i < NL; ++i) {
            const int j = blk(i);
            v2u h[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) h[k] = code_halves(static_cast<uint32_t>(piece[i][k]));
            if (unit < HD) {     // K: 16 channels (chunk c) of token t
                const int c = unit >> 4, t = unit & 15;
                uint8_t* dst = k_lds + ((j * NS + (c >> 1)) * 64 + (c & 1) * 32 + t) * 16;
                *reinterpret_cast<v4i*>(dst) = v4i{(int)h[0].x, (int)h[0].y, (int)h[1].x, (int)h[1].y};
                *reinterpret_cast<v4i*>(dst + 256) = v4i{(int)h[2].x, (int)h[2].y, (int)h[3].x, (int)h[3].y};
            } else {             // V: 16 tokens of channel d; tokens 4 g' .. go to lane group g'
                const int d = unit - HD;
                uint8_t* dst = v_lds + (((d >> 4) * 2 + (j >> 1)) * 64 + (d & 15)) * 16 + (j & 1) * 8;
#pragma unroll
                for (int k = 0; k < 4; ++k) *reinterpret_cast<v2u*>(dst + k * 256) = h[k];
            }
        }
    };

    v4f acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = -INFINITY, l_run = 0.0f, unit_scale = 0x1p-100f;   // acc counts in unit_scale * 2^-15
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
        }
        __syncthreads();                         // everyone is done with the tile before
        store_tile();
        __syncthreads();
        if (turn + 1 < turns && at != 63) load_tile(at + 1);
        if (tile >= tile_end || !any_row) continue;
        TileHead head;
        heads.scales_of(at, head);
        const int tok0 = tile * kTileTokens;
        v4f s[kTileBlocks];
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            s[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                const v8h kk = *reinterpret_cast<const v8h*>(k_lds + ((j * NS + k) * 64 + lane) * 16);
#pragma unroll
                for (int t = 0; t < TERMS; ++t) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kk, q[t][k], s[j], 0, 0, 0);
            }
        }
        float top = -INFINITY;
        const bool masked = __any(tok0 + kTileTokens > limit);
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            const float f = qs * head.ks[j];
#pragma unroll
            for (int i = 0; i < 4; ++i) s[j][i] *= f;
            if (masked) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (tok0 + kBlockRows * j + 4 * g + i >= limit) s[j][i] = -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s[j][i]);
        }
        top = across_groups_max(top);
        const float m_new = fmaxf(m_run, top), m_safe = m_new == -INFINITY ? 0.0f : m_new;
        // The largest V scale until now; one that is not a number poisons the rows
        // that see its block.
        float v_top = unit_scale;
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            v_top = fmaxf(v_top, head.vs[j]);
            if (head.vs[j] != head.vs[j] && tok0 + kBlockRows * j < limit) poison = true;
        }
        const float v_inv = pow2_inverse(v_top);
        const float alpha = fast_exp2(m_run - m_safe);
        const float shrink = alpha * (unit_scale * v_inv);
        m_run = m_new;
        unit_scale = v_top;
        float sum = 0.0f;
        v8h w[TERMS][2];
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            const float f = head.vs[j] == head.vs[j] ? head.vs[j] * v_inv * 32768.0f : 0.0f;
            float x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = fast_exp2(s[j][i] - m_safe);
                sum += e;
                x[i] = e * f;
            }
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
        l_run = l_run * alpha + sum;
        if (__any(shrink != 1.0f)) {
#pragma unroll
            for (int i = 0; i < ND; ++i) acc[i] *= shrink;
        }
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const v8h vv = *reinterpret_cast<const v8h*>(v_lds + ((i * 2 + k) * 64 + lane) * 16);
#pragma unroll
                for (int t = 0; t < TERMS; ++t) acc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vv, w[t][k], acc[i], 0, 0, 0);
            }
    }

    // Join the teams in LDS: (m, l, acc) per row of all but the first.
    float l = across_groups_sum(l_run);
    if (poison) l = __builtin_nanf("");
    const float to_values = unit_scale * (1.0f / 32768.0f);
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] *= to_values;
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
        l *= f1;
#pragma unroll
        for (int t = 0; t < TEAMS - 1; ++t) {
            f2[t] = fast_exp2(others[t * kMergeFloats] - m_safe);
            l += others[t * kMergeFloats + 1] * f2[t];
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
        join_splits(partial + jr * (HD + 2), kMergeFloats, my_splits, d, m, ls, o);
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
