// swiftkv_block.hip -- kernels of the block cache: append, values, attention,
// eviction.  Layout and numerics: swiftkv_block.hpp, include/swiftkv.h.
#include "swiftkv_block_device.hpp"

namespace swiftkv {
namespace {

using namespace dev;

// Larger rows are taken as infinite: a code 64 of scale 2^122 would stand for 2^128.
constexpr float kRowMax = 0x1.fcp+126f;          // 127 * 2^120

// ---------------------------------------------------------------- codes

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) x = fmaxf(x, __shfl_xor(x, d));
    return x;
}

// The smallest power of two s = 2^e, e >= -100, with amax <= 127 * s.  With
// amax = 1.f * 2^x that is e = x - 6, and one more where 1.f > 127 / 64.
__device__ __forceinline__ float code_scale(float amax) {
    const uint32_t u = __float_as_uint(amax);
    const int e = static_cast<int>(u >> 23) - 133 + ((u & 0x7fffffu) > 0x7e0000u ? 1 : 0);
    return __uint_as_float(static_cast<uint32_t>(max(e, -100) + 127) << 23);
}

__device__ __forceinline__ uint32_t code_byte(float x) {
    return static_cast<uint32_t>(static_cast<int32_t>(__builtin_rintf(x))) & 0xffu;
}

__device__ __forceinline__ float byte_value(uint32_t word, int i) {
    return static_cast<float>(static_cast<int8_t>(static_cast<uint8_t>(word >> (8 * i))));
}

// 16 codes under a larger scale.
__device__ __forceinline__ v4i rescaled(v4i o, float ratio) {
    v4i w = {0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < 16; ++j)
        w[j >> 2] |= static_cast<int32_t>(code_byte(byte_value(static_cast<uint32_t>(o[j >> 2]), j & 3) * ratio)
                                          << (8 * (j & 3)));
    return w;
}

// A row value's magnitude, infinite for all that a scale cannot cover (NaN too).
__device__ __forceinline__ float row_magnitude(float x) { return fabsf(x) <= kRowMax ? fabsf(x) : INFINITY; }

// A block's scale after rows of largest magnitude amax join it.
__device__ __forceinline__ float joined_scale(float amax, bool held, float old) {
    float s = code_scale(amax);
    if (held) s = old >= s || old != old ? old : s;
    return amax == INFINITY ? __builtin_nanf("") : s;
}

// What a wave needs to append rows to one block: where its tokens and rows lie.
template <typename T>
struct BlockRows {
    int tok0;             // the block's first token
    int p, end;           // tokens [p, end) are new
    const T* rows;        // the new rows of this key/value head: token p's
    int64_t stride;
    bool held;            // the block keeps rows of earlier calls
    float old;            // its scale then
};

// One wave appends a block's K rows: lane = (token, 16-channel chunks c and
// c + 4).  A block that keeps its scale has only the new rows written.  Returns
// the scale.
template <typename T, int HD>
__device__ __forceinline__ float append_k(const BlockRows<T>& r, int8_t* record, int lane) {
    constexpr int NC = HD / 64;
    const int t = lane >> 2, c = lane & 3, tok = r.tok0 + t;
    const bool fresh = tok >= r.p && tok < r.end;
    float x[NC][16];
    float amax = 0.0f;
    // Every lane loads a row, the nearest new one where its own is not new: no
    // branch that the loads would wait at.
    const T* src = r.rows + (min(max(tok, r.p), r.end - 1) - r.p) * r.stride + c * 16;
    Vec8<T> lo[NC], hi[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        lo[i] = *reinterpret_cast<const Vec8<T>*>(src + i * 64);
        hi[i] = *reinterpret_cast<const Vec8<T>*>(src + i * 64 + 8);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[i][j] = fresh ? static_cast<float>(lo[i].v[j]) : 0.0f;
            x[i][8 + j] = fresh ? static_cast<float>(hi[i].v[j]) : 0.0f;
        }
    }
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            amax = fmaxf(amax, row_magnitude(x[i][j]));
        }
    const float s = joined_scale(wave_max(amax), r.held, r.old);
    const bool poisoned = s != s;
    const float inv = poisoned ? 0.0f : pow2_inverse(s);
    const float ratio = r.old * inv;
    const bool requantize = r.held && !poisoned && r.old != s;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int at = (c + 4 * i) * (kBlockRows * 16) + t * 16;
        v4i w = {0, 0, 0, 0};
        if (fresh && !poisoned) {
#pragma unroll
            for (int j = 0; j < 16; ++j) w[j >> 2] |= static_cast<int32_t>(code_byte(x[i][j] * inv) << (8 * (j & 3)));
        }
        if (requantize && !fresh) {
            w = rescaled(*reinterpret_cast<const v4i*>(record + at), ratio);
        }
        if (fresh || !r.held || requantize) *reinterpret_cast<v4i*>(record + at) = w;
    }
    return s;
}

// The same for V: lane = channels NC * lane .., each a run of 16 tokens that the
// lane alone holds, so new bytes merge into it without a race.
template <typename T, int HD>
__device__ __forceinline__ float append_v(const BlockRows<T>& r, int8_t* record, int lane) {
    constexpr int NC = HD / 64;
    struct alignas(sizeof(T) * NC) Pack { T v[NC]; };
    const T* src = r.rows + lane * NC;
    v4i o[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        o[i] = v4i{0, 0, 0, 0};
        if (r.held) o[i] = *reinterpret_cast<const v4i*>(record + (lane * NC + i) * kBlockRows);
    }
    float x[kBlockRows][NC];
    float amax = 0.0f;
#pragma unroll
    for (int t = 0; t < kBlockRows; ++t) {
        const int tok = r.tok0 + t;
        const Pack w = *reinterpret_cast<const Pack*>(src + (min(max(tok, r.p), r.end - 1) - r.p) * r.stride);
#pragma unroll
        for (int i = 0; i < NC; ++i) x[t][i] = tok >= r.p && tok < r.end ? static_cast<float>(w.v[i]) : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < kBlockRows; ++t)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            amax = fmaxf(amax, row_magnitude(x[t][i]));
        }
    const float s = joined_scale(wave_max(amax), r.held, r.old);
    const bool poisoned = s != s;
    const float inv = poisoned ? 0.0f : pow2_inverse(s);
    const float ratio = r.old == s || poisoned ? 1.0f : r.old * inv;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        v4i w = {0, 0, 0, 0};
#pragma unroll
        for (int t = 0; t < kBlockRows; ++t) {
            const int tok = r.tok0 + t;
            const bool fresh = tok >= r.p && tok < r.end;
            const float kept = byte_value(static_cast<uint32_t>(o[i][t >> 2]), t & 3) * ratio;
            const float v = fresh ? (poisoned ? 0.0f : x[t][i] * inv) : kept;
            w[t >> 2] |= static_cast<int32_t>(code_byte(v) << (8 * (t & 3)));
        }
        *reinterpret_cast<v4i*>(record + (lane * NC + i) * kBlockRows) = w;
    }
    return s;
}

// Workgroup (key/value head, touched block, sequence): wave 0 appends the
// block's K rows, wave 1 its V rows.  Reading the rows and writing the codes
// bound it.
template <typename T, int HD>
__global__ __launch_bounds__(128) void block_append_kernel(const BlockRowsArgs a) {
    const int kh = blockIdx.x, b = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int p = a.positions[b];
    if (p < 0) return;
    const int blk = p / kBlockRows + static_cast<int>(blockIdx.y);
    BlockRows<T> r;
    r.tok0 = blk * kBlockRows;
    r.p = p;
    r.end = p + a.n;
    if (r.tok0 >= r.end) return;
    const int64_t page = block_page(a.view, a.slot0 + b, a.layer, kh);
    int8_t* const base = a.view.base + page * a.view.page_bytes;
    const int rec = a.view.table[page * a.view.blocks + blk];
    int8_t* const record = base + static_cast<int64_t>(rec) * (2 * kBlockRows * HD) + wave * (kBlockRows * HD);
    float* const scale = reinterpret_cast<float*>(base + static_cast<int64_t>(a.view.blocks) * (2 * kBlockRows * HD)) +
                         2 * rec + wave;
    r.stride = wave == 0 ? a.k_stride : a.v_stride;
    r.rows = static_cast<const T*>(wave == 0 ? a.k : a.v) + static_cast<int64_t>(b) * a.n * r.stride + kh * HD;
    r.held = r.tok0 < p;
    r.old = r.held ? *scale : 0.0f;
    const float s = wave == 0 ? append_k<T, HD>(r, record, lane) : append_v<T, HD>(r, record, lane);
    if (lane == 0 && !(r.held && r.old == s)) *scale = s;
}

// The reverse, with the same lanes: values of cached rows, rounded once.
template <typename T, int HD>
__global__ __launch_bounds__(128) void block_values_kernel(const BlockRowsArgs a) {
    constexpr int NC = HD / 64;
    const int kh = blockIdx.x, b = blockIdx.z;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int p = a.positions[b];
    if (p < 0) return;
    const int blk = p / kBlockRows + static_cast<int>(blockIdx.y);
    const int tok0 = blk * kBlockRows, end = p + a.n;
    if (tok0 >= end) return;
    const int64_t page = block_page(a.view, a.slot0 + b, a.layer, kh);
    const int8_t* const base = a.view.base + page * a.view.page_bytes;
    const int rec = a.view.table[page * a.view.blocks + blk];
    const int8_t* const record = base + static_cast<int64_t>(rec) * (2 * kBlockRows * HD) + wave * (kBlockRows * HD);
    const float s = reinterpret_cast<const float*>(base + static_cast<int64_t>(a.view.blocks) * (2 * kBlockRows * HD))[
        2 * rec + wave];
    const int64_t row0 = static_cast<int64_t>(b) * a.n - p;
    const int64_t stride = static_cast<int64_t>(a.view.kv_heads) * HD;
    if (wave == 0) {
        const int t = lane >> 2, c = lane & 3, tok = tok0 + t;
        if (tok < p || tok >= end) return;
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const v4i o = *reinterpret_cast<const v4i*>(record + (c + 4 * i) * (kBlockRows * 16) + t * 16);
            T* dst = static_cast<T*>(a.k_out) + (row0 + tok) * stride + kh * HD + (c + 4 * i) * 16;
            Vec8<T> w[2];
#pragma unroll
            for (int j = 0; j < 16; ++j)
                w[j >> 3].v[j & 7] = static_cast<T>(byte_value(static_cast<uint32_t>(o[j >> 2]), j & 3) * s);
            *reinterpret_cast<Vec8<T>*>(dst) = w[0];
            *reinterpret_cast<Vec8<T>*>(dst + 8) = w[1];
        }
    } else {
        v4i o[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) o[i] = *reinterpret_cast<const v4i*>(record + (lane * NC + i) * kBlockRows);
        T* dst = static_cast<T*>(a.v_out) + kh * HD + lane * NC;
#pragma unroll
        for (int t = 0; t < kBlockRows; ++t) {
            const int tok = tok0 + t;
            if (tok < p || tok >= end) continue;
            struct alignas(sizeof(T) * NC) Pack { T v[NC]; } w;
#pragma unroll
            for (int i = 0; i < NC; ++i)
                w.v[i] = static_cast<T>(byte_value(static_cast<uint32_t>(o[i][t >> 2]), t & 3) * s);
            *reinterpret_cast<Pack*>(dst + (row0 + tok) * stride) = w;
        }
    }
}

__global__ __launch_bounds__(256) void block_table_kernel(uint16_t* table, int64_t n, int blocks) {
    const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; i < n; i += step)
        table[i] = static_cast<uint16_t>(i % blocks);
}

// ---------------------------------------------------------------- attention

// softmax(scale q k^T) v of the rows of one chunk -- query tokens times the
// query heads that share a key/value head, 4, 8 or 16 of them -- over the
// tiles of one split.  Both products run on the 8-bit matrix instructions
// straight from the codes (D[16][16] += A[16][64] B[64][16]):
//
//   scores  A: the queries as integers q = m 2^E (E for a row, |m| <= 2^30), the
//           four signed bytes of m as four rows, so a 16-row A holds 4 queries;
//           B: the K codes as they lie.  The byte sums are exact; one lane has the
//           four of a (row, token) and joins them into m.k.
//   output  A: p v as a fraction of 2^30, in four signed bytes, p = 2^(score - the tile's
//           largest), v its block's V scale, over the power of two above the largest p v
//           that the row has in the tile (a block's scale alone says nothing: the row may
//           not see the block, or hardly weigh it);
//           B: the V codes as they lie, 64 tokens of 16 channels at a time.
//
// So a code is never converted, the operator is bound by reading the codes
// (2 * head_dim + 0.5 bytes a token), and what a product rounds is 2^-30 of a
// row's largest query value and 2^-30 of its largest p v in a tile: less than
// FP32 products would.
//
// Wave w takes tiles w, w + 4, ... of the split, each with its own running
// (max, sum, output); the waves meet in LDS.  A tile's loads all go out together;
// with up to 4 rows four workgroups fill a CU (128 registers), so that others' loads
// fly while one computes: 64 sequences x 32 heads of 4096 tokens 308 us, 7.0 TB/s.
// Asking for the next tile's codes ahead took 154 registers and 328 us.  Heads of 128
// with 8 rows take 161 to 178 registers (two or three workgroups a CU), with 16 rows 202
// to 256 (one), where little hides a tile's loads: 64 sequences of 4096 tokens, 8
// key/value heads, 86.5, 94 and 138 us for 4, 8 and 16 rows.
//
// ONCE (one row chunk, so each page is read once): the codes are read past the
// caches (nontemporal; 64 sequences of 4096 tokens, 8 key/value heads, 82 us
// against 100.6 in an earlier form), and the call's new rows may be appended here: each workgroup
// appends to the blocks of its own range, at most two (n <= 16), writes them to
// the cache and keeps them in LDS, from where the wave that scans their tile
// takes them.
//
// A sequence's splits publish (m, l, acc) with write-through stores and count
// themselves; the last to arrive joins them in split order, so the result does
// not depend on who that is.
constexpr int kAttendThreads = 256;
constexpr int kAttendWaves4 = 4;
constexpr int kDigitStride = kTileTokens + 16;   // bytes between rows of digits: rows of a 4-row step apart in banks
constexpr int kScaleBits = 127 - 100;            // exponent bits of the smallest scale
// A sum of weights times values may leave FP32's range where its quotient does not (2^17
// tokens, values below 2^127): a wave sums in a power of two of its own, 2^kUnitMin at
// least, and waves and splits join what they have over 2^kJoinExp.
constexpr float kUnitMin = -200.0f;
constexpr int kJoinExp = 18;

template <int HD, int RT>
struct AttendShared {
    static constexpr int kQueryBytes = RT * (HD / 64) * 1024;
    static constexpr int kDigitBytes = kAttendWaves4 * RT * 16 * kDigitStride;
    static constexpr int kRows = RT * kRowTile;
    static constexpr int kMergeBytes = kAttendWaves4 * kRows * (HD + 2) * 4;
    static constexpr int kScanBytes = kQueryBytes + kDigitBytes;
    static constexpr int kBytes = kScanBytes > kMergeBytes ? kScanBytes : kMergeBytes;
};

// The queries of a chunk as A operands: [row tile][64-channel step][lane][16
// bytes], lane = (chunk g of the step) * 16 + (row * 4 + byte); scales in q_scale.
//
// With b = 0x00808080 the bytes of (m + b) ^ b are the signed digits of m: adding
// b carries exactly where a byte's digit is negative.
constexpr uint32_t kDigitBias = 0x00808080u;
__device__ __forceinline__ uint32_t signed_digits(int32_t m) {
    return (static_cast<uint32_t>(m) + kDigitBias) ^ kDigitBias;
}

// Bytes k of four words, as one word.
__device__ __forceinline__ uint32_t bytes_of(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, int k) {
    const uint32_t low = __builtin_amdgcn_perm(w1, w0, 0x0c0c0400u + 0x0101u * k);
    const uint32_t high = __builtin_amdgcn_perm(w3, w2, 0x04000c0cu + 0x01010000u * k);
    return low | high;
}

template <typename T, int HD, int RT>
__device__ __forceinline__ void stage_queries(const BlockAttendArgs& a, int b, int kh, int row_first, int rows,
                                              uint8_t* lds, float* q_scale) {
    constexpr int kPieces = HD / 8;              // lanes of a row, 8 channels each
    static_assert(RT * kRowTile * kPieces <= kAttendThreads, "a row's piece for each thread");
    const int row = threadIdx.x / kPieces, piece = threadIdx.x % kPieces;
    if (row >= RT * kRowTile) return;
    const int r = row_first + min(row, rows - 1), i = row_token(a, r);
    const Vec8<T> w = *reinterpret_cast<const Vec8<T>*>(
        static_cast<const T*>(a.q) + (static_cast<int64_t>(b) * a.n + i) * a.q_stride +
        (kh * a.group + r - i * a.group) * HD + piece * 8);
    float x[8];
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        x[j] = row < rows ? static_cast<float>(w.v[j]) : 0.0f;
        amax = fmaxf(amax, fabsf(x[j]) <= kFloatMax ? fabsf(x[j]) : INFINITY);
    }
#pragma unroll
    for (int d = 1; d < kPieces; d <<= 1) amax = fmaxf(amax, __shfl_xor(amax, d));
    const bool poison = amax == INFINITY;
    const int e = poison ? 0 : max(static_cast<int>(__float_as_uint(amax) >> 23) - 126, -90);   // amax < 2^e
    if (piece == 0) q_scale[row] = poison ? __builtin_nanf("") : ldexpf(a.scale, e - 30);
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)                  // |m| <= 2^30
        u[j] = signed_digits(poison ? 0 : static_cast<int32_t>(__builtin_rintf(ldexpf(x[j], 30 - e))));
    // 8 channels: half (piece & 1) of chunk piece / 2 = 4 * step + g
    const int chunk = piece >> 1, step = chunk >> 2, g = chunk & 3;
    uint8_t* dst = lds + (((row >> 2) * (HD / 64) + step) * 64 + g * 16 + (row & 3) * 4) * 16 + (piece & 1) * 8;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        *reinterpret_cast<v2u*>(dst + k * 16) = v2u{bytes_of(u[0], u[1], u[2], u[3], k), bytes_of(u[4], u[5], u[6], u[7], k)};
}

__device__ __forceinline__ float row16_max_f(float x) {
    x = fmaxf(x, dpp_f<kDppQuadXor1>(x));
    x = fmaxf(x, dpp_f<kDppQuadXor2>(x));
    x = fmaxf(x, dpp_f<kDppHalfMirror>(x));
    return fmaxf(x, dpp_f<kDppRowRor8>(x));
}
__device__ __forceinline__ float row16_sum_f(float x) {
    x += dpp_f<kDppQuadXor1>(x);
    x += dpp_f<kDppQuadXor2>(x);
    x += dpp_f<kDppHalfMirror>(x);
    return x + dpp_f<kDppRowRor8>(x);
}

// A workgroup appends the call's rows to the (at most two) blocks `first` ..
// of its range: to the cache and to `tail`, whose copies the scan reads.  Small
// code, for it runs once a workgroup: its rows are few.
template <typename T, int HD>
__device__ __forceinline__ void append_here(const BlockAttendArgs& a, int b, int kh, int p, int first, int touched,
                                            int64_t page, int8_t* base, int8_t* scale_base, int8_t* tail,
                                            uint32_t* tail_max, float* tail_scale) {
    constexpr int NC = HD / 64, kRecord = 2 * kBlockRows * HD, kPieces = kRecord / 16;
    struct alignas(sizeof(T) * NC) Pack { T v[NC]; };
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int piece = min(tid, kPieces - 1), is_v = piece >= kPieces / 2;       // a thread's 16 bytes of a record
    int rec[2];
    v4i o[2];
    float old[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        rec[t] = a.view.table[page * a.view.blocks + min(first + t, first + touched - 1)];
        o[t] = *reinterpret_cast<const v4i*>(base + static_cast<int64_t>(rec[t]) * kRecord + piece * 16);
        old[t] = reinterpret_cast<const float*>(scale_base)[2 * rec[t] + is_v];
    }
    if (tid < 4) tail_max[tid] = 0;
    __syncthreads();
    // A wave takes the K or the V part of one row after another.
    auto rows = [&](auto&& f) {
        for (int i = wave; i < 2 * a.n; i += kAttendWaves4) {
            const int tok = p + (i >> 1), t = tok / kBlockRows - first;
            if (t < 0 || t >= touched) continue;
            const T* src = static_cast<const T*>(i & 1 ? a.v : a.k) +
                           (static_cast<int64_t>(b) * a.n + (i >> 1)) * (i & 1 ? a.v_stride : a.k_stride) + kh * HD;
            const Pack w = *reinterpret_cast<const Pack*>(src + lane * NC);
            f(w, i & 1, t, tok % kBlockRows);
        }
    };
    rows([&](const Pack& w, int v, int t, int) {
        float amax = 0.0f;
#pragma unroll
        for (int i = 0; i < NC; ++i) amax = fmaxf(amax, row_magnitude(static_cast<float>(w.v[i])));
        amax = wave_max(amax);
        if (lane == 0) atomicMax(&tail_max[2 * t + v], __float_as_uint(amax));
    });
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        if (t >= touched || tid >= kPieces) continue;
        const bool held = (first + t) * kBlockRows < p;
        const float s = joined_scale(__uint_as_float(tail_max[2 * t + is_v]), held, old[t]);
        if (!held) o[t] = v4i{0, 0, 0, 0};
        else if (s > old[t]) o[t] = rescaled(o[t], old[t] * pow2_inverse(s));
        *reinterpret_cast<v4i*>(tail + t * kRecord + piece * 16) = o[t];
        if (piece % (kPieces / 2) == 0) {
            tail_scale[2 * t + is_v] = s;
            reinterpret_cast<float*>(scale_base)[2 * rec[t] + is_v] = s;
        }
    }
    __syncthreads();
    rows([&](const Pack& w, int v, int t, int slot) {
        const float s = tail_scale[2 * t + v], inv = s != s ? 0.0f : pow2_inverse(s);
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            const int c = lane * NC + i;
            const float x = s != s ? 0.0f : static_cast<float>(w.v[i]) * inv;
            tail[t * kRecord + (v ? kBlockRows * HD + c * kBlockRows + slot : (c >> 4) * (kBlockRows * 16) + slot * 16 + (c & 15))] =
                static_cast<int8_t>(code_byte(x));
        }
    });
    __syncthreads();
#pragma unroll
    for (int t = 0; t < 2; ++t)
        if (t < touched && tid < kPieces)
            *reinterpret_cast<v4i*>(base + static_cast<int64_t>(rec[t]) * kRecord + piece * 16) =
                *reinterpret_cast<const v4i*>(tail + t * kRecord + piece * 16);
}

template <typename T, int HD, int RT, bool LSE, bool ONCE>
__global__ __launch_bounds__(kAttendThreads, RT == 4 ? 1 : RT == 2 ? 2 : 4) void block_attend_kernel(const BlockAttendArgs a) {
    using S = AttendShared<HD, RT>;
    constexpr int NS = HD / 64;                  // 64-channel steps of a score
    constexpr int ND = HD / 16;                  // 16-channel tiles of an output
    constexpr int kPolicy = ONCE ? 2 : 0;        // nontemporal
    constexpr int kRecord = 2 * kBlockRows * HD;
    constexpr int kRows = S::kRows;
    __shared__ __align__(16) uint8_t lds[S::kBytes];
    __shared__ __align__(16) int8_t tail[ONCE ? 2 * kRecord : 16];   // the blocks that this call appends to
    __shared__ uint32_t tail_max[4];
    __shared__ float tail_scale[4];
    __shared__ float q_scale[kRows];
    __shared__ uint32_t arrived;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g = lane >> 4, n16 = lane & 15;
    const int b = a.order[blockIdx.y];
    int id = blockIdx.x;
    const int kh = id % a.view.kv_heads;         // heads fastest: a head's workgroups share an XCD's L2
    id /= a.view.kv_heads;
    const int split = id % a.splits, chunk = id / a.splits;
    const int all_rows = a.group * a.n;
    const int row_first = chunk * kRows, rows = min(kRows, all_rows - row_first);
    const int p = a.positions[b];
    // tokens that the chunk's last row sees
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
    int8_t* const scale_base = base + static_cast<int64_t>(a.view.blocks) * kRecord;

    // A tile's codes, by the two halves of its table entry.
    v4i kb[kTileBlocks][NS], vb[ND];
    auto load_k = [&](uint32_t low, uint32_t high) {
#pragma unroll
        for (int j = 0; j < kTileBlocks; ++j) {
            const int at = static_cast<int>(((j & 2 ? high : low) >> (16 * (j & 1))) & 0xffffu) * kRecord;
#pragma unroll
            for (int s = 0; s < NS; ++s)
                kb[j][s] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, lane * 16, at + s * 1024, kPolicy);
        }
    };
    auto load_v = [&](uint32_t low, uint32_t high) {
        const uint32_t mine = ((g & 2 ? high : low) >> (16 * (g & 1))) & 0xffffu;
        const int at = static_cast<int>(mine) * kRecord + kBlockRows * HD + n16 * 16;
#pragma unroll
        for (int i = 0; i < ND; ++i) vb[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at, i * 256, kPolicy);
    };

    // (a wave without a tile, and lanes past its last, ask for the split's last)
    const int last_tile = max(tile_begin, tile_end - 1);
    int tile0 = tile_begin + wave;               // first of the 64 tiles whose heads the wave holds
    TileHeads heads;
    auto start = [&]() {
        heads.load_entries(table, tile0 + lane * kAttendWaves4, last_tile);
        heads.load_scales(scale_base);
    };
    start();

    stage_queries<T, HD, RT>(a, b, kh, row_first, rows, lds, q_scale);
    // Blocks of this range that new rows go to.
    int touch_begin = tile_end * kTileBlocks, touched = 0;
    if (ONCE && a.k != nullptr && p >= 0) {
        touch_begin = max(p / kBlockRows, tile_begin * kTileBlocks);
        touched = min((p + a.n - 1) / kBlockRows + 1, tile_end * kTileBlocks) - touch_begin;
    }

    if (touched > 0) append_here<T, HD>(a, b, kh, p, touch_begin, touched, page, base, scale_base, tail, tail_max, tail_scale);
    __syncthreads();

    v4i qa[RT][NS];
    float qs[RT], m_run[RT], l_run[RT];
    float acc[RT][ND], unit[RT];                 // acc counts in 2^(m_run + unit)
    int limit[RT];                               // tokens that row (rt, g) sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
        for (int s = 0; s < NS; ++s) qa[rt][s] = *reinterpret_cast<const v4i*>(lds + ((rt * NS + s) * 64 + lane) * 16);
        const int row = rt * kRowTile + g;
        qs[rt] = q_scale[row];
        limit[rt] = row < rows && p >= 0 ? p + row_token(a, row_first + row) + 1 : 0;
        m_run[rt] = -INFINITY;
        l_run[rt] = 0.0f;
        unit[rt] = kUnitMin;
#pragma unroll
        for (int i = 0; i < ND; ++i) acc[rt][i] = 0.0f;
    }
    // Which bytes a lane k of a quad takes: of its own word and its neighbours' (k ^ 1,
    // then k ^ 2 and k ^ 3), byte k of token i to place i.
    const int k4 = n16 & 3;
    auto at_place = [](int byte, int place) { return static_cast<uint32_t>(byte) << (8 * place); };
    const uint32_t turn_a = (0x0c0c0c0cu & ~(at_place(0xff, k4) | at_place(0xff, k4 ^ 1))) | at_place(k4, k4) |
                            at_place(4 + k4, k4 ^ 1);
    const uint32_t turn_b = (0x0c0c0c0cu & ~(at_place(0xff, k4 ^ 2) | at_place(0xff, k4 ^ 3))) | at_place(k4, k4 ^ 2) |
                            at_place(4 + k4, k4 ^ 3);
    uint8_t* const digits = lds + S::kQueryBytes + wave * (RT * 16 * kDigitStride);
    const int64_t head_row = (static_cast<int64_t>(b) * a.view.kv_heads + kh) * all_rows + row_first;

    // One tile.  FROM_LDS: it has blocks that this call appends to, which come
    // from LDS over what was loaded; such a tile is its wave's last.  (A second
    // body, not a branch in one: the loop would wait for all loads at its join.)
    auto scan = [&](auto from_lds, int tile, int at) {
        TileHead head;
        const uint32_t low = heads.low(at), high = heads.high(at);
        load_k(low, high);
        load_v(low, high);
        __builtin_amdgcn_sched_barrier(0);
        heads.scales_of(at, head);
        if constexpr (decltype(from_lds)::value) {
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
                const int t = tile * kTileBlocks + j - touch_begin;
                if (t < 0 || t >= touched) continue;
#pragma unroll
                for (int s = 0; s < NS; ++s)
                    kb[j][s] = *reinterpret_cast<const v4i*>(tail + t * kRecord + s * 1024 + lane * 16);
                if (g == j) {
#pragma unroll
                    for (int i = 0; i < ND; ++i)
                        vb[i] = *reinterpret_cast<const v4i*>(tail + t * kRecord + kBlockRows * HD + i * 256 + n16 * 16);
                }
                head.ks[j] = tail_scale[2 * t];
                head.vs[j] = tail_scale[2 * t + 1];
            }
        }
        const int tok0 = tile * kTileTokens;

        float s[RT][kTileBlocks];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
                v4i c = {0, 0, 0, 0};
#pragma unroll
                for (int k = 0; k < NS; ++k) c = __builtin_amdgcn_mfma_i32_16x16x64_i8(qa[rt][k], kb[j][k], c, 0, 0, 0);
                const float lower = static_cast<float>(c[0] + c[1] * 256);     // below 2^30
                const float upper = static_cast<float>(c[2] + c[3] * 256);
                s[rt][j] = __builtin_fmaf(upper, 65536.0f, lower) * (qs[rt] * head.ks[j]);
                if (tok0 + kBlockRows * j + n16 >= limit[rt]) s[rt][j] = -INFINITY;
            }

        v4i pa[RT];
        float acc_mul[RT], v_mul[RT], block_sum[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float top = -INFINITY;
            bool poison = false;                 // by a V scale that is not a number, where the row sees its block
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
                if (head.vs[j] != head.vs[j] && tok0 + kBlockRows * j < limit[rt]) poison = true;
                top = fmaxf(top, s[rt][j]);
            }
            top = row16_max_f(top);
            const float top_safe = top == -INFINITY ? 0.0f : top;    // a row that sees nothing here
            float sum = 0.0f, largest = 0.0f;    // of the weights times their V scales
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
                const float w = fast_exp2(s[rt][j] - top_safe);
                s[rt][j] = w;
                sum += w;
                largest = fmaxf(largest, w * head.vs[j]);
            }
            // largest < 2^(e - 126)
            const int e = max(static_cast<int>(__float_as_uint(row16_max_f(largest)) >> 23), kScaleBits);
#pragma unroll
            for (int j = 0; j < kTileBlocks; ++j) {
                const uint32_t u = signed_digits(static_cast<int32_t>(__builtin_rintf(ldexpf(s[rt][j] * head.vs[j], 156 - e))));
                // The four lanes of a quad turn their words (a token's digits) into
                // digit n16 & 3 of the quad's four tokens.
                const uint32_t x1 = dpp_u<kDppQuadXor1>(u), x2 = dpp_u<kDppQuadXor2>(u), x3 = dpp_u<kDppQuadXor1>(x2);
                const uint32_t turned = __builtin_amdgcn_perm(x1, u, turn_a) | __builtin_amdgcn_perm(x3, x2, turn_b);
                *reinterpret_cast<uint32_t*>(digits + (rt * 16 + g * 4 + (n16 & 3)) * kDigitStride + j * kBlockRows +
                                             (n16 & ~3)) = turned;
            }
            if (LSE) {
                // log2 of each block's sum, by the lane n16 == j
                float mine_sum = 0.0f;
#pragma unroll
                for (int j = 0; j < kTileBlocks; ++j) {
                    const float t = row16_sum_f(s[rt][j]);
                    if (n16 == j) mine_sum = t;
                }
                block_sum[rt] = top_safe + __log2f(mine_sum);
            }
            const float m_new = fmaxf(m_run[rt], top);
            const float m_safe = m_new == -INFINITY ? 0.0f : m_new;
            const float fall = m_run[rt] - m_safe, below = top - m_safe;   // 0 or less
            l_run[rt] = l_run[rt] * fast_exp2(fall) + sum * fast_exp2(below);
            m_run[rt] = m_new;
            const float tile_unit = static_cast<float>(e - 126);
            const float to = fmaxf(fmaxf(unit[rt] + ceilf(fall), tile_unit + ceilf(below)), kUnitMin);
            acc_mul[rt] = fast_exp2(fall + (unit[rt] - to));
            v_mul[rt] = poison ? __builtin_nanf("") : fast_exp2(below + (tile_unit - 30.0f - to));
            unit[rt] = to;
        }
        // The digits were written by other lanes of this wave, whose LDS accesses
        // stay in order; the fences keep the compiler to it.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
            pa[rt] = *reinterpret_cast<const v4i*>(digits + (rt * 16 + n16) * kDigitStride + g * 16);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int i = 0; i < ND; ++i)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                v4i c = {0, 0, 0, 0};
                c = __builtin_amdgcn_mfma_i32_16x16x64_i8(pa[rt], vb[i], c, 0, 0, 0);
                const float lower = static_cast<float>(c[0] + c[1] * 256);     // below 2^29
                const float upper = static_cast<float>(c[2] + c[3] * 256);
                acc[rt][i] = __builtin_fmaf(__builtin_fmaf(upper, 65536.0f, lower), v_mul[rt], acc[rt][i] * acc_mul[rt]);
            }
        if (LSE) {
            // The lane n16 == j < 4 has block j's.
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                const int row = rt * kRowTile + g;
                if (n16 < kTileBlocks && row < rows) {
                    float* dst = a.block_lse + (head_row + row) * a.view.blocks + tile * kTileBlocks + n16;
                    if (my_splits > 1) publish(dst, block_sum[rt]);
                    else *dst = block_sum[rt];
                }
            }
        }
    };
    const int plain_end = min(tile_end, touch_begin / kTileBlocks);     // tiles without appended blocks end here
    while (tile0 < tile_end) {
        heads.arrive();
        const int end = min(tile_end, tile0 + 64 * kAttendWaves4);
        int tile = tile0, at = 0;
        for (; tile < min(end, plain_end); tile += kAttendWaves4, ++at)
            scan(std::false_type{}, tile, at);
        if (ONCE && tile < end) scan(std::true_type{}, tile, at);
        tile0 += 64 * kAttendWaves4;
        if (tile0 < tile_end) start();
    }

    // With weights: the block that the thread adds first, its weight until now and
    // its log-sums of each row, asked for before the joins that they wait for.
    float* const weights = LSE && ONCE ? a.weights + (static_cast<int64_t>(b) * a.view.kv_heads + kh) * a.view.blocks : nullptr;
    const int first_blk = min(static_cast<int>(threadIdx.x), a.view.blocks - 1);
    float first_weight = 0.0f, first_sums[LSE && ONCE ? kRows : 1];
    auto ask_sums = [&]() {
        if constexpr (LSE && ONCE) {
            first_weight = weights[first_blk];
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                first_sums[r] = fetch(a.block_lse + (head_row + min(r, rows - 1)) * a.view.blocks + first_blk);
        }
    };
    // The waves' partials meet in LDS.
    if (LSE) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");    // the block sums have arrived
    __syncthreads();
    if (my_splits == 1) ask_sums();
    float* const merge = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float* dst = merge + (wave * kRows + rt * kRowTile + g) * (HD + 2);
        const float l = row16_sum_f(l_run[rt]);
        if (n16 == 0) {
            dst[0] = m_run[rt];
            dst[1] = l;
        }
#pragma unroll
        for (int i = 0; i < ND; ++i) dst[2 + i * 16 + n16] = ldexpf(acc[rt][i], static_cast<int>(unit[rt]) - kJoinExp);
    }
    __syncthreads();
    constexpr int kItems = kRows * HD / kAttendThreads;      // outputs of a thread
    const int64_t pair = (static_cast<int64_t>(b) * a.view.kv_heads + kh) * a.chunks + chunk;
    float* const partial = a.partials + pair * a.splits * kRows * (HD + 2);
    float m_all[kItems], l_all[kItems], o_all[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int i = threadIdx.x + k * kAttendThreads, row = i / HD, d = i % HD;
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < kAttendWaves4; ++w) m = fmaxf(m, merge[(w * kRows + row) * (HD + 2)]);
        const float m_safe = m == -INFINITY ? 0.0f : m;
        float l = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < kAttendWaves4; ++w) {
            const float* src = merge + (w * kRows + row) * (HD + 2);
            const float f = fast_exp2(src[0] - m_safe);
            l = __builtin_fmaf(src[1], f, l);
            o = __builtin_fmaf(src[2 + d], f, o);
        }
        m_all[k] = m;
        l_all[k] = l;
        o_all[k] = o;
        if (my_splits > 1) {
            float* dst = partial + (static_cast<int64_t>(split) * kRows + row) * (HD + 2);
            if (d == 0) {
                publish(dst, m);
                publish(dst + 1, l);
            }
            publish(dst + 2 + d, o);
        }
    }
    if (my_splits > 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // what was published has arrived
    __syncthreads();
    if (my_splits > 1) {
        uint32_t* const counter = a.counters + pair * kCounterStride;
        if (threadIdx.x == 0)
            arrived = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        __syncthreads();
        if (static_cast<int>(arrived) != my_splits - 1) return;
        // The last split: everybody's partials, in split order.  The counter is
        // zero again for the next launch.
        if (threadIdx.x == 0) __hip_atomic_store(counter, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        ask_sums();
#pragma unroll
        for (int k = 0; k < kItems; ++k) {
            const int i = threadIdx.x + k * kAttendThreads, row = i / HD, d = i % HD;
            join_splits<false>(partial + row * (HD + 2), kRows * (HD + 2), my_splits, d, m_all[k], l_all[k], o_all[k]);
        }
    }
    float* const lse = merge;                    // log2 of each row's sum
    if (LSE) __syncthreads();
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
        const int i = threadIdx.x + k * kAttendThreads, row = i / HD, d = i % HD;
        if (row >= rows) break;
        const int r = row_first + row, i_q = row_token(a, r);
        const int64_t token = static_cast<int64_t>(b) * a.n + i_q;
        static_cast<T*>(a.out)[token * a.out_stride + (kh * a.group + r - i_q * a.group) * HD + d] =
            static_cast<T>(l_all[k] == 0.0f ? 0.0f : o_all[k] / l_all[k] * (1 << kJoinExp));
        if (LSE && d == 0) {
            const float v = (m_all[k] == -INFINITY ? 0.0f : m_all[k]) + __log2f(l_all[k]);
            if (ONCE) lse[row] = v;
            else a.row_lse[head_row + row] = v;
        }
    }
    if (LSE && ONCE) {
        // All rows are here: weights[block] += sum over rows of 2^(the block's
        // log-sum - the row's), rows in order.
        __syncthreads();
        if (p < 0) return;
        const int held = (p + a.n - 1) / kBlockRows + 1;
        if (static_cast<int>(threadIdx.x) < held) {
            float sum = 0.0f;
#pragma unroll
            for (int r = 0; r < kRows; ++r)
                if (r < rows && first_blk * kBlockRows <= p + row_token(a, r)) sum += fast_exp2(first_sums[r] - lse[r]);
            weights[first_blk] = first_weight + sum;
        }
        for (int blk = threadIdx.x + kAttendThreads; blk < held; blk += kAttendThreads) {
            float sum = 0.0f;
            for (int r = 0; r < rows; ++r)
                if (blk * kBlockRows <= p + row_token(a, r))
                    sum += fast_exp2(fetch(a.block_lse + (head_row + r) * a.view.blocks + blk) - lse[r]);
            weights[blk] += sum;
        }
    }
}

// weights[block] += sum over rows of 2^(the block's log-sum - the row's): rows in
// order, so a block's sum has one order whatever ran first.
__global__ __launch_bounds__(256) void block_weights_kernel(const BlockAttendArgs a) {
    const int blk = blockIdx.x * 256 + threadIdx.x, kh = blockIdx.y, b = blockIdx.z;
    const int p = a.positions[b], rows = a.group * a.n;
    if (p < 0 || blk * kBlockRows >= p + a.n) return;
    const int64_t head = static_cast<int64_t>(b) * a.view.kv_heads + kh;
    float sum = 0.0f;
    for (int r = 0; r < rows; ++r)
        if (blk * kBlockRows <= p + r / a.group)
            sum += fast_exp2(a.block_lse[(head * rows + r) * a.view.blocks + blk] - a.row_lse[head * rows + r]);
    a.weights[head * a.view.blocks + blk] += sum;
}

// ---------------------------------------------------------------- eviction

// Workgroup (kv head, sequence, layer); a thread has blocks tid, tid + 256, ...
// (PER of them) in registers.  The smallest weight that stays is found by three
// passes over the weights' bits, 11 from the top, 11 and 9 (non-negative floats
// order as their bits): a histogram in LDS, then the bin where the count from the
// top reaches what is wanted.  (8-bit passes put the few exponents of real weights
// into few bins, whose atomics wait for each other: 32 layers x 8 sequences x 8
// heads of 2032 blocks took 32.8 us.)  Ballots and one prefix over (turn, wave)
// give each block its place.  A few KiB are read and written a workgroup: latency
// bounds it, twice where PER is 8, whose 88 registers leave 1280 of those 2048
// workgroups resident.  That launch takes 21.6 us on weights as they gather, and 20.5 on
// what an eviction left, mostly zeros.
constexpr int kEvictThreads = 256;
constexpr int kEvictBins = 2048;

// counts[0 .. n) -> exclusive prefix, by one wave; n <= 128.
__device__ __forceinline__ void prefix_counts(uint32_t* counts, int n, int lane) {
    const uint32_t c0 = 2 * lane < n ? counts[2 * lane] : 0, c1 = 2 * lane + 1 < n ? counts[2 * lane + 1] : 0;
    uint32_t sum = c0 + c1;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const uint32_t t = __shfl_up(sum, d);
        if (lane >= d) sum += t;
    }
    sum -= c0 + c1;
    if (2 * lane < n) counts[2 * lane] = sum;
    if (2 * lane + 1 < n) counts[2 * lane + 1] = sum + c0;
}

template <int PER>
__global__ __launch_bounds__(kEvictThreads) void block_evict_kernel(const BlockEvictArgs a) {
    __shared__ __align__(16) uint32_t bins[kEvictBins];
    __shared__ uint32_t found[2];                // the bin, and how many keys lie above it
    __shared__ uint32_t wave_sum[4];
    __shared__ uint32_t counts[2][4 * PER];      // of each (turn, wave): equal to the threshold; staying
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int kh = blockIdx.x, b = blockIdx.y, blocks = a.view.blocks;
    const int p = a.positions[b];
    if (p < 0) return;
    const int nb = (p + kBlockRows - 1) / kBlockRows;
    const int64_t row = (static_cast<int64_t>(blockIdx.z) * a.batch + a.b0 + b) * a.view.kv_heads + kh;
    float* const weights = a.weights + row * blocks;
    int32_t* const kept = a.kept ? a.kept + row * a.keep : nullptr;
    if (nb <= a.keep) {
        for (int i = nb + tid; i < blocks; i += kEvictThreads) weights[i] = 0.0f;
        if (kept)
            for (int i = tid; i < a.keep; i += kEvictThreads) kept[i] = i < nb ? i : -1;
        return;
    }
    uint16_t* const table = a.view.table + block_page(a.view, a.slot0 + a.b0 + b, a.layer0 + blockIdx.z, kh) * blocks;
    float w[PER];
    uint16_t old[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = min(k * kEvictThreads + tid, nb - 1);
        w[k] = weights[i];
        old[k] = table[i];
    }
    const int lo = a.sinks, hi = nb - a.recent;
    uint32_t want = a.keep - a.sinks - a.recent;     // of [lo, hi), which holds more
    uint32_t key[PER];                           // plus 1; 0 outside [lo, hi)
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * kEvictThreads + tid;
        key[k] = i >= lo && i < hi ? (w[k] > 0.0f ? __float_as_uint(w[k]) : 0u) + 1u : 0u;
    }
    uint32_t threshold = 0xffffffffu, prefix = 0;
    if (want > 0) {
        for (int pass = 0; pass < 3; ++pass) {
            const int shift = pass == 0 ? 20 : pass == 1 ? 9 : 0, above_bits = pass == 1 ? 11 : 9;
            uint4* const mine = reinterpret_cast<uint4*>(bins) + 2 * tid;
            mine[0] = mine[1] = make_uint4(0, 0, 0, 0);
            __syncthreads();
            uint32_t zeros = 0;                  // blocks nobody attended to: many, counted by the wave
#pragma unroll
            for (int k = 0; k < PER; ++k) {
                const uint32_t v = key[k] - 1;
                zeros += __popcll(__ballot(v == 0));
                if (key[k] > 1 && (pass == 0 || v >> (shift + above_bits) == prefix))
                    atomicAdd(&bins[(v >> shift) & (pass == 2 ? 511u : 2047u)], 1u);
            }
            if (lane == 0 && prefix == 0) atomicAdd(&bins[0], zeros);
            __syncthreads();
            const uint4 c0 = mine[0], c1 = mine[1];
            const uint32_t c[8] = {c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w};
            uint32_t sum = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += c[j];
            uint32_t above = sum;                // from the top lane down to this one
#pragma unroll
            for (int d = 1; d < 64; d <<= 1) {
                const uint32_t t = __shfl_down(above, d);
                if (lane + d < 64) above += t;
            }
            if (lane == 0) wave_sum[wave] = above;
            __syncthreads();
            above -= sum;
            for (int v = wave + 1; v < 4; ++v) above += wave_sum[v];
#pragma unroll
            for (int j = 7; j >= 0; --j) {
                if (above < want && above + c[j] >= want) {
                    found[0] = 8 * tid + j;
                    found[1] = above;
                }
                above += c[j];
            }
            __syncthreads();
            prefix = (prefix << (pass == 0 ? 0 : pass == 1 ? 11 : 9)) | found[0];
            want -= found[1];
        }
        threshold = prefix + 1;
    }
    // Keys above the threshold stay, and the first `want` that equal it.
    uint64_t equal[PER], stays[PER];
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        equal[k] = __ballot(key[k] == threshold);
        if (lane == 0) counts[0][4 * k + wave] = __popcll(equal[k]);
    }
    __syncthreads();
    if (wave == 0) prefix_counts(counts[0], 4 * PER, lane);
    __syncthreads();
    const uint64_t below = (1ull << lane) - 1;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * kEvictThreads + tid;
        const bool first = key[k] == threshold && counts[0][4 * k + wave] + __popcll(equal[k] & below) < want;
        stays[k] = __ballot(i < nb && (key[k] == 0 || (key[k] > threshold) || first));
        if (lane == 0) counts[1][4 * k + wave] = __popcll(stays[k]);
    }
    __syncthreads();
    if (wave == 0) prefix_counts(counts[1], 4 * PER, lane);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int i = k * kEvictThreads + tid;
        if (i >= nb) continue;
        const int at = counts[1][4 * k + wave] + __popcll(stays[k] & below);
        if ((stays[k] >> lane) & 1) {
            weights[at] = w[k];
            table[at] = old[k];
            if (kept) kept[at] = i;
        } else {
            table[a.keep + i - at] = old[k];
        }
    }
    for (int i = a.keep + tid; i < blocks; i += kEvictThreads) weights[i] = 0.0f;
}

}  // namespace

hipError_t launch_block_table(const BlockView& v, int64_t pages, hipStream_t s) {
    block_table_kernel<<<1024, 256, 0, s>>>(v.table, pages * v.blocks, v.blocks);
    return hipGetLastError();
}

namespace {
template <typename T, int HD>
void append_or_values(const BlockRowsArgs& a, int batch, bool values, hipStream_t s) {
    const dim3 grid(a.view.kv_heads, (a.n + 2 * kBlockRows - 2) / kBlockRows, batch);
    if (values) block_values_kernel<T, HD><<<grid, 128, 0, s>>>(a);
    else block_append_kernel<T, HD><<<grid, 128, 0, s>>>(a);
}
hipError_t launch_rows(const BlockRowsArgs& a, int batch, ElementType t, bool values, hipStream_t s) {
    with_type(t, [&](auto tag) {
        using T = decltype(tag);
        if (a.view.head_dim == 64) append_or_values<T, 64>(a, batch, values, s);
        else append_or_values<T, 128>(a, batch, values, s);
    });
    return hipGetLastError();
}

template <typename T, int HD, int RT, bool LSE>
void attend(const BlockAttendArgs& a, int batch, hipStream_t s) {
    const dim3 grid(a.view.kv_heads * a.splits * a.chunks, batch);
    if (a.chunks == 1) {
        block_attend_kernel<T, HD, RT, LSE, true><<<grid, kAttendThreads, 0, s>>>(a);
        return;
    }
    if constexpr (RT == kMaxRowTiles && LSE) {   // more rows without weights: the prompt kernel
        block_attend_kernel<T, HD, RT, true, false><<<grid, kAttendThreads, 0, s>>>(a);
        int most = 0;
        for (int b = 0; b < batch; ++b) most = a.positions[b] + a.n > most ? a.positions[b] + a.n : most;
        const int blocks = (most + kBlockRows - 1) / kBlockRows;
        if (blocks > 0)
            block_weights_kernel<<<dim3((blocks + 255) / 256, a.view.kv_heads, batch), 256, 0, s>>>(a);
    }
}
}  // namespace

hipError_t launch_block_append(const BlockRowsArgs& a, int batch, ElementType t, hipStream_t s) {
    return launch_rows(a, batch, t, false, s);
}
hipError_t launch_block_values(const BlockRowsArgs& a, int batch, ElementType t, hipStream_t s) {
    return launch_rows(a, batch, t, true, s);
}

hipError_t launch_block_attend(const BlockAttendArgs& a, int batch, int row_tiles, ElementType t, hipStream_t s) {
    with_type(t, [&](auto tag) {
        using T = decltype(tag);
        auto shaped = [&](auto hd, auto rt) {
            if (a.weights) attend<T, decltype(hd)::value, decltype(rt)::value, true>(a, batch, s);
            else attend<T, decltype(hd)::value, decltype(rt)::value, false>(a, batch, s);
        };
        auto tiled = [&](auto hd) {
            if (row_tiles == 1) shaped(hd, std::integral_constant<int, 1>{});
            else if (row_tiles == 2) shaped(hd, std::integral_constant<int, 2>{});
            else shaped(hd, std::integral_constant<int, 4>{});
        };
        if (a.view.head_dim == 64) tiled(std::integral_constant<int, 64>{});
        else tiled(std::integral_constant<int, 128>{});
    });
    return hipGetLastError();
}

hipError_t launch_block_evict(const BlockEvictArgs& a, int layers, int batch, hipStream_t s) {
    int most = 0;
    for (int b = 0; b < batch; ++b) most = a.positions[b] > most ? a.positions[b] : most;
    const int per = ((most + kBlockRows - 1) / kBlockRows + kEvictThreads - 1) / kEvictThreads;
    const dim3 grid(a.view.kv_heads, batch, layers);
    if (per <= 1) block_evict_kernel<1><<<grid, kEvictThreads, 0, s>>>(a);
    else if (per <= 2) block_evict_kernel<2><<<grid, kEvictThreads, 0, s>>>(a);
    else if (per <= 4) block_evict_kernel<4><<<grid, kEvictThreads, 0, s>>>(a);
    else if (per <= 8) block_evict_kernel<8><<<grid, kEvictThreads, 0, s>>>(a);
    else if (per <= 16) block_evict_kernel<16><<<grid, kEvictThreads, 0, s>>>(a);
    else block_evict_kernel<32><<<grid, kEvictThreads, 0, s>>>(a);
    return hipGetLastError();
}

}  // namespace swiftkv
