// swiftkv_block.hpp -- layout and kernel arguments of the block cache and the
// rotation, shared by swiftkv_block_capi.cpp and the kernels
// (swiftkv_block.hip, swiftkv_rotary.hip).
#pragma once

#include "swiftkv_common.hpp"

namespace swiftkv {

constexpr int kBlockRows = 16;       // tokens of a block
constexpr int kTileBlocks = 4;       // blocks of a tile, the unit of a scan: 64 tokens
constexpr int kTileTokens = kBlockRows * kTileBlocks;
constexpr int kBlockMaxSeq = 131072;
constexpr int kBlockWeightQueries = 8;

// Sequences per launch: positions travel by value in the kernel arguments, and
// 256 of them made every launch 0.9 us longer on the host (4.1 us against 3.2).
constexpr int kBlockBatch = 64;

// Element types of the tensors.
enum ElementType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };
inline size_t element_bytes(int t) { return t == kF32 ? 4 : 2; }

// Page of one (sequence, layer, key/value head): `blocks` records, each
//   K codes [head_dim / 16][16 tokens][16 channels] | V codes [head_dim][16 tokens]
// then the scales [blocks] {K, V} as FP32.  A record is the B operand of the
// 8-bit matrix instructions as it lies: 16 bytes are 16 channels of a token (K)
// or 16 tokens of a channel (V), the run that one lane holds, so a wave's 64
// lanes load 1 KiB of consecutive bytes and nothing is transposed on the way.
// The table [blocks] of a page holds the record of each block in the
// sequence's order.
struct BlockView {
    int8_t* base;         // pages ordered [slot][layer][kv head]
    uint16_t* table;      // [slot][layer][kv head][blocks]
    int64_t page_bytes;
    int32_t blocks;       // per page, a multiple of kTileBlocks
    int32_t layers;
    int32_t kv_heads;
    int32_t head_dim;
};
__host__ __device__ inline int64_t block_page(const BlockView& v, int slot, int layer, int kv_head) {
    return (static_cast<int64_t>(slot) * v.layers + layer) * v.kv_heads + kv_head;
}

// Rows of K and V appended to, or values read from, one layer.
struct BlockRowsArgs {
    BlockView view;
    const void* k;        // append: [batch * n] rows
    const void* v;
    int64_t k_stride;     // elements between rows
    int64_t v_stride;
    void* k_out;          // values: dense rows
    void* v_out;
    int32_t layer;
    int32_t slot0;
    int32_t n;
    int32_t positions[kBlockBatch];   // negative: the sequence is skipped
};

struct BlockAttendArgs {
    BlockView view;
    const void* q;
    void* out;
    const void* k;        // new rows, appended by the same launch (chunks == 1 only); null: none
    const void* v;
    int64_t q_stride;
    int64_t out_stride;
    int64_t k_stride;
    int64_t v_stride;
    float scale;          // log2(e) times the caller's
    int32_t group;        // query heads per key/value head
    uint32_t group_magic; // ceil(2^32 / group), 0 for 1: r / group is its product with r, shifted (r < 2^26)
    int32_t n;
    int32_t layer;
    int32_t slot0;
    int32_t chunks;       // row chunks per (sequence, key/value head)
    int32_t splits;       // of the longest sequence
    int32_t split_tiles;  // tiles per split at most, a multiple of 4
    float* partials;      // [pair][split][rows of a chunk][2 + head_dim]: m, l, acc, each kernel's own units
    uint32_t* counters;   // [pair] arrived splits, kCounterStride apart, zero between launches
    float* block_lse;     // null, or [sequence][kv head][row][blocks]: log2 of each block's sum of 2^score
    float* row_lse;       // [sequence][kv head][row]: the same of the whole row
    float* weights;       // [sequence][kv head][blocks]
    int32_t positions[kBlockBatch];
    uint8_t order[kBlockBatch];   // the sequence of each grid row, longest first
};

struct BlockEvictArgs {
    BlockView view;
    float* weights;       // [layers][batch][kv_heads][blocks]
    int32_t* kept;        // [layers][batch][kv_heads][keep] or null
    int32_t layer0;
    int32_t slot0;
    int32_t b0;           // first sequence of this launch, of `batch`
    int32_t batch;
    int32_t keep;
    int32_t sinks;
    int32_t recent;
    int32_t positions[kBlockBatch];
};

struct RotaryArgs {
    const void* x;
    void* out;
    const float2* table;  // [positions][rotary_dim / 2] (cos, sin)
    int64_t x_stride;
    int64_t out_stride;
    int32_t heads;
    int32_t head_dim;
    int32_t rotary_dim;
    int32_t n;
    int32_t positions[kBlockBatch];
};

// Rows (query tokens times grouped heads) that one attention workgroup holds.
constexpr int kRowTile = 4;          // rows of one matrix instruction, four limbs each
constexpr int kMaxRowTiles = 4;
// Rows of a workgroup of the prompt kernel, for calls with more rows than that.
constexpr int kPromptRows = 64;
// Words between the arrival counts of two pairs: a 128-byte line each.
constexpr int kCounterStride = 32;

hipError_t launch_block_table(const BlockView& v, int64_t pages, hipStream_t s);
hipError_t launch_block_append(const BlockRowsArgs& a, int batch, ElementType t, hipStream_t s);
hipError_t launch_block_values(const BlockRowsArgs& a, int batch, ElementType t, hipStream_t s);
// row_tiles: 1, 2 or 4
hipError_t launch_block_attend(const BlockAttendArgs& a, int batch, int row_tiles, ElementType t, hipStream_t s);
// a.chunks of kPromptRows rows; a.k, a.weights null
hipError_t launch_block_prompt(const BlockAttendArgs& a, int batch, ElementType t, hipStream_t s);
hipError_t launch_block_evict(const BlockEvictArgs& a, int layers, int batch, hipStream_t s);
hipError_t launch_rotary(const RotaryArgs& a, int batch, ElementType t, bool halves, bool inverse, hipStream_t s);

}  // namespace swiftkv
