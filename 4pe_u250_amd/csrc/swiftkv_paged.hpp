// swiftkv_paged.hpp -- layout and kernel arguments of the paged cache, shared by
// swiftkv_paged_capi.cpp and the kernels (swiftkv_paged.hip,
// swiftkv_paged_attend.hip, swiftkv_paged_many.hip).
#pragma once

#include "swiftkv_block.hpp"
#include "swiftkv_paged_rows.hpp"

namespace swiftkv {

constexpr int kPageTokens = 64;
constexpr int kStepTokens = 32;          // half a page: the unit of a scan and of the layout
constexpr int kPageSteps = kPageTokens / kStepTokens;
constexpr int kTreeTokens = 64;
constexpr int kPagedMaxSeq = 131072;

// Sequences per launch, and bytes of trees (or accepted tokens) that one launch
// carries by value beside their positions.
constexpr int kPagedBatch = 64;
constexpr int kTreeBytes = 2048;
constexpr uint8_t kTreeRoot = 255;       // a tree byte: the parent, or these
constexpr uint8_t kTreeNone = 254;

// Record of one (layer, page, key/value head): two steps of 32 tokens, each
//   K [head_dim / 32][2][4][16] cells | V [head_dim / 16][4][16] cells
// of 16 bytes.  A K cell is 8 channels of a token, a V cell 8 tokens of a channel:
// what one lane of a 16-bit matrix instruction holds of its A operand.  Cells lie
// in the order of the lanes of the 16x16x32 form, so that a wave loads 1 KiB of
// consecutive bytes, nothing is transposed on the way, and the scores' lanes
// already hold the weights as the second product's B operand (the 32x32x16 form
// takes the same cells, each half wave 512 consecutive bytes):
//   K  channels 32 i + 8 g .., token t = 8 (m >> 2) + 4 h + (m & 3): cell [i][h][g][m]
//   V  channel 16 i + m, tokens 8 g ..: cell [i][g][m]
// The append moves more for it: a token's V row lies in head_dim cells.
struct PagedView {
    uint8_t* base;        // [layer][page][kv head] records
    int32_t* table;       // [slot][entries]: the page of each 64 tokens, or -1
    int64_t pages;
    int32_t entries;      // per slot
    int32_t layers;
    int32_t kv_heads;
    int32_t head_dim;
};
__host__ __device__ inline int64_t paged_step_bytes(int head_dim) { return 2 * kStepTokens * 2 * static_cast<int64_t>(head_dim); }
__host__ __device__ inline int64_t paged_record_bytes(int head_dim) { return kPageSteps * paged_step_bytes(head_dim); }
__host__ __device__ inline int64_t paged_record(const PagedView& v, int layer, int64_t page, int kv_head) {
    return ((static_cast<int64_t>(layer) * v.pages + page) * v.kv_heads + kv_head) * paged_record_bytes(v.head_dim);
}

// Exponents by which a weight may lie above those of a row's reference score.
constexpr float kScoreSlack = 4.0f;

// The rotation of a call's queries and keys; table null: none.
struct PagedRotation {
    const float2* table;  // [positions][rotary_dim / 2] (cos, sin)
    int32_t rotary_dim;
    int32_t halves;
};

// A byte for each of a launch's tokens, [sequence][padded(n)].  They are read as words at
// uniform addresses, 64 bytes a sequence whatever its number (hence the bytes behind the
// last): the argument block lies far from the GPU, and only scalar loads of it are quick.
struct TreeBytes {
    uint32_t words[kTreeBytes / 4 + kTreeTokens / 4];
};
constexpr int tree_pitch(int n) { return (n + 3) & ~3; }

// Parents of a launch's tokens.
struct PagedTree {
    TreeBytes parents;
};
struct PagedChain {};

// A grid row's sequence, counted from slot0 and its tensors' first, and its cached tokens.
struct PagedRow {
    int32_t position;
    int32_t sequence;
};

// Rows appended to one layer, or values read from several.
struct PagedRowsArgs {
    PagedView view;
    PagedRotation rotation;
    const void* k;
    const void* v;
    int64_t k_stride;     // elements between rows
    int64_t v_stride;
    void* k_out;          // values: dense rows [layer][batch * n]
    void* v_out;
    int64_t layer_rows;   // rows between two layers' values
    int32_t layer;        // the first
    int32_t slot0;
    int32_t n;
    int32_t positions[kPagedBatch];   // negative: the sequence is skipped
};

struct PagedAttendArgs {
    PagedView view;
    PagedRotation rotation;
    const void* q;
    void* out;
    const void* k;        // new rows, appended by the same launch (n <= kTreeTokens); null: none
    const void* v;
    int64_t q_stride;
    int64_t out_stride;
    int64_t k_stride;
    int64_t v_stride;
    float scale;          // log2(e) times the caller's magnitude
    float slack;          // kScoreSlack over it
    int32_t negative;     // the caller's scale is: queries change their sign
    int32_t group;        // query heads per key/value head
    uint32_t group_magic; // ceil(2^32 / group), 0 for 1
    int32_t n;
    int32_t layer;
    int32_t slot0;
    int32_t chunks;       // row chunks per (sequence, key/value head)
    int32_t splits;       // of the longest sequence
    int32_t split_steps;  // steps per split at most, a multiple of kSplitQuantumSteps
    float* partials;      // [pair][split]: stats [rows of a chunk][2], then sums [rows][head_dim]
    uint32_t* counters;   // [pair] arrived splits, kCounterStride apart, zero between launches
    PagedRow order[kPagedBatch];      // of each grid row, longest first
    // Not 0: the grid is one row of so many splits, first_split[y] the sum of those before
    // order[y]'s (two a word; all ones behind the last).
    int32_t all_splits;
    int32_t batch;
    uint32_t first_split[kPagedBatch / 2];
};

struct PagedKeepArgs {
    PagedView view;
    int32_t layer0;
    int32_t slot0;
    int32_t m;
    int32_t positions[kPagedBatch];
    TreeBytes accepted;               // 255 past the path's end
};

constexpr int kMapEntries = 512;
struct PagedMapArgs {
    int32_t* entries;
    int32_t n;
    int32_t pages[kMapEntries];
};

// A split is a multiple of so many steps.
constexpr int kSplitQuantumSteps = 4;

hipError_t launch_paged_map(const PagedMapArgs& a, hipStream_t s);
// tree null: chains
hipError_t launch_paged_append(const PagedRowsArgs& a, const PagedTree* tree, int batch, ElementType t, hipStream_t s);
hipError_t launch_paged_values(const PagedRowsArgs& a, int layers, int batch, hipStream_t s);
hipError_t launch_paged_keep(const PagedKeepArgs& a, int layers, int batch, hipStream_t s);
hipError_t launch_paged_copy(const PagedView& v, int64_t from, int64_t to, hipStream_t s);
// rows: of a chunk, 16 (a.chunks == 1), 32, 48 or 64
hipError_t launch_paged_attend(const PagedAttendArgs& a, const PagedTree* tree, int batch, int rows, ElementType t, hipStream_t s);
// rows: 128 or 256
hipError_t launch_paged_many(const PagedAttendArgs& a, const PagedTree* tree, int batch, int rows, ElementType t, hipStream_t s);
// The splits of such calls, of more than 16 rows
hipError_t launch_paged_join(const PagedAttendArgs& a, const PagedTree* tree, int batch, int rows, ElementType t, hipStream_t s);

}  // namespace swiftkv
