// swiftkv_block_capi.cpp -- host side of the rotary positions and the block
// cache (include/swiftkv.h): objects, argument checks, launch plans.  Kernels:
// swiftkv_block.hip, swiftkv_rotary.hip.  As in swiftkv_capi.cpp no exception
// crosses the C boundary, and a refused call enqueues nothing.
#include "swiftkv_block_host.hpp"

#include <algorithm>
#include <cstring>
#include <new>

using namespace swiftkv;

struct swiftkv_block_cache {
    swiftkv_context* ctx = nullptr;
    int32_t max_batch = 0;
    int32_t heads = 0;
    int32_t capacity = 0;      // tokens
    BlockView view{};
    size_t bytes = 0;
    // Log-sums of the rows and blocks of one launch with weights, for the most
    // queries that such a call takes (a graph may record it at any time):
    // allocated with the first of them.
    float* log_sums = nullptr;
};

namespace {

static_assert(SWIFTKV_BLOCK_TOKENS == kBlockRows && SWIFTKV_BLOCK_MAX_SEQ == kBlockMaxSeq, "block geometry");
static_assert(SWIFTKV_BLOCK_WEIGHT_QUERIES == kBlockWeightQueries, "queries with weights");
static_assert(SWIFTKV_F32 == kF32 && SWIFTKV_BF16 == kBF16 && SWIFTKV_F16 == kF16, "element types");

constexpr float kLog2E = 1.4426950408889634f;
// Workgroups of up to 1024 threads that a launch's x extent holds.
constexpr int64_t kMaxPromptGroups = int64_t(1) << 22;
// Workgroups of an attention launch that splits its sequences, at most, and
// what their partials take (17 MB).
constexpr int64_t kMaxSplitGroups = 2048;
constexpr size_t kPartialFloats = static_cast<size_t>(kMaxSplitGroups) * kMaxRowTiles * kRowTile * (2 + 128);

int check_type(int32_t dtype) {
    return dtype < kF32 || dtype > kF16 ? fail(SWIFTKV_EINVAL, "unknown element type %d", dtype) : SWIFTKV_OK;
}

// What every call on a range of sequences of a block cache checks; n tokens at
// positions[b] (negative: skipped, if `skips`) have to fit.
int check_rows(const swiftkv_context* ctx, const swiftkv_block_cache* c, int32_t layer, int32_t layers, int32_t seq0,
               const int32_t* positions, int32_t batch, int32_t n) {
    if (int rc = check_idle_io(ctx)) return rc;
    if (!c || c->ctx != ctx) return fail(SWIFTKV_EINVAL, "cache is null or belongs to another context");
    if (!positions) return fail(SWIFTKV_EINVAL, "null positions");
    if (layers < 1 || layer < 0 || static_cast<int64_t>(layer) + layers > c->view.layers)
        return fail(SWIFTKV_ERANGE, "layers [%d, %lld) outside [0, %d)", layer, static_cast<long long>(layer) + layers,
                    c->view.layers);
    if (batch < 1 || seq0 < 0 || static_cast<int64_t>(seq0) + batch > c->max_batch)
        return fail(SWIFTKV_ERANGE, "sequences [%d, %lld) outside [0, %d)", seq0,
                    static_cast<long long>(seq0) + batch, c->max_batch);
    if (n < 0 || n > c->capacity) return fail(SWIFTKV_ERANGE, "n = %d outside [0, %d]", n, c->capacity);
    for (int32_t b = 0; b < batch; ++b)
        if (static_cast<int64_t>(positions[b]) + n > c->capacity)
            return fail(SWIFTKV_ERANGE, "positions[%d] = %d: %d more tokens exceed the capacity %d", b, positions[b], n,
                        c->capacity);
    return SWIFTKV_OK;
}

template <typename Args>
void set_positions(Args& a, const int32_t* positions, int32_t nb) {
    std::memcpy(a.positions, positions, sizeof(int32_t) * static_cast<size_t>(nb));
}

int append_rows(const swiftkv_context* ctx, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                int32_t dtype, const swiftkv_block_cache* c, int32_t layer, int32_t seq0, const int32_t* positions,
                int32_t batch, int32_t n) {
    const size_t size = element_bytes(dtype);
    BlockRowsArgs a{};
    a.view = c->view;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.layer = layer;
    a.n = n;
    for (int32_t b0 = 0; b0 < batch; b0 += kBlockBatch) {
        const int32_t nb = std::min<int32_t>(kBlockBatch, batch - b0);
        const int64_t row = static_cast<int64_t>(b0) * n;
        a.k = static_cast<const char*>(k) + row * k_stride * static_cast<int64_t>(size);
        a.v = static_cast<const char*>(v) + row * v_stride * static_cast<int64_t>(size);
        a.slot0 = seq0 + b0;
        set_positions(a, positions + b0, nb);
        SKV_HIP(launch_block_append(a, nb, static_cast<ElementType>(dtype), ctx->stream));
    }
    return SWIFTKV_OK;
}

// Tokens per split, in tiles.  Splits make a workgroup for each CU where the
// (sequence, key/value head, row chunk) triples alone do not, and no more than the
// square root of a sequence's tiles, or 16, since the last of them joins all: us
// of a step with this rule's tokens against others, 8 key/value heads: batch 1 at
// 4096 512 (8 splits) 11.1; 256 11.7, 1024 12.4; at 16000 1024 (16) 15.6; 512 17.6,
// 2048 18.3; at 32000 2048 (16) 21.0; 1024 22.0, 4096 27.8; batch 4 at 4096 512 (8)
// 12.7; 256 15.6, 1024 14.0; batch 8 1024 (4) 16.8; 512 18.0, 2048 20.1; batch 16
// 2048 (2) 27.0; 1024 27.5; batch 4 at 32000 4096 (8) 44.9; 2048 48.6, 8192 52.1.
// Sequences of different lengths take a quarter more workgroups: 16 of 2000 to
// 32511 tokens 105.8 with 8192 tokens, 116.9 with the 9700 of one for each CU.
//
// Rows (query tokens times grouped heads) choose the kernel: the digits' row tiles
// of 4, 8 or 16, the fewest that hold the rows, and half floats, 64 rows a
// workgroup, for more than 16 without weights.  us of a step onto 4095 tokens, 64 / 8 /
// 1 sequences, 8 key/value heads (4 where groups are 5), the kernel taken against the
// next: 4 rows 86.5 / 17.7 / 10.8 against 88.7 / 19.9 / 13.2; 5 rows 47.6 / 14.5 / 12.9
// against 67.0 / 20.8 / 19.3; 8 rows 93.7 / 20.4 / 15.7 against 137 / 31.2 / 23.9; 16 rows
// 140 / 31.9 / 23.5 against 129 / 37.5 / 25.8 (FP32 139 / 31.8 / 23.4 against 163 / 43.4 /
// 28.5); more rows, half floats against 16 at a time: 20 rows 72.9 / 31.3 / 26.9 against
// 99.3 / 34.7 / 26.9, 32 rows 128 / 40.5 / 30.9 against 181 / 48.1 / 27.3 (FP32 168 / 47.1 /
// 34.4 against 184 / 46.2 / 26.2).
//
// One row chunk may append the call's rows in the attention's own launch, which
// costs each sequence's last workgroup five trips to memory, or leave them to a
// launch before it.  us of a step, own launch against one before: batch 1 / 8 /
// 32 at 4096 tokens and 8 key/value heads 11.9 / 18.3 / 49.4 against 15.0 / 21.8 /
// 51.8, batch 64 at 128 tokens 9.1 against 12.8; but batch 64 at 4096 tokens 89.4
// against 85.7, with 32 heads 343 against 316, and those at 1024 tokens 96.6
// against 92.1.  So: before it where no sequence is split and pairs times tokens
// reach kAppendBefore.
constexpr int64_t kAppendBefore = int64_t(1) << 21;
struct AttendPlan {
    int32_t row_tiles;   // 0: the prompt kernel
    int32_t chunks, splits, split_tiles;
    bool appends;
};
AttendPlan attend_plan(const swiftkv_context* ctx, const BlockView& view, int32_t group, int32_t n,
                       const int32_t* positions, int32_t batch, bool weights) {
    AttendPlan p{};
    const int64_t rows = static_cast<int64_t>(group) * n;
    const bool prompt = rows > kMaxRowTiles * kRowTile && !weights;
    p.row_tiles = prompt ? 0 : rows <= kRowTile ? 1 : rows <= 2 * kRowTile ? 2 : kMaxRowTiles;
    const int32_t chunk = prompt ? kPromptRows : p.row_tiles * kRowTile;
    p.chunks = static_cast<int32_t>((rows + chunk - 1) / chunk);
    const int64_t pairs = static_cast<int64_t>(batch) * view.kv_heads * p.chunks;
    int32_t longest = 0;
    int64_t total = 0;
    for (int32_t b = 0; b < batch; ++b) {
        const int32_t len = positions[b] < 0 ? 0 : positions[b] + n;
        longest = std::max(longest, len);
        total += (len + kTileTokens - 1) / kTileTokens;
    }
    const int64_t tiles = std::max(1, (longest + kTileTokens - 1) / kTileTokens);
    total *= view.kv_heads * p.chunks;
    const int64_t most_splits = std::min<int64_t>(16, std::ceil(std::sqrt(static_cast<double>(tiles))));
    const int64_t groups = total * 5 < pairs * tiles * 4 ? ctx->cus * 5 / 4 : ctx->cus;
    int64_t per = std::max<int64_t>((total + groups - 1) / groups, (tiles + most_splits - 1) / most_splits);
    if (ctx->split_tokens > 0) per = ctx->split_tokens / kTileTokens;
    // what the workspace holds
    const int64_t most = kMaxSplitGroups * kMaxRowTiles * kRowTile / std::max(chunk, kMaxRowTiles * kRowTile) / pairs;
    if (most <= 1) per = tiles;
    else per = std::max(per, (tiles + most - 1) / most);
    per = (per + 3) / 4 * 4;
    p.split_tiles = static_cast<int32_t>(per);
    p.splits = static_cast<int32_t>((tiles + per - 1) / per);
    p.appends = !prompt && p.chunks == 1 && (p.splits > 1 || pairs * longest < kAppendBefore);
    return p;
}

}  // namespace

extern "C" {

// ---------------------------------------------------------------- rotary

int swiftkv_rotary_create(swiftkv_context* ctx, int32_t rotary_dim, int32_t positions, double theta,
                          const swiftkv_rope_scaling* scaling, swiftkv_rotary_table** out) {
    if (!ctx || !out) return fail(SWIFTKV_EINVAL, "null argument");
    *out = nullptr;
    if (int rc = not_capturing(ctx, "swiftkv_rotary_create")) return rc;
    if (rotary_dim < 2 || rotary_dim > 256 || rotary_dim % 2 != 0)
        return fail(SWIFTKV_EINVAL, "rotary_dim %d: must be even and within [2, 256]", rotary_dim);
    if (positions < 1 || positions > SWIFTKV_ROTARY_MAX_POSITIONS)
        return fail(SWIFTKV_ERANGE, "positions %d outside [1, %d]", positions, SWIFTKV_ROTARY_MAX_POSITIONS);
    double freq[128], magnitude = 1.0;
    int rc = rope_frequencies(rotary_dim, theta, scaling, freq, &magnitude);
    if (rc) return rc;
    if ((rc = set_device(ctx))) return rc;
    const int32_t half = rotary_dim / 2;
    const size_t entries = static_cast<size_t>(positions) * half;
    float2* host = new (std::nothrow) float2[entries];
    swiftkv_rotary_table* t = new (std::nothrow) swiftkv_rotary_table();
    void* p = nullptr;
    if (!host || !t || hipMalloc(&p, entries * sizeof(float2)) != hipSuccess) {
        delete[] host;
        delete t;
        return fail(SWIFTKV_ENOMEM, "no memory for a rotary table of %zu bytes", entries * sizeof(float2));
    }
    for (int32_t i = 0; i < positions; ++i)
        for (int32_t j = 0; j < half; ++j) {
            const double angle = static_cast<double>(i) * freq[j];
            host[static_cast<size_t>(i) * half + j] = make_float2(static_cast<float>(magnitude * std::cos(angle)),
                                                                  static_cast<float>(magnitude * std::sin(angle)));
        }
    const hipError_t e = hipMemcpy(p, host, entries * sizeof(float2), hipMemcpyHostToDevice);
    delete[] host;
    if (e != hipSuccess) {
        (void)hipFree(p);
        delete t;
        return fail(SWIFTKV_EHIP, "rotary table upload: %s", hipGetErrorString(e));
    }
    t->ctx = ctx;
    t->rotary_dim = rotary_dim;
    t->positions = positions;
    t->table = static_cast<float2*>(p);
    ++ctx->children;
    *out = t;
    return ok();
}

int swiftkv_rotary_destroy(swiftkv_rotary_table* table) {
    if (!table) return ok();
    swiftkv_context* ctx = table->ctx;
    if (int rc = not_capturing(ctx, "swiftkv_rotary_destroy")) return rc;
    (void)hipSetDevice(ctx->device);
    (void)hipStreamSynchronize(ctx->stream);
    (void)hipFree(table->table);
    delete table;
    release_child(ctx);
    return ok();
}

int swiftkv_rotary(swiftkv_context* ctx, const swiftkv_rotary_table* table, const void* x, int64_t x_stride,
                   void* out, int64_t out_stride, int32_t dtype, int32_t halves, int32_t inverse,
                   const int32_t* positions, int32_t batch, int32_t n, int32_t heads, int32_t head_dim) {
    int rc = check_idle_io(ctx);
    if (rc) return rc;
    if (!table || table->ctx != ctx) return fail(SWIFTKV_EINVAL, "table is null or belongs to another context");
    if (!x || !out || !positions) return fail(SWIFTKV_EINVAL, "null x, out or positions");
    if ((rc = check_type(dtype))) return rc;
    if (batch < 1 || n < 0 || heads < 1 || heads > 65536)
        return fail(SWIFTKV_EINVAL, "batch %d, n %d, heads %d: batch >= 1, n >= 0 and 1 <= heads <= 65536", batch, n, heads);
    if (head_dim < table->rotary_dim || head_dim > 1024)
        return fail(SWIFTKV_EINVAL, "head_dim %d outside [%d, 1024]", head_dim, table->rotary_dim);
    const int64_t row = static_cast<int64_t>(heads) * head_dim;
    for (const int64_t stride : {x_stride, out_stride})
        if (stride < row || stride > (int64_t(1) << 40))
            return fail(SWIFTKV_EINVAL, "stride %lld outside [heads * head_dim = %lld, 2^40]",
                        static_cast<long long>(stride), static_cast<long long>(row));
    const size_t size = element_bytes(dtype);
    if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(out)) % size != 0)
        return fail(SWIFTKV_EINVAL, "x and out must be aligned to their elements");
    if (x == out && x_stride != out_stride) return fail(SWIFTKV_EINVAL, "in place x and out have one stride");
    for (int32_t b = 0; b < batch; ++b)
        if (positions[b] < 0 || static_cast<int64_t>(positions[b]) + n > table->positions)
            return fail(SWIFTKV_ERANGE, "positions[%d] = %d: tokens [%d, %lld) outside the table (%d)", b, positions[b],
                        positions[b], static_cast<long long>(positions[b]) + n, table->positions);
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;
    RotaryArgs a{};
    a.table = table->table;
    a.x_stride = x_stride;
    a.out_stride = out_stride;
    a.heads = heads;
    a.head_dim = head_dim;
    a.rotary_dim = table->rotary_dim;
    a.n = n;
    for (int32_t b0 = 0; b0 < batch; b0 += kBlockBatch) {
        const int32_t nb = std::min<int32_t>(kBlockBatch, batch - b0);
        const int64_t first = static_cast<int64_t>(b0) * n;
        a.x = static_cast<const char*>(x) + first * x_stride * static_cast<int64_t>(size);
        a.out = static_cast<char*>(out) + first * out_stride * static_cast<int64_t>(size);
        set_positions(a, positions + b0, nb);
        SKV_HIP(launch_rotary(a, nb, static_cast<ElementType>(dtype), halves != 0, inverse != 0, ctx->stream));
    }
    return ok();
}

// ---------------------------------------------------------------- block cache

int swiftkv_block_cache_create(swiftkv_context* ctx, int32_t layers, int32_t max_batch, int32_t heads,
                               int32_t kv_heads, int32_t head_dim, int32_t max_seq_len,
                               swiftkv_block_cache** out) {
    if (!ctx || !out) return fail(SWIFTKV_EINVAL, "null argument");
    *out = nullptr;
    if (int rc = not_capturing(ctx, "swiftkv_block_cache_create")) return rc;
    if (layers < 1 || layers > 256) return fail(SWIFTKV_EINVAL, "layers %d outside [1, 256]", layers);
    if (max_batch < 1 || max_batch > 4096) return fail(SWIFTKV_EINVAL, "max_batch %d outside [1, 4096]", max_batch);
    if (kv_heads < 1 || kv_heads > 256 || heads < kv_heads || heads % kv_heads != 0 || heads / kv_heads > 64)
        return fail(SWIFTKV_EINVAL, "heads %d, kv_heads %d: kv_heads within [1, 256], heads a multiple of it, at most 64 "
                    "times", heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) return fail(SWIFTKV_EINVAL, "head_dim %d: must be 64 or 128", head_dim);
    if (max_seq_len < 1 || max_seq_len > kBlockMaxSeq)
        return fail(SWIFTKV_EINVAL, "max_seq_len %d outside [1, %d]", max_seq_len, kBlockMaxSeq);
    int rc = set_device(ctx);
    if (rc) return rc;
    if (!ctx->block_workspace) {
        void* p = nullptr;
        const size_t counters = kMaxSplitGroups * kCounterStride * sizeof(uint32_t);
        const size_t bytes = counters + kPartialFloats * sizeof(float);
        if (hipMalloc(&p, bytes) != hipSuccess) return fail(SWIFTKV_ENOMEM, "hipMalloc of %zu bytes failed", bytes);
        const hipError_t e = hipMemsetAsync(p, 0, counters, ctx->stream);
        if (e != hipSuccess) {
            (void)hipFree(p);
            return fail(SWIFTKV_EHIP, "split counters: %s", hipGetErrorString(e));
        }
        ctx->block_workspace = static_cast<uint32_t*>(p);
    }
    swiftkv_block_cache* c = new (std::nothrow) swiftkv_block_cache();
    if (!c) return fail(SWIFTKV_ENOMEM, "out of host memory");
    c->ctx = ctx;
    c->max_batch = max_batch;
    c->heads = heads;
    c->capacity = (max_seq_len + kTileTokens - 1) / kTileTokens * kTileTokens;
    c->view.blocks = c->capacity / kBlockRows;
    c->view.layers = layers;
    c->view.kv_heads = kv_heads;
    c->view.head_dim = head_dim;
    c->view.page_bytes =
        (static_cast<int64_t>(c->view.blocks) * (2 * kBlockRows * head_dim + 8) + 255) / 256 * 256;
    const int64_t pages = static_cast<int64_t>(max_batch) * layers * kv_heads;
    const size_t page_total = static_cast<size_t>(pages) * static_cast<size_t>(c->view.page_bytes);
    const size_t table_total = static_cast<size_t>(pages) * static_cast<size_t>(c->view.blocks) * sizeof(uint16_t);
    c->bytes = page_total + table_total;
    void* p = nullptr;
    if (hipMalloc(&p, c->bytes) != hipSuccess) {
        const size_t bytes = c->bytes;
        delete c;
        return fail(SWIFTKV_ENOMEM, "hipMalloc of a block cache (%zu bytes) failed", bytes);
    }
    c->view.base = static_cast<int8_t*>(p);
    c->view.table = reinterpret_cast<uint16_t*>(c->view.base + page_total);
    hipError_t e = hipMemsetAsync(p, 0, page_total, ctx->stream);
    if (e == hipSuccess) e = launch_block_table(c->view, pages, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
        (void)hipFree(p);
        delete c;
        return fail(SWIFTKV_EHIP, "block cache: %s", hipGetErrorString(e));
    }
    ++ctx->children;
    *out = c;
    return ok();
}

int swiftkv_block_cache_destroy(swiftkv_block_cache* cache) {
    if (!cache) return ok();
    swiftkv_context* ctx = cache->ctx;
    if (int rc = not_capturing(ctx, "swiftkv_block_cache_destroy")) return rc;
    (void)hipSetDevice(ctx->device);
    (void)hipStreamSynchronize(ctx->stream);
    (void)hipFree(cache->view.base);
    if (cache->log_sums) (void)hipFree(cache->log_sums);
    delete cache;
    release_child(ctx);
    return ok();
}

size_t swiftkv_block_cache_bytes(const swiftkv_block_cache* cache) { return cache ? cache->bytes : 0; }
int32_t swiftkv_block_cache_blocks(const swiftkv_block_cache* cache) { return cache ? cache->view.blocks : 0; }

int swiftkv_block_append(swiftkv_context* ctx, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                         int32_t dtype, swiftkv_block_cache* cache, int32_t layer_index, int32_t seq0,
                         const int32_t* positions, int32_t batch, int32_t n) {
    int rc = check_rows(ctx, cache, layer_index, 1, seq0, positions, batch, n);
    if (rc) return rc;
    if ((rc = check_type(dtype))) return rc;
    const int64_t row = static_cast<int64_t>(cache->view.kv_heads) * cache->view.head_dim;
    if ((rc = check_tensor("k", k, k_stride, row, dtype))) return rc;
    if ((rc = check_tensor("v", v, v_stride, row, dtype))) return rc;
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;
    if ((rc = append_rows(ctx, k, k_stride, v, v_stride, dtype, cache, layer_index, seq0, positions, batch, n)))
        return rc;
    return ok();
}

int swiftkv_block_values(swiftkv_context* ctx, const swiftkv_block_cache* cache, int32_t layer_index, int32_t seq0,
                         const int32_t* positions, int32_t batch, int32_t n, int32_t dtype, void* k, void* v) {
    int rc = check_rows(ctx, cache, layer_index, 1, seq0, positions, batch, n);
    if (rc) return rc;
    if ((rc = check_type(dtype))) return rc;
    const int64_t row = static_cast<int64_t>(cache->view.kv_heads) * cache->view.head_dim;
    if ((rc = check_tensor("k", k, row, row, dtype))) return rc;
    if ((rc = check_tensor("v", v, row, row, dtype))) return rc;
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;
    BlockRowsArgs a{};
    a.view = cache->view;
    a.layer = layer_index;
    a.n = n;
    for (int32_t b0 = 0; b0 < batch; b0 += kBlockBatch) {
        const int32_t nb = std::min<int32_t>(kBlockBatch, batch - b0);
        const int64_t first = static_cast<int64_t>(b0) * n * row * static_cast<int64_t>(element_bytes(dtype));
        a.k_out = static_cast<char*>(k) + first;
        a.v_out = static_cast<char*>(v) + first;
        a.slot0 = seq0 + b0;
        set_positions(a, positions + b0, nb);
        SKV_HIP(launch_block_values(a, nb, static_cast<ElementType>(dtype), ctx->stream));
    }
    return ok();
}

int swiftkv_block_attention(swiftkv_context* ctx, const void* q, int64_t q_stride, const void* k, int64_t k_stride,
                            const void* v, int64_t v_stride, int32_t dtype, swiftkv_block_cache* cache,
                            int32_t layer_index, int32_t seq0, const int32_t* positions, int32_t batch, int32_t n,
                            float scale, float* weights, void* out, int64_t out_stride) {
    int rc = check_rows(ctx, cache, layer_index, 1, seq0, positions, batch, n);
    if (rc) return rc;
    if ((rc = check_type(dtype))) return rc;
    const BlockView& view = cache->view;
    const int64_t kv_row = static_cast<int64_t>(view.kv_heads) * view.head_dim;
    const int64_t q_row = static_cast<int64_t>(cache->heads) * view.head_dim;
    if ((rc = check_tensor("q", q, q_stride, q_row, dtype))) return rc;
    if ((rc = check_tensor("out", out, out_stride, q_row, dtype))) return rc;
    if ((k == nullptr) != (v == nullptr)) return fail(SWIFTKV_EINVAL, "k and v must both be set or both be null");
    if (k && (rc = check_tensor("k", k, k_stride, kv_row, dtype))) return rc;
    if (v && (rc = check_tensor("v", v, v_stride, kv_row, dtype))) return rc;
    if (!std::isfinite(scale)) return fail(SWIFTKV_EINVAL, "scale must be finite");
    if (weights && n > kBlockWeightQueries)
        return fail(SWIFTKV_ERANGE, "weights are gathered from at most %d queries a call, not %d", kBlockWeightQueries, n);
    if (reinterpret_cast<uintptr_t>(weights) & 3u) return fail(SWIFTKV_EINVAL, "weights must be aligned to 4 bytes");
    const int32_t group = cache->heads / view.kv_heads;
    if (!weights && (static_cast<int64_t>(group) * n + kPromptRows - 1) / kPromptRows * view.kv_heads >= kMaxPromptGroups)
        return fail(SWIFTKV_ERANGE, "n = %d: %d heads take %lld workgroups and more", n, cache->heads,
                    static_cast<long long>(kMaxPromptGroups));
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;

    BlockAttendArgs a{};
    a.view = view;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.scale = (scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(view.head_dim)) : scale) * kLog2E;
    a.group = group;
    a.group_magic = a.group == 1 ? 0u : static_cast<uint32_t>(((uint64_t(1) << 32) + a.group - 1) / a.group);
    a.n = n;
    a.layer = layer_index;
    a.counters = ctx->block_workspace;
    a.partials = reinterpret_cast<float*>(ctx->block_workspace + kMaxSplitGroups * kCounterStride);
    if (weights) {
        const size_t rows =
            static_cast<size_t>(std::min(cache->max_batch, kBlockBatch)) * cache->heads * kBlockWeightQueries;
        if (!cache->log_sums) {
            if ((rc = not_capturing(ctx, "the first attention with weights"))) return rc;
            const size_t bytes = rows * (static_cast<size_t>(view.blocks) + 1) * sizeof(float);
            void* p = nullptr;
            if (hipMalloc(&p, bytes) != hipSuccess) return fail(SWIFTKV_ENOMEM, "hipMalloc of %zu bytes failed", bytes);
            cache->log_sums = static_cast<float*>(p);
            cache->bytes += bytes;
        }
        a.row_lse = cache->log_sums;
        a.block_lse = cache->log_sums + rows;
    }
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    const int64_t size = static_cast<int64_t>(element_bytes(dtype));
    for (int32_t b0 = 0; b0 < batch; b0 += kBlockBatch) {
        const int32_t nb = std::min<int32_t>(kBlockBatch, batch - b0);
        const AttendPlan plan = attend_plan(ctx, view, a.group, n, positions + b0, nb, weights != nullptr);
        const int64_t first = static_cast<int64_t>(b0) * n;
        a.q = static_cast<const char*>(q) + first * q_stride * size;
        a.out = static_cast<char*>(out) + first * out_stride * size;
        a.k = a.v = nullptr;
        if (k) {
            const char* kb = static_cast<const char*>(k) + first * k_stride * size;
            const char* vb = static_cast<const char*>(v) + first * v_stride * size;
            if (plan.appends) {
                a.k = kb;
                a.v = vb;
            } else if ((rc = append_rows(ctx, kb, k_stride, vb, v_stride, dtype, cache, layer_index, seq0 + b0,
                                         positions + b0, nb, n))) {
                return rc;
            }
        }
        a.weights = weights ? weights + static_cast<int64_t>(b0) * view.kv_heads * view.blocks : nullptr;
        a.slot0 = seq0 + b0;
        a.chunks = plan.chunks;
        a.splits = plan.splits;
        a.split_tiles = plan.split_tiles;
        set_positions(a, positions + b0, nb);
        for (int32_t b = 0; b < nb; ++b) a.order[b] = static_cast<uint8_t>(b);
        if (nb > 1)
            std::sort(a.order, a.order + nb, [&](uint8_t x, uint8_t y) {
                return a.positions[x] != a.positions[y] ? a.positions[x] > a.positions[y] : x < y;
            });
        const ElementType type = static_cast<ElementType>(dtype);
        SKV_HIP(plan.row_tiles == 0 ? launch_block_prompt(a, nb, type, ctx->stream)
                                    : launch_block_attend(a, nb, plan.row_tiles, type, ctx->stream));
    }
    return ok();
}

int swiftkv_block_evict(swiftkv_context* ctx, swiftkv_block_cache* cache, int32_t layer0, int32_t layers,
                        int32_t seq0, const int32_t* positions, int32_t batch, int32_t keep, int32_t sinks,
                        int32_t recent, float* weights, int32_t* kept, int32_t* out_positions) {
    int rc = check_rows(ctx, cache, layer0, layers, seq0, positions, batch, 0);
    if (rc) return rc;
    if (!weights) return fail(SWIFTKV_EINVAL, "null weights");
    if ((reinterpret_cast<uintptr_t>(weights) | reinterpret_cast<uintptr_t>(kept)) & 3u)
        return fail(SWIFTKV_EINVAL, "weights and kept must be aligned to 4 bytes");
    if (sinks < 0 || recent < 1 || keep > cache->view.blocks || static_cast<int64_t>(sinks) + recent > keep)
        return fail(SWIFTKV_EINVAL, "keep %d, sinks %d, recent %d: 0 <= sinks, 1 <= recent, sinks + recent <= keep <= %d",
                    keep, sinks, recent, cache->view.blocks);
    if ((rc = set_device(ctx))) return rc;
    BlockEvictArgs a{};
    a.view = cache->view;
    a.weights = weights;
    a.kept = kept;
    a.layer0 = layer0;
    a.slot0 = seq0;
    a.batch = batch;
    a.keep = keep;
    a.sinks = sinks;
    a.recent = recent;
    for (int32_t b0 = 0; b0 < batch; b0 += kBlockBatch) {
        const int32_t nb = std::min<int32_t>(kBlockBatch, batch - b0);
        a.b0 = b0;
        set_positions(a, positions + b0, nb);
        SKV_HIP(launch_block_evict(a, layers, nb, ctx->stream));
    }
    if (out_positions)
        for (int32_t b = 0; b < batch; ++b) {
            const int32_t held = positions[b] < 0 ? 0 : (positions[b] + kBlockRows - 1) / kBlockRows;
            out_positions[b] = positions[b] - kBlockRows * std::max(0, held - keep);
        }
    return ok();
}

}  // extern "C"
