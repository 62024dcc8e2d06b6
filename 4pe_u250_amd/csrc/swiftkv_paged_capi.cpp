// swiftkv_paged_capi.cpp -- host side of the paged cache (include/swiftkv.h):
// objects, argument checks, launch plans.  Kernels: swiftkv_paged.hip,
// swiftkv_paged_attend.hip, swiftkv_paged_many.hip.  As in swiftkv_capi.cpp no exception crosses the C
// boundary, and a refused call enqueues nothing.
#include "swiftkv_block_host.hpp"

#include <algorithm>
#include <cstring>
#include <iterator>
#include <new>

#include "swiftkv_paged.hpp"
#include "swiftkv_paged_host.hpp"

using namespace swiftkv;

struct swiftkv_paged_cache {
    swiftkv_context* ctx = nullptr;
    int32_t max_batch = 0;
    int32_t heads = 0;
    int32_t capacity = 0;      // tokens of a sequence
    ElementType type = kBF16;
    PagedView view{};
    size_t bytes = 0;
    PageTable* table = nullptr;
};

namespace {

static_assert(SWIFTKV_PAGE_TOKENS == kPageTokens && SWIFTKV_TREE_TOKENS == kTreeTokens, "page and tree size");
static_assert(SWIFTKV_PAGED_MAX_SEQ == kPagedMaxSeq, "sequence length");

constexpr float kLog2E = 1.4426950408889634f;
// Workgroups of 256 threads that a launch's x extent holds.
constexpr int64_t kMaxGroups = int64_t(1) << 23;
// Workgroups of an attention launch that splits its sequences, at most, and the
// rows of their partials.
constexpr int64_t kMaxSplitGroups = 2048;
constexpr int64_t kMaxPartialRows = int64_t(1) << 16;
constexpr size_t kPartialFloats = static_cast<size_t>(kMaxPartialRows) * (2 + 128);

constexpr int32_t kXcds = 8;

// Turns (plan_attention) from which they are many.
constexpr int64_t kManyTurns = 32768;

// What every call on a range of sequences of a paged cache checks.
int check_call(const swiftkv_context* ctx, const swiftkv_paged_cache* c, int32_t layer, int32_t layers, int32_t seq0,
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
    return SWIFTKV_OK;
}

// Tokens [0, positions + count) of a sequence have pages, and with `own` those
// from `first` on pages that nobody else names.
int check_pages(const swiftkv_paged_cache* c, int32_t seq, int32_t b, int32_t position, int32_t count, bool own) {
    const int64_t end = static_cast<int64_t>(position) + count;
    if (end > c->capacity)
        return fail(SWIFTKV_ERANGE, "positions[%d] = %d: %d more tokens exceed the capacity %d", b, position, count,
                    c->capacity);
    if (!c->table->holds(seq, end, kPageTokens))
        return fail(SWIFTKV_ESTATE, "sequence %d has no pages for all of tokens [0, %lld)", seq, static_cast<long long>(end));
    if (own) {
        const int32_t e = c->table->not_own(seq, position, static_cast<int32_t>(end), kPageTokens);
        if (e >= 0)
            return fail(SWIFTKV_ESTATE, "sequence %d would write tokens of page %d, which another entry names too", seq,
                        c->table->page(seq, e));
    }
    return SWIFTKV_OK;
}

// The tokens, trees and rotary positions of a call; `counts` of the sequence b.
int check_tokens(const swiftkv_paged_cache* c, const swiftkv_rotary_table* table, const int32_t* parents, int32_t seq0,
                 const int32_t* positions, int32_t batch, int32_t n, bool writes) {
    if (table && table->ctx != c->ctx) return fail(SWIFTKV_EINVAL, "table belongs to another context");
    if (table && table->rotary_dim > c->view.head_dim)
        return fail(SWIFTKV_EINVAL, "the table's %d rotary channels exceed head_dim %d", table->rotary_dim, c->view.head_dim);
    if (parents && n > kTreeTokens) return fail(SWIFTKV_ERANGE, "a tree of %d tokens: at most %d", n, kTreeTokens);
    for (int32_t b = 0; b < batch; ++b) {
        int32_t count = n, depth = n - 1;
        if (parents) {
            const int32_t* tree = parents + static_cast<int64_t>(b) * n;
            count = tree_tokens(tree, n);
            if (count < 0)
                return fail(SWIFTKV_EINVAL, "parents of sequence %d: token %d has parent %d", b, -1 - count, tree[-1 - count]);
            depth = tree_depth(tree, count);
        }
        if (positions[b] < 0) continue;
        if (int rc = check_pages(c, seq0 + b, b, positions[b], count, writes)) return rc;
        if (table && !turns_within(positions[b], depth, table->positions))
            return fail(SWIFTKV_ERANGE, "positions[%d] = %d: token positions up to %lld outside the table (%d)", b, positions[b],
                        static_cast<long long>(positions[b]) + depth, table->positions);
    }
    return SWIFTKV_OK;
}

PagedRotation rotation_of(const swiftkv_rotary_table* table, int32_t halves) {
    return table ? PagedRotation{table->table, table->rotary_dim, halves != 0} : PagedRotation{nullptr, 0, 0};
}

// Sequences of one launch of n tokens each.
int32_t launch_batch(bool tree, int32_t n) { return tree ? std::min<int32_t>(kPagedBatch, kTreeBytes / tree_pitch(n)) : kPagedBatch; }

// Rows b0 .. b0 + nb - 1 of [batch][n] numbers below 64 as bytes, -1 and -2 as these.
void set_bytes(TreeBytes& t, const int32_t* numbers, int32_t b0, int32_t nb, int32_t n, uint8_t minus_one, uint8_t minus_two) {
    uint8_t* dst = reinterpret_cast<uint8_t*>(t.words);
    const int32_t pitch = tree_pitch(n);
    for (int32_t b = 0; b < nb; ++b, dst += pitch) {
        const int32_t* src = numbers + static_cast<int64_t>(b0 + b) * n;
        for (int32_t i = 0; i < n; ++i) dst[i] = src[i] == -1 ? minus_one : src[i] == -2 ? minus_two : static_cast<uint8_t>(src[i]);
        for (int32_t i = n; i < pitch; ++i) dst[i] = minus_two;
    }
}

const PagedTree* tree_of(PagedTree& t, const int32_t* parents, int32_t b0, int32_t nb, int32_t n) {
    if (!parents) return nullptr;
    set_bytes(t.parents, parents, b0, nb, n, kTreeRoot, kTreeNone);
    return &t;
}

int append_rows(const swiftkv_context* ctx, const PagedRotation& rotation, const void* k, int64_t k_stride, const void* v,
                int64_t v_stride, const swiftkv_paged_cache* c, int32_t layer, int32_t seq0, const int32_t* positions,
                const int32_t* parents, int32_t batch, int32_t n) {
    PagedRowsArgs a{};
    a.view = c->view;
    a.rotation = rotation;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.layer = layer;
    a.n = n;
    const int32_t most = launch_batch(parents != nullptr, n);
    for (int32_t b0 = 0; b0 < batch; b0 += most) {
        const int32_t nb = std::min(most, batch - b0);
        const int64_t row = static_cast<int64_t>(b0) * n;
        a.k = static_cast<const char*>(k) + row * k_stride * 2;
        a.v = static_cast<const char*>(v) + row * v_stride * 2;
        a.slot0 = seq0 + b0;
        std::memcpy(a.positions, positions + b0, sizeof(int32_t) * static_cast<size_t>(nb));
        PagedTree tree;
        SKV_HIP(launch_paged_append(a, tree_of(tree, parents, b0, nb, n), nb, c->type, ctx->stream));
    }
    return SWIFTKV_OK;
}

// The kernel of a call goes by its rows (query tokens times grouped heads) and by turns,
// steps times chunks of 256 rows times key/value heads.  Up to 16 and 32 rows a workgroup
// holds them all.  Where turns are many, its cells shall be read by few workgroups: 48 rows
// (three tiles of 16 a wave: loads bound these), 64 (two of 32), 128 or 256 (cells shared in
// LDS).  Where they are few, workgroups shall be many: 32 rows, or 64 where 32 would leave a
// CU more than one.  us of a call onto 4031 tokens, 32 heads of 128 over 8, the kernel taken
// against others: 64 sequences x 12 tokens (48 rows) 48 190, 64 192, 32 207; x 16 64 195, 32 210,
// 128 216; x 24 128 225, 64 255, 32 261; x 64 256 351, 128 407, 64 467; 8 x 16 32 31.4, 64 35.2; x
// 24 32 35.0, 64 38.5, 128 43.3; x 64 64 56.6, 32 65.4, 256 66.5; one sequence x 26 32 16.1, 64
// 20.3; x 512 64 53.5, 32 58.8, 256 67.6; x 1024 64 102, 32 111, 256 114; 4 x 512 256 171, 64 185; a
// prompt of 4096 tokens onto none 256 178, 128 207.
//
// What the rule does not see: a chunk of a prompt scans what it sees and turns count as if
// each saw all, so prompts onto none get more rows than is best (512 tokens 64 19.4, 32 16.0;
// 1024 64 35.8, 32 31.0; 2048 64 81.7, 32 74.4), and 8 x 32 tokens are where the two meet (64
// 40.0, 32 36.8).
//
// Splits make a workgroup for each CU and not more, of at most 32 a sequence and at most the
// square root of its 64-token tiles, since they are joined: us of a step, tokens of this
// rule's splits against others: one sequence at 4096 512 10.9; 256 12.0, 1024 12.6; 4 at 4096
// 512 16.5; 1024 19.6; 8 at 4096 1024 26.3; 512 29.3, 2048 30.5; 32 at 4096 none 85.6; 2048
// 90.7; 64 none 169; 2048 180; one at 32000 1408 29.6; 1024 30.1, 2048 31.4, 4096 46.0.  It goes by
// how many workgroups there are, not by what each scans: one sequence of 32000 among 63 of 100
// is not split (280; in 4 splits 84).
PagedPlan plan_attention(int32_t cus, int32_t split_tokens, int32_t forced_rows, int32_t group, int32_t kv_heads, int32_t n,
                         const int32_t* positions, int32_t batch) {
    PagedPlan p{};
    const int64_t rows = static_cast<int64_t>(group) * n;
    auto steps_of = [&](int32_t b) {
        return positions[b] < 0 ? 0 : (static_cast<int64_t>(positions[b]) + n + kStepTokens - 1) / kStepTokens;
    };
    int64_t turns = 0, longest = 1, live = 0;
    for (int32_t b = 0; b < batch; ++b) {
        live += positions[b] >= 0;
        turns += steps_of(b);
        longest = std::max(longest, steps_of(b));
    }
    turns *= (rows + 255) / 256 * kv_heads;
    if (rows <= 16) p.rows = 16;
    else if (forced_rows > 0) p.rows = forced_rows;
    else if (rows <= 32 || (turns < kManyTurns && rows * kv_heads * live < 32 * cus)) p.rows = 32;
    else if (turns < kManyTurns) p.rows = 64;
    else p.rows = rows <= 48 ? 48 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    p.chunks = static_cast<int32_t>((rows + p.rows - 1) / p.rows);
    const int64_t pairs = static_cast<int64_t>(batch) * kv_heads * p.chunks;
    auto whole = [](int64_t steps) { return (steps + kSplitQuantumSteps - 1) / kSplitQuantumSteps * kSplitQuantumSteps; };
    auto groups = [&](int64_t per) {
        int64_t sum = 0;
        for (int32_t b = 0; b < batch; ++b) sum += (steps_of(b) + per - 1) / per;
        return sum * kv_heads * p.chunks;
    };
    const int64_t most_splits = std::min<int64_t>(32, std::ceil(std::sqrt(longest / 2.0)));
    int64_t low = whole((longest + most_splits - 1) / most_splits), per = whole(longest);
    if (live * kv_heads * p.chunks < cus)
        while (low < per) {              // the fewest steps with which the workgroups find a CU each
            const int64_t middle = whole((low + per - kSplitQuantumSteps) / 2);
            if (groups(middle) <= cus) per = middle;
            else low = middle + kSplitQuantumSteps;
        }
    if (split_tokens > 0) per = split_tokens / kStepTokens;
    // what the workspace holds
    const int64_t most = std::min(kMaxSplitGroups, kMaxPartialRows / p.rows) / pairs;
    if (most <= 1) per = longest;
    else per = std::max(per, (longest + most - 1) / most);
    per = whole(per);
    p.split_steps = static_cast<int32_t>(per);
    p.splits = static_cast<int32_t>((longest + per - 1) / per);
    p.appends = n <= kTreeTokens;
    return p;
}

}  // namespace

extern "C" {

int swiftkv_paged_cache_create(swiftkv_context* ctx, int32_t layers, int32_t pages, int32_t max_batch, int32_t heads,
                               int32_t kv_heads, int32_t head_dim, int32_t max_seq_len, int32_t dtype,
                               swiftkv_paged_cache** out) {
    if (!ctx || !out) return fail(SWIFTKV_EINVAL, "null argument");
    *out = nullptr;
    if (int rc = not_capturing(ctx, "swiftkv_paged_cache_create")) return rc;
    if (layers < 1 || layers > 256) return fail(SWIFTKV_EINVAL, "layers %d outside [1, 256]", layers);
    if (pages < 1 || pages > (1 << 24)) return fail(SWIFTKV_EINVAL, "pages %d outside [1, 2^24]", pages);
    if (max_batch < 1 || max_batch > 4096) return fail(SWIFTKV_EINVAL, "max_batch %d outside [1, 4096]", max_batch);
    if (kv_heads < 1 || kv_heads > 256 || heads < kv_heads || heads % kv_heads != 0 || heads / kv_heads > 64)
        return fail(SWIFTKV_EINVAL, "heads %d, kv_heads %d: kv_heads within [1, 256], heads a multiple of it, at most 64 "
                    "times", heads, kv_heads);
    if (head_dim != 64 && head_dim != 128) return fail(SWIFTKV_EINVAL, "head_dim %d: must be 64 or 128", head_dim);
    if (max_seq_len < 1 || max_seq_len > kPagedMaxSeq)
        return fail(SWIFTKV_EINVAL, "max_seq_len %d outside [1, %d]", max_seq_len, kPagedMaxSeq);
    if (dtype != kBF16 && dtype != kF16) return fail(SWIFTKV_EINVAL, "element type %d: must be SWIFTKV_BF16 or SWIFTKV_F16", dtype);
    int rc = set_device(ctx);
    if (rc) return rc;
    if (!ctx->paged_workspace) {
        void* p = nullptr;
        const size_t counters = kMaxSplitGroups * kCounterStride * sizeof(uint32_t);
        const size_t bytes = counters + kPartialFloats * sizeof(float);
        if (!device_malloc(&p, bytes)) return fail(SWIFTKV_ENOMEM, "hipMalloc of %zu bytes failed", bytes);
        const hipError_t e = hipMemsetAsync(p, 0, counters, ctx->stream);
        if (e != hipSuccess) {
            (void)hipFree(p);
            return fail(SWIFTKV_EHIP, "split counters: %s", hipGetErrorString(e));
        }
        ctx->paged_workspace = static_cast<uint32_t*>(p);
    }
    const int32_t entries = (max_seq_len + kPageTokens - 1) / kPageTokens;
    swiftkv_paged_cache* c = new (std::nothrow) swiftkv_paged_cache();
    if (!c) return fail(SWIFTKV_ENOMEM, "out of host memory");
    try {
        c->table = new PageTable(max_batch, entries, pages);
    } catch (const std::bad_alloc&) {
        delete c;
        return fail(SWIFTKV_ENOMEM, "out of host memory");
    }
    c->ctx = ctx;
    c->max_batch = max_batch;
    c->heads = heads;
    c->capacity = entries * kPageTokens;
    c->type = static_cast<ElementType>(dtype);
    c->view.pages = pages;
    c->view.entries = entries;
    c->view.layers = layers;
    c->view.kv_heads = kv_heads;
    c->view.head_dim = head_dim;
    const size_t records = static_cast<size_t>(layers) * static_cast<size_t>(pages) * static_cast<size_t>(kv_heads) *
                           static_cast<size_t>(paged_record_bytes(head_dim));
    const size_t table = static_cast<size_t>(max_batch) * static_cast<size_t>(entries) * sizeof(int32_t);
    c->bytes = records + table;
    void* p = nullptr;
    if (!device_malloc(&p, c->bytes)) {
        const size_t bytes = c->bytes;
        delete c->table;
        delete c;
        return fail(SWIFTKV_ENOMEM, "hipMalloc of a paged cache (%zu bytes) failed", bytes);
    }
    c->view.base = static_cast<uint8_t*>(p);
    c->view.table = reinterpret_cast<int32_t*>(c->view.base + records);
    hipError_t e = hipMemsetAsync(p, 0, records, ctx->stream);
    if (e == hipSuccess) e = hipMemsetAsync(c->view.table, 0xff, table, ctx->stream);
    if (e == hipSuccess) e = hipStreamSynchronize(ctx->stream);
    if (e != hipSuccess) {
        (void)hipFree(p);
        delete c->table;
        delete c;
        return fail(SWIFTKV_EHIP, "paged cache: %s", hipGetErrorString(e));
    }
    ++ctx->children;
    *out = c;
    return ok();
}

int swiftkv_paged_cache_destroy(swiftkv_paged_cache* cache) {
    if (!cache) return ok();
    swiftkv_context* ctx = cache->ctx;
    if (int rc = not_capturing(ctx, "swiftkv_paged_cache_destroy")) return rc;
    (void)hipSetDevice(ctx->device);
    (void)hipStreamSynchronize(ctx->stream);
    (void)hipFree(cache->view.base);
    delete cache->table;
    delete cache;
    release_child(ctx);
    return ok();
}

size_t swiftkv_paged_cache_bytes(const swiftkv_paged_cache* cache) { return cache ? cache->bytes : 0; }

int swiftkv_paged_map(swiftkv_context* ctx, swiftkv_paged_cache* cache, int32_t seq, int32_t first, const int32_t* pages,
                      int32_t n) {
    int rc = check_idle_io(ctx);
    if (rc) return rc;
    if ((rc = not_capturing(ctx, "swiftkv_paged_map"))) return rc;
    if (!cache || cache->ctx != ctx) return fail(SWIFTKV_EINVAL, "cache is null or belongs to another context");
    if (!pages) return fail(SWIFTKV_EINVAL, "null pages");
    if (seq < 0 || seq >= cache->max_batch) return fail(SWIFTKV_ERANGE, "sequence %d outside [0, %d)", seq, cache->max_batch);
    if (n < 0 || first < 0 || static_cast<int64_t>(first) + n > cache->view.entries)
        return fail(SWIFTKV_ERANGE, "entries [%d, %lld) outside [0, %d)", first, static_cast<long long>(first) + n,
                    cache->view.entries);
    const int32_t bad = cache->table->first_bad(pages, n);
    if (bad < n) return fail(SWIFTKV_ERANGE, "pages[%d] = %d outside [-1, %d)", bad, pages[bad], cache->table->pages());
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;
    for (int32_t i0 = 0; i0 < n; i0 += kMapEntries) {
        PagedMapArgs a{};
        a.entries = cache->view.table + static_cast<int64_t>(seq) * cache->view.entries + first + i0;
        a.n = std::min(kMapEntries, n - i0);
        std::memcpy(a.pages, pages + i0, sizeof(int32_t) * static_cast<size_t>(a.n));
        SKV_HIP(launch_paged_map(a, ctx->stream));
        cache->table->assign(seq, first + i0, pages + i0, a.n);
    }
    return ok();
}

int swiftkv_paged_copy(swiftkv_context* ctx, swiftkv_paged_cache* cache, int32_t from, int32_t to) {
    int rc = check_idle_io(ctx);
    if (rc) return rc;
    if (!cache || cache->ctx != ctx) return fail(SWIFTKV_EINVAL, "cache is null or belongs to another context");
    const int32_t pages = cache->table->pages();
    if (from < 0 || from >= pages || to < 0 || to >= pages)
        return fail(SWIFTKV_ERANGE, "pages %d and %d outside [0, %d)", from, to, pages);
    if (from == to) return ok();
    if (cache->table->uses(to) > 1) return fail(SWIFTKV_ESTATE, "page %d is named by %d entries", to, cache->table->uses(to));
    if ((rc = set_device(ctx))) return rc;
    SKV_HIP(launch_paged_copy(cache->view, from, to, ctx->stream));
    return ok();
}

int swiftkv_paged_append(swiftkv_context* ctx, const swiftkv_rotary_table* table, int32_t halves, const void* k,
                         int64_t k_stride, const void* v, int64_t v_stride, swiftkv_paged_cache* cache,
                         int32_t layer_index, int32_t seq0, const int32_t* positions, const int32_t* parents,
                         int32_t batch, int32_t n) {
    int rc = check_call(ctx, cache, layer_index, 1, seq0, positions, batch, n);
    if (rc) return rc;
    const int64_t row = static_cast<int64_t>(cache->view.kv_heads) * cache->view.head_dim;
    if ((rc = check_tensor("k", k, k_stride, row, cache->type))) return rc;
    if ((rc = check_tensor("v", v, v_stride, row, cache->type))) return rc;
    if ((rc = check_tokens(cache, table, parents, seq0, positions, batch, n, true))) return rc;
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;
    if ((rc = append_rows(ctx, rotation_of(table, halves), k, k_stride, v, v_stride, cache, layer_index, seq0, positions,
                          parents, batch, n)))
        return rc;
    return ok();
}

int swiftkv_paged_values(swiftkv_context* ctx, const swiftkv_paged_cache* cache, int32_t layer0, int32_t layers,
                         int32_t seq0, const int32_t* positions, int32_t batch, int32_t n, void* k, void* v) {
    int rc = check_call(ctx, cache, layer0, layers, seq0, positions, batch, n);
    if (rc) return rc;
    const int64_t row = static_cast<int64_t>(cache->view.kv_heads) * cache->view.head_dim;
    if ((rc = check_tensor("k", k, row, row, cache->type))) return rc;
    if ((rc = check_tensor("v", v, row, row, cache->type))) return rc;
    if ((rc = check_tokens(cache, nullptr, nullptr, seq0, positions, batch, n, false))) return rc;
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;
    PagedRowsArgs a{};
    a.view = cache->view;
    a.layer = layer0;
    a.n = n;
    a.layer_rows = static_cast<int64_t>(batch) * n;
    for (int32_t b0 = 0; b0 < batch; b0 += kPagedBatch) {
        const int32_t nb = std::min<int32_t>(kPagedBatch, batch - b0);
        const int64_t at = static_cast<int64_t>(b0) * n * row * 2;
        a.k_out = static_cast<char*>(k) + at;
        a.v_out = static_cast<char*>(v) + at;
        a.slot0 = seq0 + b0;
        std::memcpy(a.positions, positions + b0, sizeof(int32_t) * static_cast<size_t>(nb));
        SKV_HIP(launch_paged_values(a, layers, nb, ctx->stream));
    }
    return ok();
}

int swiftkv_paged_attention(swiftkv_context* ctx, const swiftkv_rotary_table* table, int32_t halves, const void* q,
                            int64_t q_stride, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                            swiftkv_paged_cache* cache, int32_t layer_index, int32_t seq0, const int32_t* positions,
                            const int32_t* parents, int32_t batch, int32_t n, float scale, void* out,
                            int64_t out_stride) {
    int rc = check_call(ctx, cache, layer_index, 1, seq0, positions, batch, n);
    if (rc) return rc;
    const PagedView& view = cache->view;
    const int64_t kv_row = static_cast<int64_t>(view.kv_heads) * view.head_dim;
    const int64_t q_row = static_cast<int64_t>(cache->heads) * view.head_dim;
    if ((rc = check_tensor("q", q, q_stride, q_row, cache->type))) return rc;
    if ((rc = check_tensor("out", out, out_stride, q_row, cache->type))) return rc;
    if ((k == nullptr) != (v == nullptr)) return fail(SWIFTKV_EINVAL, "k and v must both be set or both be null");
    if (k && (rc = check_tensor("k", k, k_stride, kv_row, cache->type))) return rc;
    if (v && (rc = check_tensor("v", v, v_stride, kv_row, cache->type))) return rc;
    const float magnitude = std::fabs(scale);
    if (scale != 0.0f && !(magnitude >= 0x1p-100f && magnitude <= 0x1p100f))
        return fail(SWIFTKV_EINVAL, "scale must be 0 or of a magnitude within [2^-100, 2^100]");
    const int32_t group = cache->heads / view.kv_heads;
    if ((static_cast<int64_t>(group) * n + 15) / 16 * view.kv_heads >= kMaxGroups)
        return fail(SWIFTKV_ERANGE, "n = %d: %d heads take %lld workgroups and more", n, cache->heads,
                    static_cast<long long>(kMaxGroups));
    if ((rc = check_tokens(cache, table, parents, seq0, positions, batch, n, k != nullptr))) return rc;
    if (n == 0) return ok();
    if ((rc = set_device(ctx))) return rc;

    PagedAttendArgs a{};
    a.view = view;
    a.rotation = rotation_of(table, halves);
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.scale = (scale == 0.0f ? 1.0f / std::sqrt(static_cast<float>(view.head_dim)) : magnitude) * kLog2E;
    a.slack = kScoreSlack / a.scale;
    a.negative = scale < 0.0f;
    a.group = group;
    a.group_magic = group == 1 ? 0u : static_cast<uint32_t>(((uint64_t(1) << 32) + group - 1) / group);
    a.n = n;
    a.layer = layer_index;
    a.counters = ctx->paged_workspace;
    a.partials = reinterpret_cast<float*>(ctx->paged_workspace + kMaxSplitGroups * kCounterStride);
    const int32_t most = launch_batch(parents != nullptr, n);
    for (int32_t b0 = 0; b0 < batch; b0 += most) {
        const int32_t nb = std::min(most, batch - b0);
        const PagedPlan plan = plan_attention(ctx->cus, ctx->split_tokens, ctx->paged_rows, group, view.kv_heads, n, positions + b0, nb);
        const int64_t first = static_cast<int64_t>(b0) * n;
        a.q = static_cast<const char*>(q) + first * q_stride * 2;
        a.out = static_cast<char*>(out) + first * out_stride * 2;
        a.k = a.v = nullptr;
        if (k && plan.appends) {
            a.k = static_cast<const char*>(k) + first * k_stride * 2;
            a.v = static_cast<const char*>(v) + first * v_stride * 2;
        } else if (k && (rc = append_rows(ctx, a.rotation, static_cast<const char*>(k) + first * k_stride * 2, k_stride,
                                          static_cast<const char*>(v) + first * v_stride * 2, v_stride, cache, layer_index,
                                          seq0 + b0, positions + b0, parents ? parents + first : nullptr, nb, n))) {
            return rc;
        }
        a.slot0 = seq0 + b0;
        a.chunks = plan.chunks;
        a.splits = plan.splits;
        a.split_steps = plan.split_steps;
        for (int32_t b = 0; b < nb; ++b) a.order[b] = {positions[b0 + b], b};
        if (nb > 1)
            std::sort(a.order, a.order + nb, [](const PagedRow& x, const PagedRow& y) {
                return x.position != y.position ? x.position > y.position : x.sequence < y.sequence;
            });
        a.batch = nb;
        a.all_splits = 0;
        if (plan.splits > 1) {
            std::fill(std::begin(a.first_split), std::end(a.first_split), ~0u);
            for (int32_t y = 0; y < nb; ++y) {
                uint32_t& word = a.first_split[y / 2];
                const uint32_t first = static_cast<uint32_t>(a.all_splits);
                word = y % 2 ? (word & 0xffffu) | first << 16 : (word & 0xffff0000u) | first;
                const int32_t steps = a.order[y].position < 0 ? 0 : (a.order[y].position + n + kStepTokens - 1) / kStepTokens;
                a.all_splits += std::max(1, (steps + plan.split_steps - 1) / plan.split_steps);
            }
            // Finding its split costs a workgroup 1 us, for nothing where none is missing or
            // each is a workgroup on every XCD anyway.
            if (a.all_splits == nb * plan.splits || view.kv_heads % kXcds == 0) a.all_splits = 0;
        }
        PagedTree tree;
        const PagedTree* const trees = tree_of(tree, parents, b0, nb, n);
        SKV_HIP(plan.rows <= 64 ? launch_paged_attend(a, trees, nb, plan.rows, cache->type, ctx->stream)
                                : launch_paged_many(a, trees, nb, plan.rows, cache->type, ctx->stream));
        if (plan.splits > 1 && plan.rows > 16)
            SKV_HIP(launch_paged_join(a, trees, nb, plan.rows, cache->type, ctx->stream));
    }
    return ok();
}

int swiftkv_paged_keep(swiftkv_context* ctx, swiftkv_paged_cache* cache, int32_t layer0, int32_t layers, int32_t seq0,
                       const int32_t* positions, const int32_t* accepted, int32_t batch, int32_t m,
                       int32_t* out_positions) {
    int rc = check_call(ctx, cache, layer0, layers, seq0, positions, batch, 0);
    if (rc) return rc;
    if (!accepted) return fail(SWIFTKV_EINVAL, "null accepted");
    if (m < 0 || m > kTreeTokens) return fail(SWIFTKV_ERANGE, "m = %d outside [0, %d]", m, kTreeTokens);
    for (int32_t b = 0; b < batch; ++b) {
        const int32_t* path = accepted + static_cast<int64_t>(b) * m;
        const int32_t count = accepted_tokens(path, m);
        if (count < 0)
            return fail(SWIFTKV_EINVAL, "accepted tokens of sequence %d: [%d] = %d", b, -1 - count, path[-1 - count]);
        if (positions[b] < 0) continue;
        if ((rc = check_pages(cache, seq0 + b, b, positions[b], count == 0 ? 0 : path[count - 1] + 1, false))) return rc;
        for (int32_t j = 0; j < count; ++j)      // rows that move write their target's page
            if (path[j] != j) {
                if ((rc = check_pages(cache, seq0 + b, b, positions[b] + j, count - j, true))) return rc;
                break;
            }
    }
    if (m > 0) {
        if ((rc = set_device(ctx))) return rc;
        PagedKeepArgs a{};
        a.view = cache->view;
        a.layer0 = layer0;
        a.m = m;
        const int32_t most = launch_batch(true, m);
        for (int32_t b0 = 0; b0 < batch; b0 += most) {
            const int32_t nb = std::min(most, batch - b0);
            a.slot0 = seq0 + b0;
            std::memcpy(a.positions, positions + b0, sizeof(int32_t) * static_cast<size_t>(nb));
            set_bytes(a.accepted, accepted, b0, nb, m, 255, 255);
            SKV_HIP(launch_paged_keep(a, layers, nb, ctx->stream));
        }
    }
    if (out_positions)
        for (int32_t b = 0; b < batch; ++b)
            out_positions[b] = positions[b] < 0 ? positions[b]
                                                : positions[b] + accepted_tokens(accepted + static_cast<int64_t>(b) * m, m);
    return ok();
}

int swiftkv_debug_set_paged_rows(swiftkv_context* ctx, int32_t rows) {
    if (!ctx) return fail(SWIFTKV_EINVAL, "null context");
    if (rows != 0 && rows != 32 && rows != 48 && rows != 64 && rows != 128 && rows != 256)
        return fail(SWIFTKV_EINVAL, "rows %d: must be 0, 32, 48, 64, 128 or 256", rows);
    ctx->paged_rows = rows;
    return ok();
}

int swiftkv_debug_paged_plan(int32_t cus, int32_t split_tokens, int32_t heads, int32_t kv_heads, int32_t n,
                             const int32_t* positions, int32_t batch, int32_t* out_rows, int32_t* out_chunks,
                             int32_t* out_splits, int32_t* out_split_tokens) {
    if (!positions || !out_rows || !out_chunks || !out_splits || !out_split_tokens) return fail(SWIFTKV_EINVAL, "null argument");
    if (cus < 1 || split_tokens < 0 || kv_heads < 1 || kv_heads > 256 || heads < kv_heads || heads % kv_heads != 0 ||
        heads / kv_heads > 64 || n < 1 || n > kPagedMaxSeq || batch < 1 || batch > kPagedBatch)
        return fail(SWIFTKV_EINVAL, "cus %d, heads %d over %d, n %d, batch %d", cus, heads, kv_heads, n, batch);
    const PagedPlan p = plan_attention(cus, split_tokens, 0, heads / kv_heads, kv_heads, n, positions, batch);
    *out_rows = p.rows;
    *out_chunks = p.chunks;
    *out_splits = p.splits;
    *out_split_tokens = p.split_steps * kStepTokens;
    return ok();
}

}  // extern "C"
