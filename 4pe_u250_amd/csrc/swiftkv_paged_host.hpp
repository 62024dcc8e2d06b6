// swiftkv_paged_host.hpp -- the paged cache's host-side rules, without a device:
// which pages a sequence has, and what a tree of drafted tokens may look like.
#pragma once

#include <cstddef>
#include <cstdint>
#include <vector>

namespace swiftkv {

// The table as the host knows it: the page of each entry (64 tokens) of each
// sequence, how many entries name a page, how many entries from the first on have
// one.
class PageTable {
public:
    // May throw std::bad_alloc.
    PageTable(int32_t sequences, int32_t entries, int32_t pages)
        : entries_(entries), pages_(pages), page_(static_cast<size_t>(sequences) * entries, -1),
          uses_(static_cast<size_t>(pages), 0), leading_(static_cast<size_t>(sequences), 0) {}

    int32_t entries() const { return entries_; }
    int32_t pages() const { return pages_; }
    int32_t page(int32_t seq, int32_t entry) const { return page_[at(seq, entry)]; }
    int32_t uses(int32_t page) const { return uses_[static_cast<size_t>(page)]; }

    // The first index of `pages` that is neither -1 nor a page, or n.
    int32_t first_bad(const int32_t* pages, int32_t n) const {
        for (int32_t i = 0; i < n; ++i)
            if (pages[i] < -1 || pages[i] >= pages_) return i;
        return n;
    }

    void assign(int32_t seq, int32_t first, const int32_t* pages, int32_t n) {
        for (int32_t i = 0; i < n; ++i) {
            int32_t& p = page_[at(seq, first + i)];
            if (p >= 0) --uses_[static_cast<size_t>(p)];
            p = pages[i];
            if (p >= 0) ++uses_[static_cast<size_t>(p)];
        }
        int32_t& lead = leading_[static_cast<size_t>(seq)];
        if (first > lead) return;
        lead = first;
        while (lead < entries_ && page_[at(seq, lead)] >= 0) ++lead;
    }

    // Whether the entries of tokens [0, end) all have a page.
    bool holds(int32_t seq, int64_t end, int32_t page_tokens) const {
        return end <= static_cast<int64_t>(leading_[static_cast<size_t>(seq)]) * page_tokens;
    }

    // A page among those of tokens [begin, end) that another entry names too, or that
    // is missing: its entry, or -1.
    int32_t not_own(int32_t seq, int32_t begin, int32_t end, int32_t page_tokens) const {
        if (begin >= end) return -1;
        for (int32_t e = begin / page_tokens; e <= (end - 1) / page_tokens; ++e) {
            const int32_t p = page_[at(seq, e)];
            if (p < 0 || uses_[static_cast<size_t>(p)] != 1) return e;
        }
        return -1;
    }

private:
    size_t at(int32_t seq, int32_t entry) const { return static_cast<size_t>(seq) * entries_ + entry; }
    int32_t entries_, pages_;
    std::vector<int32_t> page_, uses_, leading_;
};

// Tokens of a tree: parents[i] within [-1, i), or -2 for all from some i on.
// Returns their number, or -1 - i for a parent that breaks the rule.
inline int32_t tree_tokens(const int32_t* parents, int32_t n) {
    int32_t count = 0;
    while (count < n && parents[count] != -2) {
        if (parents[count] < -1 || parents[count] >= count) return -1 - count;
        ++count;
    }
    for (int32_t i = count; i < n; ++i)
        if (parents[i] != -2) return -1 - i;
    return count;
}

// The largest depth of a tree's tokens (n <= 64); -1 without one.
inline int32_t tree_depth(const int32_t* parents, int32_t count) {
    int32_t depth[64], most = -1;
    for (int32_t i = 0; i < count; ++i) {
        depth[i] = parents[i] < 0 ? 0 : depth[parents[i]] + 1;
        if (depth[i] > most) most = depth[i];
    }
    return most;
}

// Accepted tokens of a tree: rising within [0, 64), then -1.  Returns their
// number, or -1 - j for one that breaks the rule.
inline int32_t accepted_tokens(const int32_t* accepted, int32_t m) {
    int32_t count = 0;
    while (count < m && accepted[count] != -1) {
        if (accepted[count] < 0 || accepted[count] >= 64 || (count > 0 && accepted[count] <= accepted[count - 1]))
            return -1 - count;
        ++count;
    }
    for (int32_t j = count; j < m; ++j)
        if (accepted[j] != -1) return -1 - j;
    return count;
}

// The launch of one attention call.
struct PagedPlan {
    int32_t rows;        // of a workgroup's chunk
    int32_t chunks, splits, split_steps;
    bool appends;        // in the attention's own launch
};

}  // namespace swiftkv
