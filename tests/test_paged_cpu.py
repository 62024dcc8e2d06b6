"""The paged cache without a device: what its entries refuse, the host's rules for pages, trees and accepted paths, the
launch plan."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

RULES = r"""
#include <cassert>
#include "swiftkv_paged_host.hpp"
using namespace swiftkv;
int main() {
    PageTable t(2, 4, 3);
    const int32_t a[4] = {2, 0, -1, 1}, one[1] = {2}, none[2] = {-1, -1}, bad[3] = {0, 3, -2};
    assert(t.first_bad(a, 4) == 4 && t.first_bad(bad, 3) == 1 && t.first_bad(bad + 2, 1) == 0);
    assert(t.holds(0, 0, 64) && !t.holds(0, 1, 64));
    t.assign(0, 0, a, 4);
    assert(t.holds(0, 128, 64) && !t.holds(0, 129, 64));
    assert(t.not_own(0, 0, 128, 64) == -1 && t.not_own(0, 5, 5, 64) == -1 && t.not_own(0, 127, 129, 64) == 2);
    t.assign(1, 0, one, 1);                       // shares page 2
    assert(t.uses(2) == 2 && t.not_own(0, 63, 64, 64) == 0 && t.not_own(0, 64, 65, 64) == -1 && t.not_own(1, 0, 1, 64) == 0);
    t.assign(0, 0, none, 2);
    assert(t.uses(2) == 1 && t.uses(0) == 0 && !t.holds(0, 1, 64) && t.not_own(1, 0, 64, 64) == -1);
    t.assign(0, 2, one, 1);                       // behind a gap
    assert(!t.holds(0, 1, 64));
    t.assign(0, 0, a, 2);                         // page 2 twice in one sequence
    assert(t.holds(0, 256, 64) && t.uses(2) == 3 && t.not_own(0, 0, 1, 64) == 0);

    const int32_t tree[5] = {-1, 0, 0, -2, -2}, gap[3] = {-1, -2, 0}, self[2] = {-1, 1}, later[2] = {1, -1}, low[1] = {-3};
    assert(tree_tokens(tree, 5) == 3 && tree_tokens(tree, 0) == 0 && tree_tokens(tree + 3, 2) == 0);
    assert(tree_tokens(gap, 3) == -3 && tree_tokens(self, 2) == -2 && tree_tokens(later, 2) == -1 && tree_tokens(low, 1) == -1);
    assert(tree_depth(tree, 3) == 1 && tree_depth(tree, 0) == -1);
    int32_t chain[64];
    for (int i = 0; i < 64; ++i) chain[i] = i - 1;
    assert(tree_tokens(chain, 64) == 64 && tree_depth(chain, 64) == 63);

    const int32_t path[4] = {0, 3, 63, -1}, same[2] = {1, 1}, hole[2] = {-1, 4}, high[1] = {64}, minus[1] = {-2};
    assert(accepted_tokens(path, 4) == 3 && accepted_tokens(path + 3, 1) == 0 && accepted_tokens(same, 2) == -2);
    assert(accepted_tokens(hole, 2) == -2 && accepted_tokens(high, 1) == -1 && accepted_tokens(minus, 1) == -1);
    return 0;
}
"""


def test_host_rules(tmp_path):
    src = tmp_path / "rules.cpp"
    src.write_text(RULES)
    exe = str(tmp_path / "rules")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-D_GLIBCXX_ASSERTIONS", "-I",
                    os.path.join(REPO, "4pe_u250_amd", "csrc"), str(src), "-o", exe], check=True)
    subprocess.run([exe], check=True)


def run_rules(tmp_path, text):
    src = tmp_path / "rules.cpp"
    src.write_text(text)
    exe = str(tmp_path / "rules")
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-D_GLIBCXX_ASSERTIONS", "-I",
                    os.path.join(REPO, "4pe_u250_amd", "csrc"), str(src), "-o", exe], check=True)
    subprocess.run([exe], check=True)


APPENDED_ROWS = r"""
#include <cassert>
#include <initializer_list>
#include "swiftkv_paged_rows.hpp"
using namespace swiftkv;
int main() {
    for (int n : {1, 2, 7, 31, 32, 33, 64, 65, 100})
        for (int p = 0; p < 200; ++p)
            for (int count = 0; count <= n; ++count) {       // of a tree; n for a chain
                int stored = 0;
                for (int y = 0; y < (n + 62) / 32; ++y) {    // the launch's steps
                    const int tok0 = (p / 32 + y) * 32, end = p + count;
                    if (!step_has_new(tok0, p, end)) continue;
                    for (int tok = tok0; tok < tok0 + 32; ++tok) {
                        const int i = nearest_row(tok, p, end);
                        assert(i >= 0 && i < count);         // every load is of a row that is there
                        if (tok >= p && tok < end) {
                            assert(i == tok - p);
                            ++stored;
                        }
                    }
                }
                assert(stored == count);
            }
    return 0;
}
"""


def test_rows_that_an_append_reads(tmp_path):
    """None before a sequence's first or behind its last, for trees without tokens too."""
    run_rules(tmp_path, APPENDED_ROWS)


TURNED_POSITIONS = r"""
#include <cassert>
#include <initializer_list>
#include "swiftkv_paged_host.hpp"
#include "swiftkv_paged_rows.hpp"
using namespace swiftkv;
int main() {
    for (int positions : {1, 2, 64, 100})
        for (int n : {1, 2, 7, 64})
            for (int p : {-2147483647 - 1, -64, -5, -1, 0, 1, 36, 63, 64, 93, 98, 99, 100, 101}) {
                // a chain, and trees of every number of tokens: chains, and stars under one token
                if (turns_within(p, n - 1, positions))
                    for (int i = 0; i < n; ++i) {
                        const int at = turn_position(p, i, true);
                        assert(at >= 0 && at < positions && (p < 0 || at == p + i));
                    }
                for (int count = 0; count <= n; ++count)
                    for (int star = 0; star < 2; ++star) {
                        int parents[64], depth[64];
                        for (int i = 0; i < n; ++i) {
                            parents[i] = i >= count ? -2 : star && i > 0 ? 0 : i - 1;
                            depth[i] = parents[i] < 0 ? 0 : depth[parents[i]] + 1;
                        }
                        assert(tree_tokens(parents, n) == count);
                        if (!turns_within(p, tree_depth(parents, count), positions)) continue;
                        for (int i = 0; i < n; ++i) {        // rows without a token too: their queries are read
                            const int at = turn_position(p, depth[i], i < count);
                            assert(at >= 0 && at < positions && (p < 0 || i >= count || at == p + depth[i]));
                        }
                    }
            }
    assert(!turns_within(2147483647, 63, 2147483647) && turns_within(100, -1, 100) && !turns_within(100, 0, 100));
    return 0;
}
"""


def test_positions_that_are_looked_up(tmp_path):
    """All within the table for every call that the check lets pass: full sequences that bring no tokens, sequences that
    sit out, rows without a token."""
    run_rules(tmp_path, TURNED_POSITIONS)


def test_null_checks_without_device(skv):
    L = skv.lib()
    pos = np.zeros(1, np.int32).ctypes.data_as(C.c_void_p)
    h = C.c_void_p()
    assert L.swiftkv_paged_cache_create(None, 1, 1, 1, 1, 1, 64, 64, skv.BF16, C.byref(h)) == skv.EINVAL
    assert L.swiftkv_paged_map(None, None, 0, 0, pos, 1) == skv.EINVAL
    assert L.swiftkv_paged_copy(None, None, 0, 0) == skv.EINVAL
    assert L.swiftkv_paged_append(None, None, 0, None, 0, None, 0, None, 0, 0, pos, None, 1, 1) == skv.EINVAL
    assert L.swiftkv_paged_values(None, None, 0, 1, 0, pos, 1, 1, None, None) == skv.EINVAL
    assert L.swiftkv_paged_attention(None, None, 0, None, 0, None, 0, None, 0, None, 0, 0, pos, None, 1, 1, 0.0, None,
                                     0) == skv.EINVAL
    assert b"null" in L.swiftkv_last_error()
    assert L.swiftkv_paged_keep(None, None, 0, 1, 0, pos, pos, 1, 1, None) == skv.EINVAL
    assert L.swiftkv_debug_set_paged_rows(None, 0) == skv.EINVAL
    assert L.swiftkv_paged_cache_bytes(None) == 0 and L.swiftkv_paged_cache_destroy(None) == skv.OK


@pytest.mark.parametrize("heads,kv", [(32, 32), (32, 8), (20, 4), (64, 1), (256, 256)])
@pytest.mark.parametrize("n", [1, 3, 8, 26, 64, 512, 5000])
@pytest.mark.parametrize("batch", [1, 3, 64])
@pytest.mark.parametrize("split", [0, 256, 4096])
def test_plan_stays_within_the_workspace(skv, heads, kv, n, batch, split):
    """Every row has a chunk, every token a split, and the splits' counters and partial rows fit the workspace."""
    rng = np.random.default_rng(n * batch)
    for longest in (0, 1, 200, 4095, 120000):
        at = [longest] + [int(x) for x in rng.integers(-1, longest + 1, batch - 1)]
        rows, chunks, splits, tokens = skv.paged_plan(heads, kv, n, at, split_tokens=split)
        assert rows in (16, 32, 48, 64, 128, 256) and (rows > 16 or chunks == 1)
        assert rows * chunks >= n * (heads // kv) > rows * (chunks - 1)
        assert tokens % 128 == 0 and splits * tokens >= longest + n > (splits - 1) * tokens
        if splits > 1:
            assert batch * kv * chunks * splits <= 2048
            assert batch * kv * chunks * splits * rows <= 65536
