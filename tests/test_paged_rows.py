"""Positions of packed rows (csrc/paged_rows.hpp), evaluated by the host compiler over offsets that
ascend and ones that do not: a row that a kernel goes on with has a position below its sequence's keys."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "slang_amd", "csrc")

# seq_of_row and seq_rows as the kernels run them: 64 offsets at a time, counted by a ballot
PROLOGUE = """
#include <cstdint>
#include <initializer_list>
#include "paged_rows.hpp"
using namespace g4a;
constexpr int kSeqs = 130;
struct Cu {
    int n = 0, at[kSeqs + 1] = {};
};
constexpr int seq_of_row(const Cu& cu, int tok) {
    int b = 0;
    for (int s0 = 0; s0 < cu.n; s0 += 64) {
        int count = 0;
        for (int s = s0; s < s0 + 64; ++s) count += s < cu.n && cu.at[s + 1] <= tok;
        b += count;
        if (count < 64) break;
    }
    return b;
}
constexpr Cu offsets(std::initializer_list<int> v) {
    Cu c;
    c.n = (int)v.size() - 1;
    int i = 0;
    for (int x : v) c.at[i++] = x;
    return c;
}
constexpr Cu random_offsets(uint32_t seed, int n, int lo, int hi) {
    Cu c;
    c.n = n;
    for (int i = 0; i <= n; ++i) {
        seed = seed * 1664525u + 1013904223u;
        c.at[i] = lo + (int)((seed >> 8) % (uint32_t)(hi - lo + 1));
    }
    return c;
}
"""


def holds(tmp_path, body):
    cxx = shutil.which("g++") or shutil.which("clang++")
    if cxx is None:
        pytest.skip("no host C++ compiler")
    src = tmp_path / "rows.cpp"
    src.write_text(PROLOGUE + body)
    limit = ["-fconstexpr-ops-limit=400000000", "-fconstexpr-loop-limit=10000000"] if "g++" in os.path.basename(cxx) \
        and "clang" not in cxx else ["-fconstexpr-steps=400000000"]
    p = subprocess.run([cxx, "-std=c++17", "-fsyntax-only", *limit, f"-I{CSRC}", str(src)], capture_output=True, text=True)
    assert p.returncode == 0, p.stderr


def test_no_row_past_the_keys(tmp_path):
    """Every row of every list: the position is below the sequence's keys, or the row is left out."""
    holds(tmp_path, """
constexpr bool within(const Cu& cu, int tokens, int keys) {
    for (int tok = 0; tok < tokens; ++tok) {
        const int b = seq_of_row(cu, tok);
        if (b >= cu.n) continue;
        const SeqRows r = cut_rows(cu.at[b], cu.at[b + 1], tokens, keys);
        if (r.lo < 0 || r.hi < r.lo || r.hi > tokens) return false;
        if (holds(r, tok) && row_position(r, tok) >= keys) return false;
    }
    return true;
}
static_assert(within(offsets({0, 500, 5, 10}), 500, 600) && within(offsets({0, 660, 0, 0}), 660, 700), "");
static_assert(within(offsets({0, -5, 2147483647, -2147483647 - 1, 3}), 40, 10), "");
constexpr bool any() {
    for (uint32_t seed = 1; seed <= 60; ++seed)
        if (!within(random_offsets(seed, 1 + (int)(seed * 37 % kSeqs), -20, 120), 100, 1 + (int)(seed % 7) * 30)) return false;
    return true;
}
static_assert(any(), "a row past its sequence's keys");
// what `holds` keeps out: without it these rows' positions pass the keys by the packed rows before them
constexpr SeqRows none = cut_rows(5, 10, 500, 600);
static_assert(!holds(none, 499) && row_position(none, 499) == 1089, "");
""")


def test_ascending_offsets_reach_every_row(tmp_path):
    """Each packed row belongs to the sequence that lists it, empty ones between, rows behind to nobody."""
    holds(tmp_path, """
constexpr bool all() {
    for (int n : {1, 3, 63, 64, 65, 129, 130}) {
        Cu c;
        c.n = n;
        for (int i = 0; i < n; ++i) c.at[i + 1] = c.at[i] + (i * 7 + n) % 4;
        const int tokens = c.at[n] + 5;
        for (int b = 0; b < n; ++b)
            for (int i = c.at[b]; i < c.at[b + 1]; ++i) {
                const SeqRows r = cut_rows(c.at[b], c.at[b + 1], tokens, 50);
                if (seq_of_row(c, i) != b || !holds(r, i) || row_position(r, i) != 50 - (c.at[b + 1] - i)) return false;
            }
        for (int i = c.at[n]; i < tokens; ++i)
            if (seq_of_row(c, i) != n) return false;
    }
    return true;
}
static_assert(all(), "a row of another sequence");
""")


def test_tiles_of_the_longest_blocks(tmp_path):
    """Up to 2^30 keys: no step of the count, of a size class (63 classes of tiles) or of a piece's range (8 pieces)
    overflows, and a count that went through a 32-bit float is not taken for less than it is."""
    holds(tmp_path, """
constexpr int kMost = 1 << 30;
constexpr bool fits(int keys, int S, int bq, int kt, int window) {
    const int nb = (S + bq - 1) / bq;
    for (int qb : {0, nb / 2, nb - 1}) {
        const int64_t p0 = (int64_t)keys - S + (int64_t)qb * bq, hi = p0 + bq < keys ? p0 + bq : keys;
        const int64_t first = window > 0 && p0 + 1 > window ? p0 + 1 - window : 0, span = hi - first / 16 * 16;
        const int64_t want = span > 0 ? (span + kt - 1) / kt : 0;
        const int n = key_tiles(keys - S, S, qb, bq, kt, window);
        if (n != want || (int64_t)n * 63 > 0x7fffffff || (int64_t)n * 8 > 0x7fffffff) return false;
    }
    return true;
}
constexpr bool all() {
    for (int keys : {1, 15, 16, 17, 1000, kMost - 33, kMost - 1, kMost})
        for (int S : {1, 16, 100, 4000, 1 << 26})
            for (int bq : {16, 32, 64, 128})
                for (int kt : {32, 64})
                    for (int window : {0, 1, 16, 512, kMost})
                        if (!fits(keys, S, bq, kt, window)) return false;
    return true;
}
static_assert(all(), "a count that overflows");
constexpr bool bounded() {
    for (int n = 1; n < 1 << 25; n += n < 1 << 23 ? n / 8 + 1 : 997)
        if (tiles_at_least((int)(float)n) < n || (n <= 1 << 24 && n != 1 << 24 && tiles_at_least((int)(float)n) != n)) return false;
    return tiles_at_least((int)(float)(1 << 25)) >= 1 << 25;
}
static_assert(bounded(), "a count taken for less");
constexpr int n = key_tiles(32 * ((1 << 24) + 1) - 1, 1, 0, 16, 32, 0);
static_assert(n > 1 << 24 && (int)(float)n < n && tiles_at_least((int)(float)n) >= n, "");
""")
