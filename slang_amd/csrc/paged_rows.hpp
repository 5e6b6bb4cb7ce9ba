// Which packed rows are a sequence's, and at which positions, apart from the kernels so that a host
// compiler can evaluate it over offsets that no caller should pass (tests/test_paged_rows.py).
#pragma once

namespace g4a {

constexpr int cut_to(int x, int lo, int hi) { return x < lo ? lo : x > hi ? hi : x; }

// the packed rows [lo, hi) of a sequence and its keys: row lo + i is the token at position
// keys - (hi - lo) + i. Offsets outside [0, n_tokens] are cut to it, one below its predecessor to that.
struct SeqRows {
    int lo, hi, keys;
};
constexpr SeqRows cut_rows(int begin, int end, int n_tokens, int keys) {
    const int lo = cut_to(begin, 0, n_tokens), hi = cut_to(end, lo, n_tokens);
    return SeqRows{lo, hi, keys};
}
// The test and the position go together: offsets that do not ascend lead seq_of_row to a sequence whose
// rows `tok` is not among, where the position would pass the keys, and with them the RoPE tables.
constexpr bool holds(const SeqRows& r, int tok) { return tok >= r.lo && tok < r.hi; }
constexpr int row_position(const SeqRows& r, int tok) { return r.keys - r.hi + tok; }  // below keys if r holds tok

// Key tiles of query block qb of a sequence whose S tokens start at position `start`: keys
// [first & ~15, min(p0 + bq, start + S)), first the first one that the block attends.
constexpr int key_tiles(int start, int S, int qb, int bq, int kt, int window) {
    const int p0 = start + qb * bq, hi = p0 + bq < start + S ? p0 + bq : start + S;
    const int front = p0 + 1 - window, first = window > 0 ? (front > 0 ? front : 0) : 0;
    const int n = (hi - (first & ~15) + kt - 1) / kt;
    return n > 0 ? n : 0;
}
// A bound of a count (2^25 at most) that went through a 32-bit float, which above 2^24 may have made it one
// less: a longest block taken for shorter than it is would be cut where no partial has room.
constexpr int tiles_at_least(int rounded) { return rounded + (rounded >> 24); }

}  // namespace g4a
