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

}  // namespace g4a
