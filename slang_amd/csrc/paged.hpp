// The paged K/V cache as the kernels see it, and the host checks that its entry points share.
#pragma once

#include "common.hpp"
#include "paged_rows.hpp"

namespace g4a {

// Position p of sequence b is row p % page_size of page table[b * stride + p / page_size] of the
// pools [n_pages][page_size][kvH][hd]. Everything read from the device is bounded before it is
// used: lengths by max_len (the host's bound, which the table's cols cover), an entry outside
// [0, n_pages) is a page that is not there.
struct PageTab {
    const int32_t* table;
    const int32_t* key_len;
    int n_seq, stride, cols, n_pages, shift, max_len;
};

// keys of sequence b, those of this call included
__device__ __forceinline__ int paged_len(const PageTab& t, int b) { return min(max(t.key_len[b], 0), t.max_len); }

__device__ __forceinline__ bool page_ok(const PageTab& t, int page) { return (unsigned)page < (unsigned)t.n_pages; }

// the table entry of position p < max_len
__device__ __forceinline__ int page_at(const PageTab& t, int b, int p) {
    return t.table[(size_t)b * t.stride + (p >> t.shift)];
}

// Inclusive prefix sum over the 64 lanes on DPP row shifts and broadcasts (wave_prefix_sum without its six
// trips through the LDS crossbar).
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false);  // row_shr:1
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1 and 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2 and 3
    return x;
}

// rows of a 16-key block that lie in front of its end, n = end - block start, wave-uniform. (The clamp
// is a vector instruction; left in a vector register it would make the buffer resource it enters look
// divergent, and every load through it a loop over lanes.)
__device__ __forceinline__ int clamp16(int n) { return __builtin_amdgcn_readfirstlane(min(max(n, 0), 16)); }

// element offset of a position's row in the pools, `row` = kvH * hd elements
__device__ __forceinline__ size_t paged_row(const PageTab& t, int page, int p, int row) {
    return (((size_t)page << t.shift) + (size_t)(p & ((1 << t.shift) - 1))) * (size_t)row;
}

__device__ __forceinline__ SeqRows seq_rows(const PageTab& t, const int32_t* cu, int n_tokens, int b) {
    return cut_rows(cu[b], cu[b + 1], n_tokens, paged_len(t, b));
}

// The sequence of packed row `tok`: how many sequences end at or before it, 64 offsets a load
// (cu ascends; if it does not, any sequence). n_seq: a row behind the last sequence. Every lane of the wave must call it.
__device__ __forceinline__ int seq_of_row(const int32_t* cu, int n_seq, int tok) {
    const int lane = threadIdx.x & 63;
    int b = 0;
    for (int s0 = 0; s0 < n_seq; s0 += 64) {
        const int s = s0 + lane;
        const unsigned long long m = __ballot(s < n_seq && cu[s < n_seq ? s + 1 : 0] <= tok);
        b += __builtin_popcountll(m);
        if (m != ~0ull) break;
    }
    return b;
}

// checks of a g4a_paged and the config that goes with it; 0 or the error code (g4a_last_error set)
int check_paged(const g4a_cfg* cfg, const g4a_paged* pg, bool need_group_le8);
// ... of the operands that paged decode and prefill share, n_tokens rows of q and out
int check_paged_call(const g4a_cfg* cfg, int n_tokens, const float* q, const float* q_gain, const float* rcos,
                     const float* rsin, const void* out);
int check_tokens(const g4a_cfg* cfg, int n_tokens, const int32_t* cu);
int check_rope(const float* rcos, const float* rsin);
int check_steps(float k_in_q, float v_in_q);
PageTab page_tab(const g4a_paged* pg);

}  // namespace g4a
