// Attention of drafted trees over a paged K/V cache, for gfx950 on f16 MFMA.
//
// A tree's n tokens are its sequence's last rows, token i at row start + i, start = key_len - n. parents[i] < i names
// the token that i continues, anything else makes it a root, whose parent is the history's last key. So token i stands at
// position start + depth(i) and attends the history's keys t with start + depth(i) - t < W, and itself and its ancestors j
// with depth(i) - depth(j) < W. Everything else is paged_prefill.hip's: the same unit of columns x key tiles
// (paged_tiles.hpp), P and V as f16 operands, sums in f32, K/V rows through the page table. Scores are plain decoding's, so that
// drafts are checked as it would choose: q is a pair of f16 operands, and so are K and P over f32 caches (products of one
// remainder, not of two).
//
// Few tokens over a long history: the rows of K and V are read once for all of a tree's tokens, so the call is bound by
// them, and the history is what gets cut over the card. Three launches: rows (RoPE by depth, the k/v rows into their
// pages, q in two f16 operands, the tokens' bits, and in the first workgroup the work list), units, and the merge of their partials.
#include <algorithm>

#include "paged_tiles.hpp"

namespace g4a {

constexpr int kTreeSlots = 768;   // pieces with partials in a call
constexpr int kTreePieces = 256;  // pieces a query block is cut into
constexpr int kPlanThreads = 256;
constexpr int tree_columns(int HD) { return HD == 256 ? 128 : 64; }  // of a unit: tokens times heads of a kv head

struct TreeRowArgs : PagedTreeArgs {
    const void* k_new;
    const void* v_new;
    const float* k_gain;
    void* k_pages;
    void* v_pages;
    PageTab rows;  // the cache's own table (t is the f16 copy's where there is one)
    PagedKv16Args conv;
    int v_norm, q_groups;  // groups of four heads
    int conv_x, conv_z;    // f32 caches: the conversion's workgroups a sequence and 16 rows; 0: none
    float k_in_q, v_in_q;
};

__device__ __forceinline__ SeqRows tree_rows(const PageTab& t, const int32_t* cu, int n_tokens, int b) {
    return cut_tree(seq_rows(t, cu, n_tokens, b));
}

// ---------------------------------------------------------------- the work list
// Cost of a piece beside its tiles, of its partial and of the merge, in key tiles (about 2 us). (At hd 512 prices of 4 to 9 a piece
// and 1 to 2.5 a partial are within 1 % of each other over eight batches.)
struct TreeCost {
    float unit, part, merge;
};
__device__ __forceinline__ TreeCost tree_cost(int kt) { return kt == 64 ? TreeCost{4.8f, 1.5f, 2.0f} : TreeCost{6.0f, 2.5f, 2.0f}; }

// Pieces of the longest block in candidate c of 64: 1 .. 32, then every seventh up to 256.
__device__ __forceinline__ int tree_candidate(int c) { return c < 32 ? c + 1 : 32 + 7 * (c - 31); }

// floor(x / d) of x in [0, 2^31), r = 1 / d on the transcendental unit: the first product is off by 2^-22 of itself, the
// second, of what is left, by less than one, which the remainder puts right. A division by an unknown d takes the
// compiler some 35 dependent instructions, and the list is waited for by everything.
struct Over {
    int d;
    float r;
    __device__ __forceinline__ explicit Over(int d_) : d(d_), r(__builtin_amdgcn_rcpf((float)d_)) {}
    __device__ __forceinline__ int operator()(int x) const {
        int q = (int)((float)x * r), rest = x - q * d;
        const int more = (int)((float)rest * r);
        q += more;
        rest -= more * d;
        return q + (rest >= d ? 1 : rest < 0 ? -1 : 0);
    }
    __device__ __forceinline__ int up(int x) const { return (*this)(x + d - 1); }
};

// Written by one workgroup of kPlanThreads threads. A sequence's blocks all read its whole history, so they take the same
// number of pieces, ceil(tiles of the last block / st) for one st, the tiles that a piece may have. Lane c of every
// wave prices candidate c of st over a quarter of the sequences: units that all fit the card at once end with the longest
// of them; more end at the mean load of a CU, and half a unit.
__device__ void plan_trees(const TreeRowArgs& a) {
    __shared__ int s_lo[kPlanThreads], s_S[kPlanThreads], s_start[kPlanThreads], s_nt[kPlanThreads];
    __shared__ int s_at[3][kPlanThreads + 1], s_wave[3][kPlanThreads / 64], s_long;
    __shared__ float s_sum[kPlanThreads / 64][3][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int chunks = (a.t.n_seq + kPlanThreads - 1) / kPlanThreads, log_bq = 31 - __builtin_clz((unsigned)a.bq);
    if (tid == 0) s_long = 0;
    // the sequences c * kPlanThreads .. into LDS
    auto load_chunk = [&](int c) {
        __syncthreads();
        const int b = c * kPlanThreads + tid;
        SeqRows r{0, 0, 0};
        if (b < a.t.n_seq) r = tree_rows(a.t, a.cu, a.n_tokens, b);
        const int S = r.hi - r.lo, start = r.keys - S;
        s_lo[tid] = r.lo;
        s_S[tid] = S;
        s_start[tid] = start;
        s_nt[tid] = S > 0 ? tree_tiles(start, S, (S - 1) >> log_bq, a.bq, a.kt, a.window) : 0;
        __syncthreads();
    };
    load_chunk(0);
    for (int c = 0; c < chunks; ++c) {
        if (c > 0) load_chunk(c);
        atomicMax(&s_long, s_nt[tid]);
    }
    __syncthreads();
    const int longest = max(s_long, 1);
    int st = longest;
    if (a.max_slots > 0 && longest > 1) {  // workgroup-uniform
        const int my = max(Over(tree_candidate(lane)).up(longest), 1);
        const Over per(my);
        float units = 0.0f, slots = 0.0f, tiles = 0.0f;
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) load_chunk(c);
            for (int i = wave; i < min(kPlanThreads, a.t.n_seq - c * kPlanThreads); i += kPlanThreads / 64) {
                const int nb = (s_S[i] + a.bq - 1) >> log_bq, np = max(per.up(s_nt[i]), 1);
                units += (float)(nb * np);  // exact up to 2^24, far above the slots that there are
                slots += np > 1 ? (float)(nb * np) : 0.0f;
                tiles += (float)nb * (float)s_nt[i];
            }
        }
        s_sum[wave][0][lane] = units;
        s_sum[wave][1][lane] = slots;
        s_sum[wave][2][lane] = tiles;
        __syncthreads();
        units = slots = tiles = 0.0f;
#pragma unroll
        for (int w = 0; w < kPlanThreads / 64; ++w) {
            units += s_sum[w][0][lane];
            slots += s_sum[w][1][lane];
            tiles += s_sum[w][2][lane];
        }
        const float kvh = (float)a.n_kv_heads;
        units *= kvh;
        slots *= kvh;
        tiles *= kvh;
        const TreeCost pc = tree_cost(a.kt);
        const float piece = (float)my + pc.unit + (slots > 0.0f ? pc.part : 0.0f);
        float cost = units <= (float)kCus ? piece
                                          : fmaxf((tiles + units * pc.unit + slots * pc.part) * (1.0f / kCus) + 0.5f * piece, piece);
        if (slots > 0.0f) cost += pc.merge + 0.01f * slots;
        if (slots > (float)a.max_slots) cost = __builtin_huge_valf();
        const float best = -wave_max(-cost);
        const unsigned long long m = __ballot(cost == best);
        const int pick = __builtin_ctzll(m | 1ull << 63);
        st = __builtin_amdgcn_readlane(my, pick);
        __syncthreads();
    }
    const Over over_st(st);
    int at[3] = {0, 0, 0};  // units, slots, merges of the chunks before
    for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) load_chunk(c);
        const int nb = (s_S[tid] + a.bq - 1) >> log_bq, np = max(over_st.up(s_nt[tid]), 1);
        const int n[3] = {nb * np * a.n_kv_heads, np > 1 ? nb * np * a.n_kv_heads : 0, np > 1 ? nb * a.n_kv_heads : 0};
        int incl[3];
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            incl[i] = wave_scan(n[i]);
            if (lane == 63) s_wave[i][wave] = incl[i];
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            for (int w = 0; w < wave; ++w) incl[i] += s_wave[i][w];
            s_at[i][tid + 1] = at[i] + incl[i];
            if (tid == 0) s_at[i][0] = at[i];
        }
        __syncthreads();
        const int u0 = s_at[0][0], u1 = s_at[0][kPlanThreads];
        for (int u = u0 + tid; u < min(u1, a.max_units); u += kPlanThreads) {
            int lo = 0, hi = min(kPlanThreads, a.t.n_seq - c * kPlanThreads);  // s_at[0][lo] <= u < s_at[0][lo + 1]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_at[0][mid] <= u) lo = mid;
                else hi = mid;
            }
            const int pieces = max(over_st.up(s_nt[lo]), 1);
            const Over over_pieces(pieces);
            const int start = s_start[lo], S = s_S[lo], b = c * kPlanThreads + lo;
            // The blocks that read the same keys (stream kh * pieces + p) come every eighth, which is the same XCD: its L2
            // then reads them once (hd 512: 16 trees after up to 16384 keys 97 -> 92.5 us a call). Eight streams at a time, the last
            // ones as many as there are.
            const int k = u - s_at[0][lo], nb = (S + a.bq - 1) >> log_bq, streams = pieces * a.n_kv_heads;
            const int group = Over(8 * nb)(k), in = k - group * 8 * nb, wide = min(8, streams - 8 * group);
            const int qb = Over(wide)(in), stream = 8 * group + in - qb * wide;
            const int kh = over_pieces(stream), p = stream - kh * pieces;
            const int nt = tree_tiles(start, S, qb, a.bq, a.kt, a.window);
            // (pieces of ceil(nt / pieces) tiles or one less, so that no product passes 32 bits)
            const int each = over_pieces(nt), more = nt - each * pieces, t0 = p * each + min(p, more);
            PagedUnit w{b, qb, kh, pieces, 0, t0, t0 + each + (p < more ? 1 : 0), s_lo[lo], S, start, {-1, -1, -1, -1}, 0, 0};
            const int key0 = (tree_first(start, a.window) & ~(a.kt - 1)) + w.t0 * a.kt;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // (a group past the table's columns has no rows)
                const int col = (key0 + 16 * i) >> a.t.shift;
                w.page[i] = nt > 0 && col < a.t.cols ? a.rows.table[(size_t)b * a.rows.stride + col] : -1;
                if (a.conv_x) w.page[i] = page_ok(a.rows, w.page[i]) ? b * a.t.cols + col : -1;  // as the conversion names it
            }
            if (pieces > 1) {  // the prices have kept to max_slots
                const int slot0 = s_at[1][lo] + (qb * a.n_kv_heads + kh) * pieces;
                w.slot = slot0;
                if (p == 0) a.merges[s_at[2][lo] + qb * a.n_kv_heads + kh] = w;
                w.slot = slot0 + p;
            }
            a.units[u] = w;
        }
#pragma unroll
        for (int i = 0; i < 3; ++i) at[i] = s_at[i][kPlanThreads];
        __syncthreads();
    }
    if (tid == 0) {
        a.counts[0] = min(at[0], a.max_units);
        a.counts[1] = at[2];
    }
}

// ---------------------------------------------------------------- rows
// Calls f(j, steps from i) for token i of the tree whose parents are `par`, then for its ancestors, nearest first;
// returns its depth. i is wave-uniform and below kTreeMax; every lane of the wave must call it. Up to 64 tokens
// sit in the lanes, more in `lds`, the wave's own kTreeMax words. One step after the other: a call of 253 tokens after 300 keys takes 29 us
// as a star and 49 as a chain, of 1024 55 and 149.
template <typename F>
__device__ __forceinline__ int walk_up(const int32_t* par, int i, int* lds, int lane, F f) {
    int j = i, d = 0;
    if (i < 64) {
        const int mine = lane <= i ? par[lane] : -1;
        while (true) {
            f(j, d);
            const int p = __builtin_amdgcn_readlane(mine, j);
            if ((unsigned)p >= (unsigned)j) return d;
            j = p;
            ++d;
        }
    }
    for (int k = lane; k <= i; k += 64) lds[k] = par[k];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    while (true) {
        f(j, d);
        const int p = __builtin_amdgcn_readfirstlane(lds[j]);
        if ((unsigned)p >= (unsigned)j) return d;
        j = p;
        ++d;
    }
}

// Workgroup 0: the work list. Then a wave per token and four heads: q as paged_prep_kernel makes it, at the token's
// depth, in f16 and what that leaves, and once a token its depth and bits. Then, with new rows, a workgroup per token and kv head: paged_write's row at
// its own place, rotated by its depth, in the cache and in an f32 cache's f16 copies. Then the copies' other rows, which need
// none of that: one launch where rows, copy, q and list took three (3 trees of 253, 123 and 60 after 500 to 5000 keys 10 us a call less).
template <int HD, typename IT, typename CT>
__global__ __launch_bounds__(256) void tree_rows_kernel(TreeRowArgs a) {
    __shared__ int s_par[4][kTreeMax];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int blk = blockIdx.x;
    if (blk == 0) {
        plan_trees(a);
        return;
    }
    const int waves = a.n_tokens * a.q_groups, q_blocks = (waves + 3) / 4;  // (n_tokens * n_q_heads fits 32 bits with room)
    if (blk <= q_blocks) {
        constexpr int E = HD / 64, NH = 4;
        typedef float vec_t __attribute__((ext_vector_type(E)));
        typedef half_t hvec_t __attribute__((ext_vector_type(E)));
        const int w = (blk - 1) * 4 + wave;
        if (w >= waves) return;
        const int tok = w / a.q_groups, h0 = (w - tok * a.q_groups) * NH;
        vec_t x[NH], gv;
        const float* qr = a.q + ((size_t)tok * a.n_q_heads + h0) * HD + E * lane;
#pragma unroll
        for (int i = 0; i < NH; ++i) x[i] = *reinterpret_cast<const vec_t*>(qr + (h0 + i < a.n_q_heads ? i * HD : 0));
        if (a.q_gain) gv = *reinterpret_cast<const vec_t*>(a.q_gain + E * lane);
        const int b = seq_of_row(a.cu, a.t.n_seq, tok);
        if (b >= a.t.n_seq) return;  // a row of nobody
        const SeqRows r = tree_rows(a.t, a.cu, a.n_tokens, b);
        if (!holds(r, tok)) return;  // offsets that do not ascend, or a row behind the tree's last
        const int i0 = tok - r.lo, start = r.keys - (r.hi - r.lo), off = start & 63;
        unsigned long long bits = 0;  // lane k: word k
        const int depth = walk_up(a.parents + r.lo, i0, s_par[wave], lane, [&](int j, int d) {
            if (lane == (off + j) >> 6 && (a.window == 0 || d < a.window)) bits |= 1ull << ((off + j) & 63);
        });
        const int pos = start + depth;
        if (h0 == 0) {
            // the history in the first word: keys start - off .. start - 1 that the window holds
            if (lane == 0) {
                const int from = a.window > 0 ? min(max(pos + 1 - a.window - (start - off), 0), off) : 0;
                bits |= ((1ull << off) - 1) & ~((1ull << from) - 1);
                a.depth[tok] = depth;
            }
            if (lane < a.words) a.bits[(size_t)tok * a.words + lane] = bits;
        }
        const int p = max(pos, 0);
        vec_t c, sn;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            c[e] = 1.0f;
            sn[e] = 0.0f;
        }
        if (a.rcos) {
            c = *reinterpret_cast<const vec_t*>(a.rcos + (size_t)p * (HD / 2) + E * (lane & 31));
            sn = *reinterpret_cast<const vec_t*>(a.rsin + (size_t)p * (HD / 2) + E * (lane & 31));
        }
#pragma unroll
        for (int i = 0; i < NH; ++i) {
            if (a.q_gain) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < E; ++e) ss = __builtin_fmaf(x[i][e], x[i][e], ss);
                const float rs = 1.0f / sqrtf(wave_sum(ss) / (float)HD + a.eps);
#pragma unroll
                for (int e = 0; e < E; ++e) x[i][e] = x[i][e] * rs * gv[e];
            }
            hvec_t hv, lo;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const float2 pr = pair32(x[i][e]);  // (lane < 32: this lane's, its partner's), the same pair in both
                const float y = lane < 32 ? pr.y : pr.x;
                const float z = pin(lane < 32 ? __builtin_fmaf(x[i][e], c[e], -(y * sn[e])) : __builtin_fmaf(x[i][e], c[e], y * sn[e]));
                hv[e] = (half_t)z;
                lo[e] = (half_t)(z - (float)hv[e]);
            }
            if (h0 + i < a.n_q_heads) {
                const size_t at = ((size_t)tok * a.n_q_heads + h0 + i) * HD + E * lane;
                *reinterpret_cast<hvec_t*>(a.q16 + at) = hv;
                *reinterpret_cast<hvec_t*>(a.q16_lo + at) = lo;
            }
        }
        return;
    }
    blk -= 1 + q_blocks;
    const int row_blocks = a.k_new ? a.n_tokens * a.n_kv_heads : 0;
    if (blk >= row_blocks) {
        if constexpr (sizeof(CT) == 4) {
            blk -= row_blocks;  // < conv_x * n_seq * conv_z by the grid
            const int x = blk % a.conv_x, bz = blk / a.conv_x;
            kv16_rows<true>(a.conv, x, bz / a.conv_z, bz % a.conv_z, a.conv_z);
        }
        return;
    }
    // one (token, kv head); every exit is the whole workgroup's
    constexpr int HALF = HD / 2;
    __shared__ float red[2 * (HALF / 64)];
    const int t = threadIdx.x, tok = blk / a.n_kv_heads, kh = blk - tok * a.n_kv_heads;
    const int b = seq_of_row(a.cu, a.rows.n_seq, tok);
    if (b >= a.rows.n_seq) return;
    const SeqRows r = tree_rows(a.rows, a.cu, a.n_tokens, b);
    if (!holds(r, tok)) return;
    const int at = row_position(r, tok);
    if (at < 0) return;
    const int page = page_at(a.rows, b, at);
    if (!page_ok(a.rows, page)) return;
    const size_t row = ((size_t)tok * a.n_kv_heads + kh) * HD;
    const IT* kin = reinterpret_cast<const IT*>(a.k_new) + row;
    const IT* vin = reinterpret_cast<const IT*>(a.v_new) + row;
    float k0 = 0.0f, k1 = 0.0f, v0 = 0.0f, v1 = 0.0f;
    if (t < HALF) {
        k0 = (float)kin[t];
        k1 = (float)kin[t + HALF];
        v0 = (float)vin[t];
        v1 = (float)vin[t + HALF];
    }
    const int depth = walk_up(a.parents + r.lo, tok - r.lo, s_par[wave], lane, [](int, int) {});
    const int p = max(r.keys - (r.hi - r.lo) + depth, 0);
    kv_pair_prep<HD>(k0, k1, v0, v1, a.k_gain, a.rcos ? a.rcos + (size_t)p * HALF : nullptr,
                     a.rsin ? a.rsin + (size_t)p * HALF : nullptr, a.v_norm != 0, a.eps, a.k_in_q, a.v_in_q, red, t);
    if (t >= HALF) return;
    const size_t crow = paged_row(a.rows, page, at, a.n_kv_heads * HD) + (size_t)kh * HD;
    CT* kc = reinterpret_cast<CT*>(a.k_pages) + crow;
    CT* vc = reinterpret_cast<CT*>(a.v_pages) + crow;
    store_elem(kc + t, k0);
    store_elem(kc + t + HALF, k1);
    store_elem(vc + t, v0);
    store_elem(vc + t + HALF, v1);
    if constexpr (sizeof(CT) == 4) {
        const size_t copy = paged_row(a.rows, b * a.t.cols + (at >> a.rows.shift), at, a.n_kv_heads * HD) + (size_t)kh * HD;
        a.conv.ko[copy + t] = (half_t)k0;
        a.conv.ko[copy + t + HALF] = (half_t)k1;
        a.conv.klo[copy + t] = rest16(k0);
        a.conv.klo[copy + t + HALF] = rest16(k1);
        a.conv.vo[copy + t] = (half_t)v0;
        a.conv.vo[copy + t + HALF] = (half_t)v1;
    }
}

// ---------------------------------------------------------------- merge
// out = sum_p o_p l_p 2^(m_p - M) / sum_p l_p 2^(m_p - M), M = max_p m_p, of a block's pieces (o_p = O_p / l_p). A
// workgroup's item is a wave's block of 32 columns x 256 dims of an entry of the merge list, and of its 16 runs of 8 values
// x 64 lanes one, so that many workgroups share the bytes (four runs an item: 8 trees of 16 after 2000 keys 29 -> 35 us a
// call, 64 after 3000 111 -> 116). Its four waves take every fourth piece, each relative to its own largest m so far, and
// join through LDS: one trip to memory for up to 16 pieces.
constexpr int kMergeGrid = 2048;
template <typename OUTT, int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(PagedTreeArgs a) {
    constexpr int NCOL = tree_columns(HD), NV = NCOL * HD, BLK = NV * 3;  // values and bytes of a piece's block
    constexpr int NW = 4;                                                 // waves' blocks
    __shared__ float s_o[4][8][64], s_l[4][64], s_m[4][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int merges = a.counts[1], G = a.n_q_heads / a.n_kv_heads, BQ = NCOL / G;
    for (int item = blockIdx.x; item < merges * NW * 16; item += gridDim.x) {
        const PagedUnit pu = a.merges[item / (NW * 16)];
        const int w = item / 16 % NW, k = item % 16, qb = pu.qb, kh = pu.kh, n_pieces = pu.n_pieces, w32 = HD == 256 ? w : w & 1;
        if (qb * BQ + 32 * w32 / G >= pu.S) continue;  // no token in these 32 columns
        const int c = 32 * w32 + (lane & 31), s_idx = qb * BQ + c / G;
        const bool ok = s_idx < pu.S;
        const float2* ml = a.part_ml + (size_t)pu.slot * NCOL + c;
        const char* base = reinterpret_cast<const char*>(a.part_o) + (size_t)pu.slot * BLK;
        float o[8] = {}, L = 0.0f, M = kNegInf;
        const int run = w * (32 * 256) + k * 512 + 8 * lane;
        for (int p0 = wave; p0 < n_pieces; p0 += 16) {
            float2 mp[4];
            v4u32 hi[4];
            v2u32 lo[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int p = p0 + 4 * e;
                mp[e] = make_float2(kNegInf, 0.0f);
                hi[e] = v4u32{0, 0, 0, 0};
                lo[e] = v2u32{0, 0};
                if (ok && p < n_pieces) {
                    mp[e] = ml[(size_t)p * NCOL];
                    hi[e] = *reinterpret_cast<const v4u32*>(base + (size_t)p * BLK + 2 * run);
                    lo[e] = *reinterpret_cast<const v2u32*>(base + (size_t)p * BLK + 2 * NV + run);
                }
            }
            const float top = fmaxf(M, fmaxf(fmaxf(mp[0].x, mp[1].x), fmaxf(mp[2].x, mp[3].x)));
            const float back = M == kNegInf ? 0.0f : fexp2(M - top);
            M = top;
            L *= back;
#pragma unroll
            for (int i = 0; i < 8; ++i) o[i] *= back;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                // a piece with no attended key (l = 0) counts for nothing, whatever it holds; one of NaN scores alone
                // (l NaN, m -inf) makes all NaN
                const bool none = mp[e].y == 0.0f;
                const float wt = none ? 0.0f : mp[e].y * fexp2(mp[e].x - M);
                L += wt;
#pragma unroll
                for (int i = 0; i < 8; ++i) o[i] = __builtin_fmaf(none ? 0.0f : unpack24(hi[e], lo[e], i), wt, o[i]);
            }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s_o[wave][e][lane] = o[e];
        s_l[wave][lane] = L;
        s_m[wave][lane] = M;
        __syncthreads();
        // wave w finishes values 2w and 2w + 1 of each run
        if (ok) {
            M = fmaxf(fmaxf(s_m[0][lane], s_m[1][lane]), fmaxf(s_m[2][lane], s_m[3][lane]));
            float x = 0.0f, y = 0.0f;
            L = 0.0f;
#pragma unroll
            for (int v = 0; v < 4; ++v) {
                const float l = s_l[v][lane], f = l == 0.0f ? 0.0f : fexp2(s_m[v][lane] - M);
                L += l * f;
                x = __builtin_fmaf(l == 0.0f ? 0.0f : s_o[v][2 * wave][lane], f, x);
                y = __builtin_fmaf(l == 0.0f ? 0.0f : s_o[v][2 * wave + 1][lane], f, y);
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            OUTT* orow = reinterpret_cast<OUTT*>(a.out) + ((size_t)(pu.row0 + s_idx) * a.n_q_heads + kh * G + c % G) * HD +
                         (HD == 256 ? 0 : 256 * (w >> 1));
            // run k: dims tile k/2, 4-row pair k%2
            OUTT* to = orow + 32 * (k >> 1) + 16 * (k & 1) + 8 * (wave >> 1) + 4 * h + 2 * (wave & 1);
            store_elem(to, srq(x * inv, a.out_q));
            store_elem(to + 1, srq(y * inv, a.out_q));
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- host side
typedef void (*tree_fn)(PagedTreeArgs);
typedef void (*tree_rows_fn)(TreeRowArgs);

template <int G, int HD, bool K32>
static tree_fn pick_out(bool out32) {
    return out32 ? paged_kernel_w256<G, float, PagedTreeArgs, HD, K32> : paged_kernel_w256<G, half_t, PagedTreeArgs, HD, K32>;
}
template <int G>
static tree_fn pick_form(int HD, bool kv32, bool out32) {
    if (HD == 256) return kv32 ? pick_out<G, 256, true>(out32) : pick_out<G, 256, false>(out32);
    return kv32 ? pick_out<G, 512, true>(out32) : pick_out<G, 512, false>(out32);
}
static tree_fn pick_units(int HD, int G, bool kv32, bool out32) {  // G: 1, 2, 4 or 8 (check_cfg)
    switch (G) {
        case 1: return pick_form<1>(HD, kv32, out32);
        case 2: return pick_form<2>(HD, kv32, out32);
        case 4: return pick_form<4>(HD, kv32, out32);
        default: return pick_form<8>(HD, kv32, out32);
    }
}
static tree_fn pick_merge(int HD, bool out32) {
    if (HD == 256) return out32 ? tree_merge_kernel<float, 256> : tree_merge_kernel<half_t, 256>;
    return out32 ? tree_merge_kernel<float, 512> : tree_merge_kernel<half_t, 512>;
}
template <int HD>
static tree_rows_fn pick_rows(bool in16, bool c32) {
    if (in16) return c32 ? tree_rows_kernel<HD, half_t, float> : tree_rows_kernel<HD, half_t, half_t>;
    return c32 ? tree_rows_kernel<HD, float, float> : tree_rows_kernel<HD, float, half_t>;
}

// What the host can bound, and the workspace [counts][units][merges][depth][bits][q16][its remainders][partials][(m, l)][K16][its
// remainders][V16][table16].
// Every part grows with n_tokens, n_seq and max_key_len, so that one reserved for the largest call holds all.
struct TreePlan {
    int bq, kt, max_units, max_slots, words, cols16;
    size_t units, merges, depth, bits, q16, q16_lo, part_o, part_ml, k16, k16_lo, v16, tab16, total;
};
static bool tree_plan(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens, TreePlan& p) {
    const int HD = (int)cfg->head_dim, G = (int)(cfg->n_q_heads / cfg->n_kv_heads);
    const int64_t kvh = cfg->n_kv_heads;
    p.bq = tree_columns(HD) / G;
    p.kt = HD == 256 ? 64 : 32;
    p.words = tree_words(n_tokens);
    const int64_t blocks = std::min<int64_t>(n_tokens, (int64_t)n_tokens / p.bq + pg->n_seq);
    const int64_t keys = pg->max_key_len;
    const int64_t most = std::min<int64_t>((keys + p.kt - 1) / p.kt + 1, kTreePieces);  // pieces of a block
    const int slots = (int)std::min<int64_t>(blocks * kvh * most, kTreeSlots);
    p.max_slots = slots;
    const int64_t units = blocks * kvh + slots;
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    size_t at = 256;
    auto part = [&](size_t bytes) {
        const size_t x = at;
        at += al(bytes);
        return x;
    };
    p.max_units = (int)units;
    p.units = part((size_t)units * sizeof(PagedUnit));
    p.merges = part((size_t)slots * sizeof(PagedUnit));
    p.depth = part((size_t)n_tokens * sizeof(int32_t));
    p.bits = part((size_t)n_tokens * p.words * sizeof(unsigned long long));
    p.q16 = part((size_t)n_tokens * cfg->n_q_heads * HD * sizeof(half_t));
    p.q16_lo = part((size_t)n_tokens * cfg->n_q_heads * HD * sizeof(half_t));
    p.part_o = part((size_t)slots * tree_columns(HD) * HD * 3);
    p.part_ml = part((size_t)slots * tree_columns(HD) * sizeof(float2));
    p.k16 = p.k16_lo = p.v16 = p.tab16 = at;
    p.cols16 = 0;
    int64_t pages16 = 0;
    if (cfg->flags & G4A_KV_F32) {
        p.cols16 = (pg->max_key_len + pg->page_size - 1) / pg->page_size;
        pages16 = (int64_t)pg->n_seq * p.cols16;
        const size_t pool = (size_t)pages16 * pg->page_size * kvh * HD * sizeof(half_t);
        p.k16 = part(pool);
        p.k16_lo = part(pool);
        p.v16 = part(pool);
        p.tab16 = part((size_t)pages16 * sizeof(int32_t));
    }
    p.total = at;
    if (units > 0x7fffffff || pages16 > 0x7fffffff || (int64_t)n_tokens * (cfg->n_q_heads + kvh) > 0x7fffffff - 64) {
        set_error("n_tokens * heads or n_seq * max_key_len too large");
        return false;
    }
    return true;
}

}  // namespace g4a

using namespace g4a;

extern "C" size_t g4a_paged_tree_ws_bytes(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens) {
    if (check_paged(cfg, pg, true) || check_tokens(cfg, n_tokens, pg->key_len)) return 0;
    TreePlan p;
    return tree_plan(cfg, pg, n_tokens, p) ? p.total : 0;
}

extern "C" int g4a_paged_tree(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens, const int32_t* cu_q,
                              const int32_t* parents, const float* q, const float* q_gain, const float* rope_cos,
                              const float* rope_sin, const void* k_new, const void* v_new, float k_in_q, float v_in_q,
                              const float* k_gain, void* out, void* ws, size_t ws_bytes, void* stream_) {
    if (const int rc = check_paged(cfg, pg, true)) return rc;
    if (const int rc = check_tokens(cfg, n_tokens, cu_q)) return rc;
    if (const int rc = check_paged_call(cfg, n_tokens, q, q_gain, rope_cos, rope_sin, out)) return rc;
    if (const int rc = check_steps(k_in_q, v_in_q)) return rc;
    if (!parents || (uintptr_t)parents % 4) {
        set_error("parents must be non-NULL and 4-byte aligned");
        return G4A_EINVAL;
    }
    if ((k_new == nullptr) != (v_new == nullptr)) {
        set_error("k_new and v_new must both be given or both be NULL");
        return G4A_EINVAL;
    }
    if ((uintptr_t)k_new % 16 || (uintptr_t)v_new % 16 || (uintptr_t)k_gain % 16) {
        set_error("k_new, v_new and k_gain must be 16-byte aligned");
        return G4A_EINVAL;
    }
    if (cfg->flags & G4A_Q_HILO) {
        set_error("g4a_paged_tree holds q at f32 accuracy by itself (G4A_Q_HILO not supported)");
        return G4A_EUNSUPPORTED;
    }
    const int HD = (int)cfg->head_dim, G = (int)(cfg->n_q_heads / cfg->n_kv_heads);
    TreePlan p;
    if (!tree_plan(cfg, pg, n_tokens, p)) return G4A_EINVAL;
    if (!ws || (uintptr_t)ws % 256 || ws_bytes < p.total) {
        set_error("paged tree workspace needs %zu bytes (256-byte aligned), got %zu", p.total, ws ? ws_bytes : (size_t)0);
        return G4A_EWORKSPACE;
    }
    const hipStream_t stream = (hipStream_t)stream_;
    char* w = (char*)ws;
    TreeRowArgs a;
    a.t = a.rows = page_tab(pg);
    a.cu = cu_q;
    a.q = q;
    a.q_gain = q_gain;
    a.rcos = rope_cos;
    a.rsin = rope_sin;
    a.kc = a.k_pages = pg->k_pages;
    a.vc = a.v_pages = pg->v_pages;
    a.out = out;
    a.q16 = (half_t*)(w + p.q16);
    a.units = (PagedUnit*)(w + p.units);
    a.merges = (PagedUnit*)(w + p.merges);
    a.counts = (int*)w;
    a.part_o = w + p.part_o;
    a.part_ml = (float2*)(w + p.part_ml);
    a.n_tokens = n_tokens;
    a.n_q_heads = (int)cfg->n_q_heads;
    a.n_kv_heads = (int)cfg->n_kv_heads;
    a.window = (int)cfg->window;
    a.max_units = p.max_units;
    a.max_slots = p.max_slots;
    a.bq = p.bq;
    a.kt = p.kt;
    a.scale_log2 = cfg->scale * kLog2e;
    a.eps = cfg->eps;
    a.out_q = cfg->out_q;
    a.parents = parents;
    a.bits = (unsigned long long*)(w + p.bits);
    a.depth = (int32_t*)(w + p.depth);
    a.q16_lo = (half_t*)(w + p.q16_lo);
    a.kc_lo = nullptr;
    a.words = p.words;
    a.k_new = k_new;
    a.v_new = v_new;
    a.k_gain = k_gain;
    a.v_norm = (cfg->flags & G4A_NO_V_NORM) ? 0 : 1;
    a.k_in_q = k_in_q;
    a.v_in_q = v_in_q;
    a.q_groups = (a.n_q_heads + 3) / 4;
    const bool kv32 = (cfg->flags & G4A_KV_F32) != 0, in16 = (cfg->flags & G4A_IN_F16) != 0;
    const tree_rows_fn rows = HD == 256 ? pick_rows<256>(in16, kv32) : pick_rows<512>(in16, kv32);
    int64_t blocks = 1 + ((int64_t)n_tokens * a.q_groups + 3) / 4 + (k_new ? (int64_t)n_tokens * a.n_kv_heads : 0);
    hipError_t e;
    a.conv = PagedKv16Args{};
    a.conv_x = a.conv_z = 0;
    if (kv32) {
        PagedKv16Args& k = a.conv;
        k.t = a.rows;
        k.cu = cu_q;
        k.kc = (const float*)pg->k_pages;
        k.vc = (const float*)pg->v_pages;
        k.ko = (half_t*)(w + p.k16);
        k.vo = (half_t*)(w + p.v16);
        k.klo = (half_t*)(w + p.k16_lo);
        k.tab = (int32_t*)(w + p.tab16);
        k.n_tokens = n_tokens;
        k.row = a.n_kv_heads * HD;
        k.cols = p.cols16;
        k.window = a.window;
        k.rows_given = k_new != nullptr;
        a.conv_x = (pg->max_key_len + 15) / 16;
        a.conv_z = (k.row + 511) / 512;
        blocks += (int64_t)a.conv_x * pg->n_seq * a.conv_z;
        // the units read the f16 copy by its own table
        a.kc = w + p.k16;
        a.kc_lo = w + p.k16_lo;
        a.vc = w + p.v16;
        a.t.table = (const int32_t*)(w + p.tab16);
        a.t.cols = a.t.stride = p.cols16;
        a.t.n_pages = pg->n_seq * p.cols16;
    }
    if (blocks > 0x7fffffff) {
        set_error("n_tokens or n_seq * max_key_len too large");
        return G4A_EINVAL;
    }
    hipLaunchKernelGGL(rows, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged tree preparation launch");
    const bool out32 = (cfg->flags & G4A_OUT_F32) != 0;
    const PagedTreeArgs& t = a;
    hipLaunchKernelGGL(pick_units(HD, G, kv32, out32), dim3((unsigned)p.max_units), dim3(256), 0, stream, t);
    if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged tree launch");
    // a block of the merge list has two slots at least
    const int items = p.max_slots / 2 * 4 * 16;
    hipLaunchKernelGGL(pick_merge(HD, out32), dim3((unsigned)std::max(std::min(items, kMergeGrid), 1)), dim3(256), 0, stream, t);
    if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged tree merge launch");
    return G4A_OK;
}
