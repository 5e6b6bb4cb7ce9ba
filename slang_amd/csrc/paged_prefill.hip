// Causal attention of packed prompts over a paged K/V cache, for gfx950 on f16 MFMA.
//
// The mathematics is prefill.hip's: per query column an online softmax over key tiles, scores formed
// transposed (S^T = K . Q^T), so that they are the B operand of O^T += V^T . P^T, all sums in f32. q and P
// are rounded to f16, and f32 caches too, because the matrix units take f16 operands at 16 times
// the rate of f32 ones: half a step (2^-11) of a query, key, weight or value, which puts outputs 4 to 5e-4 of
// the largest off where 32-bit products with an f16 output are 2e-4 off. Partials of split blocks keep 24
// bits, half a step of which is 2^-16, and move three quarters of the bytes. What differs from prefill.hip is what
// a server's batch brings:
//   * Lengths are device data, so nothing can be planned on the host. One launch prepares q in f16 and,
//     in its first workgroup, writes the work list: a unit is a query block (128 columns: the G heads
//     of a kv head x 128/G positions) of one sequence and kv head, or a piece of its keys. A list
//     sorted by length, longest first, keeps ragged prompts from leaving one long block running alone
//     at the end; blocks longer than what a CU gets on average are cut into up to kMaxPieces pieces
//     whose partials the merge kernel joins.
//   * K/V rows come through the page table. Tiles start at a multiple of 16 keys, so 16 rows of a tile
//     lie in one page; each wave moves rows of one such group and holds the table entries of 64 tiles
//     in its lanes, one readlane a tile. Rows outside [first attended, last] and pages that are not there
//     read as zeros through the buffer range, whatever memory holds; their scores are masked.
// f32 caches are first converted to f16 pages in the workspace (the rounding of prefill.hip's form
// without G4A_Q_HILO), with a table of their own.
#include <algorithm>
#include <type_traits>

#include "paged.hpp"
#include "prefill_tiles.hpp"

namespace g4a {

constexpr int kMaxPieces = 8;  // pieces a query block is cut into
constexpr int kMaxSlots = 768; // pieces with partials in a call
// P, rounded to f16 for its product, is at most 2^kMaxLag. A maximum that moves is set this many powers of two
// below the score, so that a key keeps all bits down to 2^-18 of the largest weight and is zero only below
// 2^-29 (2^-14 and 2^-25 without, while the sum still counts it: 32768 such keys are 2^-10 of it), and it moves
// again when a score passes the largest so far by 2^11. Each move rescales O^T: 0 / 2 / 4 / 8 powers took
// prefill_hd512 824 / 831 / 840 / 900 us, prefill_mixed 128 / 128 / 128 / 135.
constexpr float kPagedLift = 4.0f;
constexpr int kCus = 256;      // compute units of the MI355X; the kernels run one workgroup a CU

struct PagedUnit {
    int b, qb, kh, n_pieces;   // sequence, query block, kv head; pieces of the block
    int slot, t0, t1, row0;    // partial block of this piece (merge list: of the first); key tiles; packed row of the
    int S, start;              // sequence's first token, its tokens in this call, the position of the first
    int page[4];               // table entries of the first tile's 16-row groups
    int pad0, pad1;
};

struct PagedPrefillArgs {
    PageTab t;
    const int32_t* cu;
    const float* q;
    const float* q_gain;
    const float* rcos;
    const float* rsin;
    const void* kc;  // f16 pages
    const void* vc;
    void* out;
    half_t* q16;
    PagedUnit* units;
    PagedUnit* merges;
    int* counts;  // units, merges
    void* part_o;
    float2* part_ml;
    int n_tokens, n_q_heads, n_kv_heads, window, max_units, max_slots, bq, kt;
    float scale_log2, eps, out_q;
};

// ---------------------------------------------------------------- the work list
__device__ __forceinline__ int block_tiles(const PagedPrefillArgs& a, int start, int S, int qb) {
    return key_tiles(start, S, qb, a.bq, a.kt, a.window);
}

// Cost of the units, in key tiles: a unit's own beside its tiles (q, epilogue), a partial's store and
// merge (its 3 bytes a value go to memory and back at a CU's share of the bandwidth, 20 GB/s), and
// the merge launch, set when a tile took about 1.9 us at hd 256 and 2.4 us at hd 512. At hd 256 a unit takes
// 9 us beside its tiles, half of it while others run: a price of 4.8 for 2.4 moves calls by -2.5 to +2.5 % (16
// sequences of 64 tokens over 0 to 15000 keys 118.3 -> 115.3 us, 6 prompts of 300 27.7 -> 28.4, the cases +-0).
struct PlanCost {
    float unit, part, merge;
};
__host__ __device__ inline PlanCost plan_cost(int kt) { return kt == 64 ? PlanCost{2.4f, 4.6f, 2.0f} : PlanCost{4.0f, 7.5f, 2.0f}; }

constexpr int kPlanThreads = 256;
constexpr int kBins = 64;  // size classes of the sorted list

// How the units of one candidate split would end: sums over a lane's sequences, whose blocks' tiles run
// linearly from u to v over m blocks.
struct SplitSums {
    float units = 0.0f, slots = 0.0f, over[4] = {};  // over: pieces of at least (4 - i)/4 of the longest
};
__device__ __forceinline__ float ramp_over(float v, float m, float slope, float x) {  // blocks of more than x tiles
    return v <= x ? 0.0f : m * fminf((v - x) * slope, 1.0f);
}
__device__ __forceinline__ void ramp_sums(SplitSums& t, float u, float v, float m, float st) {
    const float slope = __builtin_amdgcn_rcpf(fmaxf(v - u, 1.0f));
    float units = m, c1 = 0.0f;
#pragma unroll
    for (int j = 1; j < kMaxPieces; ++j) {
        const float c = ramp_over(v, m, slope, st * (float)j);
        if (j == 1) c1 = c;
        units += c;
    }
    const float slots = units - m + c1;
    t.units += units;
    t.slots += slots;
    // pieces of cut blocks count as longest (they hold half of st at least)
#pragma unroll
    for (int i = 0; i < 4; ++i) t.over[i] += slots + fmaxf(ramp_over(v, m, slope, st * (float)(4 - i) * 0.25f - 0.5f) - c1, 0.0f);
}

// Written by one workgroup of kPlanThreads threads.
// How many pieces: st, the most tiles a piece may have, is longest / 1 .. longest / kMaxPieces. Units
// dealt longest first to kCus CUs end, to a good approximation, at the larger of the mean load and, for
// any c, ceil(c / kCus) units of the size of the c-th longest; the st with the lowest such cost is
// taken, from each sequence's block sizes as two linear ramps (first block to middle to last).
// The list: size classes from the longest. (Dealing the blocks that read the same K/V to one XCD was
// tried: L2 hits stayed at 80-85 %, the kernels' times within 3 %.)
__device__ void plan_units(const PagedPrefillArgs& a) {
    __shared__ int s_lo[kPlanThreads], s_S[kPlanThreads], s_start[kPlanThreads], s_blk[kPlanThreads + 1];
    __shared__ int s_wave[kPlanThreads / 64], s_max, s_cut, s_bin[kBins], s_slot, s_merge;
    __shared__ float s_blocks;
    __shared__ float s_sum[kMaxPieces + 1][7];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int chunks = (a.t.n_seq + kPlanThreads - 1) / kPlanThreads;
    if (tid < kBins) s_bin[tid] = 0;
    if (tid == 0) {
        s_max = s_cut = s_slot = s_merge = 0;
        s_blocks = 0.0f;
    }

    // the sequences c * kPlanThreads .. into LDS, with the prefix sum of their query blocks
    auto load_chunk = [&](int c) {
        __syncthreads();
        const int b = c * kPlanThreads + tid;
        SeqRows r{0, 0, 0};
        if (b < a.t.n_seq) r = seq_rows(a.t, a.cu, a.n_tokens, b);
        const int S = r.hi - r.lo, nb = (S + a.bq - 1) / a.bq;
        s_lo[tid] = r.lo;
        s_S[tid] = S;
        s_start[tid] = r.keys - S;
        const int incl = wave_scan(nb);
        if (lane == 63) s_wave[wave] = incl;
        __syncthreads();
        int base = 0;
        for (int w = 0; w < wave; ++w) base += s_wave[w];
        s_blk[tid + 1] = base + incl;
        if (tid == 0) s_blk[0] = 0;
        __syncthreads();
    };
    // f(sequence of the chunk, its index there, query block, its tiles, i, n) for every block, by n lanes in a
    // row (i = 0 .. n - 1), the largest n = 2^0 .. 2^log_most for which there are threads
    auto for_blocks = [&](int log_most, auto f) {
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) load_chunk(c);
            const int blocks = s_blk[kPlanThreads];
            int sh = log_most;
            while (sh > 0 && blocks > kPlanThreads >> sh) --sh;
            for (int js = tid; js < blocks << sh; js += kPlanThreads) {
                const int j = js >> sh;
                int lo = 0, hi = min(kPlanThreads, a.t.n_seq);  // s_blk[lo] <= j < s_blk[hi]
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s_blk[mid] <= j) lo = mid;
                    else hi = mid;
                }
                f(c * kPlanThreads + lo, lo, j - s_blk[lo], block_tiles(a, s_start[lo], s_S[lo], j - s_blk[lo]), js & ((1 << sh) - 1), 1 << sh);
            }
        }
    };
    load_chunk(0);

    // the longest block: tiles do not fall along a sequence, but for a short last block
    for (int c = 0; c < chunks; ++c) {
        if (chunks > 1) load_chunk(c);
        const int nb = s_blk[tid + 1] - s_blk[tid];
        int mx = 0;
        if (nb > 0) mx = block_tiles(a, s_start[tid], s_S[tid], nb - 1);
        if (nb > 1) mx = max(mx, block_tiles(a, s_start[tid], s_S[tid], nb - 2));
        mx = (int)wave_max((float)mx);
        const float blocks = wave_sum((float)((s_S[tid] + a.bq - 1) / a.bq));
        if (lane == 0) {
            atomicMax(&s_max, mx);
            atomicAdd(&s_blocks, blocks);
        }
    }
    __syncthreads();
    // Ascending offsets make no more blocks than this. Others can list the packed rows once a sequence, more
    // than the sums below can count: no block runs then
    if (s_blocks > 1.01f * ((float)a.n_tokens / (float)a.bq + (float)a.t.n_seq) + 64.0f) {
        if (tid == 0) a.counts[0] = a.counts[1] = 0;
        return;
    }
    const int longest = tiles_at_least(s_max);
    const int st_min = a.kt == 64 ? 2 : 4;  // tiles a piece at least
    const auto cut = [&](int k) { return max((longest + k - 1) / k, k == 1 ? 1 : st_min); };
    int st = cut(1);
    if (a.max_slots > 0 && longest > st_min) {  // workgroup-uniform
        // wave w takes candidates w + 1, w + 5, .., a sequence a lane
        SplitSums t[2];
        float tiles = 0.0f;
        static_assert(kMaxPieces == 2 * (kPlanThreads / 64), "two candidates a wave");
        for (int c = 0; c < chunks; ++c) {
            if (chunks > 1) load_chunk(c);
            for (int i = lane; i < min(kPlanThreads, a.t.n_seq - c * kPlanThreads); i += 64) {
                const int nb = s_blk[i + 1] - s_blk[i];
                if (nb == 0) continue;
                const int S = s_S[i], start = s_start[i];
                const float n0 = (float)block_tiles(a, start, S, 0), n1 = (float)block_tiles(a, start, S, nb / 2);
                const float n2 = (float)block_tiles(a, start, S, nb > 1 ? nb - 2 : 0), m1 = (float)(nb / 2), m2 = (float)(nb - nb / 2);
                tiles += 0.5f * ((n0 + n1) * m1 + (n1 + n2) * m2);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    ramp_sums(t[q], n0, n1, m1, (float)cut(wave + 1 + 4 * q));
                    ramp_sums(t[q], n1, n2, m2, (float)cut(wave + 1 + 4 * q));
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const float v[7] = {wave_sum(t[q].units), wave_sum(t[q].slots), wave_sum(t[q].over[0]), wave_sum(t[q].over[1]),
                                wave_sum(t[q].over[2]), wave_sum(t[q].over[3]), wave_sum(tiles)};
            if (lane == 0)
#pragma unroll
                for (int i = 0; i < 7; ++i) s_sum[wave + 1 + 4 * q][i] = v[i];
        }
        __syncthreads();
        // lane k of every wave prices candidate k
        const PlanCost pc = plan_cost(a.kt);
        float cost = __builtin_huge_valf();
        if (lane >= 1 && lane <= kMaxPieces) {
            float v[7];
#pragma unroll
            for (int i = 0; i < 7; ++i) {
                v[i] = s_sum[lane][i] * (float)a.n_kv_heads;
            }
            const float stk = (float)cut(lane), part = v[1] > 0.5f ? pc.part : 0.0f;
            cost = (v[6] + v[0] * pc.unit + v[1] * pc.part) * (1.0f / kCus);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (v[2 + i] >= 0.5f) cost = fmaxf(cost, ceilf(v[2 + i] * (1.0f / kCus)) * (stk * (float)(4 - i) * 0.25f + pc.unit + part));
            if (v[1] > 0.5f) cost += pc.merge;
            if (v[1] > (float)a.max_slots) cost = __builtin_huge_valf();
        }
        const float best = -wave_max(-cost);
        const unsigned long long m = __ballot(cost == best && lane >= 1 && lane <= kMaxPieces);
        if (m) st = cut(__builtin_ctzll(m));
    }
    const auto pieces = [&](int nt) { return min(max(1, (nt + st - 1) / st), kMaxPieces); };
    // class 0: the longest pieces
    const auto bin_of = [&](int nt, int np) { return kBins - 1 - min((nt + np - 1) / np * (kBins - 1) / st, kBins - 1); };
    for (int round = 0; round < 2; ++round) {
        for_blocks(0, [&](int, int, int, int nt, int, int) {
            const int np = pieces(nt);
            atomicAdd(&s_bin[bin_of(nt, np)], np * a.n_kv_heads);
            if (np > 1) atomicAdd(&s_cut, np * a.n_kv_heads);
        });
        __syncthreads();
        if (s_cut <= a.max_slots) break;
        // the ramps missed: more pieces than there is room for their partials, so none at all
        __syncthreads();
        st = max(longest, 1);
        if (tid < kBins) s_bin[tid] = 0;
        if (tid == 0) s_cut = 0;
        __syncthreads();
    }
    if (wave == 0) {  // first unit of each class
        const int n = s_bin[lane], incl = wave_scan(n);
        s_bin[lane] = incl - n;
        if (lane == 63) a.counts[0] = min(incl, a.max_units);
    }
    __syncthreads();
    // (a lane waits for the table entries of one piece after the other, so few blocks' pieces go to lanes of
    // their own: 2 tokens over 595 keys, 8 kv heads 11.4 -> 7.8 us, 6 prompts without a cut 7.0 -> 7.3)
    static_assert(kMaxPieces == 8);
    for_blocks(3, [&](int b, int s, int qb, int nt, int lane0, int lanes) {
        const int np = pieces(nt);
        int at = 0, slot = 0, mg = 0;
        if (lane0 == 0) {
            at = atomicAdd(&s_bin[bin_of(nt, np)], np * a.n_kv_heads);
            if (np > 1) {
                slot = atomicAdd(&s_slot, np * a.n_kv_heads);
                mg = atomicAdd(&s_merge, a.n_kv_heads);
            }
        }
        if (lanes > 1) {
            at = __shfl(at, lane - lane0);
            slot = __shfl(slot, lane - lane0);
            mg = __shfl(mg, lane - lane0);
        }
        PagedUnit u{b, qb, 0, np, 0, 0, 0, s_lo[s], s_S[s], s_start[s], {-1, -1, -1, -1}, 0, 0};
        const int p0 = s_start[s] + qb * a.bq, key0 = a.window > 0 ? max(0, p0 + 1 - a.window) & ~15 : 0;
        for (int p = lane0; p < np; p += lanes) {
            u.t0 = (p * nt + np - 1) / np;
            u.t1 = ((p + 1) * nt + np - 1) / np;
#pragma unroll
            for (int i = 0; i < 4; ++i) {  // (a group past the table's columns has no rows)
                const int col = (key0 + u.t0 * a.kt + 16 * i) >> a.t.shift;
                u.page[i] = nt > 0 && col < a.t.cols ? a.t.table[(size_t)b * a.t.stride + col] : -1;
            }
            for (int kh = 0; kh < a.n_kv_heads; ++kh) {
                u.kh = kh;
                u.slot = slot + kh * np + p;
                const int i = at + kh * np + p;
                // (offsets out of order could list more blocks than there are packed rows: cut to the room)
                if (i < a.max_units) a.units[i] = u;
                if (np > 1 && p == 0) a.merges[mg + kh] = u;
            }
        }
    });
    __syncthreads();
    if (tid == 0) a.counts[1] = s_merge;
}

// q of packed rows to f16: RMSNorm * gain, then RoPE at the row's position (qprep_row512_kernel's
// arithmetic). A wave takes four heads of a token; lane l holds dims E l .. E l + E - 1, whose RoPE
// partners sit in lane l ^ 32. The first workgroup writes the work list meanwhile (about 7 us, what a call of few
// tokens waits for). Many tokens: the bytes (15252 of 8 x 256, 187 MB: 36 us = 5.2 TB/s, a copy's rate).
template <int HD>
__global__ __launch_bounds__(256) void paged_prep_kernel(PagedPrefillArgs a) {
    if (blockIdx.x == 0) {
        plan_units(a);
        return;
    }
    constexpr int E = HD / 64, NH = 4;
    typedef float vec_t __attribute__((ext_vector_type(E)));
    typedef half_t hvec_t __attribute__((ext_vector_type(E)));
    const int lane = threadIdx.x & 63, hg = (a.n_q_heads + NH - 1) / NH;
    const int w = ((int)blockIdx.x - 1) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int tok = w / hg, h0 = (w - tok * hg) * NH;
    if (tok >= a.n_tokens) return;
    vec_t x[NH], gv;
    const float* qr = a.q + ((size_t)tok * a.n_q_heads + h0) * HD + E * lane;
#pragma unroll
    for (int i = 0; i < NH; ++i) x[i] = *reinterpret_cast<const vec_t*>(qr + (h0 + i < a.n_q_heads ? i * HD : 0));
    if (a.q_gain) gv = *reinterpret_cast<const vec_t*>(a.q_gain + E * lane);
    const int b = seq_of_row(a.cu, a.t.n_seq, tok);
    if (b >= a.t.n_seq) return;  // a row of nobody
    const SeqRows r = seq_rows(a.t, a.cu, a.n_tokens, b);
    if (!holds(r, tok)) return;  // offsets that do not ascend
    const int p = max(row_position(r, tok), 0);
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
        hvec_t hv;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float2 pr = pair32(x[i][e]);  // (lane < 32: this lane's, its partner's), the same pair in both
            const float y = lane < 32 ? pr.y : pr.x;
            hv[e] = (half_t)pin(lane < 32 ? __builtin_fmaf(x[i][e], c[e], -(y * sn[e])) : __builtin_fmaf(x[i][e], c[e], y * sn[e]));
        }
        if (h0 + i < a.n_q_heads)
            __builtin_nontemporal_store(hv, reinterpret_cast<hvec_t*>(a.q16 + ((size_t)tok * a.n_q_heads + h0 + i) * HD + E * lane));
    }
}

// The rows of f32 pages that the call attends, as f16 pages of the workspace: page i of sequence b is
// page b * cols + i of ko / vo, and the table written to tab names it if the cache's own is there.
struct PagedKv16Args {
    PageTab t;
    const int32_t* cu;
    const float* kc;
    const float* vc;
    half_t* ko;
    half_t* vo;
    int32_t* tab;
    int n_tokens, row, cols, window;
};
__global__ __launch_bounds__(256) void paged_kv16_kernel(PagedKv16Args a) {
    const int b = blockIdx.y, k0 = 16 * blockIdx.x, ps = 1 << a.t.shift;
    const SeqRows r = seq_rows(a.t, a.cu, a.n_tokens, b);
    const int page = k0 >> a.t.shift;
    if (page >= a.cols) return;
    const int first = a.window > 0 ? max(0, r.keys - (r.hi - r.lo) + 1 - a.window) & ~15 : 0;
    const bool used = k0 < r.keys && r.hi > r.lo && (page + 1) << a.t.shift > first;
    const int from = used ? page_at(a.t, b, k0) : -1;
    const bool ok = page_ok(a.t, from);
    const int to = b * a.cols + page;
    if ((k0 & (ps - 1)) == 0 && threadIdx.x == 0 && blockIdx.z == 0) a.tab[to] = ok ? to : -1;
    if (!ok || k0 < first) return;
    const size_t src = paged_row(a.t, from, k0, a.row), dst = paged_row(a.t, to, k0, a.row);
    const int n8 = min(16, r.keys - k0) * a.row / 8;
    for (int i = threadIdx.x + 256 * blockIdx.z; i < n8; i += 256 * gridDim.z) {
        *reinterpret_cast<half8*>(a.ko + dst + 8 * (size_t)i) = load8h(a.kc + src + 8 * (size_t)i);
        *reinterpret_cast<half8*>(a.vo + dst + 8 * (size_t)i) = load8h(a.vc + src + 8 * (size_t)i);
    }
}

// ---------------------------------------------------------------- pages of a workgroup's tiles
// Lane j holds, for tile t0 + j (64 at a time), the table entry of the 16 rows that its wave moves and a
// bit for each 16 rows of the tile whose page is not there.
template <int KT>
struct TilePages {
    int entry = -1, gone = 0;
    __device__ __forceinline__ void load(const PageTab& t, int b, int key0, int own, int lane) {
        const rsrc_t rt = make_rsrc(t.table + (size_t)b * t.stride, (uint32_t)t.cols * 4);
        int e[KT / 16];
#pragma unroll
        for (int i = 0; i < KT / 16; ++i)
            e[i] = __builtin_amdgcn_raw_buffer_load_b32(rt, ((key0 + KT * lane + 16 * i) >> t.shift) * 4, 0, 0);
        gone = 0;
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) {
            entry = i == own ? e[i] : entry;
            gone |= page_ok(t, e[i]) ? 0 : 1 << i;
        }
    }
};
// the 16 rows of keys k0 .. of a page as a buffer resource: rows at or past kv_hi, and all of a page that
// is not there, read as zeros
__device__ __forceinline__ rsrc_t page_rows(const PageTab& t, const void* pool, int entry, int k0, int kv_hi, int row,
                                            int kh_off) {
    const bool ok = page_ok(t, entry);
    const uint32_t bytes = ok ? (uint32_t)(clamp16(kv_hi - k0) * row * 2) : 0u;
    return make_rsrc(reinterpret_cast<const half_t*>(pool) + paged_row(t, ok ? entry : 0, k0, row) + kh_off, bytes);
}
constexpr int kNoRow = 0x7fff0000;  // an offset past every such range (64 MiB at most), with room for a row's own bytes

// A transposed read that does not wait for the DMAs in flight. The compiler cannot tell that those fill other
// tiles and would wait for all of them (vmcnt 0) before the first read of a tile's V; the __restrict puts the
// read in an alias scope of its own. The tile loop's own wait and barrier order it behind the DMAs of its tile.
__device__ __forceinline__ half4 read_tr16(const half_t* __restrict p) { return lds_tr16(p); }

// ---------------------------------------------------------------- hd 256
// 32 query columns a wave, 128 a workgroup, key tiles of 64 moved straight into LDS and double
// buffered: the LDS layout and swizzles of prefill_kernel_w32, its tile loop pipelined by hand (below).
// 7856 tokens, kvH 2, up to 3000 keys: 112 us = 770 TFLOP/s (123 us with the plain loop, 118 waiting for the
// DMAs at V's first read). A tile takes 2200 cycles of MFMA and about 3500 of LDS: K rows 1024, V's
// transposed reads 1490, the DMAs' writes 1024; beside the tiles a unit takes about 9 us (its page entries,
// q, the first scores, the epilogue), which bounds short prompts and windows (15252 tokens, window 512: 121 us).
template <int G, typename OUTT>
__global__ __launch_bounds__(256) void paged_prefill_kernel_256(PagedPrefillArgs a) {
    constexpr int HD = 256, KT = 64, NCOL = 128, BQ = NCOL / G;
    constexpr int ROWB = HD * 2;      // bytes per LDS tile row
    constexpr int TILEB = KT * ROWB;  // one K or V tile
    __shared__ __attribute__((aligned(1024))) char lds[2 * 2 * TILEB];  // [buffer][K, V]

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n32 = lane & 31, h = lane >> 5;
    if ((int)blockIdx.x >= a.counts[0]) return;  // past the work list
    const PagedUnit wu = a.units[blockIdx.x];
    const int start_pos = wu.start, S = wu.S, row0 = wu.row0;
    const int T_total = start_pos + S;
    const int kh = wu.kh, qb = wu.qb, n_pieces = wu.n_pieces;

    // ---- key range of the workgroup [wg_lo, kv_hi) in tiles; with a key split this
    // workgroup takes tiles [t0, t1) of its query block
    const int p0 = start_pos + qb * BQ;
    const int kv_hi = min(p0 + BQ, T_total);
    const int first = a.window > 0 ? max(0, p0 + 1 - a.window) : 0;  // first attended key
    const int wg_lo = first & ~15;
    const int t0 = wu.t0, t1 = wu.t1;

    // ---- this lane's query column (head hh, position offset pl) and 8-dim half h
    const int c = 32 * wave + n32;
    const int hh = c % G, pl = c / G;
    const int s_raw = qb * BQ + pl;
    const bool col_ok = s_raw < S;
    const int s_idx = col_ok ? s_raw : S - 1;
    const int pos = start_pos + s_idx;

    // K/V rows of this kv head; wave w moves rows 16w .. 16w + 15 of a tile, two rows (1 KiB) an instruction
    const int rowg = a.n_kv_heads * HD * 2;  // bytes per cache row
    TilePages<KT> pages;
    // this wave's 16 rows of tile t from the page of `entry`; past the last tile: an empty range
    const auto tile_rows = [&](const void* pool, int t, int entry) {
        const int kg = wg_lo + t * KT + 16 * wave;
        return page_rows(a.t, pool, entry, kg, t < t1 ? kv_hi : kg, rowg / 2, kh * HD);
    };
    // DMA j of a wave's eight for a tile: two rows. swz: K's or V's chunk places
    const auto dma = [&](rsrc_t rp, char* dst, int j, int off) {
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rp, (__attribute__((address_space(3))) void*)(dst + (16 * wave + 2 * j) * ROWB),
                                                 16, off, 0, 0, 0);
    };
    const auto k_off = [&](int j) { return (2 * j + h) * rowg + 16 * (n32 ^ ((16 * wave + 2 * j + h) & 31)); };
    const auto v_off = [&](int j) { return (2 * j + h) * rowg + 16 * (n32 ^ vswz(2 * j + h)); };
    const auto tile_k = [&](int t) { return lds + (t & 1) * 2 * TILEB; };
    const auto tile_v = [&](int t) { return lds + (t & 1) * 2 * TILEB + TILEB; };

    // ---- q: lane (column, h) holds dims 16s + 8h + i (s < 16, i < 8), the B operand of the 32x32x16
    // MFMA. Wave w DMAs the f16 q rows of its own 32 columns (two 512-byte rows an instruction, chunk
    // n32 of a row from logical chunk n32 ^ (row % 32)) into the LDS stage that tile t0 + 1 takes over
    // later, then reads them back in that layout; rows past the block's last token read as zeros.
    half8 qf[16];
    int entry1, gone0, gone1 = 0;  // tile t + 1's page, the 16-row groups of tiles t and t + 1 without one
    {
        const rsrc_t rq = make_rsrc(a.q16 + ((size_t)row0 + qb * BQ) * a.n_q_heads * HD, (uint32_t)min(BQ, S - qb * BQ) * a.n_q_heads * ROWB);
        char* qs = lds + ((t0 + 1) & 1) * 2 * TILEB;
        pages.load(a.t, wu.b, wg_lo + t0 * KT, wave, lane);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
            const int r = 32 * wave + 2 * j + h;  // column of the row this lane moves
            const int qo = ((r / G) * a.n_q_heads + kh * G + r % G) * ROWB + 16 * (n32 ^ (r & 31));
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (__attribute__((address_space(3))) void*)(qs + (32 * wave + 2 * j) * ROWB),
                                                     16, qo, 0, 0, 0);
        }
        entry1 = wu.page[0];  // this wave's group
        gone0 = 0;
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) {
            entry1 = i == wave ? wu.page[i] : entry1;
            gone0 |= page_ok(a.t, wu.page[i]) ? 0 : 1 << i;
        }
        if (t0 < t1) {  // tile t0: of the block's first tile, rows in front of the first attended key read as zeros
            const rsrc_t rk = tile_rows(a.kc, t0, entry1), rv = tile_rows(a.vc, t0, entry1);
            const int skip = first - (wg_lo + t0 * KT + 16 * wave);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                dma(rk, tile_k(t0), j, 2 * j + h < skip ? kNoRow : k_off(j));
                dma(rv, tile_v(t0), j, 2 * j + h < skip ? kNoRow : v_off(j));
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        const char* qrow = qs + c * ROWB;
#pragma unroll
        for (int s = 0; s < 16; ++s) qf[s] = *reinterpret_cast<const half8*>(qrow + 16 * ((2 * s + h) ^ n32));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // stage free for tile t0 + 1's DMA
        if (!col_ok) {
#pragma unroll
            for (int s = 0; s < 16; ++s) qf[s] = half8{0, 0, 0, 0, 0, 0, 0, 0};
        }
        // q is only ever an MFMA B operand, which may sit in AGPRs: that leaves the VGPRs to
        // the O^T accumulators, the scores and the LDS operand batches
#pragma unroll
        for (int s = 0; s < 16; ++s) asm volatile("" : "+a"(qf[s]));
    }

    // ---- key ranges: this wave [w_lo, wp1], this column [col_lo, pos]
    const int wp0 = p0 + (32 * wave) / G;
    const int wp1 = min(p0 + (32 * wave + 31) / G, T_total - 1);
    const int col_lo = a.window > 0 ? pos + 1 - a.window : 0;

    float16v oacc[8];  // O^T[32dt + 8(r/4) + 4h + r%4][column]
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) oacc[dt] = float16v{};
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) asm volatile("" : "+a"(oacc[dt]));
    float m_use = kNegInf, l_run = 0.0f;
    bool started = false;

    // transposed V reads: 16-lane group (h, half16), lane m supplies row 4h + m/4 (+8, +16u),
    // dims 32dt + 16 half16 + 4(m%4) .. +3
    const int m16 = lane & 15, half16 = (lane >> 4) & 1;
    const int vr0 = 4 * h + (m16 >> 2);
    const int vc0 = 2 * half16 + ((m16 & 3) >> 1);  // chunk within a 32-dim tile
    const int vb0 = 8 * (m16 & 1);                   // byte within the chunk
    const int vsw = vswz(vr0);                        // rows 16u + vr0 (+8) share r % 4

    // A tile's scores, S^T = K . Q^T: two 32-key sub-tiles, 16 k-steps of 16 dims, the two accumulator
    // chains in turn (a chain of dependent MFMAs issues at half rate).
    // Masks of tile t's scores: key kb + 4h + 32kt + 8(r/4) + r%4 of this lane's column; tiles inside every
    // column's range skip it.
    auto mask = [&](int t, int gone, float16v (&sc)[2]) {
        const int kb = wg_lo + t * KT;
        if ((kb + KT - 1 > wp0) || (a.window > 0 && kb < wp1 + 1 - a.window)) {
            const int rel_hi = pos - (kb + 4 * h), rel_lo = col_lo - (kb + 4 * h);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int o = 32 * kt + 8 * (r >> 2) + (r & 3);
                    sc[kt][r] = (o <= rel_hi && o >= rel_lo) ? sc[kt][r] : kNegInf;
                }
        }
        if (gone) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[kt][r] = gone >> (2 * kt + (r >> 3)) & 1 ? kNegInf : sc[kt][r];
        }
    };

    // One tile. A wave has its SIMD to itself, so what is to overlap has to be interleaved in its own
    // instruction stream (the order below is kept by the sched_barriers):
    //   * the 32 score MFMAs of tile t + 1 with the exponentials of tile t -- a step's two MFMAs take the
    //     matrix unit 64 cycles, in which two exponentials of three stages (argument, exp2, sum and
    //     rounding of the step before) and the operand reads two steps ahead issue -- and with the DMAs
    //     of V(t + 1) and K(t + 2), which issue one a step: all 16 at once hold the wave up while the
    //     CU's four waves queue for the 64 B/clk path into LDS (1190 of 5300 cycles a tile);
    //   * the 32 P.V MFMAs of tile t with the maxima of tile t + 1.
    // So K is fetched two tiles ahead, V one: K(t + 2) into the buffer of K(t), whose scores are done,
    // V(t + 1) into that of V(t - 1).
    float mnext = kNegInf;  // this lane's maximum of the scores of the next tile
    auto tile = [&](int t, float16v (&sacc)[2], float16v (&snext)[2]) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part of V(t) and K(t + 1) is in LDS
        __syncthreads();                                    // all parts; K(t) and V(t - 1) fully consumed
        const int gone = gone1, entry = entry1;             // of tile t + 1
        {
            const int j = (t + 2 - t0) & 63;
            if (j == 0) pages.load(a.t, wu.b, wg_lo + (t + 2) * KT, wave, lane);
            entry1 = __builtin_amdgcn_readlane(pages.entry, j);
            gone1 = __builtin_amdgcn_readlane(pages.gone, j);
        }
        const float mloc = max32(mnext) * a.scale_log2;  // the column's other half sits in lane ^ 32 (scale > 0)
        // move the running maxima only when a score passes one by more than 2^kMaxLag
        const bool bump = mloc > m_use + kMaxLag;
        if (__any(bump)) {
            const float m_new = fmaxf(m_use, mloc - kPagedLift);
            const float corr = m_use == kNegInf ? 0.0f : fexp2(m_use - m_new);
            l_run *= corr;
            if (started) {
                // one 16-register tile at a time: copied to VGPRs, scaled, pinned back into
                // AGPRs (left to itself the compiler moves all of them at once)
                asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"  // the last MFMA's writes, as in the epilogue
                             : "+a"(oacc[0]), "+a"(oacc[1]), "+a"(oacc[2]), "+a"(oacc[3]), "+a"(oacc[4]),
                               "+a"(oacc[5]), "+a"(oacc[6]), "+a"(oacc[7]));
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) {
                    float16v x = oacc[dt];
                    asm volatile("" : "+v"(x));
                    x *= corr;
                    asm volatile("" : "+v"(x));
                    oacc[dt] = x;
                    asm volatile("" : "+a"(oacc[dt]));
                }
            }
            m_use = m_new;
        }
        started = true;
        const float msub = m_use == kNegInf ? 0.0f : m_use;
        half8 pb[4];
        float ps = 0.0f;
        {
            const char* krow0 = tile_k(t + 1) + n32 * ROWB;
            const char* krow1 = krow0 + 32 * ROWB;
            half8 kr[3][2];
            auto read_k = [&](int s) {
                const int cb = 16 * ((2 * s + h) ^ n32);
                kr[s % 3][0] = *reinterpret_cast<const half8*>(krow0 + cb);
                kr[s % 3][1] = *reinterpret_cast<const half8*>(krow1 + cb);
            };
            // exponential v of the lane's 32 in three stages
            float ex[2][2], ev[2][2];
            auto arg = [&](int v) { ex[(v >> 1) & 1][v & 1] = __builtin_fmaf(sacc[v >> 4][v & 15], a.scale_log2, -msub); };
            auto expo = [&](int v) { ev[(v >> 1) & 1][v & 1] = fexp2(ex[(v >> 1) & 1][v & 1]); };
            auto take = [&](int v) {
                const float e = ev[(v >> 1) & 1][v & 1];
                ps += e;
                pb[v >> 3][v & 7] = (half_t)e;
            };
            read_k(0);
            read_k(1);
            arg(0);
            arg(1);
            const rsrc_t rv = tile_rows(a.vc, t + 1, entry), rk = tile_rows(a.kc, t + 2, entry1);
            snext[0] = snext[1] = float16v{};
#pragma unroll
            for (int s = 0; s < 16; ++s) {
                if (s + 2 < 16) read_k(s + 2);
                snext[0] = mfma32(kr[s % 3][0], qf[s], snext[0]);
                expo(2 * s);
                expo(2 * s + 1);
                if (s > 0) {
                    take(2 * s - 2);
                    take(2 * s - 1);
                }
                snext[1] = mfma32(kr[s % 3][1], qf[s], snext[1]);
                if (s < 15) {
                    arg(2 * s + 2);
                    arg(2 * s + 3);
                }
                if (s < 8) dma(rv, tile_v(t + 1), s, v_off(s));
                else dma(rk, tile_k(t + 2), s - 8, k_off(s - 8));
                __builtin_amdgcn_sched_barrier(0);
            }
            take(30);
            take(31);
        }
        l_run += ps;
        // (here, not where they are used behind the masks' branches: the compiler would sink them there)
        asm volatile("" : "+v"(pb[0]), "+v"(pb[1]), "+v"(pb[2]), "+v"(pb[3]), "+v"(l_run));
        if (t + 1 < t1) mask(t + 1, gone, snext);

        // O^T += V^T . P^T over four 16-key steps; k-slot i < 4 is key 16u + 4h + i, i >= 4 is key
        // 16u + 8 + 4h + i - 4, matching the S^T accumulator rows in pb. Transposed V reads (two an
        // MFMA) kPvAhead MFMAs ahead.
        {
            const char* V = tile_v(t);
            half8 av[kPvAhead + 1];
            auto read_v = [&](int i) {
                const int u = i >> 3, ch = 4 * (i & 7) + vc0;
                const char* vp = V + (16 * u + vr0) * ROWB + 16 * (ch ^ vsw) + vb0;
                const half4 lo = read_tr16(reinterpret_cast<const half_t*>(vp));
                const half4 hi = read_tr16(reinterpret_cast<const half_t*>(vp + 8 * ROWB));
                av[i % (kPvAhead + 1)] = half8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
            mnext = kNegInf;
#pragma unroll
            for (int i = 0; i < kPvAhead; ++i) read_v(i);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (i + kPvAhead < 32) read_v(i + kPvAhead);
                mfma32_acc(oacc[i & 7], av[i % (kPvAhead + 1)], pb[i >> 3]);
                if (i >= 8 && i < 24) mnext = fmaxf(mnext, fmaxf(snext[(i - 8) >> 3][2 * (i & 7)], snext[(i - 8) >> 3][2 * (i & 7) + 1]));
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" : "+v"(mnext));
        }
    };
    if (t0 < t1) {
        float16v sa[2] = {float16v{}, float16v{}}, sb[2];
        __syncthreads();  // K(t0), V(t0); every wave has its q
        entry1 = __builtin_amdgcn_readlane(pages.entry, 1);
        gone1 = __builtin_amdgcn_readlane(pages.gone, 1);
        const rsrc_t rk = tile_rows(a.kc, t0 + 1, entry1);
#pragma unroll
        for (int j = 0; j < 8; ++j) dma(rk, tile_k(t0 + 1), j, k_off(j));
        const char* krow0 = tile_k(t0) + n32 * ROWB;
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            const int cb = 16 * ((2 * s + h) ^ n32);
            sa[0] = mfma32(*reinterpret_cast<const half8*>(krow0 + cb), qf[s], sa[0]);
            sa[1] = mfma32(*reinterpret_cast<const half8*>(krow0 + 32 * ROWB + cb), qf[s], sa[1]);
        }
        mask(t0, gone0, sa);
#pragma unroll
        for (int r = 0; r < 16; ++r) mnext = fmaxf(mnext, fmaxf(sa[0][r], sa[1][r]));
        for (int t = t0;;) {  // the two score sets change roles every tile
            tile(t, sa, sb);
            if (++t >= t1) break;
            tile(t, sb, sa);
            if (++t >= t1) break;
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last tile's (empty) DMAs, before LDS is used again
    }

    // ---- epilogue: column sum over both halves, normalise, srq, store 4 dims at a time
    // (the accumulators must not be read within 18 wait states of the last MFMA writing them, which the
    // compiler does not see)
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
                 : "+a"(oacc[0]), "+a"(oacc[1]), "+a"(oacc[2]), "+a"(oacc[3]), "+a"(oacc[4]), "+a"(oacc[5]),
                   "+a"(oacc[6]), "+a"(oacc[7]));
    const float l_tot = add32(l_run);
    if (n_pieces > 1) {  // a piece of a split query block: O / l and (m, l)
        const float inv_p = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) store_part<true, HD, NCOL * HD>(a.part_o, true, wu.slot, wave, dt, lane, oacc[dt], inv_p);
        if (h == 0) a.part_ml[(size_t)wu.slot * NCOL + c] = make_float2(m_use, l_tot);
        return;
    }
    const float inv = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
    if constexpr (sizeof(OUTT) == 2) {
        // f16 rows through LDS: each wave stages its 32 output rows (528-byte stride: the
        // 8-byte writes of a store instruction fall on distinct banks), then stores two whole
        // 512-byte rows an instruction. Written straight from the accumulator layout, every
        // store instruction put 16 bytes into each of 32 rows.
        constexpr int OSTR = HD * 2 + 16;
        __syncthreads();  // every wave is done with the last tile's K/V
        char* ost = lds + wave * 32 * OSTR;
        auto stage = [&](auto quantise) {  // (one test of the step for all of them)
#pragma unroll
            for (int dt = 0; dt < 8; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float4v v = float4v{oacc[dt][4 * j], oacc[dt][4 * j + 1], oacc[dt][4 * j + 2], oacc[dt][4 * j + 3]} * inv;
                    if constexpr (decltype(quantise)::value) v = srq4(v, a.out_q);
                    store4(reinterpret_cast<half_t*>(ost + n32 * OSTR) + 32 * dt + 8 * j + 4 * h, v);
                }
        };
        if (a.out_q == 0.0f) stage(std::false_type{});
        else stage(std::true_type{});
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int rr = 2 * i + h, cc = 32 * wave + rr;  // lanes 32h..: the wave's row rr
            const int so = qb * BQ + cc / G;
            const half8 val = *reinterpret_cast<const half8*>(ost + rr * OSTR + 16 * n32);
            if (so < S)
                *reinterpret_cast<half8*>(reinterpret_cast<half_t*>(a.out) +
                                          ((size_t)(row0 + so) * a.n_q_heads + kh * G + cc % G) * HD + 8 * n32) = val;
        }
    } else if (col_ok) {
        OUTT* orow = reinterpret_cast<OUTT*>(a.out) + ((size_t)(row0 + s_idx) * a.n_q_heads + kh * G + hh) * HD;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4v v = float4v{oacc[dt][4 * j], oacc[dt][4 * j + 1], oacc[dt][4 * j + 2],
                                          oacc[dt][4 * j + 3]} * inv;
                store4(orow + 32 * dt + 8 * j + 4 * h, srq4(v, a.out_q));
            }
    }
}

// ---------------------------------------------------------------- hd 512
// Every wave holds all 512 dims of its 32 columns, key tiles of 32: the LDS layout and register placement
// (O^T in AGPRs, q in VGPRs) of prefill_kernel_w32h, the tile loop interleaved as at hd 256. 13500 tokens in
// three prompts: 831 us = 840 TFLOP/s at the 1.7 GHz that the card's power allows (before kPagedLift 800 to 820, and
// then 873 us with the plain loop, 867 interleaved but waiting for its DMAs at V's first read); LDS is busy
// 3700 cycles a tile. Times at hd 256 and here are the least of 12 in a trace; the median here is 914.
template <int G, typename OUTT>
__global__ __launch_bounds__(256) void paged_prefill_kernel_512(PagedPrefillArgs a) {
    constexpr int HD = 512, KT = 32, NCOL = 128, BQ = NCOL / G;
    constexpr int ROWB = HD * 2;       // 1 KiB rows
    constexpr int TILEB = KT * ROWB;   // one K or V tile: 32 KiB
    constexpr int OSTR = HD * 2 + 16;  // the epilogue's staged f16 output rows (1040 B apart)
    constexpr int LDS_BYTES = 2 * 2 * TILEB > 4 * 32 * OSTR ? 2 * 2 * TILEB : 4 * 32 * OSTR;
    __shared__ __attribute__((aligned(1024))) char lds[LDS_BYTES];  // [buffer][K, V]; output rows

    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n32 = lane & 31, h = lane >> 5;
    if ((int)blockIdx.x >= a.counts[0]) return;  // past the work list
    const PagedUnit wu = a.units[blockIdx.x];
    const int start_pos = wu.start, S = wu.S, row0 = wu.row0;
    const int T_total = start_pos + S;
    const int kh = wu.kh, qb = wu.qb, n_pieces = wu.n_pieces;

    const int p0 = start_pos + qb * BQ;
    const int kv_hi = min(p0 + BQ, T_total);
    const int first = a.window > 0 ? max(0, p0 + 1 - a.window) : 0;  // first attended key
    const int wg_lo = first & ~15;
    const int t0 = wu.t0, t1 = wu.t1;

    // ---- this lane's query column (head hh, position offset pl) and 8-dim half h
    const int c = 32 * wave + n32;
    const int hh = c % G, pl = c / G;
    const int s_raw = qb * BQ + pl;
    const bool col_ok = s_raw < S;
    const int s_idx = col_ok ? s_raw : S - 1;
    const int pos = start_pos + s_idx;

    // K/V rows: wave w moves rows 8w .. 8w + 7 of a tile, one 1 KiB row an instruction. (The lane index
    // passes through an empty asm each time, so the source offsets are formed where they are used rather
    // than held in registers across the loop.)
    const int rowg = a.n_kv_heads * HD * 2;
    TilePages<KT> pages;
    // the 16 rows of tile t that this wave's 8 belong to, from the page of `entry`; past the last tile: an
    // empty range
    const auto tile_rows = [&](const void* pool, int t, int entry) {
        const int kg = wg_lo + t * KT + 16 * (wave >> 1);
        return page_rows(a.t, pool, entry, kg, t < t1 ? kv_hi : kg, rowg / 2, kh * HD);
    };
    const auto dma = [&](rsrc_t rp, char* dst, int j, int row_off, int swz) {
        int ln = lane;
        asm volatile("" : "+v"(ln));
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rp, (__attribute__((address_space(3))) void*)(dst + (8 * wave + j) * ROWB), 16,
                                                 row_off + 16 * (ln ^ swz), 0, 0, 0);
    };
    const auto row_off = [&](int j) { return (8 * (wave & 1) + j) * rowg; };
    const auto k_swz = [&](int j) { return (8 * wave + j) & 31; };
    const auto v_swz = [&](int j) { return vswz(j); };
    const auto tile_k = [&](int t) { return lds + (t & 1) * 2 * TILEB; };
    const auto tile_v = [&](int t) { return lds + (t & 1) * 2 * TILEB + TILEB; };

    // ---- q: lane (column c, half h) holds dims 16s + 8h .. +7 (s < 32), the B operand layout. Wave w
    // DMAs the f16 q rows of its 32 columns, whole 1 KiB rows (chunk n of a row from logical chunk
    // n ^ (column % 32)), into its 16 KiB of the LDS stage that tile t0 + 1 takes over later, in two
    // rounds of 16 rows, and reads each round back in that layout; tile t0's DMA goes out after the
    // first round's. Rows past the block's last token read as zeros.
    half8 qf[32];
    int entry1 = wave >> 1 ? wu.page[1] : wu.page[0];  // tile t + 1's page
    // the 16-row groups of tiles t and t + 1 without one
    int gone0 = (page_ok(a.t, wu.page[0]) ? 0 : 1) | (page_ok(a.t, wu.page[1]) ? 0 : 2), gone1 = 0;
    {
        const rsrc_t rq = make_rsrc(a.q16 + ((size_t)row0 + qb * BQ) * a.n_q_heads * HD, (uint32_t)min(BQ, S - qb * BQ) * a.n_q_heads * ROWB);
        pages.load(a.t, wu.b, wg_lo + t0 * KT, wave >> 1, lane);
        char* qs = lds + ((t0 + 1) & 1) * 2 * TILEB + wave * 16 * ROWB;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            int ln = lane;
            asm volatile("" : "+v"(ln));
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int cj = 32 * wave + 16 * r + j;  // the column whose row this DMA moves
                const int qo = ((cj / G) * a.n_q_heads + kh * G + cj % G) * ROWB + 16 * (ln ^ (16 * r + j));
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (__attribute__((address_space(3))) void*)(qs + j * ROWB),
                                                         16, qo, 0, 0, 0);
            }
            if (r == 0 && t0 < t1) {
                // of the block's first tile, rows in front of the first attended key read as zeros
                const rsrc_t rk = tile_rows(a.kc, t0, entry1), rv = tile_rows(a.vc, t0, entry1);
                const int skip = first - (wg_lo + t0 * KT + 16 * (wave >> 1));
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int ro = 8 * (wave & 1) + j < skip ? kNoRow : row_off(j);
                    dma(rk, tile_k(t0), j, ro, k_swz(j));
                    dma(rv, tile_v(t0), j, ro, v_swz(j));
                }
                asm volatile("s_waitcnt vmcnt(16)" ::: "memory");  // the 16 q DMAs before tile t0's
            } else {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            }
            if ((n32 >> 4) == r) {
                const char* qrow = qs + (n32 & 15) * ROWB;
#pragma unroll
                for (int s = 0; s < 32; ++s) qf[s] = *reinterpret_cast<const half8*>(qrow + 16 * ((2 * s + h) ^ n32));
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // this wave's 16 KiB free again
        }
        if (!col_ok) {
#pragma unroll
            for (int s = 0; s < 32; ++s) qf[s] = half8{0, 0, 0, 0, 0, 0, 0, 0};
        }
    }

    // ---- key ranges: this wave [w_lo, wp1], this column [col_lo, pos]
    const int wp0 = p0 + (32 * wave) / G;
    const int wp1 = min(p0 + (32 * wave + 31) / G, T_total - 1);
    const int col_lo = a.window > 0 ? pos + 1 - a.window : 0;

    // LDS read offsets. K operand k-step s of this lane: row n32, chunk (2s + h) ^ n32, i.e.
    // byte kofs ^ 32s with kofs = 1024 n32 + 16 (h ^ n32). Transposed V reads (as
    // prefill_kernel_w32's): row 16u + 8i + vr0, chunk (4dt + vc0) ^ vsw, i.e. byte
    // (vofs ^ 64dt) + 1024 (16u + 8i) with vofs = 1024 vr0 + 16 (vc0 ^ vsw) + vb0. Both offsets
    // pass through an empty asm every tile, so the compiler forms the 32 + 16 XORs in the
    // loop instead of holding 48 hoisted addresses.
    const int m16 = lane & 15, half16 = (lane >> 4) & 1;
    const int vr0 = 4 * h + (m16 >> 2);
    const int vc0 = 2 * half16 + ((m16 & 3) >> 1);
    const int vb0 = 8 * (m16 & 1);
    const int kofs0 = 1024 * n32 + 16 * (h ^ n32);
    const int vofs0 = 1024 * vr0 + 16 * (vc0 ^ vswz(vr0)) + vb0;

    float16v oacc[16];  // O^T[32dt + 8(r/4) + 4h + r%4][column]
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) oacc[dt] = float16v{};
#pragma unroll
    for (int dt = 0; dt < 16; ++dt) asm volatile("" : "+a"(oacc[dt]));
    float m_use = kNegInf, l_run = 0.0f;
    bool started = false;
    // Masks of tile t's scores: key kb + 4h + 8(r/4) + r%4 of this lane's column; tiles inside every column's
    // range skip it.
    auto mask = [&](int t, int gone, float16v& sc) {
        const int kb = wg_lo + t * KT;
        if ((kb + KT - 1 > wp0) || (a.window > 0 && kb < wp1 + 1 - a.window)) {
            const int rel_hi = pos - (kb + 4 * h), rel_lo = col_lo - (kb + 4 * h);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int o = 8 * (r >> 2) + (r & 3);
                sc[r] = (o <= rel_hi && o >= rel_lo) ? sc[r] : kNegInf;
            }
        }
        if (gone) {
#pragma unroll
            for (int r = 0; r < 16; ++r) sc[r] = gone >> (r >> 3) & 1 ? kNegInf : sc[r];
        }
    };

    // One tile, interleaved as in the hd-256 kernel: the 32 score MFMAs of tile t + 1 (even and odd k-steps
    // in two chains, added at the end) with the 16 exponentials of tile t and the DMAs of V(t + 1) and
    // K(t + 2); the 32 P.V MFMAs of tile t with the maxima of tile t + 1. On entry sacc holds tile t's
    // scores, on return tile t + 1's.
    float16v sacc = float16v{};
    float mnext = kNegInf;  // this lane's maximum of them
    auto tile = [&](int t) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's rows of V(t) and K(t + 1) are in LDS
        __syncthreads();
        const int gone = gone1, entry = entry1;             // of tile t + 1
        {
            const int j = (t + 2 - t0) & 63;
            if (j == 0) pages.load(a.t, wu.b, wg_lo + (t + 2) * KT, wave >> 1, lane);
            entry1 = __builtin_amdgcn_readlane(pages.entry, j);
            gone1 = __builtin_amdgcn_readlane(pages.gone, j);
        }
        const float mloc = max32(mnext) * a.scale_log2;
        const bool bump = mloc > m_use + kMaxLag;  // the running maxima move only past 2^kMaxLag
        if (__any(bump)) {
            const float m_new = fmaxf(m_use, mloc - kPagedLift);
            const float corr = m_use == kNegInf ? 0.0f : fexp2(m_use - m_new);
            l_run *= corr;
            if (started) {
                // one 16-register tile at a time: copied to VGPRs, scaled, pinned back into
                // AGPRs (left to itself the compiler moves all 256 through VGPRs and spills)
                asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"  // the last MFMA's writes, as in the epilogue
                             : "+a"(oacc[0]), "+a"(oacc[1]), "+a"(oacc[2]), "+a"(oacc[3]), "+a"(oacc[4]),
                               "+a"(oacc[5]), "+a"(oacc[6]), "+a"(oacc[7]), "+a"(oacc[8]), "+a"(oacc[9]),
                               "+a"(oacc[10]), "+a"(oacc[11]), "+a"(oacc[12]), "+a"(oacc[13]), "+a"(oacc[14]),
                               "+a"(oacc[15]));
#pragma unroll
                for (int dt = 0; dt < 16; ++dt) {
                    float16v x = oacc[dt];
                    asm volatile("" : "+v"(x));
                    x *= corr;
                    asm volatile("" : "+v"(x));
                    oacc[dt] = x;
                    asm volatile("" : "+a"(oacc[dt]));
                }
            }
            m_use = m_new;
        }
        started = true;
        const float msub = m_use == kNegInf ? 0.0f : m_use;
        half8 pb[2];
        float ps = 0.0f;
        float16v se = float16v{}, so = float16v{};
        {
            int kofs = ((t + 1) & 1) * 2 * TILEB + kofs0;
            asm volatile("" : "+v"(kofs));
            half8 kr[3][2];
            auto read_k = [&](int s) {
                kr[s % 3][0] = *reinterpret_cast<const half8*>(lds + (kofs ^ (64 * s)));
                kr[s % 3][1] = *reinterpret_cast<const half8*>(lds + (kofs ^ (64 * s + 32)));
            };
            // exponential v of the lane's 16 in three stages
            float ex[2], ev[2];
            auto arg = [&](int v) { ex[v & 1] = __builtin_fmaf(sacc[v], a.scale_log2, -msub); };
            auto take = [&](int v) {
                ps += ev[v & 1];
                pb[v >> 3][v & 7] = (half_t)ev[v & 1];
            };
            read_k(0);
            read_k(1);
            arg(0);
            const rsrc_t rv = tile_rows(a.vc, t + 1, entry), rk = tile_rows(a.kc, t + 2, entry1);
#pragma unroll
            for (int s = 0; s < 16; ++s) {
                if (s + 2 < 16) read_k(s + 2);
                se = mfma32(kr[s % 3][0], qf[2 * s], se);
                ev[s & 1] = fexp2(ex[s & 1]);
                if (s > 0) take(s - 1);
                so = mfma32(kr[s % 3][1], qf[2 * s + 1], so);
                if (s < 15) arg(s + 1);
                if (s < 8) dma(rv, tile_v(t + 1), s, row_off(s), v_swz(s));
                else dma(rk, tile_k(t + 2), s - 8, row_off(s - 8), k_swz(s - 8));
                __builtin_amdgcn_sched_barrier(0);
            }
            take(15);
        }
        l_run += ps;
        sacc = se + so;
        // (here, not where they are used behind the masks' branches: the compiler would sink them there)
        asm volatile("" : "+v"(pb[0]), "+v"(pb[1]), "+v"(l_run), "+v"(sacc));
        if (t + 1 < t1) mask(t + 1, gone, sacc);

        // O^T += V^T . P^T over two 16-key steps, 16 dims tiles each; transposed V reads (two an MFMA) kPvAhead
        // MFMAs ahead
        {
            int vofs = (t & 1) * 2 * TILEB + TILEB + vofs0;
            asm volatile("" : "+v"(vofs));
            half8 av[kPvAhead + 1];
            auto read_v = [&](int i) {
                const char* vp = lds + (vofs ^ (64 * (i & 15))) + 16 * (i >> 4) * ROWB;
                const half4 lo = read_tr16(reinterpret_cast<const half_t*>(vp));
                const half4 hi = read_tr16(reinterpret_cast<const half_t*>(vp + 8 * ROWB));
                av[i % (kPvAhead + 1)] = half8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
            mnext = kNegInf;
#pragma unroll
            for (int i = 0; i < kPvAhead; ++i) read_v(i);
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                if (i + kPvAhead < 32) read_v(i + kPvAhead);
                mfma32_acc(oacc[i & 15], av[i % (kPvAhead + 1)], pb[i >> 4]);
                if (i >= 8 && i < 16) mnext = fmaxf(mnext, fmaxf(sacc[2 * (i - 8)], sacc[2 * (i - 8) + 1]));
                __builtin_amdgcn_sched_barrier(0);
            }
            asm volatile("" : "+v"(mnext));
        }
    };
    if (t0 < t1) {
        __syncthreads();  // K(t0), V(t0); every wave has its q
        entry1 = __builtin_amdgcn_readlane(pages.entry, 1);
        gone1 = __builtin_amdgcn_readlane(pages.gone, 1);
        const rsrc_t rk = tile_rows(a.kc, t0 + 1, entry1);
#pragma unroll
        for (int j = 0; j < 8; ++j) dma(rk, tile_k(t0 + 1), j, row_off(j), k_swz(j));
        float16v se = float16v{}, so = float16v{};
        const int kofs = (t0 & 1) * 2 * TILEB + kofs0;
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            se = mfma32(*reinterpret_cast<const half8*>(lds + (kofs ^ (64 * s))), qf[2 * s], se);
            so = mfma32(*reinterpret_cast<const half8*>(lds + (kofs ^ (64 * s + 32))), qf[2 * s + 1], so);
        }
        sacc = se + so;
        mask(t0, gone0, sacc);
#pragma unroll
        for (int r = 0; r < 16; ++r) mnext = fmaxf(mnext, sacc[r]);
        for (int t = t0; t < t1; ++t) tile(t);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the last tile's (empty) DMAs, before LDS is used again
    }

    // ---- epilogue: the 512 dims of this wave's 32 columns. The accumulators are read by
    // VALU instructions below, which must not issue within 18 wait states of the last MFMA
    // writing them (the compiler does not see the asm MFMAs); the asm also orders every read
    // after the wait, since each accumulator passes through it.
    asm volatile("s_nop 7\n\ts_nop 7\n\ts_nop 3"
                 : "+a"(oacc[0]), "+a"(oacc[1]), "+a"(oacc[2]), "+a"(oacc[3]), "+a"(oacc[4]), "+a"(oacc[5]),
                   "+a"(oacc[6]), "+a"(oacc[7]), "+a"(oacc[8]), "+a"(oacc[9]), "+a"(oacc[10]), "+a"(oacc[11]),
                   "+a"(oacc[12]), "+a"(oacc[13]), "+a"(oacc[14]), "+a"(oacc[15]));
    const float l_tot = add32(l_run);
    if (n_pieces > 1) {  // a piece of a split query block: O / l and (m, l)
        const float inv_p = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
#pragma unroll
        for (int dt = 0; dt < 16; ++dt) store_part<false, HD, NCOL * HD>(a.part_o, true, wu.slot, wave, dt, lane, oacc[dt], inv_p);
        if (h == 0) a.part_ml[(size_t)wu.slot * NCOL + c] = make_float2(m_use, l_tot);
        return;
    }
    const float inv = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
    if constexpr (sizeof(OUTT) == 2) {
        // f16 rows through LDS: each wave stages its 32 output rows, then stores one whole 1 KiB row
        // an instruction
        __syncthreads();  // every wave is done with the last tile's K/V
        char* ost = lds + wave * 32 * OSTR;
        auto stage = [&](auto quantise) {  // (one test of the step for all of them)
#pragma unroll
            for (int dt = 0; dt < 16; ++dt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float4v v = float4v{oacc[dt][4 * j], oacc[dt][4 * j + 1], oacc[dt][4 * j + 2], oacc[dt][4 * j + 3]} * inv;
                    if constexpr (decltype(quantise)::value) v = srq4(v, a.out_q);
                    store4(reinterpret_cast<half_t*>(ost + n32 * OSTR) + 32 * dt + 8 * j + 4 * h, v);
                }
        };
        if (a.out_q == 0.0f) stage(std::false_type{});
        else stage(std::true_type{});
#pragma unroll
        for (int rr = 0; rr < 32; ++rr) {
            const int cc = 32 * wave + rr, so = qb * BQ + cc / G;
            const half8 val = *reinterpret_cast<const half8*>(ost + rr * OSTR + 16 * lane);
            if (so < S)
                *reinterpret_cast<half8*>(reinterpret_cast<half_t*>(a.out) +
                                          ((size_t)(row0 + so) * a.n_q_heads + kh * G + cc % G) * HD + 8 * lane) = val;
        }
    } else if (col_ok) {
        OUTT* orow = reinterpret_cast<OUTT*>(a.out) + ((size_t)(row0 + s_idx) * a.n_q_heads + kh * G + hh) * HD;
#pragma unroll
        for (int dt = 0; dt < 16; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float4v v = float4v{oacc[dt][4 * j], oacc[dt][4 * j + 1], oacc[dt][4 * j + 2],
                                          oacc[dt][4 * j + 3]} * inv;
                store4(orow + 32 * dt + 8 * j + 4 * h, srq4(v, a.out_q));
            }
    }
}

// Merge of the pieces of a split query block, as prefill_merge_kernel: with each piece holding
// o_p = O_p / l_p, out = sum_p o_p l_p 2^(m_p - M) / sum_p l_p 2^(m_p - M), M = max_p m_p. One workgroup
// per (entry of the merge list, wave block of 32 columns x 256 dims); thread (k, lane) owns the lane's
// 8-dim runs k, k + 4, .. of the 16 (dims tile, 4-row pair) runs. 4 to 5 us, a launch and one trip to memory;
// 0.9 when the plan has cut nothing.
template <typename OUTT, int HD>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedPrefillArgs a) {
    constexpr int NCOL = 128, MAXP = kMaxPieces;
    constexpr int NV = NCOL * HD, BLK = NV * 3;  // values and bytes of a piece's block
    if ((int)blockIdx.x >= a.counts[1]) return;
    const PagedUnit pu = a.merges[blockIdx.x];
    const int qb = pu.qb, w = blockIdx.y, kh = pu.kh, n_pieces = pu.n_pieces, tid = threadIdx.x;
    const int lane = tid & 63, k0 = tid >> 6;
    const int c = (HD == 256 ? 32 * w : 32 * (w >> 1)) + (lane & 31), h = lane >> 5;
    const int dbase = HD == 256 ? 0 : 256 * (w & 1);
    const int G = a.n_q_heads / a.n_kv_heads, BQ = NCOL / G;
    const int s_idx = qb * BQ + c / G;
    const size_t blk0 = (size_t)pu.slot;
    // buffer ranges end at the block's last piece: the loads of absent pieces read zeros,
    // so all of them issue at once with no branch
    const rsrc_t rml = make_rsrc(a.part_ml + blk0 * NCOL, (uint32_t)n_pieces * NCOL * 8);
    const rsrc_t ro = make_rsrc(reinterpret_cast<const char*>(a.part_o) + blk0 * BLK, (uint32_t)(n_pieces * BLK));
    float2 ml[MAXP];
    v4u32 ov[MAXP][4];
    v2u32 ob[MAXP][4];
#pragma unroll
    for (int p = 0; p < MAXP; ++p) ml[p] = bload_f32x2(rml, (p * NCOL + c) * 8);
#pragma unroll
    for (int p = 0; p < MAXP; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // run k = k0 + 4i: dims tile k/2, 4-row pair k%2
            const int run = w * (32 * 256) + (k0 + 4 * i) * 512 + 8 * lane;
            ov[p][i] = __builtin_amdgcn_raw_buffer_load_b128(ro, p * BLK + 2 * run, 0, 0);
            ob[p][i] = __builtin_amdgcn_raw_buffer_load_b64(ro, p * BLK + 2 * NV + run, 0, 0);
        }
    float wt[MAXP];
    float M = kNegInf;
#pragma unroll
    for (int p = 0; p < MAXP; ++p) {
        if (p >= n_pieces) ml[p] = make_float2(kNegInf, 0.0f);
        M = fmaxf(M, ml[p].x);
    }
    float L = 0.0f;
#pragma unroll
    for (int p = 0; p < MAXP; ++p) {  // a piece with no attended key weighs 0
        wt[p] = ml[p].x == kNegInf ? 0.0f : ml[p].y * fexp2(ml[p].x - M);
        L += wt[p];
    }
    float4v o[8];  // o[2i + e]: rows 8e.. of run i
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = float4v{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int p = 0; p < MAXP; ++p) {
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                v[e] = unpack24(ov[p][i], ob[p][i], e);
            o[2 * i] += float4v{v[0], v[1], v[2], v[3]} * wt[p];
            o[2 * i + 1] += float4v{v[4], v[5], v[6], v[7]} * wt[p];
        }
    if (s_idx >= pu.S) return;
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    OUTT* orow = reinterpret_cast<OUTT*>(a.out) + ((size_t)(pu.row0 + s_idx) * a.n_q_heads + kh * G + c % G) * HD + dbase;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int k = k0 + 4 * i, d = 32 * (k >> 1) + 16 * (k & 1) + 8 * e + 4 * h;
            store4(orow + d, srq4(o[2 * i + e] * inv, a.out_q));
        }
}


// ---------------------------------------------------------------- host side
typedef void (*paged_prefill_fn)(PagedPrefillArgs);

template <int G>
static paged_prefill_fn pick_out(int HD, bool out32) {
    if (HD == 256) return out32 ? paged_prefill_kernel_256<G, float> : paged_prefill_kernel_256<G, half_t>;
    return out32 ? paged_prefill_kernel_512<G, float> : paged_prefill_kernel_512<G, half_t>;
}
static paged_prefill_fn pick_paged(int HD, int G, bool out32) {  // G: 1, 2, 4 or 8 (check_cfg)
    switch (G) {
        case 1: return pick_out<1>(HD, out32);
        case 2: return pick_out<2>(HD, out32);
        case 4: return pick_out<4>(HD, out32);
        default: return pick_out<8>(HD, out32);
    }
}
static paged_prefill_fn pick_paged_merge(int HD, bool out32) {
    if (HD == 256) return out32 ? paged_merge_kernel<float, 256> : paged_merge_kernel<half_t, 256>;
    return out32 ? paged_merge_kernel<float, 512> : paged_merge_kernel<half_t, 512>;
}

// What the host can bound: query blocks (each sequence's last one may be short), units and partials; and
// the workspace [counts][units][merges][q16][partials][(m, l)][K16][V16][table16]. A server reserves one
// for its largest call and runs smaller ones in it, so every part grows with n_tokens, n_seq and
// max_key_len: there is room for partials also in a call too large to split.
struct PagedPlan {
    int bq, kt, max_units, max_slots, cols16;
    size_t units, merges, q16, part_o, part_ml, k16, v16, tab16, total;
};
static bool paged_plan(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens, PagedPlan& p) {
    const int HD = (int)cfg->head_dim, G = (int)(cfg->n_q_heads / cfg->n_kv_heads);
    const int64_t kvh = cfg->n_kv_heads;
    p.bq = 128 / G;
    p.kt = HD == 256 ? 64 : 32;
    const int64_t blocks = std::min<int64_t>(n_tokens, (int64_t)n_tokens / p.bq + pg->n_seq);
    // a split is of use only if the longest block can outlast the mean load of a CU (plan_units)
    int64_t keys = pg->max_key_len;
    if (cfg->window > 0) keys = std::min<int64_t>(keys, (int64_t)cfg->window + p.bq + 15);
    const PlanCost pc = plan_cost(p.kt);
    const double longest = (double)((keys + p.kt - 1) / p.kt) + pc.unit;
    const double load = (double)(n_tokens / p.bq) * (double)kvh * (1.0 + pc.unit) / kCus;
    const bool split = longest > load;
    const int slots = (int)std::min<int64_t>(blocks * kvh * kMaxPieces, kMaxSlots);
    p.max_slots = split ? slots : 0;
    const int64_t units = blocks * kvh + p.max_slots;
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    size_t at = 256;
    auto part = [&](size_t bytes) {
        const size_t x = at;
        at += al(bytes);
        return x;
    };
    p.max_units = (int)units;
    p.units = part((size_t)(blocks * kvh + slots) * sizeof(PagedUnit));
    p.merges = part((size_t)slots * sizeof(PagedUnit));
    p.q16 = part((size_t)n_tokens * cfg->n_q_heads * HD * sizeof(half_t));
    p.part_o = part((size_t)slots * 128 * HD * 3);
    p.part_ml = part((size_t)slots * 128 * sizeof(float2));
    p.k16 = p.v16 = p.tab16 = at;
    p.cols16 = 0;
    int64_t pages16 = 0;
    if (cfg->flags & G4A_KV_F32) {
        p.cols16 = (pg->max_key_len + pg->page_size - 1) / pg->page_size;
        pages16 = (int64_t)pg->n_seq * p.cols16;
        const size_t pool = (size_t)pages16 * pg->page_size * kvh * HD * sizeof(half_t);
        p.k16 = part(pool);
        p.v16 = part(pool);
        p.tab16 = part((size_t)pages16 * sizeof(int32_t));
    }
    p.total = at;
    if (units > 0x7fffffff || pages16 > 0x7fffffff) {
        set_error("n_tokens * n_kv_heads or n_seq * max_key_len too large");
        return false;
    }
    return true;
}

}  // namespace g4a

using namespace g4a;

extern "C" size_t g4a_paged_prefill_ws_bytes(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens) {
    if (check_paged(cfg, pg, true) || check_tokens(cfg, n_tokens, pg->key_len)) return 0;
    PagedPlan p;
    return paged_plan(cfg, pg, n_tokens, p) ? p.total : 0;
}

extern "C" int g4a_paged_prefill(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens, const int32_t* cu_q,
                                 const float* q, const float* q_gain, const float* rope_cos, const float* rope_sin,
                                 void* out, void* ws, size_t ws_bytes, void* stream_) {
    if (const int rc = check_paged(cfg, pg, true)) return rc;
    if (const int rc = check_tokens(cfg, n_tokens, cu_q)) return rc;
    if (const int rc = check_paged_call(cfg, n_tokens, q, q_gain, rope_cos, rope_sin, out)) return rc;
    if (cfg->flags & G4A_Q_HILO) {
        set_error("g4a_paged_prefill rounds q to f16 (G4A_Q_HILO not supported)");
        return G4A_EUNSUPPORTED;
    }
    const int HD = (int)cfg->head_dim, G = (int)(cfg->n_q_heads / cfg->n_kv_heads);
    PagedPlan p;
    if (!paged_plan(cfg, pg, n_tokens, p)) return G4A_EINVAL;
    if (!ws || (uintptr_t)ws % 256 || ws_bytes < p.total) {
        set_error("paged prefill workspace needs %zu bytes (256-byte aligned), got %zu", p.total, ws ? ws_bytes : (size_t)0);
        return G4A_EWORKSPACE;
    }
    const hipStream_t stream = (hipStream_t)stream_;
    char* w = (char*)ws;
    PagedPrefillArgs a;
    a.t = page_tab(pg);
    a.cu = cu_q;
    a.q = q;
    a.q_gain = q_gain;
    a.rcos = rope_cos;
    a.rsin = rope_sin;
    a.kc = pg->k_pages;
    a.vc = pg->v_pages;
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
    hipError_t e;
    if (cfg->flags & G4A_KV_F32) {
        PagedKv16Args k;
        k.t = a.t;
        k.cu = cu_q;
        k.kc = (const float*)pg->k_pages;
        k.vc = (const float*)pg->v_pages;
        k.ko = (half_t*)(w + p.k16);
        k.vo = (half_t*)(w + p.v16);
        k.tab = (int32_t*)(w + p.tab16);
        k.n_tokens = n_tokens;
        k.row = (int)cfg->n_kv_heads * HD;
        k.cols = p.cols16;
        k.window = a.window;
        // a workgroup per 16 rows, and per 512 elements of a row: four loads a thread (595 keys of 8 x 256: 11.4
        // us with one workgroup per 16 rows, 5 so)
        hipLaunchKernelGGL(paged_kv16_kernel, dim3((unsigned)((pg->max_key_len + 15) / 16), pg->n_seq, (unsigned)((k.row + 511) / 512)),
                           dim3(256), 0, stream, k);
        if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged cache conversion launch");
        // from here on the f16 copy and its table
        a.kc = w + p.k16;
        a.vc = w + p.v16;
        a.t.table = (const int32_t*)(w + p.tab16);
        a.t.cols = a.t.stride = p.cols16;
        a.t.n_pages = pg->n_seq * p.cols16;
    }
    const int64_t rows = (int64_t)n_tokens * ((a.n_q_heads + 3) / 4);  // waves, each four heads of a token
    const dim3 pgrid((unsigned)((rows + 3) / 4 + 1));
    if (HD == 256) hipLaunchKernelGGL(paged_prep_kernel<256>, pgrid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(paged_prep_kernel<512>, pgrid, dim3(256), 0, stream, a);
    if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged prefill preparation launch");
    const bool out32 = (cfg->flags & G4A_OUT_F32) != 0;
    hipLaunchKernelGGL(pick_paged(HD, G, out32), dim3((unsigned)p.max_units), dim3(256), 0, stream, a);
    if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged prefill launch");
    if (p.max_slots > 0) {  // a block of the merge list has two slots at least
        hipLaunchKernelGGL(pick_paged_merge(HD, out32), dim3((unsigned)p.max_slots / 2, 4 * (HD / 256)), dim3(256), 0, stream, a);
        if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged prefill merge launch");
    }
    return G4A_OK;
}
