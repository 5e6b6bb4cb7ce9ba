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

#include "paged_tiles.hpp"

namespace g4a {

constexpr int kMaxPieces = 8;  // pieces a query block is cut into
constexpr int kMaxSlots = 768; // pieces with partials in a call

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

__global__ __launch_bounds__(256) void paged_kv16_kernel(PagedKv16Args a) { kv16_rows<false>(a, blockIdx.x, blockIdx.y, blockIdx.z, gridDim.z); }

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
    if (HD == 256) return out32 ? paged_kernel_w256<G, float> : paged_kernel_w256<G, half_t>;
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
        k.klo = nullptr;
        k.tab = (int32_t*)(w + p.tab16);
        k.n_tokens = n_tokens;
        k.row = (int)cfg->n_kv_heads * HD;
        k.cols = p.cols16;
        k.window = a.window;
        k.rows_given = 0;
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
