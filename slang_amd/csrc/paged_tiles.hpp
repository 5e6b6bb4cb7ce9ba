// The attention of packed rows over a paged K/V cache on f16 MFMA: one work unit, a block of 128 query columns
// (the G heads of a kv head x 128/G tokens; trees at hd 512: 64) times the key tiles of a piece. paged_prefill.hip runs it over
// prompts, whose tokens attend every earlier row, paged_tree.hip over drafted trees, whose tokens attend their
// ancestors among the rows of the call (bits of a row per token, and per 64 keys a word).
#pragma once

#include <type_traits>

#include "paged.hpp"
#include "prefill_tiles.hpp"

namespace g4a {

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

// What a call over drafted trees has beside that. Bit k of a packed row's words is the row's answer for key
// (start & ~63) + k of its sequence (start: the row of the first token): attended or not, its ancestors and itself among
// the rows of the call, and the history in front of them in the same 64.
struct PagedTreeArgs : PagedPrefillArgs {
    const int32_t* parents;
    unsigned long long* bits;  // [n_tokens][words]
    int32_t* depth;            // [n_tokens]: the token's position is start + depth
    half_t* q16_lo;            // what f16 leaves of q, as q16
    const void* kc_lo;         // f32 caches: what f16 leaves of K, as kc
    int words;
};

// The rows of f32 pages that the call attends, as f16 pages of the workspace: page i of sequence b is
// page b * cols + i of ko / vo, and the table written to tab names it if the cache's own is there.
struct PagedKv16Args {
    PageTab t;
    const int32_t* cu;
    const float* kc;
    const float* vc;
    half_t* ko;
    half_t* vo;
    half_t* klo;  // what f16 leaves of K, or NULL
    int32_t* tab;
    int n_tokens, row, cols, window;
    int rows_given;  // the call's own rows are stored in both by whoever makes them
};
// What f16 leaves of x. (Of one beyond f16 -inf or inf: such a K shows as NaN in what attends it, as it does in decoding.)
__device__ __forceinline__ half_t rest16(float x) { return (half_t)(x - (float)(half_t)x); }
// rows 16 x .. of sequence b, part z of nz of their elements, by a workgroup of 256 threads. LO: K's remainders too
template <bool LO>
__device__ __forceinline__ void kv16_rows(const PagedKv16Args& a, int x, int b, int z, int nz) {
    const int k0 = 16 * x, ps = 1 << a.t.shift;
    const SeqRows r = seq_rows(a.t, a.cu, a.n_tokens, b);
    const int page = k0 >> a.t.shift;
    if (page >= a.cols) return;
    const int first = a.window > 0 ? max(0, r.keys - (r.hi - r.lo) + 1 - a.window) & ~15 : 0;
    const bool used = k0 < r.keys && r.hi > r.lo && (page + 1) << a.t.shift > first;
    const int from = used ? page_at(a.t, b, k0) : -1;
    const bool ok = page_ok(a.t, from);
    const int to = b * a.cols + page;
    if ((k0 & (ps - 1)) == 0 && threadIdx.x == 0 && z == 0) a.tab[to] = ok ? to : -1;
    if (!ok || k0 < first) return;
    const size_t src = paged_row(a.t, from, k0, a.row), dst = paged_row(a.t, to, k0, a.row);
    const int end = a.rows_given ? cut_tree(r).keys - (cut_tree(r).hi - r.lo) : r.keys;
    const int n8 = min(16, end - k0) * a.row / 8;
    for (int i = threadIdx.x + 256 * z; i < n8; i += 256 * nz) {
        if constexpr (LO) {
            const float4v x0 = *reinterpret_cast<const float4v*>(a.kc + src + 8 * (size_t)i);
            const float4v x1 = *reinterpret_cast<const float4v*>(a.kc + src + 8 * (size_t)i + 4);
            half8 hi, lo;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = e < 4 ? x0[e] : x1[e - 4];
                hi[e] = (half_t)x;
                lo[e] = rest16(x);
            }
            *reinterpret_cast<half8*>(a.ko + dst + 8 * (size_t)i) = hi;
            *reinterpret_cast<half8*>(a.klo + dst + 8 * (size_t)i) = lo;
        } else {
            *reinterpret_cast<half8*>(a.ko + dst + 8 * (size_t)i) = load8h(a.kc + src + 8 * (size_t)i);
        }
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
__device__ __forceinline__ half8 read_h8(const half8* __restrict p) { return *p; }
__device__ __forceinline__ float4v read_f4(const float* __restrict p) { return *reinterpret_cast<const float4v*>(p); }

// ---------------------------------------------------------------- 256 dims a wave
// 32 query columns a wave, 128 a workgroup, key tiles of 64 moved straight into LDS and double
// buffered: the LDS layout and swizzles of prefill_kernel_w32, its tile loop pipelined by hand (below).
// 7856 tokens, kvH 2, up to 3000 keys: 112 us = 770 TFLOP/s (123 us with the plain loop, 118 waiting for the
// DMAs at V's first read). A tile takes 2200 cycles of MFMA and about 3500 of LDS: K rows 1024, V's
// transposed reads 1490, the DMAs' writes 1024; beside the tiles a unit takes about 9 us (its page entries,
// q, the first scores, the epilogue), which bounds short prompts and windows (15252 tokens, window 512: 121 us).
//
// Trees run it at both head sizes, q always as a pair of f16 operands, so that drafts are checked as plain decoding
// chooses, whose scores are as exact:
//   * hd 512: two waves share 32 columns, each with 256 of their dims, whose halves of the scores meet in LDS behind P.V (64
//     columns a workgroup, key tiles of 32, as large as those of 64 at hd 256). A wave with all 512 dims of its columns, as in the
//     prompts' kernel, has no registers for q's second operand (q 128 and O 256 of 512). Against that kernel with q in f16: 8 trees
//     of 16 after 2000 keys 36 us a call for 41, 3 of 60 to 253 55 for 57; where history streams, twice the columns a K/V
//     byte tell: 16 of 5 to 40 after up to 16384 92 for 83.
//   * K32, over f32 caches: K's remainder in f16 is a second tile, multiplied by q's high operand behind the first. Both have
//     one place in LDS, which is filled again as soon as its products are done: high, low, P.V, each tile is on its way for two
//     of a tile's three phases, and the waits are counted so that the next one's fetch goes on. Half as many bytes again as
//     with K in f16 alone: 16 trees after up to 8192 keys at hd 512 160 us a call for 129 (15 more with each low tile fetched
//     and waited for within its own tile), 32 after up to 2000 at hd 256 52 for 45. P keeps its remainder too, on the V operands that
//     are there: outputs are 2.9e-4 off, 3.1 to 3.2e-4 without it, of which 2.1e-4 each are V's and the output's rounding to
//     f16 (1 to 5 % of a call; a V beyond f16 makes its outputs NaN where a weight leaves no remainder).
template <int G, typename OUTT, typename ARGS = PagedPrefillArgs, int HD = 256, bool K32 = false>
__global__ __launch_bounds__(256) void paged_kernel_w256(ARGS a) {
    constexpr bool TREE = std::is_same<ARGS, PagedTreeArgs>::value;
    static_assert(TREE || (HD == 256 && !K32), "prompts at hd 512 have a kernel of their own");
    constexpr int PAIR = HD / 256;                          // waves that share 32 columns
    constexpr int KT = 64 / PAIR, NS = KT / 32, NCOL = 128 / PAIR, BQ = NCOL / G;
    constexpr bool STAGED = !K32 && PAIR == 1;              // q through LDS
    constexpr bool LATE = !K32 && PAIR == 2;                // the next tile's scores are whole only behind P.V
    constexpr int ROWB = HD * 2;                            // bytes per LDS tile row
    constexpr int TILEB = KT * ROWB;                        // one K or V tile: 32 KiB
    constexpr int XCHB = PAIR == 2 ? 4 * 16 * 64 * 4 : 0;   // halves of scores: [wave][4 rows][lane][4]
    __shared__ __attribute__((aligned(1024))) char lds[2 * 2 * TILEB + XCHB];  // [buffer][K, V]

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
    // first attended key (of a tree: by a root)
    const int first = a.window > 0 ? max(0, (TREE ? start_pos : p0) + 1 - a.window) : 0;
    const int wg_lo = first & (TREE ? ~(KT - 1) : ~15);
    const int t0 = wu.t0, t1 = wu.t1;

    // ---- this lane's query column (head hh, position offset pl) and 8-dim half h
    const int cg = PAIR == 2 ? wave & 1 : wave, d0 = PAIR == 2 ? 256 * (wave >> 1) : 0;  // the wave's columns and dims
    const int c = 32 * cg + n32;
    const int hh = c % G, pl = c / G;
    const int s_raw = qb * BQ + pl;
    const bool col_ok = s_raw < S;
    const int s_idx = col_ok ? s_raw : S - 1;
    int pos = start_pos + s_idx;
    if constexpr (TREE) pos = start_pos + a.depth[row0 + s_idx];

    // K/V rows of this kv head; wave w moves rows 16w .. 16w + 15 of a tile, two rows (1 KiB) an instruction (hd 512: 8w ..
    // 8w + 7, one)
    const int rowg = a.n_kv_heads * HD * 2;  // bytes per cache row
    const void* kc_lo = nullptr;
    if constexpr (K32) kc_lo = a.kc_lo;
    TilePages<KT> pages;
    // this wave's 16 rows of tile t from the page of `entry`; past the last tile: an empty range
    const auto tile_rows = [&](const void* pool, int t, int entry) {
        const int kg = wg_lo + t * KT + 16 * (wave / PAIR);
        return page_rows(a.t, pool, entry, kg, t < t1 ? kv_hi : kg, rowg / 2, kh * HD);
    };
    // DMA j of a wave's eight for a tile: two rows (hd 512: one). row_of: this lane's of the wave's 16-row group; k_off, v_off:
    // its source, K's or V's chunk places
    const auto dma = [&](rsrc_t rp, char* dst, int j, int off) {
        const int row = PAIR == 2 ? 8 * wave + j : 16 * wave + 2 * j;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rp, (__attribute__((address_space(3))) void*)(dst + row * ROWB), 16, off, 0, 0, 0);
    };
    const int ln = PAIR == 2 ? lane : n32;  // this lane's chunk of a row
    const auto row_of = [&](int j) { return PAIR == 2 ? 8 * (wave & 1) + j : 2 * j + h; };
    const auto k_off = [&](int j) { return row_of(j) * rowg + 16 * (ln ^ ((16 * (wave / PAIR) + row_of(j)) & 31)); };
    const auto v_off = [&](int j) { return row_of(j) * rowg + 16 * (ln ^ vswz(row_of(j))); };
    const auto tile_k = [&](int t) { return lds + (K32 ? 0 : (t & 1) * 2 * TILEB); };
    const auto tile_k_lo = [&] { return lds + 2 * TILEB; };  // K32
    const auto tile_v = [&](int t) { return lds + (t & 1) * 2 * TILEB + TILEB; };

    // ---- q: lane (column, h) holds dims 16s + 8h + i (s < 16, i < 8), the B operand of the 32x32x16
    // MFMA. Wave w DMAs the f16 q rows of its own 32 columns (two 512-byte rows an instruction, chunk
    // n32 of a row from logical chunk n32 ^ (row % 32)) into the LDS stage that tile t0 + 1 takes over
    // later, then reads them back in that layout; rows past the block's last token read as zeros.
    // (A tree's second operand, what f16 leaves of q, goes straight into registers, and the first too where that stage is not
    // free or rows are longer. Outputs are 2.1 to 2.6e-4 off 64 bits instead of 4.2 to 5.2e-4 with q in f16, where an f16 output
    // alone is 2.1e-4; 16 long histories take 71 us for 65.7, one short one 10.2 for 8.4.)
    half8 qf[16], ql[TREE ? 16 : 1];
    int entry1, gone0, gone1 = 0;  // tile t + 1's page, the 16-row groups of tiles t and t + 1 without one
    {
        const rsrc_t rq = make_rsrc(a.q16 + ((size_t)row0 + qb * BQ) * a.n_q_heads * HD, (uint32_t)min(BQ, S - qb * BQ) * a.n_q_heads * ROWB);
        char* qs = lds + ((t0 + 1) & 1) * 2 * TILEB;
        pages.load(a.t, wu.b, wg_lo + t0 * KT, wave / PAIR, lane);
        const int qo = (pl * a.n_q_heads + kh * G + hh) * ROWB + 2 * d0 + 16 * h;
        if constexpr (TREE) {
            const rsrc_t rl = make_rsrc(a.q16_lo + ((size_t)row0 + qb * BQ) * a.n_q_heads * HD, (uint32_t)min(BQ, S - qb * BQ) * a.n_q_heads * ROWB);
#pragma unroll
            for (int s = 0; s < 16; ++s) ql[s] = bload_h8(rl, qo + 32 * s);
        }
        if constexpr (STAGED) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int r = 32 * wave + 2 * j + h;  // column of the row this lane moves
                const int qr = ((r / G) * a.n_q_heads + kh * G + r % G) * ROWB + 16 * (n32 ^ (r & 31));
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rq, (__attribute__((address_space(3))) void*)(qs + (32 * wave + 2 * j) * ROWB),
                                                         16, qr, 0, 0, 0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 16; ++s) qf[s] = bload_h8(rq, qo + 32 * s);
        }
        entry1 = wu.page[0];  // this wave's group
        gone0 = 0;
#pragma unroll
        for (int i = 0; i < KT / 16; ++i) {
            entry1 = i == wave / PAIR ? wu.page[i] : entry1;
            gone0 |= page_ok(a.t, wu.page[i]) ? 0 : 1 << i;
        }
        if (t0 < t1) {  // tile t0: of the block's first tile, rows in front of the first attended key read as zeros
            const rsrc_t rk = tile_rows(a.kc, t0, entry1), rv = tile_rows(a.vc, t0, entry1);
            const int skip = first - (wg_lo + t0 * KT + 16 * (wave / PAIR));
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                dma(rk, tile_k(t0), j, row_of(j) < skip ? kNoRow : k_off(j));
                dma(rv, tile_v(t0), j, row_of(j) < skip ? kNoRow : v_off(j));
            }
            if constexpr (K32) {
                const rsrc_t rkl = tile_rows(kc_lo, t0, entry1);
#pragma unroll
                for (int j = 0; j < 8; ++j) dma(rkl, tile_k_lo(), j, row_of(j) < skip ? kNoRow : k_off(j));
            }
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        if constexpr (STAGED) {
            const char* qrow = qs + c * ROWB;
#pragma unroll
            for (int s = 0; s < 16; ++s) qf[s] = *reinterpret_cast<const half8*>(qrow + 16 * ((2 * s + h) ^ n32));
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // stage free for tile t0 + 1's DMA
        }
        if constexpr (TREE) {
#pragma unroll
            for (int s = 0; s < 16; ++s) asm volatile("" : "+v"(ql[s]));
        }
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
    int lo_max = 0;  // tree: the last column's first attended key of the history
    if constexpr (TREE) {
        lo_max = col_lo;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) lo_max = max(lo_max, __shfl_xor(lo_max, d));
        lo_max = __builtin_amdgcn_readfirstlane(lo_max);
    }
    // tree: the word of tile t for this lane's column, if the tile holds rows of the call
    const auto tree_word = [&](int t) {
        unsigned long long w = ~0ull;
        if constexpr (TREE) {
            const int kb = wg_lo + t * KT;
            if (t < t1 && kb + KT > start_pos) {
                const unsigned long long* row = a.bits + (size_t)(row0 + s_idx) * a.words;
                if constexpr (KT == 64) w = row[(kb - (start_pos & ~63)) >> 6];
                else w = reinterpret_cast<const uint32_t*>(row)[(kb - (start_pos & ~63)) >> 5];
            }
        }
        return w;
    };

    float16v oacc[8];  // O^T[d0 + 32dt + 8(r/4) + 4h + r%4][column]
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

    // A tile's scores, S^T = K . Q^T: two 32-key sub-tiles (hd 512: one), 16 k-steps of 16 dims, the two accumulator
    // chains in turn (a chain of dependent MFMAs issues at half rate).
    // Masks of tile t's scores: key kb + 4h + 32kt + 8(r/4) + r%4 of this lane's column; tiles inside every
    // column's range skip it.
    auto mask = [&](int t, int gone, unsigned long long word, float16v (&sc)[NS]) {
        const int kb = wg_lo + t * KT;
        if constexpr (TREE) {
            if (kb + KT > start_pos) {
                const uint32_t w[2] = {(uint32_t)word >> (4 * h), (uint32_t)(word >> 32) >> (4 * h)};
#pragma unroll
                for (int kt = 0; kt < NS; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[kt][r] = w[kt] >> (8 * (r >> 2) + (r & 3)) & 1 ? sc[kt][r] : kNegInf;
            } else if (a.window > 0 && kb < lo_max) {
                const int rel_lo = col_lo - (kb + 4 * h);
#pragma unroll
                for (int kt = 0; kt < NS; ++kt)
#pragma unroll
                    for (int r = 0; r < 16; ++r) sc[kt][r] = 32 * kt + 8 * (r >> 2) + (r & 3) >= rel_lo ? sc[kt][r] : kNegInf;
            }
        } else if ((kb + KT - 1 > wp0) || (a.window > 0 && kb < wp1 + 1 - a.window)) {
            const int rel_hi = pos - (kb + 4 * h), rel_lo = col_lo - (kb + 4 * h);
#pragma unroll
            for (int kt = 0; kt < NS; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int o = 32 * kt + 8 * (r >> 2) + (r & 3);
                    sc[kt][r] = (o <= rel_hi && o >= rel_lo) ? sc[kt][r] : kNegInf;
                }
        }
        if (gone) {
#pragma unroll
            for (int kt = 0; kt < NS; ++kt)
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
    // Where the next scores are LATE, P.V comes before the other wave's half, masks and maxima.
    float mnext = kNegInf;  // this lane's maximum of the scores of the next tile
    // operands of k-step s of a K tile
    const auto read_k = [&](const char* K, int s, half8 (&kr)[NS]) {
        const int cb = 16 * ((2 * s + d0 / 8 + h) ^ n32);
#pragma unroll
        for (int n = 0; n < NS; ++n) {
            const half8* p = reinterpret_cast<const half8*>(K + (n32 + 32 * n) * ROWB + cb);
            kr[n] = K32 ? read_h8(p) : *p;
        }
    };
    // K32: S += K_lo . Q_hi. f(s) issues what is fetched meanwhile.
    const auto add_lo = [&](float16v (&sc)[NS], auto f) {
        half8 kr[3][NS];
        float16v alt = float16v{};  // one sub-tile: every other step, so that two chains take turns
        read_k(tile_k_lo(), 0, kr[0]);
        read_k(tile_k_lo(), 1, kr[1]);
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            if (s + 2 < 16) read_k(tile_k_lo(), s + 2, kr[(s + 2) % 3]);
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                if (NS == 1 && (s & 1)) alt = mfma32(kr[s % 3][n], qf[s], alt);
                else sc[n] = mfma32(kr[s % 3][n], qf[s], sc[n]);
            }
            f(s);
            __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (NS == 1) sc[0] += alt;
    };
    float* const xch = reinterpret_cast<float*>(lds + 2 * 2 * TILEB);
    const auto give = [&](const float16v& sc) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4v*>(xch + ((wave * 4 + j) * 64 + lane) * 4) = float4v{sc[4 * j], sc[4 * j + 1], sc[4 * j + 2], sc[4 * j + 3]};
    };
    // barriers that do not wait, as __syncthreads would, for the tiles on their way: for none, for all but the last (eight DMAs)
    const auto meet = [] { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // (which counts on the order that they were issued in: each kind in a phase of its own, or behind this)
    const auto in_order = [] { asm volatile("" ::: "memory"); __builtin_amdgcn_sched_barrier(0); };
    const auto meet_but_last = [] { asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    const auto take_other = [&](float16v& sc) {  // (a + b is b + a: both waves have the same scores)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float4v v = read_f4(xch + (((wave ^ 2) * 4 + j) * 64 + lane) * 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[4 * j + e] += v[e];
        }
    };
    auto tile = [&](int t, float16v (&sacc)[NS], float16v (&snext)[NS]) {
        if constexpr (K32) {
            meet_but_last();  // V(t) and K(t + 1) are in LDS, its low tile on its way; V(t - 1) fully consumed
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's part of V(t) and K(t + 1) is in LDS
            __syncthreads();                                    // all parts; K(t) and V(t - 1) fully consumed
        }
        const int gone = gone1, entry = entry1;  // of tile t + 1
        const unsigned long long word = tree_word(t + 1);
        {
            const int j = (t + 2 - t0) & 63;
            if (j == 0) pages.load(a.t, wu.b, wg_lo + (t + 2) * KT, wave / PAIR, lane);
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
        half8 pb[2 * NS], pl[K32 ? 2 * NS : 1];
        float ps = 0.0f;
        const rsrc_t rv = tile_rows(a.vc, t + 1, entry), rk = tile_rows(a.kc, t + 2, entry1);
        {
            half8 kr[3][NS];
            // exponentials NS s .. of the lane's 16 NS in three stages
            float ex[2][NS], ev[2][NS];
            auto arg = [&](int s) {
#pragma unroll
                for (int e = 0; e < NS; ++e) ex[s & 1][e] = __builtin_fmaf(sacc[(NS * s + e) >> 4][(NS * s + e) & 15], a.scale_log2, -msub);
            };
            auto expo = [&](int s) {
#pragma unroll
                for (int e = 0; e < NS; ++e) ev[s & 1][e] = fexp2(ex[s & 1][e]);
            };
            auto take = [&](int s) {
#pragma unroll
                for (int e = 0; e < NS; ++e) {
                    const half_t p = (half_t)ev[s & 1][e];
                    pb[(NS * s + e) >> 3][(NS * s + e) & 7] = p;
                    // (a tree's sum is of the weights as they enter the product: the leading ones' roundings cancel, f16 caches 2.9 ->
                    // 2.6e-4 off in the same time)
                    ps += TREE && !K32 ? (float)p : ev[s & 1][e];
                    if constexpr (K32) pl[(NS * s + e) >> 3][(NS * s + e) & 7] = (half_t)(ev[s & 1][e] - (float)p);
                }
            };
            read_k(tile_k(t + 1), 0, kr[0]);
            read_k(tile_k(t + 1), 1, kr[1]);
            arg(0);
#pragma unroll
            for (int n = 0; n < NS; ++n) snext[n] = float16v{};
            float16v alt = float16v{};  // one sub-tile: the products with q's low operand
#pragma unroll
            for (int s = 0; s < 16; ++s) {
                if (s + 2 < 16) read_k(tile_k(t + 1), s + 2, kr[(s + 2) % 3]);
                snext[0] = mfma32(kr[s % 3][0], qf[s], snext[0]);
                expo(s);
                if (s > 0) take(s - 1);
                if constexpr (NS == 2) snext[1] = mfma32(kr[s % 3][1], qf[s], snext[1]);
                if constexpr (TREE && NS == 2) snext[0] = mfma32(kr[s % 3][0], ql[s], snext[0]);
                if constexpr (TREE && NS == 1) alt = mfma32(kr[s % 3][0], ql[s], alt);
                if (s < 15) arg(s + 1);
                if constexpr (TREE && NS == 2) snext[1] = mfma32(kr[s % 3][1], ql[s], snext[1]);
                if (s < 8) dma(rv, tile_v(t + 1), s, v_off(s));
                else if (!K32) dma(rk, tile_k(t + 2), s - 8, k_off(s - 8));
                __builtin_amdgcn_sched_barrier(0);
            }
            take(15);
            if constexpr (NS == 1) snext[0] += alt;
        }
        l_run += ps;
        // (here, not where they are used behind the masks' branches: the compiler would sink them there)
#pragma unroll
        for (int u = 0; u < 2 * NS; ++u) {
            asm volatile("" : "+v"(pb[u]));
            if constexpr (K32) asm volatile("" : "+v"(pl[u]));
        }
        asm volatile("" : "+v"(l_run));
        if constexpr (K32) {
            meet_but_last();  // K(t + 1)'s low tile is in LDS, V(t + 1) on its way; its high tile fully consumed
            add_lo(snext, [&](int s) {
                if (s < 8) dma(rk, tile_k(t + 2), s, k_off(s));
            });
            if constexpr (PAIR == 2) give(snext[0]);
            meet();  // the low tile fully consumed, both halves there
            if constexpr (PAIR == 2) take_other(snext[0]);
        }
        if constexpr (LATE) give(snext[0]);
        else if (t + 1 < t1) mask(t + 1, gone, word, snext);

        // O^T += V^T . P^T over four 16-key steps (hd 512: two); k-slot i < 4 is key 16u + 4h + i, i >= 4 is key
        // 16u + 8 + 4h + i - 4, matching the S^T accumulator rows in pb. Transposed V reads (two an
        // MFMA) kPvAhead MFMAs ahead.
        {
            constexpr int N = 16 * NS;
            const char* V = tile_v(t);
            half8 av[kPvAhead + 1];
            auto read_v = [&](int i) {
                const int u = i >> 3, ch = 4 * (i & 7) + d0 / 8 + vc0;
                const char* vp = V + (16 * u + vr0) * ROWB + 16 * (ch ^ vsw) + vb0;
                const half4 lo = read_tr16(reinterpret_cast<const half_t*>(vp));
                const half4 hi = read_tr16(reinterpret_cast<const half_t*>(vp + 8 * ROWB));
                av[i % (kPvAhead + 1)] = half8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
            mnext = kNegInf;
            const rsrc_t rkl = K32 ? tile_rows(kc_lo, t + 2, entry1) : rk;
#pragma unroll
            for (int i = 0; i < kPvAhead; ++i) read_v(i);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                // (the remainders' products one behind, so that no two in turn have the same sum)
                if (K32 && i > 0) mfma32_acc(oacc[(i - 1) & 7], av[(i - 1) % (kPvAhead + 1)], pl[(i - 1) >> 3]);
                if (i + kPvAhead < N) read_v(i + kPvAhead);
                mfma32_acc(oacc[i & 7], av[i % (kPvAhead + 1)], pb[i >> 3]);
                constexpr int I0 = 4 * NS;
                if (!LATE && i >= I0 && i < 3 * I0)
                    mnext = fmaxf(mnext, fmaxf(snext[(i - I0) >> 3][2 * ((i - I0) & 7)], snext[(i - I0) >> 3][2 * ((i - I0) & 7) + 1]));
                if (K32 && i < 8) dma(rkl, tile_k_lo(), i, k_off(i));
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (K32) mfma32_acc(oacc[(N - 1) & 7], av[(N - 1) % (kPvAhead + 1)], pl[(N - 1) >> 3]);
            asm volatile("" : "+v"(mnext));
        }
        if constexpr (LATE) {
            meet();  // both halves are there
            take_other(snext[0]);
            if (t + 1 < t1) mask(t + 1, gone, word, snext);
#pragma unroll
            for (int n = 0; n < NS; ++n)
#pragma unroll
                for (int r = 0; r < 16; ++r) mnext = fmaxf(mnext, snext[n][r]);
        }
    };
    // A wave without a token (trees are short) moves its rows and leaves LDS and the matrix units to the others. It
    // meets every barrier that those meet.
    if (TREE && qb * BQ + 32 * cg / G >= S) {
        if (t0 < t1) {
            const auto fetch = [&](const void* pool, char* dst, int t, int entry, bool v) {
                const rsrc_t r = tile_rows(pool, t, entry);
#pragma unroll
                for (int i = 0; i < 8; ++i) dma(r, dst, i, v ? v_off(i) : k_off(i));
            };
            __syncthreads();                                 // K(t0), V(t0)
            if constexpr (K32 || PAIR == 2) __syncthreads();  // the scores of t0
            entry1 = __builtin_amdgcn_readlane(pages.entry, 1);
            fetch(a.kc, tile_k(t0 + 1), t0 + 1, entry1, false);
            in_order();
            if constexpr (K32) fetch(kc_lo, tile_k_lo(), t0 + 1, entry1, false);
            for (int t = t0; t < t1; ++t) {
                if constexpr (K32) {
                    meet_but_last();
                } else {
                    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                    __syncthreads();
                }
                const int j = (t + 2 - t0) & 63, entry = entry1;
                if (j == 0) pages.load(a.t, wu.b, wg_lo + (t + 2) * KT, wave / PAIR, lane);
                entry1 = __builtin_amdgcn_readlane(pages.entry, j);
                fetch(a.vc, tile_v(t + 1), t + 1, entry, true);
                if constexpr (K32) meet_but_last();
                fetch(a.kc, tile_k(t + 2), t + 2, entry1, false);
                if constexpr (K32 || PAIR == 2) meet();
                if constexpr (K32) fetch(kc_lo, tile_k_lo(), t + 2, entry1, false);
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        if (sizeof(OUTT) == 2 && n_pieces == 1) __syncthreads();  // the epilogue's
        return;
    }
    if (t0 < t1) {
        float16v sa[NS], sb[NS];
#pragma unroll
        for (int n = 0; n < NS; ++n) sa[n] = float16v{};
        __syncthreads();  // K(t0), V(t0); every wave has its q
        entry1 = __builtin_amdgcn_readlane(pages.entry, 1);
        gone1 = __builtin_amdgcn_readlane(pages.gone, 1);
        const rsrc_t rk = tile_rows(a.kc, t0 + 1, entry1);
        const auto next_k = [&] {
#pragma unroll
            for (int j = 0; j < 8; ++j) dma(rk, tile_k(t0 + 1), j, k_off(j));
            if constexpr (K32) {
                in_order();
                const rsrc_t rkl = tile_rows(kc_lo, t0 + 1, entry1);
#pragma unroll
                for (int j = 0; j < 8; ++j) dma(rkl, tile_k_lo(), j, k_off(j));
            }
        };
        if constexpr (!K32) next_k();
#pragma unroll
        for (int s = 0; s < 16; ++s) {
            half8 kr[NS];
            read_k(tile_k(t0), s, kr);
#pragma unroll
            for (int n = 0; n < NS; ++n) sa[n] = mfma32(kr[n], qf[s], sa[n]);
            if constexpr (TREE) {
#pragma unroll
                for (int n = 0; n < NS; ++n) sa[n] = mfma32(kr[n], ql[s], sa[n]);
            }
        }
        if constexpr (K32) add_lo(sa, [](int) {});
        if constexpr (PAIR == 2) give(sa[0]);
        if constexpr (K32 || PAIR == 2) __syncthreads();  // K(t0) fully consumed, both halves there
        if constexpr (K32) next_k();
        if constexpr (PAIR == 2) take_other(sa[0]);
        mask(t0, gone0, tree_word(t0), sa);
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int n = 0; n < NS; ++n) mnext = fmaxf(mnext, sa[n][r]);
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
        if (TREE && !col_ok) return;  // few tokens: columns of none move no bytes
        const float inv_p = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) store_part<true, 256, NCOL * HD>(a.part_o, true, wu.slot, wave, dt, lane, oacc[dt], inv_p);
        if (h == 0 && d0 == 0) a.part_ml[(size_t)wu.slot * NCOL + c] = make_float2(m_use, l_tot);
        return;
    }
    const float inv = l_tot > 0.0f ? 1.0f / l_tot : 0.0f;
    if constexpr (sizeof(OUTT) == 2) {
        // f16 rows through LDS: each wave stages its 32 output rows' 256 dims (528-byte stride: the
        // 8-byte writes of a store instruction fall on distinct banks), then stores two whole
        // 512-byte rows an instruction. Written straight from the accumulator layout, every
        // store instruction put 16 bytes into each of 32 rows.
        constexpr int OSTR = 256 * 2 + 16;
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
            const int rr = 2 * i + h, cc = 32 * cg + rr;  // lanes 32h..: the wave's row rr
            const int so = qb * BQ + cc / G;
            const half8 val = *reinterpret_cast<const half8*>(ost + rr * OSTR + 16 * n32);
            if (so < S)
                *reinterpret_cast<half8*>(reinterpret_cast<half_t*>(a.out) +
                                          ((size_t)(row0 + so) * a.n_q_heads + kh * G + cc % G) * HD + d0 + 8 * n32) = val;
        }
    } else if (col_ok) {
        OUTT* orow = reinterpret_cast<OUTT*>(a.out) + ((size_t)(row0 + s_idx) * a.n_q_heads + kh * G + hh) * HD + d0;
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

}  // namespace g4a
