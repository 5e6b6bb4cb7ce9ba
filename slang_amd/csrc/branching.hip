// What a server does with a paged cache once a sequence has branched: the walk that accepts drafts (g4a_tree_accept), the
// accepted rows moved up to where plain steps would have put them (g4a_paged_keep), and the tables, pages and rows of
// beams that follow their parents (g4a_paged_fork). Whole numbers and copies: nothing here is rounded, and every
// result is the same whatever order the workgroups run in.
#include <algorithm>

#include "paged.hpp"

namespace g4a {

typedef unsigned uint4v __attribute__((ext_vector_type(4)));

__device__ __forceinline__ SeqRows tree_rows(const PageTab& t, const int32_t* cu, int n_tokens, int b) {
    return cut_tree(seq_rows(t, cu, n_tokens, b));
}

// ---------------------------------------------------------------- accepting drafts
struct AcceptArgs {
    const int32_t* cu;
    const int32_t* parents;
    const int32_t* drafts;
    const int32_t* targets;
    const int32_t* key_len;
    int32_t* path;
    int32_t* n_path;
    int32_t* next;
    int32_t* kept;
    int n_tokens, n_seq, max_path;
};

// path[0] = 0; then, while there is one, the first child c of the last token whose draft is the last token's target. Children
// follow their parents, so one pass over the tokens finds the whole path: a wave a sequence, 64 tokens a ballot, 256
// tokens' loads at once. Latency: cu, then the tokens, then the stores.
__global__ __launch_bounds__(256) void tree_accept_kernel(AcceptArgs a) {
    const int lane = threadIdx.x & 63, b = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (b >= a.n_seq) return;
    const SeqRows all = cut_rows(a.cu[b], a.cu[b + 1], a.n_tokens, a.key_len[b]), r = cut_tree(all);
    const int n = r.hi - r.lo;
    int32_t* path = a.path + (size_t)b * a.max_path;
    int count = 0, cur = -1, want = -1;
    for (int base = 0; base < n; base += 256) {
        int par[4], draft[4], target[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = base + 64 * i + lane;
            const bool in = k < n;
            par[i] = in ? a.parents[r.lo + k] : -1;
            draft[i] = in ? a.drafts[r.lo + k] : 0;
            target[i] = in ? a.targets[r.lo + k] : 0;
        }
        if (base == 0) {
            cur = 0;
            want = __builtin_amdgcn_readfirstlane(target[0]);
            count = 1;
            if (lane == 0) path[0] = 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int k = base + 64 * i + lane;
            while (count < a.max_path) {
                const unsigned long long m = __ballot(k < n && k > cur && par[i] == cur && draft[i] == want);
                if (!m) break;
                const int l = __builtin_ctzll(m);
                cur = base + 64 * i + l;
                want = __builtin_amdgcn_readlane(target[i], l);
                if (lane == 0) path[count] = cur;
                ++count;
            }
        }
    }
    for (int k = count + lane; k < a.max_path; k += 64) path[k] = -1;
    if (lane == 0) {
        a.n_path[b] = count;
        a.next[b] = want;
        a.kept[b] = all.keys - (all.hi - all.lo) + count;
    }
}

// ---------------------------------------------------------------- keeping the accepted rows
constexpr int kPools = 64;  // G4A_POOLS_MAX
struct Pools {
    g4a_pool at[kPools];
};

struct KeepArgs {
    PageTab t;
    const int32_t* cu;
    const int32_t* path;
    const int32_t* n_path;
    int n_tokens, max_path;
};

// Row start + path[d] of a sequence to row start + d, in every pool. path ascends, so path[d] >= d and a row is read
// for the last time before it is written: a workgroup holds as many rows of its columns in registers as fit, stores
// them, and goes on. A workgroup per sequence, pool and 4 KB of a row's bytes; bound by the chain cu -> path -> table
// -> rows.
__global__ __launch_bounds__(256) void paged_keep_kernel(KeepArgs a, Pools pools) {
    constexpr int kPart = 4096, kRegs = 4;
    __shared__ int64_t s_src[kTreeMax], s_dst[kTreeMax];
    __shared__ int s_n;
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63;
    const g4a_pool pool = pools.at[blockIdx.y];
    const int64_t part0 = (int64_t)blockIdx.z * kPart;
    if (part0 >= pool.row_bytes) return;
    const SeqRows r = tree_rows(a.t, a.cu, a.n_tokens, b);
    const int n = r.hi - r.lo, start = r.keys - n;
    const int want = min(min(a.n_path[b], a.max_path), n);
    if (tid < 64) {  // where the rows are; the path ends at the first entry that is no token behind the one before
        int m = 0;
        for (int d0 = 0; d0 < want; d0 += 64) {
            const int d = d0 + lane;
            int from = -1, before = -1;
            if (d < want) {
                from = a.path[(size_t)b * a.max_path + d];
                if (d > 0) before = a.path[(size_t)b * a.max_path + d - 1];
            }
            const unsigned long long bad = __ballot(d < want && !(from > before && from >= 0 && from < n));
            const int ok = bad ? __builtin_ctzll(bad) : min(64, want - d0);
            if (lane < ok) {
                int64_t src = -1, dst = -1;
                if (from != d && start + d >= 0) {
                    const int ps = page_at(a.t, b, start + from), pd = page_at(a.t, b, start + d);
                    if (page_ok(a.t, ps) && page_ok(a.t, pd)) {
                        src = (int64_t)paged_row(a.t, ps, start + from, 1);
                        dst = (int64_t)paged_row(a.t, pd, start + d, 1);
                    }
                }
                s_src[d] = src;
                s_dst[d] = dst;
            }
            m = d0 + ok;
            if (bad) break;
        }
        if (lane == 0) s_n = m;
    }
    __syncthreads();
    const int m = s_n;
    const int cols = (int)(min((int64_t)kPart, pool.row_bytes - part0) / 16);  // 16-byte chunks of a row's part
    char* base = reinterpret_cast<char*>(pool.rows) + part0;
    const int rows = max(kRegs * 256 / cols, 1);  // rows in registers at a time
    for (int d0 = 0; d0 < m; d0 += rows) {
        const int items = min(rows, m - d0) * cols;
        uint4v x[kRegs];
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
            const int k = tid + 256 * i, d = d0 + k / cols;
            if (k < items && s_src[d] >= 0) x[i] = *reinterpret_cast<const uint4v*>(base + s_src[d] * pool.row_bytes + 16 * (k % cols));
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kRegs; ++i) {
            const int k = tid + 256 * i, d = d0 + k / cols;
            if (k < items && s_src[d] >= 0) *reinterpret_cast<uint4v*>(base + s_dst[d] * pool.row_bytes + 16 * (k % cols)) = x[i];
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------- forking
struct ForkArgs {
    PageTab t;  // the tables that are followed; cols is all of them here
    const int32_t* parent;
    const int32_t* free_in;
    const int32_t* n_free_in;
    int32_t* table;    // [n_new][cols]
    int32_t* len;
    int32_t* free_out;
    int32_t* n_free_out;
    int32_t* copy;     // [3][n_new]: a row's tail: from page, to page, rows
    int n_new, room, words;
};

// key rows of new row j: its parent's
__device__ __forceinline__ int fork_len(const ForkArgs& a, int p) { return (unsigned)p < (unsigned)a.t.n_seq ? paged_len(a.t, p) : 0; }
// columns [full, end) of a row of L keys are the ones that the row will write to
__device__ __forceinline__ int fork_end(const ForkArgs& a, int p, int L) {
    if ((unsigned)p >= (unsigned)a.t.n_seq) return 0;
    const int64_t end = ((int64_t)L + a.room + (1 << a.t.shift) - 1) >> a.t.shift;
    return (int)min(end, (int64_t)a.t.cols);
}
__device__ __forceinline__ bool bit(const uint32_t* map, int p) { return map[p >> 5] >> (p & 31) & 1; }
__device__ __forceinline__ void set_bit(uint32_t* map, int p) { atomicOr(map + (p >> 5), 1u << (p & 31)); }

// The marks of a call's pages: in the workspace, or in LDS where one workgroup does all of it.
struct ForkMarks {
    int32_t* owner;   // the first new row that has the page in a column it will write to
    uint32_t* was;    // bits: some old row has it;
    uint32_t* held;   //   some new row has it;
    uint32_t* full;   //   some new row has it in a column that is full
};

// Column c of new row j, whose parent has page x there: a full one is the parent's, one that the row will write to is
// claimed
__device__ __forceinline__ void mark_new(const ForkArgs& a, const ForkMarks& mk, int j, int full, int end, int c, int x) {
    int e = -1;
    if (c < end && page_ok(a.t, x)) {
        if (c < full) {
            set_bit(mk.held, x);
            set_bit(mk.full, x);
            e = x;
        } else {
            atomicMin(mk.owner + x, j);
        }
    }
    a.table[(size_t)j * a.t.cols + c] = e;
}

// The writable columns, in order of rows and columns, by one workgroup, once all is marked: a page that no other row holds
// stays, the others take pages off the end of the free list, to which the pages that no row holds any more are added
// first.
constexpr int kForkThreads = 1024;
__device__ __forceinline__ void fork_pages(const ForkArgs& a, const ForkMarks& mk) {
    __shared__ int s_wave[kForkThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // exclusive prefix of x over the workgroup, and the total
    auto scan = [&](int x, int& total) {
        const int incl = wave_scan(x);
        __syncthreads();
        if (lane == 63) s_wave[wave] = incl;
        __syncthreads();
        int before = 0;
        total = 0;
#pragma unroll
        for (int w = 0; w < kForkThreads / 64; ++w) {
            if (w < wave) before += s_wave[w];
            total += s_wave[w];
        }
        return before + incl - x;
    };
    // f(column, the parent's page there or -1, whether the row keeps it, whether it needs another) over row j of parent p
    auto columns = [&](int j, int p, int L, auto f) {
        const int end = fork_end(a, p, L);
        for (int c = L >> a.t.shift; c < end; ++c) {
            int x = a.t.table[(size_t)p * a.t.stride + c];
            if (!page_ok(a.t, x)) x = -1;
            const bool keeps = x >= 0 && !bit(mk.full, x) && mk.owner[x] == j;
            // (keys whose page is not there stay lost: a new page there would make them rows of anything)
            f(c, x, keeps, !keeps && (x >= 0 || (int64_t)c << a.t.shift >= L));
        }
    };
    const int chunks = (a.n_new + kForkThreads - 1) / kForkThreads;
    const int had = min(max(a.n_free_in[0], 0), a.t.n_pages);
    for (int i = tid; i < had; i += kForkThreads) a.free_out[i] = a.free_in[i];
    // a workgroup's barrier alone does not wait for stores and atomics to reach memory, where the others read them
    auto reached = [] {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    int p = -1, L = 0, need = 0;  // of this thread's row; of the only chunk, if there is one
    for (int ch = 0; ch < chunks; ++ch) {
        const int j = ch * kForkThreads + tid;
        if (j >= a.n_new) break;
        p = a.parent[j];
        L = fork_len(a, p);
        need = 0;
        columns(j, p, L, [&](int c, int x, bool keeps, bool needs) {
            need += needs;
            if (keeps) {
                a.table[(size_t)j * a.t.cols + c] = x;
                set_bit(mk.held, x);
            }
        });
    }
    reached();
    int m = had;
    for (int w0 = 0; w0 < a.words; w0 += kForkThreads) {
        const int w = w0 + tid;
        uint32_t gone = w < a.words ? __hip_atomic_load(mk.was + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) &
                                          ~__hip_atomic_load(mk.held + w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)
                                    : 0u;
        int total;
        int at = m + scan(__builtin_popcount(gone), total);
        for (; gone; gone &= gone - 1, ++at)
            if (at < a.t.n_pages) a.free_out[at] = 32 * w + __builtin_ctz(gone);  // (a list with pages in use could overflow)
        m += total;
    }
    m = min(m, a.t.n_pages);
    reached();
    int taken = 0;
    for (int ch = 0; ch < chunks; ++ch) {
        const int j = ch * kForkThreads + tid;
        if (chunks > 1) {
            need = 0;
            p = j < a.n_new ? a.parent[j] : -1;
            L = fork_len(a, p);
            if (j < a.n_new) columns(j, p, L, [&](int, int, bool, bool needs) { need += needs; });
        }
        int total;
        int k = taken + scan(need, total);
        if (j < a.n_new) {
            int from = -1, to = -1, rows = 0;
            if (need > 0)
                columns(j, p, L, [&](int c, int x, bool, bool needs) {
                    if (!needs) return;
                    const int at = m - 1 - k++;
                    int got = -1;
                    if (at >= 0) got = a.free_out[at];
                    if (!page_ok(a.t, got)) got = -1;
                    a.table[(size_t)j * a.t.cols + c] = got;
                    const int fill = L - (c << a.t.shift);
                    if (fill > 0) {  // the parent's last page, partly filled
                        from = x;
                        to = got;
                        rows = got >= 0 ? fill : 0;
                    }
                });
            a.copy[j] = from;
            a.copy[a.n_new + j] = to;
            a.copy[2 * a.n_new + j] = rows;
        }
        taken += total;
    }
    reached();
    const int left = max(m - taken, 0);
    for (int i = left + tid; i < a.t.n_pages; i += kForkThreads) a.free_out[i] = -1;
    if (tid == 0) a.n_free_out[0] = left;
}

// All of it by one workgroup, the marks in LDS, which holds those of 12288 pages, where table entries are few. A call without
// copies in a graph, against the three launches: 4 rows of 11 columns 5.5 and 8.7 us (with 12288 pages 7.2 and 9.9), 128 of
// 67 12.4 and 13.5, 256 of 67 (34304 entries) 19.0 and 18.3, 512 of 66 26.3 and 23.3, 1024 of 66 45.9 and 24.7, 64 of 1000 26.7 and
// 20.6. (Beyond, the free list is one workgroup's still: 500000 pages, most of them free, take 89 us.)
constexpr int kForkPages = 12288, kForkEntries = 1 << 15, kForkRows = 1024;
__global__ __launch_bounds__(kForkThreads) void fork_small_kernel(ForkArgs a) {
    __shared__ int32_t s_owner[kForkPages];
    __shared__ uint32_t s_bits[3][kForkPages / 32];
    const ForkMarks mk{s_owner, s_bits[0], s_bits[1], s_bits[2]};
    __shared__ int s_parent[kForkRows], s_full[kForkRows], s_end[kForkRows];
    constexpr int NW = kForkThreads / 64, U = 4;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, cols = a.t.cols;
    if (tid < a.n_new) {
        const int p = a.parent[tid], L = fork_len(a, p), end = fork_end(a, p, L);
        a.len[tid] = L;
        s_parent[tid] = end > 0 ? p : 0;  // (a row that is not read)
        s_full[tid] = L >> a.t.shift;
        s_end[tid] = end;
    }
    for (int i = tid; i < a.t.n_pages; i += kForkThreads) s_owner[i] = 0x7fffffff;
    for (int i = tid; i < a.words; i += kForkThreads) s_bits[0][i] = s_bits[1][i] = s_bits[2][i] = 0;
    __syncthreads();
    for (int c0 = 0; c0 < cols; c0 += 64) {  // a wave a row, the entries of eight rows' loads at once
        const int c = c0 + lane;
        for (int r0 = wave; r0 < max(a.t.n_seq, a.n_new); r0 += NW * U) {
            int was[U], heir[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + NW * u;
                was[u] = r < a.t.n_seq && c < cols ? a.t.table[(size_t)r * a.t.stride + c] : -1;
                heir[u] = r < a.n_new && c < s_end[r] ? a.t.table[(size_t)s_parent[r] * a.t.stride + c] : -1;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int r = r0 + NW * u;
                if (page_ok(a.t, was[u])) set_bit(mk.was, was[u]);
                if (r < a.n_new && c < cols) mark_new(a, mk, r, s_full[r], s_end[r], c, heir[u]);
            }
        }
    }
    __syncthreads();
    fork_pages(a, mk);
}

__global__ __launch_bounds__(256) void fork_clear_kernel(ForkArgs a, ForkMarks mk) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < a.t.n_pages) mk.owner[i] = 0x7fffffff;
    if (i < a.words) mk.was[i] = mk.held[i] = mk.full[i] = 0;
}
// A workgroup per row of either table
__global__ __launch_bounds__(256) void fork_mark_kernel(ForkArgs a, ForkMarks mk) {
    const int row = blockIdx.x;
    if (row < a.t.n_seq) {
        for (int c = threadIdx.x; c < a.t.cols; c += 256) {
            const int e = a.t.table[(size_t)row * a.t.stride + c];
            if (page_ok(a.t, e)) set_bit(mk.was, e);
        }
        return;
    }
    const int j = row - a.t.n_seq, p = a.parent[j], L = fork_len(a, p), end = fork_end(a, p, L);
    for (int c = threadIdx.x; c < a.t.cols; c += 256)
        mark_new(a, mk, j, L >> a.t.shift, end, c, c < end ? a.t.table[(size_t)p * a.t.stride + c] : -1);
    if (threadIdx.x == 0) a.len[j] = L;
}
__global__ __launch_bounds__(kForkThreads) void fork_pages_kernel(ForkArgs a, ForkMarks mk) { fork_pages(a, mk); }

// The filled rows of the pages that were replaced, in every pool: a workgroup per row, pool and 16 KB
__global__ __launch_bounds__(256) void fork_copy_kernel(ForkArgs a, Pools pools) {
    const int j = blockIdx.x, rows = a.copy[2 * a.n_new + j];
    if (rows <= 0) return;
    const g4a_pool pool = pools.at[blockIdx.y];
    const int64_t n16 = rows * pool.row_bytes / 16, page = pool.row_bytes << a.t.shift;
    const char* src = reinterpret_cast<const char*>(pool.rows) + a.copy[j] * page;
    char* dst = reinterpret_cast<char*>(pool.rows) + a.copy[a.n_new + j] * page;
    for (int64_t i0 = (int64_t)blockIdx.z * 1024; i0 < n16; i0 += (int64_t)gridDim.z * 1024) {
        uint4v x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i0 + 256 * i + threadIdx.x < n16) x[i] = *reinterpret_cast<const uint4v*>(src + 16 * (i0 + 256 * i + threadIdx.x));
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (i0 + 256 * i + threadIdx.x < n16) *reinterpret_cast<uint4v*>(dst + 16 * (i0 + 256 * i + threadIdx.x)) = x[i];
    }
}

// ---------------------------------------------------------------- host side
// Pools of the cache's pages, as the kernels take them. Rows of two pools must not share memory: their copies would race.
static int check_pools(const g4a_pool* pools, int n, const g4a_paged* pg, Pools& out, int64_t& widest) {
    if (n < 0 || n > kPools || (n > 0 && !pools)) {
        set_error("pools: 0 to %d of them (got %d)", kPools, n);
        return G4A_EINVAL;
    }
    widest = 0;
    uintptr_t lo[kPools], hi[kPools];
    for (int i = 0; i < n; ++i) {
        const g4a_pool& p = pools[i];
        if (!p.rows || (uintptr_t)p.rows % 16 || p.row_bytes <= 0 || p.row_bytes % 16 || p.row_bytes > 1 << 20) {
            set_error("pool %d: rows must be non-NULL and 16-byte aligned, row_bytes (%lld) a multiple of 16, at most 2^20", i,
                      (long long)p.row_bytes);
            return G4A_EINVAL;
        }
        lo[i] = (uintptr_t)p.rows;
        hi[i] = lo[i] + (uintptr_t)p.row_bytes * (uintptr_t)pg->n_pages * (uintptr_t)pg->page_size;
        for (int k = 0; k < i; ++k)
            if (lo[i] < hi[k] && lo[k] < hi[i]) {
                set_error("pools %d and %d share memory", k, i);
                return G4A_EINVAL;
            }
        out.at[i] = p;
        widest = std::max(widest, p.row_bytes);
    }
    return G4A_OK;
}

static int check_pool_table(const g4a_paged* pg) {
    if (!pg || !pg->page_table || !pg->key_len || (uintptr_t)pg->page_table % 4 || (uintptr_t)pg->key_len % 4) {
        set_error("pg, page_table and key_len must be non-NULL, both 4-byte aligned");
        return G4A_EINVAL;
    }
    return check_table(pg);
}

static bool bad4(const void* p) { return !p || (uintptr_t)p % 4; }

struct ForkPlan {
    int words;
    size_t was, held, full, copy, total;
};
static ForkPlan fork_plan(const g4a_paged* pg, int n_new) {
    ForkPlan p;
    p.words = (pg->n_pages + 31) / 32;
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.was = al((size_t)pg->n_pages * 4);
    p.held = p.was + al((size_t)p.words * 4);
    p.full = p.held + al((size_t)p.words * 4);
    p.copy = p.full + al((size_t)p.words * 4);
    p.total = p.copy + al((size_t)n_new * 12);
    return p;
}

static int check_new(const g4a_paged* pg, int n_new, int room) {
    if (n_new <= 0 || (int64_t)n_new + pg->n_seq > 0x7fffffff || room < 0 || room > 1 << 30) {
        set_error("n_new (%d) must be positive, room (%d) in [0, 2^30]", n_new, room);
        return G4A_EINVAL;
    }
    return G4A_OK;
}

}  // namespace g4a

using namespace g4a;

extern "C" int g4a_tree_accept(int n_tokens, int n_seq, const int32_t* cu_q, const int32_t* parents, const int32_t* drafts,
                               const int32_t* targets, const int32_t* key_len, int max_path, int32_t* path, int32_t* n_path,
                               int32_t* next, int32_t* kept, void* stream) {
    if (n_tokens <= 0 || n_seq <= 0 || max_path <= 0) {
        set_error("n_tokens (%d), n_seq (%d) and max_path (%d) must be positive", n_tokens, n_seq, max_path);
        return G4A_EINVAL;
    }
    if (bad4(cu_q) || bad4(parents) || bad4(drafts) || bad4(targets) || bad4(key_len) || bad4(path) || bad4(n_path) || bad4(next) ||
        bad4(kept)) {
        set_error("cu_q, parents, drafts, targets, key_len, path, n_path, next and kept must be non-NULL and 4-byte aligned");
        return G4A_EINVAL;
    }
    const AcceptArgs a{cu_q, parents, drafts, targets, key_len, path, n_path, next, kept, n_tokens, n_seq, max_path};
    hipLaunchKernelGGL(tree_accept_kernel, dim3((unsigned)((n_seq + 3) / 4)), dim3(256), 0, (hipStream_t)stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? G4A_OK : hip_error(e, "tree accept launch");
}

extern "C" int g4a_paged_keep(const g4a_pool* pools, int n_pools, const g4a_paged* pg, int n_tokens, const int32_t* cu_q,
                              const int32_t* path, int max_path, const int32_t* n_path, void* stream) {
    if (const int rc = check_pool_table(pg)) return rc;
    Pools ps;
    int64_t widest;
    if (const int rc = check_pools(pools, n_pools, pg, ps, widest)) return rc;
    if (n_tokens <= 0 || max_path <= 0 || bad4(cu_q) || bad4(path) || bad4(n_path)) {
        set_error("n_tokens (%d) and max_path (%d) must be positive, cu_q, path and n_path non-NULL and 4-byte aligned", n_tokens, max_path);
        return G4A_EINVAL;
    }
    if (n_pools == 0) return G4A_OK;
    const KeepArgs a{page_tab(pg), cu_q, path, n_path, n_tokens, max_path};
    hipLaunchKernelGGL(paged_keep_kernel, dim3((unsigned)pg->n_seq, (unsigned)n_pools, (unsigned)((widest + 4095) / 4096)), dim3(256), 0,
                       (hipStream_t)stream, a, ps);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? G4A_OK : hip_error(e, "paged keep launch");
}

extern "C" size_t g4a_paged_fork_ws_bytes(const g4a_paged* pg, int n_new) {
    if (check_pool_table(pg) || check_new(pg, n_new, 0)) return 0;
    return fork_plan(pg, n_new).total;
}

extern "C" int g4a_paged_fork(const g4a_pool* pools, int n_pools, const g4a_paged* pg, int n_new, const int32_t* parent, int room,
                              const int32_t* free_pages, const int32_t* n_free, int32_t* new_table, int32_t* new_len,
                              int32_t* new_free, int32_t* new_n_free, void* ws, size_t ws_bytes, void* stream_) {
    if (const int rc = check_pool_table(pg)) return rc;
    if (const int rc = check_new(pg, n_new, room)) return rc;
    Pools ps;
    int64_t widest;
    if (const int rc = check_pools(pools, n_pools, pg, ps, widest)) return rc;
    if (bad4(parent) || bad4(free_pages) || bad4(n_free) || bad4(new_table) || bad4(new_len) || bad4(new_free) || bad4(new_n_free)) {
        set_error("parent, free_pages, n_free and the outputs must be non-NULL and 4-byte aligned");
        return G4A_EINVAL;
    }
    struct Span {
        const void* p;
        size_t bytes;
    };
    const size_t cols = (size_t)pg->table_cols;
    const Span in[] = {{pg->page_table, ((size_t)(pg->n_seq - 1) * pg->table_stride + cols) * 4}, {pg->key_len, (size_t)pg->n_seq * 4},
                       {parent, (size_t)n_new * 4}, {free_pages, (size_t)pg->n_pages * 4}, {n_free, 4}};
    const Span out[] = {{new_table, (size_t)n_new * cols * 4}, {new_len, (size_t)n_new * 4}, {new_free, (size_t)pg->n_pages * 4},
                        {new_n_free, 4}};
    const auto meet = [](const Span& x, const Span& y) {
        return (uintptr_t)x.p < (uintptr_t)y.p + y.bytes && (uintptr_t)y.p < (uintptr_t)x.p + x.bytes;
    };
    for (int i = 0; i < 4; ++i) {
        for (const Span& x : in)
            if (meet(out[i], x)) {
                set_error("the new table, lengths and free list must not overlap the old ones");
                return G4A_EINVAL;
            }
        for (int k = 0; k < i; ++k)
            if (meet(out[i], out[k])) {
                set_error("two of the outputs overlap");
                return G4A_EINVAL;
            }
    }
    const ForkPlan p = fork_plan(pg, n_new);
    if (!ws || (uintptr_t)ws % 256 || ws_bytes < p.total) {
        set_error("paged fork workspace needs %zu bytes (256-byte aligned), got %zu", p.total, ws ? ws_bytes : (size_t)0);
        return G4A_EWORKSPACE;
    }
    const hipStream_t stream = (hipStream_t)stream_;
    char* w = (char*)ws;
    ForkArgs a;
    a.t = page_tab(pg);
    a.t.cols = pg->table_cols;
    a.parent = parent;
    a.free_in = free_pages;
    a.n_free_in = n_free;
    a.table = new_table;
    a.len = new_len;
    a.free_out = new_free;
    a.n_free_out = new_n_free;
    a.copy = (int32_t*)(w + p.copy);
    a.n_new = n_new;
    a.room = room;
    a.words = p.words;
    const int64_t entries = ((int64_t)pg->n_seq + n_new) * pg->table_cols;
    if (pg->n_pages <= kForkPages && n_new <= kForkRows && entries <= kForkEntries) {
        hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kForkThreads), 0, stream, a);
    } else {
        const ForkMarks mk{(int32_t*)w, (uint32_t*)(w + p.was), (uint32_t*)(w + p.held), (uint32_t*)(w + p.full)};
        hipLaunchKernelGGL(fork_clear_kernel, dim3((unsigned)((pg->n_pages + 255) / 256)), dim3(256), 0, stream, a, mk);
        hipLaunchKernelGGL(fork_mark_kernel, dim3((unsigned)(pg->n_seq + n_new)), dim3(256), 0, stream, a, mk);
        hipLaunchKernelGGL(fork_pages_kernel, dim3(1), dim3(kForkThreads), 0, stream, a, mk);
    }
    hipError_t e;
    if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged fork launch");
    if (n_pools > 0) {
        const int64_t page_parts = std::min<int64_t>(((widest << a.t.shift) + 16383) / 16384, 16);
        hipLaunchKernelGGL(fork_copy_kernel, dim3((unsigned)n_new, (unsigned)n_pools, (unsigned)page_parts), dim3(256), 0, stream, a, ps);
        if ((e = hipGetLastError()) != hipSuccess) return hip_error(e, "paged fork copy launch");
    }
    return G4A_OK;
}
