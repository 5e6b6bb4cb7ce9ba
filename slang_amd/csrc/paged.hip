// The paged K/V cache: the checks that its entry points share, and appending rows.
#include "paged.hpp"

namespace g4a {

static bool aligned16(const void* p) { return (uintptr_t)p % 16 == 0; }
int check_paged(const g4a_cfg* cfg, const g4a_paged* pg, bool need_group_le8) {
    if (!check_cfg(cfg, need_group_le8)) return G4A_EINVAL;
    if (!pg) {
        set_error("pg is NULL");
        return G4A_EINVAL;
    }
    if (!pg->k_pages || !pg->v_pages || !pg->page_table || !pg->key_len) {
        set_error("k_pages, v_pages, page_table and key_len must be non-NULL");
        return G4A_EINVAL;
    }
    if (!aligned16(pg->k_pages) || !aligned16(pg->v_pages) || (uintptr_t)pg->page_table % 4 || (uintptr_t)pg->key_len % 4) {
        set_error("k_pages and v_pages must be 16-byte aligned, page_table and key_len 4-byte aligned");
        return G4A_EINVAL;
    }
    const int ps = pg->page_size;
    if (ps < 16 || ps > 65536 || (ps & (ps - 1))) {
        set_error("page_size must be a power of two of 16 .. 65536 (got %d)", ps);
        return G4A_EUNSUPPORTED;
    }
    if (pg->n_pages <= 0 || pg->n_seq <= 0 || pg->table_cols <= 0 || pg->table_stride < pg->table_cols) {
        set_error("n_pages (%d), n_seq (%d) and table_cols (%d) must be positive, table_stride (%d) at least table_cols",
                  pg->n_pages, pg->n_seq, pg->table_cols, pg->table_stride);
        return G4A_EINVAL;
    }
    if (pg->max_key_len <= 0 || (int64_t)pg->max_key_len > (int64_t)pg->table_cols * ps || pg->max_key_len > 1 << 30) {
        set_error("max_key_len (%d) must be in [1, table_cols * page_size] and at most 2^30", pg->max_key_len);
        return G4A_EINVAL;
    }
    if (pg->reserved[0] || pg->reserved[1]) {
        set_error("g4a_paged's reserved words must be 0");
        return G4A_EINVAL;
    }
    if (cfg->head_dim != 256 && cfg->head_dim != 512) {
        set_error("head_dim %u not supported (256 or 512)", cfg->head_dim);
        return G4A_EUNSUPPORTED;
    }
    if (cfg->n_kv_heads > 4096 || cfg->n_q_heads > 32768 || (int64_t)pg->n_seq * cfg->n_kv_heads > 65535) {
        set_error("n_kv_heads (%u), n_q_heads (%u) or n_seq * n_kv_heads (n_seq %d) too large", cfg->n_kv_heads,
                  cfg->n_q_heads, pg->n_seq);
        return G4A_EINVAL;
    }
    if (cfg->window > 1u << 30) {
        set_error("window (%u) must be at most 2^30", cfg->window);
        return G4A_EINVAL;
    }
    return G4A_OK;
}

PageTab page_tab(const g4a_paged* pg) {
    // the columns that max_key_len keys use: 2^26 at most, whose bytes a buffer range holds
    const int cols = (pg->max_key_len + pg->page_size - 1) / pg->page_size;
    return PageTab{pg->page_table, pg->key_len, pg->n_seq, pg->table_stride, cols, pg->n_pages,
                   __builtin_ctz((unsigned)pg->page_size), pg->max_key_len};
}

struct PagedWriteArgs {
    PageTab t;
    const int32_t* cu;
    const void* k;
    const void* v;
    const float* k_gain;
    const float* rcos;
    const float* rsin;
    void* kc;
    void* vc;
    int n_tokens, n_kv_heads, v_norm;
    float k_in_q, v_in_q, eps;
};

// Row of token t and kv head: k <- RoPE(rms(srq(k)) * gain, p), v <- rms(srq(v)), at its position p's place. A
// workgroup of HD / 2 threads takes one (token, kv head), as kv_write's does, and through the same
// kv_pair_prep, so that the rows are kv_write's to the bit. Few rows: the chain of loads cu -> key_len -> table
// -> row (3.1 us for 16 rows, of which a launch is most). Many: vector instructions, the steps' divisions and
// the sums' shuffles, ahead of the bytes (13501 tokens of 2 x 256, f16 rows into an f32 cache, 83 MB: 21 us =
// 4.0 TB/s, where a copy reaches 5.2). Against 20.8 then, 4 or 8 rows a workgroup took 24.6 / 26.5 us, the steps
// through a refined reciprocal 22.0, the raw rows fetched before the position is known 22.3.
template <int HD, typename IT, typename CT>
__global__ __launch_bounds__(HD / 2) void paged_write_kernel(PagedWriteArgs a) {
    constexpr int HALF = HD / 2, NW = HALF / 64;
    __shared__ float red[2 * NW];
    const int t = threadIdx.x, tok = blockIdx.x, kh = blockIdx.y;
    const int b = seq_of_row(a.cu, a.t.n_seq, tok);
    if (b >= a.t.n_seq) return;
    const SeqRows r = seq_rows(a.t, a.cu, a.n_tokens, b);
    if (!holds(r, tok)) return;
    const int p = row_position(r, tok);
    if (p < 0) return;
    const int page = page_at(a.t, b, p);
    if (!page_ok(a.t, page)) return;
    const size_t row = ((size_t)tok * a.n_kv_heads + kh) * HD;
    const IT* kin = reinterpret_cast<const IT*>(a.k) + row;
    const IT* vin = reinterpret_cast<const IT*>(a.v) + row;
    float k0 = (float)kin[t], k1 = (float)kin[t + HALF], v0 = (float)vin[t], v1 = (float)vin[t + HALF];
    kv_pair_prep<HD>(k0, k1, v0, v1, a.k_gain, a.rcos ? a.rcos + (size_t)p * HALF : nullptr,
                     a.rsin ? a.rsin + (size_t)p * HALF : nullptr, a.v_norm != 0, a.eps, a.k_in_q, a.v_in_q, red, t);
    const size_t crow = paged_row(a.t, page, p, a.n_kv_heads * HD) + (size_t)kh * HD;
    CT* kc = reinterpret_cast<CT*>(a.kc) + crow;
    CT* vc = reinterpret_cast<CT*>(a.vc) + crow;
    store_elem(kc + t, k0);
    store_elem(kc + t + HALF, k1);
    store_elem(vc + t, v0);
    store_elem(vc + t + HALF, v1);
}

typedef void (*paged_write_fn)(PagedWriteArgs);
template <int HD>
static paged_write_fn pick_write(bool in16, bool c32) {
    if (in16) return c32 ? paged_write_kernel<HD, half_t, float> : paged_write_kernel<HD, half_t, half_t>;
    return c32 ? paged_write_kernel<HD, float, float> : paged_write_kernel<HD, float, half_t>;
}

static int launch_write(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens, const int32_t* cu, bool in16, const void* k,
                        const void* v, float k_in_q, float v_in_q, const float* k_gain, const float* rcos,
                        const float* rsin, hipStream_t stream) {
    PagedWriteArgs a;
    a.t = page_tab(pg);
    a.cu = cu;
    a.k = k;
    a.v = v;
    a.k_gain = k_gain;
    a.rcos = rcos;
    a.rsin = rsin;
    a.kc = pg->k_pages;
    a.vc = pg->v_pages;
    a.n_tokens = n_tokens;
    a.n_kv_heads = (int)cfg->n_kv_heads;
    a.v_norm = (cfg->flags & G4A_NO_V_NORM) ? 0 : 1;
    a.k_in_q = k_in_q;
    a.v_in_q = v_in_q;
    a.eps = cfg->eps;
    const bool c32 = (cfg->flags & G4A_KV_F32) != 0;
    hipLaunchKernelGGL(cfg->head_dim == 256 ? pick_write<256>(in16, c32) : pick_write<512>(in16, c32),
                       dim3((unsigned)n_tokens, cfg->n_kv_heads), dim3(cfg->head_dim / 2), 0, stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? G4A_OK : hip_error(e, "paged write launch");
}

int check_rope(const float* rcos, const float* rsin) {
    if ((rcos == nullptr) != (rsin == nullptr)) {
        set_error("rope_cos and rope_sin must both be given or both be NULL");
        return G4A_EINVAL;
    }
    return G4A_OK;
}
int check_steps(float k_in_q, float v_in_q) {
    if (!(k_in_q >= 0.0f) || !(v_in_q >= 0.0f)) {
        set_error("k_in_q/v_in_q must be >= 0");
        return G4A_EINVAL;
    }
    return G4A_OK;
}
int check_paged_call(const g4a_cfg* cfg, int n_tokens, const float* q, const float* q_gain, const float* rcos,
                     const float* rsin, const void* out) {
    if (const int rc = check_rope(rcos, rsin)) return rc;
    if (!q || !out) {
        set_error("q and out must be non-NULL");
        return G4A_EINVAL;
    }
    if (!aligned16(q) || !aligned16(out) || !aligned16(q_gain) || !aligned16(rcos) || !aligned16(rsin)) {
        set_error("q, out, q_gain and the rope tables must be 16-byte aligned");
        return G4A_EINVAL;
    }
    const size_t n = (size_t)n_tokens * cfg->n_q_heads * cfg->head_dim, osz = (cfg->flags & G4A_OUT_F32) ? 4 : 2;
    const uintptr_t x = (uintptr_t)q, y = (uintptr_t)out;
    if (x < y + n * osz && y < x + n * 4) {
        set_error("out must not overlap q");
        return G4A_EINVAL;
    }
    return G4A_OK;
}
int check_tokens(const g4a_cfg* cfg, int n_tokens, const int32_t* cu) {
    if (n_tokens <= 0 || !cu || (uintptr_t)cu % 4) {
        set_error("n_tokens (%d) must be positive and cu_q non-NULL and 4-byte aligned", n_tokens);
        return G4A_EINVAL;
    }
    if ((int64_t)n_tokens * cfg->n_q_heads > 0x7fffffff - 64) {
        set_error("n_tokens * n_q_heads too large");
        return G4A_EINVAL;
    }
    return G4A_OK;
}

}  // namespace g4a

using namespace g4a;

extern "C" int g4a_paged_write(const g4a_cfg* cfg, const g4a_paged* pg, int n_tokens, const int32_t* cu_q,
                               const void* k, const void* v, float k_in_q, float v_in_q, const float* k_gain,
                               const float* rope_cos, const float* rope_sin, void* stream) {
    if (const int rc = check_paged(cfg, pg, false)) return rc;
    if (const int rc = check_tokens(cfg, n_tokens, cu_q)) return rc;
    if (const int rc = check_rope(rope_cos, rope_sin)) return rc;
    if (const int rc = check_steps(k_in_q, v_in_q)) return rc;
    if (!k || !v) {
        set_error("k and v must be non-NULL");
        return G4A_EINVAL;
    }
    if (!aligned16(k) || !aligned16(v) || !aligned16(k_gain) || !aligned16(rope_cos) || !aligned16(rope_sin)) {
        set_error("k, v, k_gain and the rope tables must be 16-byte aligned");
        return G4A_EINVAL;
    }
    return launch_write(cfg, pg, n_tokens, cu_q, (cfg->flags & G4A_IN_F16) != 0, k, v, k_in_q, v_in_q, k_gain, rope_cos,
                        rope_sin, (hipStream_t)stream);
}
