// Beam search's selection over beams and vocabulary (g4a_beam_select).
//
// Scores within a beam are ordered as its logits, so a row's candidates are its n_out largest logits, and the sum of
// exponentials is needed only to compare beams. One pass over the logits: a wave takes 64 * E of a row into registers and
// writes its maximum, its sum and its n_out largest. A second launch joins a row's waves, and in the group's last row
// the beams.
//
// A logit's place in the order is a 64-bit key: its bits, made to ascend, over the complement of its token, so that
// equal logits come lowest token first and no two keys are the same; 0 is no candidate (NaN and -inf are none).
#include <algorithm>

#include "common.hpp"

namespace g4a {

constexpr int kBeams = 64;  // G4A_BEAMS_MAX
typedef unsigned long long u64;

struct BeamArgs {
    const void* logits;
    int64_t row_stride;
    const float* scores;
    const uint8_t* done;
    float* out_score;
    int32_t* out_parent;
    int32_t* out_token;
    float2* sums;     // [rows][parts]: maximum, sum of 2^(log2e (x' - maximum))
    u64* keys;        // [rows][parts][n_out], largest first
    u64* row_keys;    // [rows][n_out]
    double2* row_sum;  // [rows]: the largest x', the logarithm of the sum of exp(x' - it)
    int width, vocab, n_out, parts, pad;
    float cap;
};

// the bits of a float as a whole number that ascends with it, -0 as 0
__device__ __forceinline__ uint32_t ascending(float x) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float of_ascending(uint32_t u) {
    return __builtin_bit_cast(float, u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ u64 key_of(float x, int token) { return (u64)ascending(x) << 32 | (uint32_t)~token; }

// x' of a logit: cap tanh(x / cap) as cap - 2 cap / (1 + 2^(2 log2e x / cap)); up2 = 2 log2e / cap
__device__ __forceinline__ float capped(float x, float cap, float up2) {
    return cap == 0.0f ? x : __builtin_fmaf(-2.0f * cap, __builtin_amdgcn_rcpf(1.0f + fexp2(x * up2)), cap);
}

__device__ __forceinline__ u64 wave_max64(u64 k) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_xor(k, d);
        k = o > k ? o : k;
    }
    return k;
}

// The wave's `want` largest of the keys x[0 .. N) of all its lanes, largest first, to out (0 behind the last). Fast: the
// want-th largest of the lanes' own maxima bounds the want-th largest key from below; the few keys that pass it go to
// `list` (kList keys of the wave's own LDS), where each counts the ones above it. More than kList pass where many are
// equal: then one maximum after the other.
constexpr int kList = 128;
template <int N>
__device__ __forceinline__ void wave_top(const u64 (&x)[N], int want, u64* list, u64* out, int lane) {
    u64 mine = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) mine = x[i] > mine ? x[i] : mine;
    // the largest bound that `want` lanes' maxima reach, by its bits from the top
    uint32_t bound = 0;
    const uint32_t top = (uint32_t)(mine >> 32);
    for (int b = 31; b >= 0; --b) {
        const uint32_t t = bound | 1u << b;
        if (__builtin_popcountll(__ballot(top >= t)) >= want) bound = t;
    }
    int n = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) n += x[i] != 0 && (uint32_t)(x[i] >> 32) >= bound;
    int at = 0, total = 0;
    {
        int incl = n;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int y = __shfl_up(incl, d);
            if (lane >= d) incl += y;
        }
        at = incl - n;
        total = __builtin_amdgcn_readlane(incl, 63);
    }
    if (total <= kList) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (x[i] != 0 && (uint32_t)(x[i] >> 32) >= bound) list[at++] = x[i];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        for (int k = lane; k < total; k += 64) {
            const u64 me = list[k];
            int rank = 0;
            for (int o = 0; o < total; ++o) rank += list[o] > me;
            if (rank < want) out[rank] = me;
        }
        for (int k = total + lane; k < want; k += 64) out[k] = 0;
        __builtin_amdgcn_wave_barrier();
        return;
    }
    u64 last = ~0ull;
    for (int k = 0; k < want; ++k) {
        u64 best = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) best = x[i] < last && x[i] > best ? x[i] : best;
        best = wave_max64(best);
        if (lane == 0) out[k] = best;
        last = best;
    }
}

// A wave's 64 * E logits of a row, E / VEC loads of 16 bytes a lane. Rows may begin anywhere: a part begins at a multiple of VEC
// elements of the tensor, at or in front of the row's first.
template <typename T, int E>
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(VEC)));
    __shared__ u64 s_list[4][kList];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.y, part = blockIdx.x * 4 + wave;
    if (part >= a.parts) return;
    const int64_t first = (int64_t)row * a.row_stride, base = first & ~(int64_t)(VEC - 1);
    const int skip = (int)(first - base);
    const T* p = reinterpret_cast<const T*>(a.logits) + base;
    float x[E];
#pragma unroll
    for (int i = 0; i < E / VEC; ++i) {
        const int64_t o = (int64_t)part * (64 * E) + (i * 64 + lane) * VEC - skip;  // token of the first of VEC
        if (o >= 0 && o + VEC <= a.vocab) {
            const vec_t v = __builtin_nontemporal_load(reinterpret_cast<const vec_t*>(p + o + skip));
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[i * VEC + e] = (float)v[e];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[i * VEC + e] = o + e >= 0 && o + e < a.vocab ? (float)p[o + e + skip] : kNegInf;
        }
    }
    float m = kNegInf;
#pragma unroll
    for (int i = 0; i < E; ++i) m = fmaxf(m, x[i]);
    m = wave_max(m);
    const float up2 = 2.0f * kLog2e / a.cap, mc = capped(m, a.cap, up2);
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const float c = capped(x[i], a.cap, up2);
        // (equal to the maximum: 1, for infinities too; NaN and what is no token: 0)
        s += x[i] == m ? 1.0f : x[i] > kNegInf ? fexp2((c - mc) * kLog2e) : 0.0f;
    }
    s = wave_sum(m == kNegInf ? 0.0f : s);
    u64 k[E];
#pragma unroll
    for (int i = 0; i < E; ++i) {
        const int64_t t = (int64_t)part * (64 * E) + ((i / VEC) * 64 + lane) * VEC + i % VEC - skip;
        k[i] = x[i] > kNegInf ? key_of(x[i], (int)t) : 0;  // (what is no token is -inf)
    }
    const size_t at = (size_t)row * a.parts + part;
    if (lane == 0) a.sums[at] = make_float2(m, s);
    wave_top<E>(k, a.n_out, s_list[wave], a.keys + at * a.n_out, lane);
}

// A row: its parts' sums in 64 bits, its n_out largest keys.
__global__ __launch_bounds__(256) void beam_row_kernel(BeamArgs a) {
    __shared__ u64 s_top[4][kBeams], s_list[4][kList];
    __shared__ float s_m[4];
    __shared__ double s_s[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), row = blockIdx.x;
    const float2* sums = a.sums + (size_t)row * a.parts;
    float m = kNegInf;
    for (int i = tid; i < a.parts; i += 256) m = fmaxf(m, sums[i].x);
    m = wave_max(m);
    if (lane == 0) s_m[wave] = m;
    __syncthreads();
    m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    const auto cap64 = [&](float x) { return a.cap == 0.0f ? (double)x : (double)a.cap * tanh((double)x / (double)a.cap); };
    double s = 0.0;
    for (int i = tid; i < a.parts; i += 256) {
        const float2 v = sums[i];
        if (v.x == m) s += (double)v.y;
        else if (v.x > kNegInf) s += (double)v.y * exp(cap64(v.x) - cap64(m));
    }
    for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
    if (lane == 0) s_s[wave] = s;
    // keys: 8 a lane at a time, the wave's best so far among them
    const u64* keys = a.keys + (size_t)row * a.parts * a.n_out;
    const int64_t n = (int64_t)a.parts * a.n_out;
    for (int k = lane; k < a.n_out; k += 64) s_top[wave][k] = 0;
    for (int64_t k0 = 0; k0 < n; k0 += 4 * 64 * 7) {
        u64 x[8];
#pragma unroll
        for (int i = 0; i < 7; ++i) {
            const int64_t k = k0 + (int64_t)(i * 4 + wave) * 64 + lane;
            x[i] = k < n ? keys[k] : 0;
        }
        __builtin_amdgcn_wave_barrier();
        x[7] = lane < a.n_out ? s_top[wave][lane] : 0;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        wave_top<8>(x, a.n_out, s_list[wave], s_top[wave], lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
    __syncthreads();
    if (wave > 0) return;
    u64 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = lane < a.n_out ? s_top[i][lane] : 0;
    wave_top<4>(x, a.n_out, s_list[0], a.row_keys + (size_t)row * a.n_out, lane);
    if (lane == 0) a.row_sum[row] = make_double2(cap64(m), log(s_s[0] + s_s[1] + s_s[2] + s_s[3]));
}

// A group: candidate (beam, place) of score s + x' - lse; its place among the group's is its own place in its beam and, of
// each other beam, the candidates in front of it, found by halving.
__global__ __launch_bounds__(256) void beam_group_kernel(BeamArgs a) {
    __shared__ double s_score[kBeams * kBeams];
    __shared__ int s_token[kBeams * kBeams], s_n[kBeams];
    const int g = blockIdx.x, tid = threadIdx.x, W = a.width, K = a.n_out;
    for (int i = tid; i < W * K; i += 256) {
        const int w = i / K, k = i - w * K, row = g * W + w;
        const double at = (double)a.scores[row];
        const bool done = a.done && a.done[row];
        double score = (double)kNegInf;
        int token = -1;
        if (done) {
            if (k == 0) {
                score = at;
                token = a.pad;
            }
        } else if (const u64 key = a.row_keys[(size_t)row * K + k]) {
            const float x = of_ascending((uint32_t)(key >> 32));
            const double2 sum = a.row_sum[row];
            const double c = a.cap == 0.0f ? (double)x : (double)a.cap * tanh((double)x / (double)a.cap);
            score = at + ((c == sum.x ? 0.0 : c - sum.x) - sum.y);  // (the largest may be +inf)
            token = ~(int)(uint32_t)key;
        }
        if (!(score > (double)kNegInf)) score = (double)kNegInf;
        s_score[i] = score;
        s_token[i] = token;
    }
    __syncthreads();
    if (tid < W) {  // the beam's candidates: the ones that are there come first, and no rounding puts two out of order
        int n = 0;
        double least = (double)__builtin_huge_valf();
        for (int k = 0; k < K; ++k) {
            least = fmin(least, s_score[tid * K + k]);
            s_score[tid * K + k] = least;
            n += least > (double)kNegInf;
        }
        s_n[tid] = n;
    }
    __syncthreads();
    int total = 0;
    for (int w = 0; w < W; ++w) total += s_n[w];
    for (int i = tid; i < W * K; i += 256) {
        const int w = i / K, k = i - w * K;
        if (k >= s_n[w]) continue;
        const double me = s_score[i];
        int rank = k;
        for (int o = 0; o < W && rank < K; ++o) {
            if (o == w) continue;
            int lo = 0, hi = s_n[o];  // candidates of beam o in front of this one: [0, lo)
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                const double s = s_score[o * K + mid];
                if (s > me || (s == me && o < w)) lo = mid + 1;
                else hi = mid;
            }
            rank += lo;
        }
        if (rank < K) {
            const size_t at = (size_t)g * K + rank;
            a.out_score[at] = (float)me;
            a.out_parent[at] = g * W + w;
            a.out_token[at] = s_token[i];
        }
    }
    for (int k = total + tid; k < K; k += 256) {
        const size_t at = (size_t)g * K + k;
        a.out_score[at] = kNegInf;
        a.out_parent[at] = a.out_token[at] = -1;
    }
}

// Tokens that a wave takes: enough waves for the card first (four a SIMD), then long ones, whose lists are fewer.
static int beam_each(int64_t rows, int64_t vocab) { return rows * vocab >= (int64_t)64 * 32 * 4096 ? 32 : 8; }

struct BeamPlan {
    int each, parts;
    size_t keys, row_keys, row_sum, total;
};
static BeamPlan beam_plan(int n_groups, int width, int vocab, int n_out) {
    BeamPlan p;
    const int64_t rows = (int64_t)n_groups * width;
    p.each = beam_each(rows, vocab);
    p.parts = (int)(((int64_t)vocab + 7 + 64 * p.each - 1) / (64 * p.each));  // a row may begin 7 behind its part
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.keys = al((size_t)rows * p.parts * sizeof(float2));
    p.row_keys = p.keys + al((size_t)rows * p.parts * n_out * sizeof(u64));
    p.row_sum = p.row_keys + al((size_t)rows * n_out * sizeof(u64));
    p.total = p.row_sum + al((size_t)rows * sizeof(double2));
    return p;
}

static int check_beam(int n_groups, int width, int vocab, int n_out) {
    if (n_groups <= 0 || width <= 0 || vocab <= 0 || n_out <= 0 || width > kBeams || n_out > kBeams) {
        set_error("n_groups (%d) and vocab (%d) must be positive, width (%d) and n_out (%d) in [1, %d]", n_groups, vocab, width, n_out, kBeams);
        return G4A_EINVAL;
    }
    if ((int64_t)n_groups * width > 65535 || vocab > 1 << 30) {
        set_error("n_groups * width must be at most 65535 (%d * %d), vocab at most 2^30 (%d)", n_groups, width, vocab);
        return G4A_EINVAL;
    }
    return G4A_OK;
}

}  // namespace g4a

using namespace g4a;

extern "C" size_t g4a_beam_select_ws_bytes(int n_groups, int width, int vocab, int n_out) {
    return check_beam(n_groups, width, vocab, n_out) ? 0 : beam_plan(n_groups, width, vocab, n_out).total;
}

extern "C" int g4a_beam_select(int n_groups, int width, int vocab, int logits_f16, const void* logits, int64_t row_stride,
                               const float* scores, const uint8_t* done, int pad, float cap, int n_out, float* out_score,
                               int32_t* out_parent, int32_t* out_token, void* ws, size_t ws_bytes, void* stream_) {
    if (const int rc = check_beam(n_groups, width, vocab, n_out)) return rc;
    if (!logits || (uintptr_t)logits % 16 || !scores || (uintptr_t)scores % 4 || !out_score || !out_parent || !out_token ||
        ((uintptr_t)out_score | (uintptr_t)out_parent | (uintptr_t)out_token) % 4) {
        set_error("logits (16-byte aligned), scores and the outputs (4-byte aligned) must be non-NULL");
        return G4A_EINVAL;
    }
    if (row_stride < vocab || row_stride > (int64_t)1 << 40 || !(cap >= 0.0f) || !(cap < 3.0e38f)) {
        set_error("row_stride (%lld) must be at least vocab (%d), cap (%g) finite and >= 0", (long long)row_stride, vocab, (double)cap);
        return G4A_EINVAL;
    }
    if (done && (pad < 0 || pad >= vocab)) {
        set_error("pad (%d) must be a token", pad);
        return G4A_EINVAL;
    }
    const BeamPlan p = beam_plan(n_groups, width, vocab, n_out);
    if (!ws || (uintptr_t)ws % 256 || ws_bytes < p.total) {
        set_error("beam select workspace needs %zu bytes (256-byte aligned), got %zu", p.total, ws ? ws_bytes : (size_t)0);
        return G4A_EWORKSPACE;
    }
    char* w = (char*)ws;
    const BeamArgs a{logits, row_stride, scores, done, out_score, out_parent, out_token, (float2*)w, (u64*)(w + p.keys),
                     (u64*)(w + p.row_keys), (double2*)(w + p.row_sum), width, vocab, n_out, p.parts, pad, cap};
    const hipStream_t stream = (hipStream_t)stream_;
    const dim3 grid((unsigned)((p.parts + 3) / 4), (unsigned)(n_groups * width));
    void (*part)(BeamArgs) = logits_f16 ? (p.each == 32 ? beam_part_kernel<half_t, 32> : beam_part_kernel<half_t, 8>)
                                        : (p.each == 32 ? beam_part_kernel<float, 32> : beam_part_kernel<float, 8>);
    hipLaunchKernelGGL(part, grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL(beam_row_kernel, dim3((unsigned)(n_groups * width)), dim3(256), 0, stream, a);
    hipLaunchKernelGGL(beam_group_kernel, dim3((unsigned)n_groups), dim3(256), 0, stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? G4A_OK : hip_error(e, "beam select launch");
}
