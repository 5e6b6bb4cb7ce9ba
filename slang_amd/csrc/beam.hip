// Beam search's selection over beams and vocabulary (g4a_beam_select).
//
// Scores within a beam are ordered as its logits, so a row's candidates are its n_out largest logits, and the sum of
// exponentials is needed only to compare beams. One pass over the logits: a wave walks a part of a row, 64 * E at a time
// in registers while the next are on their way, and keeps the maximum, the sum relative to it and the n_out largest. A second
// launch, a workgroup a group, joins each row's parts and then the beams.
//
// Logits are ranked by 64-bit keys: a logit's bits, made to ascend, over the complement of its token, so that equal
// logits come lowest token first and no two keys are the same; 0 is no candidate (NaN and -inf are none).
#include <algorithm>

#include "paged.hpp"

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
    int width, vocab, n_out, parts, steps, pad;  // a part is 64 * E * steps logits
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

// A logit x counts as x' = cap tanh(x / cap), or as it is without a cap. What the kernels hold is x' times log2e / unit:
//   kNoCap    unit log2e: the difference of two logits, which is exact where it matters, is rounded last.
//   kCap      unit 1: cap - 2 cap / (1 + 2^(2 log2e x / cap)), off by 2.5 2^-23 of the cap, whatever x is. Its reciprocal cap is
//             kept finite for caps near the smallest numbers, where 0 times infinity would be no number.
//   kWideCap  unit log2e, for caps above kCapTo: tanh by its series, x + x u^2 (-1/3 + 2/15 u^2 - 17/315 u^4 + 62/2835 u^6), where
//             |u| = |x / cap| < 0.3 (the next term is below 2^-24), else 1 - 2 / (1 + 2^(2 log2e u)): off by 4.5 2^-23 of x'.
//             A logit takes twelve instructions more than with kCap: 128 rows of 262144 in f32 54.5 us a call for 46.8.
enum { kNoCap, kCap, kWideCap };
constexpr float kCapTo = 64.0f;
struct Cap {
    float cap, up;  // kCap: cap log2e, 2 log2e / cap; kWideCap: cap, 1 / cap
};
template <int CAP>
__device__ __forceinline__ Cap cap_of(float cap) {
    return CAP == kCap ? Cap{cap * kLog2e, fminf(2.0f * kLog2e / cap, 3.40282347e38f)} : Cap{cap, 1.0f / cap};
}
template <int CAP>
__device__ __forceinline__ float capped(float x, const Cap& c) {
    if (CAP == kCap) return __builtin_fmaf(-2.0f * c.cap, __builtin_amdgcn_rcpf(1.0f + fexp2(x * c.up)), c.cap);
    if (CAP == kWideCap) {
        const float u = x * c.up, u2 = u * u;
        const float far = c.cap * __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + fexp2(u * (2.0f * kLog2e))), 1.0f);
        float p = __builtin_fmaf(u2, 62.0f / 2835.0f, -17.0f / 315.0f);
        p = __builtin_fmaf(u2, p, 2.0f / 15.0f);
        p = __builtin_fmaf(u2, p, -1.0f / 3.0f);
        return fabsf(u) < 0.3f ? __builtin_fmaf(x, u2 * p, x) : far;
    }
    return x;
}
// 2^ of the difference of two
template <int CAP>
__device__ __forceinline__ float weight(float d) { return fexp2(CAP == kCap ? d : d * kLog2e); }
// x' in 64 bits, where beams are compared (not by tanh(), whose 64 bits take a microsecond): off by 2^-51 of the cap; for
// caps above kCapTo by the series below |u| = 0.05, whose next term is below 2^-50
template <int CAP>
__device__ __forceinline__ double capped64(float x_, float cap_) {
    const double x = x_, cap = cap_;
    if (CAP == kNoCap) return x;
    const double u = x / cap, u2 = u * u;
    if (CAP == kWideCap && fabs(u) < 0.05)
        return x + x * (u2 * (-1.0 / 3.0 + u2 * (2.0 / 15.0 + u2 * (-17.0 / 315.0 + u2 * (62.0 / 2835.0)))));
    return cap - 2.0 * cap / (1.0 + exp(2.0 * u));
}

__device__ __forceinline__ u64 wave_max64(u64 k) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const u64 o = __shfl_xor(k, d);
        k = o > k ? o : k;
    }
    return k;
}

// The upper 16 bits of a value that `want` lanes' `top` reach (0: fewer do), found from the highest bit down. Where
// `top` is the largest of a lane's values, at least `want` values reach it, and not many more do.
__device__ __forceinline__ uint32_t wave_bound(uint32_t top, int want) {
    uint32_t bound = 0;
#pragma unroll
    for (int b = 31; b >= 16; --b) {
        const uint32_t t = bound | 1u << b;
        if (__builtin_popcountll(__ballot(top >= t)) >= want) bound = t;
    }
    return bound;
}

// Sorts the `total` keys of the wave's list, largest first, and drops all behind the first `want`: each counts the ones
// above it. Returns how many are left.
constexpr int kList = 128;
__device__ __forceinline__ int wave_rank(u64* list, int total, int want, int lane) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const u64 me = lane < total ? list[lane] : 0, far = 64 + lane < total ? list[64 + lane] : 0;
    int rank = 0, far_rank = 0;
    if (total <= 64) {
#pragma unroll 4
        for (int o = 0; o < total; ++o) rank += list[o] > me;
    } else {
#pragma unroll 4
        for (int o = 0; o < total; ++o) {
            rank += list[o] > me;
            far_rank += list[o] > far;
        }
    }
    __builtin_amdgcn_wave_barrier();
    if (me && rank < want) list[rank] = me;
    if (far && far_rank < want) list[far_rank] = far;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    return min(total, want);
}

// What a part's sum, relative to its own maximum, counts relative to M
template <int CAP>
__device__ __forceinline__ float part_weight(float2 v, float M, const Cap& c) {
    return v.x == M ? v.y : v.x > kNegInf ? v.y * weight<CAP>(capped<CAP>(v.x, c) - capped<CAP>(M, c)) : 0.0f;
}

// Rows may begin anywhere, and which tokens a lane sums must not depend on where: equal rows have equal sums to the bit, so
// that equal beams tie. So a part begins at a token, and 16 bytes are loaded from any element on (128 rows of 262144, one
// element off 16 bytes: 44.0 us a call for 44.2 in f32, 46.1 for 44.2 in f16).
template <typename T, int E, int CAP>
__global__ __launch_bounds__(256) void beam_part_kernel(BeamArgs a) {
    constexpr int VEC = 16 / sizeof(T);
    typedef T vec_t __attribute__((ext_vector_type(VEC), aligned(sizeof(T))));
    __shared__ u64 s_list[4][kList];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row = blockIdx.y, part = blockIdx.x * 4 + wave, K = a.n_out;
    if (part >= a.parts) return;
    u64* list = s_list[wave];
    const T* p = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row_stride;
    const int64_t wave0 = (int64_t)part * a.steps * (64 * E), part0 = wave0 + lane * VEC;  // tokens of the first values
    const auto load = [&](int step, float (&x)[E]) {
        const int64_t w0 = wave0 + (int64_t)step * (64 * E), o0 = part0 + (int64_t)step * (64 * E);
        if (w0 + 64 * E <= a.vocab) {  // wave-uniform
            vec_t v[E / VEC];
#pragma unroll
            for (int i = 0; i < E / VEC; ++i) v[i] = __builtin_nontemporal_load(reinterpret_cast<const vec_t*>(p + o0) + i * 64);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] = (float)v[i / VEC][i % VEC];
        } else {  // a row's end: 16 bytes where a lane has them, so that this wave is not the one that the launch ends with
#pragma unroll
            for (int i = 0; i < E / VEC; ++i) {
                const int64_t o = o0 + i * 64 * VEC;
                vec_t v;
#pragma unroll
                for (int k = 0; k < VEC; ++k) v[k] = (T)kNegInf;
                if (o + VEC <= a.vocab) {
                    v = *reinterpret_cast<const vec_t*>(p + o);
                } else if (o < a.vocab) {
#pragma unroll
                    for (int k = 0; k < VEC; ++k)
                        if (o + k < a.vocab) v[k] = p[o + k];
                }
#pragma unroll
                for (int k = 0; k < VEC; ++k) x[i * VEC + k] = (float)v[k];
            }
        }
    };
    const Cap cap = cap_of<CAP>(a.cap);
    float m = kNegInf, s = 0.0f;
    float least = -3.40282347e38f;  // what a logit has to reach to be a candidate: nothing below can be among the largest
    int count = 0, sorted = 0;      // candidates in the list; of them in order and above all that came before them
    float x[E], y[E];
    load(0, y);
    for (int step = 0; step < a.steps; ++step) {
#pragma unroll
        for (int i = 0; i < E; ++i) {  // (copied here, so that no wait below is for the loads that follow)
            x[i] = y[i];
            asm volatile("" : "+v"(x[i]));
        }
        if (step + 1 < a.steps) load(step + 1, y);
        float mine = kNegInf, low = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {  // (both pass over NaN)
            mine = fmaxf(mine, x[i]);
            if (CAP) low = fminf(low, x[i]);
        }
        const float mx = wave_max(mine);
        if (mx > m) {
            const float d = capped<CAP>(m, cap) - capped<CAP>(mx, cap);
            s = m == kNegInf ? 0.0f : s * weight<CAP>(d);
            m = mx;
        }
        const float mc = capped<CAP>(m, cap);
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < E; ++i) {
            const float d = capped<CAP>(x[i], cap) - mc;
            sum += weight<CAP>(d);
        }
        // with -inf, which a cap would make finite, or NaN, which are no tokens, or +inf, which is all there is: with care
        if (__ballot(!(sum < __builtin_huge_valf()) || (CAP && low == kNegInf))) {
            sum = 0.0f;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                x[i] = fmaxf(x[i], kNegInf);
                const float d = capped<CAP>(x[i], cap) - mc;
                sum += x[i] == kNegInf ? 0.0f : x[i] == m ? 1.0f : weight<CAP>(d);
            }
        }
        s += sum;
        if (step == 0) least = fmaxf(least, of_ascending(wave_bound(ascending(mine), K)));  // (NaN: as it was)
        if (__ballot(mine >= least)) {
            int n = 0;
#pragma unroll
            for (int i = 0; i < E; ++i) n += x[i] >= least;
            const int t0 = (int)(part0 + (int64_t)step * (64 * E));
            int incl = wave_scan(n), total = __builtin_amdgcn_readlane(incl, 63);
            if (count + total > kList) {
                if (count > K) count = wave_rank(list, count, K, lane);
                if (count + total > kList) {  // many are equal, or ascend: this step's largest, one after the other
                    u64 last = ~0ull;
                    for (int k = 0; k < K; ++k) {
                        u64 best = 0;
#pragma unroll
                        for (int i = 0; i < E; ++i) {
                            const u64 key = x[i] >= least ? key_of(x[i], t0 + (i / VEC) * 64 * VEC + i % VEC) : 0;
                            best = key < last && key > best ? key : best;
                        }
                        last = wave_max64(best);
                        if (last == 0) break;
                        if (lane == 0) list[count] = last;
                        ++count;
                    }
                    total = 0;
                }
            }
            if (total > 0) {
                int k = count + incl - n;
#pragma unroll
                for (int i = 0; i < E; ++i)
                    if (x[i] >= least) list[k++] = key_of(x[i], t0 + (i / VEC) * 64 * VEC + i % VEC);
                count += total;
            }
            if (count >= K && (count > kList / 2 || step == 0) && step + 1 < a.steps) {
                // of equal logits the earlier token is taken, so a later one has to be above the last
                count = sorted = wave_rank(list, count, K, lane);
                least = fmaxf(least, of_ascending((uint32_t)(list[K - 1] >> 32) + 1));
            }
        }
    }
    s = wave_sum(s);
    const size_t at = (size_t)row * a.parts + part;
    if (lane == 0) a.sums[at] = make_float2(m, s);
    if (count != sorted) count = wave_rank(list, count, K, lane);
    if (lane < K) a.keys[at * K + lane] = lane < count ? list[lane] : 0;
}

// A group. A wave a row: its parts' sums, in 64 bits, and the n_out largest of its parts' keys, whose lists descend. Then a
// candidate's place among the group's is its own place in its beam and, of each other beam, the number of candidates in
// front of it, found by halving.
constexpr int kGroupWaves = 16;
template <int CAP>
__global__ __launch_bounds__(64 * kGroupWaves) void beam_group_kernel(BeamArgs a) {
    __shared__ u64 s_list[kGroupWaves][kList];
    __shared__ union {
        u64 key;
        double score;
    } s_cand[kBeams * kBeams];
    __shared__ double s_final[kBeams * kBeams];
    __shared__ int s_token[kBeams * kBeams], s_n[kBeams], s_done[kBeams];
    __shared__ double s_score[kBeams];
    __shared__ double s_log[kBeams], s_most[kBeams];  // of a row: log of the sum of exp(x' - the largest x'), and that x'
    const int g = blockIdx.x, tid = threadIdx.x, threads = blockDim.x, W = a.width, K = a.n_out;
    const Cap cap = cap_of<CAP>(a.cap);
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (tid < W) {
        s_n[tid] = 0;
        s_score[tid] = (double)a.scores[g * W + tid];
        s_done[tid] = a.done && a.done[g * W + tid];
    }
    for (int w = wave; w < W; w += threads >> 6) {
        const size_t row = (size_t)g * W + w;
        const float2* sums = a.sums + row * a.parts;
        const u64* keys = a.keys + row * a.parts * K;
        float m = kNegInf;
        uint32_t top = 0;
        for (int i = lane; i < a.parts; i += 64) {
            m = fmaxf(m, sums[i].x);
            top = max(top, (uint32_t)(keys[(size_t)i * K] >> 32));
        }
        m = wave_max(m);
        const uint32_t bound = max(wave_bound(top, K), 1u);  // (0 is no key)
        double s = 0.0;
        int total = 0;
        for (int i0 = 0; i0 < a.parts; i0 += 64) {  // wave-uniform
            const int i = i0 + lane;
            const float2 v = i < a.parts ? sums[i] : make_float2(kNegInf, 0.0f);
            s += (double)part_weight<CAP>(v, m, cap);
            bool more = i < a.parts;
            for (int k = 0; k < K; ++k) {
                const u64 key = more ? keys[(size_t)i * K + k] : 0;
                more = (uint32_t)(key >> 32) >= bound;
                const unsigned long long in = __ballot(more);
                if (!in) break;
                const int at = total + __builtin_popcountll(in & ((1ull << lane) - 1));
                if (more && at < kList) s_list[wave][at] = key;
                total += __builtin_popcountll(in);
            }
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) s += __shfl_xor(s, d);
        if (lane == 0) s_log[w] = log(s);
        if (total <= kList) {
            total = wave_rank(s_list[wave], total, K, lane);
            if (lane < K) s_cand[w * K + lane].key = lane < total ? s_list[wave][lane] : 0;
        } else {  // many are equal, or fewer parts than n_out, where no bound is found, have more than the list holds: one after the
                  // other (4 rows of 32000 in 63 parts: n_out 16 11.2 us a call, 64 112)
            u64 last = ~0ull;
            for (int k = 0; k < K; ++k) {
                u64 best = 0;
                for (int i = lane; i < a.parts; i += 64)
                    for (int j = 0; j < K; ++j) {
                        const u64 key = keys[(size_t)i * K + j];
                        if (key >= last) continue;
                        best = key > best ? key : best;
                        break;
                    }
                last = wave_max64(best);
                if (lane == 0) s_cand[w * K + k].key = last;
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    for (int i = tid; i < W * K; i += threads) {
        const u64 key = s_cand[i].key;
        const double c = capped64<CAP>(of_ascending((uint32_t)(key >> 32)), a.cap);
        s_token[i] = key ? ~(int)(uint32_t)key : -1;
        s_cand[i].score = c;
        if (i % K == 0) s_most[i / K] = c;
    }
    __syncthreads();
    for (int i = tid; i < W * K; i += threads) {
        const int w = i / K, k = i - w * K;
        double score = (double)kNegInf;
        if (s_done[w]) {
            if (k == 0) {
                score = s_score[w];
                s_token[i] = a.pad;
            }
        } else if (s_token[i] >= 0) {
            double c = s_cand[i].score;  // no rounding puts two of a beam out of order
#pragma unroll 4
            for (int j = 0; j < k; ++j) c = fmin(c, s_cand[i - 1 - j].score);
            score = s_score[w] + ((c == s_most[w] ? 0.0 : c - s_most[w]) - s_log[w]);  // (the largest may be +inf)
        }
        s_final[i] = score > (double)kNegInf ? score : (double)kNegInf;
        if (score > (double)kNegInf) atomicAdd(&s_n[w], 1);  // a beam's candidates come first
    }
    __syncthreads();
    int total = 0;
#pragma unroll 4
    for (int w = 0; w < W; ++w) total += s_n[w];
    for (int i = tid; i < W * K; i += threads) {
        const int w = i / K, k = i - w * K;
        if (k >= s_n[w]) continue;
        const double me = s_final[i];
        int rank = k;
        for (int o0 = 0; o0 < W && rank < K; o0 += 4) {  // four beams' searches at once: LDS answers in 130 cycles
            int front[4] = {}, n[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) n[u] = o0 + u < W && o0 + u != w ? s_n[o0 + u] : 0;
            for (int step = kBeams; step; step >>= 1) {
                if (step > K) continue;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int o = o0 + u, at = front[u] + step;
                    const double s = s_final[at <= n[u] ? o * K + at - 1 : i];
                    if (at <= n[u] && (s > me || (s == me && o < w))) front[u] = at;
                }
            }
            rank += front[0] + front[1] + front[2] + front[3];
        }
        if (rank < K) {
            const size_t at = (size_t)g * K + rank;
            a.out_score[at] = (float)me;
            a.out_parent[at] = g * W + w;
            a.out_token[at] = s_token[i];
        }
    }
    for (int k = total + tid; k < K; k += threads) {
        const size_t at = (size_t)g * K + k;
        a.out_score[at] = kNegInf;
        a.out_parent[at] = a.out_token[at] = -1;
    }
}

typedef void (*beam_fn)(BeamArgs);
template <typename T, int CAP>
static beam_fn pick_each(int each) { return each == 32 ? beam_part_kernel<T, 32, CAP> : beam_part_kernel<T, 8, CAP>; }
template <int CAP>
static beam_fn pick_part(bool f16, int each) { return f16 ? pick_each<half_t, CAP>(each) : pick_each<float, CAP>(each); }
struct BeamFns {
    beam_fn part, group;
};
static BeamFns pick_beam(bool f16, int each, float cap) {
    if (cap == 0.0f) return {pick_part<kNoCap>(f16, each), beam_group_kernel<kNoCap>};
    if (cap > kCapTo) return {pick_part<kWideCap>(f16, each), beam_group_kernel<kWideCap>};
    return {pick_part<kCap>(f16, each), beam_group_kernel<kCap>};
}

// Few logits: 512 a wave, one step, so that many waves share them. Many, or rows so long that their parts would be many to
// join: steps of 2048, as many (to the nearest) as leave the card kPartWaves waves. A call in a graph with steps of 512 and of
// 2048: 4 rows of 32000 9.3 and 10.6 us, of 65536 9.9 and 10.2, of 100000 11.6 and 10.5, of 262144 14.7 and 11.4; 128 rows of
// 32000 in f16 with a cap 19.2 and 25.1, of 50000 22.1 and 21.5, of 65536 23.9 and 21.8, of 262144 56.5 and 40.3; 1024 rows of
// 8192 20.1 and 20.4.
// A wave pays for its first step's bound and order, so longer walks are cheaper, and fewer waves hide less: the kernel takes
// 33.6 us for 128 rows of 262144 in f32 with a cap with 2 steps of 2048 (4.0 TB/s), 33.8 with 1 (whose parts take the join a
// microsecond more), 34.5 with 4; 29.4 without a cap. What bounds it: a logit with
// a cap takes two exponentials, a reciprocal and six more instructions, about 72 cycles a wave of 64, 15 us of the card's
// VALU beside the 26 us that the bytes take, and a wave's first step's ballots and LDS trips.
constexpr int kPartWaves = 8192;
struct BeamPlan {
    int each, steps, parts;
    size_t keys, total;
};
static BeamPlan beam_plan(int n_groups, int width, int vocab, int n_out) {
    BeamPlan p;
    const int64_t rows = (int64_t)n_groups * width, span = vocab;
    p.each = vocab > 1 << 16 || rows * vocab >= (int64_t)64 * 16 * kPartWaves ? 32 : 8;
    const int64_t step = (int64_t)64 * 32 * kPartWaves;
    p.steps = p.each == 8 ? 1 : (int)std::min<int64_t>(std::max<int64_t>((rows * vocab + step / 2) / step, 1), 64);
    const int64_t part = (int64_t)64 * p.each * p.steps;
    p.parts = (int)((span + part - 1) / part);
    auto al = [](size_t x) { return (x + 255) & ~(size_t)255; };
    p.keys = al((size_t)rows * p.parts * sizeof(float2));
    // (room for the parts that the shortest steps make, so that a workspace for the largest call holds every smaller one)
    const size_t most = (size_t)rows * (size_t)((span + 511) / 512);
    p.total = al(most * sizeof(float2)) + al(most * n_out * sizeof(u64));
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
    const BeamArgs a{logits, row_stride, scores, done, out_score, out_parent, out_token, (float2*)w, (u64*)(w + p.keys), width, vocab, n_out,
                     p.parts, p.steps, pad, cap};
    const hipStream_t stream = (hipStream_t)stream_;
    const dim3 grid((unsigned)((p.parts + 3) / 4), (unsigned)(n_groups * width));
    const BeamFns fn = pick_beam(logits_f16 != 0, p.each, cap);
    hipLaunchKernelGGL(fn.part, grid, dim3(256), 0, stream, a);
    hipLaunchKernelGGL(fn.group, dim3((unsigned)n_groups), dim3(64 * std::min(width, kGroupWaves)), 0, stream, a);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? G4A_OK : hip_error(e, "beam select launch");
}
