// Tile-level pieces that the prefill kernels over contiguous (prefill.hip) and paged caches
// (paged_prefill.hip) share: MFMA forms, LDS swizzles and transposed reads, partial outputs in memory.
#pragma once

#include "common.hpp"

namespace g4a {

typedef unsigned v4u32 __attribute__((ext_vector_type(4)));
typedef unsigned v2u32 __attribute__((ext_vector_type(2)));

// Most a column's running maximum lags its true maximum by (log2 units): P <= 2^15 < 65504
constexpr float kMaxLag = 15.0f;

// f32 values rounded to their upper 24 bits (a 16-bit mantissa, half a step 2^-16; an infinity and
// the NaNs that f16 operands make keep their bits), eight at a time: the upper halves, and the
// third bytes.
struct Part24 {
    v4u32 hi;
    v2u32 lo;
};
template <typename ACC>
__device__ __forceinline__ Part24 pack24(const ACC& acc, int j0, float inv) {
    uint32_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __builtin_bit_cast(uint32_t, acc[j0 + i] * inv) + 0x80u;
    Part24 r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r.hi[i] = __builtin_amdgcn_perm(x[2 * i + 1], x[2 * i], 0x07060302);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t p0 = __builtin_amdgcn_perm(x[4 * i + 1], x[4 * i], 0x0c0c0501);
        const uint32_t p1 = __builtin_amdgcn_perm(x[4 * i + 3], x[4 * i + 2], 0x0c0c0501);
        r.lo[i] = __builtin_amdgcn_perm(p1, p0, 0x05040100);
    }
    return r;
}
// value i of the eight
__device__ __forceinline__ float unpack24(v4u32 hi, v2u32 lo, int i) {
    const uint32_t sel = (i & 1 ? 0x07060000u : 0x05040000u) | (uint32_t)(i & 3) << 8 | 0x0cu;
    return __builtin_bit_cast(float, __builtin_amdgcn_perm(hi[i / 2], lo[i / 4], sel));
}

// The partial of one 32x32 accumulator tile dt of wave block w (of 32 x DIMS), times inv, as
// contiguous runs of all 64 lanes, into the piece's block `slot` of NV = NCOL x HD values. NT: on the
// non-temporal policy, which the hd-256 pieces take (their 12 MB of partials at S 1024, with the q
// rows also stored that way: config 3G 27.2 -> 26.5 us, 3S 25.2 -> 25.55 us) and the hd-512 ones
// do not (29 MB: 47.3 -> 49.2 us).
template <bool NT, int DIMS, int NV, typename ACC>
__device__ __forceinline__ void store_part(void* part_o, bool part24, int slot, int w, int dt, int lane, const ACC& acc, float inv) {
    char* base = reinterpret_cast<char*>(part_o) + (size_t)slot * (NV * (part24 ? 3 : 2));
    const int run0 = w * (32 * DIMS) + dt * 1024;
    auto put = [](auto* dst, auto v) {
        if constexpr (NT) __builtin_nontemporal_store(v, dst);
        else *dst = v;
    };
#pragma unroll
    for (int jp = 0; jp < 2; ++jp) {
        const int run = run0 + 512 * jp + 8 * lane;
        if (part24) {
            const Part24 v = pack24(acc, 8 * jp, inv);
            put(reinterpret_cast<v4u32*>(base + 2 * run), v.hi);
            put(reinterpret_cast<v2u32*>(base + 2 * NV + run), v.lo);
        } else {
            half8 v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = (half_t)(acc[8 * jp + i] * inv);
            put(reinterpret_cast<half8*>(base + 2 * run), v);
        }
    }
}

// LDS operand reads issued ahead of their MFMAs in prefill_kernel_w32: score product
// (one K read per MFMA) and P.V product (two transposed V reads per MFMA); 2-8 and 3-7
// measured within +-2 % at S 1024 and S 8192
constexpr int kQkAhead = 4;
constexpr int kPvAhead = 3;
// 4 halves of a row-major LDS tile transposed across each 16-lane group: lane n of the
// group receives element n%4 of the 8-byte chunks supplied by lanes n/4 + 4j (j < 4).
__device__ __forceinline__ half4 lds_tr16(const half_t* p) {
    typedef short short4_ __attribute__((ext_vector_type(4)));
    const short4_ t = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_*)(p));
    return __builtin_bit_cast(half4, t);
}

typedef float float16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float16v mfma32(half8 a, half8 b, float16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ int vswz(int r) { return (0x6CA0 >> (4 * (r & 3))) & 15; }

// acc += a . b with the accumulator in AGPRs (the file's MFMAs are built in VGPR form). The
// leading s_nop covers a VALU write of a or b just before (2 wait states); the MFMA pipe
// takes 32 cycles an instruction, so it costs no issue slot the pipe could have used.
__device__ __forceinline__ void mfma32_acc(float16v& acc, half8 a, half8 b) {
    asm("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(acc) : "v"(a), "v"(b));
}

}  // namespace g4a
