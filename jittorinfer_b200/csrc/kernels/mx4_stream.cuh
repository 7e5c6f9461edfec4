// What the products of a few rows of activations with packed 4-bit weights share: a chunk of weights times tiles of 8 rows by mma, the loads
// that bring chunks, and the order in which a warp reads activations.
//
// Up to 16 rows the stream of weights counts, 2048 weights in 1088 bytes.  A weight is decoded once for all rows: per eight weights of a lane four
// conversions, four products and an mma for each tile of 8 rows.  The mma bound it: 14 clocks each on a quarter of an SM, 70 weights a
// clock and SM for one tile (the memory delivers 43), 35 for two.
//
// Activations are fp16, each row scaled by a power of two to a largest magnitude in [2^14, 2^15): exact for bf16 values down to 2^-29 of
// the row's largest, and within 2^-39 of it below.  They are read as fragments of B: for a chunk, a tile of 8 rows and a pair of 16-column
// steps, lane 4 n + t holds 16 bytes, columns 2t, 2t + 1, 2t + 8, 2t + 9 of the first step and of the second of row n.
#pragma once
#include <cuda_bf16.h>

#include "mx4.cuh"
#include "sm100.cuh"

namespace mx4 {

constexpr int FRAG = 4 * 32 * 16;             // bytes of a chunk's fragments for one tile of 8 rows

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Two chunks, `apart` bytes from one another in memory, side by side to this warp's shared memory: read once, so past the L1 and first to leave the
// L2 (with sm100::l2_policy_evict_first).
__device__ __forceinline__ void copy16(uint32_t dst, const void * src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
__device__ __forceinline__ void copy_chunks(uint32_t dst, const uint8_t * src, size_t apart, uint64_t policy) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int u = 0; u < 2; ++u) copy16(dst + m * CHUNK + (u * 32 + lane) * 16, src + m * apart + (u * 32 + lane) * 16, policy);
    if (lane < 8) copy16(dst + (lane >> 2) * CHUNK + SCALES + (lane & 3) * 16, src + (lane >> 2) * apart + SCALES + (lane & 3) * 16, policy);
}
// The same through no cache policy; `bytes` 16, or 0: zeros.
__device__ __forceinline__ void copy16_or_zero(uint32_t dst, const void * src, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last n groups of copies are there (n: 0 .. 3).
__device__ __forceinline__ void copies_wait(int n) {
    if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// y[m] (row g: columns 2t, 2t + 1; row g + 8) += chunk m x the same fragments: frag(n, pair) gives this lane's 16 bytes.
template <int NT, typename F>
__device__ __forceinline__ void chunks_mma(const uint8_t * chunks, float (&y)[2][NT][4], F frag) {
    const int lane = threadIdx.x & 31;
    uint2 f[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) f[m] = *(const uint2 *) (chunks + m * CHUNK + SCALES + (lane >> 2) * 8);
    uint4 q[2];
#pragma unroll
    for (int p = 0; p < 4; ++p) {          // 32 columns: two steps, one scale a row
        if ((p & 1) == 0)
#pragma unroll
            for (int m = 0; m < 2; ++m) q[m] = *(const uint4 *) (chunks + m * CHUNK + ((p >> 1) * 32 + lane) * 16);
        uint4 v[NT];
#pragma unroll
        for (int n = 0; n < NT; ++n) v[n] = frag(n, p);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const uint32_t s0 = scale2(f[m].x, p), s1 = scale2(f[m].y, p);
            uint32_t a[4];
            decode(p & 1 ? q[m].z : q[m].x, s0, s1, a);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(y[m][n], a, v[n].x, v[n].y);
            decode(p & 1 ? q[m].w : q[m].y, s0, s1, a);
#pragma unroll
            for (int n = 0; n < NT; ++n) mma16816(y[m][n], a, v[n].z, v[n].w);
        }
    }
}

// A bounded wait in few instructions, for kernels whose loops have to stay in the instruction cache: up to 2^21 tries that a thread may be suspended
// in for a microsecond each.
__device__ __forceinline__ bool wait(uint64_t * bar, uint32_t parity) {
    const uint32_t at = sm100::smem_u32(bar);
    uint32_t ok = 0;
#pragma unroll 1
    for (int i = 0; i < 1 << 21; ++i) {
        asm volatile("{\n\t.reg .pred P;\n\tmbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, 1000;\n\tselp.b32 %0, 1, 0, P;\n\t}"
                     : "=r"(ok) : "r"(at), "r"(parity) : "memory");
        if (ok) break;
    }
    return ok != 0;
}
__device__ __forceinline__ bool wait_all(uint64_t * bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); }

// The exponent of a largest magnitude (bits of the fp32 value): values times 2^(14 - exponent) fit fp16.  0 and what is below 2^-112 count as that.
__device__ __forceinline__ int top_exponent(uint32_t bits) { return max(min((int) (bits >> 23), 254) - 127, -112); }

// Columns 16 s + 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of a row, scaled, as two registers of fp16 (zeros from column K on; K a multiple of 16).
__device__ __forceinline__ uint2 frag_step(const __nv_bfloat16 * row, int s, int t, int K, float unit) {
    if (16 * s >= K) return make_uint2(0u, 0u);
    const float2 a = __bfloat1622float2(*(const __nv_bfloat162 *) (row + 16 * s + 2 * t)), b = __bfloat1622float2(*(const __nv_bfloat162 *) (row + 16 * s + 2 * t + 8));
    const __half2 x = __floats2half2_rn(a.x * unit, a.y * unit), y = __floats2half2_rn(b.x * unit, b.y * unit);
    return make_uint2(*(const uint32_t *) &x, *(const uint32_t *) &y);
}

// `bytes` (a multiple of 16) to shared memory.
__device__ __forceinline__ void bulk_load(void * dst, const void * src, uint32_t bytes, uint64_t * bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ float gated(float z, float u, int act) {
    const float a = act == JIB_ACT_GELU_TANH ? 1.5957691216057308f * (z + 0.044715f * z * z * z) : z;
    return __fdividef(z, 1.f + expf(-a)) * u;          // (the quotient is 0 where the divisor is above 2^126)
}

}  // namespace mx4
