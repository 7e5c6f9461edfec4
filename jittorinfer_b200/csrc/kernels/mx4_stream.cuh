// What the products of a few rows of activations with packed 4-bit weights share: 32 rows of a chunk of weights times tiles of 8 rows of activations by
// mma, the copies that bring chunks, and the order in which a warp reads activations.
//
// Up to 8 rows, one tile, the stream of weights counts, 4096 weights in 2176 bytes, and the instructions on its way: at the memory's rate an SM gets 43
// weights a clock, 2.8 issue slots (of 32 lanes) a weight.  A weight is decoded once for all rows.  The mma bound it in the end: 14 clocks each
// on a quarter of an SM, 70 weights a clock and SM.  (A second tile halves that; more rows run as tiled products.)
//
// Activations are fp16, each row scaled by a power of two to a largest magnitude in [2^14, 2^15): exact for bf16 values down to 2^-29 of
// the row's largest, and within 2^-39 of it below.  They are read as fragments of B: for a chunk, a tile of 8 rows and two steps 2 p, 2 p + 1, lane 4 n + t
// holds the eight columns 32 t + 8 p .. of row n.
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

constexpr int SLOT = 32 * (CODES + SCALES);      // 32 rows of a chunk in shared memory: codes, then factors

// Read once: first to leave the L2 (with sm100::l2_policy_evict_first).
__device__ __forceinline__ void copy16(uint32_t dst, const void * src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "l"(policy) : "memory");
}
// 32 rows of a chunk: this lane's first 16 bytes of codes and factors (of the first eight lanes).
__device__ __forceinline__ void copy_chunk(uint32_t dst, const uint8_t * codes, const uint8_t * factors, uint64_t policy) {
    const int lane = threadIdx.x & 31;
    dst += lane * 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) copy16(dst + i * 512, codes + i * 512, policy);
    if (lane < 8) copy16(dst + 32 * CODES, factors, policy);
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// All but the last n groups of copies are there (n: 0 .. 3).
__device__ __forceinline__ void copies_wait(int n) {
    if (n == 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
    else if (n == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (n == 2) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 3;" ::: "memory");
}

// y[m] (row g: columns 2t, 2t + 1; row g + 8) += rows 16 m .. of a chunk x the same fragments: frag(p) gives this lane's 16 bytes.
template <typename F>
__device__ __forceinline__ void chunk_mma(const uint8_t * chunk, float (&y)[2][4], F frag) {
    const int lane = threadIdx.x & 31;
    uint32_t s[2][2];
    uint4 q[2][2];
#pragma unroll
    for (int m = 0; m < 2; ++m)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = (m * 16 + h * 8) * 4 + lane;          // 4 (row) + t
            s[m][h] = factor2(chunk[32 * CODES + at]);
            q[m][h] = ((const uint4 *) chunk)[at];
        }
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const uint4 v = frag(p);
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const uint4 & a = q[m][0], & b = q[m][1];
            uint32_t f[2][4];
            decode(p == 0 ? a.x : p == 1 ? a.y : p == 2 ? a.z : a.w, p == 0 ? b.x : p == 1 ? b.y : p == 2 ? b.z : b.w, s[m][0], s[m][1], f);
            mma16816(y[m], f[0], v.x, v.y);
            mma16816(y[m], f[1], v.z, v.w);
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

// Eight columns of a row from k on, scaled, as fp16 (zeros from column K on; K a multiple of 32).
__device__ __forceinline__ uint4 frag_of(const __nv_bfloat16 * row, int k, int K, float unit) {
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (k >= K) return v;
    const uint4 in = *(const uint4 *) (row + k);
    const uint32_t w[4] = {in.x, in.y, in.z, in.w};
    uint32_t o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(*(const __nv_bfloat162 *) &w[i]);
        const __half2 h = __floats2half2_rn(f.x * unit, f.y * unit);
        o[i] = *(const uint32_t *) &h;
    }
    return make_uint4(o[0], o[1], o[2], o[3]);
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
