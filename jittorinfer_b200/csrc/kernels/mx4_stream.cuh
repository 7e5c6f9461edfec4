// What the products of a few rows of activations with packed 4-bit weights share: a chunk of weights times tiles of 8 rows by mma, the bulk
// copies that bring chunks into shared memory, and the order in which a warp reads activations.
//
// Up to 16 rows the stream of weights counts, 2176 weights in 1088 bytes, and the instructions that take a weight out of its four bits:
// eleven integer ones, four products and NT mma for eight weights of a lane, about 160 a warp and chunk, 80 % of the machine's issue
// slots at the memory's rate.  So a weight is decoded once for all rows, and nothing else is done per weight.
//
// Activations are read as fragments of B: for a chunk, a tile of 8 rows and a pair of 16-column steps, lane 4 n + t holds 16 bytes, columns
// 2t, 2t + 1, 2t + 8, 2t + 9 of the first step and of the second of row n.
#pragma once
#include "mx4.cuh"
#include "sm100.cuh"

namespace mx4 {

constexpr int FRAG = 4 * 32 * 16;             // bytes of a chunk's fragments for one tile of 8 rows

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// c (row g: columns 2t, 2t + 1; row g + 8) += chunk (in shared memory) x fragments
template <int NT>
__device__ __forceinline__ void chunk_mma(const uint8_t * chunk, const uint4 (&b)[NT][4], float (&c)[NT][4]) {
    const int lane = threadIdx.x & 31;
    const uint2 f = ((const uint2 *) (chunk + SCALES))[lane >> 2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        const uint4 q = ((const uint4 *) chunk)[u * 32 + lane];
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t a[4];
            decode(w[i], scale2(f.x, 2 * u + i / 2), scale2(f.y, 2 * u + i / 2), a);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const uint4 & v = b[n][2 * u + i / 2];
                mma16816(c[n], a, i & 1 ? v.z : v.x, i & 1 ? v.w : v.y);
            }
        }
    }
}

// 16 bytes of fragments: row n's columns of steps 2 pair and 2 pair + 1 of chunk c (zeros from column K on; K a multiple of 16).
__device__ __forceinline__ uint4 gather_frag(const __nv_bfloat16 * row, int c, int pair, int t, int K) {
    const int k = c * COLS + pair * 32 + 2 * t;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    if (c * COLS + pair * 32 < K) {
        v.x = *(const uint32_t *) (row + k);
        v.y = *(const uint32_t *) (row + k + 8);
    }
    if (c * COLS + pair * 32 + 16 < K) {
        v.z = *(const uint32_t *) (row + k + 16);
        v.w = *(const uint32_t *) (row + k + 24);
    }
    return v;
}

// `bytes` (a multiple of 16) of weights to shared memory, first to leave the L2.
__device__ __forceinline__ void bulk_load(void * dst, const void * src, uint32_t bytes, uint64_t * bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;"
                 ::"r"(sm100::smem_u32(dst)), "l"(src), "r"(bytes), "r"(sm100::smem_u32(bar)), "l"(policy)
                 : "memory");
}

__device__ __forceinline__ float gated(float z, float u, int act) {
    const float a = act == JIB_ACT_GELU_TANH ? 1.5957691216057308f * (z + 0.044715f * z * z * z) : z;
    return z / (1.f + expf(-a)) * u;
}

}  // namespace mx4
