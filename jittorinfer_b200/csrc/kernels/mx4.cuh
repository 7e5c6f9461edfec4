// Microscaled 4-bit weights in the order in which the products read them.
//
// A matrix [N][K] is cut into chunks of 128 columns.  codes [chunk][row][64 bytes], scales [chunk][row][4 bytes], rows padded to a multiple of 32, all
// zeros behind the last row or column; codes two to a byte, the lower half first, scales E8M0.  A gated pair is one matrix in which 16 rows of the
// gate alternate with 16 of the up matrix.  So a tile of rows is one block of memory for the tensor maps of the tiled products, and 32
// rows of a chunk are 2048 + 128 bytes in a row for the products of a few tokens.  Those read `factors` in place of the scales (below).
//
// The latter feed mma.m16n8k16 in fp16.  The order of columns within a chunk is free as long as the activations share it: lane 4 g + t
// holds the 32 columns 32 t .. of rows g and g + 8, that is 16 bytes and one scale each, and step s of the chunk's eight multiplies its columns 4 s
// .. 4 s + 3.  Decoding is one conversion instruction a byte (E2M1 pair to fp16 pair) and one product with the block's scale.  (Masks and shifts to
// bf16 took eleven integer instructions for eight weights; 16 warps of an SM decoded and multiplied 38 weights a clock so, 66 with the
// conversion.)  fp16 cannot hold every scale, so a factor is relative to the largest scale of its row's blocks with a value: the upper byte of 2^(13 -
// (largest - scale)) in fp16, exact up to 27 binades below the largest and 0 beyond, where a weight is less than 2^-24 of the row's largest (6 2^-28
// of a value that is half its scale at least): layers of weights that have such rows run as tiled products.  A row has an exponent (int) that its sum
// is multiplied with.  A block without a number (scale 255) has codes 0 and a factor of infinity.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace mx4 {

constexpr int COLS = 128;             // columns of a chunk
constexpr int CODES = 64, SCALES = 4; // bytes of a row in it
constexpr int ROWS = 32;              // rows are padded to
constexpr int TOP = 13;               // the largest scale of a row is 2^TOP: 6 * 2^13 is a number in fp16

__host__ __device__ inline int chunks(int K) { return (K + COLS - 1) / COLS; }
// Rows of a matrix, of a gated pair.
__host__ __device__ inline int rows_of(int N, bool pair) { return pair ? (N + 15) / 16 * 32 : (N + ROWS - 1) / ROWS * ROWS; }

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t s) {
    __half2 x, y;
    *(uint32_t *) &x = a;
    *(uint32_t *) &y = s;
    x = __hmul2(x, y);
    return *(uint32_t *) &x;
}

// The fragments (four registers of two fp16) of two steps from four bytes of row g and of row g + 8; s0, s1: their scales, twice in a register.
__device__ __forceinline__ void decode(uint32_t w0, uint32_t w1, uint32_t s0, uint32_t s1, uint32_t (&a)[2][4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3, c0, c1, c2, c3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %8;\n\t"
        "mov.b32 {c0, c1, c2, c3}, %9;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, c0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, c1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %4, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %5, c2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %6, b3;\n\t"
        "cvt.rn.f16x2.e2m1x2 %7, c3;\n\t}"
        : "=r"(a[0][0]), "=r"(a[0][1]), "=r"(a[0][2]), "=r"(a[0][3]), "=r"(a[1][0]), "=r"(a[1][1]), "=r"(a[1][2]), "=r"(a[1][3])
        : "r"(w0), "r"(w1));
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        a[s][0] = mul2(a[s][0], s0);
        a[s][1] = mul2(a[s][1], s1);
        a[s][2] = mul2(a[s][2], s0);
        a[s][3] = mul2(a[s][3], s1);
    }
}

// A factor's byte as a pair of fp16.
__device__ __forceinline__ uint32_t factor2(uint32_t f) { return f * 0x01000100u; }

// 2^e in fp32 for -126 <= e <= 127; 0 or infinity outside
__device__ __forceinline__ float pow2_normal(int e) { return __uint_as_float((uint32_t) (min(max(e, -127), 128) + 127) << 23); }
// 2^e in fp32, 0 below 2^-149 and infinity above 2^127.
__device__ __forceinline__ float pow2(int e) {
    if (e >= -126) return __uint_as_float((uint32_t) (min(e, 128) + 127) << 23);
    return e < -149 ? 0.f : __uint_as_float(1u << (e + 149));
}
// v 2^e for |e| <= 252, without an overflow or underflow on the way
__device__ __forceinline__ float times_pow2(float v, int e) {
    const int h = e >> 1;
    return v * pow2_normal(h) * pow2_normal(e - h);
}

}  // namespace mx4
