// Microscaled 4-bit weights in the order in which the products read them.
//
// A matrix [N][K] is cut into row blocks of 16 rows and chunks of 128 columns.  A chunk is 1088 bytes: two units of 64 columns, 16 bytes for
// each lane of a warp (lane = 4 g + t, word i = columns 16 i .. 16 i + 15 of the unit), then 8 scale bytes for each g: the four blocks of 32
// columns of row g, those of row g + 8.  The chunks of a row block follow one another, a gated pair alternates row blocks (gate, up), and
// everything behind the last row or column is zero.  A word's bytes are what one lane feeds mma.m16n8k16 as the fragment of A: row g
// columns 2t, 2t + 1; row g + 8 the same; row g columns 2t + 8, 2t + 9; row g + 8 the same.
//
// Decoding is one conversion instruction a byte (E2M1 pair to fp16 pair) and one product with the block's scale.  (Masks and shifts to bf16 took
// eleven integer instructions a word; 16 warps of an SM decoded and multiplied 38 weights a clock so, 66 with the conversion.)  fp16 cannot
// hold every scale, so scales are kept relative to the largest of their row: the scale byte is the upper byte of 2^(13 - (largest - scale)) in fp16,
// exact up to 27 binades below the largest and 0 beyond, where a weight is less than 2^-25 of the row's largest; and a row has an exponent
// (int, next to the packed bytes) that its sum is multiplied with.  Infinity times the code 0 makes a block NaN.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

namespace mx4 {

constexpr int ROWS = 16;              // rows of a block
constexpr int COLS = 128;             // columns of a chunk
constexpr int CHUNK = 1088;           // bytes of a chunk: 2 * 512 + 8 * 8
constexpr int SCALES = 1024;          // offset of the scales in a chunk
constexpr int TOP = 13;               // the largest scale of a row is 2^TOP: 6 * 2^13 is a number in fp16

__host__ __device__ inline int chunks(int K) { return (K + COLS - 1) / COLS; }
__host__ __device__ inline int row_blocks(int N) { return (N + ROWS - 1) / ROWS; }

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t s) {
    __half2 x, y;
    *(uint32_t *) &x = a;
    *(uint32_t *) &y = s;
    x = __hmul2(x, y);
    return *(uint32_t *) &x;
}

// The fragment (four registers of two fp16) of a word; s0, s1: scales of row g and row g + 8, twice in a register.
__device__ __forceinline__ void decode(uint32_t w, uint32_t s0, uint32_t s1, uint32_t (&a)[4]) {
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
        : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3])
        : "r"(w));
    a[0] = mul2(a[0], s0);
    a[1] = mul2(a[1], s1);
    a[2] = mul2(a[2], s0);
    a[3] = mul2(a[3], s1);
}

// Scale byte `j` of a word as a pair of fp16.
__device__ __forceinline__ uint32_t scale2(uint32_t f, int j) { return __byte_perm(f, 0u, 0x0404u | (uint32_t) j << 4 | (uint32_t) j << 12); }

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
