// Microscaled 4-bit weights in the order in which the products read them.
//
// A matrix [N][K] is cut into row blocks of 16 rows and chunks of 128 columns.  A chunk is 1088 bytes: two units of 64 columns, 16 bytes for
// each lane of a warp (lane = 4 g + t, word i = columns 16 i .. 16 i + 15 of the unit), then 8 scale bytes for each g: the four blocks of 32
// columns of row g, those of row g + 8.  The chunks of a row block follow one another, a gated pair alternates row blocks (gate, up), and
// everything behind the last row or column is zero.  A word's eight weights are what one lane feeds mma.m16n8k16 as the fragment of A: row g
// columns 2t, 2t + 1; row g + 8 the same; row g columns 2t + 8, 2t + 9; row g + 8 the same.
//
// A weight's bits s e1 e0 m stand where they have to be in bf16 (s at 15, e1 e0 m at 8..6, a value of 2^-126 times the weight), or, for the
// pairs 1 and 2, 3 and 6 places below, so that a shift and a mask take out two weights at a time; pair 3 gets the four bits that are left.
// The scale byte f is the exponent field of the bf16 number 2^126 * 2^(E - 127 - shift), multiplied into the pair: exact, as both factors
// are or carry powers of two.  `shift` is one per matrix, 0 unless a scale is above 2 (then the product's epilogue multiplies it back in).
#pragma once
#include <cuda_bf16.h>
#include <stdint.h>

namespace mx4 {

constexpr int ROWS = 16;              // rows of a block
constexpr int COLS = 128;             // columns of a chunk
constexpr int CHUNK = 1088;           // bytes of a chunk: 2 * 512 + 8 * 8
constexpr int SCALES = 1024;          // offset of the scales in a chunk

__host__ __device__ inline int chunks(int K) { return (K + COLS - 1) / COLS; }
__host__ __device__ inline int row_blocks(int N) { return (N + ROWS - 1) / ROWS; }

// One 16-bit half of pair `j` for a code (the other half is the same, 16 places up).
__host__ __device__ inline uint32_t place(uint32_t c, int j) {
    switch (j) {
        case 0: return (c & 8) << 12 | (c & 7) << 6;
        case 1: return (c & 8) << 9 | (c & 7) << 3;
        case 2: return (c & 8) << 6 | (c & 7);
        default: return (c & 8) << 11 | (c & 4) << 11 | (c & 3) << 10;
    }
}

__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t s) {
    __nv_bfloat162 x, y;
    *(uint32_t *) &x = a;
    *(uint32_t *) &y = s;
    x = __hmul2(x, y);
    return *(uint32_t *) &x;
}

// The fragment (four registers of two bf16) of a word; s0, s1: scales of row g and row g + 8, twice in a register.
__device__ __forceinline__ void decode(uint32_t w, uint32_t s0, uint32_t s1, uint32_t (&a)[4]) {
    constexpr uint32_t M = 0x81C081C0u;
    a[0] = mul2(w & M, s0);
    a[1] = mul2((w << 3) & M, s1);
    a[2] = mul2((w << 6) & M, s0);
    a[3] = mul2(((w << 1) & 0x80008000u) | ((w >> 4) & 0x00C000C0u) | ((w >> 5) & 0x01000100u), s1);
}

// Scale byte `j` of a word as a pair of bf16.
__device__ __forceinline__ uint32_t scale2(uint32_t f, int j) { return ((f >> (8 * j)) & 0xffu) * 0x00800080u; }

}  // namespace mx4
