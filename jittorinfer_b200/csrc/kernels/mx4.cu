// Microscaled 4-bit tensors (codes E2M1 in blocks of 32 along a row, one power-of-two scale a block): quantising rows, expanding them,
// laying weights out for the products, and the product on CUDA cores.
//
// The reference keeps block-quantised weights in GGUF files and multiplies them through its device library (ggml/src/ggml-cann/
// aclnn_ops.cpp, quantised mul_mat); it has no microscaled type.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "jib_kernels.h"
#include "mx4_stream.cuh"
#include "pdl.cuh"

namespace {

typedef __nv_bfloat16 bf16;

__device__ __forceinline__ float to_f(bf16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f(float v) { return v; }
__device__ __forceinline__ void from_f(float v, bf16 & o) { o = __float2bfloat16(v); }
__device__ __forceinline__ void from_f(float v, __half & o) { o = __float2half(v); }
__device__ __forceinline__ void from_f(float v, float & o) { o = v; }

template <typename T>
struct alignas(16) Vec8 {
    T v[8];
};

// Eight values to eight codes, the first in the lowest four bits: nearest, ties to even, at most 6 in magnitude.
__device__ __forceinline__ uint32_t to_e2m1(const float (&y)[8]) {
    uint32_t r;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(r)
        : "f"(y[0]), "f"(y[1]), "f"(y[2]), "f"(y[3]), "f"(y[4]), "f"(y[5]), "f"(y[6]), "f"(y[7]));
    return r;
}

// ---- quantise: four lanes a block, eight values each ---------------------------------------------------------------------------
// Scale 2^e with e = floor(log2 max) - 2, so that the largest value lies in [4, 8) and the largest code is 6; the exponent field of
// the largest value is floor(log2) + 127, hence the byte e + 127 = field - 2, at least 0.  Dividing by 2^e is a product with
// 2^-e, exact.  A block with an infinity or NaN gets the scale NaN (255) and codes 0.
// A thread keeps its eight columns and walks down the rows (no division by the row's length: 36 us with one), ROWS loads in flight.  Bound by memory:
// 4096 x 5120 bf16 to 4 bits and back in 23 us, 4.6 TB/s.
constexpr int ROWS = 4;

template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T * __restrict__ x, long long ld, uint32_t * __restrict__ codes,
                                                       uint8_t * __restrict__ scales, long long ld_s, int rows, int per_row, int vec) {
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    const int col = blockIdx.x * blockDim.x + threadIdx.x;
#pragma unroll 1
    for (long long r0 = (long long) blockIdx.y * ROWS; r0 < rows; r0 += (long long) gridDim.y * ROWS) {
        Vec8<T> in[ROWS];
#pragma unroll
        for (int h = 0; h < ROWS; ++h) {
            const T * p = x + (r0 + h) * ld + (long long) col * 8;
            if (r0 + h >= rows || col >= per_row)
#pragma unroll
                for (int j = 0; j < 8; ++j) from_f(0.f, in[h].v[j]);
            else if (vec) in[h] = *(const Vec8<T> *) p;
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) in[h].v[j] = p[j];
        }
#pragma unroll
        for (int h = 0; h < ROWS; ++h) {
            float y[8];
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[j] = to_f(in[h].v[j]);
                top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
            }
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
            if (r0 + h >= rows || col >= per_row) continue;
            const int field = (int) (top >> 23);
            const int byte = field == 255 ? 255 : max(field - 2, 0);
            const float inv = __uint_as_float((uint32_t) (254 - byte) << 23);          // 2^(127 - byte)
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= inv;
            codes[(r0 + h) * per_row + col] = byte == 255 ? 0u : to_e2m1(y);
            if ((col & 3) == 0) scales[(r0 + h) * ld_s + (col >> 2)] = (uint8_t) byte;
        }
    }
}

__device__ __forceinline__ float code_value(uint32_t c) {
    const uint32_t m = c & 7;
    const float v = m < 2 ? 0.5f * m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
    return c & 8 ? -v : v;
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t * __restrict__ codes, const uint8_t * __restrict__ scales, long long ld_s,
                                                         T * __restrict__ out, long long rows, int per_row) {
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    const int col = blockIdx.x * blockDim.x + threadIdx.x;
    if (col >= per_row) return;
#pragma unroll 1
    for (long long r0 = (long long) blockIdx.y * ROWS; r0 < rows; r0 += (long long) gridDim.y * ROWS) {
        uint32_t w[ROWS], s[ROWS];
#pragma unroll
        for (int h = 0; h < ROWS; ++h) {
            w[h] = r0 + h < rows ? codes[(r0 + h) * per_row + col] : 0u;
            s[h] = r0 + h < rows ? scales[(r0 + h) * ld_s + (col >> 2)] : 0u;
        }
#pragma unroll
        for (int h = 0; h < ROWS; ++h) {
            if (r0 + h >= rows) break;
            // 2^(s - 127), of s = 0 below the normal numbers
            const float unit = __uint_as_float(s[h] == 255 ? 0x7fffffffu : s[h] == 0 ? 0x00400000u : s[h] << 23);
            Vec8<T> o;
#pragma unroll
            for (int j = 0; j < 8; j += 2) {
                uint32_t two;
                asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(two) : "r"(w[h] >> (4 * j)));
                const float2 f = __half22float2(*(const __half2 *) &two);
                from_f(f.x * unit, o.v[j]);
                from_f(f.y * unit, o.v[j + 1]);
            }
            *(Vec8<T> *) (out + ((r0 + h) * per_row + col) * 8) = o;
        }
    }
}

// ---- weights: row-major codes to the order of mx4.cuh ----------------------------------------------------------------------------
// Where row r of a matrix stands: of a pair's member `first` of `step` 2, in blocks of 16 rows that alternate.
__device__ __forceinline__ int packed_row(int r, int step, int first) { return step == 1 ? r : (r / 16 * 2 + first) * 16 + r % 16; }

// Whether a block's codes are all 0 or -0.
__device__ __forceinline__ bool no_value(uint4 v) { return ((v.x | v.y | v.z | v.w) & 0x77777777u) == 0u; }

// Exponents of the rows: the largest scale of a block with a value (1 for a row without one) less 127 and TOP.  (A block of zeros can have any scale.)  One
// warp a row.
__global__ void __launch_bounds__(128) row_exponent_kernel(const uint4 * __restrict__ codes, const uint8_t * __restrict__ scales, long long ld_s,
                                                           int * __restrict__ exps, int N, int K, int R, int step, int first) {
    const int lane = threadIdx.x & 31, r = blockIdx.x * 4 + (threadIdx.x >> 5), m = blockIdx.y;
    if (r >= R / step) return;
    int top = -1;
    if (r < N)
        for (int i = lane; i < K / 32; i += 32) {
            const int e = scales[((size_t) m * N + r) * ld_s + i];
            if (e != 255 && !no_value(codes[((size_t) m * N + r) * (K / 32) + i])) top = max(top, e);
        }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) exps[(size_t) m * R + packed_row(r, step, first)] = (top < 0 ? 127 : top) - 127 - mx4::TOP;
}

// A thread moves 32 columns of a row: 16 bytes and a scale.
__global__ void __launch_bounds__(256) pack_kernel(const uint8_t * __restrict__ codes, const uint8_t * __restrict__ scales, long long ld_s,
                                                   const int * __restrict__ exps, uint4 * __restrict__ out, uint8_t * __restrict__ out_scales,
                                                   uint8_t * __restrict__ factors, int * __restrict__ lost, int N, int K, int R, int step, int first) {
    const int C = mx4::chunks(K), rows = R / step, m = blockIdx.y;
    const long long id = (long long) blockIdx.x * blockDim.x + threadIdx.x;
    if (id >= (long long) C * rows * 4) return;
    const int t = (int) (id & 3), r = (int) (id / 4 % rows), c = (int) (id / 4 / rows), b = c * 4 + t;
    const int row = packed_row(r, step, first);
    const size_t at = (((size_t) m * C + c) * R + row) * 4 + t;
    uint4 v = make_uint4(0u, 0u, 0u, 0u);
    int e = 0, f = 0;
    if (r < N && b < K / 32) {
        e = scales[((size_t) m * N + r) * ld_s + b];
        if (factors != nullptr) f = e == 255 ? 31 : min(max(0, 15 + e - 127 - exps[(size_t) m * R + row]), 30);        // (above 15 + TOP only for a block of zeros)
        if (e != 255) v = ((const uint4 *) codes)[((size_t) m * N + r) * (K / 32) + b];
        if (lost != nullptr && f == 0 && !no_value(v)) *lost = 1;
    }
    out[at] = v;
    out_scales[at] = (uint8_t) e;
    if (factors != nullptr) factors[at] = (uint8_t) (f << 2);
}

// ---- the product of fp32 activations, on CUDA cores ------------------------------------------------------------------
// A warp holds 16 rows (of a pair: 16 of each matrix) for eight rows of x; a lane multiplies its columns of rows g and g + 8, four lanes share a row.
constexpr int ST = 8;

template <bool PAIR>
__global__ void __launch_bounds__(128) product_kernel(const jib_mx4_desc d, unsigned first_tile) {
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    constexpr int M = PAIR ? 2 : 1;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, e = blockIdx.z;
    const int C = mx4::chunks(d.K), R = mx4::rows_of(d.N, PAIR), b = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (b * 16 >= d.N) return;
    long long base = 0, rows = d.T;
    if (d.seg != nullptr) {
        base = d.seg[e];
        rows = d.seg[e + 1] - base;
    }
    const long long t0 = (long long) (first_tile + blockIdx.y) * ST;
    if (t0 >= rows) return;
    const int nt = (int) (rows - t0 < ST ? rows - t0 : ST);
    const float * xr[ST];
#pragma unroll
    for (int j = 0; j < ST; ++j) {
        const long long r = base + t0 + (j < nt ? j : 0);
        xr[j] = (const float *) d.x + (d.src != nullptr ? (long long) d.src[r] : r) * d.ldx;
    }
    float acc[M][2][ST] = {};
    for (int c = 0; c < C; ++c) {
        const int k = c * mx4::COLS + 32 * t;
        if (k >= d.K) continue;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const size_t row = ((size_t) e * C + c) * R + (b * M + m) * 16 + h * 8 + g;
                const uint4 q = ((const uint4 *) d.w)[row * 4 + t];
                const uint32_t s = d.w_scales[row * 4 + t], word[4] = {q.x, q.y, q.z, q.w};
                const float unit = s == 255 ? __uint_as_float(0x7fffffffu) : mx4::pow2((int) s - 127);
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float w = code_value(word[i] >> (4 * j)) * unit;
#pragma unroll
                        for (int n = 0; n < ST; ++n)
                            if (n < nt) acc[m][h][n] += w * xr[n][k + 8 * i + j];
                    }
            }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int j = 0; j < ST; ++j) {
            float s[M];
#pragma unroll
            for (int m = 0; m < M; ++m) {
                s[m] = acc[m][h][j];
                s[m] += __shfl_xor_sync(0xffffffffu, s[m], 1);
                s[m] += __shfl_xor_sync(0xffffffffu, s[m], 2);
            }
            const int n = b * 16 + 8 * h + g;
            if (t != 0 || j >= nt || n >= d.N) continue;
            const long long r = base + t0 + j;
            float y = PAIR ? mx4::gated(s[0], s[M - 1], d.act) : s[0];
            if (d.residual != nullptr) {
                const long long ri = r * d.ldr + n;
                y += d.res_f32 ? ((const float *) d.residual)[ri] : to_f(((const bf16 *) d.residual)[ri]);
            }
            if (d.out_f32) ((float *) d.out)[r * d.ldo + n] = y;
            else ((bf16 *) d.out)[r * d.ldo + n] = __float2bfloat16(y);
        }
}

int launched() { return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH; }

// Threads of a CTA and a grid for `per_row` threads a row and ROWS rows a step: x along a row, y down the rows, a few waves at most (the kernels stride on).
dim3 grid_for(long long rows, int per_row, int * threads) {
    const int nx = (per_row + 255) / 256;
    *threads = ((per_row + nx - 1) / nx + 31) / 32 * 32;
    const int sms = jib::sm_count();
    const long long most = ((long long) (sms > 0 ? sms : 148) * 4096 / *threads + nx - 1) / nx, ny = (rows + ROWS - 1) / ROWS;
    return dim3((unsigned) nx, (unsigned) (ny < most ? ny : most < 65535 ? most : 65535));
}

}  // namespace

extern "C" {

// x [rows][cols], rows ld elements apart; type 0 bf16, 1 fp16, 2 fp32.  codes [rows][cols / 2], scales [rows][cols / 32], rows ld_s bytes apart.
JIB_EXPORT int jib_mx4_quantize(const void * x, int type, long long ld, void * codes, void * scales, long long ld_s, int rows, int cols, void * stream) {
    if (rows <= 0) return 0;
    if (cols <= 0 || cols % 32 || ld_s < cols / 32 || type < 0 || type > 2) return JIB_E_ARG;
    const int el = type == 2 ? 4 : 2, per_row = cols / 8, vec = ((uintptr_t) x | (uintptr_t) (ld * el)) % (size_t) 16 == 0;
    int th;
    const dim3 grid = grid_for(rows, per_row, &th);
    cudaStream_t s = (cudaStream_t) stream;
    if (type == 0) JIB_LAUNCH((quantize_kernel<bf16>), grid, th, 0, s, (const bf16 *) x, ld, (uint32_t *) codes, (uint8_t *) scales, ld_s, rows, per_row, vec);
    if (type == 1) JIB_LAUNCH((quantize_kernel<__half>), grid, th, 0, s, (const __half *) x, ld, (uint32_t *) codes, (uint8_t *) scales, ld_s, rows, per_row, vec);
    if (type == 2) JIB_LAUNCH((quantize_kernel<float>), grid, th, 0, s, (const float *) x, ld, (uint32_t *) codes, (uint8_t *) scales, ld_s, rows, per_row, vec);
    return launched();
}

// The values of `rows` rows, to out [rows][cols] of the type.
JIB_EXPORT int jib_mx4_dequantize(const void * codes, const void * scales, long long ld_s, void * out, int type, long long rows, int cols, void * stream) {
    if (rows <= 0) return 0;
    if (cols <= 0 || cols % 32 || ld_s < cols / 32 || type < 0 || type > 2) return JIB_E_ARG;
    int th;
    const dim3 grid = grid_for(rows, cols / 8, &th);
    cudaStream_t s = (cudaStream_t) stream;
    if (type == 0) JIB_LAUNCH((dequantize_kernel<bf16>), grid, th, 0, s, (const uint32_t *) codes, (const uint8_t *) scales, ld_s, (bf16 *) out, rows, cols / 8);
    if (type == 1) JIB_LAUNCH((dequantize_kernel<__half>), grid, th, 0, s, (const uint32_t *) codes, (const uint8_t *) scales, ld_s, (__half *) out, rows, cols / 8);
    if (type == 2) JIB_LAUNCH((dequantize_kernel<float>), grid, th, 0, s, (const uint32_t *) codes, (const uint8_t *) scales, ld_s, (float *) out, rows, cols / 8);
    return launched();
}

// Row-major codes and scales of `batch` matrices [N][K] to the order that the products read: out, out_scales, factors and exps of all (of pairs, with step 2, the
// member `first`).  factors and exps NULL: not made.  lost (or NULL): set to 1 where a weight's factor is 0 and the weight is not.
JIB_EXPORT int jib_mx4_pack(const void * codes, const void * scales, long long ld_s, void * out, void * out_scales, void * factors, int * exps, int * lost, int batch,
                            int N, int K, int step, int first, void * stream) {
    if (batch <= 0) return 0;
    if (N <= 0 || K <= 0 || K % 32 || ld_s < K / 32 || batch > 65535 || step < 1 || step > 2 || first < 0 || first >= step ||
        (factors == nullptr) != (exps == nullptr) || (lost != nullptr && factors == nullptr))
        return JIB_E_ARG;
    if (((uintptr_t) codes | (uintptr_t) out) & 15) return JIB_E_ALIGN;
    const int R = mx4::rows_of(N, step == 2);
    const long long n = (long long) mx4::chunks(K) * (R / step) * 4;
    if ((n + 255) / 256 > 0x7fffffffll) return JIB_E_ARG;
    cudaStream_t s = (cudaStream_t) stream;
    if (exps != nullptr) row_exponent_kernel<<<dim3((R / step + 3) / 4, batch), 128, 0, s>>>((const uint4 *) codes, (const uint8_t *) scales, ld_s, exps, N, K, R, step, first);
    pack_kernel<<<dim3((unsigned) ((n + 255) / 256), batch), 256, 0, s>>>((const uint8_t *) codes, (const uint8_t *) scales, ld_s, exps, (uint4 *) out,
                                                                         (uint8_t *) out_scales, (uint8_t *) factors, lost, N, K, R, step, first);
    return launched();
}

JIB_EXPORT int jib_mx4_product_simt(const jib_mx4_desc * d, void * stream) {
    if (d->T <= 0) return 0;
    if (d->N <= 0 || d->K <= 0 || d->K % 32 || d->batch < 1 || d->batch > 65535) return JIB_E_ARG;
    const long long rows = d->seg != nullptr ? d->max_rows : d->T;
    cudaStream_t s = (cudaStream_t) stream;
    // A grid is 65535 tiles of rows high at most.  (A kernel that strides on took 432 us for a row of 10944 by 2048 instead of 393; rows along the grid's other
    // side 713 for 300 by 2048 x 2048 instead of 646.)
    const long long tiles = (rows + ST - 1) / ST;
    for (long long t = 0; t < tiles; t += 65535) {
        const dim3 grid(((d->N + 15) / 16 + 3) / 4, (unsigned) (tiles - t < 65535 ? tiles - t : 65535), d->batch);
        if (d->gated) JIB_LAUNCH((product_kernel<true>), grid, 128, 0, s, *d, (unsigned) t);
        else JIB_LAUNCH((product_kernel<false>), grid, 128, 0, s, *d, (unsigned) t);
    }
    return launched();
}

}  // extern "C"
