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
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const T * __restrict__ x, long long ld, uint32_t * __restrict__ codes,
                                                       uint8_t * __restrict__ scales, long long ld_s, long long n8, int per_row, int vec) {
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    for (long long i0 = (long long) blockIdx.x * blockDim.x; i0 < n8; i0 += (long long) gridDim.x * blockDim.x) {
        const long long i = i0 + threadIdx.x;
        const long long row = i / per_row;
        float y[8];
        uint32_t top = 0;
        if (i < n8) {
            const T * p = x + row * ld + (i - row * per_row) * 8;
            Vec8<T> in;
            if (vec) in = *(const Vec8<T> *) p;
            else
#pragma unroll
                for (int j = 0; j < 8; ++j) in.v[j] = p[j];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                y[j] = to_f(in.v[j]);
                top = max(top, __float_as_uint(y[j]) & 0x7fffffffu);
            }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (i >= n8) continue;
        const int field = (int) (top >> 23);
        const int byte = field == 255 ? 255 : max(field - 2, 0);
        const float inv = __uint_as_float((uint32_t) (254 - byte) << 23);          // 2^(127 - byte)
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] *= inv;
        codes[i] = byte == 255 ? 0u : to_e2m1(y);
        if ((i & 3) == 0) scales[row * ld_s + ((i - row * per_row) >> 2)] = (uint8_t) byte;
    }
}

__device__ __forceinline__ float code_value(uint32_t c) {
    const uint32_t m = c & 7;
    const float v = m < 2 ? 0.5f * m : __uint_as_float(((m >> 1) + 126) << 23 | (m & 1) << 22);
    return c & 8 ? -v : v;
}

template <typename T>
__global__ void __launch_bounds__(256) dequantize_kernel(const uint32_t * __restrict__ codes, const uint8_t * __restrict__ scales, long long ld_s,
                                                         T * __restrict__ out, long long n8, int per_row) {
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    for (long long i = (long long) blockIdx.x * blockDim.x + threadIdx.x; i < n8; i += (long long) gridDim.x * blockDim.x) {
        const long long row = i / per_row;
        const uint32_t w = codes[i], s = scales[row * ld_s + ((i - row * per_row) >> 2)];
        Vec8<T> o;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            // 2^(s - 127) in two steps: s = 0 is below the normal numbers
            const float v = s == 255 ? __uint_as_float(0x7fffffffu)
                                     : code_value(w >> (4 * j)) * __uint_as_float((s > 0 ? s : 1u) << 23) * (s > 0 ? 1.f : 0.5f);
            from_f(v, o.v[j]);
        }
        *(Vec8<T> *) (out + i * 8) = o;
    }
}

// ---- weights: row-major codes to the order of mx4.cuh ----------------------------------------------------------------------------
// Exponents of the rows: the largest scale of a row less 127 and TOP (a row without a number: of scale 1).  One warp a row; step, first: a
// gated pair's matrices take every second row block.
__global__ void __launch_bounds__(128) row_exponent_kernel(const uint8_t * __restrict__ scales, long long ld_s, int * __restrict__ exps, int N, int K, int step,
                                                           int first) {
    const int lane = threadIdx.x & 31, r = blockIdx.x * 4 + (threadIdx.x >> 5), m = blockIdx.y, rows = mx4::row_blocks(N) * mx4::ROWS;
    if (r >= rows) return;
    int top = -1;
    if (r < N)
        for (int i = lane; i < K / 32; i += 32) {
            const int e = scales[((size_t) m * N + r) * ld_s + i];
            if (e != 255) top = max(top, e);
        }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) exps[((size_t) m * (rows / mx4::ROWS) * step + (r / mx4::ROWS) * step + first) * mx4::ROWS + r % mx4::ROWS] = (top < 0 ? 127 : top) - 127 - mx4::TOP;
}

// One warp a chunk.
__global__ void __launch_bounds__(128) pack_kernel(const uint8_t * __restrict__ codes, const uint8_t * __restrict__ scales,
                                                   long long ld_s, const int * __restrict__ exps, uint8_t * __restrict__ out, int N, int K,
                                                   long long out_stride, int step, int first) {
    const int C = mx4::chunks(K), lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const long long id = (long long) blockIdx.x * 4 + (threadIdx.x >> 5);
    const int B = mx4::row_blocks(N);
    if (id >= (long long) B * C) return;
    const int b = (int) (id / C), c = (int) (id % C), m = blockIdx.y;
    codes += (size_t) m * N * (K / 2);
    scales += (size_t) m * N * ld_s;
    uint8_t * dst = out + (size_t) m * out_stride + ((size_t) (b * step + first) * C + c) * mx4::CHUNK;
    const int r0 = b * mx4::ROWS + g, r1 = r0 + 8, k0 = c * mx4::COLS;
    auto pair = [&](int r, int k) -> uint32_t {       // two codes of row r, columns k and k + 1
        if (r >= N || k >= K || scales[(size_t) r * ld_s + k / 32] == 255) return 0u;
        return codes[(size_t) r * (K / 2) + k / 2];
    };
    for (int u = 0; u < 2; ++u) {
        uint32_t w[4];
        for (int i = 0; i < 4; ++i) {
            const int k = k0 + 64 * u + 16 * i + 2 * t;
            w[i] = pair(r0, k) | pair(r1, k) << 8 | pair(r0, k + 8) << 16 | pair(r1, k + 8) << 24;
        }
        ((uint4 *) dst)[u * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (t < 2) {
        const int r = t == 0 ? r0 : r1, top = exps[((size_t) m * B * step + b * step + first) * mx4::ROWS + r % mx4::ROWS] + 127 + mx4::TOP;
        uint32_t f = 0;
        for (int blk = 0; blk < 4; ++blk) {
            const int kb = k0 / 32 + blk;
            if (r >= N || kb >= K / 32) continue;
            const int e = scales[(size_t) r * ld_s + kb];
            f |= (uint32_t) (e == 255 ? 31 : max(0, 15 + mx4::TOP - (top - e))) << (8 * blk + 2);
        }
        ((uint32_t *) (dst + mx4::SCALES))[g * 2 + t] = f;
    }
}

// ---- the product on CUDA cores: fp32 activations, and every shape ------------------------------------------------------------------
// A warp holds one row block (of a pair: two) for eight rows of x; a lane multiplies its weights of rows g and g + 8, four lanes share a row.
constexpr int ST = 8;

template <typename T, bool PAIR>
__global__ void __launch_bounds__(128) product_kernel(const jib_mx4_desc d) {
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    constexpr int M = PAIR ? 2 : 1;
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, e = blockIdx.z;
    const int C = mx4::chunks(d.K), b = blockIdx.x * 4 + (threadIdx.x >> 5);
    if (b >= mx4::row_blocks(d.N)) return;
    long long base = 0, rows = d.T;
    if (d.seg != nullptr) {
        base = d.seg[e];
        rows = d.seg[e + 1] - base;
    }
    const long long t0 = (long long) blockIdx.y * ST;
    if (t0 >= rows) return;
    const int nt = (int) (rows - t0 < ST ? rows - t0 : ST);
    const T * xr[ST];
#pragma unroll
    for (int j = 0; j < ST; ++j) {
        const long long r = base + t0 + (j < nt ? j : 0);
        xr[j] = (const T *) d.x + (d.src != nullptr ? (long long) d.src[r] : r) * d.ldx;
    }
    const uint8_t * w = (const uint8_t *) d.w + (size_t) e * d.w_stride + (size_t) b * M * C * mx4::CHUNK;
    const int * ex = d.w_exp + ((size_t) e * mx4::row_blocks(d.N) + b) * M * mx4::ROWS;
    float unit[M][2];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        unit[m][0] = mx4::pow2(ex[m * mx4::ROWS + g]);
        unit[m][1] = mx4::pow2(ex[m * mx4::ROWS + g + 8]);
    }
    float acc[M][2][ST] = {};
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const uint8_t * p = w + ((size_t) m * C + c) * mx4::CHUNK;
            const uint2 f = ((const uint2 *) (p + mx4::SCALES))[g];
            for (int u = 0; u < 2; ++u) {
                const uint4 q = ((const uint4 *) p)[u * 32 + lane];
                const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int k = c * mx4::COLS + u * 64 + i * 16 + 2 * t;
                    if (k >= d.K) break;
                    uint32_t a[4];
                    mx4::decode(word[i], mx4::scale2(f.x, 2 * u + i / 2), mx4::scale2(f.y, 2 * u + i / 2), a);
                    float2 v[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        v[j] = __half22float2(*(const __half2 *) &a[j]);
                        v[j].x *= unit[m][j & 1];
                        v[j].y *= unit[m][j & 1];
                    }
#pragma unroll
                    for (int j = 0; j < ST; ++j) {
                        if (j >= nt) break;
                        const float x0 = to_f(xr[j][k]), x1 = to_f(xr[j][k + 1]), x2 = to_f(xr[j][k + 8]), x3 = to_f(xr[j][k + 9]);
                        acc[m][0][j] += v[0].x * x0 + v[0].y * x1 + v[2].x * x2 + v[2].y * x3;
                        acc[m][1][j] += v[1].x * x0 + v[1].y * x1 + v[3].x * x2 + v[3].y * x3;
                    }
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
            const int n = b * mx4::ROWS + 8 * h + g;
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

// CTAs of `per` items each, at most a few waves (the kernels stride on).
unsigned grid_for(long long items, int per) {
    const long long n = (items + per - 1) / per;
    const int sms = jib::sm_count();
    const long long most = (long long) (sms > 0 ? sms : 148) * 32;
    return (unsigned) (n < most ? n : most);
}

}  // namespace

extern "C" {

// x [rows][cols], rows ld elements apart; type 0 bf16, 1 fp16, 2 fp32.  codes [rows][cols / 2], scales [rows][cols / 32], rows ld_s bytes apart.
JIB_EXPORT int jib_mx4_quantize(const void * x, int type, long long ld, void * codes, void * scales, long long ld_s, int rows, int cols, void * stream) {
    if (rows <= 0) return 0;
    if (cols <= 0 || cols % 32 || ld_s < cols / 32 || type < 0 || type > 2) return JIB_E_ARG;
    const int el = type == 2 ? 4 : 2, per_row = cols / 8;
    const long long n8 = (long long) rows * per_row;
    const int vec = ((uintptr_t) x | (uintptr_t) (ld * el)) % (size_t) 16 == 0;
    const unsigned grid = grid_for(n8, 256);
    cudaStream_t s = (cudaStream_t) stream;
    if (type == 0) JIB_LAUNCH((quantize_kernel<bf16>), grid, 256, 0, s, (const bf16 *) x, ld, (uint32_t *) codes, (uint8_t *) scales, ld_s, n8, per_row, vec);
    if (type == 1) JIB_LAUNCH((quantize_kernel<__half>), grid, 256, 0, s, (const __half *) x, ld, (uint32_t *) codes, (uint8_t *) scales, ld_s, n8, per_row, vec);
    if (type == 2) JIB_LAUNCH((quantize_kernel<float>), grid, 256, 0, s, (const float *) x, ld, (uint32_t *) codes, (uint8_t *) scales, ld_s, n8, per_row, vec);
    return launched();
}

// The values of `rows` rows, to out [rows][cols] of the type.
JIB_EXPORT int jib_mx4_dequantize(const void * codes, const void * scales, long long ld_s, void * out, int type, long long rows, int cols, void * stream) {
    if (rows <= 0) return 0;
    if (cols <= 0 || cols % 32 || ld_s < cols / 32 || type < 0 || type > 2) return JIB_E_ARG;
    const long long n8 = rows * (cols / 8);
    const unsigned grid = grid_for(n8, 256);
    cudaStream_t s = (cudaStream_t) stream;
    if (type == 0) JIB_LAUNCH((dequantize_kernel<bf16>), grid, 256, 0, s, (const uint32_t *) codes, (const uint8_t *) scales, ld_s, (bf16 *) out, n8, cols / 8);
    if (type == 1) JIB_LAUNCH((dequantize_kernel<__half>), grid, 256, 0, s, (const uint32_t *) codes, (const uint8_t *) scales, ld_s, (__half *) out, n8, cols / 8);
    if (type == 2) JIB_LAUNCH((dequantize_kernel<float>), grid, 256, 0, s, (const uint32_t *) codes, (const uint8_t *) scales, ld_s, (float *) out, n8, cols / 8);
    return launched();
}

// Row-major codes and scales of `batch` matrices [N][K] to the order that the products read; exps [batch][row blocks * step][16]; out_stride:
// bytes of a matrix.
JIB_EXPORT int jib_mx4_pack(const void * codes, const void * scales, long long ld_s, int * exps, void * out, int batch, int N, int K, long long out_stride,
                            int step, int first, void * stream) {
    if (batch <= 0) return 0;
    if (N <= 0 || K <= 0 || K % 32 || ld_s < K / 32 || batch > 65535 || step < 1 || first < 0 || first >= step) return JIB_E_ARG;
    const long long n = (long long) mx4::row_blocks(N) * mx4::chunks(K);
    if ((n + 3) / 4 > 0x7fffffffll || out_stride < n * step * mx4::CHUNK) return JIB_E_ARG;
    cudaStream_t s = (cudaStream_t) stream;
    row_exponent_kernel<<<dim3(mx4::row_blocks(N) * 4, batch), 128, 0, s>>>((const uint8_t *) scales, ld_s, exps, N, K, step, first);
    pack_kernel<<<dim3((unsigned) ((n + 3) / 4), batch), 128, 0, s>>>((const uint8_t *) codes, (const uint8_t *) scales, ld_s, exps, (uint8_t *) out, N, K,
                                                                     out_stride, step, first);
    return launched();
}

JIB_EXPORT int jib_mx4_product_simt(const jib_mx4_desc * d, int f32, void * stream) {
    if (d->T <= 0) return 0;
    if (d->N <= 0 || d->K <= 0 || d->K % 32 || d->batch < 1 || d->batch > 65535) return JIB_E_ARG;
    const long long rows = d->seg != nullptr ? d->max_rows : d->T;
    const dim3 grid((mx4::row_blocks(d->N) + 3) / 4, (unsigned) ((rows + ST - 1) / ST), d->batch);
    if ((rows + ST - 1) / ST > 65535) return JIB_E_ARG;
    cudaStream_t s = (cudaStream_t) stream;
    if (f32) {
        if (d->gated) JIB_LAUNCH((product_kernel<float, true>), grid, 128, 0, s, *d);
        else JIB_LAUNCH((product_kernel<float, false>), grid, 128, 0, s, *d);
    } else {
        if (d->gated) JIB_LAUNCH((product_kernel<bf16, true>), grid, 128, 0, s, *d);
        else JIB_LAUNCH((product_kernel<bf16, false>), grid, 128, 0, s, *d);
    }
    return launched();
}

}  // extern "C"
