// Products of bf16 activations with packed 4-bit weights on the block-scaled tensor cores: out[r][n] = f(sum_k x[r][k] w[n][k]) (+ residual), dense or
// grouped by expert.
//
// The weights go to the tensor cores as they are: the tensor map of type 16U4_ALIGN16B spreads 4-bit codes over bytes in shared memory and
// tcgen05.mma.kind::mxf8f6f4 takes them as E2M1 with their block's scale, 128 rows a tile.  So no instruction touches a weight.  Its other operand can have 8
// bits at most; a bf16 activation is the sum of two E4M3 numbers, the first its value rounded to four significant bits, the second what is left, each
// with a scale for 32 columns.  That sum is the bf16 value down to 2^-11 of the block's largest magnitude and within 2^-21 of the largest below.  At
// twice the rate of bf16 both planes cost what a bf16 product costs.  (Hidden units on their way to the next product are rounded to bf16, whose eight
// bits the planes then hold.)
//
// Up to 96 rows of x (WIDE) both planes are one operand of twice the rows, and the sums of the two meet in the epilogue.  Dense tiles then belong to one CTA,
// experts' tiles to two (PAIR, cta_group::2: 256 weights, each CTA keeps one plane).  Above 96 rows two CTAs share 256 weights by up to 192 rows of x, of
// which each keeps half: the products are bound by their traffic with shared memory, and the rows of x are half of it.  1531 rows by 2 x 10944 x 2048:
// 132 us with tiles of one CTA, 102 us with pairs (1.34 PFLOP/s).  Bounds: few rows, the weights' stream and a stage's fixed cost (8 rows by 12288 x 5120
// 14.1 us, 2.4 TB/s); many, the tensor cores (79 cycles an instruction of 256 x 192 x 32).
//
// A stage is one to three chunks of 128 columns: codes (16 KB in shared memory, 8 KB from memory) and planes.  Scales have a ring of their own: one thread asks
// for them, four warps move them to tensor memory (column j of an operand: lane l of every quarter holds the four scale bytes of row 32 j + l), well
// ahead of the products.  Eight warps take the sums of the last tile while the products of the next run.  With few tiles K is split among CTAs; their sums
// meet in memory, and the one that comes last adds them up in the order of K.
#include <cuda_fp8.h>
#include <math.h>

#include "jib_kernels.h"
#include "mx4_pair.cuh"
#include "mx4_stream.cuh"
#include "pdl.cuh"
#include "sm100.cuh"
#include "tma_host.cuh"

namespace {

using namespace sm100;
typedef __nv_bfloat16 bf16;

constexpr int BM = 128, MAX_BN = 192, MAX_STAGES = 8, MAX_SLOTS = 8, MAX_E = 256, PAD = 32;
constexpr int A_BYTES = BM * 128, SA_BYTES = BM * 4;
constexpr int THREADS = 512;                       // producer, issuer, one idle, producer of scales; four scale warps; eight epilogue warps
constexpr int MOST_SMEM = 227 * 1024;
constexpr int STAGED = 72, STAGED_BYTES = 2 * 16 * STAGED * 2;          // 64 hidden units of a row and room between rows; two times 16 rows
// Rows of the planes' scales: a tile reads up to MAX_BN behind the last one, 16 bytes (four rows) at a time.
__host__ __device__ inline long long scale_rows_of(long long rows) { return (rows + MAX_BN + 31) / 32 * 32; }

__host__ __device__ inline int stage_bytes(int bn) { return A_BYTES + 2 * bn * 128; }
__host__ __device__ inline int slot_bytes(int bn) { return SA_BYTES + 2 * bn * 4; }              // scales of a stage
__host__ __device__ inline int scale_cols(int n) { return (n + 127) / 128 * 4; }          // of n rows

struct Args {
    const uint8_t * w_scales;                // [matrix][chunk][R][4]
    const uint8_t * x_scales;                // [plane][chunk][x_rows][4], x_rows as scale_rows_of says
    void * out;
    const void * residual;
    const int * seg;                         // grouped: first row of each expert's rows, multiples of PAD; device int[E + 1]
    const int * count;                       // ... and how many there are
    float * part;                            // [tile][split][bn][128]
    int * counters;                          // zeros, one a tile
    int * status;
    uint8_t * h_planes, * h_scales;          // the result as planes and scales for the next product (NULL: as it is, to out); rows h_rows, h_C chunks
    long long ldo, ldr, x_rows, h_rows;
    int T, N, R, C, E, bn, m_tiles, t_tiles, splits, stages, slots, cps, h_C, gated, act, out_f32, res_f32;
};

__device__ __forceinline__ void st_cols4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_mxf8f6f4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t) accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t) accumulate)
            : "memory");
}
// E2M1 x E4M3 with E8M0 scales, m x n, the scales in byte k of their words.
__device__ __forceinline__ uint32_t idesc_e2m1_e4m3(int m, int n, uint32_t k) {
    return k << 4 | 5u << 7 | 0u << 10 | (uint32_t) (n >> 3) << 17 | 1u << 23 | (uint32_t) (m >> 4) << 24 | k << 29;
}

// A place in a ring of n and the parity of its round (divisions by the number of stages took the issuing thread as long as the products).
struct Ring {
    int at = 0;
    uint32_t round = 0;
    __device__ __forceinline__ void next(int n) {
        if (++at == n) { at = 0; round ^= 1; }
    }
};

// ---- bf16 values as two E4M3 numbers ----------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}
__device__ __forceinline__ float2 e4m3_values(uint32_t two) {
    return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t) two, __NV_E4M3)));
}

// Four lanes a block of 32 columns, eight of them each.  Scale 2^e with e = floor(log2 max) - 7, at least -123: the largest magnitude becomes 128 .. 256, rounded
// to hi; what is left, at most 8, times 16 is rounded to lo, whose scale is 2^(e - 4).  Returns e + 127, or 255 for a block with an infinity or NaN.
__device__ __forceinline__ int to_planes(uint4 in, uint2 & hi, uint2 & lo) {
    const uint32_t w[4] = {in.x, in.y, in.z, in.w};
    float z[8];
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 f = __bfloat1622float2(*(const __nv_bfloat162 *) &w[j]);
        z[2 * j] = f.x;
        z[2 * j + 1] = f.y;
        top = max(top, max(__float_as_uint(f.x) & 0x7fffffffu, __float_as_uint(f.y) & 0x7fffffffu));
    }
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int field = (int) (top >> 23), byte = field == 255 ? 255 : max(field - 7, 4);
    const float unit = field == 255 ? 0.f : __uint_as_float((uint32_t) (254 - byte) << 23);
#pragma unroll
    for (int j = 0; j < 8; ++j) z[j] = field == 255 ? 0.f : z[j] * unit;
    hi.x = e4m3x4(z[0], z[1], z[2], z[3]);
    hi.y = e4m3x4(z[4], z[5], z[6], z[7]);
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const float2 f = e4m3_values((j < 4 ? hi.x : hi.y) >> (j & 2) * 8);
        z[j] = (z[j] - f.x) * 16.f;
        z[j + 1] = (z[j + 1] - f.y) * 16.f;
    }
    lo.x = e4m3x4(z[0], z[1], z[2], z[3]);
    lo.y = e4m3x4(z[4], z[5], z[6], z[7]);
    return byte;
}
__device__ __forceinline__ uint8_t low_scale(int byte) { return (uint8_t) (byte == 255 ? 255 : byte - 4); }

// Sixteen columns of sums; with the planes side by side the other plane's stand `other` columns on.
__device__ __forceinline__ void sums16(uint32_t at, int other, uint32_t (&v)[16]) {
    tmem_ld16(at, v);
    if (other != 0) {
        uint32_t u[16];
        tmem_ld16(at + other, u);
        tmem_ld_wait();
#pragma unroll
        for (int k = 0; k < 16; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) + __uint_as_float(u[k]));
    } else {
        tmem_ld_wait();
    }
}

// Named barrier 1 of the eight epilogue warps, and their decision: true when `ok` is for every thread.
__device__ __forceinline__ bool all_of_256(bool ok) {
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 256, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((uint32_t) ok) : "memory");
    return all != 0;
}

// What item i is: row tile m (of a pair: the first of two), first row of x, how many, chunks c0 .. c1 - 1, matrix, tile (for sums that meet).
struct Item {
    int m, row0, rows, c0, c1, e, tile, split;
};

__device__ __forceinline__ Item item_of(const Args & g, const int * first_tile, const int2 * experts, int i) {
    Item t;
    t.m = i % g.m_tiles;
    int rest = i / g.m_tiles;
    t.e = 0;
    t.split = 0;
    t.c0 = 0;
    t.c1 = g.C;
    if (g.seg != nullptr) {                  // the expert whose tiles hold tile `rest`
        int lo = 0, hi = g.E;
#pragma unroll 1
        while (hi - lo > 1) {
            const int mid = (lo + hi) / 2;
            if (first_tile[mid] <= rest) lo = mid;
            else hi = mid;
        }
        t.e = lo;
        const int at = (rest - first_tile[lo]) * g.bn;
        t.row0 = experts[lo].x + at;
        t.rows = min(g.bn, experts[lo].y - at);
    } else {
        const int tt = rest % g.t_tiles;
        t.split = rest / g.t_tiles;
        t.row0 = tt * g.bn;
        t.rows = min(g.bn, g.T - t.row0);
        t.c0 = t.split * g.C / g.splits;
        t.c1 = (t.split + 1) * g.C / g.splits;
        rest = tt;
    }
    t.tile = rest * g.m_tiles + t.m;
    return t;
}

template <bool PAIR>
__device__ __forceinline__ int row_tile(int m, int rank) { return PAIR ? 2 * m + rank : m; }

// How many chunks item i has.
__device__ __forceinline__ int chunks_of(const Args & g, int i) {
    if (g.splits == 1) return g.C;
    const int split = i / (g.m_tiles * g.t_tiles);
    return (split + 1) * g.C / g.splits - split * g.C / g.splits;
}

template <bool PAIR, bool WIDE>
__global__ void __launch_bounds__(THREADS, 1) mx4_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const Args g) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ int first_tile[MAX_E + 1], last_s;
    __shared__ int2 experts[MAX_E];            // first row, rows
    __shared__ uint64_t bars[2 * MAX_STAGES + 3 * MAX_SLOTS + 4];
    __shared__ uint32_t tmem_slot;
    uint8_t * tiles = (uint8_t *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    uint64_t * full = bars, * empty = full + MAX_STAGES, * sl_full = empty + MAX_STAGES, * sf_full = sl_full + MAX_SLOTS, * sf_empty = sf_full + MAX_SLOTS,
             * acc_full = sf_empty + MAX_SLOTS, * acc_empty = acc_full + 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, S = g.stages, Q = g.slots, bn = g.bn, cps = g.cps;
    const int rank = PAIR ? blockIdx.x & 1 : 0, first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
    // rows of x in this CTA's shared memory: of a pair half of them, or, WIDE, all of one plane
    const int xn = PAIR ? bn / 2 : bn, SB = stage_bytes(xn), QB = slot_bytes(bn), plane = xn * 128;
    const int mn = WIDE ? 2 * bn : bn, sfc = scale_cols(mn), slab = WIDE ? 4 + sfc : 4 + 2 * sfc;
    uint8_t * scale_slots = tiles + S * cps * SB;
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); }
        for (int i = 0; i < Q; ++i) { mbar_init(&sl_full[i], 1); mbar_init(&sf_full[i], PAIR ? 8 : 4); mbar_init(&sf_empty[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], PAIR ? 16 : 8); }
        fence_barrier_init();
        prefetch_tmap(&tm_w);
        prefetch_tmap(&tm_x);
    }
    if (warp == 2) mx4::alloc_all<PAIR>(&tmem_slot);
    tc_fence_before();
    __syncthreads();
    if (PAIR) mx4::both_here();                   // barriers are arrived at from the other CTA
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    int items = g.m_tiles * g.t_tiles * g.splits;
    if (g.seg != nullptr) {
        if (warp == 0) {                     // tiles of the experts before each
            int sum = 0;
#pragma unroll 1
            for (int e0 = 0; e0 < g.E; e0 += 32) {
                const int have = e0 + lane < g.E ? g.count[e0 + lane] : 0, mine = (have + bn - 1) / bn;
                if (e0 + lane < g.E) experts[e0 + lane] = make_int2(g.seg[e0 + lane], have);
                int s = mine;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const int v = __shfl_up_sync(0xffffffffu, s, o);
                    if (lane >= o) s += v;
                }
                if (e0 + lane < g.E) first_tile[e0 + lane] = sum + s - mine;
                sum += __shfl_sync(0xffffffffu, s, 31);
            }
            if (lane == 0) first_tile[g.E] = sum;
        }
        __syncthreads();
        items = first_tile[g.E] * g.m_tiles;
    }
    const uint32_t sf0 = tmem + 2 * mn;

    if (warp == 0) {
        if (elect_one()) {
            Ring r;
            bool ok = true;
#pragma unroll 1
            for (int i = first; i < items && ok; i += step) {
                const Item t = item_of(g, first_tile, experts, i);
#pragma unroll 1
                for (int c0 = t.c0; c0 < t.c1; c0 += cps, r.next(S)) {
                    const int s = r.at, n = min(cps, t.c1 - c0);
                    if (!mbar_wait(&empty[s], r.round ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 61, i); ok = false; break; }
                    // (codes count as they are in memory; a pair's first CTA waits for both CTAs' tiles)
                    if (rank == 0) mbar_expect_tx(&full[s], n * (PAIR ? 2 : 1) * (A_BYTES / 2 + 2 * plane));
#pragma unroll 1
                    for (int j = 0; j < n; ++j) {
                        uint8_t * st = tiles + (s * cps + j) * SB;
                        mx4::load<PAIR>(st, &tm_w, &full[s], 0, row_tile<PAIR>(t.m, rank) * BM, t.e * g.C + c0 + j);
                        if (PAIR && WIDE) {
                            mx4::load<PAIR>(st + A_BYTES, &tm_x, &full[s], (c0 + j) * 128, t.row0, rank);
                        } else {
                            mx4::load<PAIR>(st + A_BYTES, &tm_x, &full[s], (c0 + j) * 128, t.row0 + rank * xn, 0);
                            mx4::load<PAIR>(st + A_BYTES + plane, &tm_x, &full[s], (c0 + j) * 128, t.row0 + rank * xn, 1);
                        }
                    }
                }
            }
            // copies in flight end before the memory is given back (the last round's; a stage that was not asked for is not waited for long)
            if (!ok && rank == 0)
                for (int i = 0; i < S; ++i) mbar_wait(&full[i], i < r.at ? r.round : r.round ^ 1);
        }
        __syncwarp();
    } else if (warp == 3) {
        if (elect_one()) {
            Ring r;
            bool ok = true;
#pragma unroll 1
            for (int i = first; i < items && ok; i += step) {
                const Item t = item_of(g, first_tile, experts, i);
                const int m0 = row_tile<PAIR>(t.m, rank) * BM, w_rows = max(0, min(BM, g.R - m0));      // (a pair's second tile may lie behind the last row)
#pragma unroll 1
                for (int c0 = t.c0; c0 < t.c1; c0 += cps, r.next(Q)) {
                    const int q = r.at, n = min(cps, t.c1 - c0);
                    if (!mbar_wait(&sf_empty[q], r.round ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 66, i); ok = false; break; }
                    mbar_expect_tx(&sl_full[q], n * (w_rows * 4 + 2 * bn * 4));
#pragma unroll 1
                    for (int c = c0; c < c0 + n; ++c) {
                        uint8_t * sc = scale_slots + (q * cps + c - c0) * QB;
                        if (!PAIR || w_rows > 0) mx4::bulk_load(sc, g.w_scales + ((size_t) (t.e * g.C + c) * g.R + m0) * 4, w_rows * 4, &sl_full[q]);
                        mx4::bulk_load(sc + SA_BYTES, g.x_scales + ((size_t) c * g.x_rows + t.row0) * 4, bn * 4, &sl_full[q]);
                        mx4::bulk_load(sc + SA_BYTES + bn * 4, g.x_scales + ((size_t) (g.C + c) * g.x_rows + t.row0) * 4, bn * 4, &sl_full[q]);
                    }
                }
            }
            if (!ok)
                for (int i = 0; i < Q; ++i) mbar_wait(&sl_full[i], i < r.at ? r.round : r.round ^ 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if ((!PAIR || rank == 0) && elect_one()) {
            Ring r, rq;
            int j = 0;
            bool ok = true;
            const uint64_t desc0 = desc_k_sw128(smem_u32(tiles));
            const uint32_t id0 = idesc_e2m1_e4m3(PAIR ? 2 * BM : BM, mn, 0), lo = (uint32_t) plane >> 4;
#pragma unroll 1
            for (int i = first; i < items && ok; i += step, ++j) {
                const int n = chunks_of(g, i);
                const int buf = j & 1;
                if (!mbar_wait(&acc_empty[buf], (j >> 1 & 1) ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 62, i); break; }
                tc_fence_after();
                const uint32_t acc = tmem + buf * mn;
                bool more = false;
#pragma unroll 1
                for (int c0 = 0; c0 < n; c0 += cps, r.next(S), rq.next(Q)) {
                    if (!mbar_wait(&sf_full[rq.at], rq.round) || !mbar_wait(&full[r.at], r.round)) {
                        jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 63, i);
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    // descriptors count in 16 bytes, a step of 32 columns is two of them; the scales' byte is in bits 4 and 29 of the other
#pragma unroll 1
                    for (int j = 0; j < min(cps, n - c0); ++j) {
                        const uint64_t a = desc0 + (uint32_t) ((r.at * cps + j) * SB >> 4), b = a + (A_BYTES >> 4);
                        const uint32_t sf = sf0 + (rq.at * cps + j) * slab;
                        if (WIDE) {
#pragma unroll
                            for (int k = 0; k < 4; ++k) mma_mxf8f6f4<PAIR>(acc, a + 2 * k, b + 2 * k, id0 + (k << 4) + ((uint32_t) k << 29), sf, sf + 4, more || k != 0);
                        } else {
#pragma unroll
                            for (int k = 0; k < 4; ++k) {
                                const uint32_t id = id0 + (k << 4) + ((uint32_t) k << 29);
                                mma_mxf8f6f4<PAIR>(acc, a + 2 * k, b + 2 * k, id, sf, sf + 4, more || k != 0);
                                mma_mxf8f6f4<PAIR>(acc, a + 2 * k, b + lo + 2 * k, id, sf, sf + 4 + sfc, true);
                            }
                        }
                        more = true;
                    }
                    mx4::commit<PAIR>(&empty[r.at]);
                    mx4::commit<PAIR>(&sf_empty[rq.at]);
                }
                mx4::commit<PAIR>(&acc_full[buf]);
            }
        }
        __syncwarp();
    } else if (warp >= 4 && warp < 8) {
        // scales to tensor memory
        const uint32_t mine = sf0 + ((uint32_t) (warp & 3) << 21);
        Ring r;
        bool ok = true;
#pragma unroll 1
        for (int i = first; i < items && ok; i += step) {
            const int n = chunks_of(g, i);
#pragma unroll 1
            for (int c0 = 0; c0 < n; c0 += cps, r.next(Q)) {
                const int q = r.at;
                ok = __all_sync(0xffffffffu, mbar_wait(&sl_full[q], r.round));
                if (!ok) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 64, i); break; }
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < min(cps, n - c0); ++c) {
                    const uint32_t * sc = (const uint32_t *) (scale_slots + (q * cps + c) * QB) + lane;
                    const uint32_t dst = mine + (q * cps + c) * slab;
                    constexpr int P = WIDE ? 1 : 2;
                    uint32_t w[4], v[P][8];
#pragma unroll
                    for (int k = 0; k < 4; ++k) w[k] = sc[k * 32];
#pragma unroll
                    for (int p = 0; p < P; ++p)
#pragma unroll
                        for (int k = 0; k < 8; ++k) v[p][k] = k * 32 + lane < mn ? sc[SA_BYTES / 4 + p * bn + k * 32] : 0u;
                    st_cols4(dst, w[0], w[1], w[2], w[3]);
#pragma unroll
                    for (int p = 0; p < P; ++p) {
                        st_cols4(dst + 4 + p * sfc, v[p][0], v[p][1], v[p][2], v[p][3]);
                        if (sfc > 4) st_cols4(dst + 8 + p * sfc, v[p][4], v[p][5], v[p][6], v[p][7]);
                    }
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mx4::arrive_first<PAIR>(&sf_full[q]);
            }
        }
    } else if (warp >= 8) {
        // two warps a quarter of the rows, they take every second 16 rows of x
        const int q = warp & 3, half = (warp - 8) >> 2;
        const uint32_t mine = tmem + ((uint32_t) q << 21);
        bf16 * staged = (bf16 *) (scale_slots + Q * cps * QB) + half * 16 * STAGED;
        int j = 0;
#pragma unroll 1
        for (int i = first; i < items; i += step, ++j) {
            const Item t = item_of(g, first_tile, experts, i);
            const int buf = j & 1;
            bool ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], j >> 1 & 1));
            if (g.h_planes != nullptr || (!PAIR && g.splits > 1)) ok = all_of_256(ok);          // (they meet below)
            if (!ok) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 65, i); break; }
            tc_fence_after();
            const uint32_t acc = mine + buf * mn;
            bool finish = true;
            float * part = g.part + ((size_t) t.tile * g.splits * bn) * BM + q * 32 + lane;
            if (!PAIR && g.splits > 1) {
                float * to = part + (size_t) t.split * bn * BM;
#pragma unroll 1
                for (int c = 16 * half; c < t.rows; c += 32) {
                    uint32_t v[16];
                    sums16(acc + c, WIDE ? bn : 0, v);
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (c + k < t.rows) __stcg(to + (size_t) (c + k) * BM, __uint_as_float(v[k]));
                }
                __threadfence();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 256) {
                    last_s = atomicAdd(g.counters + t.tile, 1) == g.splits - 1;
                    __threadfence();
                }
                asm volatile("bar.sync 1, 256;" ::: "memory");
                finish = last_s != 0;
                asm volatile("bar.sync 1, 256;" ::: "memory");
            }
            // lane = row n of the tile (of pairs: 16 of the gate, 16 of the up matrix), 16 rows of x at a time
            const int m = row_tile<PAIR>(t.m, rank), n = g.gated ? m * 64 + q * 16 + (lane & 15) : m * BM + q * 32 + lane;
#pragma unroll 1
            for (int c = 16 * half; c < t.rows && finish; c += 32) {
                float y[16];
                if (!PAIR && g.splits > 1) {
#pragma unroll
                    for (int k = 0; k < 16; ++k) y[k] = 0.f;
#pragma unroll 1
                    for (int s = 0; s < g.splits; s += 2) {
                        float v[2][16];
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int k = 0; k < 16; ++k)
                                v[h][k] = c + k < t.rows && s + h < g.splits ? __ldcg(part + ((size_t) (s + h) * bn + c + k) * BM) : 0.f;
#pragma unroll
                        for (int h = 0; h < 2; ++h)
#pragma unroll
                            for (int k = 0; k < 16; ++k) y[k] += v[h][k];
                    }
                } else {
                    uint32_t v[16];
                    sums16(acc + c, WIDE ? bn : 0, v);
#pragma unroll
                    for (int k = 0; k < 16; ++k) y[k] = __uint_as_float(v[k]);
                }
                if (PAIR && g.h_planes != nullptr) {
                    // four warps: 16 rows of 64 units, in bf16, through shared memory; then a thread eight units of a row
                    bf16 * at = staged + (lane >> 4) * STAGED + q * 16 + (lane & 15);
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? y[k + 1] : y[k], 16);
                        const float v = mx4::gated(lane < 16 ? y[k] : other, lane < 16 ? other : y[k + 1], g.act);
                        at[k * STAGED] = __float2bfloat16(n < g.N ? v : 0.f);
                    }
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
                    const int id = threadIdx.x & 127, row = id >> 3, col = m * 64 + (id & 7) * 8;
                    uint2 hi, lo;
                    const int byte = to_planes(*(const uint4 *) (staged + row * STAGED + (id & 7) * 8), hi, lo);
                    if (c + row < t.rows && col < g.h_C * 128) {
                        const long long r = t.row0 + c + row, width = g.h_C * 128;
                        *(uint2 *) (g.h_planes + r * width + col) = hi;
                        *(uint2 *) (g.h_planes + (g.h_rows + r) * width + col) = lo;
                        if ((id & 3) == 0) {
                            const long long rows = scale_rows_of(g.h_rows);
                            uint8_t * sc = g.h_scales + ((col >> 7) * rows + r) * 4 + (col >> 5 & 3);
                            sc[0] = (uint8_t) byte;
                            sc[g.h_C * rows * 4] = low_scale(byte);
                        }
                    }
                    asm volatile("bar.sync %0, 128;" ::"r"(2 + half) : "memory");
                    continue;
                }
                if (g.gated) {
                    // a gate's lane takes the even rows of x, the up matrix's lane 16 above it the odd ones
                    bf16 * to = (bf16 *) g.out + (long long) (t.row0 + c + (lane >> 4)) * g.ldo + n;
#pragma unroll
                    for (int k = 0; k < 16; k += 2) {
                        const float other = __shfl_xor_sync(0xffffffffu, lane < 16 ? y[k + 1] : y[k], 16);
                        const float v = mx4::gated(lane < 16 ? y[k] : other, lane < 16 ? other : y[k + 1], g.act);
                        if (n < g.N && c + k + (lane >> 4) < t.rows) {
                            if (g.out_f32) ((float *) g.out)[(long long) (t.row0 + c + k + (lane >> 4)) * g.ldo + n] = v;
                            else *to = __float2bfloat16(v);
                        }
                        to += 2 * g.ldo;
                    }
                    continue;
                }
                if (n >= g.N) continue;
                if (g.residual != nullptr)
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (c + k < t.rows) {
                            const long long at = (long long) (t.row0 + c + k) * g.ldr + n;
                            y[k] += g.res_f32 ? ((const float *) g.residual)[at] : __bfloat162float(((const bf16 *) g.residual)[at]);
                        }
                bf16 * to = (bf16 *) g.out + (long long) (t.row0 + c) * g.ldo + n;
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                    if (c + k < t.rows) {
                        if (g.out_f32) ((float *) g.out)[(long long) (t.row0 + c + k) * g.ldo + n] = y[k];
                        else *to = __float2bfloat16(y[k]);
                    }
                    to += g.ldo;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mx4::arrive_first<PAIR>(&acc_empty[buf]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) mx4::both_here();                   // neither leaves while the other arrives at its barriers or multiplies its rows
    if (warp == 2) mx4::free_all<PAIR>(tmem);
}

// ---- bf16 rows as two E4M3 planes ------------------------------------------------------------------------------------------------
// A thread keeps its eight columns and walks down the rows.  Bound by memory and two dependent loads with src (4 thousand rows of 2048 columns gathered from
// 515: 12 us).  src: row r is x[src[r]] (zeros where that is negative); limit: rows from *limit on are left alone.
constexpr int ROWS = 4;                             // of a thread's columns, their loads in flight together

__global__ void __launch_bounds__(256) planes_kernel(const bf16 * __restrict__ x, long long ldx, const int * __restrict__ src, const int * __restrict__ limit,
                                                     uint8_t * __restrict__ planes, uint8_t * __restrict__ scales, long long rows, long long scale_rows, int K, int C,
                                                     int * __restrict__ zeros, int n_zeros) {
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    const int id = (blockIdx.y * gridDim.x + blockIdx.x) * blockDim.x + threadIdx.x, k = (blockIdx.x * blockDim.x + threadIdx.x) * 8;
    for (int i = id; i < n_zeros; i += gridDim.x * gridDim.y * blockDim.x) zeros[i] = 0;
    const long long most = limit != nullptr ? min(rows, (long long) *limit) : rows;
#pragma unroll 1
    for (long long r0 = (long long) blockIdx.y * ROWS; r0 < most; r0 += (long long) gridDim.y * ROWS) {
        uint4 in[ROWS];
#pragma unroll
        for (int h = 0; h < ROWS; ++h) {
            const long long from = r0 + h >= most ? -1 : src != nullptr ? src[r0 + h] : r0 + h;
            in[h] = from >= 0 && k < K ? *(const uint4 *) (x + from * ldx + k) : make_uint4(0u, 0u, 0u, 0u);
        }
#pragma unroll
        for (int h = 0; h < ROWS; ++h) {
            uint2 hi, lo;
            const int byte = to_planes(in[h], hi, lo);
            if (r0 + h >= most || k >= C * 128) continue;
            uint8_t * to = planes + (r0 + h) * (long long) (C * 128) + k;
            *(uint2 *) to = hi;
            *(uint2 *) (to + rows * (long long) (C * 128)) = lo;
            if ((k >> 3 & 3) == 0) {
                uint8_t * sc = scales + ((long long) (k >> 7) * scale_rows + r0 + h) * 4 + (k >> 5 & 3);
                sc[0] = (uint8_t) byte;
                sc[(long long) C * scale_rows * 4] = low_scale(byte);
            }
        }
    }
}

// ---- pairs by expert, each expert's rows at a multiple of PAD -------------------------------------------------------------------------
// first[e] and count[e] of the padded order (first[E]: its end), the token of each of its rows (-1: none) and the row of each pair (-1: an id outside the experts).
// 4 thousand pairs: 7 us; by the framework's own sort and a launch that spreads its places 18.  One CTA: counts, their sums, places, with a table for each warp (tokens that choose alike would queue for one).  Which of its warp's rows a pair gets is left
// to chance; what is computed from a row does not depend on where it stands.
constexpr int SORT_NT = 1024, SORT_AHEAD = 4;

__global__ void __launch_bounds__(SORT_NT) sort_kernel(const int * __restrict__ ids, int n, int k, int E, int * __restrict__ first, int * __restrict__ count,
                                                       int * __restrict__ row_src, int * __restrict__ pair_row) {
    __shared__ int places[SORT_NT / 32][MAX_E], count_s[MAX_E], first_s[MAX_E + 1];
    const int tid = threadIdx.x, lane = tid & 31;
    int * mine = places[tid >> 5];
    auto ask = [&](int b, int (&e)[SORT_AHEAD]) {        // -1: none
#pragma unroll
        for (int j = 0; j < SORT_AHEAD; ++j) {
            const int i = b + j * SORT_NT + tid, id = i < n ? ids[i] : -1;
            e[j] = (unsigned) id < (unsigned) E ? id : -1;
        }
    };
    for (int i = tid; i < SORT_NT / 32 * MAX_E; i += SORT_NT) (&places[0][0])[i] = 0;
    __syncthreads();
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    for (int b = 0; b < n; b += SORT_NT * SORT_AHEAD) {
        int e[SORT_AHEAD];
        ask(b, e);
#pragma unroll
        for (int j = 0; j < SORT_AHEAD; ++j)
            if (e[j] >= 0) atomicAdd(&mine[e[j]], 1);
    }
    __syncthreads();
    if (tid < E) {                       // each warp's first place among its expert's rows
        int sum = 0;
#pragma unroll 8
        for (int w = 0; w < SORT_NT / 32; ++w) {
            const int have = places[w][tid];
            places[w][tid] = sum;
            sum += have;
        }
        count_s[tid] = sum;
    }
    __syncthreads();
    if (tid < 32) {
        int sum = 0;
#pragma unroll 1
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + lane, rows = e < E ? (count_s[e] + PAD - 1) / PAD * PAD : 0;
            int s = rows;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int v = __shfl_up_sync(0xffffffffu, s, o);
                if (lane >= o) s += v;
            }
            if (e < E) first_s[e] = sum + s - rows;
            sum += __shfl_sync(0xffffffffu, s, 31);
        }
        if (lane == 0) first_s[E] = sum;
    }
    __syncthreads();
    for (int e = tid; e <= E; e += SORT_NT) {
        first[e] = first_s[e];
        if (e < E) count[e] = count_s[e];
    }
    for (int i = tid; i < E * PAD; i += SORT_NT) {       // rows behind an expert's last
        const int e = i / PAD, r = first_s[e] + count_s[e] + i % PAD;
        if (r < first_s[e + 1]) row_src[r] = -1;
    }
    for (int b = 0; b < n; b += SORT_NT * SORT_AHEAD) {
        int e[SORT_AHEAD];
        ask(b, e);
#pragma unroll
        for (int j = 0; j < SORT_AHEAD; ++j) {
            const int i = b + j * SORT_NT + tid;
            int r = -1;
            if (e[j] >= 0) {
                r = first_s[e[j]] + atomicAdd(&mine[e[j]], 1);
                row_src[r] = i / k;
            }
            if (i < n) pair_row[i] = r;
        }
    }
}

int launched() { return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH; }

// Tensor map of the packed codes: 4-bit elements spread over bytes, boxes of 128 rows of a chunk.
int weights_map(CUtensorMap * out, const void * codes, long long R, long long z) {
    jib::TmaEncodeFn fn = jib::tma_encode_fn();
    if (!fn) return JIB_E_DRIVER;
    if ((uintptr_t) codes & 31) return JIB_E_ALIGN;
    const cuuint64_t dims[3] = {128, (cuuint64_t) R, (cuuint64_t) z}, strides[2] = {mx4::CODES, (cuuint64_t) R * mx4::CODES};
    const cuuint32_t box[3] = {128, BM, 1}, step[3] = {1, 1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 3, const_cast<void *>(codes), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : JIB_E_TENSORMAP;
}

int planes_map(CUtensorMap * out, const void * planes, long long rows, long long bytes, int bn) {
    jib::TmaEncodeFn fn = jib::tma_encode_fn();
    if (!fn) return JIB_E_DRIVER;
    if ((uintptr_t) planes & 15) return JIB_E_ALIGN;
    const cuuint64_t dims[3] = {(cuuint64_t) bytes, (cuuint64_t) rows, 2}, strides[2] = {(cuuint64_t) bytes, (cuuint64_t) (bytes * rows)};
    const cuuint32_t box[3] = {128, (cuuint32_t) bn, 1}, step[3] = {1, 1, 1};
    return fn(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, const_cast<void *>(planes), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS
               ? 0
               : JIB_E_TENSORMAP;
}

// Up to this many rows of x the planes are one operand (two buffers of sums and the scales fit in tensor memory).
constexpr int MAX_WIDE = 96;

int sm_count() { return jib::sm_count() > 0 ? jib::sm_count() : 148; }

template <bool WIDE>
int pair_count() {
    static std::atomic<int> known[jib::MAX_DEVICES];
    static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
    return mx4::pair_count(mx4_gemm_kernel<true, WIDE>, THREADS, MOST_SMEM - 5120, known, attr_done);
}

// Rows of x in a tile and splits of K of a dense product.  What a chunk costs a CTA is its traffic with shared memory: 128 bytes written a row of either operand
// and plane, and as many read by each instruction.  In rows of x (512 bytes): w + 64 with the planes as one operand; in a pair w / 2 + 96, or w for its
// products where that is more.  Where the tiles leave SMs idle, K is split, four chunks a split at least.
void shape_of(long long T, int R, int C, int * bn, int * splits) {
    const int sms = sm_count(), pairs = R > BM ? pair_count<false>() : 0;
    const long long m_tiles = (R + BM - 1) / BM;
    long long best = -1;
    for (int w = T > 16 ? 32 : 16; w <= (pairs > 0 ? MAX_BN : MAX_WIDE); w += 32) {
        const bool pair = w > MAX_WIDE;
        const long long tiles = (pair ? (m_tiles + 1) / 2 : m_tiles) * ((T + w - 1) / w), at_once = pair ? pairs : sms;
        const long long cost = (tiles + at_once - 1) / at_once * (!pair ? w + 64 : w > w / 2 + 96 ? w : w / 2 + 96);
        if (best < 0 || cost <= best) { best = cost; *bn = w; }
        if (w >= T) break;
    }
    const long long tiles = m_tiles * ((T + *bn - 1) / *bn);
    int s = (int) (sms / tiles);
    if (s > C / 4) s = C / 4;
    if (s > 16) s = 16;
    *splits = s < 1 || *bn > MAX_WIDE ? 1 : s;
}

// What a product needs besides its operands: planes and their scales; sums and counters of splits.
struct Scratch {
    long long scales, part, counters, bytes;             // (planes come first)
    int bn = 0, splits = 1, tiles = 0;                   // of a dense product
    Scratch(long long rows, int N, int K, bool gated, bool grouped) {
        const int C = mx4::chunks(K), R = mx4::rows_of(N, gated), m_tiles = (R + BM - 1) / BM;
        scales = 2 * rows * C * 128;
        part = planes(rows, C);
        counters = part;
        if (!grouped) {
            shape_of(rows, R, C, &bn, &splits);
            if (splits > 1) {
                tiles = (int) (m_tiles * ((rows + bn - 1) / bn));
                counters = part + 4ll * tiles * splits * bn * BM;
            }
        }
        bytes = counters + 4ll * tiles;
    }
    static long long planes(long long rows, int C) { return 2 * rows * C * 128 + 2ll * C * scale_rows_of(rows) * 4; }
};

}  // namespace

extern "C" {

// Bytes that jib_mx4_gemm needs for `rows` rows.
JIB_EXPORT long long jib_mx4_gemm_scratch(long long rows, int N, int K, int gated, int grouped) { return Scratch(rows, N, K, gated != 0, grouped != 0).bytes; }

// Whether a grouped product can hand its results to the next one as planes.
JIB_EXPORT int jib_mx4_gemm_joins(int N, int gated) { return gated && mx4::rows_of(N, true) > BM && pair_count<true>() > 0 && pair_count<false>() > 0; }

// ids [n / k][k]; first: E + 1 ints, count: E, row_src: room for n pairs and PAD - 1 more rows of each expert that has any, pair_row: n.
JIB_EXPORT int jib_mx4_sort(const int * ids, int n, int k, int E, int * first, int * count, int * row_src, int * pair_row, void * stream) {
    if (E < 1 || E > MAX_E || n < 1 || k < 1) return JIB_E_ARG;
    JIB_LAUNCH((sort_kernel), 1, SORT_NT, 0, (cudaStream_t) stream, ids, n, k, E, first, count, row_src, pair_row);
    return launched();
}

// The tiled product of bf16 rows d->x: as planes, then multiplied.  Grouped: d->seg = first, count, d->src = row_src of jib_mx4_sort (NULL: x in that order), T
// rows at most.  scratch: jib_mx4_gemm_scratch(T, ..) bytes on this device at least; ready: it holds the planes already (then d->x is not read).  next (grouped pairs of more than one
// tile of weights, see jib_mx4_gemm_joins): the scratch of a product of the results, which go there as planes and not to d->out.
JIB_EXPORT int jib_mx4_gemm(const jib_mx4_desc * d, const int * count, void * scratch, long long scratch_bytes, void * next, long long next_bytes, int ready,
                            void * stream) {
    if (d->T <= 0) return 0;
    if (d->N <= 0 || d->K <= 0 || d->K % 32 || d->batch < 1 || d->batch > MAX_E || (d->seg != nullptr && (count == nullptr || d->residual != nullptr)) ||
        (next != nullptr && (!jib_mx4_gemm_joins(d->N, d->gated) || d->seg == nullptr || !d->gated || ((uintptr_t) next & 15))) || (ready && d->seg == nullptr))
        return JIB_E_ARG;
    if (((uintptr_t) d->x | (uintptr_t) (d->ldx * 2) | (uintptr_t) scratch | (uintptr_t) d->w_scales) & 15) return JIB_E_ALIGN;
    const Scratch sc(d->T, d->N, d->K, d->gated != 0, d->seg != nullptr);
    if (scratch_bytes < sc.bytes || (next != nullptr && next_bytes < Scratch::planes(d->T, mx4::chunks(d->N)))) return JIB_E_SCRATCH;
    uint8_t * planes = (uint8_t *) scratch, * x_scales = planes + sc.scales;
    const int sms = sm_count();
    Args g;
    g.w_scales = d->w_scales; g.x_scales = x_scales; g.out = d->out; g.residual = d->residual; g.seg = d->seg; g.count = count;
    g.part = (float *) (planes + sc.part); g.counters = (int *) (planes + sc.counters); g.status = d->status; g.ldo = d->ldo; g.ldr = d->ldr; g.x_rows = scale_rows_of(d->T);
    g.T = d->T; g.N = d->N; g.R = mx4::rows_of(d->N, d->gated != 0); g.C = mx4::chunks(d->K); g.E = d->batch;
    g.gated = d->gated; g.act = d->act; g.out_f32 = d->out_f32; g.res_f32 = d->res_f32;
    g.h_planes = (uint8_t *) next; g.h_rows = d->T; g.h_C = mx4::chunks(d->N); g.h_scales = g.h_planes + 2ll * d->T * g.h_C * 128;
    g.m_tiles = (g.R + BM - 1) / BM;
    long long items;
    if (d->seg != nullptr) {
        // an expert's rows on average and twice their spread: most experts then take one tile
        const float avg = (float) d->max_rows / d->batch;
        const int w = ((int) (avg + 2.f * sqrtf(avg)) + 31) / 32 * 32;
        const int most = g.R > BM && pair_count<false>() > 0 ? MAX_BN : MAX_WIDE;
        g.bn = w < 32 ? 32 : w > most ? most : w;
        g.splits = 1;
        g.t_tiles = 1;
        items = sms;
    } else {
        g.bn = sc.bn;
        g.splits = sc.splits;
        g.t_tiles = (d->T + g.bn - 1) / g.bn;
        items = (long long) g.m_tiles * g.t_tiles * g.splits;
    }
    // pairs: tiles of more rows, and experts' tiles (of the 66-expert layer 17 rows take 95.5 us alone, 92 in pairs, 515 rows 159 and 143)
    const bool wide = g.bn <= MAX_WIDE, pair = !wide || (d->seg != nullptr && g.R > BM && pair_count<true>() > 0);
    const int at_once = !pair ? sms : wide ? pair_count<true>() : pair_count<false>(), xn = pair ? g.bn / 2 : g.bn;
    if (pair) {
        g.m_tiles = (g.m_tiles + 1) / 2;
        items = d->seg != nullptr ? at_once : (long long) g.m_tiles * g.t_tiles;
    }
    if (items > 0x3fffffff) return JIB_E_ARG;
    // Chunks of a stage: its waits and commits take the issuing thread as long as a few products.  8 rows by 12288 x 5120: 21 us with one, 16.5 with two, 14.3
    // with three; 17 rows of the 66-expert layer (16 and 11 chunks) 122 and 96 us with one and two, 107 with three; 515 rows 191 and 160.  The rule goes by the
    // tile's width alone: numbers of chunks that three divides were not measured.
    g.cps = g.bn <= 16 ? 3 : g.bn <= MAX_WIDE ? 2 : 1;
    g.slots = !wide ? (512 - 2 * g.bn) / (4 + 2 * scale_cols(g.bn)) : (512 - 4 * g.bn) / (g.cps * (4 + scale_cols(2 * g.bn)));
    if (g.slots > MAX_SLOTS) g.slots = MAX_SLOTS;
    const int staged = next != nullptr ? STAGED_BYTES : 0;
    g.stages = (MOST_SMEM - 5120 - 1024 - staged - g.slots * g.cps * slot_bytes(g.bn)) / (g.cps * stage_bytes(xn));        // (5 KB: barriers and tables)
    if (g.stages > MAX_STAGES) g.stages = MAX_STAGES;
    const size_t smem = g.cps * (g.stages * stage_bytes(xn) + g.slots * slot_bytes(g.bn)) + staged + 1024;
    CUtensorMap mw, mx;
    int rc = weights_map(&mw, d->w, g.R, (long long) g.C * d->batch);
    if (rc) return rc;
    rc = planes_map(&mx, planes, d->T, (long long) g.C * 128, wide ? g.bn : xn);
    if (rc) return rc;
    static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
    if (!pair && !jib::ensure_dyn_smem(mx4_gemm_kernel<false, true>, MOST_SMEM - 5120, attr_done)) return JIB_E_LAUNCH;
    // a thread keeps its eight columns and walks down the rows
    const int nx = (g.C * 16 + 255) / 256, th = ((g.C * 16 + nx - 1) / nx + 31) / 32 * 32;
    const long long ny = (d->T + ROWS - 1) / ROWS, most = ((long long) sms * 4096 / th + nx - 1) / nx;
    if (!ready)
        JIB_LAUNCH((planes_kernel), dim3(nx, (unsigned) (ny < most ? ny : most < 65535 ? most : 65535)), th, 0, (cudaStream_t) stream, (const bf16 *) d->x, d->ldx, d->src,
               d->seg != nullptr ? d->seg + d->batch : nullptr, planes, x_scales, (long long) d->T, g.x_rows, d->K, g.C, g.counters, sc.tiles);
    const unsigned grid = (unsigned) (items < at_once ? items : at_once);
    if (pair && wide) (void) jib::launch_pdl_pairs(mx4_gemm_kernel<true, true>, grid, dim3(THREADS), smem, (cudaStream_t) stream, mw, mx, g);
    else if (pair) (void) jib::launch_pdl_pairs(mx4_gemm_kernel<true, false>, grid, dim3(THREADS), smem, (cudaStream_t) stream, mw, mx, g);
    else JIB_LAUNCH((mx4_gemm_kernel<false, true>), grid, THREADS, smem, (cudaStream_t) stream, mw, mx, g);
    return launched();
}

}  // extern "C"
