// Product of two microscaled 4-bit operands on the 4-bit tensor cores: out[t][n] = sum_k a[t][k] b[n][k].
//
// tcgen05.mma.kind::mxf4.block_scale multiplies E2M1 codes and applies the blocks' scales itself, 64 columns an instruction: nothing is
// expanded.  b (the weights) is operand A of the instruction, 128 rows a tile, a's rows are its columns, up to 208 a tile: so few tokens cost
// a narrow tile.  The scales live in tensor memory: column j of a slab holds, in lane l of every quarter, the four scale bytes of row 32 j + l
// for 128 columns of K.  They come in boxes of 16 bytes a row (512 columns, two stages) in a ring of their own, and four warps move them to tensor
// memory ahead of their stage.  (Read from global memory by those warps, stage by stage, they took 1200 clocks a stage, three times the products.)
#include "sm100.cuh"
#include "jib_kernels.h"
#include "pdl.cuh"
#include "tma_host.cuh"

namespace {

using namespace sm100;
typedef __nv_bfloat16 bf16;

constexpr int BM = 128, MAX_BN = 208, STAGES = 4, KS = 256;       // weights a tile, tokens at most, stages, columns a stage
constexpr int A_BYTES = BM * 128, B_BYTES = MAX_BN * 128, STAGE_BYTES = A_BYTES + B_BYTES;
constexpr int BOXES = 3, BOX_BYTES = (BM + MAX_BN) * 16;         // scales of two stages
constexpr int SMEM = STAGES * STAGE_BYTES + BOXES * BOX_BYTES + 1024 + 256;
constexpr int SLAB = 12;                                         // columns of the scales of 128 columns of K: 4 of A, 8 of B
constexpr int SF0 = 2 * MAX_BN;                                  // two accumulators, then the scales of each stage
constexpr int THREADS = 512;                                     // producer, issuer, one idle, producer of scales; four scale warps; eight epilogue warps
static_assert(SF0 + STAGES * 2 * SLAB <= 512, "tensor memory");

struct Args {
    void * out;
    long long ldo;
    int * status;
    int T, N, K, bn, out_f32, m_tiles, items;
};

__device__ __forceinline__ void st_cols4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t) accumulate)
        : "memory");
}
// E2M1 x E2M1 with E8M0 scales, 128 x n, the scales in bytes `half` and `half` + 1 of their words.
__device__ __forceinline__ uint32_t idesc_mxf4(int n, uint32_t half) {
    return half << 4 | 1u << 7 | 1u << 10 | (uint32_t) (n >> 3) << 17 | 1u << 23 | (uint32_t) (BM >> 4) << 24 | half << 29;
}

__global__ void __launch_bounds__(THREADS, 1) mx4_matmul_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                                                                const __grid_constant__ CUtensorMap tm_as, const __grid_constant__ CUtensorMap tm_bs, const Args g) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t * tiles = (uint8_t *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    uint8_t * boxes = tiles + STAGES * STAGE_BYTES;
    uint64_t * full = (uint64_t *) (boxes + BOXES * BOX_BYTES), * empty = full + STAGES, * sf_full = empty + STAGES, * acc_full = sf_full + STAGES,
             * acc_empty = acc_full + 2, * box_full = acc_empty + 2, * box_empty = box_full + BOXES;
    uint32_t * tmem_slot = (uint32_t *) (box_empty + BOXES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); mbar_init(&sf_full[i], 4); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], 8); }
        for (int i = 0; i < BOXES; ++i) { mbar_init(&box_full[i], 1); mbar_init(&box_empty[i], 4); }
        fence_barrier_init();
        prefetch_tmap(&tm_as);
        prefetch_tmap(&tm_bs);
        prefetch_tmap(&tm_a);
        prefetch_tmap(&tm_b);
    }
    if (warp == 2) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    const int n_stages = (g.K + KS - 1) / KS;

    if (warp == 0) {
        if (elect_one()) {
            int it = 0;
            bool ok = true;
            for (int item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
                const int n0 = item % g.m_tiles * BM, t0 = item / g.m_tiles * g.bn;
                for (int kb = 0; kb < n_stages; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&empty[s], (it / STAGES & 1) ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 41, item); ok = false; break; }
                    uint8_t * st = tiles + s * STAGE_BYTES;
                    mbar_expect_tx(&full[s], A_BYTES + g.bn * 128);
                    tma_load_2d(st, &tm_b, &full[s], kb * 128, n0);
                    tma_load_2d(st + A_BYTES, &tm_a, &full[s], kb * 128, t0);
                }
            }
            // copies in flight end before the memory is given back
            if (!ok)
                for (int i = it - STAGES < 0 ? 0 : it - STAGES; i < it; ++i) mbar_wait(&full[i % STAGES], i / STAGES & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (elect_one()) {
            const uint64_t desc0 = desc_k_sw128(smem_u32(tiles));
            const uint32_t id0 = idesc_mxf4(g.bn, 0), id1 = idesc_mxf4(g.bn, 2);
            int it = 0, j = 0;
            bool ok = true;
            for (int item = blockIdx.x; item < g.items && ok; item += gridDim.x, ++j) {
                const int buf = j & 1;
                if (!mbar_wait(&acc_empty[buf], (j >> 1 & 1) ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 42, item); break; }
                tc_fence_after();
                const uint32_t acc = tmem + buf * MAX_BN;
                for (int kb = 0; kb < n_stages; ++kb, ++it) {
                    const int s = it % STAGES;
                    const uint32_t ph = it / STAGES & 1;
                    if (!mbar_wait(&full[s], ph) || !mbar_wait(&sf_full[s], ph)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 43, item); ok = false; break; }
                    tc_fence_after();
                    const uint64_t a = desc0 + (uint32_t) (s * STAGE_BYTES >> 4), b = a + (A_BYTES >> 4);       // (descriptors count in 16 bytes)
                    const uint32_t sf = tmem + SF0 + s * 2 * SLAB;
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        mma_mxf4(acc, a + 2 * q, b + 2 * q, q & 1 ? id1 : id0, sf + q / 2 * SLAB, sf + q / 2 * SLAB + 4, (kb | q) != 0);
                    mma_commit(&empty[s]);
                }
                mma_commit(&acc_full[buf]);
            }
        }
        __syncwarp();
    } else if (warp == 3) {
        if (elect_one()) {
            int it = 0;
            bool ok = true;
            for (int item = blockIdx.x; item < g.items && ok; item += gridDim.x) {
                const int n0 = item % g.m_tiles * BM, t0 = item / g.m_tiles * g.bn;
                for (int kb = 0; kb < n_stages; kb += 2, ++it) {
                    const int s = it % BOXES;
                    if (!mbar_wait(&box_empty[s], (it / BOXES & 1) ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 46, item); ok = false; break; }
                    mbar_expect_tx(&box_full[s], (BM + g.bn) * 16);
                    tma_load_2d(boxes + s * BOX_BYTES, &tm_bs, &box_full[s], kb * 8, n0);
                    tma_load_2d(boxes + s * BOX_BYTES + BM * 16, &tm_as, &box_full[s], kb * 8, t0);
                }
            }
            if (!ok)
                for (int i = it - BOXES < 0 ? 0 : it - BOXES; i < it; ++i) mbar_wait(&box_full[i % BOXES], i / BOXES & 1);
        }
        __syncwarp();
    } else if (warp >= 4 && warp < 8) {
        // scales of a stage: eight bytes a row
        const uint32_t mine = tmem + ((uint32_t) (warp & 3) << 21) + SF0;
        const int valid = g.K / 32;
        int it = 0, box = -1;
        bool ok = true;
        for (int item = blockIdx.x; item < g.items && ok; item += gridDim.x)
            for (int kb = 0; kb < n_stages; ++kb, ++it) {
                const int s = it % STAGES, n = valid - kb * 8;
                if ((kb & 1) == 0) {
                    ++box;
                    ok = __all_sync(0xffffffffu, mbar_wait(&box_full[box % BOXES], box / BOXES & 1));
                    if (!ok) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 47, item); break; }
                }
                // bytes behind the last block: 1 (the codes there are zero)
                const uint64_t keep = n >= 8 ? ~0ull : (1ull << (8 * n)) - 1, ones = 0x7f7f7f7f7f7f7f7full & ~keep;
                const uint8_t * rows = boxes + box % BOXES * BOX_BYTES + (kb & 1) * 8 + lane * 16;
                uint2 v[12];
#pragma unroll
                for (int j = 0; j < 12; ++j) {
                    uint64_t w = 0;
                    if (j < 4 || (j - 4) * 32 + lane < g.bn) w = *(const uint64_t *) (rows + j * 512);
                    w = (w & keep) | ones;
                    v[j] = make_uint2((uint32_t) w, (uint32_t) (w >> 32));
                }
                if ((kb & 1) != 0 || kb == n_stages - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&box_empty[box % BOXES]);
                }
                ok = __all_sync(0xffffffffu, mbar_wait(&empty[s], (it / STAGES & 1) ^ 1));
                if (!ok) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 44, item); break; }
                tc_fence_after();
                const uint32_t dst = mine + s * 2 * SLAB;
#pragma unroll
                for (int q = 0; q < 3; ++q) {
                    st_cols4(dst + 4 * q, v[4 * q].x, v[4 * q + 1].x, v[4 * q + 2].x, v[4 * q + 3].x);
                    st_cols4(dst + SLAB + 4 * q, v[4 * q].y, v[4 * q + 1].y, v[4 * q + 2].y, v[4 * q + 3].y);
                }
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sf_full[s]);
            }
    } else if (warp >= 8) {
        // two warps a quarter of the rows, they take every second 16 tokens
        const uint32_t mine = tmem + ((uint32_t) (warp & 3) << 21);
        const int half = (warp - 8) >> 2;
        int j = 0;
        for (int item = blockIdx.x; item < g.items; item += gridDim.x, ++j) {
            const int n = item % g.m_tiles * BM + (warp & 3) * 32 + lane, t0 = item / g.m_tiles * g.bn, buf = j & 1, cols = min(g.bn, g.T - t0);
            if (!__all_sync(0xffffffffu, mbar_wait(&acc_full[buf], j >> 1 & 1))) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 45, item); break; }
            tc_fence_after();
            for (int c = 16 * half; c < cols; c += 32) {
                uint32_t v[16];
                tmem_ld16(mine + buf * MAX_BN + c, v);
                tmem_ld_wait();
                if (n >= g.N) continue;
                bf16 * to = (bf16 *) g.out + (long long) (t0 + c) * g.ldo + n;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (c + i < cols) {
                        if (g.out_f32) ((float *) g.out)[(long long) (t0 + c + i) * g.ldo + n] = __uint_as_float(v[i]);
                        else *to = __float2bfloat16(__uint_as_float(v[i]));
                    }
                    to += g.ldo;
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buf]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 2) tmem_dealloc(tmem, 512);
}

}  // namespace

// a [T][K], b [N][K] in 4 bits: codes row-major and dense, scale rows a_ld / b_ld bytes apart (multiples of 16, the arrays 16-byte aligned).
extern "C" JIB_EXPORT int jib_mx4_matmul(const void * a_codes, const void * a_scales, long long a_ld, const void * b_codes, const void * b_scales,
                                         long long b_ld, void * out, long long ldo, int out_f32, int T, int N, int K, int * status, void * stream) {
    if (T <= 0) return 0;
    if (N <= 0 || K <= 0 || K % 32 || a_ld < K / 32 || b_ld < K / 32) return JIB_E_ARG;
    if (((uintptr_t) a_scales | (uintptr_t) b_scales | (uintptr_t) a_ld | (uintptr_t) b_ld) & 15) return JIB_E_ALIGN;
    // The width of a token tile: the one whose rounds over the machine cost least (a tile's fixed part is worth some 24 tokens).
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148, m_tiles = (N + BM - 1) / BM;
    int bn = 16;
    long long best = -1;
    for (int w = 16; w <= MAX_BN; w += 16) {
        const long long tiles = (long long) m_tiles * ((T + w - 1) / w), cost = (tiles + sms - 1) / sms * (w + 24);
        if (best < 0 || cost <= best) { best = cost; bn = w; }
        if (w >= T) break;
    }
    Args g;
    g.out = out; g.ldo = ldo; g.status = status; g.T = T; g.N = N; g.K = K; g.bn = bn; g.out_f32 = out_f32; g.m_tiles = m_tiles;
    const long long items = (long long) m_tiles * ((T + bn - 1) / bn);
    if (items > 0x3fffffff) return JIB_E_ARG;
    g.items = (int) items;
    CUtensorMap ma, mb;
    int rc = jib::tma_rows_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, a_codes, T, K / 2, K / 2, bn);
    if (rc) return rc;
    rc = jib::tma_rows_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, b_codes, N, K / 2, K / 2, BM);
    if (rc) return rc;
    CUtensorMap mas, mbs;
    rc = jib::tma_bytes_map(&mas, a_scales, T, a_ld, 16, bn);
    if (rc) return rc;
    rc = jib::tma_bytes_map(&mbs, b_scales, N, b_ld, 16, BM);
    if (rc) return rc;
    static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
    if (!jib::ensure_dyn_smem(mx4_matmul_kernel, SMEM, attr_done)) return JIB_E_LAUNCH;
    JIB_LAUNCH((mx4_matmul_kernel), (unsigned) (items < sms ? items : sms), THREADS, SMEM, (cudaStream_t) stream, ma, mb, mas, mbs, g);
    return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH;
}
