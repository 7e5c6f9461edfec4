// Product of two microscaled 4-bit operands on the 4-bit tensor cores: out[t][n] = sum_k a[t][k] b[n][k].
//
// tcgen05.mma.kind::mxf4.block_scale multiplies E2M1 codes and applies the blocks' scales itself, 64 columns an instruction: nothing is
// expanded.  b (the weights) is operand A of the instruction, 128 rows a tile, a's rows are its columns, up to 208 a tile: so few tokens cost
// a narrow tile.  Where it costs less, two CTAs (PAIR, cta_group::2) share 256 weights by up to 192 tokens, of which each keeps half.
//
// The scales live in tensor memory: column j of a slab holds, in lane l of every quarter, the four scale bytes of row 32 j + l for 128 columns of K.  They
// come in boxes of 16 bytes a row (512 columns, two stages) in a ring of their own, and eight warps, four a stage in turn, move them to tensor
// memory ahead of their stage.  (Read from global memory by those warps, stage by stage, they took 1200 clocks a stage, three times the products; four
// warps for them took longer than the products of a pair.)  2048 x 5120 by 12288, quantising included: 91 us with four warps for scales and four for
// results, 81 with eight for results, 67 with eight for scales and pairs (3.85 PFLOP/s; pairs alone 86); bound by the scales' way and shared memory.
#include "sm100.cuh"
#include "jib_kernels.h"
#include "mx4_pair.cuh"
#include "pdl.cuh"
#include "tma_host.cuh"

namespace {

using namespace sm100;
typedef __nv_bfloat16 bf16;

constexpr int BM = 128, KS = 256;                                // weights a tile, columns a stage
constexpr int A_BYTES = BM * 128;
constexpr int BOXES = 3;
constexpr int SLAB = 12;                                         // columns of the scales of 128 columns of K: 4 of A, 8 of B
constexpr int THREADS = 640;                                     // producer, issuer, one idle, producer of scales; eight scale warps; eight epilogue warps

template <bool PAIR>
struct Shape {
    static constexpr int MAX_BN = PAIR ? 192 : 208, STAGES = PAIR ? 5 : 4;         // tokens of a tile at most
    static constexpr int STAGE_BYTES = A_BYTES + (PAIR ? MAX_BN / 2 : MAX_BN) * 128;
    static constexpr int BOX_BYTES = (BM + MAX_BN) * 16;                           // scales of two stages
    static constexpr int SMEM = STAGES * STAGE_BYTES + BOXES * BOX_BYTES + 1024 + 256;
    static constexpr int SF0 = 2 * MAX_BN;                                         // two accumulators, then the scales of each stage
    static_assert(SF0 + STAGES * 2 * SLAB <= 512 && SMEM <= 227 * 1024, "tensor memory, shared memory");
};

struct Args {
    void * out;
    long long ldo;
    int * status;
    int T, N, K, bn, out_f32, m_tiles, items;
};

__device__ __forceinline__ void st_cols4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
template <bool PAIR>
__device__ __forceinline__ void mma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, bool accumulate) {
    if (PAIR)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t) accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %6, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
            ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"((uint32_t) accumulate)
            : "memory");
}
// E2M1 x E2M1 with E8M0 scales, m x n, the scales in bytes `half` and `half` + 1 of their words.
__device__ __forceinline__ uint32_t idesc_mxf4(int m, int n, uint32_t half) {
    return half << 4 | 1u << 7 | 1u << 10 | (uint32_t) (n >> 3) << 17 | 1u << 23 | (uint32_t) (m >> 4) << 24 | half << 29;
}

template <bool PAIR>
__global__ void __launch_bounds__(THREADS, 1) mx4_matmul_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
                                                                const __grid_constant__ CUtensorMap tm_as, const __grid_constant__ CUtensorMap tm_bs, const Args g) {
    using S = Shape<PAIR>;
    constexpr int STAGES = S::STAGES, STAGE_BYTES = S::STAGE_BYTES, BOX_BYTES = S::BOX_BYTES, SF0 = S::SF0, MAX_BN = S::MAX_BN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * tiles = (uint8_t *) (((uintptr_t) smem_raw + 1023) & ~(uintptr_t) 1023);
    uint8_t * boxes = tiles + STAGES * STAGE_BYTES;
    uint64_t * full = (uint64_t *) (boxes + BOXES * BOX_BYTES), * empty = full + STAGES, * sf_full = empty + STAGES, * acc_full = sf_full + STAGES,
             * acc_empty = acc_full + 2, * box_full = acc_empty + 2, * box_empty = box_full + BOXES;
    uint32_t * tmem_slot = (uint32_t *) (box_empty + BOXES);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    // of a pair each CTA has 128 rows of weights and keeps half of the tokens
    const int rank = PAIR ? blockIdx.x & 1 : 0, first = PAIR ? blockIdx.x >> 1 : blockIdx.x, step = PAIR ? gridDim.x >> 1 : gridDim.x;
    const int rows = PAIR ? 2 * BM : BM, an = PAIR ? g.bn / 2 : g.bn;
    if (threadIdx.x == 0) {
        for (int i = 0; i < STAGES; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], 1); mbar_init(&sf_full[i], PAIR ? 8 : 4); }
        for (int i = 0; i < 2; ++i) { mbar_init(&acc_full[i], 1); mbar_init(&acc_empty[i], PAIR ? 16 : 8); }
        for (int i = 0; i < BOXES; ++i) { mbar_init(&box_full[i], 1); mbar_init(&box_empty[i], 8); }
        fence_barrier_init();
        prefetch_tmap(&tm_as);
        prefetch_tmap(&tm_bs);
        prefetch_tmap(&tm_a);
        prefetch_tmap(&tm_b);
    }
    if (warp == 2) mx4::alloc_all<PAIR>(tmem_slot);
    tc_fence_before();
    __syncthreads();
    if (PAIR) mx4::both_here();              // barriers are arrived at from the other CTA
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    const int n_stages = (g.K + KS - 1) / KS;

    if (warp == 0) {
        if (elect_one()) {
            int it = 0;
            bool ok = true;
            for (int item = first; item < g.items && ok; item += step) {
                const int n0 = item % g.m_tiles * rows + rank * BM, t0 = item / g.m_tiles * g.bn;
                for (int kb = 0; kb < n_stages; ++kb, ++it) {
                    const int s = it % STAGES;
                    if (!mbar_wait(&empty[s], (it / STAGES & 1) ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 41, item); ok = false; break; }
                    uint8_t * st = tiles + s * STAGE_BYTES;
                    if (rank == 0) mbar_expect_tx(&full[s], (PAIR ? 2 : 1) * (A_BYTES + an * 128));
                    mx4::load<PAIR>(st, &tm_b, &full[s], kb * 128, n0);
                    mx4::load<PAIR>(st + A_BYTES, &tm_a, &full[s], kb * 128, t0 + rank * an);
                }
            }
            // copies in flight end before the memory is given back
            if (!ok && rank == 0)
                for (int i = it - STAGES < 0 ? 0 : it - STAGES; i < it; ++i) mbar_wait(&full[i % STAGES], i / STAGES & 1);
        }
        __syncwarp();
    } else if (warp == 1) {
        if (rank == 0 && elect_one()) {
            const uint64_t desc0 = desc_k_sw128(smem_u32(tiles));
            const uint32_t id0 = idesc_mxf4(rows, g.bn, 0), id1 = idesc_mxf4(rows, g.bn, 2);
            int it = 0, j = 0;
            bool ok = true;
            for (int item = first; item < g.items && ok; item += step, ++j) {
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
                        mma_mxf4<PAIR>(acc, a + 2 * q, b + 2 * q, q & 1 ? id1 : id0, sf + q / 2 * SLAB, sf + q / 2 * SLAB + 4, (kb | q) != 0);
                    mx4::commit<PAIR>(&empty[s]);
                }
                mx4::commit<PAIR>(&acc_full[buf]);
            }
        }
        __syncwarp();
    } else if (warp == 3) {
        if (elect_one()) {
            int it = 0;
            bool ok = true;
            for (int item = first; item < g.items && ok; item += step) {
                const int n0 = item % g.m_tiles * rows + rank * BM, t0 = item / g.m_tiles * g.bn;
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
    } else if (warp >= 4 && warp < 12) {
        // scales of a stage, eight bytes a row: four warps take the even stages of a tile, four the odd ones
        const uint32_t mine = tmem + ((uint32_t) (warp & 3) << 21) + SF0;
        const int valid = g.K / 32, odd = (warp - 4) >> 2;
        int it = odd, box = 0;
        bool ok = true;
        for (int item = first; item < g.items && ok; item += step, it -= n_stages & 1)
            for (int kb = odd; kb < n_stages + odd; kb += 2, it += 2, ++box) {          // (the odd ones' last turn may have a box and no stage)
                const int s = it % STAGES, n = valid - kb * 8;
                ok = __all_sync(0xffffffffu, mbar_wait(&box_full[box % BOXES], box / BOXES & 1));
                if (!ok) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 47, item); break; }
                // bytes behind the last block: 1 (the codes there are zero)
                const uint64_t keep = n >= 8 ? ~0ull : n <= 0 ? 0ull : (1ull << (8 * n)) - 1, ones = 0x7f7f7f7f7f7f7f7full & ~keep;
                const uint8_t * at = boxes + box % BOXES * BOX_BYTES + odd * 8 + lane * 16;
                uint2 v[12];
#pragma unroll
                for (int j = 0; j < 12; ++j) {
                    uint64_t w = 0;
                    if (j < 4 || (j - 4) * 32 + lane < g.bn) w = *(const uint64_t *) (at + j * 512);
                    w = (w & keep) | ones;
                    v[j] = make_uint2((uint32_t) w, (uint32_t) (w >> 32));
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&box_empty[box % BOXES]);
                if (kb >= n_stages) continue;
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
                if (lane == 0) mx4::arrive_first<PAIR>(&sf_full[s]);
            }
    } else if (warp >= 12) {
        // two warps a quarter of the rows, they take every second 16 tokens
        const uint32_t mine = tmem + ((uint32_t) (warp & 3) << 21);
        const int half = (warp - 12) >> 2;
        int j = 0;
        for (int item = first; item < g.items; item += step, ++j) {
            const int n = item % g.m_tiles * rows + rank * BM + (warp & 3) * 32 + lane, t0 = item / g.m_tiles * g.bn, buf = j & 1, cols = min(g.bn, g.T - t0);
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
            if (lane == 0) mx4::arrive_first<PAIR>(&acc_empty[buf]);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) mx4::both_here();              // neither leaves while the other arrives at its barriers or multiplies its rows
    if (warp == 2) mx4::free_all<PAIR>(tmem);
}

int pair_count() {
    static std::atomic<int> known[jib::MAX_DEVICES];
    static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
    return mx4::pair_count(mx4_matmul_kernel<true>, THREADS, Shape<true>::SMEM, known, attr_done);
}

}  // namespace

// a [T][K], b [N][K] in 4 bits: codes row-major and dense, scale rows a_ld / b_ld bytes apart (multiples of 16, the arrays 16-byte aligned).
extern "C" JIB_EXPORT int jib_mx4_matmul(const void * a_codes, const void * a_scales, long long a_ld, const void * b_codes, const void * b_scales,
                                         long long b_ld, void * out, long long ldo, int out_f32, int T, int N, int K, int * status, void * stream) {
    if (T <= 0) return 0;
    if (N <= 0 || K <= 0 || K % 32 || a_ld < K / 32 || b_ld < K / 32) return JIB_E_ARG;
    if (((uintptr_t) a_scales | (uintptr_t) b_scales | (uintptr_t) a_ld | (uintptr_t) b_ld) & 15) return JIB_E_ALIGN;
    // The width of a token tile, of a CTA alone or a pair: whose rounds over the machine cost least.  A stage costs its traffic with shared memory: 128 bytes of
    // each row written and read, of a pair half of the tokens'.
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148, tiles_n = (N + BM - 1) / BM, pairs = N > BM ? pair_count() : 0;
    int bn = 16;
    bool pair = false;
    long long best = -1;
    for (int w = 16; w <= Shape<false>::MAX_BN; w += 16) {
        const long long tt = (T + w - 1) / w, cost = (tiles_n * tt + sms - 1) / sms * (w + BM);
        if (best < 0 || cost <= best) { best = cost; bn = w; pair = false; }
        if (pairs > 0 && w % 32 == 0 && w <= Shape<true>::MAX_BN) {
            const long long both = ((tiles_n + 1) / 2 * tt + pairs - 1) / pairs * (w / 2 + BM);
            if (both < best) { best = both; bn = w; pair = true; }
        }
        if (w >= T) break;
    }
    const int m_tiles = pair ? (tiles_n + 1) / 2 : tiles_n, at_once = pair ? pairs : sms;
    Args g;
    g.out = out; g.ldo = ldo; g.status = status; g.T = T; g.N = N; g.K = K; g.bn = bn; g.out_f32 = out_f32; g.m_tiles = m_tiles;
    const long long items = (long long) m_tiles * ((T + bn - 1) / bn);
    if (items > 0x3fffffff) return JIB_E_ARG;
    g.items = (int) items;
    CUtensorMap ma, mb;
    int rc = jib::tma_rows_map(&ma, CU_TENSOR_MAP_DATA_TYPE_UINT8, a_codes, T, K / 2, K / 2, pair ? bn / 2 : bn);
    if (rc) return rc;
    rc = jib::tma_rows_map(&mb, CU_TENSOR_MAP_DATA_TYPE_UINT8, b_codes, N, K / 2, K / 2, BM);
    if (rc) return rc;
    CUtensorMap mas, mbs;
    rc = jib::tma_bytes_map(&mas, a_scales, T, a_ld, 16, bn);
    if (rc) return rc;
    rc = jib::tma_bytes_map(&mbs, b_scales, N, b_ld, 16, BM);
    if (rc) return rc;
    const unsigned grid = (unsigned) (items < at_once ? items : at_once);
    if (pair) {
        (void) jib::launch_pdl_pairs(mx4_matmul_kernel<true>, grid, dim3(THREADS), Shape<true>::SMEM, (cudaStream_t) stream, ma, mb, mas, mbs, g);
    } else {
        static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
        if (!jib::ensure_dyn_smem(mx4_matmul_kernel<false>, Shape<false>::SMEM, attr_done)) return JIB_E_LAUNCH;
        JIB_LAUNCH((mx4_matmul_kernel<false>), grid, THREADS, Shape<false>::SMEM, (cudaStream_t) stream, ma, mb, mas, mbs, g);
    }
    return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH;
}
