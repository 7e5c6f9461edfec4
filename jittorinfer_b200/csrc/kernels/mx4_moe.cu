// A mixture-of-experts layer over packed 4-bit experts for up to 8 tokens, in two launches: the router's outputs, then everything else --
// choice of experts, gate and up products, activation, down products, weighted sum, residual.
//
// The reference runs router, choice, sorting, grouped products and the weighted sum as some dozen launches
// (src/llama-graph-ffn.cpp:145-260); the bf16 path here takes five.  Width 2048, 64 experts of 1408, 6 chosen + 2 shared, norm included: 1 token 33.7 us, 8
// tokens 66 (bf16: 43 and 119); alone, 8 tokens read their 170 MB of weights at 2.5 TB/s over the whole layer, at 3.4 TB/s within its two loops.
//
// The layer is bound by the stream of the chosen experts' weights, and on the way by instructions: a weight has 2.8 issue slots at the memory's rate.  So
// the second launch is two plain loops over chunks and a meeting of its CTAs in between; every warp is alike, and keeps a ring of weights of its
// own filled with asynchronous copies.  (Versions with units drawn one by one, special warps for copies and sums, and waits for single
// experts' hidden units overlapped more and took twice the time: their code did not stay in the instruction cache.)
//
// Gate and up: GW warps share 16 hidden units of an expert, each a part of K, and add their sums up in order in shared memory.  Hidden units go to
// memory as fragments, fp16, each 16 of a token scaled by a power of two that is kept beside them.  Groups draw their units from a counter, so every
// unit is done by a CTA that runs; a CTA whose groups find none left waits until all are done: nothing waits for a CTA that has not started.
// Down: the chunks of 64 rows x all chosen experts' hidden units are one line, cut into equal pieces, one for each CTA.  Where a piece ends inside 64
// rows, the sums meet in memory, and the CTA that comes last adds them up in their order.
#include "gate.cuh"
#include "jib_kernels.h"
#include "mx4_stream.cuh"
#include "pdl.cuh"

namespace {

using namespace sm100;

constexpr int MAX_T = 8, MAX_K = 32;                          // tokens, choices of a token
constexpr int NW = 16, THREADS = NW * 32;                     // warps
constexpr int MOST_SMEM = 227 * 1024, MAX_DEPTH = 4, KNOWN = 8, AHEAD = 3;       // units of a group: that it remembers, that it draws ahead
constexpr int BIAS = 113;                                     // top_exponent() + BIAS is 1 .. 240
constexpr uint64_t WAIT_NS = JIB_WAIT_NS;                     // for the other CTAs' hidden units

struct MoeArgs {
    const bf16 * residual;                   // may be NULL
    const uint4 * xf;                        // fragments of x, then the exponents of its 8 rows
    const float * logits, * bias;            // logits NULL: ids and weights are given
    const int * ids;
    const float * wts;
    const uint8_t * gu, * down, * gu_factors, * down_factors;
    const int * gu_exp, * down_exp;
    __half * h;                              // hidden units: [slot][chunks of F] fragments, each 16 of a token scaled by a power of two ...
    uint8_t * h_exp;                         // ... [slot][chunk][token][16 units], BIAS more than its exponent
    float * part;                            // [pieces][512]
    bf16 * out;
    int * sync;                              // zeros: units of gate and up drawn, units done (and two more), the largest byte of h_exp of each slot and token
                                             // [slots][8], pieces done of each 64 rows
    int * status;
    long long ldr;
    int T, max_slots, d, F, E, k, n_group, topk_group, norm, sigmoid, n_shared, group_top2, act, gw, depth1, depth2;
    float scale;
};

// Shared memory: tables; sums, three times; the warps' rings of chunks, for gate and up behind the tokens' fragments.
struct Layout {
    static_assert((48 + 4 * KNOWN * 8) % 16 == 0, "the exponents' place");
    static constexpr int SUMS = 8;                                // of a lane
    static constexpr int RED = NW * 32 * SUMS * 4;
    static constexpr int BUFFERS = 3;                             // of sums (see where a unit of gate and up is finished)
    static_assert(BUFFERS * RED >= NW * (MAX_E + 32) * 4, "scratch of the choice");
    __host__ __device__ static int frags(int d) { return mx4::chunks(d) * mx4::FRAG; }
    __host__ __device__ static int tables(int slots) { return (slots * 32 + MAX_E * 4 * 3 + MAX_T * MAX_K * 8 + 64 + 4 * KNOWN * (8 + 128) + 127) / 128 * 128; }
    __host__ __device__ static int base(int slots) { return 128 + tables(slots) + BUFFERS * RED; }
    __host__ __device__ static int bytes(int d, int slots, int depth1, int depth2) {
        const int a = frags(d) + NW * depth1 * mx4::SLOT, b = NW * depth2 * mx4::SLOT;
        return base(slots) + (a > b ? a : b);
    }
};

// 2^-n in fp16, twice 
__device__ __forceinline__ uint32_t below(int n) {
    const float f = __uint_as_float((uint32_t) min(max(127 - n, 0), 127) << 23);
    const __half2 h = __floats2half2_rn(f, f);
    return *(const uint32_t *) &h;
}

__device__ __forceinline__ int ld_acquire(const int * p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

__global__ void __launch_bounds__(THREADS, 1) mx4_moe_kernel(const MoeArgs g) {
    using L = Layout;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * base = (uint8_t *) (((uintptr_t) smem_raw + 127) & ~(uintptr_t) 127);
    float * wtab = (float *) base;                                 // [slot][8] weight of each token, 0: not chosen
    int * slot_of = (int *) (wtab + g.max_slots * 8), * expert_of = slot_of + MAX_E, * mask = expert_of + MAX_E;
    int * ids_s = mask + MAX_E;
    float * wts_s = (float *) (ids_s + MAX_T * MAX_K);
    uint64_t * acts_full = (uint64_t *) (wts_s + MAX_T * MAX_K);
    int * word = (int *) (acts_full + 1);                          // [0] slots, [1] units done by this CTA, [2] pieces done
    long long * drawn = (long long *) (word + 10);                 // (48 bytes behind the barrier) of each group (at most 4) the last KNOWN units: number << 32 | unit
    int * exps = (int *) (drawn + 4 * KNOWN);                      // ... and the exponents of their 32 rows: 16-byte copies, 304 bytes behind the barrier
    float * red = (float *) (base + L::tables(g.max_slots));
    uint8_t * work = (uint8_t *) (red + L::BUFFERS * L::RED / 4);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g4 = lane >> 2, t2 = 2 * (lane & 3);

    if (threadIdx.x == 0) {
        mbar_init(acts_full, 1);
        fence_barrier_init();
    }
    for (int i = threadIdx.x; i < g.max_slots * 8; i += THREADS) wtab[i] = 0.f;
    for (int i = threadIdx.x; i < MAX_E; i += THREADS) { slot_of[i] = 0; mask[i] = 0; }
    if (threadIdx.x < 4 * KNOWN) drawn[threadIdx.x] = -1;
    __syncthreads();
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    if (warp % g.gw == 0) {
        // one draw for all: a group stops at its first unit that is none, so its units have to ascend, and lanes' own draws come in any order
        const int unit0 = __shfl_sync(0xffffffffu, lane == 0 ? atomicAdd(g.sync, AHEAD) : 0, 0);
        if (lane < AHEAD) drawn[warp / g.gw * KNOWN + lane] = (long long) lane << 32 | (unit0 + lane);
    }
    if (threadIdx.x == THREADS - 1) {
        word[1] = 0;
        mbar_expect_tx(acts_full, L::frags(g.d));
        mx4::bulk_load(work, g.xf, L::frags(g.d), acts_full);
    }

    // ---- which experts, for which tokens, with which weights ----
    const int kk = g.k + g.n_shared;
    if (g.logits != nullptr) {
        const int E = g.E - g.n_shared;
        if (warp < g.T)
            gate_token(g.logits + (size_t) warp * E, g.bias, nullptr, nullptr, warp, E, g.k, g.n_group, g.topk_group, g.scale, g.norm, g.sigmoid, g.n_shared,
                       g.group_top2, red + warp * (MAX_E + 32), red + warp * (MAX_E + 32) + MAX_E, ids_s, wts_s);
    } else {
        for (int i = threadIdx.x; i < g.T * kk; i += THREADS) { ids_s[i] = g.ids[i]; wts_s[i] = g.wts[i]; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < g.T * kk; i += THREADS)
        if ((unsigned) ids_s[i] < (unsigned) g.E) slot_of[ids_s[i]] = 1;
    __syncthreads();
    if (warp == 0) {
        int n = 0;
#pragma unroll 4
        for (int e = lane; e < (g.E + 31) / 32 * 32; e += 32) {
            const bool hit = slot_of[e] != 0;
            const unsigned m = __ballot_sync(0xffffffffu, hit);
            const int s = n + __popc(m & ((1u << lane) - 1));
            slot_of[e] = s;
            if (hit) expert_of[s] = e;
            n += __popc(m);
        }
        if (lane == 0) word[0] = n;
    }
    __syncthreads();
    // a thread a choice; of an expert that a token chose several times the first adds the weights up, in their order
    for (int i = threadIdx.x; i < g.T * kk; i += THREADS) {
        const int e = ids_s[i], t = i / kk;
        if ((unsigned) e >= (unsigned) g.E) continue;
        float w = 0.f;
        bool repeated = false;
#pragma unroll 4
        for (int j = t * kk; j < (t + 1) * kk; ++j)
            if (ids_s[j] == e) {
                w += wts_s[j];
                repeated |= j < i;
            }
        if (repeated) continue;
        wtab[slot_of[e] * 8 + t] = w;
        atomicOr(&mask[slot_of[e]], 1 << t);
    }
    __syncthreads();
    const int slots = word[0], C1 = mx4::chunks(g.d), C2 = mx4::chunks(g.F), RB1 = g.F / 16, G = gridDim.x, U = slots * RB1;
    int * done = g.sync + 1, * h_top = g.sync + 4, * pieces_done = h_top + g.max_slots * 8;
    const uint64_t policy = l2_policy_evict_first();

    // ---- gate and up ----
    if (!mx4::wait_all(acts_full, 0) && lane == 0) jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 51, warp);
    {
        const int group = warp / g.gw, wg = warp % g.gw, count = (C1 - wg + g.gw - 1) / g.gw, depth = min(g.depth1, max(2 * count, 1));
        const uint8_t * ring = work + L::frags(g.d) + warp * g.depth1 * mx4::SLOT;
        const uint32_t ring_s = smem_u32(ring);
        const uint4 * acts = (const uint4 *) work + lane;
        const int R1 = 2 * g.F;
        int * rows_of = exps + group * KNOWN * 32;
        // The group's unit number i, once it is drawn (by the group's first warp, which draws number i + 3 before it begins with number i + 1).
        auto unit = [&](int i) -> int {
            volatile const long long * at = drawn + group * KNOWN + i % KNOWN;
#pragma unroll 1
            for (int tries = 0; tries < 1 << 22; ++tries) {
                const long long v = *at;
                if ((int) (v >> 32) == i) return (int) v;
            }
            jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 53, i);
            return U;
        };
        // Asks for this warp's next chunks: of unit after unit the chunks wg, wg + gw .., at most two units ahead; and for the exponents of a unit's rows.
        int ia = 0, ka = wg, at = 0, ua = 0;
        const uint8_t * codes = nullptr, * factors = nullptr;           // of this lane's next 16 bytes (NULL: of a unit not begun)
        const size_t step = (size_t) g.gw * R1;
        auto ask = [&] {
            if (codes == nullptr && ua < U) ua = unit(ia);
            if (ua < U && ka < C1) {
                if (codes == nullptr) {
                    const int slot = ua / RB1, rb = ua - slot * RB1, e = expert_of[slot];
                    const size_t row = ((size_t) e * C1 + wg) * R1 + rb * 32;
                    codes = g.gu + row * mx4::CODES + lane * 16;
                    factors = g.gu_factors + row * mx4::SCALES + lane * 16;
                    if (lane < 8 && wg < 1)
                        mx4::copy16(smem_u32(rows_of + (ia % KNOWN) * 32 + lane * 4), g.gu_exp + (size_t) e * R1 + rb * 32 + lane * 4, policy);
                }
                mx4::copy_chunk(ring_s + at * mx4::SLOT, codes, factors, policy);
                at = at + 1 == depth ? 0 : at + 1;
                codes += step * mx4::CODES;
                factors += step * mx4::SCALES;
                ka += g.gw;
                if (ka >= C1) {
                    ka = wg;
                    codes = nullptr;
                    ++ia;
                }
            }
            mx4::copies_commit();
        };
#pragma unroll 1
        for (int i = 0; i < depth; ++i) ask();
        int here = 0, i = 0;
        const int set = wg >> 1, job = wg & 1, col = t2 + job;
        const int xe = ((const int *) ((const uint8_t *) g.xf + L::frags(g.d)))[col];
#pragma unroll 1
        for (int u; (u = unit(i)) < U; ++i) {
            const int parity = i & 1;
            float * sums = red + i % L::BUFFERS * (L::RED / 4);
            int next = 0;
            if (wg == 0 && lane == 0) next = atomicAdd(g.sync, 1);
            float acc[2][4] = {};
#pragma unroll 1
            for (int k = wg; k < C1; k += g.gw) {
                mx4::copies_wait(depth - 1);
                __syncwarp();
                const uint4 * b = acts + k * 128;
                mx4::chunk_mma(ring + here * mx4::SLOT, acc, [&](int p) { return b[p * 32]; });
                here = here + 1 == depth ? 0 : here + 1;
                __syncwarp();
                ask();
            }
            if (wg == 0 && lane == 0) *(volatile long long *) (drawn + group * KNOWN + (i + AHEAD) % KNOWN) = (long long) (i + AHEAD) << 32 | next;
            // the group's sums, in the order of its warps: [gate or up][register][lane]
            float * mine = sums + warp * L::SUMS * 32 + lane;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int c = 0; c < 4; ++c) mine[(m * 4 + c) * 32] = acc[m][c];
            // Two warps finish the unit: the first two and the next two take turns, and the two whose turn it is not go on without waiting: they wait for all
            // at the next unit, so that a buffer is free again three units later.
            const int barrier = 1 + group * 2 + parity;
            if (set == (parity ^ 1)) asm volatile("bar.arrive %0, %1;" ::"r"(barrier), "r"(g.gw * 32) : "memory");
            else asm volatile("bar.sync %0, %1;" ::"r"(barrier), "r"(g.gw * 32) : "memory");
            if (set == parity) {
                // token col, hidden units f + g and f + g + 8
                const int slot = u / RB1, f = (u - slot * RB1) * 16;
                const float * from = sums + (warp - wg) * L::SUMS * 32 + job * 32 + lane;
                float z[2] = {0.f, 0.f}, v[2] = {0.f, 0.f};
#pragma unroll 4
                for (int w = 0; w < g.gw; ++w)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        z[c] += from[w * L::SUMS * 32 + 64 * c];
                        v[c] += from[w * L::SUMS * 32 + 128 + 64 * c];
                    }
                const int * rows = rows_of + i % KNOWN * 32 + g4;
                uint32_t most = 0;
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    v[c] = mx4::gated(mx4::times_pow2(z[c], rows[8 * c] + xe), mx4::times_pow2(v[c], rows[16 + 8 * c] + xe), g.act);
                    most = max(most, __float_as_uint(v[c]) & 0x7fffffffu);
                }
#pragma unroll
                for (int o = 4; o < 32; o *= 2) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
                if (mask[slot] >> col & 1) {
                    const int he = mx4::top_exponent(most);
                    const float up = mx4::pow2_normal(14 - he);
                    const size_t tile = (size_t) slot * C2 + f / mx4::COLS;
                    __half * to = g.h + ((tile * 4 + f % 32 / 8) * 32 + col * 4 + f % mx4::COLS / 32) * 8 + g4;
                    to[0] = __float2half_rn(v[0] * up);
                    to[32 * 8] = __float2half_rn(v[1] * up);
                    if (g4 == 0) {
                        g.h_exp[(tile * 8 + col) * 8 + f % mx4::COLS / 16] = (uint8_t) (he + BIAS);
                        atomicMax(h_top + slot * 8 + col, he + BIAS);
                    }
                }
            }
        }
        mx4::copies_wait(0);
        __threadfence();
        if (wg == 0 && lane == 0) atomicAdd(&word[1], i);
        __syncthreads();
        if (threadIdx.x == 0) atomicAdd(done, word[1]);
    }

    // ---- down: places (64 rows, chunk of an expert's hidden units) i0 .. i1 - 1 of the line ----
    const int P = slots * C2, groups = (g.d + 63) / 64;
    const long long N = (long long) groups * P;
    const int pieces = N < G ? (int) N : G;
    if (N == 0) {                                 // no expert: the residual, or zeros
        for (int i = blockIdx.x * THREADS + threadIdx.x; i < g.T * g.d; i += G * THREADS) {
            const int t = i / g.d, o = i % g.d;
            g.out[i] = g.residual != nullptr ? g.residual[t * g.ldr + o] : __float2bfloat16(0.f);
        }
        return;
    }
    if ((int) blockIdx.x >= pieces) return;
    const int i0 = (int) (blockIdx.x * N / pieces), i1 = (int) ((blockIdx.x + 1) * N / pieces);
    const int pair = warp >> 3, wj = warp & 7, depth = g.depth2;
    const uint8_t * ring = work + warp * depth * mx4::SLOT;
    const uint32_t ring_s = smem_u32(ring);
    // This warp's places: of each piece of 64 rows' places [a, b) those at a + wj, a + wj + 8, ..
    struct Place {
        int gr, p, end, slot, c;        // rows, place (slot * C2 + c) and the piece's end there
    };
    auto start = [&](Place & x, int gr, int p) {
        x.gr = gr;
        x.p = p + wj;
        x.end = min(P, i1 - gr * P);
        x.slot = x.p / C2;
        x.c = x.p - x.slot * C2;
    };
    auto advance = [&](Place & x) {              // past the last place: p >= end in the last rows
        x.p += 8;
        x.c += 8;
#pragma unroll 1
        while (x.c >= C2) { x.c -= C2; ++x.slot; }
#pragma unroll 1
        while (x.p >= x.end && (x.gr + 1) * P < i1) start(x, x.gr + 1, 0);
    };
    auto begin = [&](Place & x) {
        start(x, i0 / P, i0 % P);
#pragma unroll 1
        while (x.p >= x.end && (x.gr + 1) * P < i1) start(x, x.gr + 1, 0);
    };
    Place xa, xh;                                // asked for: chunks; hidden units
    begin(xa);
    begin(xh);
    int at = 0;
    auto first_row = [&](const Place & x) { return x.gr * 64 + pair * 32 < g.d ? x.gr * 64 + pair * 32 : 0; };      // (rows behind the last: any)
    auto ask = [&] {
        if (xa.p < xa.end) {
            const size_t row = ((size_t) expert_of[xa.slot] * C2 + xa.c) * g.d + first_row(xa);
            mx4::copy_chunk(ring_s + at * mx4::SLOT, g.down + row * mx4::CODES + lane * 16, g.down_factors + row * mx4::SCALES + lane * 16, policy);
            at = at + 1 == depth ? 0 : at + 1;
            advance(xa);
        }
        mx4::copies_commit();
    };
    // A place's hidden units: fragments (zeros for tokens that have not chosen this expert, and behind the last hidden unit), their exponents' bytes, the
    // largest byte of this lane's token; the exponents of this lane's rows.
    struct Hidden {
        uint4 b[4];
        uint32_t ex;
        int top, row[4];
    } next;
    auto fetch = [&] {
        if (xh.p >= xh.end) return;
        const size_t tile = xh.slot * C2 + xh.c;
        const int m = mask[xh.slot], * rows = g.down_exp + (size_t) expert_of[xh.slot] * g.d + first_row(xh) + g4;
        const bool units = xh.c * mx4::COLS + 32 * (lane & 3) < g.F;
#pragma unroll
        for (int i = 0; i < 4; ++i) next.row[i] = __ldg(rows + 8 * i);
        const bool chosen = m >> g4 & 1;
        next.ex = 0u;
        next.top = 0;
        if (chosen) {
            next.ex = __ldcg((const unsigned short *) g.h_exp + (tile * 8 + g4) * 4 + (lane & 3));
            next.top = __ldcg(h_top + xh.slot * 8 + g4);
        }
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            next.b[p] = make_uint4(0u, 0u, 0u, 0u);
            if (chosen && units) next.b[p] = __ldcg((const uint4 *) g.h + (tile * 4 + p) * 32 + lane);
        }
    };
#pragma unroll 1
    for (int i = 0; i < depth; ++i) ask();
    // the other CTAs' hidden units
    if (threadIdx.x == 0) {
        const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
        while (ld_acquire(done) < U) {
            if (globaltimer_ns() - t0 > WAIT_NS) {
                jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 52, blockIdx.x);
                break;
            }
            __nanosleep(32);
        }
    }
    __syncthreads();
    fetch();
    int here = 0;
#pragma unroll 1
    for (int gr = i0 / P; gr * P < i1; ++gr) {
        const int a = max(0, i0 - gr * P), b = min(P, i1 - gr * P);
        float acc[2][4] = {};
#pragma unroll 1
        while (xh.gr == gr && xh.p < xh.end) {
            Hidden h = next;
            const int slot = xh.slot;
            // all hidden units of a token to the power of two of its largest ones
            const uint32_t f0 = below(h.top - (int) (h.ex & 0xff)), f1 = below(h.top - (int) (h.ex >> 8));
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint4 & v = h.b[q];
                v.x = mx4::mul2(v.x, q < 2 ? f0 : f1);
                v.y = mx4::mul2(v.y, q < 2 ? f0 : f1);
                v.z = mx4::mul2(v.z, q < 2 ? f0 : f1);
                v.w = mx4::mul2(v.w, q < 2 ? f0 : f1);
            }
            advance(xh);
            fetch();
            mx4::copies_wait(depth - 1);
            __syncwarp();
            float y[2][4] = {};
            mx4::chunk_mma(ring + here * mx4::SLOT, y, [&](int q) { return h.b[q]; });
            here = here + 1 == depth ? 0 : here + 1;
            __syncwarp();
            ask();
            float r[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = mx4::pow2(h.row[i]);
            const float2 wt = *(const float2 *) (wtab + slot * 8 + t2);
            const int e0 = __shfl_sync(0xffffffffu, h.top, 4 * t2), e1 = __shfl_sync(0xffffffffu, h.top, 4 * t2 + 4);
            const float w0 = wt.x * mx4::pow2_normal(e0 - BIAS - 14), w1 = wt.y * mx4::pow2_normal(e1 - BIAS - 14);
            // (a token that has not chosen this expert takes nothing from it, were its weights NaN)
            const int chosen = mask[slot] >> t2;
#pragma unroll
            for (int m = 0; m < 2; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    // (the factors first: either alone may take y out of fp32's range where the result is well inside)
                    if (chosen & (i & 1 ? 2 : 1)) acc[m][i] += y[m][i] * (r[2 * m + (i >> 1)] * (i & 1 ? w1 : w0));
        }
        float * mine = red + (gr & 1) * (L::RED / 4) + warp * L::SUMS * 32 + lane;
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) mine[(m * 4 + i) * 32] = acc[m][i];
        __syncthreads();
        // thread = (two row blocks, register, lane): its row of one row block, then of the other
        const int half = warp >> 3, m = warp >> 2 & 1, reg = warp & 3, o = gr * 64 + (2 * half + m) * 16 + g4 + 8 * (reg >> 1);
        const float * src = red + (gr & 1) * (L::RED / 4) + half * 8 * L::SUMS * 32 + (m * 4 + reg) * 32 + lane;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < 8; ++w) v += src[w * L::SUMS * 32];
        if (a > 0 || b < P) {
            // pieces first .. last hold places of these rows
            const int first = (int) ((((long long) gr * P + 1) * pieces - 1) / N), last = (int) ((((long long) gr + 1) * P * pieces - 1) / N);
            float * part = g.part + ((size_t) (first + 2 * gr)) * THREADS + threadIdx.x;
            __stcg(part + (blockIdx.x - first) * THREADS, v);
            __threadfence();
            __syncthreads();
            if (threadIdx.x == 0) {
                word[2] = atomicAdd(pieces_done + gr, 1);
                __threadfence();
            }
            __syncthreads();
            if (word[2] != last - first) continue;
            v = 0.f;
#pragma unroll 1
            for (int q0 = 0; q0 <= last - first; q0 += 8) {
                float x[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) x[q] = q0 + q <= last - first ? __ldcg(part + (q0 + q) * THREADS) : 0.f;
#pragma unroll
                for (int q = 0; q < 8; ++q) v += x[q];
            }
        }
        const int t = t2 + (reg & 1);
        if (o < g.d && t < g.T) {
            if (g.residual != nullptr) v += __bfloat162float(g.residual[t * g.ldr + o]);
            g.out[(size_t) t * g.d + o] = __float2bfloat16(v);
        }
    }
    mx4::copies_wait(0);
}

// The layer's first launch: CTAs below E compute router outputs [T][E], the others a token's fragments each (8 of them, zeros from T on); zeros where
// the next launch counts.
__global__ void __launch_bounds__(GATE_NT) mx4_prepare_kernel(const bf16 * __restrict__ x, long long ldx, const float * __restrict__ w_router,
                                                              float * __restrict__ logits, uint4 * __restrict__ xf, int * __restrict__ sync, int n_sync, int T,
                                                              int d, int E) {
    __shared__ float red[GATE_NT / 32][GATE_TG];
    const bool router = (int) blockIdx.x < E;
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    for (int i = blockIdx.x * GATE_NT + threadIdx.x; i < n_sync; i += gridDim.x * GATE_NT) sync[i] = 0;
    if (router) {
        router_rows(x, w_router, nullptr, 0.f, nullptr, logits, 0, T, T, d, E, blockIdx.x, red, nullptr);
        return;
    }
    const int n = blockIdx.x - E, lane = threadIdx.x & 31, C = mx4::chunks(d);
    const bf16 * row = x + n * ldx;
    uint32_t top = 0;
    if (n < T)
        for (int i = threadIdx.x; i < d / 2; i += GATE_NT) {
            const float2 v = __bfloat1622float2(((const __nv_bfloat162 *) row)[i]);
            top = max(top, max(__float_as_uint(v.x) & 0x7fffffffu, __float_as_uint(v.y) & 0x7fffffffu));
        }
    top = __reduce_max_sync(0xffffffffu, top);
    if (lane == 0) red[threadIdx.x >> 5][0] = __uint_as_float(top);
    __syncthreads();
#pragma unroll
    for (int w = 0; w < GATE_NT / 32; ++w) top = max(top, __float_as_uint(red[w][0]));
    const int ex = mx4::top_exponent(top);
    const float unit = mx4::pow2(14 - ex);
    if (threadIdx.x == 0) ((int *) (xf + (size_t) C * 128))[n] = ex - 14;
    for (int i = threadIdx.x; i < C * 16; i += GATE_NT) {          // eight columns
        const int p = i & 3, t = i >> 2 & 3, c = i >> 4;
        xf[(c * 4 + p) * 32 + n * 4 + t] = n < T ? mx4::frag_of(row, c * mx4::COLS + 32 * t + 8 * p, d, unit) : make_uint4(0u, 0u, 0u, 0u);
    }
}

// Stages of chunks that fit, at most MAX_DEPTH (0: not one).
int depth_of(int d, int slots, bool down) {
    using L = Layout;
    for (int i = MAX_DEPTH; i > 0; --i)
        if ((down ? L::bytes(0, slots, 0, i) : L::bytes(d, slots, i, 0)) <= MOST_SMEM) return i;
    return 0;
}

int launch(const MoeArgs & a, cudaStream_t s) {
    using L = Layout;
    static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
    MoeArgs g = a;
    g.depth1 = depth_of(g.d, g.max_slots, false);
    g.depth2 = depth_of(g.d, g.max_slots, true);
    // Warps that share 16 hidden units: whatever takes the fullest group the least time, in chunks of one warp (finishing a unit is worth one more).
    // Two finish a unit, and two more take turns with them.
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148;
    const long long units = (long long) g.max_slots * (g.F / 16);
    long long best = -1;
    for (int gw = 4; gw <= NW; gw *= 2) {
        const long long groups = (long long) sms * (NW / gw), cost = (units + groups - 1) / groups * ((mx4::chunks(g.d) + gw - 1) / gw + 1);
        if (best < 0 || cost < best) { best = cost; g.gw = gw; }
    }
    if (!jib::ensure_dyn_smem(mx4_moe_kernel, MOST_SMEM, attr_done)) return JIB_E_LAUNCH;
    JIB_LAUNCH(mx4_moe_kernel, sms, THREADS, L::bytes(g.d, g.max_slots, g.depth1, g.depth2), s, g);
    return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH;
}

// Experts that T tokens can choose.
int slots_of(int T, int k, int E) { return T * k < E ? T * k : E; }

}  // namespace

extern "C" {

// Whether the two-launch form takes a layer (else 0), and the sizes of its buffers: bytes of xf and of h, floats of part, ints of sync.
JIB_EXPORT int jib_mx4_moe_sizes(int T, int d, int F, int E, int k, long long * sizes) {
    if (T < 1 || T > MAX_T || k < 1 || k > MAX_K || E < 1 || E > MAX_E || d % 32 || F % 32 || d < 32 || F < 32 || d > GATE_MAXC * GATE_NT * 8) return 0;
    const long long slots = slots_of(T, k, E);
    if (depth_of(d, (int) slots, false) == 0) return 0;
    const long long tiles = slots * mx4::chunks(F);
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148, groups = (d + 63) / 64;
    if (tiles * groups > (1 << 30) || slots * (F / 16) > (1 << 30)) return 0;
    sizes[0] = Layout::frags(d) + 32;
    sizes[1] = tiles * (mx4::FRAG + 64);
    sizes[2] = (long long) (sms + 2 * groups) * THREADS;
    sizes[3] = 4 + slots * 8 + groups;
    return 1;
}

// The layer's first launch: x as the second one reads it, zeros in sync, and with w_router [E][d] the router's outputs [T][E].
JIB_EXPORT int jib_mx4_moe_prepare(const void * x, long long ldx, const float * w_router, float * logits, void * xf, int * sync, int n_sync, int T, int d, int E,
                                   void * stream) {
    if (w_router == nullptr) E = 0;
    if (T < 1 || T > MAX_T || E < 0 || E > MAX_E || d % 32 || d > GATE_MAXC * GATE_NT * 8 || (E > 0 && ldx != d)) return JIB_E_ARG;
    if (((uintptr_t) x | (uintptr_t) (ldx * 2) | (uintptr_t) xf | (uintptr_t) w_router) & 15) return JIB_E_ALIGN;
    JIB_LAUNCH((mx4_prepare_kernel), E + 8, GATE_NT, 0, (cudaStream_t) stream, (const bf16 *) x, ldx, w_router, logits, (uint4 *) xf, sync, n_sync, T, d, E);
    return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH;
}

// out = residual + sum over the choices of weight * down(act(gate) * up).  With logits the launch chooses the experts itself (the gate's arguments are
// those of jib_moe_gate; the last n_shared of the E experts take every token), else ids and wts [T][k] do (n_shared 0).
JIB_EXPORT int jib_mx4_moe(const jib_mx4_moe_desc * m, void * stream) {
    long long sizes[4];
    if (m->T <= 0) return 0;
    if (m->n_shared < 0 || m->k < 1 || !jib_mx4_moe_sizes(m->T, m->d, m->F, m->E, m->k + m->n_shared, sizes)) return JIB_E_ARG;
    if (m->logits == nullptr ? (m->ids == nullptr || m->wts == nullptr || m->n_shared != 0)
                             : (m->n_shared >= m->E || m->k > m->E - m->n_shared || m->n_group < 1 || m->n_group > 32 || (m->E - m->n_shared) % m->n_group))
        return JIB_E_ARG;
    if (((uintptr_t) m->gu | (uintptr_t) m->down | (uintptr_t) m->gu_factors | (uintptr_t) m->down_factors | (uintptr_t) m->gu_exp | (uintptr_t) m->h | (uintptr_t) m->xf | (uintptr_t) m->part | (uintptr_t) m->sync | (uintptr_t) m->down_exp) & 15)
        return JIB_E_ALIGN;
    if (m->part_floats < sizes[2]) return JIB_E_SCRATCH;          // (goes by the device's SMs)
    MoeArgs a;
    a.xf = (const uint4 *) m->xf; a.residual = (const bf16 *) m->residual; a.logits = m->logits; a.bias = m->bias; a.ids = m->ids; a.wts = m->wts;
    a.gu = (const uint8_t *) m->gu; a.down = (const uint8_t *) m->down; a.gu_exp = m->gu_exp; a.down_exp = m->down_exp;
    a.max_slots = slots_of(m->T, m->k + m->n_shared, m->E);
    a.h = (__half *) m->h; a.h_exp = (uint8_t *) m->h + (long long) a.max_slots * mx4::chunks(m->F) * mx4::FRAG; a.part = m->part; a.out = (bf16 *) m->out; a.sync = m->sync; a.status = m->status;
    a.ldr = m->ldr; a.gu_factors = m->gu_factors; a.down_factors = m->down_factors;
    a.T = m->T; a.d = m->d; a.F = m->F; a.E = m->E; a.k = m->k; a.n_group = m->n_group; a.topk_group = m->topk_group; a.norm = m->norm; a.sigmoid = m->sigmoid;
    a.n_shared = m->n_shared; a.group_top2 = m->group_top2; a.act = m->act; a.scale = m->scale;
    return launch(a, (cudaStream_t) stream);
}

}  // extern "C"
