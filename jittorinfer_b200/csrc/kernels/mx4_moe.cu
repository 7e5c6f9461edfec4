// A mixture-of-experts layer over packed 4-bit experts for up to 16 tokens, in two launches: the router's outputs, then everything else --
// choice of experts, gate and up products, activation, down products, weighted sum, residual.
//
// The reference runs router, choice, sorting, grouped products and the weighted sum as some dozen launches
// (src/llama-graph-ffn.cpp:145-260); the bf16 path here takes five.
//
// The layer is bound by the stream of the chosen experts' weights, so the second launch is one stream: every CTA draws units from a counter,
// first 32 hidden units of an expert (rows of gate and up), then 64 rows of down over a share of the chosen experts' hidden units.  A unit of the
// second kind needs hidden units that other CTAs store: an expert's counter says how many of its gate and up units are done.  Units are drawn
// in order and a CTA works them off in order, those of the first kind never wait, so whatever a unit waits for is being worked on: the
// launch ends however few of its CTAs run at a time.
// A stage is NP places along K times four row blocks (gate, up, gate, up; or four of down), and a place's activations.  Roles: 2 NP warps
// multiply two row blocks each at one place, each with its own ring of weights that it keeps filled with asynchronous copies; one thread draws
// units; one warp waits for hidden units and copies them to shared memory; FIN warps take turns in adding a unit's NP sums up, in the
// order of the warps, and finishing its rows.  Sums of shares meet in memory, the share that comes last adds them up in their order.
// Five roles in one kernel are much code, and what runs beside one another has to stay in the instruction cache: waits are short loops, what one thread
// can work out for all (the drawing one) is worked out once, and only the products are unrolled.  (With every wait and index in line the kernel
// was 140 KB and took twice the time.)
#include "gate.cuh"
#include "jib_kernels.h"
#include "mx4_stream.cuh"
#include "pdl.cuh"

namespace {

using namespace sm100;

constexpr int MAX_T = 16, MAX_K = 32;                         // tokens, choices of a token
constexpr int MAX_SHARES = 24, MOST_SMEM = 227 * 1024;
constexpr int BIAS = 113;                                     // top_exponent() + BIAS is 1 .. 240
constexpr uint64_t WAIT_NS = JIB_WAIT_NS;                     // for hidden units that another CTA stores
constexpr int NP = 8, NW = 2 * NP;                            // places of a stage; multiplying warps

struct MoeArgs {
    const bf16 * residual;                   // may be NULL
    const uint4 * xf;                        // fragments of x, then the exponents of its 16 rows
    const float * logits, * bias;            // logits NULL: ids and weights are given
    const int * ids;
    const float * wts;
    const uint8_t * gu, * down;
    const int * gu_exp, * down_exp;
    __half * h;                              // hidden units: [slot][chunks of F][NT] fragments, each 16 of a token scaled by a power of two ...
    uint8_t * h_exp;                         // ... [slot][chunk][token][step], BIAS more than its exponent
    float * part;                            // [d / 64][shares][512 NT]
    bf16 * out;
    int * sync;                              // zeros: next unit (and three more), done gate and up units of each slot [MAX_E], the largest byte of h_exp of
                                             // each slot and token [slots][16], shares done of each 64 rows
    int * status;
    long long ldr, gu_stride, down_stride;
    int T, max_slots, d, F, E, k, n_group, topk_group, norm, sigmoid, n_shared, group_top2, act, shares, ring, depth;
    float scale;
};

// A drawn unit, in shared memory.
struct Unit {
    const uint8_t * weights;      // of its first row block: of the expert's pairs; or of the first expert's matrix of down
    int id, n;                    // id -1: the end; places along K
    int slot, col;                // of down: the first place's expert and chunk
};

// Shared memory: the tokens' fragments; a ring of stages' hidden units (for each place fragments, their exponents' bytes, the exponents of 64 rows, the
// largest bytes of 16 tokens); sums; tables; barriers.
template <int NT>
struct Layout {
    static constexpr int FIN = 2;                                 // finishing warps, each with a buffer of sums
    static constexpr int THREADS = (NW + 2 + FIN) * 32;
    static constexpr int H_EXP = NP * NT * mx4::FRAG, H_ROW = H_EXP + NP * NT * 64, H_TOP = H_ROW + NP * 256, HID = H_TOP + NP * 64;
    static constexpr int SUMS = 8 * NT;                           // of a lane
    static constexpr int RED = NW * 32 * SUMS * 4;                // one unit's sums of every warp
    static constexpr int MAX_RING = 3, QUEUE = 2;                 // stages of hidden units; units drawn and not begun by all
    static constexpr int DEEP = NW * 2 * mx4::CHUNK, MAX_DEPTH = 4;       // weights of a stage; stages asked for ahead
    static constexpr int BARS = 16 + (2 * MAX_RING + 2 * QUEUE + 2 * FIN + 1) * 8 + QUEUE * (int) sizeof(Unit) + (FIN + 1) * 4;
    static_assert(FIN * RED >= 8 * (MAX_E + 32) * 4, "scratch of the choice");
    __host__ __device__ static int frags(int d) { return mx4::chunks(d) * NT * mx4::FRAG; }
    __host__ __device__ static int tables(int slots) { return slots * 64 + MAX_E * 4 * 3 + MAX_T * MAX_K * 8; }
    __host__ __device__ static int bytes(int d, int slots, int ring, int depth) { return 128 + depth * DEEP + ring * HID + frags(d) + FIN * RED + tables(slots) + BARS; }
};

// 2^-n in fp16, twice (n below 0, from a byte that no hidden unit goes with, counts as 0)
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

template <int NT>
__global__ void __launch_bounds__(Layout<NT>::THREADS, 1) mx4_moe_kernel(const MoeArgs g) {
    using L = Layout<NT>;
    constexpr int FIN = L::FIN;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * ring = (uint8_t *) (((uintptr_t) smem_raw + 127) & ~(uintptr_t) 127);
    uint8_t * acts = ring + g.ring * L::HID, * weights = (uint8_t *) (((uintptr_t) smem_raw + L::bytes(g.d, g.max_slots, g.ring, 0) - 1) & ~(uintptr_t) 15);
    float * red = (float *) (acts + L::frags(g.d));
    float * wtab = red + FIN * L::RED / 4;                         // [slot][16] weight of each token, 0: not chosen
    int * slot_of = (int *) (wtab + g.max_slots * 16), * expert_of = slot_of + MAX_E, * mask = expert_of + MAX_E;
    int * ids_s = mask + MAX_E;
    float * wts_s = (float *) (ids_s + MAX_T * MAX_K);
    float * sel = red, * gscore = red + 8 * MAX_E;                 // the choice's scratch, before the first sums
    uint64_t * hid_full = (uint64_t *) (wts_s + MAX_T * MAX_K), * hid_empty = hid_full + L::MAX_RING;
    uint64_t * drawn = hid_empty + L::MAX_RING, * worked = drawn + L::QUEUE, * red_full = worked + L::QUEUE, * red_empty = red_full + FIN;
    uint64_t * acts_full = red_empty + FIN;
    Unit * queue = (Unit *) (acts_full + 1);
    int * red_unit = (int *) (queue + L::QUEUE), * n_slots_s = red_unit + FIN;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = g.ring;

    if (threadIdx.x == 0) {
        for (int i = 0; i < R; ++i) { mbar_init(&hid_full[i], 1); mbar_init(&hid_empty[i], NW); }
        for (int i = 0; i < L::QUEUE; ++i) { mbar_init(&drawn[i], 1); mbar_init(&worked[i], NW + 1); }
        mbar_init(acts_full, 1);
        for (int i = 0; i < FIN; ++i) { mbar_init(&red_full[i], NW); mbar_init(&red_empty[i], 1); }
        fence_barrier_init();
    }
    for (int i = threadIdx.x; i < g.max_slots * 16; i += L::THREADS) wtab[i] = 0.f;
    for (int i = threadIdx.x; i < MAX_E; i += L::THREADS) { slot_of[i] = 0; mask[i] = 0; }
    __syncthreads();
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    int first_unit = 0;
    if (threadIdx.x == NW * 32) {          // the drawing thread: its first unit, the tokens' fragments
        first_unit = atomicAdd(g.sync, 1);
        mbar_expect_tx(acts_full, L::frags(g.d));
        mx4::bulk_load(acts, g.xf, L::frags(g.d), acts_full);
    }

    // ---- which experts, for which tokens, with which weights ----
    const int kk = g.k + g.n_shared;
    if (g.logits != nullptr) {
        const int E = g.E - g.n_shared;
        if (warp < 8)
            for (int t = warp; t < g.T; t += 8)
                gate_token(g.logits + (size_t) t * E, g.bias, nullptr, nullptr, t, E, g.k, g.n_group, g.topk_group, g.scale, g.norm, g.sigmoid, g.n_shared,
                           g.group_top2, sel + warp * MAX_E, gscore + warp * 32, ids_s, wts_s);
    } else {
        for (int i = threadIdx.x; i < g.T * kk; i += L::THREADS) { ids_s[i] = g.ids[i]; wts_s[i] = g.wts[i]; }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < g.T * kk; i += L::THREADS)
        if ((unsigned) ids_s[i] < (unsigned) g.E) slot_of[ids_s[i]] = 1;
    __syncthreads();
    if (warp == 0) {
        int n = 0;
        for (int e = lane; e < MAX_E; e += 32) {
            const bool hit = slot_of[e] != 0;
            const unsigned m = __ballot_sync(0xffffffffu, hit);
            const int s = n + __popc(m & ((1u << lane) - 1));
            slot_of[e] = s;
            if (hit) expert_of[s] = e;
            n += __popc(m);
        }
        if (lane == 0) *n_slots_s = n;
        __syncwarp();
        if (lane < g.T)
            for (int j = 0; j < kk; ++j) {
                const int e = ids_s[lane * kk + j];
                if ((unsigned) e >= (unsigned) g.E) continue;
                wtab[slot_of[e] * 16 + lane] += wts_s[lane * kk + j];
                atomicOr(&mask[slot_of[e]], 1 << lane);
            }
    }
    __syncthreads();
    const int slots = *n_slots_s, C1 = mx4::chunks(g.d), C2 = mx4::chunks(g.F), UPE = g.F / 32, RB2 = g.d / 16, UPS = (g.d + 63) / 64;
    const int P = slots * C2, shares = min(g.shares, max(1, (P + NP - 1) / NP));      // a share is a stage at least
    const int U1 = slots * UPE, U = U1 + UPS * shares;
    int * done = g.sync + 4, * h_top = done + MAX_E, * shares_done = h_top + g.max_slots * 16;

    if (warp == NW) {
        // ---- units ----
        if (lane == 0)
#pragma unroll 1
            for (int i = 0;; ++i) {
                const int q = i % L::QUEUE, id = i == 0 ? first_unit : atomicAdd(g.sync, 1);
                if (!mx4::wait(&worked[q], (i / L::QUEUE & 1) ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 51, i); break; }
                Unit & u = queue[q];
                u.id = id < U ? id : -1;
                if (id < U1) {
                    u.n = C1;
                    u.slot = u.col = 0;
                    u.weights = g.gu + (size_t) expert_of[id / UPE] * g.gu_stride + (size_t) (id % UPE) * 4 * C1 * mx4::CHUNK;
                } else if (id < U) {
                    const int share = (id - U1) % shares, lo = share * P / shares;
                    u.n = (share + 1) * P / shares - lo;
                    u.slot = lo / C2;
                    u.col = lo % C2;
                    u.weights = g.down + (size_t) ((id - U1) / shares) * 4 * C2 * mx4::CHUNK;
                }
                mbar_arrive(&drawn[q]);
                if (id >= U) break;
            }
        __syncwarp();
        return;
    }

    if (warp == NW + 1) {
        // ---- hidden units ----
        int st = 0;                          // stages of down
        bool ok = true;
#pragma unroll 1
        for (int i = 0; ok; ++i) {
            ok = mx4::wait_all(&drawn[i % L::QUEUE], i / L::QUEUE & 1);
            if (!ok) break;
            const Unit u = queue[i % L::QUEUE];
            if (u.id < 0) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(&worked[i % L::QUEUE]);
            if (u.id < U1) continue;
            const int rb = (u.id - U1) / shares * 4, row_bytes = min(4, RB2 - rb) * 64;
            int slot = u.slot, c = u.col + lane;             // of this lane's place
#pragma unroll 1
            for (int p0 = 0; p0 < u.n; p0 += NP, c += NP, ++st) {
                const int s = st % R, n = min(NP, u.n - p0);
                while (c >= C2) { c -= C2; ++slot; }
                ok = mx4::wait_all(&hid_empty[s], (st / R & 1) ^ 1);
                const uint64_t t0 = globaltimer_ns();
#pragma unroll 1
                for (bool there = lane >= n; ok;) {
                    if (!there) there = ld_acquire(done + slot) >= UPE;
                    if (__all_sync(0xffffffffu, there)) break;
                    ok = __all_sync(0xffffffffu, globaltimer_ns() - t0 <= WAIT_NS);
                    __nanosleep(20);
                }
                if (!ok) break;
                asm volatile("fence.proxy.async.global;" ::: "memory");      // stored by ordinary stores, read by copies
                if (lane == 0) mbar_expect_tx(&hid_full[s], n * (NT * (mx4::FRAG + 64) + row_bytes + 64));
                __syncwarp();
                if (lane < n) {
                    uint8_t * hid = ring + s * L::HID;
                    const size_t tile = (size_t) (slot * C2 + c) * NT;
                    mx4::bulk_load(hid + lane * NT * mx4::FRAG, (const uint8_t *) g.h + tile * mx4::FRAG, NT * mx4::FRAG, &hid_full[s]);
                    mx4::bulk_load(hid + L::H_EXP + lane * NT * 64, g.h_exp + tile * 64, NT * 64, &hid_full[s]);
                    mx4::bulk_load(hid + L::H_ROW + lane * 256, g.down_exp + ((size_t) expert_of[slot] * RB2 + rb) * 16, row_bytes, &hid_full[s]);
                    mx4::bulk_load(hid + L::H_TOP + lane * 64, h_top + slot * 16, 64, &hid_full[s]);
                }
                __syncwarp();
            }
        }
        if (!ok) {
            if (lane == 0) jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 52, st);
            // copies in flight end before the memory is given back
            for (int i = st - R < 0 ? 0 : st - R; i < st; ++i) mx4::wait(&hid_full[i % R], i / R & 1);
        }
        return;
    }

    if (warp < NW) {
        // ---- products ----
        float acc[2][NT][4];                 // gate and up, or two row blocks of the weighted sum
        const int pair = warp / NP, g4 = lane >> 2, t2 = 2 * (lane & 3);
        // Two walks over the same stages, places p0 .. p0 + n - 1 of a unit, of which this warp has p0 + j if j < n: one asks for weights, up to
        // `depth` stages ahead of the other, which multiplies.  Places go around the warps, wherever units end.
        const uint64_t policy = l2_policy_evict_first();
        const int depth = g.depth;
        const uint8_t * mine = weights + warp * depth * (2 * mx4::CHUNK);
        Unit u;                                                   // the asking walk's unit, its place and the place in the ring
        int u_i = -1, u_p0 = 0, u_turn = 0, at_ask = 0, ahead = 0;
        u.id = u.n = 0;
        int id = 0, n_places = 0, slot0 = 0, col0 = 0, now_i = -1, p0 = 0, turn = 0, at_now = 0, sums = 0, st = 0;
        bool ok = mx4::wait_all(acts_full, 0);
#pragma unroll 1
        while (ok) {
            // ask, as far as units are known (with nothing on its way: wait for one)
#pragma unroll 1
            while (ahead < depth && u.id >= 0) {
                u_p0 += NP;
                if (u_i < 0 || u_p0 >= u.n) {
                    const int q = (u_i + 1) % L::QUEUE, ph = (u_i + 1) / L::QUEUE & 1;
                    if (ahead > 0 && !__all_sync(0xffffffffu, mbar_test_wait(&drawn[q], ph))) {
                        u_p0 -= NP;
                        break;
                    }
                    ok = mx4::wait_all(&drawn[q], ph);
                    if (!ok) break;
                    ++u_i;
                    u = queue[q];
                    u_p0 = 0;
                }
                const int j = (warp - u_turn) & (NP - 1), n = min(NP, u.n - u_p0);
                if (u.id >= 0) {
                    u_turn += n;
                    if (j < n) {
                        const bool down = u.id >= U1;
                        int slot = u.slot, c = u.col + u_p0 + j;
                        const uint8_t * at = u.weights;
                        if (down) {
                            while (c >= C2) { c -= C2; ++slot; }
                            at += (size_t) expert_of[slot] * g.down_stride;
                        }
                        const size_t apart = (size_t) (down ? C2 : C1) * mx4::CHUNK;
                        if (!down || (u.id - U1) / shares * 4 + 2 * pair < RB2) at += 2 * pair * apart;      // (two row blocks behind the last: any)
                        mx4::copy_chunks(smem_u32(mine) + at_ask * (2 * mx4::CHUNK), at + c * mx4::CHUNK, apart, policy);
                    }
                }
                mx4::copies_commit();
                at_ask = at_ask + 1 == depth ? 0 : at_ask + 1;
                ++ahead;
            }
            if (!ok) break;
            // the stage to multiply
            p0 += NP;
            if (now_i < 0 || p0 >= n_places) {
                ++now_i;
                const Unit & v = queue[now_i % L::QUEUE];           // (the asking walk has seen that it is there)
                id = v.id;
                n_places = v.n;
                slot0 = v.slot;
                col0 = v.col;
                p0 = 0;
                if (id < 0) break;
                __syncwarp();
                if (lane == 0) mbar_arrive(&worked[now_i % L::QUEUE]);
            }
            const bool down = id >= U1, first = p0 == 0, last = p0 + NP >= n_places;
            const int n_now = min(NP, n_places - p0), j_now = (warp - turn) & (NP - 1);
            turn += n_now;
            // its weights are here when at most those asked for behind them are not
            if (ahead == 1) mx4::copies_wait<0>();
            else if (ahead == 2) mx4::copies_wait<1>();
            else if (ahead == 3) mx4::copies_wait<2>();
            else mx4::copies_wait<3>();
            __syncwarp();
            const uint8_t * chunks = mine + at_now * (2 * mx4::CHUNK);
            if (first) {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int t = 0; t < NT; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[m][t][i] = 0.f;
            }
            if (!down) {
                if (j_now < n_now) {
                    const uint4 * b = (const uint4 *) acts + (p0 + j_now) * NT * 128 + lane;
                    float y[2][NT][4];
                    mx4::chunks_mma<NT>(chunks, y, [&](int t, int p) { return b[(t * 4 + p) * 32]; });
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int t = 0; t < NT; ++t)
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[m][t][i] += y[m][t][i];
                }
            } else if (n_now > 0) {
                const int s = st % R;
                ok = mx4::wait_all(&hid_full[s], st / R & 1);
                ++st;
                if (!ok) break;
                if (j_now < n_now) {
                    const uint8_t * hid = ring + s * L::HID;
                    int slot = slot0, c = col0 + p0 + j_now;
                    while (c >= C2) { c -= C2; ++slot; }
                    const uint4 * b = (const uint4 *) hid + j_now * NT * 128 + lane;
                    const int * tops = (const int *) (hid + L::H_TOP) + j_now * 16, * rows = (const int *) (hid + L::H_ROW) + j_now * 64 + pair * 32 + g4;
                    uint2 ex[NT];
                    int top[NT];
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        ex[t] = ((const uint2 *) (hid + L::H_EXP))[(j_now * NT + t) * 8 + g4];
                        top[t] = tops[t * 8 + g4];
                    }
                    float y[2][NT][4];
                    mx4::chunks_mma<NT>(chunks, y, [&](int t, int p) {
                        // all hidden units of a token to the same power of two: its largest one's
                        uint4 v = make_uint4(0u, 0u, 0u, 0u);
                        if (c * mx4::COLS + p * 32 < g.F) {
                            v = b[(t * 4 + p) * 32];
                            const uint32_t two = (p < 2 ? ex[t].x : ex[t].y) >> (16 * (p & 1));
                            const uint32_t f0 = below(top[t] - (int) (two & 0xff)), f1 = below(top[t] - (int) (two >> 8 & 0xff));
                            v.x = mx4::mul2(v.x, f0);
                            v.y = mx4::mul2(v.y, f0);
                            v.z = mx4::mul2(v.z, f1);
                            v.w = mx4::mul2(v.w, f1);
                        }
                        return v;
                    });
                    int re[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) re[i] = rows[8 * i] - BIAS - 14;
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        const float2 wt = *(const float2 *) (wtab + slot * 16 + t * 8 + t2);
                        const int2 te = *(const int2 *) (tops + t * 8 + t2);
                        const int chosen = mask[slot] >> (t * 8 + t2);
#pragma unroll
                        for (int m = 0; m < 2; ++m)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (chosen >> (i & 1) & 1)                // else there are no hidden units
                                    acc[m][t][i] += (i & 1 ? wt.y : wt.x) * mx4::pow2_normal(re[2 * m + (i >> 1)] + (i & 1 ? te.y : te.x)) * y[m][t][i];
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&hid_empty[s]);
            }
            __syncwarp();
            at_now = at_now + 1 == depth ? 0 : at_now + 1;
            --ahead;
            if (last) {
                const int buf = sums % FIN;
                ok = mx4::wait_all(&red_empty[buf], (sums / FIN & 1) ^ 1);
                if (!ok) break;
                float4 * dst = (float4 *) red + (buf * NW + warp) * (L::SUMS / 4) * 32 + lane;
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int t = 0; t < NT; ++t) dst[(m * NT + t) * 32] = make_float4(acc[m][t][0], acc[m][t][1], acc[m][t][2], acc[m][t][3]);
                if (warp == 0 && lane == 0) red_unit[buf] = id;
                __syncwarp();
                if (lane == 0) mbar_arrive(&red_full[buf]);
                ++sums;
            }
        }
        mx4::copies_wait<0>();
        if (!ok && lane == 0) jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 53, warp);
        // the end, for every finishing warp
#pragma unroll 1
        for (int i = 0; i < FIN; ++i, ++sums) {
            const int buf = sums % FIN;
            mx4::wait(&red_empty[buf], (sums / FIN & 1) ^ 1);
            if (warp == 0 && lane == 0) red_unit[buf] = -1;
            __syncwarp();
            if (lane == 0) mbar_arrive(&red_full[buf]);
        }
        return;
    }

    // ---- finished rows: a warp a unit; a lane holds row g of columns 2t, 2t + 1 and row g + 8 of the same ----
    constexpr int AT_ONCE = NT == 1 ? 3 : 1;                 // shares
    const int fin = warp - NW - 2, row0 = lane >> 2, col0 = 2 * (lane & 3);
    int x_exp[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int p = 0; p < 2; ++p) x_exp[n][p] = ((const int *) ((const uint8_t *) g.xf + L::frags(g.d)))[n * 8 + col0 + p];
#pragma unroll 1
    for (int round = 0;; ++round) {
        if (!mx4::wait_all(&red_full[fin], round & 1)) {
            if (lane == 0) jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 54, round);
            break;
        }
        const int unit = red_unit[fin];
        if (unit < 0) break;
        int ex[4][2];                        // exponents of this lane's rows of gate and up
        const int slot = unit < U1 ? unit / UPE : 0;
        if (unit < U1) {
            const int * rows = g.gu_exp + ((size_t) expert_of[slot] * UPE + unit % UPE) * 64 + row0;
#pragma unroll
            for (int i = 0; i < 8; ++i) ex[i >> 1][i & 1] = __ldg(rows + 8 * i);
        }
        float s[4][NT][4];
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 4; ++i) s[m][n][i] = 0.f;
#pragma unroll
                for (int w = 0; w < NP; ++w) {
                    const float4 v = ((const float4 *) red)[((fin * NW + (m >> 1) * NP + w) * (L::SUMS / 4) + (m & 1) * NT + n) * 32 + lane];
                    s[m][n][0] += v.x;
                    s[m][n][1] += v.y;
                    s[m][n][2] += v.z;
                    s[m][n][3] += v.w;
                }
            }
        __syncwarp();
        if (lane == 0) mbar_arrive(&red_empty[fin]);
        if (unit < U1) {
            const int f0 = unit % UPE * 32, m = mask[slot];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const size_t tile = ((size_t) slot * C2 + f0 / mx4::COLS) * NT + n;
#pragma unroll 1
                for (int st = 0; st < 2; ++st) {             // 16 hidden units each
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        v[i] = mx4::gated(mx4::times_pow2(s[2 * st][n][i], ex[2 * st][i >> 1] + x_exp[n][i & 1]),
                                          mx4::times_pow2(s[2 * st + 1][n][i], ex[2 * st + 1][i >> 1] + x_exp[n][i & 1]), g.act);
#pragma unroll
                    for (int p = 0; p < 2; ++p) {
                        // those of token 8 n + col, scaled together
                        const int col = col0 + p;
                        uint32_t top = max(__float_as_uint(v[p]) & 0x7fffffffu, __float_as_uint(v[p + 2]) & 0x7fffffffu);
#pragma unroll
                        for (int o = 4; o < 32; o *= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
                        if (m >> (n * 8 + col) & 1) {
                            const int he = mx4::top_exponent(top);
                            const float up = mx4::pow2(14 - he);
                            // hidden unit f0 + 16 st + row in its place among the fragments
                            __half * to = g.h + ((tile * 4 + f0 % mx4::COLS / 32) * 32 + col * 4 + row0 / 2) * 8 + st * 4 + (row0 & 1);
                            to[0] = __float2half_rn(v[p] * up);
                            to[2] = __float2half_rn(v[p + 2] * up);
                            if (row0 == 0) {
                                g.h_exp[(tile * 8 + col) * 8 + f0 % mx4::COLS / 16 + st] = (uint8_t) (he + BIAS);
                                atomicMax(h_top + slot * 16 + n * 8 + col, he + BIAS);
                            }
                        }
                    }
                }
            }
            __threadfence();
            __syncwarp();
            if (lane == 0) atomicAdd(done + slot, 1);
            continue;
        }
        const int rb = (unit - U1) / shares, share = (unit - U1) % shares;
        if (shares > 1) {
            float4 * part = (float4 *) g.part + (size_t) rb * shares * (4 * NT * 32) + lane;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
                    __stcg(part + ((share * 4 + m) * NT + n) * 32, make_float4(s[m][n][0], s[m][n][1], s[m][n][2], s[m][n][3]));
            __threadfence();
            __syncwarp();
            int others = 0;
            if (lane == 0) {
                others = atomicAdd(shares_done + rb, 1);
                __threadfence();
            }
            if (__shfl_sync(0xffffffffu, others, 0) != shares - 1) continue;
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) s[m][n][i] = 0.f;
#pragma unroll 1
            for (int i0 = 0; i0 < shares; i0 += AT_ONCE) {
                float4 v[AT_ONCE][4 * NT];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                    for (int k = 0; k < 4 * NT; ++k)
                        v[i][k] = i0 + i < shares ? __ldcg(part + ((i0 + i) * 4 * NT + k) * 32) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                    for (int k = 0; k < 4 * NT; ++k) {
                        s[k / NT][k % NT][0] += v[i][k].x;
                        s[k / NT][k % NT][1] += v[i][k].y;
                        s[k / NT][k % NT][2] += v[i][k].z;
                        s[k / NT][k % NT][3] += v[i][k].w;
                    }
            }
        }
        if (g.residual != nullptr)           // (all read before the first result is stored)
#pragma unroll
            for (int m = 0; m < 4; ++m)
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int t = n * 8 + col0 + (i & 1), o = rb * 64 + m * 16 + row0 + 8 * (i >> 1);
                        if (t < g.T && o < g.d) s[m][n][i] += __bfloat162float(g.residual[t * g.ldr + o]);
                    }
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int t = n * 8 + col0 + (i & 1), o = rb * 64 + m * 16 + row0 + 8 * (i >> 1);
                    if (t < g.T && o < g.d) g.out[(size_t) t * g.d + o] = __float2bfloat16(s[m][n][i]);
                }
    }
}

// The layer's first launch: CTAs below E compute router outputs [T][E], the others a token's fragments each (8 NT of them, zeros from T on); zeros where
// the next launch counts.
__global__ void __launch_bounds__(GATE_NT) mx4_prepare_kernel(const bf16 * __restrict__ x, long long ldx, const float * __restrict__ w_router,
                                                              float * __restrict__ logits, uint4 * __restrict__ xf, int * __restrict__ sync, int n_sync, int T,
                                                              int d, int E, int NT, int warm) {
    __shared__ float red[GATE_NT / 32][GATE_TG];
    const bool router = (int) blockIdx.x < E;
    PDL_TRIGGER_TOP();
    if (warm && router) router_rows(x, w_router, nullptr, 0.f, nullptr, logits, 0, min(T, GATE_TG), T, d, E, blockIdx.x, red, nullptr, true);
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
    if (threadIdx.x == 0) ((int *) (xf + (size_t) C * NT * 128))[n] = ex - 14;
    for (int i = threadIdx.x; i < C * 16; i += GATE_NT) {          // chunk, pair of steps, quarter of a step
        const int t = i & 3, pair = i >> 2 & 3, c = i >> 4;
        uint2 a = make_uint2(0u, 0u), b = a;
        if (n < T) {
            a = mx4::frag_step(row, c * 8 + pair * 2, t, d, unit);
            b = mx4::frag_step(row, c * 8 + pair * 2 + 1, t, d, unit);
        }
        xf[((c * NT + (n >> 3)) * 4 + pair) * 32 + (n & 7) * 4 + t] = make_uint4(a.x, a.y, b.x, b.y);
    }
}

template <int NT>
int launch(const MoeArgs & a, cudaStream_t s) {
    using L = Layout<NT>;
    static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
    MoeArgs g = a;
    g.ring = 2;
    g.depth = (MOST_SMEM - L::bytes(g.d, g.max_slots, g.ring, 0)) / L::DEEP;
    if (g.depth > L::MAX_DEPTH) {
        g.depth = L::MAX_DEPTH;
        if (L::bytes(g.d, g.max_slots, 3, g.depth) <= MOST_SMEM) g.ring = 3;
    }
    if (g.depth < 1) return JIB_E_SCRATCH;
    if (!jib::ensure_dyn_smem(mx4_moe_kernel<NT>, MOST_SMEM, attr_done)) return JIB_E_LAUNCH;
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148;
    JIB_LAUNCH((mx4_moe_kernel<NT>), sms, L::THREADS, L::bytes(g.d, g.max_slots, g.ring, g.depth), s, g);
    return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH;
}

// Shares that 64 rows of down are cut into at most: two, three or four units for each SM, whichever leaves the last round fullest.
int shares_of(int d) {
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148, groups = (d + 63) / 64;
    int best = 1;
    double fill = 0;
    for (int k = 2; k <= 4; ++k) {
        int n = k * sms / groups;
        n = n < 1 ? 1 : n > MAX_SHARES ? MAX_SHARES : n;
        const int rounds = (groups * n + sms - 1) / sms;
        const double f = (double) groups * n / ((double) rounds * sms);
        if (f > fill + 0.02) { fill = f; best = n; }
    }
    return best;
}

// Experts that T tokens can choose.
int slots_of(int T, int k, int E) { return T * k < E ? T * k : E; }

}  // namespace

extern "C" {

// Whether the two-launch form takes a layer (else 0), and the sizes of its buffers: bytes of xf and of h, floats of part, ints of sync.
JIB_EXPORT int jib_mx4_moe_sizes(int T, int d, int F, int E, int k, long long * sizes) {
    if (T < 1 || T > MAX_T || k < 1 || k > MAX_K || E < 1 || E > MAX_E || d % 32 || F % 32 || d < 32 || F < 32 || d > GATE_MAXC * GATE_NT * 8) return 0;
    const int NT = T <= 8 ? 1 : 2;
    const long long slots = slots_of(T, k, E);
    if ((NT == 1 ? Layout<1>::bytes(d, (int) slots, 2, 1) : Layout<2>::bytes(d, (int) slots, 2, 1)) > MOST_SMEM) return 0;
    const long long tiles = slots * mx4::chunks(F) * NT;
    if (slots * (F / 32) + (long long) (d / 32) * MAX_SHARES > (1ll << 30) || tiles > (1 << 25)) return 0;
    sizes[0] = (NT == 1 ? Layout<1>::frags(d) : Layout<2>::frags(d)) + 64;
    sizes[1] = tiles * (mx4::FRAG + 64);
    sizes[2] = (long long) ((d + 63) / 64) * shares_of(d) * 512 * NT;
    sizes[3] = 4 + MAX_E + slots * 16 + (d + 63) / 64;
    return 1;
}

// The layer's first launch: x as the second one reads it, zeros in sync, and with w_router [E][d] the router's outputs [T][E].
JIB_EXPORT int jib_mx4_moe_prepare(const void * x, long long ldx, const float * w_router, float * logits, void * xf, int * sync, int n_sync, int T, int d, int E,
                                   void * stream) {
    if (w_router == nullptr) E = 0;
    if (T < 1 || T > MAX_T || E < 0 || E > MAX_E || d % 32 || d > GATE_MAXC * GATE_NT * 8 || (E > 0 && ldx != d)) return JIB_E_ARG;
    if (((uintptr_t) x | (uintptr_t) (ldx * 2) | (uintptr_t) xf) & 15) return JIB_E_ALIGN;
    const int NT = T <= 8 ? 1 : 2;
    JIB_LAUNCH((mx4_prepare_kernel), E + 8 * NT, GATE_NT, 0, (cudaStream_t) stream, (const bf16 *) x, ldx, w_router, logits, (uint4 *) xf, sync, n_sync, T, d, E, NT,
               jib::warm_for(T));
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
    if (((uintptr_t) m->gu | (uintptr_t) m->down | (uintptr_t) m->gu_stride | (uintptr_t) m->down_stride | (uintptr_t) m->h | (uintptr_t) m->xf | (uintptr_t) m->part | (uintptr_t) m->sync | (uintptr_t) m->down_exp) & 15)
        return JIB_E_ALIGN;
    MoeArgs a;
    a.xf = (const uint4 *) m->xf; a.residual = (const bf16 *) m->residual; a.logits = m->logits; a.bias = m->bias; a.ids = m->ids; a.wts = m->wts;
    a.gu = (const uint8_t *) m->gu; a.down = (const uint8_t *) m->down; a.gu_exp = m->gu_exp; a.down_exp = m->down_exp;
    a.max_slots = slots_of(m->T, m->k + m->n_shared, m->E);
    a.h = (__half *) m->h; a.h_exp = (uint8_t *) m->h + (long long) a.max_slots * mx4::chunks(m->F) * (m->T <= 8 ? 1 : 2) * mx4::FRAG; a.part = m->part; a.out = (bf16 *) m->out; a.sync = m->sync; a.status = m->status;
    a.ldr = m->ldr; a.gu_stride = m->gu_stride; a.down_stride = m->down_stride;
    a.T = m->T; a.d = m->d; a.F = m->F; a.E = m->E; a.k = m->k; a.n_group = m->n_group; a.topk_group = m->topk_group; a.norm = m->norm; a.sigmoid = m->sigmoid;
    a.n_shared = m->n_shared; a.group_top2 = m->group_top2; a.act = m->act; a.scale = m->scale;
    a.shares = shares_of(m->d);
    return m->T <= 8 ? launch<1>(a, (cudaStream_t) stream) : launch<2>(a, (cudaStream_t) stream);
}

}  // extern "C"
