// A mixture-of-experts layer over packed 4-bit experts for up to 16 tokens, in two launches: the router's outputs, then everything else --
// choice of experts, gate and up products, activation, down products, weighted sum, residual.
//
// The reference runs router, choice, sorting, grouped products and the weighted sum as some dozen launches
// (src/llama-graph-ffn.cpp:145-260); the bf16 path here takes five.
//
// The layer is bound by the stream of the chosen experts' weights, so the second launch is one stream: every CTA draws units from a counter,
// first rows of gate and up (16 hidden units of one expert), then rows of down (16 outputs over a share of the experts), and one thread
// keeps a ring of stages filled with what the units read, across units and ahead of the sums.  A unit of the second kind waits until the
// hidden units it reads are stored: an expert's counter says how many of its gate and up units are done.  Units are drawn in order and a CTA
// works them off in order, those of the first kind never wait, so whatever a unit waits for is being worked on: the launch ends
// however few of its CTAs run at a time.
// Roles: NW warps multiply (a chunk of 16 rows x 128 columns each, mx4_stream.cuh), one thread copies, four warps add the NW sums up in warp
// order and finish the rows.  Sums of shares of experts meet in memory, the share that comes last adds them up in their order.
#include "gate.cuh"
#include "jib_kernels.h"
#include "mx4_stream.cuh"
#include "pdl.cuh"

namespace {

using namespace sm100;

constexpr int MAX_T = 16, MAX_K = 32, SPC = 16;               // tokens, choices of a token, chunks of a stage
constexpr int STAGE = SPC * mx4::CHUNK;
constexpr int MAX_SHARES = 8;
constexpr int FIN = 4;                                        // finishing warps

struct MoeArgs {
    const bf16 * x, * residual;              // residual may be NULL
    const float * logits, * bias;            // logits NULL: ids and weights are given
    const int * ids;
    const float * wts;
    const uint8_t * gu, * down;
    const float * gu_scale, * gu_scale2, * down_scale;
    bf16 * h;                                // [slot][chunks of F][NT] fragments
    float * part;                            // [d / 16][shares][128 NT]
    bf16 * out;
    int * sync;                              // zeros: next unit, done gate and up units of each slot [MAX_E], shares done of each row block
    int * status;
    long long ldx, ldr, gu_stride, down_stride;
    int T, d, F, E, k, n_group, topk_group, norm, sigmoid, n_shared, group_top2, act, shares, ring, limit_ms;
    float scale;
};

// A stage's contents, in shared memory beside it.
struct Header {
    int unit;                // -1: the end
    int p0, n;               // positions of the unit's stream: p0 .. p0 + n - 1
    int turn;                // chunks before this stage, modulo NW: chunk c belongs to warp (c + turn) mod NW
    int last;                // the unit ends here
    int pad[3];
};

template <int NT, int NW>
struct Layout {
    static constexpr int THREADS = (NW + 1 + FIN) * 32;
    static constexpr int RED = NW * 8 * NT * 32 * 4;              // one unit's sums of every warp
    static constexpr int TABLES = MAX_E * 16 * 4 + MAX_E * 4 * 3 + MAX_T * MAX_K * 8;
    static constexpr int MAX_RING = 12;
    static constexpr int BARS = MAX_RING * (3 * 8 + (int) sizeof(Header)) + 64;
    static_assert(2 * RED >= 8 * (MAX_E + 32) * 4, "scratch of the choice");
    __host__ __device__ static int frags(int d) { return mx4::chunks(d) * NT * mx4::FRAG; }
    __host__ __device__ static int bytes(int d, int ring) { return 128 + ring * STAGE + frags(d) + 2 * RED + TABLES + BARS; }
};

__device__ __forceinline__ int ld_acquire(const int * p) {
    int v;
    asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
    return v;
}

template <int NT, int NW>
__global__ void __launch_bounds__(Layout<NT, NW>::THREADS, 1) mx4_moe_kernel(const MoeArgs g) {
    using L = Layout<NT, NW>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t * ring = (uint8_t *) (((uintptr_t) smem_raw + 127) & ~(uintptr_t) 127);
    uint4 * xs = (uint4 *) (ring + g.ring * STAGE);
    float * red = (float *) ((uint8_t *) xs + L::frags(g.d));
    float * wtab = red + 2 * L::RED / 4;                           // [slot][16] weight of each token, 0: not chosen
    int * slot_of = (int *) (wtab + MAX_E * 16), * expert_of = slot_of + MAX_E, * mask = expert_of + MAX_E;
    int * ids_s = mask + MAX_E;
    float * wts_s = (float *) (ids_s + MAX_T * MAX_K);
    float * sel = red, * gscore = red + 8 * MAX_E;                // the choice's scratch, before the first sums
    uint64_t * full = (uint64_t *) (wts_s + MAX_T * MAX_K), * empty = full + L::MAX_RING, * meta = empty + L::MAX_RING;
    Header * hdr = (Header *) (meta + L::MAX_RING);
    uint64_t * red_full = (uint64_t *) (hdr + L::MAX_RING), * red_empty = red_full + 2;
    int * red_unit = (int *) (red_empty + 2), * n_slots_s = red_unit + 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, R = g.ring;

    if (threadIdx.x == 0) {
        for (int i = 0; i < R; ++i) { mbar_init(&full[i], 1); mbar_init(&empty[i], NW); mbar_init(&meta[i], 1); }
        for (int i = 0; i < 2; ++i) { mbar_init(&red_full[i], NW); mbar_init(&red_empty[i], FIN); }
        fence_barrier_init();
    }
    for (int i = threadIdx.x; i < MAX_E * 16; i += L::THREADS) wtab[i] = 0.f;
    for (int i = threadIdx.x; i < MAX_E; i += L::THREADS) { slot_of[i] = 0; mask[i] = 0; }
    PDL_TRIGGER_TOP();
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point

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
    const int slots = *n_slots_s, C1 = mx4::chunks(g.d), C2 = mx4::chunks(g.F), RB1 = g.F / 16, RB2 = g.d / 16;
    const int U1 = slots * RB1, U = U1 + RB2 * g.shares;
    int * done = g.sync + 1, * shares_done = done + MAX_E;

    if (warp == NW) {
        // ---- copies ----
        if (lane == 0) {
            const uint64_t policy = l2_policy_evict_first();
            int it = 0, turn = 0, unit = atomicAdd(g.sync, 1);
            bool ok = true;
            while (ok) {
                const bool end = unit >= U;
                int next = 0;
                int total = 0, lo = 0;
                const uint8_t * src = nullptr;
                if (!end) {
                    next = atomicAdd(g.sync, 1);           // on its way while this unit's copies are issued
                    if (unit < U1) {
                        total = 2 * C1;
                        src = g.gu + (size_t) expert_of[unit / RB1] * g.gu_stride + (size_t) (unit % RB1) * total * mx4::CHUNK;
                    } else {
                        const int share = (unit - U1) % g.shares;
                        lo = share * slots / g.shares;
                        total = ((share + 1) * slots / g.shares - lo) * C2;
                        src = g.down + (size_t) ((unit - U1) / g.shares) * C2 * mx4::CHUNK;
                    }
                }
                int p0 = 0;
                do {
                    const int s = it % R, n = min(SPC, total - p0);
                    if (!mbar_wait(&empty[s], (it / R & 1) ^ 1)) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 51, unit); ok = false; break; }
                    Header & q = hdr[s];
                    q.unit = end ? -1 : unit;
                    q.p0 = p0;
                    q.n = n;
                    q.turn = turn;
                    q.last = p0 + n >= total;
                    mbar_arrive(&meta[s]);
                    uint8_t * dst = ring + s * STAGE;
                    if (n > 0) {
                        mbar_expect_tx(&full[s], n * mx4::CHUNK);
                        if (unit < U1) mx4::bulk_load(dst, src + (size_t) p0 * mx4::CHUNK, n * mx4::CHUNK, &full[s], policy);
                        else
                            for (int p = p0; p < p0 + n;) {              // one copy for the chunks of one expert
                                const int c = p % C2, m = min(C2 - c, p0 + n - p);
                                mx4::bulk_load(dst + (p - p0) * mx4::CHUNK,
                                          src + (size_t) expert_of[lo + p / C2] * g.down_stride + (size_t) c * mx4::CHUNK, m * mx4::CHUNK, &full[s], policy);
                                p += m;
                            }
                    } else {
                        mbar_arrive(&full[s]);
                    }
                    ++it;
                    turn = (turn + n) % NW;
                    p0 += n;
                } while (p0 < total);
                if (end) break;
                unit = next;
            }
            // copies in flight end before the memory is given back
            if (!ok)
                for (int i = it - R < 0 ? 0 : it - R; i < it; ++i) mbar_wait(&full[i % R], i / R & 1);
        }
        __syncwarp();
        return;
    }

    // ---- the tokens as fragments ----
    for (int i = threadIdx.x < NW * 32 ? threadIdx.x : threadIdx.x - 32; i < C1 * NT * 128; i += (NW + FIN) * 32) {
        const int ln = i & 31, pair = i >> 5 & 3, nt = (i >> 7) % NT, c = (i >> 7) / NT, n = nt * 8 + (ln >> 2);
        xs[i] = n < g.T ? mx4::gather_frag(g.x + n * g.ldx, c, pair, ln & 3, g.d) : make_uint4(0u, 0u, 0u, 0u);
    }
    asm volatile("bar.sync 1, %0;" ::"n"((NW + FIN) * 32) : "memory");

    if (warp < NW) {
        // ---- products ----
        float acc[2][NT][4];                 // gate, up; or: [0] the weighted sum
        uint4 hb[NT][4];                     // the next chunk's hidden units, asked for ahead
        bool have = false, ok = true, first = true;
        int ready = 0, units = 0;            // hidden units of the slots below are stored
        // Hidden units of position p of the unit: false if they are not all stored yet and `block` is not set.
        auto fetch = [&](const Header & q, int p, bool block) -> bool {
            const int share = (q.unit - U1) % g.shares, slot = share * slots / g.shares + p / C2, c = p % C2;
            if (slot >= ready) {
                const uint64_t t0 = globaltimer_ns();
                for (int s = ready; s <= slot; ++s) {
                    bool seen = false;
                    do {
                        int v = 0;
                        if (lane == 0) v = ld_acquire(done + s);
                        seen = __shfl_sync(0xffffffffu, v, 0) >= RB1;
                        if (!seen && block) {
                            __nanosleep(40);
                            if (globaltimer_ns() - t0 > (uint64_t) g.limit_ms * 1000000ull) {
                                jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 52, s);
                                break;
                            }
                        }
                    } while (!seen && block);
                    if (!seen && !block) return false;
                }
                ready = slot + 1;
            }
            const uint4 * src = (const uint4 *) g.h + ((size_t) (slot * C2 + c) * NT) * 128 + lane;
            const int m = mask[slot];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int pair = 0; pair < 4; ++pair) {
                    const int k = c * mx4::COLS + pair * 32;
                    hb[n][pair] = make_uint4(0u, 0u, 0u, 0u);
                    if ((m >> (n * 8 + (lane >> 2)) & 1) && k < g.F) hb[n][pair] = __ldcg(src + n * 128 + pair * 32);
                }
            return true;
        };
        for (int it = 0; ok; ++it) {
            const int s = it % R;
            const uint32_t ph = it / R & 1;
            ok = __all_sync(0xffffffffu, mbar_wait(&meta[s], ph));
            if (!ok) break;
            const Header q = hdr[s];
            if (q.unit < 0) break;
            const bool down = q.unit >= U1;
            if (first) {
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[m][n][i] = 0.f;
            }
            int c = (warp - q.turn) & (NW - 1);
            if (down && c < q.n && !have) fetch(q, q.p0 + c, true);
            have = false;
            ok = __all_sync(0xffffffffu, mbar_wait(&full[s], ph));
            if (!ok) break;
            for (; c < q.n; c += NW) {
                const uint8_t * chunk = ring + s * STAGE + c * mx4::CHUNK;
                const int p = q.p0 + c;
                if (!down) {
                    uint4 b[NT][4];
                    const int kc = p < C1 ? p : p - C1;
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i) b[n][i] = xs[((kc * NT + n) * 4 + i) * 32 + lane];
                    if (p < C1) mx4::chunk_mma<NT>(chunk, b, acc[0]);
                    else mx4::chunk_mma<NT>(chunk, b, acc[1]);
                } else {
                    if (NW < SPC && c >= NW) fetch(q, p, true);
                    float y[NT][4] = {};
                    mx4::chunk_mma<NT>(chunk, hb, y);
                    const int slot = (q.unit - U1) % g.shares * slots / g.shares + p / C2;
                    const float ws = g.down_scale[expert_of[slot]];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        const float2 w = *(const float2 *) (wtab + slot * 16 + n * 8 + (lane & 3) * 2);
                        acc[0][n][0] += w.x * ws * y[n][0];
                        acc[0][n][1] += w.y * ws * y[n][1];
                        acc[0][n][2] += w.x * ws * y[n][2];
                        acc[0][n][3] += w.y * ws * y[n][3];
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&empty[s]);
            first = q.last != 0;
            if (q.last) {
                const int buf = units & 1;
                ok = __all_sync(0xffffffffu, mbar_wait(&red_empty[buf], (units >> 1 & 1) ^ 1));
                if (!ok) break;
                float * dst = red + buf * (L::RED / 4) + warp * 8 * NT * 32 + lane;
#pragma unroll
                for (int m = 0; m < 2; ++m)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (m == 0 || !down) dst[((m * NT + n) * 4 + i) * 32] = acc[m][n][i];
                if (warp == 0 && lane == 0) red_unit[buf] = q.unit;
                __syncwarp();
                if (lane == 0) mbar_arrive(&red_full[buf]);
                ++units;
            }
        }
        if (!ok) jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 53, warp);
        // the end, for the finishing warps
        const int buf = units & 1;
        mbar_wait(&red_empty[buf], (units >> 1 & 1) ^ 1);
        if (warp == 0 && lane == 0) red_unit[buf] = -1;
        __syncwarp();
        if (lane == 0) mbar_arrive(&red_full[buf]);
        return;
    }

    // ---- finished rows: thread = (register of the fragment, lane) ----
    const int fin = threadIdx.x - (NW + 1) * 32, reg = fin >> 5, row = (lane >> 2) + 8 * (reg >> 1), col = 2 * (lane & 3) + (reg & 1);
    for (int units = 0;; ++units) {
        const int buf = units & 1;
        if (!__all_sync(0xffffffffu, mbar_wait(&red_full[buf], units >> 1 & 1))) { jib_report(g.status, JIB_ERR_WAIT_TIMEOUT, 54, units); break; }
        const int unit = red_unit[buf];
        if (unit < 0) break;
        const float * src = red + buf * (L::RED / 4) + reg * 32 + lane;
        float s[2][NT];
#pragma unroll
        for (int m = 0; m < 2; ++m)
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s[m][n] = 0.f;
                if (m == 0 || unit < U1)
                    for (int w = 0; w < NW; ++w) s[m][n] += src[(w * 8 * NT + (m * NT + n) * 4) * 32];
            }
        __syncwarp();
        if (lane == 0) mbar_arrive(&red_empty[buf]);
        if (unit < U1) {
            const int slot = unit / RB1, f = unit % RB1 * 16, e = expert_of[slot];
            const float zs = g.gu_scale[e], us = g.gu_scale2[e];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                if (!(mask[slot] >> (n * 8 + col) & 1)) continue;
                // hidden unit f + row of token 8 n + col, in its place among the fragments
                const size_t at = ((((size_t) slot * C2 + f / mx4::COLS) * NT + n) * 4 + f % mx4::COLS / 32) * 32 + col * 4 + (row & 7) / 2;
                g.h[at * 8 + (f / 16 & 1) * 4 + (row >> 3) * 2 + (row & 1)] = __float2bfloat16(mx4::gated(s[0][n] * zs, s[1][n] * us, g.act));
            }
            __threadfence();
            asm volatile("bar.sync 2, %0;" ::"n"(FIN * 32) : "memory");
            if (fin == 0) atomicAdd(done + slot, 1);
            continue;
        }
        const int rb = (unit - U1) / g.shares, share = (unit - U1) % g.shares;
        if (g.shares > 1) {
            float * mine = g.part + ((size_t) rb * g.shares) * (128 * NT) + fin;
#pragma unroll
            for (int n = 0; n < NT; ++n) __stcg(mine + (share * NT + n) * 128, s[0][n]);
            __threadfence();
            asm volatile("bar.sync 2, %0;" ::"n"(FIN * 32) : "memory");
            if (fin == 0) {
                n_slots_s[1] = atomicAdd(shares_done + rb, 1);
                __threadfence();
            }
            asm volatile("bar.sync 2, %0;" ::"n"(FIN * 32) : "memory");
            const bool last = n_slots_s[1] == g.shares - 1;
            asm volatile("bar.sync 2, %0;" ::"n"(FIN * 32) : "memory");
            if (!last) continue;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                s[0][n] = 0.f;
                for (int i = 0; i < g.shares; ++i) s[0][n] += __ldcg(mine + (i * NT + n) * 128);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const int t = n * 8 + col, o = rb * 16 + row;
            if (t >= g.T) continue;
            float y = s[0][n];
            if (g.residual != nullptr) y += __bfloat162float(g.residual[t * g.ldr + o]);
            g.out[(size_t) t * g.d + o] = __float2bfloat16(y);
        }
    }
}

// Router outputs [T][E] of up to 16 tokens, and zeros where the next launch counts.
__global__ void __launch_bounds__(GATE_NT) mx4_router_kernel(const bf16 * __restrict__ x, const float * __restrict__ w_router, float * __restrict__ logits,
                                                             int * __restrict__ sync, int n_sync, int T, int d, int E, int warm) {
    __shared__ float red[GATE_NT / 32][GATE_TG];
    PDL_TRIGGER_TOP();
    if (warm) router_rows(x, w_router, nullptr, 0.f, nullptr, logits, 0, min(T, GATE_TG), T, d, E, blockIdx.x, red, nullptr, true);
    pdl_wait();      // inputs come from earlier kernels; nothing is written before this point
    for (int i = blockIdx.x * GATE_NT + threadIdx.x; i < n_sync; i += gridDim.x * GATE_NT) sync[i] = 0;
    router_rows(x, w_router, nullptr, 0.f, nullptr, logits, 0, T, T, d, E, blockIdx.x, red, nullptr);
}

template <int NT, int NW>
int launch(const MoeArgs & a, cudaStream_t s) {
    using L = Layout<NT, NW>;
    static std::atomic<unsigned char> attr_done[jib::MAX_DEVICES];
    constexpr int MOST = 227 * 1024;
    MoeArgs g = a;
    g.ring = (MOST - L::bytes(g.d, 0)) / STAGE;
    if (g.ring > L::MAX_RING) g.ring = L::MAX_RING;
    if (g.ring < 2) return JIB_E_SCRATCH;
    if (!jib::ensure_dyn_smem(mx4_moe_kernel<NT, NW>, MOST, attr_done)) return JIB_E_LAUNCH;
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148;
    JIB_LAUNCH((mx4_moe_kernel<NT, NW>), sms, L::THREADS, L::bytes(g.d, g.ring), s, g);
    return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH;
}

// Shares of the experts that a row block of down is cut into: eight units for each SM, so that the last round is short.
int shares_of(int d) {
    const int sms = jib::sm_count() > 0 ? jib::sm_count() : 148, n = (8 * sms + d / 16 - 1) / (d / 16);
    return n < 1 ? 1 : n > MAX_SHARES ? MAX_SHARES : n;
}

}  // namespace

extern "C" {

// Whether the one-launch form takes a layer, and the sizes of its buffers: bytes of h, floats of part, ints of sync.  0: it does not.
JIB_EXPORT int jib_mx4_moe_sizes(int T, int d, int F, int E, int k, long long * h_bytes, long long * part_floats, long long * sync_ints) {
    if (T < 1 || T > MAX_T || k < 1 || k > MAX_K || E < 1 || E > MAX_E || d % 32 || F % 32 || d < 32 || F < 32) return 0;
    const int NT = T <= 8 ? 1 : 2;
    if (NT == 1 ? Layout<1, 16>::bytes(d, 2) > 227 * 1024 : Layout<2, 8>::bytes(d, 2) > 227 * 1024) return 0;
    const long long slots = (long long) T * k < E ? (long long) T * k : E;
    if (slots * (F / 16) + (long long) (d / 16) * MAX_SHARES > (1ll << 30)) return 0;
    *h_bytes = slots * mx4::chunks(F) * NT * mx4::FRAG;
    *part_floats = (long long) (d / 16) * shares_of(d) * 128 * NT;
    *sync_ints = 1 + MAX_E + d / 16;
    return 1;
}

// The router's outputs of the layer's launch, and zeros in sync.
JIB_EXPORT int jib_mx4_moe_router(const void * x, const float * w_router, float * logits, int * sync, int n_sync, int T, int d, int E, void * stream) {
    if (T < 1 || T > MAX_T || E < 1 || E > MAX_E || d % 8 || d > GATE_MAXC * GATE_NT * 8) return JIB_E_ARG;
    JIB_LAUNCH((mx4_router_kernel), E, GATE_NT, 0, (cudaStream_t) stream, (const bf16 *) x, w_router, logits, sync, n_sync, T, d, E, jib::warm_for(T));
    return cudaGetLastError() == cudaSuccess ? 0 : JIB_E_LAUNCH;
}

// out = residual + sum over the choices of weight * down(act(gate) * up).  With logits the launch chooses the experts itself (the gate's arguments are
// those of jib_moe_gate; the last n_shared of the E experts take every token), else ids and wts [T][k] do (n_shared 0).
JIB_EXPORT int jib_mx4_moe(const jib_mx4_moe_desc * m, void * stream) {
    long long h, p, n;
    if (m->T <= 0) return 0;
    if (m->n_shared < 0 || m->k < 1 || !jib_mx4_moe_sizes(m->T, m->d, m->F, m->E, m->k + m->n_shared, &h, &p, &n)) return JIB_E_ARG;
    if (m->h_bytes < h || m->part_floats < p || m->sync_ints < n) return JIB_E_SCRATCH;
    if (m->logits == nullptr ? (m->ids == nullptr || m->wts == nullptr || m->n_shared != 0)
                             : (m->n_shared >= m->E || m->k > m->E - m->n_shared || m->n_group < 1 || m->n_group > 32 || (m->E - m->n_shared) % m->n_group))
        return JIB_E_ARG;
    if (((uintptr_t) m->gu | (uintptr_t) m->down | (uintptr_t) m->gu_stride | (uintptr_t) m->down_stride | (uintptr_t) m->h) & 15 || ((uintptr_t) m->x & 3) || m->ldx % 2)
        return JIB_E_ALIGN;
    MoeArgs a;
    a.x = (const bf16 *) m->x; a.residual = (const bf16 *) m->residual; a.logits = m->logits; a.bias = m->bias; a.ids = m->ids; a.wts = m->wts;
    a.gu = (const uint8_t *) m->gu; a.down = (const uint8_t *) m->down; a.gu_scale = m->gu_scale; a.gu_scale2 = m->gu_scale2; a.down_scale = m->down_scale;
    a.h = (bf16 *) m->h; a.part = m->part; a.out = (bf16 *) m->out; a.sync = m->sync; a.status = m->status;
    a.ldx = m->ldx; a.ldr = m->ldr; a.gu_stride = m->gu_stride; a.down_stride = m->down_stride;
    a.T = m->T; a.d = m->d; a.F = m->F; a.E = m->E; a.k = m->k; a.n_group = m->n_group; a.topk_group = m->topk_group; a.norm = m->norm; a.sigmoid = m->sigmoid;
    a.n_shared = m->n_shared; a.group_top2 = m->group_top2; a.act = m->act; a.scale = m->scale;
    a.shares = shares_of(m->d);
    a.limit_ms = 2000;
    return m->T <= 8 ? launch<1, 16>(a, (cudaStream_t) stream) : launch<2, 8>(a, (cudaStream_t) stream);
}

}  // extern "C"
