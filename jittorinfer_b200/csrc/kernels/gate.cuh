// Parts of the routing kernels that more than one file uses: router outputs of a few tokens, the gating of one token.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <float.h>
#include <stdint.h>

namespace {

typedef __nv_bfloat16 bf16;
constexpr int MAX_E = 256;

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Router logits in fp32: logits[t][e] = sum_i g[t][i] * w_router[e][i].
// One expert per CTA, 256 threads; thread i owns the 8-element chunks i, i + 256, ... of the d axis (its router row slice
// stays in registers), tokens are walked in groups of 8 so that every load of a group is independent -- the kernel is
// latency-bound, so memory-level parallelism is what matters.
//
// With norm_w the rows of x are first RMS-normalised: thread mapping, accumulation order and reduction tree are those of
// rmsnorm_kernel<256, *> (elementwise.cu), so the bf16 row the dot product sees -- and the row CTA (t mod gridDim.x)
// stores to g_out -- is bit for bit what that kernel would have produced.
constexpr int GATE_TG = 8;
constexpr int GATE_NT = 256;
constexpr int GATE_MAXC = 4;      // 8-element chunks per thread: d <= 4 * 256 * 8 = 8192

struct alignas(16) bf16x8 {
    __nv_bfloat162 v[4];
};

__device__ __noinline__ void router_rows(const bf16 * __restrict__ x, const float * __restrict__ w_router, const float * __restrict__ norm_w,
                                            float eps, bf16 * __restrict__ g_out, float * __restrict__ logits, int t_begin, int t_end,
                                            int T, int d, int E, int e, float (*red)[GATE_TG], float * inv_s, bool dry = false) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int nv = d / 8;
    float4 w[GATE_MAXC][2];
    float4 nw[GATE_MAXC][2];
#pragma unroll
    for (int c = 0; c < GATE_MAXC; ++c) {
        const int i = threadIdx.x + c * GATE_NT;
        const float4 z = make_float4(0.f, 0.f, 0.f, 0.f);
        w[c][0] = i < nv ? ((const float4 *) (w_router + (size_t) e * d))[2 * i] : z;
        w[c][1] = i < nv ? ((const float4 *) (w_router + (size_t) e * d))[2 * i + 1] : z;
        nw[c][0] = (norm_w != nullptr && i < nv) ? ((const float4 *) norm_w)[2 * i] : z;
        nw[c][1] = (norm_w != nullptr && i < nv) ? ((const float4 *) norm_w)[2 * i + 1] : z;
    }
    for (int t0 = t_begin; t0 < t_end; t0 += GATE_TG) {
        if (norm_w != nullptr) {
            // sum of squares per token, then 1 / rms: warp w finishes token t0 + w
            float ss[GATE_TG];
#pragma unroll
            for (int j = 0; j < GATE_TG; ++j) ss[j] = 0.f;
#pragma unroll
            for (int c = 0; c < GATE_MAXC; ++c) {
                const int i = threadIdx.x + c * GATE_NT;
                if (i < nv) {
#pragma unroll
                    for (int j = 0; j < GATE_TG; ++j) {
                        const int t = min(t0 + j, T - 1);
                        const bf16x8 a = ((const bf16x8 *) (x + (size_t) t * d))[i];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const float2 f = __bfloat1622float2(a.v[q]);
                            ss[j] += f.x * f.x + f.y * f.y;
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < GATE_TG; ++j) {
                const float s = warp_sum(ss[j]);
                if (lane == 0) red[warp][j] = s;
            }
            __syncthreads();
            {
                float t = lane < GATE_NT / 32 ? red[lane][warp] : 0.f;
                t = warp_sum(t);
                if (lane == 0) inv_s[warp] = rsqrtf(t / (float) d + eps);
            }
            __syncthreads();
        }
        float acc[GATE_TG];
#pragma unroll
        for (int j = 0; j < GATE_TG; ++j) acc[j] = 0.f;
#pragma unroll
        for (int c = 0; c < GATE_MAXC; ++c) {
            const int i = threadIdx.x + c * GATE_NT;
            if (i < nv) {
#pragma unroll
                for (int j = 0; j < GATE_TG; ++j) {
                    const int t = min(t0 + j, T - 1);
                    bf16x8 a = ((const bf16x8 *) (x + (size_t) t * d))[i];
                    if (norm_w != nullptr) {
                        const float inv = inv_s[j];
                        const float2 f0 = __bfloat1622float2(a.v[0]), f1 = __bfloat1622float2(a.v[1]);
                        const float2 f2 = __bfloat1622float2(a.v[2]), f3 = __bfloat1622float2(a.v[3]);
                        a.v[0] = __floats2bfloat162_rn(f0.x * inv * nw[c][0].x, f0.y * inv * nw[c][0].y);
                        a.v[1] = __floats2bfloat162_rn(f1.x * inv * nw[c][0].z, f1.y * inv * nw[c][0].w);
                        a.v[2] = __floats2bfloat162_rn(f2.x * inv * nw[c][1].x, f2.y * inv * nw[c][1].y);
                        a.v[3] = __floats2bfloat162_rn(f3.x * inv * nw[c][1].z, f3.y * inv * nw[c][1].w);
                        if (g_out != nullptr && !dry && t0 + j < t_end && (t0 + j) % (int) gridDim.x == (int) blockIdx.x)
                            ((bf16x8 *) (g_out + (size_t) (t0 + j) * d))[i] = a;
                    }
                    const float2 f0 = __bfloat1622float2(a.v[0]), f1 = __bfloat1622float2(a.v[1]);
                    const float2 f2 = __bfloat1622float2(a.v[2]), f3 = __bfloat1622float2(a.v[3]);
                    acc[j] += w[c][0].x * f0.x + w[c][0].y * f0.y + w[c][0].z * f1.x + w[c][0].w * f1.y +
                              w[c][1].x * f2.x + w[c][1].y * f2.y + w[c][1].z * f3.x + w[c][1].w * f3.y;
                }
            }
        }
#pragma unroll
        for (int j = 0; j < GATE_TG; ++j) {
            const float s = warp_sum(acc[j]);
            if (lane == 0) red[warp][j] = s;
        }
        __syncthreads();
        if (threadIdx.x < GATE_TG && t0 + threadIdx.x < t_end) {
            float s = 0.f;
#pragma unroll
            for (int q = 0; q < GATE_NT / 32; ++q) s += red[q][threadIdx.x];
            if (!dry) logits[(size_t) (t0 + threadIdx.x) * E + e] = s;
        }
        __syncthreads();
    }
}

// Gating of one token by one warp: softmax/sigmoid over the logits, optional group-limited masking, k rounds of arg-max.  A lane holds the
// experts lane, lane + 32, ... in registers; a round is two warp reductions of one instruction each (the largest value, then the lowest
// expert that has it) instead of ten exchanges and a walk through shared memory.
// sel: E floats and gscore: 32 floats, private to the warp, with groups only.  Not inlined: callers run it twice (a dry run, then the
// real one) and both calls must execute the same copy of the code.
constexpr int GATE_NI = MAX_E / 32;

__device__ __forceinline__ float warp_max(float v) {
    asm volatile("redux.sync.max.f32 %0, %0, 0xffffffff;" : "+f"(v));
    return v;
}

__device__ __noinline__ void gate_token(const float * __restrict__ logits_row, const float * __restrict__ bias, int * __restrict__ ids,
                                           float * __restrict__ wts, int t, int E, int k, int n_group, int topk_group, float scale,
                                           int norm, int sigmoid, int n_shared, int group_top2, float * sel,
                                           float * gscore, int * ids_copy = nullptr, float * wts_copy = nullptr, bool dry = false,
                                           const float * __restrict__ logit_bias = nullptr, int shared_gate = 0) {
    // dry: runs the same instructions on made-up logits and stores nothing to global memory -- a caller that is still waiting for its
    // inputs uses it to pull this code into the SM's instruction cache ahead of the real call
    const int lane = threadIdx.x & 31;
    const int ld = k + n_shared;
    float p[GATE_NI], v[GATE_NI];
    float mx = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < GATE_NI; ++i) {
        const int e = lane + 32 * i;
        p[i] = 0.f;
        if (32 * i < E && e < E) {              // possibly written by other CTAs: from L2
            p[i] = dry ? (float) ((e * 37 + t) & 63) : __ldcg(logits_row + e) + (logit_bias != nullptr ? logit_bias[e] : 0.f);
            mx = fmaxf(mx, p[i]);
        }
    }
    mx = warp_max(mx);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < GATE_NI; ++i)
        if (32 * i < E && lane + 32 * i < E) {
            p[i] = sigmoid ? 1.f / (1.f + expf(-p[i])) : expf(p[i] - mx);
            sum += p[i];
        }
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < GATE_NI; ++i) {
        const int e = lane + 32 * i;
        v[i] = -INFINITY;
        if (32 * i < E && e < E) {
            if (!sigmoid) p[i] = p[i] / sum;
            v[i] = p[i] + (bias && !dry ? bias[e] : 0.f);
        }
    }
    if (n_group > 1) {
#pragma unroll
        for (int i = 0; i < GATE_NI; ++i)
            if (32 * i < E && lane + 32 * i < E) sel[lane + 32 * i] = v[i];
        __syncwarp();
        const int gs = E / n_group;
        if (lane < n_group) {
            // a group's score: its best expert (DeepSeek-V2) or the sum of its two best (DeepSeek-V3)
            float m = -FLT_MAX, m2 = -FLT_MAX;
            for (int j = 0; j < gs; ++j) {
                const float x = sel[lane * gs + j];
                if (x > m) { m2 = m; m = x; } else if (x > m2) { m2 = x; }
            }
            gscore[lane] = (group_top2 && gs >= 2) ? m + m2 : m;
        }
        __syncwarp();
        // keep the topk_group best groups (ties -> lower group id): rank of my group
        if (lane < n_group) {
            int rank = 0;
            const float mine = gscore[lane];
            for (int j = 0; j < n_group; ++j) rank += (gscore[j] > mine) || (gscore[j] == mine && j < lane);
            if (rank >= topk_group)
                for (int j = 0; j < gs; ++j) sel[lane * gs + j] = -INFINITY;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < GATE_NI; ++i)
            if (32 * i < E && lane + 32 * i < E) v[i] = sel[lane + 32 * i];
        __syncwarp();
    }
    // k rounds of warp arg-max (ties -> lower expert id); lane `round` keeps that round's pick
    float wsum = 0.f, my_w = 0.f;
    int my_id = 0;
    for (int round = 0; round < k; ++round) {
        float bv = -INFINITY;
        unsigned bi = 0x7fffffffu;
#pragma unroll
        for (int i = 0; i < GATE_NI; ++i)
            if (32 * i < E && lane + 32 * i < E && (v[i] > bv || (v[i] == bv && bi == 0x7fffffffu))) { bv = v[i]; bi = lane + 32 * i; }
        const float top = warp_max(bv);
        unsigned pick = __reduce_min_sync(0xffffffffu, bv == top ? bi : 0x7fffffffu);
        if (pick >= (unsigned) E) pick = 0;     // no number among the scores; a masked -inf is re-picked when fewer than k experts are eligible
        float w = 0.f;
#pragma unroll
        for (int i = 0; i < GATE_NI; ++i)
            if ((int) (pick >> 5) == i) {
                w = p[i];
                if ((int) (pick & 31) == lane) v[i] = -INFINITY;
            }
        w = __shfl_sync(0xffffffffu, w, pick & 31);
        if (lane == round) { my_id = (int) pick; my_w = w; }
        wsum += w;
    }
    if (lane < ld) {
        // shared experts ride along as always-selected experts E, E+1, ... with weight 1, or that of their gate
        const bool routed = lane < k;
        const int id = routed ? my_id : E + (lane - k);
        float w = routed ? (norm ? my_w / wsum : my_w) * scale : 1.f;
        if (!routed && shared_gate && !dry) w = 1.f / (1.f + expf(-__ldcg(logits_row + E)));
        if (!dry && ids != nullptr) {
            ids[(size_t) t * ld + lane] = id;
            wts[(size_t) t * ld + lane] = w;
        }
        if (ids_copy != nullptr) ids_copy[t * ld + lane] = id;
        if (wts_copy != nullptr) wts_copy[t * ld + lane] = w;
    }
}

}  // namespace
