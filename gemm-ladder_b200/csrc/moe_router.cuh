// moe_router.cuh -- the router of the mixture-of-experts layer (moe_kernel.cuh): logits l_te = x_t . r_e in fp32, the
// top_k experts of each token by logit (equal logits: the lower index), their softmax weights.
//
// A latency-bound kernel (E D values of R, 1 MB at 128 experts of 4096, and a choice per token), so its work is spread
// for short chains rather than few bytes: a cluster of 8 blocks takes TG tokens, its 64 warps the experts (a warp two
// at a time, lanes along D, 16-byte loads), the logits go to the block of the cluster that chooses for the token
// through distributed shared memory, and one warp per token picks: no counters, no second kernel, R read once per TG
// tokens (from L2 after the first).
// The sums are 32 chains of D / 32 products, exact in fp32, added in fp32, then a tree: the choice between two experts
// can differ from the exact one only where their logits agree to about 2^-21 of the products' magnitude.
// It also clears the words that the experts kernel counts on.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "moe_sched.h"
#include "quant_rows.cuh"

namespace bw {

struct RouterParams {
    const uint16_t* X;  // T x D, ldx elements from row to row
    long long ldx;
    const uint16_t* R;  // E x D
    int T, E, top_k, D;
    int renormalize;    // 1: the weights' sum over the chosen experts is 1; 0: the softmax is over all experts
    int* ids;           // T x top_k, by falling logit
    float* weights;
    int* zero;
    int zero_words;
};

constexpr int kRouterBlocks = 8;  // of a cluster
constexpr int kRouterThreads = 256;

// Larger logits get larger keys; 0 is below every key (NaN, of either sign, is above every number).
__device__ __forceinline__ uint32_t router_key(float v)
{
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as 0: equal logits have equal keys
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <bool BF16, int TG>
__global__ void __cluster_dims__(kRouterBlocks, 1, 1) __launch_bounds__(kRouterThreads)
    moe_router_kernel(const RouterParams p)
{
    __shared__ float logits[kMoeMaxExperts];  // of the token this block chooses for
    griddep_launch();
    griddep_wait();
    for (int i = blockIdx.x * kRouterThreads + threadIdx.x; i < p.zero_words; i += gridDim.x * kRouterThreads)
        p.zero[i] = 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const int t0 = blockIdx.x / kRouterBlocks * TG;
    const int warps = kRouterBlocks * (kRouterThreads / 32);
    const int nv = p.D / 8;
    for (int e = rank * (kRouterThreads / 32) + warp; e < p.E; e += 2 * warps) {
        const bool two = e + warps < p.E;
        const uint4* r0 = reinterpret_cast<const uint4*>(p.R + (size_t)e * p.D);
        const uint4* r1 = reinterpret_cast<const uint4*>(p.R + (size_t)(two ? e + warps : e) * p.D);
        float acc[2][TG];
#pragma unroll
        for (int t = 0; t < TG; ++t) acc[0][t] = acc[1][t] = 0.f;
#pragma unroll(TG == 1 ? 4 : 1)
        for (int c = lane; c < nv; c += 32) {
            const uint4 w0 = r0[c], w1 = r1[c];
            uint4 x[TG];
#pragma unroll
            for (int t = 0; t < TG; ++t) {
                const int tok = t0 + t < p.T ? t0 + t : t0;  // rows past the last token repeat a row that exists
                x[t] = reinterpret_cast<const uint4*>(p.X + (size_t)tok * p.ldx)[c];
            }
            const uint32_t a0[4] = {w0.x, w0.y, w0.z, w0.w}, a1[4] = {w1.x, w1.y, w1.z, w1.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float u0, v0, u1, v1;
                unpack2<BF16>(a0[j], u0, v0);
                unpack2<BF16>(a1[j], u1, v1);
#pragma unroll
                for (int t = 0; t < TG; ++t) {
                    const uint32_t xw[4] = {x[t].x, x[t].y, x[t].z, x[t].w};
                    float xa, xb;
                    unpack2<BF16>(xw[j], xa, xb);
                    acc[0][t] = fmaf(v0, xb, fmaf(u0, xa, acc[0][t]));
                    acc[1][t] = fmaf(v1, xb, fmaf(u1, xa, acc[1][t]));
                }
            }
        }
#pragma unroll
        for (int t = 0; t < TG; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float v = acc[h][t];
#pragma unroll
                for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
                if (lane == t && (h == 0 || two)) {
                    const uint32_t dst = mapa_shared(smem_u32(&logits[e + h * warps]), (uint32_t)t);
                    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst), "f"(v) : "memory");
                }
            }
    }
    cluster_sync();  // the logits are in; nothing reaches another block's shared memory after this
    const int tok = t0 + rank;
    if (rank >= TG || tok >= p.T || warp != 0) return;
    constexpr int kPer = kMoeMaxExperts / 32;
    uint32_t key[kPer];
    uint32_t best = 0u;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < p.E ? router_key(logits[e]) : 0u;
        best = max(best, key[i]);
    }
    int mine = 0;           // the lane-th choice
    for (int j = 0; j < p.top_k; ++j) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        uint32_t at = 0xFFFFFFFFu;  // the lowest index among the largest keys
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i)
            if (key[i] == top && lane + 32 * i < p.E) at = (uint32_t)(lane + 32 * i);
        at = __reduce_min_sync(0xFFFFFFFFu, at);
        if (lane == j) mine = (int)at;
        best = 0u;
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            if ((uint32_t)(lane + 32 * i) == at) key[i] = 0u;
            best = max(best, key[i]);
        }
    }
    const float first = logits[__shfl_sync(0xFFFFFFFFu, mine, 0)];  // the largest
    const float ex = lane < p.top_k ? expf(logits[mine] - first) : 0.f;
    float sum = 0.f;
    if (p.renormalize) {
        sum = ex;
    } else {
        for (int e = lane; e < p.E; e += 32) sum += expf(logits[e] - first);
    }
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, m);
    if (lane < p.top_k) {
        p.ids[(size_t)tok * p.top_k + lane] = mine;
        p.weights[(size_t)tok * p.top_k + lane] = ex / sum;
    }
}

}  // namespace bw
