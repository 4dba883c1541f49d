// moe_router.cuh -- the router of the mixture-of-experts layer (moe_kernel.cuh): logits l_te = x_t . r_e in fp32, the
// top_k experts of each token by logit (equal logits: the lower index), their softmax weights.
//
// A latency-bound kernel (E D values of R, 1 MB at 128 experts of 4096, and a choice per token), so its work is spread
// for short chains: a cluster of 8 blocks takes TG tokens; each of its 128 warps takes four experts and one of `ds`
// ranges of D (as many ranges as the experts leave warps for), so that a value of X or R is unpacked once for four
// products and a warp's loads are all in flight at once.  The ranges are summed in shared memory, the logits go to the
// block of the cluster that chooses for the token through distributed shared memory, and one warp per token picks: no
// counters, no second kernel.
// A logit is a chain of D / (32 ds) fp32 additions per lane (of products that are exact in fp32), a tree of five and a chain
// over the ds ranges, so within (D / (32 ds) + 5 + ds) 2^-24 of the sum of its products' magnitudes: 2^-19.6 at 64 experts of
// 2048 (ds 8), 2^-18.6 at 128 of 4096 (ds 4), 2^-17 at 256 of 8192 (ds 2).  The choice between two experts can differ from
// the exact one only where their logits agree that far.
// Measured: 3.0 us at one token over 64 experts of 2048, 4.6 us at 8 over 128 of 4096, 8 us at 64.
// It also clears the words that the experts kernel counts on, and lays the tokens out for its copies.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernel_common.cuh"
#include "moe_sched.h"
#include "quant_rows.cuh"

namespace bw {

struct RouterParams {
    const uint16_t* X;  // T x D, ldx elements from row to row
    long long ldx;
    const uint16_t* R;  // E x D
    int T, E, top_k, D;
    int ranges;         // router_ranges(E)
    int renormalize;    // 1: the weights' sum over the chosen experts is 1; 0: the softmax is over all experts
    uint8_t* XT;        // the tokens as the experts' MMAs read them (moe_token_bytes)
    int* ids;           // T x top_k, by falling logit
    float* weights;
    int* zero;
    int zero_words;
};

constexpr int kRouterBlocks = 8;     // of a cluster
constexpr int kRouterThreads = 512;
constexpr int kRouterWarps = kRouterThreads / 32;
constexpr int kRouterTE = 4;         // experts of a warp

// The ranges of D (a power of two up to a block's warps) that E experts leave warps for.
__host__ __device__ inline int router_ranges(int E)
{
    const int groups = (E + kRouterTE - 1) / kRouterTE;
    int ds = kRouterWarps;
    while (ds > 1 && kRouterBlocks * (kRouterWarps / ds) < groups) ds >>= 1;
    return ds;
}

// Larger logits get larger keys; 0 is below every key (NaN, of either sign, is above every number).
__device__ __forceinline__ uint32_t router_key(float v)
{
    if (v != v) return 0xFFFFFFFFu;
    const uint32_t u = __float_as_uint(v + 0.0f);  // -0 as 0: equal logits have equal keys
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A block's shared memory: NV sums of each warp; the logits of the token the block chooses for.
template <int NV, int EMAX>
struct RouterSmem {
    float part[kRouterWarps][NV];
    float logits[EMAX];
};

// TG tokens per cluster; up to 32 PER experts.
template <bool BF16, int TG, int PER>
__global__ void __cluster_dims__(kRouterBlocks, 1, 1) __launch_bounds__(kRouterThreads, 2)
    moe_router_kernel(const RouterParams p)
{
    constexpr int TE = kRouterTE, NV = TE * TG;
    using Smem = RouterSmem<NV, 32 * PER>;
#ifdef BW_EMULATE
    Smem& sm = *reinterpret_cast<Smem*>(emu::cta_smem());
#else
    __shared__ Smem sm;
#endif
    auto& part = sm.part;
    auto& logits = sm.logits;
    // Another block's shared memory may be written once that block has started: the first stores wait below, behind the
    // dot products.
    cluster_arrive();
    if (threadIdx.x == 0) BW_TRACE_AT(12);
    for (int i = blockIdx.x * kRouterThreads + threadIdx.x; i < p.zero_words; i += gridDim.x * kRouterThreads)
        p.zero[i] = 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const int t0 = blockIdx.x / kRouterBlocks * TG;
    const int ds = p.ranges, gpb = kRouterWarps / ds;  // ranges of D; groups of experts per block
    for (int i = rank * kRouterThreads + threadIdx.x; i < TG * (p.D / 8); i += kRouterBlocks * kRouterThreads) {
        const int t = t0 + i / (p.D / 8), c = i % (p.D / 8);
        if (t < p.T)
            *reinterpret_cast<uint4*>(p.XT + moe_token_bytes(p.T, c >> 3, t, c & 7)) =
                reinterpret_cast<const uint4*>(p.X + (size_t)t * p.ldx)[c];
    }
    const int nv = p.D / 8, v0 = nv * (warp % ds) / ds, v1 = nv * (warp % ds + 1) / ds;
    for (int g0 = 0; g0 * TE < p.E; g0 += kRouterBlocks * gpb) {
        const int e0 = (g0 + rank * gpb + warp / ds) * TE;
        float acc[TE][TG];
#pragma unroll
        for (int i = 0; i < TE; ++i)
#pragma unroll
            for (int t = 0; t < TG; ++t) acc[i][t] = 0.f;
        if (e0 < p.E) {
#pragma unroll(TG == 1 ? 4 : 1)
            for (int c = v0 + lane; c < v1; c += 32) {
                uint4 w[TE], x[TG];
#pragma unroll
                for (int i = 0; i < TE; ++i)  // (experts past the last repeat one that exists, tokens too)
                    w[i] = reinterpret_cast<const uint4*>(p.R + (size_t)(e0 + i < p.E ? e0 + i : e0) * p.D)[c];
#pragma unroll
                for (int t = 0; t < TG; ++t)
                    x[t] = reinterpret_cast<const uint4*>(p.X + (size_t)(t0 + t < p.T ? t0 + t : t0) * p.ldx)[c];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float u[TE], v[TE];
#pragma unroll
                    for (int i = 0; i < TE; ++i) {
                        const uint32_t ww[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                        unpack2<BF16>(ww[j], u[i], v[i]);
                    }
#pragma unroll
                    for (int t = 0; t < TG; ++t) {
                        const uint32_t xw[4] = {x[t].x, x[t].y, x[t].z, x[t].w};
                        float xa, xb;
                        unpack2<BF16>(xw[j], xa, xb);
#pragma unroll
                        for (int i = 0; i < TE; ++i) acc[i][t] = fmaf(v[i], xb, fmaf(u[i], xa, acc[i][t]));
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < TE; ++i)
#pragma unroll
            for (int t = 0; t < TG; ++t) {
                float v = acc[i][t];
#pragma unroll
                for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, m);
                if (lane == (i * TG + t) % 32) part[warp][i * TG + t] = v;
            }
        __syncthreads();
        if (g0 == 0) cluster_wait();
        // a logit per thread: its ranges in order, to the block that chooses for its token
        for (int n = threadIdx.x; n < gpb * NV; n += kRouterThreads) {
            const int g = n / NV, i = n % NV / TG, t = n % TG, e = (g0 + rank * gpb + g) * TE + i;
            float v = 0.f;
            for (int r = 0; r < ds; ++r) v += part[g * ds + r][i * TG + t];
            if (e < p.E) {
                st_cluster_f32(mapa_shared(smem_u32(&logits[e]), (uint32_t)t), v);
            }
        }
        if ((g0 + kRouterBlocks * gpb) * TE < p.E) __syncthreads();  // the sums are read before the next ones
    }
    if (threadIdx.x == 0) BW_TRACE_AT(13);
    cluster_sync();  // the logits are in; nothing reaches another block's shared memory after this
    const int tok = t0 + rank;
    if (rank >= TG || tok >= p.T || warp != 0) return;
    if (threadIdx.x == 0) BW_TRACE_AT(14);
    uint32_t key[PER];
    uint32_t best = 0u;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int e = lane + 32 * i;
        key[i] = e < p.E ? router_key(logits[e]) : 0u;
        best = max(best, key[i]);
    }
    int mine = 0;           // the lane-th choice
    for (int j = 0; j < p.top_k; ++j) {
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, best);
        uint32_t at = 0xFFFFFFFFu;  // the lowest index among the largest keys
#pragma unroll
        for (int i = PER - 1; i >= 0; --i)
            if (key[i] == top && lane + 32 * i < p.E) at = (uint32_t)(lane + 32 * i);
        at = __reduce_min_sync(0xFFFFFFFFu, at);
        if (lane == j) mine = (int)at;
        best = 0u;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
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
    if (threadIdx.x == 0) BW_TRACE_AT(15);
}

}  // namespace bw
