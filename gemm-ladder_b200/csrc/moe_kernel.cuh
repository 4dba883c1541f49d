// moe_kernel.cuh -- a mixture-of-experts MLP layer for few tokens (T <= 128), in two kernels:
//
//   router    logits l_te = x_t . r_e;  S_t = the top_k experts of token t (equal logits: the lower index);
//             p_te = exp(l_te - max) / sum over S_t (or over all experts)
//   experts   g = x_t W1[e][:F]^T, u = x_t W1[e][F:]^T;  h_te = p_te silu(g) u (0 where e is not in S_t);
//             y_t = sum_e h_te W2[e]^T
//
// With few tokens the layer is a stream of the active experts' weights: 6 D F bytes each, read once, against 2 T
// multiplications per weight at most.  So the experts kernel is one persistent block per SM whose TMA producer streams
// weights without a pause from the first to the last byte:
//   - as in the swap-AB GEMM the weights fill the MMA's 128 rows (two MMAs per stage: gate and up rows, or 256 rows of
//     W2) and the tokens its N.  All T tokens are multiplied with every active expert (the tensor core idles anyway);
//     a token that did not choose the expert gets h = 0, so no rows are gathered or sorted.
//   - the router's weights are folded into h, so that the down product of all experts is one product whose K is the
//     active experts' F one after the other: the sum over the experts happens in the accumulator.
//   - both products are cut evenly over the blocks by K-blocks (moe_sched.h); split tiles are summed in block order
//     (the same bits on every run).
//   - between the products a block waits for the activations it needs, by active expert, but only its token-side loads
//     do: the weights of W2 are already on their way into the ring (up to 160 KB per SM, 24 MB in all), so the wait
//     costs no memory time.
// Roles: one thread of warp 0 the weights' producer, one of warp 10 the tokens', one of warp 1 the MMA issuer, warps 2-9
// the epilogue.  The blocks wait for one another, so the launch is cooperative (all blocks
// resident); every wait is bounded (ptx.cuh).
//
// Measured on a B200, router included, under load: 33 tokens over 8 experts of 4096 x 14336 (2.8 GB of weights, bf16) 466 us,
// 6.4 TB/s in the streams; 8 tokens over 128 of 4096 x 1344 (51 active, 1.7 GB) 272 us; 64 tokens over 128 of 4096 x 1280
// 686 us; 128 tokens over 32 of 2880 x 2880 380 us, where the SMs take in 58 to 75 GB/s each of weights and tokens;
// one token, top 8 of 64 of 2048 x 1024 (100 MB) 44 us, of which the stream is 15.
//
// Roundings: h to two values of the tokens' type (the MMA's operand; moe_plane_rows of moe_sched.h; p is folded in before, in
// fp32), y once at the end; sums in fp32.
#pragma once
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "kernel_common.cuh"
#include "moe_sched.h"

namespace bw {

constexpr int kMoeThreads = 352;  // 11 warps
constexpr int kMoeEpiThreads = 256;
constexpr int kMoeXBytes = 32768; // a stage of the weights' ring: 256 rows x 64 values
constexpr int kMoeMaxStages = 5;  // as fast as 6 or 1 % faster from 1 to 16 tokens (3: up to 5 % slower, 8 % at 128): deeper
                                   // rings make the counts and partials queue behind more weights in flight
constexpr int kMoeEpiThread0 = 64;

struct MoeParams {
    int T, Tp;          // tokens; rounded up to 16 (the gate/up MMA's N)
    int E, top_k, D, F;
    int bf16;           // the tokens', weights' and results' type: 1 bf16, 0 fp16
    int stages, slots;  // of the weights' ring and of the tokens'
    int slot_bytes;
    const int* ids;     // T x top_k
    const float* weights;
    const uint16_t* W2; // (the tensor maps hold the weights' addresses otherwise)
    const uint8_t* X;   // the tokens, by K-blocks (moe_token_bytes)
    uint8_t* H;         // the activations of each active expert, likewise, two planes
    long long plane;
    uint16_t* Y;        // T x D
    float* partials;
    long long slot_floats;
    int* ready;         // finished gate/up tiles per active expert
    int* counters;      // the split tiles' (moe_counter)
    unsigned long long wait_ns;
};

// Shared memory after the ring (offsets from its end).
struct MoeSmem {
    static constexpr int kBars = 0;  // weights in and out, tokens in and out (5 each), tfull, tempty (2 each), drain
    static constexpr int kMisc = (kBars + (4 * kMoeMaxStages + 5) * 8 + 15) / 16 * 16;  // tmem slot, flags
    static constexpr int kMask = kMisc + 64;                       // a bit per expert
    static constexpr int kExpert = kMask + kMoeMaxExperts / 8;     // the active experts, 16 bits each
    static constexpr int kGate = kExpert + 2 * kMoeMaxExperts;     // p of every token for the epilogue's expert (on 16 bytes)
    static constexpr int kBytes = kGate + 4 * kMoeMaxTokens;
    static_assert(kGate % 16 == 0, "read by 16 bytes");
};
// The weights and the tokens have rings of their own: a slot of tokens holds both planes of a K-block of h, and beyond 96
// tokens 4 stages of weights fit beside 3 such slots (from L2, so soon there) where only 3 stages of both would.
__host__ __device__ inline int moe_slot_bytes(int T) { return 2 * moe_plane_rows(T) * 128; }
inline void moe_rings(int T, int* stages, int* slots)
{
    const int room = BW_SMEM_LIMIT - 1024 - MoeSmem::kBytes;
    for (int s = kMoeMaxStages;; --s) {
        const int fit = (room - s * kMoeXBytes) / moe_slot_bytes(T);
        *stages = s;
        *slots = fit < s ? fit : s;
        if (fit >= s - 1) return;  // (at 4 stages always)
    }
}
inline int moe_smem_bytes(const MoeParams& p)
{
    return 1024 + p.stages * kMoeXBytes + p.slots * p.slot_bytes + MoeSmem::kBytes;
}

// The accumulators in tensor memory: two buffers of `cols` columns, each of both weight blocks, `n` columns apart (the
// MMA's N).  A down product of more than 64 tokens takes both buffers as one (2 x 2 x 2 Tp columns are not there).
struct MoeAcc {
    int n0, n1;  // gate/up, down
    int cols;
    bool both;   // the down product takes both buffers
    __device__ explicit MoeAcc(int T)
    {
        n0 = moe_padded(T);
        n1 = 2 * moe_plane_rows(T);
        both = n0 > 64;
        cols = both ? 2 * n0 : 2 * n1;
    }
    __device__ __forceinline__ int n(int phase) const { return phase ? n1 : n0; }
    __device__ __forceinline__ bool joint(int phase) const { return phase && both; }
    __device__ __forceinline__ uint32_t base(int phase, int acc) const { return joint(phase) ? 0u : (uint32_t)(acc * cols); }
};

// Spins until the counter at p reaches `want`, the abort flag rises or the limit passes.  One thread calls it.
__device__ __noinline__ bool moe_wait_count(const int* p, int want, volatile int* abort_flag, uint64_t limit_ns,
                                            uint32_t where, int seg)
{
    const uint64_t t0 = globaltimer_ns();
    for (uint32_t i = 1;; ++i) {
        if (ld_acquire_gpu(p) >= want) return true;
        if ((i & 15u) == 0) {
            if (*abort_flag) return false;
            if (globaltimer_ns() - t0 > limit_ns) {
                record_timeout(abort_flag, where, seg);
                return false;
            }
        }
    }
}

// A producer's loads in flight land before its block may leave (on the normal path they all have): the last S stages
// it filled.
__device__ __forceinline__ void moe_drain(uint64_t* full, int issued, int S, uint64_t limit_ns)
{
    const int n = issued < S ? issued : S;
    for (int i = 1; i <= n; ++i) wait_drain(&full[(issued - i) % S], (uint32_t)(((issued - i) / S) & 1), limit_ns);
}

__device__ __forceinline__ uint16_t moe_bits16(float v, int bf16)
{
    if (bf16) {
        const __nv_bfloat16 b = __float2bfloat16_rn(v);
        return *reinterpret_cast<const uint16_t*>(&b);
    }
    const __half h = __float2half_rn(v);
    return *reinterpret_cast<const uint16_t*>(&h);
}

// The parts of a split tile summed (a: this block's own part, the two weight blocks' rows, 8 tokens from c0), in block
// order so that the bits do not depend on who is last.  Two parts' loads are in flight at once, unconditional ones (a
// load under a condition is waited for before the next is issued): this block's own slot, parts past the last and
// tokens past the last group of four are read from a slot or group that exists and left out of the sum.
__device__ __forceinline__ void moe_sum_parts(const MoeParams& p, const MoeSeg& g, int c, int row, int c0, int tq,
                                              float (&a)[2][8])
{
    float own[2][8];
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            own[w][j] = a[w][j];
            a[w][j] = 0.f;
        }
    const int g0 = c0 / 4, g1 = min(g0 + 1, tq - 1);  // the groups of four tokens
#pragma unroll 1
    for (int b0 = g.first; b0 < g.first + g.nseg; b0 += 2) {
        float4 v[2][2][2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int b = min(b0 + i, g.first + g.nseg - 1);
            const float4* src = reinterpret_cast<const float4*>(p.partials + (size_t)moe_slot(g, b) * p.slot_floats) + row;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                v[i][w][0] = __ldcg(src + (size_t)(w * tq + g0) * 128);
                v[i][w][1] = __ldcg(src + (size_t)(w * tq + g1) * 128);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int b = b0 + i;
            const bool in = b < g.first + g.nseg, mine = b == c;
#pragma unroll
            for (int w = 0; w < 2; ++w)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const float u[4] = {v[i][w][j].x, v[i][w][j].y, v[i][w][j].z, v[i][w][j].w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) a[w][4 * j + e] += mine ? own[w][4 * j + e] : in ? u[e] : 0.f;
                }
        }
    }
}

constexpr float kMoeNotChosen = -1.f;  // in the place of p, which is no negative number (0 where it underflowed)

// h = p silu(g) u of 8 tokens, without a branch so that their chains overlap (the last whole gate/up tile's epilogue is
// what the down product waits for).  The fast exponential and division are within (2 + 1.16 |g|) 2^-23 and 2^-22 (below
// g = -87.3, where 1 + exp(-g) passes 2^126, the division gives 0 for up to 2^-119 |u|).  A token that did not choose the
// expert (kMoeNotChosen) contributes nothing, whatever its products.
__device__ __forceinline__ void moe_activation(const float (&a)[2][8], const float* gate, float (&v)[8])
{
    const float4 p0 = *reinterpret_cast<const float4*>(gate), p1 = *reinterpret_cast<const float4*>(gate + 4);
    const float pr[8] = {p0.x, p0.y, p0.z, p0.w, p1.x, p1.y, p1.z, p1.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        v[j] = pr[j] * (__fdividef(a[0][j], 1.0f + __expf(-a[0][j])) * a[1][j]);
        v[j] = pr[j] == kMoeNotChosen ? 0.f : v[j];
    }
}

// 8 values in the tokens' type (one test of it for all).
__device__ __forceinline__ void moe_bits8(const float (&v)[8], int bf16, uint16_t (&h)[8])
{
    if (bf16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = moe_bits16(v[j], 1);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) h[j] = moe_bits16(v[j], 0);
    }
}
// What rounding v (scaled) to h left, at the second plane's scale (exact in fp32), 0 where h is an infinity.
__device__ __forceinline__ float moe_left(float v, uint16_t h, int bf16)
{
    if (bf16) return (h & 0x7FFFu) == 0x7F80u ? 0.f : v - __uint_as_float((uint32_t)h << 16);
    __half x;
    *reinterpret_cast<uint16_t*>(&x) = h;
    return (h & 0x7FFFu) == 0x7C00u ? 0.f : (v - __half2float(x)) * (kMoeLoScale / kMoeHiScale);
}

// 8 tokens' sums from c0 of both weight blocks (tbase: the lane's accumulator, n columns per block); lo: the columns from
// the first plane of h to the second (0: there is one plane), both brought to scale and added.
__device__ __forceinline__ void moe_load8(uint32_t tbase, int n, int c0, int lo, int bf16, uint32_t (&r)[2][8])
{
    tmem_ld8(tbase + (uint32_t)c0, r[0]);
    tmem_ld8(tbase + (uint32_t)(n + c0), r[1]);
    tmem_wait_ld();
    if (!lo) return;
    uint32_t x[2][8];
    tmem_ld8(tbase + (uint32_t)(lo + c0), x[0]);
    tmem_ld8(tbase + (uint32_t)(n + lo + c0), x[1]);
    tmem_wait_ld();
    const float sh = bf16 ? 1.f : 1.f / kMoeHiScale, sl = bf16 ? 1.f : 1.f / kMoeLoScale;
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
        for (int j = 0; j < 8; ++j)
            r[w][j] = __float_as_uint(fmaf(__uint_as_float(x[w][j]), sl, __uint_as_float(r[w][j]) * sh));
}

__device__ __forceinline__ bool moe_finite(float v) { return fabsf(v) <= 3.4028235e38f; }
__device__ __forceinline__ float moe_shfl_xor(float v, int m)
{
    return __uint_as_float(__shfl_xor_sync(0xFFFFFFFFu, __float_as_uint(v), m));
}

// This block's part of a down tile's results: of the tile's n items (four tokens of one column) [n mine / nseg, n (mine + 1) /
// nseg).
__device__ __forceinline__ void moe_down_items(const MoeSeg& g, int c, int tq, int& i0, int& i1)
{
    const int items = 2 * tq * 128, mine = c - g.first;
    i0 = (int)((long long)items * mine / g.nseg);
    i1 = (int)((long long)items * (mine + 1) / g.nseg);
}

// Its sum over a split tile's parts; true if all of it is finite.  With few tokens there are fewer items than threads: 2^ls lanes then share an item, each
// adding every 2^ls-th part in block order, and their sums meet in a tree (ls depends on the sizes alone).
__device__ __noinline__ bool moe_sum_down(const MoeParams& p, const MoeSeg& g, int c, int tq, int tid, int lane)
{
    int i0, i1;
    moe_down_items(g, c, tq, i0, i1);
    bool fine = true;
    int ls = 0;
    while (ls < 5 && (1 << ls) < g.nseg && ((i1 - i0) << (ls + 1)) <= kMoeEpiThreads) ++ls;
    const int per = 32 >> ls, sub = lane / per;  // items per warp; this lane's share of its item
    for (int base = i0 + (tid >> 5) * per; base < i1; base += (kMoeEpiThreads / 32) * per) {
        const int x = base + lane % per;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (x < i1) {
            // eight parts' loads in flight: unconditional ones (past the last part, the last again), since a load
            // under a condition is waited for before the next is issued
#pragma unroll 1
            for (int b0 = g.first + sub; b0 < g.first + g.nseg; b0 += 8 << ls) {
                float4 u[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int b = min(b0 + (j << ls), g.first + g.nseg - 1);
                    u[j] = __ldcg(reinterpret_cast<const float4*>(p.partials + (size_t)moe_slot(g, b) * p.slot_floats) + x);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const bool in = b0 + (j << ls) < g.first + g.nseg;
                    v.x += in ? u[j].x : 0.f;
                    v.y += in ? u[j].y : 0.f;
                    v.z += in ? u[j].z : 0.f;
                    v.w += in ? u[j].w : 0.f;
                }
            }
        }
        for (int m = 16; m >= per; m >>= 1) {
            v.x += moe_shfl_xor(v.x, m);
            v.y += moe_shfl_xor(v.y, m);
            v.z += moe_shfl_xor(v.z, m);
            v.w += moe_shfl_xor(v.w, m);
        }
        const int w = x / (tq * 128), t0 = (x - w * tq * 128) / 128 * 4;
        const int d = g.tile * 256 + w * 128 + (x & 127);
        if (x >= i1 || sub || d >= p.D) continue;
        uint16_t* dst = p.Y + (size_t)t0 * p.D + d;
        dst[0] = moe_bits16(v.x, p.bf16);
        if (t0 + 1 < p.T) dst[(size_t)p.D] = moe_bits16(v.y, p.bf16);
        if (t0 + 2 < p.T) dst[2 * (size_t)p.D] = moe_bits16(v.z, p.bf16);
        if (t0 + 3 < p.T) dst[3 * (size_t)p.D] = moe_bits16(v.w, p.bf16);
        fine &= moe_finite(v.x) & (moe_finite(v.y) | (t0 + 1 >= p.T)) & (moe_finite(v.z) | (t0 + 2 >= p.T)) &
                (moe_finite(v.w) | (t0 + 3 >= p.T));
    }
    return fine;
}

__device__ __forceinline__ float moe_value(uint32_t bits, int bf16)
{
    if (bf16) return __uint_as_float(bits << 16);
    __half h;
    *reinterpret_cast<uint16_t*>(&h) = (uint16_t)bits;
    return __half2float(h);
}
// This block's results that are no finite numbers, again: each as the sum over its own token's experts alone, h put
// together before it is multiplied.  In the shared accumulators the zeros of tokens that did not choose an expert meet an
// infinity or a NaN of its W2 (0 x inf), and h's second value meets it with a sign of its own.  A warp per element, for
// results that were no numbers anyway: ordinary calls pay a flag.
__device__ __noinline__ void moe_redo(const MoeParams& p, const uint32_t* mask, int active, int tid, int lane)
{
    const MoeSched s = moe_sched(p.T, p.D, p.F, active, gridDim.x);
    const int c = blockIdx.x, tq = (p.T + 3) / 4;
    MoeIter it(s, c);
    MoeSeg g;
    const uint16_t inf = p.bf16 ? 0x7F80u : 0x7C00u;
    const float sh = p.bf16 ? 1.f : 1.f / kMoeHiScale, sl = p.bf16 ? 1.f : 1.f / kMoeLoScale;
    while (it.next(s, g)) {
        if (!g.phase) continue;
        int i0, i1;
        moe_down_items(g, c, tq, i0, i1);
        for (int x = i0 + (tid >> 5); x < i1; x += kMoeEpiThreads / 32) {
            const int w = x / (tq * 128), t0 = (x - w * tq * 128) / 128 * 4;
            const int d = g.tile * 256 + w * 128 + (x & 127);
            for (int t = t0; d < p.D && t < t0 + 4 && t < p.T; ++t) {
                uint16_t* y = p.Y + (size_t)t * p.D + d;
                if ((*y & 0x7FFFu) < inf) continue;
                float v = 0.f;
                for (int j = 0; j < p.top_k; ++j) {
                    const int e = p.ids[t * p.top_k + j];
                    int at = __popc(mask[e >> 5] & ((1u << (e & 31)) - 1u));
                    for (int i = 0; i < e >> 5; ++i) at += __popc(mask[i]);
                    ld_acquire_gpu(p.ready + at);  // (complete: h is in)
                    const uint16_t* w2 = p.W2 + ((size_t)e * p.D + d) * p.F;
                    for (int f = 8 * lane; f < p.F; f += 256) {
                        const uint8_t* h = p.H + moe_token_bytes(p.T, at * s.kbf + (f >> 6), t, f >> 3 & 7);
                        const uint4 a = __ldcg(reinterpret_cast<const uint4*>(h));
                        const uint4 b = __ldcg(reinterpret_cast<const uint4*>(h + p.plane));
                        const uint4 m = __ldcg(reinterpret_cast<const uint4*>(w2 + f));
                        const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
                        const uint32_t mv[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const int r = (i & 1) * 16;
                            const float hi = moe_value(av[i / 2] >> r & 0xFFFFu, p.bf16);
                            const float lo = moe_value(bv[i / 2] >> r & 0xFFFFu, p.bf16);
                            v = fmaf(fmaf(lo, sl, hi * sh), moe_value(mv[i / 2] >> r & 0xFFFFu, p.bf16), v);
                        }
                    }
                }
                for (int m = 16; m >= 1; m >>= 1) v += moe_shfl_xor(v, m);
                __syncwarp();  // every lane has read what was there
                if (lane == 0) *y = moe_bits16(v, p.bf16);
            }
        }
    }
}

// kind::f16 with fp16 (format 0) or bf16 (format 1) operands, both K-major, fp32 accumulators.
__device__ __forceinline__ uint32_t moe_idesc(int n, int bf16)
{
    return (1u << 4) | ((uint32_t)bf16 << 7) | ((uint32_t)bf16 << 10) | ((uint32_t)(n >> 3) << 17) | (8u << 24);
}

// tmw1: W1 as {D, F, 2 E} (gate and up halves of an expert are two planes), boxes of 64 x 128; tmw2: W2 as {F, D, E},
// boxes of 64 x 256.  Zeros outside both.
__global__ void __launch_bounds__(kMoeThreads, 1)
    moe_experts_kernel(const __grid_constant__ CUtensorMap tmw1, const __grid_constant__ CUtensorMap tmw2,
                       const MoeParams p)
{
#ifdef BW_EMULATE
    uint8_t* smem_raw = emu::cta_smem();
#else
    extern __shared__ uint8_t smem_raw[];
#endif
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint8_t* ring_x = smem + (size_t)p.stages * kMoeXBytes;
    uint8_t* misc = ring_x + (size_t)p.slots * p.slot_bytes;
    uint64_t* wfull = reinterpret_cast<uint64_t*>(misc + MoeSmem::kBars);  // a barrier per stage and producer, so that
    uint64_t* wempty = wfull + kMoeMaxStages;                              // each can drain its own loads
    uint64_t* xfull = wempty + kMoeMaxStages;
    uint64_t* xempty = xfull + kMoeMaxStages;
    uint64_t* tfull = xempty + kMoeMaxStages;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(misc + MoeSmem::kMisc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* epi_go = abort_flag + 1;    // two slots, alternating by segment
    volatile int* epi_sum = abort_flag + 3;   // two slots: this block sums the segment's tile
    volatile int* epi_pend = abort_flag + 5;  // two slots: a split down tile's parts are all there
    volatile int* epi_odd = abort_flag + 7;   // a result of this block is not finite
    uint32_t* mask = reinterpret_cast<uint32_t*>(misc + MoeSmem::kMask);
    uint16_t* expert = reinterpret_cast<uint16_t*>(misc + MoeSmem::kExpert);
    float* gate = reinterpret_cast<float*>(misc + MoeSmem::kGate);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, c = blockIdx.x;
    const int S = p.stages, Tp = p.Tp;
    const MoeAcc A(p.T);
    const int lo_rows = moe_plane_rows(p.T);  // from h's first plane to its second
    int tmem_cols = 32;
    while (tmem_cols < 2 * A.cols) tmem_cols *= 2;

    if (threadIdx.x == 0) {
        for (int i = 1; i < 12; ++i) BW_TRACE_VAL(i, 0);  // (12 to 15 are the router's)
        BW_TRACE_AT(0);
        for (int i = 0; i < S; ++i) {
            mbar_init(&wfull[i], 1);   // the producer's arrive.expect_tx
            mbar_init(&wempty[i], 1);  // one tcgen05.commit
        }
        for (int i = 0; i < p.slots; ++i) {
            mbar_init(&xfull[i], 1);
            mbar_init(&xempty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], kMoeEpiThreads / 32);  // one arrival per epilogue warp
        }
        mbar_init(drain, 1);
        *abort_flag = 0;
        *epi_odd = 0;
        fence_barrier_init();
    }
    if (threadIdx.x < kMoeMaxExperts / 32) mask[threadIdx.x] = 0u;
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmw1);
        prefetch_tmap(&tmw2);
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, (uint32_t)tmem_cols);
        tmem_relinquish();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (threadIdx.x == 0) BW_TRACE_AT(1);

    // the experts that some token chose, in index order
    for (int i = threadIdx.x; i < p.T * p.top_k; i += kMoeThreads) {
        const int e = p.ids[i];
        atomicOr(&mask[e >> 5], 1u << (e & 31));
    }
    __syncthreads();
    int active = 0;
    for (int w = 0; w < (p.E + 31) / 32; ++w) active += __popc(mask[w]);
    for (int e = threadIdx.x; e < p.E; e += kMoeThreads) {
        if (!(mask[e >> 5] >> (e & 31) & 1u)) continue;
        int pos = __popc(mask[e >> 5] & ((1u << (e & 31)) - 1u));
        for (int w = 0; w < e >> 5; ++w) pos += __popc(mask[w]);
        expert[pos] = (uint16_t)e;
    }
    __syncthreads();
    const MoeSched s = moe_sched(p.T, p.D, p.F, active, gridDim.x);
    if (threadIdx.x == 0) BW_TRACE_AT(3);

    if (warp == 0) {
        // ---------------------------------------------------------- the weights' producer
        if (lane == 0) {
            const uint64_t pol = policy_evict_first();  // read once
            MoeIter it(s, c);
            MoeSeg sg;
            int stage = 0, seg = 0, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            while (ok && it.next(s, sg)) {
                for (int kb = sg.k0; kb < sg.k1; ++kb) {
                    if (!wait_bounded(&wempty[stage], ph ^ 1u, abort_flag, p.wait_ns, site(0, 1, stage), seg)) {
                        ok = false;
                        break;
                    }
                    uint8_t* dst = smem + (size_t)stage * kMoeXBytes;
                    mbar_arrive_expect_tx(&wfull[stage], kMoeXBytes);
                    if (sg.phase == 0) {
                        const int e = expert[sg.tile / s.f_tiles], f0 = sg.tile % s.f_tiles * 128;
                        tma_load_3d_hint(dst, &tmw1, kb * 64, f0, 2 * e, &wfull[stage], pol);
                        tma_load_3d_hint(dst + kMoeXBytes / 2, &tmw1, kb * 64, f0, 2 * e + 1, &wfull[stage], pol);
                    } else {
                        const int sl = kb / s.kbf;
                        tma_load_3d_hint(dst, &tmw2, (kb - sl * s.kbf) * 64, sg.tile * 256, expert[sl], &wfull[stage],
                                         pol);
                    }
                    ++issued;
                    if (++stage == S) {
                        stage = 0;
                        ph ^= 1u;
                    }
                }
                ++seg;
            }
            moe_drain(wfull, issued, S, p.wait_ns);
        }
    } else if (warp == 10) {
        // ---------------------------------------------------------- the tokens' producer
        if (lane == 0) {
            MoeIter it(s, c);
            MoeSeg sg;
            int slot = 0, seg = 0, seen = -1, issued = 0;
            uint32_t ph = 0;
            bool ok = true;
            while (ok && it.next(s, sg)) {
                for (int kb = sg.k0; kb < sg.k1; ++kb) {
                    if (!wait_bounded(&xempty[slot], ph ^ 1u, abort_flag, p.wait_ns, site(3, 1, slot), seg)) {
                        ok = false;
                        break;
                    }
                    const int sl = sg.phase ? kb / s.kbf : 0;
                    if (sg.phase && sl != seen) {  // the expert's activations are complete and visible to the TMA engine
                        if (!moe_wait_count(p.ready + sl, s.f_tiles, abort_flag, p.wait_ns, site(3, 10, sl & 255), seg)) {
                            ok = false;
                            break;
                        }
                        fence_proxy_async_global();
                        seen = sl;
                    }
                    uint8_t* dst = ring_x + (size_t)slot * p.slot_bytes;
                    // the T rows of the K-block (what the MMA reads past them only fills accumulator columns past T)
                    const uint32_t bytes = (uint32_t)p.T * 128u;
                    mbar_arrive_expect_tx(&xfull[slot], sg.phase ? 2 * bytes : bytes);
                    bulk_load(dst, (sg.phase == 0 ? p.X : p.H) + (size_t)kb * bytes, bytes, &xfull[slot]);
                    if (sg.phase) bulk_load(dst + lo_rows * 128, p.H + p.plane + (size_t)kb * bytes, bytes, &xfull[slot]);
                    ++issued;
                    if (++slot == p.slots) {
                        slot = 0;
                        ph ^= 1u;
                    }
                }
                ++seg;
            }
            moe_drain(xfull, issued, p.slots, p.wait_ns);
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------- the MMA issuer
        if (lane == 0) {
#ifdef BW_TRACE
            bool in_down = false;
#endif
            MoeIter it(s, c);
            MoeSeg sg;
            int stage = 0, slot = 0, acc = 0, seg = 0;
            uint32_t ph = 0, xph = 0, aph = 0;
            bool ok = true;
            while (ok && it.next(s, sg)) {
                const int n = A.n(sg.phase);
                const bool joint = A.joint(sg.phase);
                if (!wait_bounded(&tempty[acc], aph ^ 1u, abort_flag, p.wait_ns, site(1, 3, acc), seg)) break;
                if (joint && !wait_bounded(&tempty[acc ^ 1], aph ^ (uint32_t)acc ^ 1u, abort_flag, p.wait_ns,
                                           site(1, 3, acc ^ 1), seg))
                    break;
                tc_fence_after();
                const uint32_t d = tmem_base + A.base(sg.phase, acc), idesc = moe_idesc(n, p.bf16);
                for (int kb = sg.k0; kb < sg.k1; ++kb) {
                    if (!wait_bounded(&wfull[stage], ph, abort_flag, p.wait_ns, site(1, 0, stage), seg) ||
                        !wait_bounded(&xfull[slot], xph, abort_flag, p.wait_ns, site(1, 12, slot), seg)) {
                        ok = false;
                        break;
                    }
#ifdef BW_TRACE
                    if (seg == 0 && kb == sg.k0) BW_TRACE_AT(4);     // the first weights are in
                    if (sg.phase == 1 && !in_down) BW_TRACE_AT(6);   // the first activations are in
                    in_down = sg.phase == 1;
                    if (!in_down) BW_TRACE_AT(5);                    // the last gate/up stage
                    else BW_TRACE_AT(7);                             // the last down stage
#endif
                    tc_fence_after();
                    const uint32_t sx = smem_u32(smem + (size_t)stage * kMoeXBytes);
                    const uint32_t sy = smem_u32(ring_x + (size_t)slot * p.slot_bytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const uint32_t accumulate = (kb > sg.k0 || k > 0) ? 1u : 0u;
                        mma_f16(d, desc_kmajor(sx, k), desc_kmajor(sy, k), idesc, accumulate);
                        mma_f16(d + (uint32_t)n, desc_kmajor(sx + kMoeXBytes / 2, k), desc_kmajor(sy, k), idesc, accumulate);
                    }
                    mma_commit(&wempty[stage]);
                    mma_commit(&xempty[slot]);
                    if (++slot == p.slots) {
                        slot = 0;
                        xph ^= 1u;
                    }
                    if (++stage == S) {
                        stage = 0;
                        ph ^= 1u;
                    }
                }
                if (!ok) break;
                mma_commit(&tfull[acc]);
                if (joint) {  // (acc as before, in the next phase)
                    mma_commit(&tfull[acc ^ 1]);
                    aph ^= 1u;
                } else if (++acc == 2) {
                    acc = 0;
                    aph ^= 1u;
                }
                ++seg;
            }
            mma_commit(drain);  // the MMAs in flight finish before the tensor memory is freed
            wait_drain(drain, 0, p.wait_ns);
        }
        __syncwarp();
    } else {
        // ---------------------------------------------------------- the epilogue
        // warps 2-9: two per quarter of the TMEM lanes, taking turns at the groups of 8 tokens
        const int q = warp & 3, row = q * 32 + lane;  // the TMEM lane: a row of each of the stage's two weight blocks
        const int half = (warp - 2) >> 2;
        const int tq = (p.T + 3) / 4;                 // groups of four tokens
        const int tid = threadIdx.x - kMoeEpiThread0;
        MoeIter it(s, c);
        MoeSeg sg, pend[2];
        int acc = 0, seg = 0, n_pend = 0, gate_slot = -1;
        uint32_t aph = 0;
        bool ok = true, fine = true;  // fine: this thread's results are finite so far
        // a partial: [block w of 2][group of 4 tokens][row][4]
        auto slot_of = [&](int blk, const MoeSeg& g) {
            return reinterpret_cast<float4*>(p.partials + (size_t)moe_slot(g, blk) * p.slot_floats);
        };
        while (it.next(s, sg)) {
            int* counter = p.counters + moe_counter(sg);
            const int sl = sg.tile / s.f_tiles, f = sg.tile % s.f_tiles * 128 + row;  // (gate/up)
            if (sg.phase == 0 && sl != gate_slot) {  // p of every token for this expert, while the MMAs run
                named_bar_sync(1, kMoeEpiThreads);   // the previous expert's have been read
                if (tid < Tp) {  // (a group of 8 tokens reads 8)
                    const int e = expert[sl];
                    float v = kMoeNotChosen;
                    for (int j = 0; tid < p.T && j < p.top_k; ++j) {
                        const float pr = p.weights[tid * p.top_k + j];
                        if (p.ids[tid * p.top_k + j] == e) v = pr;
                    }
                    gate[tid] = v;  // (read after the barrier below)
                }
                gate_slot = sl;
            }
            if (threadIdx.x == kMoeEpiThread0) {
                bool in = wait_bounded(&tfull[acc], aph, abort_flag, p.wait_ns, site(2, 2, acc), seg);
                if (in && A.joint(sg.phase))
                    in = wait_bounded(&tfull[acc ^ 1], aph ^ (uint32_t)acc, abort_flag, p.wait_ns, site(2, 2, acc ^ 1), seg);
                epi_go[seg & 1] = in ? 1 : 0;
                // a split gate/up tile whose other parts are all there is summed here, without writing this one
                epi_sum[seg & 1] = sg.nseg == 1 || (sg.phase == 0 && ld_acquire_gpu(counter) == sg.nseg - 1) ? 1 : 0;
            }
            named_bar_sync(1, kMoeEpiThreads);
            if (epi_go[seg & 1] != 1) {
                ok = false;
                break;
            }
            tc_fence_after();
            const uint32_t tbase = tmem_base + ((uint32_t)(q * 32) << 16) + A.base(sg.phase, acc);
            const int n = A.n(sg.phase), lo = sg.phase ? lo_rows : 0;
            bool sum_here = epi_sum[seg & 1] != 0;
            if (!sum_here) {
                float4* dst = slot_of(c, sg) + row;
#pragma unroll 1
                for (int c0 = 8 * half; c0 < p.T; c0 += 16) {
                    uint32_t r[2][8];
                    moe_load8(tbase, n, c0, lo, p.bf16, r);
#pragma unroll
                    for (int w = 0; w < 2; ++w)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            if (c0 + 4 * j < p.T)
                                __stcg(dst + (size_t)(w * tq + c0 / 4 + j) * 128,
                                       make_float4(__uint_as_float(r[w][4 * j]), __uint_as_float(r[w][4 * j + 1]),
                                                   __uint_as_float(r[w][4 * j + 2]), __uint_as_float(r[w][4 * j + 3])));
                }
                named_bar_sync(1, kMoeEpiThreads);  // every thread's part is written (and epi_sum read)
                if (threadIdx.x == kMoeEpiThread0) {
                    const int old = atom_add_acq_rel_gpu(counter, 1);  // after every thread's stores (the barrier)
                    epi_sum[seg & 1] = sg.phase == 0 && old == sg.nseg - 1 ? 1 : 0;
                }
                if (sg.phase == 0) {  // the last block of a split gate/up tile sums it
                    named_bar_sync(1, kMoeEpiThreads);
                    sum_here = epi_sum[seg & 1] != 0;
                } else {
                    pend[n_pend++] = sg;  // a split down tile is summed below, by all its blocks
                }
            }
            if (sum_here) {
#pragma unroll 1
                for (int c0 = 8 * half; c0 < p.T; c0 += 16) {
                    float a[2][8];
                    {
                        uint32_t r[2][8];
                        moe_load8(tbase, n, c0, lo, p.bf16, r);
#pragma unroll
                        for (int w = 0; w < 2; ++w)
#pragma unroll
                            for (int j = 0; j < 8; ++j) a[w][j] = __uint_as_float(r[w][j]);
                    }
                    if (sg.nseg > 1) moe_sum_parts(p, sg, c, row, c0, tq, a);
                    if (sg.phase == 0) {
                        float v[8];
                        uint16_t h[8];
                        moe_activation(a, gate + c0, v);
                        if (!p.bf16) {
#pragma unroll
                            for (int j = 0; j < 8; ++j) v[j] *= kMoeHiScale;
                        }
                        moe_bits8(v, p.bf16, h);
                        // row c0 + j (c0 a multiple of 8), value f % 64 of K-block f / 64: a warp fills 64 bytes of a row
                        uint8_t* dst = p.H + moe_token_bytes(p.T, sl * s.kbf + (f >> 6), c0, 0) + (f & 7) * 2;
                        const int chunk = f >> 3 & 7;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (c0 + j < p.T && f < p.F)
                                *reinterpret_cast<uint16_t*>(dst + j * 128 + ((chunk ^ j) << 4)) = h[j];
                        // what the rounding left, to the second plane
#pragma unroll
                        for (int j = 0; j < 8; ++j) v[j] = moe_left(v[j], h[j], p.bf16);
                        moe_bits8(v, p.bf16, h);
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            if (c0 + j < p.T && f < p.F)
                                *reinterpret_cast<uint16_t*>(dst + p.plane + j * 128 + ((chunk ^ j) << 4)) = h[j];
                    } else {
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const int d = sg.tile * 256 + w * 128 + row;
                            if (d >= p.D) continue;
#pragma unroll
                            for (int j = 0; j < 8; ++j)
                                if (c0 + j < p.T) {
                                    p.Y[(size_t)(c0 + j) * p.D + d] = moe_bits16(a[w][j], p.bf16);
                                    fine &= moe_finite(a[w][j]);
                                }
                        }
                    }
                }
                if (sg.phase == 0) {
                    named_bar_sync(1, kMoeEpiThreads);
                    if (threadIdx.x == kMoeEpiThread0) {
                        red_add_release_gpu(p.ready + sl, 1);  // h before the count
                        BW_TRACE_AT(8);  // this block's last gate/up tile is done
                    }
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&tempty[acc]);  // the accumulator is read
            if (A.joint(sg.phase)) {
                if (lane == 0) mbar_arrive(&tempty[acc ^ 1]);
                aph ^= 1u;
            } else if (++acc == 2) {
                acc = 0;
                aph ^= 1u;
            }
            ++seg;
        }
        if (threadIdx.x == kMoeEpiThread0) BW_TRACE_AT(9);  // this block's partials are written
        // the split down tiles (at most two per block): every block of a tile sums a part of it once all have written
        // theirs.  A block writes its own partials before it waits for any, so no wait can close a circle.
        for (int i = 0; ok && i < n_pend; ++i) {
            const MoeSeg& g = pend[i];
            if (threadIdx.x == kMoeEpiThread0)
                epi_pend[i] = moe_wait_count(p.counters + moe_counter(g), g.nseg, abort_flag, p.wait_ns,
                                             site(2, 11, g.first & 255), seg)
                                  ? 1
                                  : 0;
            named_bar_sync(1, kMoeEpiThreads);
            ok = epi_pend[i] != 0;
            if (threadIdx.x == kMoeEpiThread0) BW_TRACE_AT(10);  // the others' partials are in
            if (ok) fine &= moe_sum_down(p, g, c, tq, tid, lane);
        }
        if (ok && !fine) *epi_odd = 1;
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp >= 2 && warp < 10 && *epi_odd)  // (this block's results are written: the barrier)
        moe_redo(p, mask, active, threadIdx.x - kMoeEpiThread0, lane);
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, (uint32_t)tmem_cols);
    }
    if (threadIdx.x == 0) BW_TRACE_AT(11);
}

}  // namespace bw
