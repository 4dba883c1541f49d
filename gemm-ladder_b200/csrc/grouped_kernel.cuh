// grouped_kernel.cuh -- products grouped by expert with ragged numbers of rows, and products in 8-bit floating point with
// a scale per block of 128: one kernel.
//
//   Y[t, n] = sum_k X[t, k] W_e[n, k]     t in the rows of expert e, n < N            (kGx16: fp16 or bf16)
//   Y[t, n] = sum_b xs[t, b] ws_e[n / 128, b] sum_{k in block b} X[t, k] W_e[n, k]    (kGxF8*: e4m3, blocks of 128 of K)
// or W as E x K x N (kGx16), or silu(gate) * up of two of W's rows per output column.  One expert and no offsets: a plain
// product.
//
// A pair of SMs (cta_group::2) holds a tile of 256 weight rows x up to 256 tokens: each block loads its 128 weight rows
// and half of the tokens, the leader issues the MMA over both blocks' shared memory.  The weights are the MMA's M, so the
// ragged dimension is its N, set per tile (grouped_sched.h).  Roles of a block's 12 warps:
//   warp 0      TMA producer: a ring of stages of 128 bytes of K (64 16-bit values or 128 e4m3).
//   warp 1      tensor memory; one lane of the leader's issues the MMAs into a ring of accumulators.  One lane of the other
//               block's deals out the whole tiles.
//   warp 2      the plan: the pair's segments (a tile and its K-blocks) one after the other, as descriptors in a ring in
//               shared memory that the other warps follow.  (Each warp on its own held the schedule's state in registers that
//               the epilogue's sums need.)
//   warp 3      e4m3: the products of two scales, four K-blocks at a time, into a ring in shared memory.
//   warps 4-11  epilogue: TMEM lanes 32 (warp % 4) .. + 31, the first or second half of the columns.
// e4m3: the accumulator is taken out of tensor memory once per K-block of 128, scaled and added in fp32 registers; the MMAs of
// the next K-blocks run into the other accumulators meanwhile.  The scales differ from block to block, so no MMA may run
// across two.  With the weights as M (kGxF8Weights) a column's scale is the same in all lanes and comes from shared memory, 4
// bytes per product: 256 tokens would take 1024 cycles a K-block (128 bytes a cycle) beside 512 of MMA.  So with more
// tokens (gx_form has the bounds) they are the M (kGxF8Tokens): a lane is a token with one scale, a half of the columns one block of
// weights with another, and the product of the two is all a K-block needs.  Few tokens: the K-blocks go to the epilogue in
// groups of 128 columns (4 K-blocks of 32 tokens), since a hand-over costs more than the sums of 32 columns.
// What bounds it (one B200, device time of a call in bursts on a cold L2):
//   16384 rows over 64 experts of 2048 x 2816, bf16: 182 us, 1037 TFLOP/s (8191 rows, 32 x (5760, 2880), activation: 266 us, 1021):
//     the operands' way from L2 to the SMs.  A K-block is 64 KB per pair for 512 cycles of MMA, 10 TB/s over all SMs; the tensor
//     pipe is active 56 % of the cycles and DRAM 63 %.
//   24 rows over 64 experts of 2048 x 1024, bf16: 31 us, 22 in a graph: two launches, one tile's latency, a split tile's sum.
//   8192^3 in e4m3, the quantiser included: 581 us, 1890 TFLOP/s: the sums in the epilogue (0.55 us per K-block of a 256 x 256
//     tile; MMAs and loads alone 0.39).  8192 rows over 64 experts of 4096 x 2048: 200 us: the same, and tiles half empty.
//   17 x 8192 x 28672 in e4m3: 65 us, the weights at 3.6 TB/s: the parts of the split tiles (3.4 MB out and in), start
//     and quantiser beside 36 us of weights.
// Every wait is bounded (wait_lean, ptx.cuh).  A thread of the epilogue whose wait gave up goes on to the end of its segment
// without waiting or writing, through every barrier and every instruction that its warp executes as one, and then leaves.
#pragma once
#include <type_traits>

#include "grouped_sched.h"
#include "kernel_common.cuh"

namespace bw {

#ifdef BW_TRACE
#define GX_CLOCK(...) __VA_ARGS__
#else
#define GX_CLOCK(...)
#endif

constexpr int kGxThreads = 384;
constexpr int kGxEpi0 = 128;         // the first epilogue thread
constexpr int kGxEpiThreads = 256;
constexpr int kGxXBytes = 128 * 128;  // a block's weight rows of a stage
constexpr int kGxMaxStages = 12;
constexpr int kGxBatch = 4;           // K-blocks whose scale products are handed over at once
constexpr int kGxBatches = 2;         // such batches held
constexpr int kGxDescs = 4;           // descriptors held at most
constexpr int kGxOtherRegs = 72, kGxEpiRegs = 216;
static_assert(128 * kGxOtherRegs + 256 * kGxEpiRegs <= kGxThreads * 168, "registers moved within what the launch holds");
constexpr int kGxAccs = 8;            // accumulators in tensor memory at most
constexpr int kGxScaleBytes = kGxBatches * kGxBatch * 2 * 128 * 4;  // [batch][K-block][gate, up or half][token]
constexpr int kGxBars = 2 * kGxMaxStages + 2 * kGxAccs + 2 * kGxBatches + 2 * kGxDescs + 2 + 1;

// fp16 or bf16; e4m3 with the weight rows as the MMA's M; e4m3 with the tokens as its M.
enum : int { kGx16 = 0, kGxF8Weights = 1, kGxF8Tokens = 2 };
// What silu * up pairs: nothing; rows 256 g + i with 256 g + 128 + i; rows f with N / 2 + f.
enum : int { kGxPlain = 0, kGxGluBlocks = 1, kGxGluHalves = 2 };

struct GxParams {
    const int* offsets;    // E + 1 ascending row numbers; null: one expert with all T rows
    int E, T;              // experts, rows of X
    int N, Nout;           // weight rows per expert; columns of C
    int nt, kblocks;       // weight tiles per expert, K-blocks
    int cap, box, wbox;    // the most tokens of a tile; rows of one TMA box of X, of W
    int stages, stage_bytes, ring_bytes;
    int descs;             // descriptors held: tiles planned ahead
    int accs, group;       // accumulators in tensor memory; K-blocks of one (e4m3), cap columns each
    int mn_major;          // W is E x K x N
    int glu, out;          // kGx*; BW_TYPE_* (0 fp16, 1 bf16, 2 fp32)
    uint32_t idesc;        // without N
    void* C;               // T x Nout, contiguous
    const float* xs;       // e4m3: scale of token t, K-block b at xs[b * xs_ld + t]
    long long xs_ld;
    const float* ws;       // e4m3: [e][block of 128 rows][K-block]
    int ws_rows;           // blocks of 128 rows per expert
    float* work;           // parts of split tiles: slots of 2 x 128 x cap
    int* counters;         // two per split tile, zero at the start of a call
    int* next;             // the whole tiles given out, zero at the start of a call
    unsigned long long wait_ns;
};

// Offsets in shared memory of what follows the stage ring: the epilogue's buffers (per warp 16 tokens x 32 columns in fp32, or
// kGxLineBytes), the scale products, barriers, tables.
struct GxSmem {
    int buf, scales, bars, misc, tables, bytes;
};
__host__ __device__ inline GxSmem gx_smem(int kind, int ring_bytes, int E)
{
    GxSmem m;
    m.buf = ring_bytes;
    m.scales = m.buf + 8 * (kind == 2 ? 4096 : 2048);
    m.bars = m.scales + (kind ? kGxScaleBytes : 0);
    m.misc = m.bars + kGxBars * 8;
    m.misc = (m.misc + 15) / 16 * 16;
    m.tables = m.misc + 64 + kGxDescs * 64;
    m.bytes = m.tables + 2 * (E + 1) * 4;
    return m;
}

// A segment: a tile (its rows of X, its weight rows), its K-blocks, and, of a tile split along K, the parts' numbers.
struct GxDesc {
    int e, n;         // expert (-1: no segment left), weight tile
    int t0, t1;       // tokens [t0, t1)
    int N;            // MMA N: a multiple of 32
    int k0, k1;       // K-blocks
    int tile;         // its number, for a split tile's counters
    int first, last;  // parts of the tile: this pair's alone where equal
};
static_assert(sizeof(GxDesc) <= 64, "room for the descriptors");

// Follows ascending tile numbers through the experts.
struct GxFind {
    int e = 0;
    template <int KIND>
    __device__ __forceinline__ void at(const GxParams& p, const int* off, const int* cum, int tile, GxDesc& t)
    {
        while (cum[e + 1] * p.nt <= tile) ++e;
        t.e = e;
        t.tile = tile;
        const int runs = cum[e + 1] - cum[e], a = off[e], b = off[e + 1];
        int m;
        group_place(tile - cum[e] * p.nt, p.nt, runs, m, t.n);
        const int rows = KIND == kGxF8Tokens ? 256 : group_run_rows(a, b, runs);
        t.t0 = a + m * rows;
        t.t1 = t.t0 + rows < b ? t.t0 + rows : b;
        int n = t.t1 - t.t0;
        if (KIND == kGxF8Tokens) n = p.glu == kGxPlain && p.N - t.n * 256 < 256 ? p.N - t.n * 256 : 256;
        t.N = (n + 31) / 32 * 32;
    }
};

// A wait after which a warp goes on, or gives up, as one.
__device__ __forceinline__ bool gx_warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint32_t limit_ns,
                                             uint32_t where)
{
    const uint32_t b = smem_u32(bar);
    if (__all_sync(0xFFFFFFFFu, mbar_try_wait(b, parity))) return true;
    return __all_sync(0xFFFFFFFFu, wait_lean(b, parity, abort_flag, limit_ns, where));
}

// The stages still on their way, of `issued`, within one limit for all (the other block of an aborted pair may not have sent its
// half).
__device__ __forceinline__ void gx_drain(uint64_t* full, int issued, int S, uint64_t limit_ns)
{
    const uint64_t t0 = globaltimer_ns();
    if (limit_ns < 1000000000ull) limit_ns = 1000000000ull;
    for (int q = issued < S ? 0 : issued - S; q < issued; ++q)
        while (!mbar_try_wait(smem_u32(&full[q % S]), (uint32_t)((q / S) & 1)))
            if (globaltimer_ns() - t0 > limit_ns) return;
}

// An accumulator as the epilogue of kGxF8Tokens sees it: its tensor memory, its barriers, the phase it waits for next.
struct GxAcc {
    uint32_t tm;
    uint64_t* full;
    uint32_t empty;  // the leader's
    uint32_t ph;
};

// Whole tiles on demand.  A pair's first is its own; for each of the others the plans of both blocks ask (q.asked), and one lane
// of the second block (warp 1) draws a number from the call's counter and hands it to both (-1: none left).  Nothing is drawn
// ahead of need: with four tiles drawn ahead, pairs of 6 tiles each ended between 141 and 282 us.
struct GxQueue {
    uint64_t* full;   // the tile is there (each block's own)
    uint64_t* asked;  // the second block's: both have asked
    volatile int* tile;
    int i;            // tiles asked for
};
__device__ __forceinline__ void gx_deal(const GxQueue& q, int* counter, int first, int tiles, volatile int* abort_flag,
                                        uint32_t limit_ns)
{
    const uint32_t other = mapa_shared(smem_u32(const_cast<int*>(q.tile)), 0), full0 = mapa_shared(smem_u32(q.full), 0);
    for (uint32_t i = 0;; ++i) {
        if (!wait_lean(smem_u32(q.asked), i & 1u, abort_flag, limit_ns, site(6, 9, 0))) return;
        int t = first + atomicAdd(counter, 1);
        if (t >= tiles) t = -1;
        *q.tile = t;
        st_cluster_f32(other, __int_as_float(t));
        mbar_arrive(q.full);
        mbar_arrive_cluster(full0);
        if (t < 0) return;
    }
}
// The next whole tile, by one warp; -1: none left, or the wait gave up (alive false).
__device__ __forceinline__ int gx_next_tile(GxQueue& q, int own, int tiles, bool& alive, volatile int* abort_flag,
                                            uint32_t limit_ns)
{
    if (q.i++ == 0) return own < tiles ? own : -1;
    __syncwarp();  // the last answer has been read
    if ((threadIdx.x & 31) == 0) mbar_arrive_remote(mapa_shared(smem_u32(q.asked), 1));
    alive = gx_warp_wait(q.full, (uint32_t)(q.i & 1), abort_flag, limit_ns, site(5, 9, 0));
    return alive ? *q.tile : -1;
}

// 16 tokens x 32 columns of C: v[j] is token tb + j, column f + lane.  Through the warp's buffer, so that a token's 32
// columns leave as 16-byte pieces; only tokens below t1 and columns below Nout (a multiple of 8) are written.
__device__ __forceinline__ void gx_store16(const GxParams& p, const float (&v)[16], void* buf, int tb, int t1, int f, int lane,
                                           bool write)
{
    if (p.out == 2) {
        float* b = static_cast<float*>(buf);
#pragma unroll
        for (int j = 0; j < 16; ++j) b[j * 32 + lane] = v[j];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = tb + i * 4 + (lane >> 3), c = f + (lane & 7) * 4;
            if (write && t < t1 && c < p.Nout)
                *reinterpret_cast<float4*>(static_cast<float*>(p.C) + (size_t)t * p.Nout + c) =
                    *reinterpret_cast<const float4*>(b + (i * 4 + (lane >> 3)) * 32 + (lane & 7) * 4);
        }
    } else {
        uint16_t* b = static_cast<uint16_t*>(buf);
        if (p.out == 1) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const __nv_bfloat16 h = __float2bfloat16_rn(v[j]);
                b[j * 32 + lane] = *reinterpret_cast<const uint16_t*>(&h);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const __half h = __float2half_rn(v[j]);
                b[j * 32 + lane] = *reinterpret_cast<const uint16_t*>(&h);
            }
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int t = tb + i * 8 + (lane >> 2), c = f + (lane & 3) * 8;
            if (write && t < t1 && c < p.Nout)
                *reinterpret_cast<uint4*>(static_cast<uint16_t*>(p.C) + (size_t)t * p.Nout + c) =
                    *reinterpret_cast<const uint4*>(b + (i * 8 + (lane >> 2)) * 32 + (lane & 3) * 8);
        }
    }
    __syncwarp();
}

// Within 5 + 1.2 |g| steps of fp32.  (The fast quotient is 0 where the exponential passes 2^126, at g < -87.3: silu(g) u is then
// within 1.1e-36 |u| of it.  With the correctly rounded one the finish of a tile took 4.3 us more.)
__device__ __forceinline__ float gx_silu(float g) { return __fdividef(g, 1.0f + __expf(-g)); }

// 16 tokens of a finished sum to C.  With the activation a warp of gate rows (quarters 0 and 1) takes the up rows' sums
// from the warp of the same columns two quarters on, through that warp's buffer; the two meet twice.
__device__ __forceinline__ void gx_finish16(const GxParams& p, float (&v)[16], uint8_t* bufs, int ew, int q, int h, int tb,
                                            int t1, int f, int lane, bool write)
{
    uint8_t* mine = bufs + ew * 2048;
    if (p.glu == kGxPlain) {
        gx_store16(p, v, mine, tb, t1, f, lane, write);
        return;
    }
    const uint32_t bar = 2u + (uint32_t)(h * 2 + (q & 1));
    if (q >= 2) {
        float* b = reinterpret_cast<float*>(mine);
#pragma unroll
        for (int j = 0; j < 16; ++j) b[j * 32 + lane] = v[j];
        named_bar_sync(bar, 64);
        named_bar_sync(bar, 64);
    } else {
        named_bar_sync(bar, 64);
        // the up rows' warp: the same half, quarter q + 2
        const float* b = reinterpret_cast<const float*>(bufs + (ew + 2) * 2048);
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = gx_silu(v[j]) * b[j * 32 + lane];
        named_bar_sync(bar, 64);
        gx_store16(p, v, mine, tb, t1, f, lane, write);
    }
}

// Rows of C (or of a gradient) held one per lane, stored as whole lines through 4 KB of shared memory per warp: 32 rows of
// 128 bytes, the 16-byte piece j of row l at piece j ^ (l % 8), so that neither way conflicts.  (A lane that stored its own
// row would touch 32 lines a store.  Transposing by shuffles took registers that the sums need: 8192^3 668 -> 878 us.)
// gx_put16: 16 columns, the at-th of the line.  gx_flush: the line's columns from c0 on, of rows r0 + l; rows below r1 and
// columns below c1 (a multiple of 8) are written.
constexpr int kGxLineBytes = 4096;
__device__ __forceinline__ int gx_per_line(int out) { return out == 2 ? 2 : 4; }  // runs of 16 columns in 128 bytes
__device__ __forceinline__ void gx_put16(int out, uint8_t* buf, int at, int lane, const float (&v)[16])
{
    uint8_t* row = buf + lane * 128;
    if (out == 2) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float4*>(row + (((at * 4 + j) ^ (lane & 7)) * 16)) =
                make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        return;
    }
    uint32_t w[8];
    if (out == 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __nv_bfloat162 x = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const __half2 x = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
            w[j] = *reinterpret_cast<const uint32_t*>(&x);
        }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
        *reinterpret_cast<uint4*>(row + (((at * 2 + j) ^ (lane & 7)) * 16)) =
            make_uint4(w[4 * j], w[4 * j + 1], w[4 * j + 2], w[4 * j + 3]);
}
__device__ __forceinline__ void gx_flush(int out, const uint8_t* buf, void* base, size_t ld, int r0, int r1, int c0, int c1,
                                         int lane)
{
    __syncwarp();
    const int size = out == 2 ? 4 : 2, c = c0 + (lane & 7) * (16 / size);
    uint8_t* to = static_cast<uint8_t*>(base) + ((size_t)(r0 + lane / 8) * ld + c) * size;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int r = e * 4 + lane / 8;
        const uint4 x = *reinterpret_cast<const uint4*>(buf + r * 128 + (((lane & 7) ^ (r & 7)) * 16));
        if (r0 + r < r1 && c < c1) *reinterpret_cast<uint4*>(to + (size_t)(e * 4) * ld * size) = x;
    }
    __syncwarp();
}

// Part `slot` of a split tile: 128 x cap fp32 of this block's rows as [token / 4][row][4].
__device__ __forceinline__ float4* gx_slot(const GxParams& p, int slot, int rank, int row, int c4)
{
    return reinterpret_cast<float4*>(p.work) + ((size_t)(slot * 2 + rank) * (p.cap / 4) + c4) * 128 + row;
}

// The experts' rows and their running number of runs, in shared memory: off[e], cum[e].  Row numbers are clamped to
// ascend within [0, T], so that no value of the caller's leads outside X or C.  By the first warp.
__device__ __forceinline__ void gx_tables(const GxParams& p, int* off, int* cum, int lane)
{
    if (!p.offsets) {
        if (lane == 0) {
            off[0] = 0;
            off[1] = p.T;
            cum[0] = 0;
            cum[1] = group_runs(0, p.T, p.cap);
        }
        return;
    }
    const int per = (p.E + 32) / 32;  // E + 1 numbers
    const int i0 = lane * per, i1 = i0 + per < p.E + 1 ? i0 + per : p.E + 1;
#pragma unroll 4
    for (int i = lane; i < p.E + 1; i += 32) {  // (loads that do not wait for one another)
        const int v = p.offsets[i];
        off[i] = v < 0 ? 0 : v > p.T ? p.T : v;
    }
    __syncwarp();
    int top = 0;
    for (int i = i0; i < i1; ++i) {
        top = off[i] > top ? off[i] : top;
        off[i] = top;
    }
    int run = top;
    for (int d = 1; d < 32; d *= 2) {
        const int o = (int)__shfl_sync(0xFFFFFFFFu, (uint32_t)run, (lane - d) & 31);
        if (lane >= d && o > run) run = o;
    }
    int before = (int)__shfl_sync(0xFFFFFFFFu, (uint32_t)run, (lane - 1) & 31);
    if (lane == 0) before = 0;
    for (int i = i0; i < i1; ++i)
        if (off[i] < before) off[i] = before;
    __syncwarp();
    int n = 0;
    for (int i = i0; i < i1 && i < p.E; ++i) {
        n += group_runs(off[i], off[i + 1], p.cap);
    }
    int sum = n;
    for (int d = 1; d < 32; d *= 2) {
        const int o = (int)__shfl_sync(0xFFFFFFFFu, (uint32_t)sum, (lane - d) & 31);
        if (lane >= d) sum += o;
    }
    n = sum - n;
    for (int i = i0; i < i1; ++i) {
        cum[i] = n;
        if (i < p.E) n += group_runs(off[i], off[i + 1], p.cap);
    }
}

// v = the sum of 16 columns over the parts [first, last] in their order, each at at(part) and 128 vectors on.  U parts are on
// their way at once (one at a time, a tile split in 8 took 100 us to sum).
template <int U, class F>
__device__ __forceinline__ void gx_sum_parts(float (&v)[16], int first, int last, F at)
{
#pragma unroll
    for (int j = 0; j < 16; ++j) v[j] = 0.f;
#pragma unroll 1
    for (int part = first; part <= last; part += U) {
        float4 x[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float4* from = at(part + u <= last ? part + u : last);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[u][j] = __ldcg(from + j * 128);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (part + u > last) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                v[4 * j] += x[u][j].x;
                v[4 * j + 1] += x[u][j].y;
                v[4 * j + 2] += x[u][j].z;
                v[4 * j + 3] += x[u][j].w;
            }
        }
    }
}

// The counters' zeros, as a kernel of the call's own ahead of its product, whose set-up it overlaps.
__global__ void gx_zero_kernel(int* p, int n)
{
    griddep_launch();
    for (int i = threadIdx.x; i < n; i += blockDim.x) p[i] = 0;
}

template <int KIND>
__global__ void __launch_bounds__(kGxThreads, 1)
    grouped_kernel(const __grid_constant__ CUtensorMap tmw, const __grid_constant__ CUtensorMap tmx, const GxParams p)
{
    constexpr bool F8 = KIND != kGx16, TOK = KIND == kGxF8Tokens;
    constexpr int kRowElems = 64;  // a 128-byte row of a stage in the maps' 16-bit elements
#ifdef BW_EMULATE
    uint8_t* smem_raw = emu::cta_smem();
#else
    extern __shared__ uint8_t smem_raw[];
#endif
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const GxSmem L = gx_smem(KIND, p.ring_bytes, p.E);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
    uint64_t* empty = full + kGxMaxStages;
    uint64_t* tfull = empty + kGxMaxStages;
    uint64_t* tempty = tfull + kGxAccs;
    uint64_t* sfull = tempty + kGxAccs;
    uint64_t* sempty = sfull + kGxBatches;
    uint64_t* dfull = sempty + kGxBatches;
    uint64_t* dempty = dfull + kGxDescs;
    uint64_t* qfull = dempty + kGxDescs;
    uint64_t* qasked = qfull + 1;
    uint64_t* drain = qasked + 1;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L.misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* reduce_flag = abort_flag + 1;
    volatile int* epi_go = abort_flag + 2;      // two, alternating
    volatile int* queue_tile = abort_flag + 4;
    GxDesc* descs = reinterpret_cast<GxDesc*>(smem + L.misc + 64);
    float* scales = reinterpret_cast<float*>(smem + L.scales);
    int* off = reinterpret_cast<int*>(smem + L.tables);
    int* cum = off + p.E + 1;

    const int warp = warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const bool leader = rank == 0;
    const int pairs = gridDim.x / 2, c = blockIdx.x / 2;
    const int S = p.stages;
    const uint32_t limit = lean_limit(p.wait_ns);
    const int acc_cols = p.group * p.cap;       // columns of an accumulator
    const int tmem_cols = p.accs * acc_cols;    // a power of two, 256 or 512

    if (threadIdx.x == 0) {
        BW_TRACE_CLEAR();
        BW_TRACE_AT(0);
    }
    griddep_launch();
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < p.accs; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 16);  // the epilogue warps of both blocks
        }
        for (int i = 0; i < kGxBatches; ++i) {
            mbar_init(&sfull[i], 1);
            mbar_init(&sempty[i], 8);  // the epilogue warps
        }
        for (int i = 0; i < kGxDescs; ++i) {
            mbar_init(&dfull[i], 1);
            mbar_init(&dempty[i], 9u + (leader ? 1u : 0u) + (F8 ? 1u : 0u));  // producer, epilogue, MMA issuer, scales
        }
        mbar_init(qfull, 1);
        mbar_init(qasked, 2);  // both blocks' plans
        mbar_init(drain, 1);
        *abort_flag = 0;
        *reduce_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmw);
        prefetch_tmap(&tmx);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, (uint32_t)tmem_cols);
        tmem_relinquish_pair();
    }
    // The kernel ahead is the call's own (zero_counters or the quantiser): it writes the counters, and in bw_linear_f8 X and
    // its scales.  Whoever uses one of these waits for it (griddep_wait); W, its scales and the offsets were complete before it
    // began.
    if (warp == 2) gx_tables(p, off, cum, lane);
    __syncwarp();
    tc_fence_before();
    cluster_sync();  // barriers, tables and tensor memory of both blocks are there
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    // e4m3 holds up to 128 sums in registers: the epilogue's 8 warps take registers from the other 4 (384 threads are launched
    // with 168 each: 128 x 72 + 256 x 216 <= 384 x 168)
    if (F8 && warp < 4) reg_dec<kGxOtherRegs>();

    // a warp's next descriptor (false: none left, or the wait gave up)
    int asked = 0;
    auto next = [&](GxDesc& d, bool& alive) {
        const int at = asked % p.descs;
        alive = alive && gx_warp_wait(&dfull[at], (uint32_t)(asked / p.descs & 1), abort_flag, limit,
                                      site(3, 10, (uint32_t)at));
        if (!alive) return false;
        d = descs[at];
        __syncwarp();
        if (lane == 0) mbar_arrive(&dempty[at]);
        ++asked;
        return d.e >= 0;
    };

    if (warp == 0) {
        // ---------------------------------------------------------- TMA producer
        const uint32_t full0 = mapa_shared(smem_u32(full), 0);  // both blocks complete the leader's barriers
        int stage = 0, issued = 0;
        uint32_t ph = 0;
        bool alive = true;
        GxDesc t;
        while (next(t, alive)) {
            const int boxes = TOK ? 1 : (t.N / 2 + p.box - 1) / p.box;
            const uint32_t bytes = 2u * (kGxXBytes + (uint32_t)(boxes * p.box) * 128u);
            const int tok = t.t0 + rank * (TOK ? 128 : t.N / 2);
            // this block's weight rows: 128 in a row, or 64 gate and 64 up rows (TOK: its half of the tile's columns; one block
            // has the gate rows, the other the up rows)
            int w0, w1 = 0;
            if (TOK) {
                w0 = p.glu == kGxPlain      ? t.n * 256 + rank * (t.N / 2)
                     : p.glu == kGxGluBlocks ? t.n * 256 + rank * 128
                                             : t.n * 128 + rank * (p.N / 2);
            } else {
                w0 = p.glu == kGxPlain      ? t.n * 256 + rank * 128
                     : p.glu == kGxGluBlocks ? t.n * 256 + rank * 64
                                             : t.n * 128 + rank * 64;
                w1 = p.glu == kGxPlain ? w0 + 64 : p.glu == kGxGluBlocks ? w0 + 128 : p.N / 2 + w0;
            }
            auto load_w = [&](int kb, int st) {
                const uint32_t bar = full0 + 8u * (uint32_t)st;
                uint8_t* to = smem + st * p.stage_bytes;
                if (leader) mbar_arrive_expect_tx(&full[st], bytes);
                if (TOK) {
                    tma_load_3d_pair(to + kGxXBytes, &tmw, kb * kRowElems, w0, t.e, bar);
                } else if (p.mn_major) {
                    tma_load_3d_pair(to, &tmw, w0, kb * 64, t.e, bar);
                    tma_load_3d_pair(to + 8192, &tmw, w0 + 64, kb * 64, t.e, bar);
                } else {
                    tma_load_3d_pair(to, &tmw, kb * kRowElems, w0, t.e, bar);
                    if (p.glu != kGxPlain) tma_load_3d_pair(to + 8192, &tmw, kb * kRowElems, w1, t.e, bar);
                }
            };
            auto load_x = [&](int kb, int st) {
                const uint32_t bar = full0 + 8u * (uint32_t)st;
                uint8_t* to = smem + st * p.stage_bytes;
                if (TOK) {
                    tma_load_3d_pair(to, &tmx, kb * kRowElems, tok, 0, bar);
                } else {
                    for (int i = 0; i < boxes; ++i)
                        tma_load_3d_pair(to + kGxXBytes + i * p.box * 128, &tmx, kb * kRowElems, tok + i * p.box, 0, bar);
                }
            };
            int kb = t.k0;
            if (issued == 0) {  // the first stages' weights while the kernel ahead runs
                const int n = t.k1 - kb < S ? t.k1 - kb : S;
                if (elect_one())
                    for (int i = 0; i < n; ++i) load_w(kb + i, i);
                griddep_wait();
                if (elect_one())
                    for (int i = 0; i < n; ++i) load_x(kb + i, i);
                kb += n;
                issued = n;
                if (n == S) ph ^= 1u;
                else stage = n;
            }
            for (; kb < t.k1; ++kb) {
                alive = gx_warp_wait(&empty[stage], ph ^ 1u, abort_flag, limit, site(0, 1, stage));
                if (!alive) break;
                if (elect_one()) {
                    load_w(kb, stage);
                    load_x(kb, stage);
                }
                ++issued;
                if (++stage == S) {
                    stage = 0;
                    ph ^= 1u;
                }
            }
        }
        if (leader && lane == 0) {  // loads in flight land before the blocks may leave (after an abort; else they have landed)
            gx_drain(full, issued, S, p.wait_ns);
        }
    } else if (warp == 1) {
        if (leader) {
            // ------------------------------------------------------ MMA issuer
            // the descriptors' low words (a 16-byte step of the address is a step of 1) and their constant high words
            const uint64_t dx = !F8 && p.mn_major ? desc_mnmajor(smem_u32(smem), 0) : desc_kmajor(smem_u32(smem), 0);
            const uint64_t dy = desc_kmajor(smem_u32(smem) + kGxXBytes, 0);
            const uint32_t step = (uint32_t)p.stage_bytes >> 4, kx = !F8 && p.mn_major ? 128u : 2u;
            int stage = 0, acc = 0;
            uint32_t ph = 0, aph = 0;
            bool alive = true;
            GxDesc t;
            GX_CLOCK(long long w_full = 0, w_acc = 0, n_kb = 0, t_at = 0);
            while (next(t, alive)) {
                const uint32_t idesc = p.idesc | idesc_n(t.N);
                int in_group = 0;
                for (int kb = t.k0; kb < t.k1; ++kb) {
                    const uint64_t ad = dx + (uint64_t)(step * (uint32_t)stage), bd = dy + (uint64_t)(step * (uint32_t)stage);
                    const uint32_t d = tmem_base + (uint32_t)(acc * acc_cols + in_group * p.cap);
                    const bool last = kb + 1 == t.k1 || (F8 && in_group + 1 == p.group);
                    GX_CLOCK(t_at = clock64());
                    alive = gx_warp_wait(&full[stage], ph, abort_flag, limit, site(1, 0, stage));
                    GX_CLOCK(w_full += clock64() - t_at; if (n_kb++ == 0 && lane == 0) BW_TRACE_AT(2); t_at = clock64());
                    // (the accumulator last: e4m3, it is what the MMAs wait for)
                    if (F8 ? in_group == 0 : kb == t.k0)
                        alive = alive && gx_warp_wait(&tempty[acc], aph ^ 1u, abort_flag, limit, site(1, 3, acc));
                    GX_CLOCK(w_acc += clock64() - t_at);
                    if (!alive) break;
                    tc_fence_after();
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t accumulate = ((!F8 && kb > t.k0) || k > 0) ? 1u : 0u;
                            if constexpr (F8)
                                mma_f8_pair(d, ad + kx * k, bd + 2 * k, idesc, accumulate);
                            else
                                mma_f16_pair(d, ad + kx * k, bd + 2 * k, idesc, accumulate);
                        }
                        if (last) mma_commit_both(smem_u32(&tfull[acc]));
                        mma_commit_both(smem_u32(&empty[stage]));
                    }
                    __syncwarp();
                    if (F8) ++in_group;
                    if (last) {
                        in_group = 0;
                        if (++acc == p.accs) {
                            acc = 0;
                            aph ^= 1u;
                        }
                    }
                    if (++stage == S) {
                        stage = 0;
                        ph ^= 1u;
                    }
                }
            }
            if (lane == 0) {
                BW_TRACE_AT(3);
                BW_TRACE_VAL(12, w_full);
                BW_TRACE_VAL(13, w_acc);
                BW_TRACE_VAL(14, n_kb);
            }
            // the MMAs in flight finish before the tensor memory is freed
            if (elect_one()) {
                mma_commit_pair(mapa_shared(smem_u32(drain), 0));
                wait_drain(drain, 0, p.wait_ns);
            }
        } else if (lane == 0) {
            // ------------------------------------------------------ whole tiles dealt out
            const GroupSched s = group_sched(p.nt, p.kblocks, pairs, cum[p.E]);
            const GxQueue queue = {qfull, qasked, queue_tile, 0};
            griddep_wait();
            if (s.split + c < s.tiles)  // (else the plans ask for nothing)
                gx_deal(queue, p.next, s.split + pairs, s.tiles, abort_flag, limit);
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---------------------------------------------------------- plan
        const GroupSched s = group_sched(p.nt, p.kblocks, pairs, cum[p.E]);
        GxQueue queue = {qfull, qasked, queue_tile, 0};
        GroupWalk walk(s, c);
        GxFind find;
        bool alive = true;
        for (int i = 0;; ++i) {
            const int at = i % p.descs;
            alive = gx_warp_wait(&dempty[at], (uint32_t)(i / p.descs & 1) ^ 1u, abort_flag, limit, site(5, 11, (uint32_t)at));
            if (!alive) break;
            GroupSeg sg;
            GxDesc d = {};
            bool some = walk.next_part(s, sg);
            if (!some) {
                const int tile = gx_next_tile(queue, s.split + c, s.tiles, alive, abort_flag, limit);
                if (!alive) break;
                some = tile >= 0;
                if (some) GroupWalk::whole(s, tile, sg);
            }
            if (some) {
                find.at<KIND>(p, off, cum, sg.tile, d);
                d.k0 = sg.k0;
                d.k1 = sg.k1;
                if (sg.k0 != 0 || sg.k1 != s.kb) {
                    d.first = tile_first_part(s, sg.tile);
                    d.last = tile_last_part(s, sg.tile);
                }
            } else {
                d.e = -1;
            }
            if (lane == 0) {
                descs[at] = d;
                mbar_arrive(&dfull[at]);
            }
            __syncwarp();
            if (!some) break;
        }
    } else if (warp == 3) {
        // ---------------------------------------------------------- scale products
        if constexpr (F8) {
            int si = 0;
            uint32_t sph = 0;
            bool alive = true;
            GxDesc t;
            griddep_wait();
            while (next(t, alive)) {
                // the scale blocks of the weight rows: kGxF8Weights, of this block's rows (gate and up: of each); kGxF8Tokens, of the
                // tile's two halves of columns
                int r0, r1;
                if (p.glu == kGxGluHalves) {
                    r0 = t.n;
                    r1 = p.ws_rows / 2 + t.n;
                } else {
                    r0 = 2 * t.n + (!TOK && p.glu == kGxPlain ? rank : 0);
                    r1 = 2 * t.n + 1;
                }
                const bool two = TOK || p.glu != kGxPlain;
                const float* w0 = p.ws + ((size_t)t.e * p.ws_rows + (r0 < p.ws_rows ? r0 : p.ws_rows - 1)) * p.kblocks;
                const float* w1 = p.ws + ((size_t)t.e * p.ws_rows + (r1 < p.ws_rows ? r1 : p.ws_rows - 1)) * p.kblocks;
                const int tok = t.t0 + (TOK ? rank * 128 : 0) + lane, have = t.t1 - tok;  // this lane's: every 32nd from tok on
                // a batch is loaded while the one before it is in use: a load takes as long as several K-blocks of MMAs
                float x[kGxBatch][4], a[kGxBatch], b[kGxBatch];
                auto load = [&](int kb, float(&x)[4], float& a, float& b) {
                    if (kb >= t.k1) return;
                    const float* xs = p.xs + kb * p.xs_ld + tok;
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = i * 32 < have ? xs[i * 32] : 0.f;
                    a = w0[kb];
                    b = two ? w1[kb] : 0.f;
                };
#pragma unroll
                for (int d = 0; d < kGxBatch; ++d) load(t.k0 + d, x[d], a[d], b[d]);
                for (int kb = t.k0; kb < t.k1; kb += kGxBatch) {
                    alive = gx_warp_wait(&sempty[si], sph ^ 1u, abort_flag, limit, site(4, 13, (uint32_t)si));
                    if (!alive) break;
                    float* to = scales + si * kGxBatch * 256 + lane;
#pragma unroll
                    for (int d = 0; d < kGxBatch; ++d) {
                        if (kb + d >= t.k1) break;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (!TOK && i * 32 >= t.N) break;
                            to[d * 256 + i * 32] = x[d][i] * a[d];
                            if (two) to[d * 256 + 128 + i * 32] = x[d][i] * b[d];
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sfull[si]);
                    if (++si == kGxBatches) {
                        si = 0;
                        sph ^= 1u;
                    }
#pragma unroll
                    for (int d = 0; d < kGxBatch; ++d) load(kb + kGxBatch + d, x[d], a[d], b[d]);
                }
            }
        }
    } else {
        // ---------------------------------------------------------- epilogue
        if (F8) reg_inc<kGxEpiRegs>();
        const int ew = warp - 4, q = warp & 3, h = ew >> 2;
        const int row = q * 32 + lane;
        const uint32_t tempty0 = mapa_shared(smem_u32(&tempty[0]), 0);
        const uint32_t quarter = tmem_base + ((uint32_t)(q * 32) << 16);
        uint8_t* bufs = smem + L.buf;
        griddep_wait();
        int acc = 0, si = 0;
        uint32_t aph = 0, sph = 0;
        bool alive = true;
        // kGxF8Tokens: its two accumulators, the next to be used first
        GxAcc acc_a = {quarter, &tfull[0], tempty0, 0u}, acc_b = {quarter + (uint32_t)p.cap, &tfull[1], tempty0 + 8u, 0u};
        auto release = [&] {
            tc_fence_before();
            __syncwarp();
            if (alive && lane == 0) mbar_arrive_remote_relaxed(tempty0 + 8u * (uint32_t)acc);
        };
        auto next_acc = [&] {
            if (++acc == p.accs) {
                acc = 0;
                aph ^= 1u;
            }
        };
        // a part of a split tile has been stored: true in the last block of `parts` to come here, which sums them
        auto count_part = [&](int tile, int parts) {
            named_bar_sync(1, kGxEpiThreads);  // every thread's stores come before the count
            if (threadIdx.x == kGxEpi0)
                *reduce_flag = alive && atom_add_acq_rel_gpu(p.counters + tile * 2 + rank, 1) == parts - 1 ? 1 : 0;
            named_bar_sync(1, kGxEpiThreads);
            return *reduce_flag != 0;
        };
        auto store_part = [&](int slot, int column, const float(&v)[16]) {
            if (!alive) return;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                __stcg(gx_slot(p, slot, rank, row, column / 4 + j),
                       make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
        };
        auto sum_parts = [&](const GroupSched& s, int tile, int first, int last, int column, float(&v)[16]) {
            gx_sum_parts<4>(v, first, last,
                            [&](int part) { return gx_slot(p, part_slot(s, part, tile), rank, row, column / 4); });
        };
        for (;; ++asked) {
            // one thread waits for the descriptor and tells the other 255, so that all of them go on to the same barriers, or none
            const GxDesc& t = descs[asked % p.descs];
            if (threadIdx.x == kGxEpi0) {
                const bool ok = alive && wait_lean(smem_u32(&dfull[asked % p.descs]), (uint32_t)(asked / p.descs & 1),
                                                   abort_flag, limit, site(2, 10, (uint32_t)(asked % p.descs)));
                epi_go[asked & 1] = ok && t.e >= 0 ? 1 : 0;
            }
            named_bar_sync(1, kGxEpiThreads);
            if (!epi_go[asked & 1]) break;
            const int N = t.N;
            // This warp's columns, in runs of 16: half of the tile's.  TOK: the first or second 128, or with the activation
            // 64 gate columns and their 64 up columns.
            const int c0 = h * (N / 2), have = t.t1 - t.t0 - c0;
            const int nc = have < N / 2 ? have : N / 2;  // (those of tokens: not TOK)
            auto col = [&](int i) {
                if (!TOK) return c0 + i * 16;
                return p.glu == kGxPlain ? h * 128 + i * 16 : (i < 4 ? 0 : 64) + h * 64 + i * 16;
            };
            auto in_tile = [&](int i) { return TOK ? col(i) < N : i * 16 < nc; };
            if constexpr (KIND == kGx16) {
                alive = alive && gx_warp_wait(&tfull[acc], aph, abort_flag, limit, site(2, 2, (uint32_t)acc));
                tc_fence_after();
            } else {
                const int blocks = t.k1 - t.k0;
                // this batch's scales have been read: the next
                auto next_batch = [&] {
                    __syncwarp();
                    if (alive && lane == 0) mbar_arrive(&sempty[si]);
                    if (++si == kGxBatches) {
                        si = 0;
                        sph ^= 1u;
                    }
                };
                auto wait_scales = [&] {
                    alive = alive && gx_warp_wait(&sfull[si], sph, abort_flag, limit, site(2, 13, (uint32_t)si));
                };
                // The segment's scaled sums.  TOK: on to C from their registers, while the MMAs of the next segment run.
                // (Through tensor memory, as below, a tile took 6 us past its sums, 10 with the activation.)  Else back into the
                // segment's last accumulator, where the code below takes them as it does other types'.
                if constexpr (TOK) {
                    uint64_t sum[8][8];  // 8 runs of 16 columns, as pairs
#pragma unroll
                    for (int i = 0; i < 64; ++i) sum[i / 8][i % 8] = 0ull;
                    // this token's scale with the weights of this warp's first 64 columns, and of the others
                    const float* sc = scales + (p.glu == kGxPlain ? h * 128 : 0) + row;
                    const int sc1 = p.glu == kGxPlain ? 0 : 128, ca = col(0), cb = col(4);
                    int left = blocks, at = 0;  // K-blocks to come; of the batch, read
                    wait_scales();
                    float s0 = sc[si * kGxBatch * 256], s1 = sc[si * kGxBatch * 256 + sc1];
                    // one K-block; false after the last
                    auto block = [&](GxAcc& a) {
                        const uint64_t p0 = pair_f32(__float_as_uint(s0), __float_as_uint(s0));
                        const uint64_t p1 = pair_f32(__float_as_uint(s1), __float_as_uint(s1));
                        alive = alive && gx_warp_wait(a.full, a.ph, abort_flag, limit, site(2, 2, 0));
                        a.ph ^= 1u;
                        tc_fence_after();
                        --left;
#pragma unroll
                        for (int i = 0; i < 8; i += 2) {  // 32 columns leave tensor memory at a time
                            uint32_t r[2][16];
#pragma unroll
                            for (int j = 0; j < 2; ++j)  // (past the tile's columns: not used)
                                tmem_ld16(a.tm + (uint32_t)((i < 4 ? ca : cb) + (i + j) % 4 * 16), r[j]);
                            tmem_wait_ld();
                            if (i == 6) {
                                tc_fence_before();
                                __syncwarp();
                                if (alive && lane == 0) mbar_arrive_remote_relaxed(a.empty);
                            }
#pragma unroll
                            for (int j = 0; j < 2; ++j)
#pragma unroll
                                for (int k = 0; k < 8; ++k)
                                    sum[i + j][k] = fma_f32x2(pair_f32(r[j][2 * k], r[j][2 * k + 1]), i < 4 ? p0 : p1,
                                                              sum[i + j][k]);
                        }
                        if (!left) return false;
                        if (++at == kGxBatch) {
                            at = 0;
                            next_batch();
                            wait_scales();
                        }
                        const float* x = sc + (si * kGxBatch + at) * 256;
                        s0 = x[0];
                        s1 = x[sc1];
                        return true;
                    };
                    while (block(acc_a) && block(acc_b)) {
                    }
                    next_batch();
                    if (blocks % 2) {  // the segment ended in the first: the second is used next
                        const GxAcc x = acc_a;
                        acc_a = acc_b;
                        acc_b = x;
                    }
                    const bool glu = p.glu != kGxPlain;
                    const int r0 = t.t0 + rank * 128 + q * 32, r1 = alive ? t.t1 : 0, f0 = t.n * (glu ? 128 : 256);
                    const int per = gx_per_line(p.out);
                    uint8_t* line = bufs + ew * kGxLineBytes;
                    // columns of C in runs of 16; the tile ends after an even number of them
                    auto put = [&](int i, const float(&v)[16]) {
                        gx_put16(p.out, line, i % per, lane, v);
                        if (i % 2 == 1 && (i % per == per - 1 || !in_tile(i + 1))) {
                            const int at = f0 + col(i);
                            gx_flush(p.out, line, p.C, (size_t)p.Nout, r0, r1, at - i % per * 16,
                                     at + 16 < p.Nout ? at + 16 : p.Nout, lane);
                        }
                    };
                    auto run = [&](int i, float(&v)[16]) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            uint32_t a, b;
                            unpair_f32(sum[i][j], a, b);
                            v[2 * j] = __uint_as_float(a);
                            v[2 * j + 1] = __uint_as_float(b);
                        }
                    };
                    auto activate = [&](float(&v)[16], const float(&u)[16]) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = gx_silu(v[j]) * u[j];
                    };
                    const int first = t.first, last = t.last, tile = t.tile;
                    if (first == last) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            if ((glu && i >= 4) || !in_tile(i)) break;
                            float v[16];
                            run(i, v);
                            if (glu && i < 4) {
                                float u[16];
                                run((i + 4) % 8, u);
                                activate(v, u);
                            }
                            put(i, v);
                        }
                    } else {
                        const GroupSched s = group_sched(p.nt, p.kblocks, pairs, cum[p.E]);
                        const int slot = part_slot(s, c, tile);
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            if (in_tile(i)) {
                                float v[16];
                                run(i, v);
                                store_part(slot, col(i), v);
                            }
                        if (count_part(tile, last - first + 1)) {
                            const int runs = glu ? 4 : 8;
#pragma unroll 1
                            for (int i = 0; i < runs && in_tile(i); ++i) {
                                float v[16];
                                sum_parts(s, tile, first, last, col(i), v);
                                if (glu) {
                                    float u[16];
                                    sum_parts(s, tile, first, last, col(i + 4), u);
                                    activate(v, u);
                                }
                                put(i, v);
                            }
                        }
                    }
                } else {
                    // R: runs of 16 columns that this warp holds
                    auto accumulate = [&](auto runs) {
                        constexpr int R = decltype(runs)::value;
                        uint64_t sum[R][8];
#pragma unroll
                        for (int i = 0; i < R; ++i)
#pragma unroll
                            for (int j = 0; j < 8; ++j) sum[i][j] = 0ull;
                        for (int kb = 0;;) {
                            if (kb % kGxBatch == 0) wait_scales();
                            alive = alive && gx_warp_wait(&tfull[acc], aph, abort_flag, limit, site(2, 2, (uint32_t)acc));
                            tc_fence_after();
                            // the accumulator's K-blocks, 4 / R of them, cap columns each
                            const uint32_t tm = quarter + (uint32_t)(acc * acc_cols + c0);
                            const float* from =
                                scales + (si * kGxBatch + kb % kGxBatch) * 256 + (p.glu != kGxPlain && q >= 2 ? 128 : 0) + c0;
#pragma unroll
                            for (int w = 0; w < 4; w += 2) {
                                uint32_t r[2][16];
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const int u = w + j;
                                    if (kb + u / R < blocks && u % R * 16 < nc)
                                        tmem_ld16(tm + (uint32_t)(u / R * (R * 32) + u % R * 16), r[j]);
                                }
                                tmem_wait_ld();
#pragma unroll
                                for (int j = 0; j < 2; ++j) {
                                    const int u = w + j;
                                    if (kb + u / R < blocks && u % R * 16 < nc) {
#pragma unroll
                                        for (int k = 0; k < 8; k += 2) {
                                            uint64_t s0, s1;  // one address per warp: a broadcast
                                            ld_shared_2b64(from + u / R * 256 + u % R * 16 + 2 * k, s0, s1);
                                            uint64_t(&to)[8] = sum[u % R];
                                            to[k] = fma_f32x2(pair_f32(r[j][2 * k], r[j][2 * k + 1]), s0, to[k]);
                                            to[k + 1] = fma_f32x2(pair_f32(r[j][2 * k + 2], r[j][2 * k + 3]), s1, to[k + 1]);
                                        }
                                    }
                                }
                            }
                            kb += 4 / R;
                            if (kb % kGxBatch == 0 || kb >= blocks) next_batch();
                            if (kb >= blocks) break;
                            release();
                            next_acc();
                        }
                        const uint32_t tm = quarter + (uint32_t)(acc * acc_cols);
#pragma unroll
                        for (int i = 0; i < R; ++i)
                            if (in_tile(i)) {
                                uint32_t r[16];
#pragma unroll
                                for (int j = 0; j < 8; ++j) unpair_f32(sum[i][j], r[2 * j], r[2 * j + 1]);
                                tmem_st16(tm + (uint32_t)col(i), r);
                            }
                        tmem_wait_st();
                    };
                    if (p.cap == 128)
                        accumulate(std::integral_constant<int, 4>());
                    else if (p.cap == 64)
                        accumulate(std::integral_constant<int, 2>());
                    else
                        accumulate(std::integral_constant<int, 1>());
                }
            }
            if constexpr (!TOK) {
                const uint32_t tm = quarter + (uint32_t)(acc * acc_cols);
                // this segment's sum of 16 columns
                auto own = [&](int i, float(&v)[16]) {
                    uint32_t r[16];
                    tmem_ld16(tm + (uint32_t)col(i), r);
                    tmem_wait_ld();
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                };
                bool done = true;  // this block has the tile's whole sum
                const int first = t.first, last = t.last, tile = t.tile;
                if (first != last) {
                    // a part of a split tile: the last block to finish sums all parts in the order of K
                    const GroupSched s = group_sched(p.nt, p.kblocks, pairs, cum[p.E]);
                    const int slot = part_slot(s, c, tile);
#pragma unroll 1
                    for (int i = 0; in_tile(i); ++i) {
                        float v[16];
                        own(i, v);
                        store_part(slot, col(i), v);
                    }
                    done = count_part(tile, last - first + 1);
                }
                if (done) {
                    const int tb = t.t0 + c0, t1 = t.t1;
                    const int f = p.glu == kGxPlain ? t.n * 256 + rank * 128 + q * 32 : t.n * 128 + rank * 64 + (q & 1) * 32;
#pragma unroll 1
                    for (int i = 0; in_tile(i); ++i) {
                        float v[16];
                        if (first == last)
                            own(i, v);
                        else
                            sum_parts(group_sched(p.nt, p.kblocks, pairs, cum[p.E]), tile, first, last, col(i), v);
                        gx_finish16(p, v, bufs, ew, q, h, tb + i * 16, t1, f, lane, alive);
                    }
                }
                release();
                next_acc();
            }
            __syncwarp();  // the descriptor has been read
            if (alive && lane == 0) mbar_arrive(&dempty[asked % p.descs]);
        }
        if (threadIdx.x == kGxEpi0) BW_TRACE_AT(4);
    }

    __syncwarp();
    tc_fence_before();
    cluster_sync();  // neither block leaves while the other may still read its memory or arrive on its barriers
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, (uint32_t)tmem_cols);
    }
    if (threadIdx.x == 0) {
        record_abort(abort_flag);
        BW_TRACE_AT(5);
    }
}

}  // namespace bw
