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
//   warp 1      tensor memory; one thread of the leader issues the MMAs into a ring of accumulators (two of 256 columns, up to eight narrower).
//   warps 2, 3  kGxF8Weights: the products xs ws of a K-block, one per token (a warp 128 of them), into a ring in shared memory.
//   warps 4-11  epilogue: TMEM lanes 32 (warp % 4) .. + 31 (weight rows), the first or second half of the columns (tokens).
// e4m3: the accumulator is taken out of tensor memory once per K-block of 128, scaled and added in fp32 registers; the MMAs of
// the next K-blocks run into the other accumulators meanwhile.  The scales differ from block to block, so no MMA may run
// across two.  With the weights as M (kGxF8Weights) a column's scale is the same in all lanes and comes from shared memory, 4
// bytes per product: 256 tokens would take 1024 cycles a K-block (128 bytes a cycle) beside 512 of MMA.  So above 128 tokens
// per expert the tokens are the M (kGxF8Tokens): a lane is a token with one scale, a half of the columns one block of
// weights with another, and the product of the two is all a K-block needs.
// Every wait is bounded (ptx.cuh); after one that gave up the epilogue walks its segments to the end without waiting,
// reading or writing, so that all threads meet at every barrier.
#pragma once
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
constexpr int kGxScales = 4;          // K-blocks of scale products held
constexpr int kGxOtherRegs = 72, kGxEpiRegs = 216;
static_assert(128 * kGxOtherRegs + 256 * kGxEpiRegs <= kGxThreads * 168, "registers moved within what the launch holds");
constexpr int kGxAhead = 4;           // K-blocks whose scales are on their way
constexpr int kGxAccs = 8;            // accumulators in tensor memory at most
constexpr int kGxScaleBytes = kGxScales * 2 * 256 * 4;          // [K-block][gate, up][token]
constexpr int kGxBars = 2 * kGxMaxStages + 2 * kGxAccs + 2 * kGxScales + 1;

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
    int accs;              // accumulators in tensor memory
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
    m.bars = m.scales + (kind == 1 ? kGxScaleBytes : 0);
    m.misc = m.bars + kGxBars * 8;
    m.misc = (m.misc + 15) / 16 * 16;
    m.tables = m.misc + 64;
    m.bytes = m.tables + 2 * (E + 1) * 4;
    return m;
}

// A tile's rows of X and weight rows.
struct GxTile {
    int e, n;     // expert, weight tile
    int t0, t1;   // its tokens [t0, t1)
    int N;        // MMA N: a multiple of 32
};

// Follows ascending tile indices through the experts.
struct GxFind {
    int e = 0;
    template <int KIND>
    __device__ __forceinline__ GxTile at(const GxParams& p, const int* off, const int* cum, int tile)
    {
        while (cum[e + 1] * p.nt <= tile) ++e;
        GxTile t;
        t.e = e;
        const int runs = cum[e + 1] - cum[e], a = off[e], b = off[e + 1];
        int m;
        group_place(tile - cum[e] * p.nt, p.nt, runs, m, t.n);
        const int rows = KIND == kGxF8Tokens ? 256 : group_run_rows(a, b, runs);
        t.t0 = a + m * rows;
        t.t1 = t.t0 + rows < b ? t.t0 + rows : b;
        int n = t.t1 - t.t0;
        if (KIND == kGxF8Tokens) n = p.glu == kGxPlain && p.N - t.n * 256 < 256 ? p.N - t.n * 256 : 256;
        t.N = (n + 31) / 32 * 32;
        return t;
    }
};

// Warp-uniform bounded wait: all lanes see the phase complete (and what it orders), or none goes on.
__device__ __forceinline__ bool gx_warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, uint64_t limit_ns,
                                             uint32_t where, int seg)
{
    const uint32_t b = smem_u32(bar);
    if (__all_sync(0xFFFFFFFFu, mbar_try_wait(b, parity))) return true;
    uint32_t ok = 1;
    if ((threadIdx.x & 31) == 0) ok = wait_spin(b, parity, abort_flag, limit_ns, where, seg) ? 1u : 0u;
    ok = __shfl_sync(0xFFFFFFFFu, ok, 0);
    if (ok) mbar_try_wait(b, parity);  // complete: this lane acquires too
    return ok != 0;
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

// 16 tokens of a finished sum to C.  With the activation a warp of gate rows (quarters 0 and 1) takes the up rows' sums
// from the warp of the same columns two quarters on, through that warp's buffer; the two meet twice.
__device__ __forceinline__ void gx_finish16(const GxParams& p, float (&v)[16], uint8_t* bufs, int ew, int q, int h, int tb,
                                            const GxTile& t, int f, int lane, bool write)
{
    uint8_t* mine = bufs + ew * 2048;
    if (p.glu == kGxPlain) {
        gx_store16(p, v, mine, tb, t.t1, f, lane, write);
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
        for (int j = 0; j < 16; ++j) v[j] = v[j] / (1.0f + __expf(-v[j])) * b[j * 32 + lane];
        named_bar_sync(bar, 64);
        gx_store16(p, v, mine, tb, t.t1, f, lane, write);
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
    int top = 0;
    for (int i = i0; i < i1; ++i) {
        int v = p.offsets[i];
        v = v < 0 ? 0 : v > p.T ? p.T : v;
        top = v > top ? v : top;
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

// What each block's dynamic shared memory and registers hold follows from p and KIND; two blocks make a cluster.
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
    uint64_t* sempty = sfull + kGxScales;
    uint64_t* drain = sempty + kGxScales;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L.misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* reduce_flag = abort_flag + 1;
    float* scales = reinterpret_cast<float*>(smem + L.scales);
    int* off = reinterpret_cast<int*>(smem + L.tables);
    int* cum = off + p.E + 1;

    const int warp = warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const bool leader = rank == 0;
    const int pairs = gridDim.x / 2, c = blockIdx.x / 2;
    const int S = p.stages;
    const int tmem_cols = p.accs * p.cap;  // a power of two, 256 or 512

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
        for (int i = 0; i < kGxScales; ++i) {
            mbar_init(&sfull[i], 2);
            mbar_init(&sempty[i], 8);
        }
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
    griddep_wait();  // what the kernel ahead wrote (the offsets, X, its scales, the counters) is visible from here on
    if (warp == 4) gx_tables(p, off, cum, lane);
    __syncwarp();
    tc_fence_before();
    cluster_sync();  // barriers, tables and tensor memory of both blocks are there
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    const GroupSched s = group_sched(p.nt, p.kblocks, pairs, cum[p.E]);
    GroupWalk walk(s, c);
    GroupSeg sg;
    GxFind find;
    // kGxF8Tokens holds 128 sums in registers: the epilogue's 8 warps take registers from the other 4 (384 threads are launched
    // with 168 each: 128 x 72 + 256 x 216 <= 384 x 168)
    if (TOK && warp < 4) reg_dec<kGxOtherRegs>();

    if (warp == 0) {
        // ---------------------------------------------------------- TMA producer
        const uint32_t full0 = mapa_shared(smem_u32(full), 0);  // both blocks complete the leader's barriers
        int stage = 0, issued = 0, seg = 0;
        uint32_t ph = 0;
        bool alive = true;
        while (alive && walk.next(s, sg)) {
            const GxTile t = find.at<KIND>(p, off, cum, sg.tile);
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
            for (int kb = sg.k0; kb < sg.k1; ++kb) {
                alive = gx_warp_wait(&empty[stage], ph ^ 1u, abort_flag, p.wait_ns, site(0, 1, stage), seg);
                if (!alive) break;
                uint8_t* sx = smem + stage * p.stage_bytes;
                const uint32_t bar = full0 + 8u * (uint32_t)stage;
                if (elect_one()) {
                    if (leader) mbar_arrive_expect_tx(&full[stage], bytes);
                    if (TOK) {
                        tma_load_3d_pair(sx, &tmx, kb * kRowElems, tok, 0, bar);
                        tma_load_3d_pair(sx + kGxXBytes, &tmw, kb * kRowElems, w0, t.e, bar);
                    } else if (p.mn_major) {
                        tma_load_3d_pair(sx, &tmw, w0, kb * 64, t.e, bar);
                        tma_load_3d_pair(sx + 8192, &tmw, w0 + 64, kb * 64, t.e, bar);
                    } else {
                        tma_load_3d_pair(sx, &tmw, kb * kRowElems, w0, t.e, bar);
                        if (p.glu != kGxPlain) tma_load_3d_pair(sx + 8192, &tmw, kb * kRowElems, w1, t.e, bar);
                    }
                    for (int i = 0; !TOK && i < boxes; ++i)
                        tma_load_3d_pair(sx + kGxXBytes + i * p.box * 128, &tmx, kb * kRowElems, tok + i * p.box, 0, bar);
                }
                ++issued;
                if (++stage == S) {
                    stage = 0;
                    ph ^= 1u;
                }
            }
            ++seg;
        }
        if (leader && lane == 0) {  // loads in flight land before the blocks may leave (after an abort; else they have landed)
            const int n = issued < S ? issued : S;
            for (int i = 1; i <= n; ++i) {
                const int q = issued - i;
                wait_drain(&full[q % S], (uint32_t)((q / S) & 1), p.wait_ns);
            }
        }
    } else if (warp == 1) {
        // ---------------------------------------------------------- MMA issuer
        if (leader) {
            const uint32_t empty0[2] = {mapa_shared(smem_u32(empty), 0), mapa_shared(smem_u32(empty), 1)};
            const uint32_t tfull0[2] = {mapa_shared(smem_u32(tfull), 0), mapa_shared(smem_u32(tfull), 1)};
            // the descriptors' low words (a 16-byte step of the address is a step of 1) and their constant high words
            const uint64_t dx = !F8 && p.mn_major ? desc_mnmajor(smem_u32(smem), 0) : desc_kmajor(smem_u32(smem), 0);
            const uint64_t dy = desc_kmajor(smem_u32(smem) + kGxXBytes, 0);
            const uint32_t step = (uint32_t)p.stage_bytes >> 4, kx = !F8 && p.mn_major ? 128u : 2u;
            int stage = 0, acc = 0, seg = 0;
            uint32_t ph = 0, aph = 0;
            bool alive = true;
            GX_CLOCK(long long w_full = 0, w_acc = 0, n_kb = 0, t_at = 0);
            while (alive && walk.next(s, sg)) {
                const GxTile t = find.at<KIND>(p, off, cum, sg.tile);
                const uint32_t idesc = p.idesc | idesc_n(t.N);
                for (int kb = sg.k0; kb < sg.k1; ++kb) {
                    GX_CLOCK(t_at = clock64());
                    if (F8 || kb == sg.k0)
                        alive = gx_warp_wait(&tempty[acc], aph ^ 1u, abort_flag, p.wait_ns, site(1, 3, acc), seg);
                    GX_CLOCK(w_acc += clock64() - t_at; t_at = clock64());
                    alive = alive && gx_warp_wait(&full[stage], ph, abort_flag, p.wait_ns, site(1, 0, stage), seg);
                    if (!alive) break;
                    GX_CLOCK(w_full += clock64() - t_at; if (n_kb++ == 0 && lane == 0) BW_TRACE_AT(2));
                    tc_fence_after();
                    const uint64_t ad = dx + (uint64_t)(step * (uint32_t)stage), bd = dy + (uint64_t)(step * (uint32_t)stage);
                    const uint32_t d = tmem_base + (uint32_t)(acc * p.cap);
                    const bool last = F8 || kb + 1 == sg.k1;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const uint32_t accumulate = ((!F8 && kb > sg.k0) || k > 0) ? 1u : 0u;
                            if constexpr (F8)
                                mma_f8_pair(d, ad + kx * k, bd + 2 * k, idesc, accumulate);
                            else
                                mma_f16_pair(d, ad + kx * k, bd + 2 * k, idesc, accumulate);
                        }
                        mma_commit_pair(empty0[0] + 8u * (uint32_t)stage);
                        mma_commit_pair(empty0[1] + 8u * (uint32_t)stage);
                        if (last) {
                            mma_commit_pair(tfull0[0] + 8u * (uint32_t)acc);
                            mma_commit_pair(tfull0[1] + 8u * (uint32_t)acc);
                        }
                    }
                    __syncwarp();
                    if (last) {
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
                ++seg;
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
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------------------------------------------------- epilogue
        if (TOK) reg_inc<kGxEpiRegs>();
        const int ew = warp - 4, q = warp & 3, h = ew >> 2;
        const int row = q * 32 + lane;
        const uint32_t tempty0 = mapa_shared(smem_u32(&tempty[0]), 0);
        uint8_t* bufs = smem + L.buf;
        int acc = 0, seg = 0, si = 0;
        uint32_t aph = 0, sph = 0;
        bool alive = true;
        const float* sc_base = scales + (p.glu != kGxPlain && q >= 2 ? 256 : 0);
        auto release = [&](int a) {
            tc_fence_before();
            __syncwarp();
            if (alive && lane == 0) mbar_arrive_remote_relaxed(tempty0 + 8u * (uint32_t)a);
        };
        auto next_acc = [&] {
            if (++acc == p.accs) {
                acc = 0;
                aph ^= 1u;
            }
        };
        while (walk.next(s, sg)) {
            const GxTile t = find.at<KIND>(p, off, cum, sg.tile);
            // This warp's columns, in runs of 16: half of the tile's.  TOK: the first or second 128, or with the activation
            // 64 gate columns and their 64 up columns.
            const int nc = t.N / 2, c0 = h * nc;
            auto col = [&](int i) {
                if (!TOK) return c0 + i * 16;
                return p.glu == kGxPlain ? h * 128 + i * 16 : (i < 4 ? 0 : 64) + h * 64 + i * 16;
            };
            auto in_tile = [&](int i) { return TOK ? col(i) < t.N : i * 16 < nc; };
            const uint32_t quarter = tmem_base + ((uint32_t)(q * 32) << 16);
            if constexpr (KIND == kGx16) {
                if (alive)
                    alive = gx_warp_wait(&tfull[acc], aph, abort_flag, p.wait_ns, site(2, 2, (uint32_t)acc), seg);
                tc_fence_after();
            } else {
                constexpr int kRuns = TOK ? 8 : 4;
                uint64_t sum[kRuns][8];  // 16 columns a run, as pairs
#pragma unroll
                for (int i = 0; i < kRuns; ++i)
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum[i][j] = 0ull;
                int kb = sg.k0;
                if constexpr (TOK) {
                    // this token's scales and its columns' (one or two blocks of 128 weight rows), two K-blocks ahead
                    const int tok = t.t0 + rank * 128 + row;
                    const float* xs = p.xs + (tok < t.t1 ? tok : t.t0);
                    const int r0 = p.glu == kGxPlain ? 2 * t.n + h : p.glu == kGxGluBlocks ? 2 * t.n : t.n;
                    const int r1 = p.glu == kGxGluHalves ? p.ws_rows / 2 + t.n : r0 + 1;
                    const float* ws0 = p.ws + ((size_t)t.e * p.ws_rows + (r0 < p.ws_rows ? r0 : p.ws_rows - 1)) * p.kblocks;
                    const float* ws1 = p.ws + ((size_t)t.e * p.ws_rows + (r1 < p.ws_rows ? r1 : p.ws_rows - 1)) * p.kblocks;
                    struct Scale {
                        float x, w0, w1;
                    } ahead[2] = {};
                    auto load = [&](int k, Scale& a) {
                        if (k >= sg.k1) return;
                        a.x = xs[k * p.xs_ld];
                        a.w0 = ws0[k];
                        if (p.glu != kGxPlain) a.w1 = ws1[k];
                    };
                    load(kb, ahead[0]);
                    load(kb + 1, ahead[1]);
                    // one K-block; false after the last
                    auto block = [&](Scale& a) {
                        const uint32_t s0 = __float_as_uint(a.x * a.w0), s1 = __float_as_uint(a.x * a.w1);
                        const uint64_t p0 = pair_f32(s0, s0), p1 = p.glu != kGxPlain ? pair_f32(s1, s1) : p0;
                        load(kb + 2, a);
                        if (alive)
                            alive = gx_warp_wait(&tfull[acc], aph, abort_flag, p.wait_ns, site(2, 2, (uint32_t)acc), seg);
                        if (alive) {
                            tc_fence_after();
                            const uint32_t tm = quarter + (uint32_t)(acc * p.cap);
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {  // 32 columns leave tensor memory at a time
                                uint32_t r[2][16];
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    tmem_ld16(tm + (uint32_t)col(i + j), r[j]);  // (past the tile's: not used)
                                tmem_wait_ld();
#pragma unroll
                                for (int j = 0; j < 2; ++j)
#pragma unroll
                                    for (int k = 0; k < 8; ++k)
                                        sum[i + j][k] = fma_f32x2(pair_f32(r[j][2 * k], r[j][2 * k + 1]), i < 4 ? p0 : p1,
                                                                  sum[i + j][k]);
                            }
                        }
                        if (++kb == sg.k1) return false;
                        release(acc);
                        next_acc();
                        return true;
                    };
                    while (block(ahead[0]) && block(ahead[1])) {
                    }
                } else {
                    for (;;) {
                        if (alive)
                            alive = gx_warp_wait(&sfull[si], sph, abort_flag, p.wait_ns, site(2, 13, (uint32_t)si), seg) &&
                                    gx_warp_wait(&tfull[acc], aph, abort_flag, p.wait_ns, site(2, 2, (uint32_t)acc), seg);
                        if (alive) {
                            tc_fence_after();
                            const float* sc = sc_base + si * 512 + c0;
                            const uint32_t tm = quarter + (uint32_t)(acc * p.cap + c0);
                            uint32_t r[4][16];
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (in_tile(i)) tmem_ld16(tm + (uint32_t)(i * 16), r[i]);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                if (in_tile(i)) {
#pragma unroll
                                    for (int k = 0; k < 8; k += 2) {
                                        uint64_t s0, s1;  // one address per warp: a broadcast
                                        ld_shared_2b64(sc + i * 16 + 2 * k, s0, s1);
                                        sum[i][k] = fma_f32x2(pair_f32(r[i][2 * k], r[i][2 * k + 1]), s0, sum[i][k]);
                                        sum[i][k + 1] = fma_f32x2(pair_f32(r[i][2 * k + 2], r[i][2 * k + 3]), s1, sum[i][k + 1]);
                                    }
                                }
                        }
                        __syncwarp();  // every lane has read the scales
                        if (alive && lane == 0) mbar_arrive(&sempty[si]);
                        if (++si == kGxScales) {
                            si = 0;
                            sph ^= 1u;
                        }
                        if (++kb == sg.k1) break;
                        release(acc);
                        next_acc();
                    }
                }
                // the sums go back into the last accumulator, where the code below takes them for all kinds
                const uint32_t tm = quarter + (uint32_t)(acc * p.cap);
#pragma unroll
                for (int i = 0; i < kRuns; ++i)
                    if (in_tile(i)) {
                        uint32_t r[16];
#pragma unroll
                        for (int j = 0; j < 8; ++j) unpair_f32(sum[i][j], r[2 * j], r[2 * j + 1]);
                        tmem_st16(tm + (uint32_t)col(i), r);
                    }
                tmem_wait_st();
            }
            const uint32_t tm = quarter + (uint32_t)(acc * p.cap);
            // this segment's sum of 16 columns
            auto own = [&](int i, float(&v)[16]) {
                uint32_t r[16];
                tmem_ld16(tm + (uint32_t)col(i), r);
                tmem_wait_ld();
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
            };
            bool done = true;  // this block has the tile's whole sum
            int first = c, last = c;
            if (sg.k0 != 0 || sg.k1 != s.kb) {
                // a part of a split tile: the last block to finish sums all parts in the order of K
                first = tile_first_part(s, sg.tile);
                last = tile_last_part(s, sg.tile);
                int* counter = p.counters + sg.tile * 2 + rank;
                named_bar_sync(1, kGxEpiThreads);  // the flag of an earlier tile has been read
                if (threadIdx.x == kGxEpi0) *reduce_flag = alive && ld_acquire_gpu(counter) == last - first ? 1 : 0;
                named_bar_sync(1, kGxEpiThreads);
                done = *reduce_flag != 0;
                if (!done) {
                    const int slot = part_slot(s, c, sg.tile);
#pragma unroll 1
                    for (int i = 0; i < 8 && in_tile(i); ++i) {
                        float v[16];
                        own(i, v);
                        if (alive) {
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                __stcg(gx_slot(p, slot, rank, row, col(i) / 4 + j),
                                       make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]));
                        }
                    }
                    named_bar_sync(1, kGxEpiThreads);  // every thread's stores come before the count
                    if (threadIdx.x == kGxEpi0)
                        *reduce_flag = alive && atom_add_acq_rel_gpu(counter, 1) == last - first ? 1 : 0;
                    named_bar_sync(1, kGxEpiThreads);
                    done = *reduce_flag != 0;
                }
            }
            // the tile's sum of 16 columns
            auto total = [&](int i, float(&v)[16]) {
                if (first == last) {
                    own(i, v);
                    return;
                }
                float mine[16];
                own(i, mine);
#pragma unroll
                for (int j = 0; j < 16; ++j) v[j] = 0.f;
                for (int part = first; part <= last; ++part) {
                    if (part == c) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] += mine[j];
                        continue;
                    }
                    const int slot = part_slot(s, part, sg.tile);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float4 x = __ldcg(gx_slot(p, slot, rank, row, col(i) / 4 + j));
                        v[4 * j] += x.x;
                        v[4 * j + 1] += x.y;
                        v[4 * j + 2] += x.z;
                        v[4 * j + 3] += x.w;
                    }
                }
            };
            if (done) {
                if constexpr (TOK) {
                    const bool glu = p.glu != kGxPlain;
                    const int r0 = t.t0 + rank * 128 + q * 32, f0 = t.n * (glu ? 128 : 256);
                    const int per = gx_per_line(p.out), runs = glu ? 4 : 8;
                    uint8_t* line = bufs + ew * kGxLineBytes;
#pragma unroll 1
                    for (int i = 0; i < runs && in_tile(i); ++i) {
                        float v[16];
                        total(i, v);
                        if (glu) {
                            float u[16];
                            total(i + 4, u);
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = v[j] / (1.0f + __expf(-v[j])) * u[j];
                        }
                        gx_put16(p.out, line, i % per, lane, v);
                        if (i % per == per - 1 || i + 1 == runs || !in_tile(i + 1))
                            gx_flush(p.out, line, p.C, (size_t)p.Nout, r0, alive ? t.t1 : 0, f0 + col(i - i % per),
                                     f0 + col(i) + 16 < p.Nout ? f0 + col(i) + 16 : p.Nout, lane);
                    }
                } else {
                    const int tb = t.t0 + c0;
                    const int f = p.glu == kGxPlain ? t.n * 256 + rank * 128 + q * 32 : t.n * 128 + rank * 64 + (q & 1) * 32;
#pragma unroll 1
                    for (int i = 0; in_tile(i); ++i) {
                        float v[16];
                        total(i, v);
                        gx_finish16(p, v, bufs, ew, q, h, tb + i * 16, t, f, lane, alive);
                    }
                }
            }
            release(acc);
            next_acc();
            ++seg;
        }
        if (threadIdx.x == kGxEpi0) BW_TRACE_AT(4);
    } else if (KIND == kGxF8Weights) {
        // ---------------------------------------------------------- scale products
        const int t00 = (warp - 2) * 128 + lane;  // this lane's first token of a tile
        int si = 0, seg = 0;
        uint32_t sph = 0;
        bool alive = true;
        while (alive && walk.next(s, sg)) {
            const GxTile t = find.at<KIND>(p, off, cum, sg.tile);
            // the scale blocks of this block's weight rows (gate and up: of each)
            const int r0 = p.glu == kGxGluHalves ? t.n : p.glu == kGxGluBlocks ? 2 * t.n : 2 * t.n + rank;
            const int r1 = p.glu == kGxGluHalves ? p.ws_rows / 2 + t.n : 2 * t.n + 1;
            const float* w0 = p.ws + ((size_t)t.e * p.ws_rows + (r0 < p.ws_rows ? r0 : p.ws_rows - 1)) * p.kblocks;
            const float* w1 = p.ws + ((size_t)t.e * p.ws_rows + (r1 < p.ws_rows ? r1 : p.ws_rows - 1)) * p.kblocks;
            const int have = t.t1 - t.t0;
            // loaded kGxAhead K-blocks ahead: a load takes as long as several K-blocks of MMAs
            float x[kGxAhead][4], a[kGxAhead], b[kGxAhead];
            auto load = [&](int kb, float(&x)[4], float& a, float& b) {
                if (kb >= sg.k1) return;
                const float* xs = p.xs + kb * p.xs_ld + t.t0;
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = t00 + i * 32 < have ? xs[t00 + i * 32] : 0.f;
                a = w0[kb];
                b = p.glu != kGxPlain ? w1[kb] : 0.f;
            };
#pragma unroll
            for (int d = 0; d < kGxAhead; ++d) load(sg.k0 + d, x[d], a[d], b[d]);
            for (int kb = sg.k0; alive && kb < sg.k1; kb += kGxAhead) {
#pragma unroll
                for (int d = 0; d < kGxAhead; ++d) {
                    if (kb + d >= sg.k1) break;
                    alive = gx_warp_wait(&sempty[si], sph ^ 1u, abort_flag, p.wait_ns, site(4, 13, (uint32_t)si), seg);
                    if (!alive) break;
                    float* to = scales + si * 512;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (t00 + i * 32 >= t.N) break;
                        to[t00 + i * 32] = x[d][i] * a[d];
                        if (p.glu != kGxPlain) to[256 + t00 + i * 32] = x[d][i] * b[d];
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sfull[si]);
                    if (++si == kGxScales) {
                        si = 0;
                        sph ^= 1u;
                    }
                    load(kb + d + kGxAhead, x[d], a[d], b[d]);
                }
            }
            ++seg;
        }
    }

    __syncwarp();
    tc_fence_before();
    cluster_sync();  // neither block leaves while the other may still read its memory or arrive on its barriers
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, (uint32_t)tmem_cols);
    }
    if (threadIdx.x == 0) BW_TRACE_AT(5);
}

}  // namespace bw
