// grouped_dw.cuh -- the weights' gradient of a product grouped by expert:
//
//   dW_e[n, k] = sum over expert e's rows t of dY[t, n] X[t, k]          (fp16 or bf16 operands, fp32 sums)
//
// The sum runs over the ragged dimension.  A pair of SMs holds a tile of 256 rows x up to 256 columns of dW_e; both operands
// are MN-major (a row of dY or X is one k of the MMA), in stages of 64 rows.  An expert's last rows end anywhere in a stage:
// the rows after them are another expert's (perhaps not finite), so they are overwritten with zeros up to the next 16 (an
// MMA's depth) between the load and the MMAs.  For that each block's loads complete on its own barrier; its warp 2 waits
// there, clears what has to be cleared and arrives on the leader's barrier, where the MMA issuer waits for both blocks.
// Warp 3 plans; roles otherwise as in grouped_kernel.cuh; a TMEM lane is a row of dW, a column a column.
// What bounds it (one B200, bursts): 16384 rows over 64 experts, 2816 x 2048, bf16: 253 us, 746 TFLOP/s.  The gradient's 738 MB
// alone, written as zeros by the same stores, take 151 us (torch's fill 190; a DRAM that is only written takes 4 to 5 TB/s), and
// the MMAs and loads of 4 K-blocks a tile do not hide behind them whole.  1000 rows over 16, 1352 x 2048: 49 us, of which 18 are
// the 89 MB of writes; 10 tiles a pair, each with its own start and end.
#pragma once
#include "grouped_kernel.cuh"

namespace bw {

constexpr int kDwStageBytes = 32768;  // 64 rows x 128 columns of dY, the same of X
constexpr int kDwMaxStages = 6;

struct DwParams {
    const int* offsets;
    int E, T, N, K;
    int tn, tk;      // tiles along N and K
    int width;       // columns of a tile but the last (a multiple of 32)
    int stages, ring_bytes;
    int out;         // BW_TYPE_*
    uint32_t idesc;  // without N
    void* dW;        // E x N x K
    float* work;     // parts of split tiles
    int* counters;   // two per split tile, zero at the start of a call
    int* next;       // the whole tiles given out, zero at the start of a call
    unsigned long long wait_ns;
};

struct DwSmem {
    int buf, bars, misc, tables, bytes;
};
__host__ __device__ inline DwSmem dw_smem(int ring_bytes, int E)
{
    DwSmem m;
    m.buf = ring_bytes;
    m.bars = m.buf + 8 * kGxLineBytes;
    m.misc = m.bars + (3 * kDwMaxStages + 5 + 2 + 2 * kGxDescs) * 8;
    m.misc = (m.misc + 15) / 16 * 16;
    m.tables = m.misc + 64 + kGxDescs * 64;
    m.bytes = m.tables + 2 * (E + 1) * 4;
    return m;
}

// A segment: a tile, its K-blocks, and, of a split tile, the parts' numbers.
struct DwDesc {
    int e, rows;      // expert (-1: no segment left), its rows
    int t0;           // its first row
    int n0, c0;       // the tile's first row and column of dW_e
    int width;        // its columns: the MMA's N
    int k0, k1;       // K-blocks
    int tile, first, last;
    long long u0;     // the tile's first unit (split tiles)
};
static_assert(sizeof(DwDesc) <= 64, "room for the descriptors");

// Row numbers as gx_tables has them, and the running number of K-blocks of one tile of each expert.  By one warp.
__device__ __forceinline__ void dw_tables(const DwParams& p, int* off, int* cum, int lane)
{
    GxParams g;
    g.offsets = p.offsets;
    g.E = p.E;
    g.T = p.T;
    g.cap = 64;
    gx_tables(g, off, cum, lane);  // cum: runs of at most 64, 0 where an expert has no rows
    __syncwarp();
    // one more for each expert without rows: added from the end of the table on, each entry by the empty experts before it
    const int per = (p.E + 32) / 32;
    const int i0 = lane * per, i1 = i0 + per < p.E + 1 ? i0 + per : p.E + 1;
    int n = 0;
    for (int i = i0; i < i1 && i < p.E; ++i) n += off[i + 1] == off[i] ? 1 : 0;
    int sum = n;
    for (int d = 1; d < 32; d *= 2) {
        const int o = (int)__shfl_sync(0xFFFFFFFFu, (uint32_t)sum, (lane - d) & 31);
        if (lane >= d) sum += o;
    }
    n = sum - n;
    for (int i = i0; i < i1; ++i) {
        cum[i] += n;
        if (i < p.E) n += off[i + 1] == off[i] ? 1 : 0;
    }
}

__global__ void __launch_bounds__(kGxThreads, 1)
    grouped_dw_kernel(const __grid_constant__ CUtensorMap tmy, const __grid_constant__ CUtensorMap tmx, const DwParams p)
{
#ifdef BW_EMULATE
    uint8_t* smem_raw = emu::cta_smem();
#else
    extern __shared__ uint8_t smem_raw[];
#endif
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const DwSmem L = dw_smem(p.ring_bytes, p.E);
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);  // this block's loads
    uint64_t* ready = full + kDwMaxStages;                        // the leader's: both blocks' stages may be multiplied
    uint64_t* empty = ready + kDwMaxStages;
    uint64_t* tfull = empty + kDwMaxStages;
    uint64_t* tempty = tfull + 2;
    uint64_t* drain = tempty + 2;
    uint64_t* qfull = drain + 1;
    uint64_t* qasked = qfull + 1;
    uint64_t* dfull = qasked + 1;
    uint64_t* dempty = dfull + kGxDescs;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L.misc);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    volatile int* reduce_flag = abort_flag + 1;
    volatile int* epi_go = abort_flag + 2;      // two, alternating
    volatile int* queue_tile = abort_flag + 4;
    DwDesc* descs = reinterpret_cast<DwDesc*>(smem + L.misc + 64);
    int* off = reinterpret_cast<int*>(smem + L.tables);
    int* cum = off + p.E + 1;

    const int warp = warp_uniform((int)threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = (int)cluster_ctarank();
    const bool leader = rank == 0;
    const int pairs = gridDim.x / 2, c = blockIdx.x / 2;
    const int S = p.stages;
    const uint32_t limit = lean_limit(p.wait_ns);

    griddep_launch();
    if (threadIdx.x == 0) {
        for (int i = 0; i < S; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&ready[i], 2);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&tfull[i], 1);
            mbar_init(&tempty[i], 16);
        }
        mbar_init(drain, 1);
        mbar_init(qfull, 1);
        mbar_init(qasked, 2);  // both blocks' plans
        for (int i = 0; i < kGxDescs; ++i) {
            mbar_init(&dfull[i], 1);
            mbar_init(&dempty[i], 10u + (leader ? 1u : 0u));  // producer, warp 2, epilogue, MMA issuer
        }
        *abort_flag = 0;
        *reduce_flag = 0;
        fence_barrier_init();
    }
    if (warp == 0 && lane == 0) {
        prefetch_tmap(&tmy);
        prefetch_tmap(&tmx);
    }
    if (warp == 1) {
        tmem_alloc_pair(tmem_slot, 512u);
        tmem_relinquish_pair();
    }
    if (warp == 4) dw_tables(p, off, cum, lane);
    __syncwarp();
    tc_fence_before();
    cluster_sync();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    int asked = 0;
    // a warp's next descriptor (false: none left, or the wait gave up)
    auto next = [&](DwDesc& d, bool& alive) {
        const int at = asked % kGxDescs;
        alive = alive && gx_warp_wait(&dfull[at], (uint32_t)(asked / kGxDescs & 1), abort_flag, limit,
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
        int stage = 0, issued = 0;
        uint32_t ph = 0;
        bool alive = true;
        DwDesc d;
        while (next(d, alive)) {
            const int boxes = (d.width / 2 + 63) / 64;
            for (int kb = d.k0; d.rows > 0 && kb < d.k1; ++kb) {
                alive = gx_warp_wait(&empty[stage], ph ^ 1u, abort_flag, limit, site(0, 1, stage));
                if (!alive) break;
                uint8_t* sy = smem + stage * kDwStageBytes;
                const int t = d.t0 + kb * 64, y = d.n0 + rank * 128, x = d.c0 + rank * (d.width / 2);
                if (elect_one()) {
                    mbar_arrive_expect_tx(&full[stage], (uint32_t)(2 + boxes) * 8192u);
                    tma_load_3d(sy, &tmy, y, t, 0, &full[stage]);
                    tma_load_3d(sy + 8192, &tmy, y + 64, t, 0, &full[stage]);
                    tma_load_3d(sy + 16384, &tmx, x, t, 0, &full[stage]);
                    if (boxes > 1) tma_load_3d(sy + 24576, &tmx, x + 64, t, 0, &full[stage]);
                }
                ++issued;
                if (++stage == S) {
                    stage = 0;
                    ph ^= 1u;
                }
            }
        }
        if (lane == 0) gx_drain(full, issued, S, p.wait_ns);
    } else if (warp == 1) {
        // ---------------------------------------------------------- MMA issuer
        if (leader) {
            const uint64_t dy = desc_mnmajor(smem_u32(smem), 0), dx = desc_mnmajor(smem_u32(smem) + 16384u, 0);
            int stage = 0, acc = 0;
            uint32_t ph = 0, aph = 0;
            bool alive = true;
            DwDesc t;
            while (next(t, alive)) {
                if (t.rows == 0) continue;
                alive = gx_warp_wait(&tempty[acc], aph ^ 1u, abort_flag, limit, site(1, 3, acc));
                const uint32_t idesc = p.idesc | idesc_n(t.width);
                const uint32_t d = tmem_base + (uint32_t)(acc * 256);
                for (int kb = t.k0; alive && kb < t.k1; ++kb) {
                    alive = gx_warp_wait(&ready[stage], ph, abort_flag, limit, site(1, 0, stage));
                    if (!alive) break;
                    tc_fence_after();
                    const uint64_t ad = dy + (uint64_t)((uint32_t)stage * (kDwStageBytes >> 4));
                    const uint64_t bd = dx + (uint64_t)((uint32_t)stage * (kDwStageBytes >> 4));
                    const int here = t.rows - kb * 64;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (k * 16 < here) mma_f16_pair(d, ad + 128 * k, bd + 128 * k, idesc, kb > t.k0 || k > 0 ? 1u : 0u);
                        if (kb + 1 == t.k1) mma_commit_both(smem_u32(&tfull[acc]));
                        mma_commit_both(smem_u32(&empty[stage]));
                    }
                    __syncwarp();
                    if (++stage == S) {
                        stage = 0;
                        ph ^= 1u;
                    }
                }
                acc ^= 1;
                if (acc == 0) aph ^= 1u;
            }
            if (elect_one()) {
                mma_commit_pair(mapa_shared(smem_u32(drain), 0));
                wait_drain(drain, 0, p.wait_ns);
            }
        } else if (lane == 0) {
            const DwSched s = dw_sched(off, cum, p.E, p.tn * p.tk, pairs);
            const GxQueue queue = {qfull, qasked, queue_tile, 0};
            griddep_wait();  // the counters are zero (a kernel of the call's own ahead of this one writes nothing else)
            if (s.split + c < s.tiles)  // (else the plans ask for nothing)
                gx_deal(queue, p.next, s.split + pairs, s.tiles, abort_flag, limit);
        }
        __syncwarp();
    } else if (warp >= 4) {
        // ---------------------------------------------------------- epilogue
        const int q = warp & 3, h = (warp - 4) >> 2, per = gx_per_line(p.out);
        uint8_t* line = smem + L.buf + (warp - 4) * kGxLineBytes;
        const int row = q * 32 + lane;
        const uint32_t tempty0 = mapa_shared(smem_u32(&tempty[0]), 0);
        griddep_wait();
        int acc = 0;
        uint32_t aph = 0;
        bool alive = true;
        for (;; ++asked) {
            // one thread waits for the descriptor and tells the others, as in grouped_kernel.cuh
            const int at = asked % kGxDescs;
            if (threadIdx.x == kGxEpi0) {
                const bool ok = alive && wait_lean(smem_u32(&dfull[at]), (uint32_t)(asked / kGxDescs & 1), abort_flag, limit,
                                                   site(2, 10, (uint32_t)at));
                epi_go[asked & 1] = ok && descs[at].e >= 0 ? 1 : 0;
            }
            named_bar_sync(1, kGxEpiThreads);
            if (!epi_go[asked & 1]) break;
            const DwDesc t = descs[at];
            __syncwarp();
            if (alive && lane == 0) mbar_arrive(&dempty[at]);
            const int nc = t.width / 2, c0 = h * nc;
            const int r0 = t.n0 + rank * 128 + q * 32, k = t.c0 + c0;
            uint8_t* base = static_cast<uint8_t*>(p.dW) + (size_t)t.e * p.N * p.K * (p.out == 2 ? 4 : 2);
            // as whole lines; past this warp's columns (k + nc) another warp or tile writes
            const int k1 = k + nc < p.K ? k + nc : p.K;
            auto store = [&](int i, const float(&v)[16]) {
                const int at = i / 16 % per;
                gx_put16(p.out, line, at, lane, v);
                if (at == per - 1 || i + 16 >= nc)
                    gx_flush(p.out, line, base, (size_t)p.K, r0, alive ? p.N : 0, k + i - at * 16, k1, lane);
            };
            if (t.rows == 0) {
                float z[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) z[j] = 0.f;
#pragma unroll 1
                for (int i = 0; i < nc; i += 16) store(i, z);
                continue;
            }
            alive = alive && gx_warp_wait(&tfull[acc], aph, abort_flag, limit, site(2, 2, (uint32_t)acc));
            tc_fence_after();
            const uint32_t tm = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(acc * 256 + c0);
            auto slot_at = [&](int part, int i) {
                const DwSched s = dw_sched(off, cum, p.E, p.tn * p.tk, pairs);
                return reinterpret_cast<float4*>(p.work) +
                       ((size_t)(dw_slot(s, part, t.u0) * 2 + rank) * 64 + (c0 + i) / 4) * 128 + row;
            };
            bool done = true;  // this block has the tile's whole sum
            const int first = t.first, last = t.last;
            if (first != last) {
                // a part of a split tile: the last block to finish sums all parts in the order of K
#pragma unroll 1
                for (int i = 0; i < nc; i += 16) {
                    uint32_t r[16];
                    tmem_ld16(tm + (uint32_t)i, r);
                    tmem_wait_ld();
                    if (alive) {
                        float4* to = slot_at(c, i);
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            __stcg(to + j * 128, make_float4(__uint_as_float(r[4 * j]), __uint_as_float(r[4 * j + 1]),
                                                             __uint_as_float(r[4 * j + 2]), __uint_as_float(r[4 * j + 3])));
                    }
                }
                named_bar_sync(1, kGxEpiThreads);
                if (threadIdx.x == kGxEpi0)
                    *reduce_flag = alive && atom_add_acq_rel_gpu(p.counters + t.tile * 2 + rank, 1) == last - first ? 1 : 0;
                named_bar_sync(1, kGxEpiThreads);
                done = *reduce_flag != 0;
            }
            if (done) {
#pragma unroll 1
                for (int i = 0; i < nc; i += 16) {
                    float v[16];
                    if (first == last) {
                        uint32_t r[16];
                        tmem_ld16(tm + (uint32_t)i, r);
                        tmem_wait_ld();
#pragma unroll
                        for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
                    } else {
                        gx_sum_parts<4>(v, first, last, [&](int part) { return slot_at(part, i); });
                    }
                    store(i, v);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (alive && lane == 0) mbar_arrive_remote_relaxed(tempty0 + 8u * (uint32_t)acc);
            acc ^= 1;
            if (acc == 0) aph ^= 1u;
        }
    } else if (warp == 2) {
        // ---------------------------------------------------------- stages handed on, an expert's last one cleared behind it
        const uint32_t ready0 = mapa_shared(smem_u32(&ready[0]), 0);
        int stage = 0;
        uint32_t ph = 0;
        bool alive = true;
        DwDesc t;
        while (next(t, alive)) {
            for (int kb = t.k0; t.rows > 0 && kb < t.k1; ++kb) {
                alive = gx_warp_wait(&full[stage], ph, abort_flag, limit, site(4, 0, (uint32_t)stage));
                if (!alive) break;
                const int here = t.rows - kb * 64;
                if (here < 64 && here % 16) {
                    const int r1 = (here + 15) / 16 * 16;
                    uint4* box = reinterpret_cast<uint4*>(smem + stage * kDwStageBytes);  // 4 boxes of 64 rows of 8 pieces
                    const int n = (r1 - here) * 8;
                    for (int i = lane; i < 4 * n; i += 32) box[(i / n) * 512 + here * 8 + i % n] = make_uint4(0u, 0u, 0u, 0u);
                    fence_proxy_async_shared();  // the MMAs read what was written, not what was loaded
                    __syncwarp();
                }
                if (lane == 0) mbar_arrive_remote(ready0 + 8u * (uint32_t)stage);
                if (++stage == S) {
                    stage = 0;
                    ph ^= 1u;
                }
            }
        }
    } else {
        // ---------------------------------------------------------- plan
        const DwSched s = dw_sched(off, cum, p.E, p.tn * p.tk, pairs);
        GxQueue queue = {qfull, qasked, queue_tile, 0};
        DwWalk walk(s, c);
        bool alive = true;
        for (int i = 0;; ++i) {
            const int at = i % kGxDescs;
            alive = gx_warp_wait(&dempty[at], (uint32_t)(i / kGxDescs & 1) ^ 1u, abort_flag, limit, site(5, 11, (uint32_t)at));
            if (!alive) break;
            DwSeg sg;
            DwDesc d = {};
            bool some = walk.next_part(s, off, cum, sg);
            if (!some) {
                const int tile = gx_next_tile(queue, s.split + c, s.tiles, alive, abort_flag, limit);
                if (!alive) break;
                some = tile >= 0;
                if (some) DwWalk::whole(s, off, tile, sg);
            }
            if (some) {
                d.e = sg.e;
                d.t0 = off[sg.e];
                d.rows = off[sg.e + 1] - d.t0;
                const int j = sg.tile - sg.e * s.per;  // neighbouring tiles share dY's columns
                d.n0 = j / p.tk * 256;
                d.c0 = j % p.tk * p.width;
                d.width = p.K - d.c0 < p.width ? (p.K - d.c0 + 31) / 32 * 32 : p.width;
                d.k0 = sg.k0;
                d.k1 = sg.k1;
                d.tile = sg.tile;
                d.u0 = sg.u0;
                if (sg.k0 != 0 || sg.k1 != sg.kb) {
                    d.first = dw_part_of(s, sg.u0);
                    d.last = dw_part_of(s, sg.u0 + sg.kb - 1);
                } else {
                    d.first = d.last = c;
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
    }

    __syncwarp();
    tc_fence_before();
    cluster_sync();
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, 512u);
    }
    if (threadIdx.x == 0) record_abort(abort_flag);
}

}  // namespace bw
