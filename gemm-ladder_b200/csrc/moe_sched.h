// moe_sched.h -- the work of one block of the mixture-of-experts kernel (moe_kernel.cuh): which tiles of the two
// products, and which K-blocks of them.  Host and device: the kernel runs it, the CPU tests check it.
//
// Both products are streams of K-blocks (256 weight rows x 64 values, 32 KB) read once, cut evenly over the blocks
// whatever the number of active experts:
//   gate/up  tile (s, j): active expert s's gate rows [128 j, 128 j + 128) and the up rows of the same, K = D
//   down     tile i: output columns [256 i, 256 i + 256), K = the active experts' F one after the other, so the sum
//            over the experts is the accumulator's own
// A share of P >= 1 blocks out of U K-blocks: block c takes [U c / P, U (c + 1) / P), P <= U, so no share is empty.
#pragma once
#if defined(__CUDACC__)
#define BW_MOE_HD __host__ __device__
#else
#define BW_MOE_HD
#endif

namespace bw {

constexpr int kMoeMaxTokens = 128;
constexpr int kMoeMaxExperts = 512;
constexpr int kMoeMaxTopK = 32;
constexpr int kMoeMinBlocks = 4;  // K-blocks of a share at least, where there are as many: a share's fixed cost is
                                  // that of a few K-blocks

struct MoeSched {
    int T, D, F;
    int active;           // experts that some token chose
    int f_tiles;          // gate/up tiles per expert
    int kb1, kbf;         // K-blocks of a gate/up tile; of one expert in a down tile
    int d_tiles;
    long long u1, u2;     // K-blocks of each product
    int p1, p2;           // blocks that share them
};

BW_MOE_HD inline int moe_share_blocks(long long u, int grid)
{
    const long long want = u / kMoeMinBlocks;
    return want < 1 ? 1 : want < grid ? (int)want : grid;
}

BW_MOE_HD inline MoeSched moe_sched(int T, int D, int F, int active, int grid)
{
    MoeSched s;
    s.T = T;
    s.D = D;
    s.F = F;
    s.active = active;
    s.f_tiles = (F + 127) / 128;
    s.kb1 = D / 64;
    s.kbf = F / 64;
    s.d_tiles = (D + 255) / 256;
    s.u1 = (long long)active * s.f_tiles * s.kb1;
    s.u2 = (long long)s.d_tiles * active * s.kbf;
    s.p1 = moe_share_blocks(s.u1, grid);
    s.p2 = moe_share_blocks(s.u2, grid);
    return s;
}

BW_MOE_HD inline long long moe_begin(long long u, int p, int c) { return u * c / p; }
// The block whose share holds K-block g: the largest c with moe_begin(c) <= g.
BW_MOE_HD inline int moe_owner(long long u, int p, long long g) { return (int)(((g + 1) * p - 1) / u); }

struct MoeSeg {
    int phase;        // 0: gate/up, 1: down
    int tile, k0, k1; // K-blocks [k0, k1) of the tile
    int first, nseg;  // the first block that works on the tile, and how many do
};

// A block's segments in order: its share of the first product, then of the second.  In the first product its parts of
// split tiles come first (the one its share ends in, then the one it starts in), so that their sums and the waits for
// them hide behind the whole tiles; what the second product waits for at the end is one whole tile's epilogue.
struct MoeIter {
    long long begin, end;
    int phase, c, step, tile, tiles;  // step: 0 the end's part, 1 the start's part, 2 whole tiles
    BW_MOE_HD MoeIter(const MoeSched&, int c_) : begin(0), end(0), phase(-1), c(c_), step(3), tile(0), tiles(0) {}
    BW_MOE_HD bool next(const MoeSched& s, MoeSeg& seg)
    {
        for (;;) {
            if (step == 3) {
                if (++phase > 1) return false;
                const int p = phase ? s.p2 : s.p1;
                if (c >= p) continue;
                const long long u = phase ? s.u2 : s.u1;
                begin = moe_begin(u, p, c);
                end = moe_begin(u, p, c + 1);
                step = 0;
            }
            const int kb = phase ? s.active * s.kbf : s.kb1;
            const int t0 = (int)(begin / kb), t1 = (int)((end - 1) / kb);
            const int k0 = (int)(begin - (long long)t0 * kb), k1 = (int)(end - (long long)t1 * kb);
            const int at = step;
            if (step < 2) ++step;
            if (at == 0) {
                tile = k0 ? t0 + 1 : t0;                     // the whole tiles
                tiles = k1 == kb ? t1 + 1 - tile : t1 - tile;
                if (tiles < 0) tiles = 0;                    // (the share lies inside one tile)
                if (phase || k1 == kb || t0 == t1) continue; // no part of a tile at the end (or it is the start's too)
                set(s, seg, t1, 0, k1);
                return true;
            }
            if (at == 1) {
                if (t0 == t1 && (k0 || k1 < kb)) {
                    set(s, seg, t0, k0, k1);
                    return true;
                }
                if (!k0) continue;
                set(s, seg, t0, k0, kb);
                return true;
            }
            if (tiles > 0) {
                --tiles;
                set(s, seg, tile++, 0, kb);
                return true;
            }
            step = 3;
            if (phase && k1 < kb && t0 != t1) {
                set(s, seg, t1, 0, k1);
                return true;
            }
        }
    }
    BW_MOE_HD void set(const MoeSched& s, MoeSeg& seg, int t, int k0, int k1) const
    {
        const long long u = phase ? s.u2 : s.u1, kb = phase ? s.active * s.kbf : s.kb1;
        const int p = phase ? s.p2 : s.p1;
        seg.phase = phase;
        seg.tile = t;
        seg.k0 = k0;
        seg.k1 = k1;
        seg.first = moe_owner(u, p, t * kb);
        seg.nseg = moe_owner(u, p, (t + 1) * kb - 1) - seg.first + 1;
    }
};

// Block c's slot for its partial of a split tile: one for the tile its share of a product starts in, one for the tile
// it ends in (whole tiles in between need none), in each product.
BW_MOE_HD inline int moe_slot(const MoeSeg& seg, int c) { return 4 * c + 2 * seg.phase + (c == seg.first ? 1 : 0); }
// The counter of a split tile: a block is the first of at most one split tile in each product.
BW_MOE_HD inline int moe_counter(const MoeSeg& seg) { return 2 * seg.first + seg.phase; }

// The token-side operands of both products (X, and the activations h of each active expert) lie in the workspace as the
// MMA reads them: by K-blocks of 64 values, T rows of 128 bytes each, a row's 16-byte chunk c at c ^ (t % 8) (the 128-byte
// swizzle of the shared-memory descriptors), so that a stage's rows are one contiguous copy.
BW_MOE_HD inline long long moe_token_bytes(int T, int kb, int t, int chunk) { return ((long long)kb * T + t) * 128 + ((chunk ^ (t & 7)) << 4); }

// h goes to the down product as two values of the tokens' type, h rounded and what the rounding left, in two planes of the
// same layout, so that the layer's error is that of its one rounding of Y (rounded once, h would make it 1.4 times that).
// The planes are rows of one operand, each with accumulator columns of its own, so in fp16 they carry scales that keep h
// within its range: the first holds 2^-8 h (|h| up to 1.6e7), the second 2^3 times what that left (at most 2^12, so below
// 2^15), which leaves h off by 2^-23 of it or 2^-28, the larger.  bf16 has fp32's range: no scales, 2^-17 of h.
//   up to 8 tokens  the planes are rows 0 and 8 of the 16 that the MMA takes anyway: free
//   more            rows 0 and Tp (T rounded up to 16) of 2 Tp, one MMA of N = 2 Tp.  The tokens' intake of the down product
//                   doubles: 1 % of the layer's time at 16 tokens, 3 % at 33 and 64, 8 % at 128 against one value (under the
//                   power cap 4, 5 and 10 %).  (Two MMAs of N = Tp in its place: 13 to 18 %.)
BW_MOE_HD inline int moe_padded(int T) { return (T + 15) / 16 * 16; }
BW_MOE_HD inline int moe_plane_rows(int T) { return T <= 8 ? 8 : moe_padded(T); }
constexpr float kMoeHiScale = 0.00390625f, kMoeLoScale = 8.0f;  // fp16

// The workspace of a call on `grid` blocks (offsets in bytes): the chosen experts and their weights, X and the
// activations of the active experts, the partials, then the words that start at zero (a count of finished gate/up tiles per active
// expert, the split tiles' counters).
struct MoeWork {
    long long ids, weights, x, h, partials, zero, bytes;
    long long plane;  // bytes of one plane of h
    int slots, zero_words;
    long long slot_floats;
};
BW_MOE_HD inline long long moe_up(long long v) { return (v + 255) / 256 * 256; }
BW_MOE_HD inline MoeWork moe_work(int T, int E, int k, int D, int F, int grid)
{
    MoeWork w;
    w.slots = T * k < E ? T * k : E;
    w.slot_floats = 256LL * ((T + 3) / 4 * 4);
    w.ids = 0;
    w.weights = moe_up(w.ids + 4LL * T * k);
    w.x = moe_up(w.weights + 4LL * T * k);
    w.h = moe_up(w.x + 2LL * T * D);
    w.plane = 2LL * w.slots * T * F;
    w.partials = moe_up(w.h + 2 * w.plane);
    w.zero = moe_up(w.partials + 4LL * 4 * grid * w.slot_floats);
    w.zero_words = w.slots + 2 * grid;
    w.bytes = moe_up(w.zero + 4LL * w.zero_words);
    return w;
}

}  // namespace bw
