// grouped_sched.h -- how the products grouped by expert are cut into tiles and how the tiles are dealt out, on the device
// (the experts' numbers of rows are device data) and, for the tests, on the host.
//
// Expert e owns rows offsets[e] .. offsets[e + 1] - 1.  Its rows are cut evenly into runs of at most `cap` (a multiple of
// 32), its weight rows into tiles of 256 (a pair of SMs, 128 each).  The weights are the MMA's 256-row operand and the
// tokens its N, which a tile sets to its own number of tokens rounded up to 32: an expert's odd number of rows costs at
// most 31 columns, where a 256-row token tile would cost up to 255.
//
// Order: expert by expert; within one, weight tile by weight tile with up to 8 of its runs of tokens in turn, so that the
// runs share a weight tile while it is in L2 and the weight tiles a run of tokens.
//
// Dealing: with `tiles` tiles on P pairs, the first tiles % P are split along K over all pairs (the K-blocks of those
// tiles cut into P even ranges), then the others go whole to whichever pair asks next (a counter in global memory: tiles
// differ in their tokens; dealt out in turn, SMs were idle for a fifth of the time).  The parts of a split tile are summed by
// the last pair to finish it, in the order of K, so results repeat bit for bit.
#pragma once
#include <cstdint>

#ifdef __CUDACC__
#define BW_GS __host__ __device__ __forceinline__
#else
#define BW_GS inline
#endif

namespace bw {

constexpr int kGroupMax = 1024;      // experts
constexpr int kGroupRowTiles = 8;    // runs of tokens that share a weight tile in turn
// K-blocks: the shortest range a split tile is cut into (gradient of 64 x 64 rows, 1024 x 1024: 54 us with 2 and 4, 63 with 8)
constexpr int kGroupMinUnits = 4;

struct GroupSched {
    int nt;        // weight tiles per expert
    int kb;        // K-blocks per tile
    int pairs;     // pairs of SMs
    int tiles;     // all tiles
    int split;     // the first tiles, split along K
    int parts;     // pairs that take a range of them
};

BW_GS GroupSched group_sched(int nt, int kb, int pairs, int runs)
{
    GroupSched s;
    s.nt = nt;
    s.kb = kb;
    s.pairs = pairs;
    s.tiles = nt * runs;
    s.split = s.tiles % pairs;
    s.parts = s.split * kb / kGroupMinUnits;
    if (s.parts > pairs) s.parts = pairs;
    if (s.parts < s.split) s.parts = s.split;
    // a remainder that fills most of a wave goes in whole tiles (64 experts of 2048 x 2048 with 110 rows: 118 us, 122 split)
    if (s.tiles > pairs && s.split * 8 > pairs * 7) s.parts = s.split;
    return s;
}

// The runs of an expert's rows [a, b): their number, and the rows of each but the last (a multiple of 32).
BW_GS int group_runs(int a, int b, int cap) { return b > a ? (b - a + cap - 1) / cap : 0; }
BW_GS int group_run_rows(int a, int b, int runs) { return ((b - a + runs - 1) / runs + 31) / 32 * 32; }

// The first K-block (of split tile x kb) of part c, and the part that holds K-block u.  (Fewer than `pairs` tiles of at most
// 2^14 K-blocks are split into at most `pairs` parts: 32 bits hold the products, and divide in a quarter of the time.)
BW_GS int part_begin(const GroupSched& s, int c) { return (int)((unsigned)(s.split * s.kb) * (unsigned)c / (unsigned)s.parts); }
BW_GS int part_of(const GroupSched& s, int u)
{
    return (int)(((unsigned)(u + 1) * (unsigned)s.parts - 1u) / (unsigned)(s.split * s.kb));
}

struct GroupSeg {
    int tile;    // index in the order above
    int k0, k1;  // its K-blocks [k0, k1)
};

// A pair's segments in order: its range of the split tiles, then whole tiles.
struct GroupWalk {
    int u, uend;
    int tile;
    BW_GS GroupWalk(const GroupSched& s, int c)
    {
        u = uend = 0;
        if (s.split && c < s.parts) {
            u = part_begin(s, c);
            uend = part_begin(s, c + 1);
        }
        tile = s.split + c;
    }
    // its next range of a split tile
    BW_GS bool next_part(const GroupSched& s, GroupSeg& g)
    {
        if (u < uend) {
            g.tile = u / s.kb;
            g.k0 = u - g.tile * s.kb;
            const int end = (g.tile + 1) * s.kb;
            g.k1 = s.kb - (end > uend ? end - uend : 0);
            u = end > uend ? uend : end;
            return true;
        }
        return false;
    }
    static BW_GS void whole(const GroupSched& s, int tile, GroupSeg& g)
    {
        g.tile = tile;
        g.k0 = 0;
        g.k1 = s.kb;
    }
    // the same with the whole tiles dealt out in turn
    BW_GS bool next(const GroupSched& s, GroupSeg& g)
    {
        if (next_part(s, g)) return true;
        if (tile >= s.tiles) return false;
        whole(s, tile, g);
        tile += s.pairs;
        return true;
    }
};

// The parts of split tile t: [first, last]; part c's slot for it (a part's range touches at most two tiles).
BW_GS int tile_first_part(const GroupSched& s, int t) { return part_of(s, t * s.kb); }
BW_GS int tile_last_part(const GroupSched& s, int t) { return part_of(s, (t + 1) * s.kb - 1); }
BW_GS int part_slot(const GroupSched& s, int c, int t) { return 2 * c + (part_begin(s, c) / s.kb == t ? 0 : 1); }

// A tile's place in its expert: weight tile n and run m, of `runs` runs; j counts the expert's tiles.
BW_GS void group_place(int j, int nt, int runs, int& m, int& n)
{
    const int g = j / (kGroupRowTiles * nt);
    const int left = runs - g * kGroupRowTiles;
    const int rows = left < kGroupRowTiles ? left : kGroupRowTiles;
    const int r = j - g * kGroupRowTiles * nt;
    m = g * kGroupRowTiles + r % rows;
    n = r / rows;
}

// ------------------------------------------------------------------ the weights' gradient
// dW_e (N x K) in tiles of 256 rows x up to 256 columns; a tile's K-blocks are runs of 64 of expert e's rows (an expert without
// rows: one unit that only writes zeros).  Tiles in the order of experts, `per` each.  The experts' lengths differ, so the
// split tiles are dealt out by units (K-blocks): with up to two waves of tiles all of them, else the first tiles % pairs; the
// others whole, to whichever pair asks next, so that the pairs work on the same expert's rows at a time.  (8192 rows over 3
// experts of 2048 x 2048, 2.6 waves: 72 us, all split 78; 2048 over 2, 1.7 waves: all split 43, else 47.)
constexpr int kDwFewWaves = 2;

struct DwSched {
    int per, pairs, tiles, split, parts;
    long long units;  // of the split tiles
};
BW_GS int dw_blocks(int rows) { return rows > 0 ? (rows + 63) / 64 : 1; }

// cum[e]: units of one tile of each expert before e (so tile t of expert e begins at unit per cum[e] + t blocks_e).
BW_GS long long dw_tile_unit(const int* off, const int* cum, int per, int tile, int E)
{
    const int e = tile / per;
    if (e >= E) return (long long)per * cum[E];
    return (long long)per * cum[e] + (long long)(tile - e * per) * dw_blocks(off[e + 1] - off[e]);
}
BW_GS DwSched dw_sched(const int* off, const int* cum, int E, int per, int pairs)
{
    DwSched s;
    s.per = per;
    s.pairs = pairs;
    s.tiles = E * per;
    s.split = s.tiles <= kDwFewWaves * pairs ? s.tiles : s.tiles % pairs;
    s.units = dw_tile_unit(off, cum, per, s.split, E);
    long long parts = s.units / kGroupMinUnits;
    if (parts > pairs) parts = pairs;
    if (parts < 1) parts = 1;
    s.parts = (int)parts;
    return s;
}
BW_GS long long dw_begin(const DwSched& s, int c) { return s.units * c / s.parts; }
BW_GS int dw_part_of(const DwSched& s, long long u) { return (int)(((u + 1) * s.parts - 1) / s.units); }
// Part c's slot for a tile that begins at unit u0: a part's range cuts at most its first and its last tile.
BW_GS int dw_slot(const DwSched& s, int c, long long u0) { return 2 * c + (u0 <= dw_begin(s, c) ? 0 : 1); }

struct DwSeg {
    int tile, e, k0, k1, kb;  // K-blocks [k0, k1) of kb
    long long u0;             // the tile's first unit (split tiles)
};
struct DwWalk {
    long long u, uend;
    int tile, e;
    BW_GS DwWalk(const DwSched& s, int c)
    {
        u = uend = 0;
        if (s.split && c < s.parts) {
            u = dw_begin(s, c);
            uend = dw_begin(s, c + 1);
        }
        tile = s.split + c;
        e = 0;
    }
    BW_GS bool next_part(const DwSched& s, const int* off, const int* cum, DwSeg& g)
    {
        if (u < uend) {
            while ((long long)s.per * cum[e + 1] <= u) ++e;
            g.e = e;
            g.kb = dw_blocks(off[e + 1] - off[e]);
            const long long base = (long long)s.per * cum[e];
            const int i = (int)((u - base) / g.kb);
            g.tile = e * s.per + i;
            g.u0 = base + (long long)i * g.kb;
            g.k0 = (int)(u - g.u0);
            const long long end = g.u0 + g.kb;
            g.k1 = g.kb - (int)(end > uend ? end - uend : 0);
            u = end > uend ? uend : end;
            return true;
        }
        return false;
    }
    static BW_GS void whole(const DwSched& s, const int* off, int tile, DwSeg& g)
    {
        g.e = tile / s.per;
        g.kb = dw_blocks(off[g.e + 1] - off[g.e]);
        g.tile = tile;
        g.k0 = 0;
        g.k1 = g.kb;
        g.u0 = 0;
    }
};

}  // namespace bw
