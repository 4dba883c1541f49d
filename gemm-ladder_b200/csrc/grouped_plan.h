// grouped_plan.h -- host side arithmetic of the grouped kernels, shared by the library and the emulator: the token tile,
// the stage ring, the workspace, the tensor maps' sizes.
#pragma once
#include "grouped_dw.cuh"

namespace bw {

// The form of a call and the most tokens of a tile, for an average of `rows` tokens per expert.
struct GxForm {
    int kind, cap;
};
inline GxForm gx_form(int T, int E, bool grouped, bool f8)
{
    const long long rows = grouped ? ((long long)T + E - 1) / E : T;
    // e4m3, the tokens as M: measured, 32 experts of 4096 x 4096 with 32 / 64 / 128 rows each in 188 / 190 / 190 us against
    // 133 / 194 / 238 with the weights as M; one matrix of 8192 x 8192 at 128 / 160 tokens in 55 / 55 against 49 / 59
    if (f8 && rows > (grouped ? 48 : 128)) return {kGxF8Tokens, 256};
    // fp16 and bf16: a tile's MMA is as wide as the tokens it has, and a smaller cap, for more stages of weights, gained nothing
    // (64 experts of 2048 x 2048 with 28 rows each in 108 us with 64 and with 256, 8 of 4096 x 4096 with 20 in 66 with both)
    if (!f8) return {kGx16, 256};
    // e4m3, the weights as M: the smaller the cap, the more K-blocks are handed over at once (17 tokens, 8192 x 8192: 31 us with 32,
    // 35 with 128).  Experts' numbers of rows spread around the average: twice it, so that most take one run.
    const long long want = grouped ? 2 * rows : rows;
    return {kGxF8Weights, want <= 32 ? 32 : want <= 64 ? 64 : 128};
}

// Everything of a call but its addresses.
inline GxParams gx_params(int E, int T, int N, int K, GxForm form, bool bf16, bool mn_major, int glu, int out)
{
    const bool f8 = form.kind != kGx16, tokens = form.kind == kGxF8Tokens;
    GxParams p = {};
    p.E = E;
    p.T = T;
    p.N = N;
    p.Nout = glu == kGxPlain ? N : N / 2;
    p.nt = glu == kGxGluHalves ? (N / 2 + 127) / 128 : (N + 255) / 256;
    p.kblocks = f8 ? (K + 127) / 128 : (K + 63) / 64;
    p.cap = form.cap;
    p.box = tokens ? 128 : p.cap == 32 ? 16 : 32;
    p.wbox = glu == kGxPlain || tokens ? 128 : 64;
    // short tiles: more of them planned ahead, to keep the stage ring full (16 experts of 8192 x 256 with 100 rows each: 31.8 us,
    // 35.8 with two); long ones: two, since a tile planned ahead cannot go to a pair that is done earlier (64 of 2048 x 2816 with
    // 256 rows: 186 us, 190 with four)
    p.descs = p.kblocks < 8 ? kGxDescs : 2;
    p.group = form.kind == kGxF8Weights ? 128 / p.cap : 1;
    p.accs = 512 / (p.cap * p.group) < kGxAccs ? 512 / (p.cap * p.group) : kGxAccs;
    p.stage_bytes = kGxXBytes + p.cap / 2 * 128;
    const int fixed = gx_smem(form.kind, 0, E).bytes + 1024;
    p.stages = (BW_SMEM_LIMIT - fixed) / p.stage_bytes;
    if (p.stages > kGxMaxStages) p.stages = kGxMaxStages;
    p.ring_bytes = p.stages * p.stage_bytes;
    p.mn_major = mn_major ? 1 : 0;
    p.glu = glu;
    p.out = out;
    p.idesc = f8 ? idesc_e4m3_f32_m(256) : idesc_16_f32_m(256, bf16, mn_major, false);
    p.ws_rows = (N + 127) / 128;
    return p;
}

// Parts of split tiles: two slots per pair, each of both blocks' 128 rows x cap fp32.
inline size_t gx_work_bytes(int pairs, int cap) { return (size_t)pairs * 2 * 2 * 128 * (size_t)cap * 4; }

// The tensor maps in 16-bit elements (two e4m3 each): {d0, d1, d2, row stride, plane stride, box rows}, boxes of 64 x rows.
struct GxMaps {
    uint64_t w[6], x[6];
};
inline GxMaps gx_maps(const GxParams& p, int K, long long ldx, bool f8)
{
    const uint64_t k = f8 ? (uint64_t)K / 2 : (uint64_t)K, ld = f8 ? (uint64_t)ldx / 2 : (uint64_t)ldx;
    GxMaps m;
    const uint64_t n = (uint64_t)p.N, e = (uint64_t)p.E;
    if (p.mn_major) {
        const uint64_t w[6] = {n, k, e, n, n * k, 64};
        for (int i = 0; i < 6; ++i) m.w[i] = w[i];
    } else {
        const uint64_t w[6] = {k, n, e, k, n * k, (uint64_t)p.wbox};
        for (int i = 0; i < 6; ++i) m.w[i] = w[i];
    }
    const uint64_t x[6] = {k, (uint64_t)p.T, 1, ld, ld * (uint64_t)p.T, (uint64_t)p.box};
    for (int i = 0; i < 6; ++i) m.x[i] = x[i];
    return m;
}

// The weights' gradient: everything of a call but its addresses.
inline DwParams dw_params(int E, int T, int N, int K, bool bf16, int out)
{
    DwParams p = {};
    p.E = E;
    p.T = T;
    p.N = N;
    p.K = K;
    p.tn = (N + 255) / 256;
    p.tk = (K + 255) / 256;
    p.width = ((K + p.tk - 1) / p.tk + 31) / 32 * 32;
    p.stages = (BW_SMEM_LIMIT - 1024 - dw_smem(0, E).bytes) / kDwStageBytes;
    if (p.stages > kDwMaxStages) p.stages = kDwMaxStages;
    p.ring_bytes = p.stages * kDwStageBytes;
    p.out = out;
    p.idesc = idesc_16_f32_m(256, bf16, true, true);
    return p;
}
// (two counters per split tile, and the number of whole tiles given out)
inline int dw_counters(const DwParams& p, int pairs)
{
    const long long tiles = (long long)p.E * p.tn * p.tk;
    return 2 * (int)(tiles <= kDwFewWaves * pairs ? tiles : tiles % pairs) + 1;
}

}  // namespace bw
