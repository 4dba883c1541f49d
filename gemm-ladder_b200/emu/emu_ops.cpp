// emu_ops.cpp -- the host emulator over the 8-bit integer kernels (test infrastructure): emu.cpp's launcher with the
// instances and plans of csrc/gemm_i8.cuh.
//
// C entry:
//   bw_emu_gemm_i8(A, a_scale, B, b_scale, C, M, N, K, sms, out_type, swiglu, status[4], &dirty, &findings, finding, len)
#include "emu.cpp"

namespace bw {
namespace {

template <int EPI, int WM>
int launch_i8_swap(const bw_plan& q, const CUtensorMap& mx, const CUtensorMap& my, const Params& p)
{
    switch (q.bn) {
    case 16: return launch<16, true, false, EPI, WM>(q, mx, my, mx, p);
    case 32: return launch<32, true, false, EPI, WM>(q, mx, my, mx, p);
    case 48: return launch<48, true, false, EPI, WM>(q, mx, my, mx, p);
    case 64: return launch<64, true, false, EPI, WM>(q, mx, my, mx, p);
    case 80: return launch<80, true, false, EPI, WM>(q, mx, my, mx, p);
    case 96: return launch<96, true, false, EPI, WM>(q, mx, my, mx, p);
    case 112: return launch<112, true, false, EPI, WM>(q, mx, my, mx, p);
    case 128: return launch<128, true, false, EPI, WM>(q, mx, my, mx, p);
    default: return BW_ERR_ARG;
    }
}

int dispatch_i8(const bw_plan& q, const CUtensorMap& mx, const CUtensorMap& my, const Params& p, int epi)
{
    if (q.kernel == BW_KERNEL_PAIR) {
        if (epi == kEpiI8F32) return launch<256, false, true, kEpiI8F32, 1>(q, mx, my, mx, p);
        if (epi == kEpiI8SwiGLU) return launch<256, false, true, kEpiI8SwiGLU, 1>(q, mx, my, mx, p);
        if (q.bn == 512) return launch<512, false, true, kEpiI8, 1>(q, mx, my, mx, p);
        return launch<256, false, true, kEpiI8, 1>(q, mx, my, mx, p);
    }
    if (q.kernel == BW_KERNEL_TILE) return launch<128, false, false, kEpiI8, 1>(q, mx, my, mx, p);
    if (epi == kEpiI8SwiGLU) return launch_i8_swap<kEpiI8SwiGLU, 2>(q, mx, my, p);
    return q.wm == 2 ? launch_i8_swap<kEpiI8, 2>(q, mx, my, p) : launch_i8_swap<kEpiI8, 1>(q, mx, my, p);
}

}  // namespace
}  // namespace bw

extern "C" __attribute__((visibility("default"))) int bw_emu_gemm_i8(const void* A, const float* a_scale, const void* B,
                                                                     const float* b_scale, void* C, int M, int N,
                                                                     int K, int sms, int out_type, int swiglu,
                                                                     unsigned* status, int* dirty, int* findings,
                                                                     char* finding, int finding_len)
{
    using namespace bw;
    emu::g_findings = 0;
    emu::g_first_finding[0] = 0;
    emu::g_tma_count = 0;
    std::memset(g_status, 0, sizeof g_status);
    const int epi = swiglu ? kEpiI8SwiGLU : out_type == BW_TYPE_F32 ? kEpiI8F32 : kEpiI8;
    const unsigned flags = epi == kEpiI8F32      ? kPlanNoSwap | kPlanI8
                           : epi == kEpiI8SwiGLU ? kPlanGateUp | kPlanI8 | (M > 128 ? kPlanNoSplit : 0u)
                                                 : kPlanI8;
    bw_plan q = {};
    int rc = make_plan(M, N, (K + 127) / 128 * 64, sms, sms / 2, 0, &q, flags);
    if (rc) return rc;
    std::vector<float> work(q.workspace_bytes / sizeof(float) + 4, 0.f);
    std::vector<int> counters((size_t)q.counters + 1, 0);
    CUtensorMap mx, my;
    make_maps(q, A, B, M, N, K / 2, &mx, &my, true);
    Params p = make_params(q, M, N, q.kblocks * 64, C, work.data(), counters.data(), true);
    i8_params(p, a_scale, b_scale, out_type == BW_TYPE_BF16, M % 2 != 0);  // (both orders of the first loads)
    // bw_linear_i8: the quantiser writes the row scales; with BWGEMM_PDL=1 one ahead of bw_gemm_i8 may write either
    emu::g_ahead[0][0] = a_scale, emu::g_ahead[0][1] = a_scale + M;
    emu::g_ahead[1][0] = b_scale, emu::g_ahead[1][1] = b_scale + N;
    rc = dispatch_i8(q, mx, my, p, epi);
    if (status) std::memcpy(status, g_status, sizeof g_status);
    if (dirty) *dirty = (int)std::count_if(counters.begin(), counters.begin() + q.counters, [](int v) { return v != 0; });
    if (findings) *findings = emu::g_findings.load();
    if (finding && finding_len > 0) snprintf(finding, (size_t)finding_len, "%s", emu::g_first_finding);
    return rc;
}
