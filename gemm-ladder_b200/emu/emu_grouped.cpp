// emu_grouped.cpp -- the host emulator over the grouped kernels (test infrastructure; a build of its own with
// -DBW_EMU_THREADS=384, the kernels' block).
//
// C entries:
//   bw_emu_grouped(X, ldx, xs, xs_ld, W, ws, offsets, C, E, T, N, K, pairs, kind, bf16, mn_major, glu, out, cap, stages,
//                  status[4], &dirty, &findings, finding, len)
//   bw_emu_grouped_dw(dY, ldy, X, ldx, offsets, dW, E, T, N, K, pairs, bf16, out, stages, status[4], &findings, finding, len)
//   bw_emu_grouped_set(name, value): wait_ns, drop_tma, engine_delay_us, start_jitter_us, lead_skew_us, ld_delay_us
#include <future>
#include <string>
#include <thread>
#include <vector>

#include "grouped_plan.h"

namespace bw {
namespace {

void map3(CUtensorMap* m, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1, uint64_t s2, uint32_t rows)
{
    const uint64_t dims[3] = {d0, d1, d2}, strides[3] = {2, s1 * 2, s2 * 2};
    const uint32_t box[3] = {64, rows, 1};
    emu::make_map(m, base, 3, dims, strides, box);
}

// Every cluster of the grid at once, `pairs` of them.
template <class F>
void launch_pairs(int pairs, int smem_bytes, F kernel)
{
    emu::g_smem_limit = smem_bytes;
    const unsigned seq = emu::g_launch_seq++;
    std::vector<std::unique_ptr<emu::Cta>> ctas;
    std::vector<std::unique_ptr<emu::Cluster>> clusters;
    for (int c = 0; c < pairs; ++c) {
        clusters.emplace_back(new emu::Cluster());
        clusters.back()->size = 2;
        for (int r = 0; r < 2; ++r) {
            ctas.emplace_back(new emu::Cta());
            ctas.back()->rank = r;
            ctas.back()->cluster = clusters.back().get();
            clusters.back()->cta[r] = ctas.back().get();
        }
    }
    std::vector<std::thread> threads;
    std::promise<void> gate;
    std::shared_future<void> open = gate.get_future().share();
    for (int b = 0; b < 2 * pairs; ++b)
        for (int t = 0; t < emu::kCtaThreads; ++t)
            threads.emplace_back([&, b, t, open] {
                open.wait();
                emu::t_cta = ctas[(size_t)b].get();
                emu::t_tid = t;
                emu::t_met = false;
                threadIdx = dim3((unsigned)t);
                blockIdx = dim3((unsigned)b);
                gridDim = dim3((unsigned)(2 * pairs));
                blockDim = dim3((unsigned)emu::kCtaThreads);
                emu::start_jitter((unsigned)b, seq);
                if (emu::g_lead_skew_us > 0 && b % 2 == 0)
                    std::this_thread::sleep_for(std::chrono::microseconds(emu::g_lead_skew_us));
                kernel();
                emu::t_cta->left.fetch_add(1);
            });
    gate.set_value();
    for (auto& th : threads) th.join();
    for (auto& c : ctas) {
        c->tma.finish();
        c->tc.finish();
    }
}

void begin()
{
    emu::g_findings = 0;
    emu::g_first_finding[0] = 0;
    emu::g_tma_count = 0;
    std::memset(g_status, 0, sizeof g_status);
}
void end(unsigned* status, int* findings, char* finding, int len)
{
    if (status) std::memcpy(status, g_status, sizeof g_status);
    if (findings) *findings = emu::g_findings.load();
    if (finding && len > 0) snprintf(finding, (size_t)len, "%s", emu::g_first_finding);
}

}  // namespace
}  // namespace bw

#define EMU_API extern "C" __attribute__((visibility("default")))

EMU_API int bw_emu_grouped_set(const char* name, long long value)
{
    using namespace bw::emu;
    const std::string n = name;
    if (n == "wait_ns") g_wait_ns = (unsigned long long)value;
    else if (n == "drop_tma") g_drop_tma = value;
    else if (n == "engine_delay_us") g_engine_delay_us = (int)value;
    else if (n == "start_jitter_us") g_start_jitter_us = (int)value;
    else if (n == "lead_skew_us") g_lead_skew_us = (int)value;
    else if (n == "ld_delay_us") g_ld_delay_us = (int)value;
    else return -1;
    return 0;
}

EMU_API int bw_emu_grouped(const void* X, long long ldx, const float* xs, long long xs_ld, const void* W, const float* ws,
                           const int* offsets, void* C, int E, int T, int N, int K, int pairs, int kind, int bf16,
                           int mn_major, int glu, int out, int cap, int stages, unsigned* status, int* dirty, int* findings,
                           char* finding, int len)
{
    using namespace bw;
    begin();
    GxParams p = gx_params(E, T, N, K, GxForm{kind, cap}, bf16, mn_major, glu, out);
    if (stages && stages < p.stages) {
        p.stages = stages;
        p.ring_bytes = stages * p.stage_bytes;
    }
    p.offsets = offsets, p.C = C, p.xs = xs, p.xs_ld = xs_ld, p.ws = ws;
    std::vector<float> work(gx_work_bytes(pairs, p.cap) / 4, NAN);
    std::vector<int> counters(2 * (size_t)pairs + 1, 0);
    p.work = work.data(), p.counters = counters.data(), p.next = p.counters + 2 * pairs;
    p.wait_ns = emu::g_wait_ns;
    CUtensorMap mw, mx;
    const GxMaps m = gx_maps(p, K, ldx, kind != kGx16);
    map3(&mw, W, m.w[0], m.w[1], m.w[2], m.w[3], m.w[4], (uint32_t)m.w[5]);
    map3(&mx, X, m.x[0], m.x[1], m.x[2], m.x[3], m.x[4], (uint32_t)m.x[5]);
    launch_pairs(pairs, gx_smem(kind, p.ring_bytes, p.E).bytes, [&] {
        if (kind == kGxF8Weights)
            grouped_kernel<kGxF8Weights>(mw, mx, p);
        else if (kind == kGxF8Tokens)
            grouped_kernel<kGxF8Tokens>(mw, mx, p);
        else
            grouped_kernel<kGx16>(mw, mx, p);
    });
    (void)dirty;
    end(status, findings, finding, len);
    return 0;
}

EMU_API int bw_emu_grouped_dw(const void* dY, long long ldy, const void* X, long long ldx, const int* offsets, void* dW, int E,
                              int T, int N, int K, int pairs, int bf16, int out, int stages, unsigned* status, int* findings,
                              char* finding, int len)
{
    using namespace bw;
    begin();
    DwParams p = dw_params(E, T, N, K, bf16, out);
    if (stages && stages < p.stages) {
        p.stages = stages;
        p.ring_bytes = stages * kDwStageBytes;
    }
    p.offsets = offsets, p.dW = dW;
    std::vector<float> work(gx_work_bytes(pairs, 256) / 4, NAN);
    std::vector<int> counters((size_t)dw_counters(p, pairs), 0);
    p.work = work.data(), p.counters = counters.data(), p.next = p.counters + counters.size() - 1;
    p.wait_ns = emu::g_wait_ns;
    CUtensorMap my, mx;
    map3(&my, dY, (uint64_t)N, (uint64_t)T, 1, (uint64_t)ldy, (uint64_t)ldy * T, 64);
    map3(&mx, X, (uint64_t)K, (uint64_t)T, 1, (uint64_t)ldx, (uint64_t)ldx * T, 64);
    launch_pairs(pairs, dw_smem(p.ring_bytes, p.E).bytes, [&] { grouped_dw_kernel(my, mx, p); });
    end(status, findings, finding, len);
    return 0;
}
