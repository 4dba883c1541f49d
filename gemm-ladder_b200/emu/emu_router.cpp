// emu_router.cpp -- the host emulator over the mixture-of-experts router (test infrastructure; a build of its own with
// -DBW_EMU_THREADS=512, the kernel's block).  Clusters do not meet, so they run one after the other.
//
// C entry:
//   bw_emu_router(X, ldx, R, T, E, top_k, D, bf16, renormalize, ids, weights, XT, zero, zero_words, &findings, finding,
//                 len)     XT: 2 T D bytes
//   bw_emu_router_set(name, value): start_jitter_us, lead_skew_us
#include <future>
#include <string>
#include <thread>
#include <vector>

#include "moe_router.cuh"

namespace bw {
namespace {

template <bool BF16, int TG, int PER>
void run(const RouterParams& p)
{
    const int clusters = (p.T + TG - 1) / TG;
    emu::g_smem_limit = (int)sizeof(RouterSmem<kRouterTE * TG, 32 * PER>);
    for (int k = 0; k < clusters; ++k) {
        const unsigned seq = emu::g_launch_seq++;
        emu::Cluster cl;
        cl.size = kRouterBlocks;
        std::vector<std::unique_ptr<emu::Cta>> ctas;
        for (int r = 0; r < kRouterBlocks; ++r) {
            ctas.emplace_back(new emu::Cta());
            ctas.back()->rank = r;
            ctas.back()->cluster = &cl;
            cl.cta[r] = ctas.back().get();
        }
        std::vector<std::thread> threads;
        std::promise<void> gate;
        std::shared_future<void> open = gate.get_future().share();
        for (int r = 0; r < kRouterBlocks; ++r)
            for (int t = 0; t < emu::kCtaThreads; ++t)
                threads.emplace_back([&, k, r, t, open] {
                    open.wait();
                    emu::t_cta = ctas[(size_t)r].get();
                    emu::t_tid = t;
                    threadIdx = dim3((unsigned)t);
                    blockIdx = dim3((unsigned)(k * kRouterBlocks + r));
                    gridDim = dim3((unsigned)(clusters * kRouterBlocks));
                    blockDim = dim3((unsigned)emu::kCtaThreads);
                    emu::start_jitter((unsigned)r, seq);
                    if (emu::g_lead_skew_us > 0 && r == 0)
                        std::this_thread::sleep_for(std::chrono::microseconds(emu::g_lead_skew_us));
                    moe_router_kernel<BF16, TG, PER>(p);
                });
        gate.set_value();
        for (auto& th : threads) th.join();
    }
}
template <bool BF16>
void pick(const RouterParams& p)  // the library's choice of instance
{
    if (p.T <= 16)
        p.E <= 128 ? run<BF16, 1, 4>(p) : run<BF16, 1, 16>(p);
    else
        p.E <= 128 ? run<BF16, 4, 4>(p) : run<BF16, 4, 16>(p);
}

}  // namespace
}  // namespace bw

extern "C" __attribute__((visibility("default"))) int bw_emu_router_set(const char* name, long long value)
{
    using namespace bw::emu;
    const std::string n = name;
    if (n == "start_jitter_us") g_start_jitter_us = (int)value;
    else if (n == "lead_skew_us") g_lead_skew_us = (int)value;
    else return -1;
    return 0;
}

extern "C" __attribute__((visibility("default"))) int bw_emu_router(const uint16_t* X, long long ldx, const uint16_t* R,
                                                                    int T, int E, int top_k, int D, int bf16,
                                                                    int renormalize, int* ids, float* weights,
                                                                    uint8_t* XT, int* zero, int zero_words,
                                                                    int* findings, char* finding, int finding_len)
{
    using namespace bw;
    emu::g_findings = 0;
    emu::g_first_finding[0] = 0;
    const RouterParams p = {X, ldx, R, T, E, top_k, D, router_ranges(E), renormalize, XT, ids, weights, zero, zero_words};
    bf16 ? pick<true>(p) : pick<false>(p);
    if (findings) *findings = emu::g_findings.load();
    if (finding && finding_len > 0) snprintf(finding, (size_t)finding_len, "%s", emu::g_first_finding);
    return 0;
}
