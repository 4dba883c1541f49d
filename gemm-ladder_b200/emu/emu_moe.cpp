// emu_moe.cpp -- the host emulator over the mixture-of-experts kernel (test infrastructure; a build of its own with
// -DBW_EMU_THREADS=352, the kernel's block).  The blocks wait for one another, so every block of the grid runs at once,
// as the library's cooperative launch has it; the router is given (ids, weights).
//
// C entry:
//   bw_emu_moe(X, ldx, W1, W2, Y, ids, weights, T, E, top_k, D, F, grid, bf16, status[4], &findings, finding, len)
//   bw_emu_moe_set(name, value): wait_ns, drop_tma, drop_bulk, drop_red, drop_atom, first_kind (emu_runtime.h), engine_delay_us, start_jitter_us, block_ramp_us, ld_delay_us
#include <future>
#include <string>
#include <thread>
#include <vector>

#include "moe_kernel.cuh"

namespace bw {
namespace {

void map3(CUtensorMap* m, const void* base, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t s1, uint64_t s2, uint32_t rows)
{
    const uint64_t dims[3] = {d0, d1, d2}, strides[3] = {2, s1 * 2, s2 * 2};
    const uint32_t box[3] = {64, rows, 1};
    emu::make_map(m, base, 3, dims, strides, box);
}

}  // namespace
}  // namespace bw

extern "C" __attribute__((visibility("default"))) int bw_emu_moe_set(const char* name, long long value)
{
    using namespace bw::emu;
    const std::string n = name;
    if (n == "wait_ns") g_wait_ns = (unsigned long long)value;
    else if (n == "drop_tma") g_drop_tma = value;
    else if (n == "engine_delay_us") g_engine_delay_us = (int)value;
    else if (n == "start_jitter_us") g_start_jitter_us = (int)value;
    else if (n == "block_ramp_us") g_block_ramp_us = (int)value;
    else if (n == "ld_delay_us") g_ld_delay_us = (int)value;
    else if (n == "first_kind") g_first_kind = (int)value;
    else if (n == "drop_bulk") g_drop_nth[kDropBulk] = value, g_drop_count[kDropBulk] = 0;
    else if (n == "drop_red") g_drop_nth[kDropRed] = value, g_drop_count[kDropRed] = 0;
    else if (n == "drop_atom") g_drop_nth[kDropAtom] = value, g_drop_count[kDropAtom] = 0;
    else return -1;
    return 0;
}

extern "C" __attribute__((visibility("default"))) int bw_emu_moe(const uint16_t* X, long long ldx, const uint16_t* W1,
                                                                 const uint16_t* W2, uint16_t* Y, const int* ids,
                                                                 const float* weights, int T, int E, int top_k, int D,
                                                                 int F, int grid, int bf16, unsigned* status,
                                                                 int* findings, char* finding, int finding_len)
{
    using namespace bw;
    emu::g_findings = 0;
    emu::g_first_finding[0] = 0;
    emu::g_tma_count = 0;
    std::memset(g_status, 0, sizeof g_status);
    const MoeWork w = moe_work(T, E, top_k, D, F, grid);
    std::vector<uint8_t> work((size_t)w.bytes + 256, 0xFF);  // NaN: what the kernel does not write shows
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(work.data()) + 255) & ~uintptr_t(255));
    std::memset(base + w.zero, 0, 4 * (size_t)w.zero_words);
    MoeParams p = {};
    p.T = T, p.Tp = moe_padded(T), p.E = E, p.top_k = top_k, p.D = D, p.F = F, p.bf16 = bf16;
    moe_rings(T, &p.stages, &p.slots);
    p.slot_bytes = moe_slot_bytes(T);
    p.ids = ids, p.weights = weights;
    p.W2 = W2;
    p.X = base + w.x, p.H = base + w.h, p.plane = w.plane, p.Y = Y;
    for (int t = 0; t < T; ++t)  // the router's layout of the tokens
        for (int c = 0; c < D / 8; ++c)
            std::memcpy(base + w.x + moe_token_bytes(T, c >> 3, t, c & 7), X + t * ldx + 8 * c, 16);
    p.partials = reinterpret_cast<float*>(base + w.partials), p.slot_floats = w.slot_floats;
    p.ready = reinterpret_cast<int*>(base + w.zero), p.counters = p.ready + w.slots;
    p.wait_ns = emu::g_wait_ns;
    CUtensorMap m1, m2;
    map3(&m1, W1, D, F, 2 * (uint64_t)E, D, (uint64_t)F * D, 128);
    map3(&m2, W2, F, D, E, F, (uint64_t)F * D, 256);
    emu::g_smem_limit = moe_smem_bytes(p) - 1024;
    const unsigned seq = emu::g_launch_seq++;
    std::vector<std::unique_ptr<emu::Cta>> ctas;
    for (int b = 0; b < grid; ++b) ctas.emplace_back(new emu::Cta());
    std::vector<std::thread> threads;
    std::promise<void> gate;
    std::shared_future<void> open = gate.get_future().share();
    for (int b = 0; b < grid; ++b)
        for (int t = 0; t < emu::kCtaThreads; ++t)
            threads.emplace_back([&, b, t, open] {
                open.wait();
                emu::t_cta = ctas[(size_t)b].get();
                emu::t_tid = t;
                threadIdx = dim3((unsigned)t);
                blockIdx = dim3((unsigned)b);
                gridDim = dim3((unsigned)grid);
                blockDim = dim3((unsigned)emu::kCtaThreads);
                emu::start_jitter((unsigned)b, seq);
                if (emu::g_block_ramp_us > 0)
                    std::this_thread::sleep_for(std::chrono::microseconds((long long)emu::g_block_ramp_us * b));
                moe_experts_kernel(m1, m2, p);
            });
    gate.set_value();
    for (auto& th : threads) th.join();
    for (auto& c : ctas) {
        c->tma.finish();
        c->tc.finish();
    }
    if (status) std::memcpy(status, g_status, sizeof g_status);
    if (findings) *findings = emu::g_findings.load();
    if (finding && finding_len > 0) snprintf(finding, (size_t)finding_len, "%s", emu::g_first_finding);
    return 0;
}
