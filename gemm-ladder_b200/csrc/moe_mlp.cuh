// moe_mlp.cuh -- host side of the mixture-of-experts layer (bw_moe_mlp of bwgemm.h), included by bwgemm.cu: argument
// checks, the tensor maps, the caller's workspace, the two launches.
#pragma once
#include "moe_kernel.cuh"
#include "moe_router.cuh"

namespace bw {
namespace {

// A 3-D row-major array of 16-bit values {d2}{d1}{d0}, boxes of 64 x rows x 1, 128-byte swizzle, zeros outside.
bool moe_map(CUtensorMap* m, const void* base, int bf16, uint64_t d0, uint64_t d1, uint64_t d2, uint64_t ld1, uint64_t ld2,
             uint32_t rows)
{
    EncodeTiled enc = encoder();
    if (!enc) return false;
    const cuuint64_t dims[3] = {d0, d1, d2};
    const cuuint64_t strides[2] = {ld1 * 2, ld2 * 2};
    const cuuint32_t box[3] = {64, rows, 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    return enc(m, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
               dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
int moe_shape(int T, int E, int top_k, int D, int F)
{
    if (T < 0 || T > kMoeMaxTokens || E < 1 || E > kMoeMaxExperts || top_k < 1 || top_k > kMoeMaxTopK || top_k > E)
        return BW_ERR_SHAPE;
    // a row's bytes and an expert's rows within the tensor maps' and the split's 32-bit indices
    if (D < 64 || F < 64 || D % 64 || F % 64 || D > (1 << 20) || F > (1 << 20)) return BW_ERR_SHAPE;
    return BW_OK;
}

// The blocks of the experts kernel: one per SM (its shared memory allows one).
int moe_grid(const DeviceState& d) { return d.sms; }

template <bool BF16, int TG>
void router_launch(const RouterParams& r, cudaStream_t st)
{
    const int grid = kRouterBlocks * ((r.T + TG - 1) / TG);
    if (r.E <= 128)
        moe_router_kernel<BF16, TG, 4><<<grid, kRouterThreads, 0, st>>>(r);
    else
        moe_router_kernel<BF16, TG, 16><<<grid, kRouterThreads, 0, st>>>(r);
}
// A token per cluster up to 16 tokens, where the clusters fit the GPU at once; 4 above, for the reuse of R.
template <bool BF16>
cudaError_t router_launch(const RouterParams& r, cudaStream_t st)
{
    if (r.T <= 16)
        router_launch<BF16, 1>(r, st);
    else
        router_launch<BF16, 4>(r, st);
    return cudaGetLastError();
}

int moe_mlp(const void* X, long long ldx, const void* R, const void* W1, const void* W2, void* Y, int T, int E, int top_k,
            int D, int F, int type, int renormalize, int* ids, float* weights, void* work, size_t work_bytes,
            cudaStream_t st)
{
    int rc = moe_shape(T, E, top_k, D, F);
    if (rc) return rc;
    if ((type != BW_TYPE_F16 && type != BW_TYPE_BF16) || (renormalize != 0 && renormalize != 1)) return BW_ERR_ARG;
    if (ldx < D || ldx % 8 || ldx > (1LL << 32)) return BW_ERR_SHAPE;
    if (T == 0) return BW_OK;
    if (!aligned(X, 16) || !aligned(R, 16) || !aligned(W1, 16) || !aligned(W2, 16) || !aligned(Y, 2) ||
        !aligned(work, 256) || (ids && !aligned(ids, 4)) || (weights && !aligned(weights, 4)))
        return BW_ERR_ARG;
    DeviceState* d = nullptr;
    if ((rc = device_state(&d))) return rc;
    const int grid = moe_grid(*d);
    const MoeWork w = moe_work(T, E, top_k, D, F, grid);
    if ((size_t)w.bytes > work_bytes) return scratch_fail((size_t)w.bytes, work_bytes);
    uint8_t* ws = static_cast<uint8_t*>(work);
    if (!ids) ids = reinterpret_cast<int*>(ws + w.ids);
    if (!weights) weights = reinterpret_cast<float*>(ws + w.weights);

    MoeParams p = {};
    p.T = T;
    p.Tp = moe_padded(T);
    p.E = E;
    p.top_k = top_k;
    p.D = D;
    p.F = F;
    p.bf16 = type == BW_TYPE_BF16;
    moe_rings(T, &p.stages, &p.slots);
    p.slot_bytes = moe_slot_bytes(T);
    p.ids = ids;
    p.weights = weights;
    p.W2 = static_cast<const uint16_t*>(W2);
    p.X = ws + w.x;
    p.H = ws + w.h;
    p.plane = w.plane;
    p.Y = static_cast<uint16_t*>(Y);
    p.partials = reinterpret_cast<float*>(ws + w.partials);
    p.slot_floats = w.slot_floats;
    p.ready = reinterpret_cast<int*>(ws + w.zero);
    p.counters = p.ready + w.slots;
    p.wait_ns = g_wait_ns;

    CUtensorMap m1, m2;
    if (!moe_map(&m1, W1, p.bf16, D, F, 2 * (uint64_t)E, D, (uint64_t)F * D, 128) ||
        !moe_map(&m2, W2, p.bf16, F, D, E, F, (uint64_t)F * D, 256)) {
        snprintf(g_errbuf, sizeof g_errbuf, "cuTensorMapEncodeTiled failed");
        return BW_ERR_LAUNCH;
    }
    cudaError_t e;
    static std::atomic<bool> limit_set[kMaxDevices];  // the kernel's shared-memory limit, once per device
    std::atomic<bool>& done = limit_set[d - g_dev];
    if (!done.load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(moe_experts_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BW_SMEM_LIMIT);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        done.store(true, std::memory_order_release);
    }

    RouterParams r = {static_cast<const uint16_t*>(X), ldx, static_cast<const uint16_t*>(R), T, E, top_k, D,
                      router_ranges(E), renormalize, ws + w.x, ids, weights, p.ready, w.zero_words};
    e = p.bf16 ? router_launch<true>(r, st) : router_launch<false>(r, st);
    if (e != cudaSuccess) return cuda_fail(e, "kernel launch (router)");

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(kMoeThreads);
    cfg.dynamicSmemBytes = (size_t)moe_smem_bytes(p);
    cfg.stream = st;
    // the blocks wait for one another, so all of them have to be resident.  (A cooperative launch does not overlap the
    // router's end: measured, programmatic serialisation has no effect on it; without the cooperative attribute it saves
    // 3.7 us a call, but then two overlapping calls could each hold SMs the other needs.)
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeCooperative;
    attr[0].val.cooperative = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, moe_experts_kernel, m1, m2, p);
    if (e != cudaSuccess) return cuda_fail(e, "kernel launch (experts)");
    return BW_OK;
}

}  // namespace
}  // namespace bw

BW_API int bw_moe_work_bytes(int T, int E, int top_k, int D, int F, size_t* bytes)
{
    using namespace bw;
    if (!bytes) return BW_ERR_ARG;
    *bytes = 0;
    int rc = moe_shape(T, E, top_k, D, F);
    if (rc || T == 0) return rc;
    DeviceState* d = nullptr;
    if ((rc = device_state(&d))) return rc;
    *bytes = (size_t)moe_work(T, E, top_k, D, F, moe_grid(*d)).bytes;
    return BW_OK;
}

BW_API int bw_moe_mlp(const void* X, long long ldx, const void* R, const void* W1, const void* W2, void* Y, int T, int E,
                      int top_k, int D, int F, int type, int renormalize, void* ids, void* weights, void* work,
                      size_t work_bytes, void* stream)
{
    return bw::moe_mlp(X, ldx, R, W1, W2, Y, T, E, top_k, D, F, type, renormalize, static_cast<int*>(ids),
                       static_cast<float*>(weights), work, work_bytes, static_cast<cudaStream_t>(stream));
}
