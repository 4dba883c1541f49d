// grouped.cuh -- host side of the products grouped by expert and in 8-bit floating point (bw_gemm_grouped,
// bw_gemm_grouped_dw, bw_quant_f8, bw_quant_blocks_f8, bw_gemm_f8, bw_linear_f8 of bwgemm.h), included by bwgemm.cu:
// argument checks, the tensor maps, the caller's workspace, the launches.
#pragma once
#include "grouped_plan.h"
#include "quant_f8.cuh"

namespace bw {
namespace {

// Sizes within the tensor maps' and the schedule's 32-bit indices.
bool gx_sizes_ok(int E, int T, int N, int K)
{
    if (E < 1 || E > kGroupMax || T < 0 || T > (1 << 30) || N < 1 || K < 1 || N > (1 << 20) || K > (1 << 20)) return false;
    return ((long long)T / 32 + E) * ((N + 255) / 256) < (1LL << 30) && (long long)E * N <= 0x7FFFFFFFLL;
}

// Pairs of SMs a call runs on.
int gx_pairs(DeviceState& d, int* pairs)
{
    std::lock_guard<std::mutex> lock(g_mu);
    int rc = pair_occupancy(d);
    if (rc) return rc;
    if (d.pairs < 1) {
        snprintf(g_errbuf, sizeof g_errbuf, "this device holds no pairs of SMs");
        return BW_ERR_LAUNCH;
    }
    *pairs = d.pairs;
    return BW_OK;
}

// The workspace of a call: [linear: quantised rows, their scales][parts of split tiles][their counters].
struct GxWork {
    size_t q, scale, parts, counters, bytes;
    long long lds;
    int n_counters;
};
GxWork gx_work(int T, int K, int cap, int pairs, bool linear)
{
    GxWork w = {};
    size_t at = 0;
    if (linear) {
        w.lds = ((long long)T + 3) / 4 * 4;
        at = up256((size_t)T * K);
        w.scale = at;
        at = up256(at + (size_t)w.lds * ((K + 127) / 128) * sizeof(float));
    }
    w.parts = at;
    at = up256(at + gx_work_bytes(pairs, cap));
    w.counters = at;
    w.n_counters = 2 * pairs + 1;
    w.bytes = up256(at + (size_t)w.n_counters * sizeof(int));
    return w;
}

// A kernel on pairs of SMs, overlapping with the one ahead of it on the stream, which is the call's own and launched in plain
// stream order.
template <class P>
int launch_pairs(DeviceState& d, void (*kernel)(CUtensorMap, CUtensorMap, P), std::atomic<bool>* limit_set, const CUtensorMap& m0,
                 const CUtensorMap& m1, const P& p, int pairs, int smem, cudaStream_t st)
{
    std::atomic<bool>& done = limit_set[&d - g_dev];  // the kernel's shared-memory limit, once per device
    cudaError_t e;
    if (!done.load(std::memory_order_acquire)) {
        e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, BW_SMEM_LIMIT);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        done.store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(2 * pairs));
    cfg.blockDim = dim3(kGxThreads);
    cfg.dynamicSmemBytes = (size_t)(1024 + smem);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    e = cudaLaunchKernelEx(&cfg, kernel, m0, m1, p);
    return e == cudaSuccess ? BW_OK : cuda_fail(e, "kernel launch (grouped)");
}
int zero_counters(int* counters, int n, cudaStream_t st)
{
    gx_zero_kernel<<<1, 256, 0, st>>>(counters, n);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? BW_OK : cuda_fail(e, "kernel launch (counters)");
}

template <int KIND>
int gx_launch(DeviceState& d, const GxParams& p, const CUtensorMap& mw, const CUtensorMap& mx, int pairs, cudaStream_t st)
{
    static std::atomic<bool> limit_set[kMaxDevices];
    return launch_pairs(d, grouped_kernel<KIND>, limit_set, mw, mx, p, pairs, gx_smem(KIND, p.ring_bytes, p.E).bytes, st);
}

// The product of p (its addresses but the workspace's filled in); zeroed: the kernel ahead of it on the stream, one of the
// call's own launched in plain order, zeroes the counters.
int gx_product(DeviceState& d, GxParams& p, const GxForm& form, const GxMaps& m, const void* X, const void* W,
               const GxWork& w, uint8_t* work, int pairs, bool zeroed, cudaStream_t st)
{
    p.work = reinterpret_cast<float*>(work + w.parts);
    p.counters = reinterpret_cast<int*>(work + w.counters);
    p.next = p.counters + 2 * pairs;
    p.wait_ns = g_wait_ns;
    CUtensorMap mw, mx;
    if (!moe_map(&mw, W, 0, m.w[0], m.w[1], m.w[2], m.w[3], m.w[4], (uint32_t)m.w[5]) ||
        !moe_map(&mx, X, 0, m.x[0], m.x[1], m.x[2], m.x[3], m.x[4], (uint32_t)m.x[5])) {
        snprintf(g_errbuf, sizeof g_errbuf, "cuTensorMapEncodeTiled failed");
        return BW_ERR_LAUNCH;
    }
    if (!zeroed) {
        const int rc = zero_counters(p.counters, w.n_counters, st);
        if (rc) return rc;
    }
    switch (form.kind) {
    case kGxF8Tokens: return gx_launch<kGxF8Tokens>(d, p, mw, mx, pairs, st);
    case kGxF8Weights: return gx_launch<kGxF8Weights>(d, p, mw, mx, pairs, st);
    default: return gx_launch<kGx16>(d, p, mw, mx, pairs, st);
    }
}

int grouped_check(int E, int M, int N, int K, int layout, int swiglu)
{
    if ((layout != BW_LAYOUT_KN && layout != BW_LAYOUT_NK) || (swiglu != 0 && swiglu != 1) ||
        (swiglu && layout != BW_LAYOUT_NK))
        return BW_ERR_ARG;
    if (!gx_sizes_ok(E, M, N, K) || N % 8 || K % 8 || (swiglu && N % 16)) return BW_ERR_SHAPE;
    return BW_OK;
}

int gemm_grouped(const void* X, long long ldx, const void* B, const int* offsets, void* C, int E, int M, int N, int K,
                 int type, int layout, int swiglu, void* work, size_t work_bytes, cudaStream_t st)
{
    if (type != BW_TYPE_F16 && type != BW_TYPE_BF16) return BW_ERR_ARG;
    int rc = grouped_check(E, M, N, K, layout, swiglu);
    if (rc) return rc;
    if (ldx < K || ldx % 8 || ldx > (1LL << 32)) return BW_ERR_SHAPE;
    if (M == 0) return BW_OK;
    if (!aligned(X, 16) || !aligned(B, 16) || !aligned(C, 16) || !aligned(offsets, 4) || !aligned(work, 256)) return BW_ERR_ARG;
    DeviceState* d = nullptr;
    int pairs = 0;
    if ((rc = device_state(&d)) || (rc = gx_pairs(*d, &pairs))) return rc;
    const GxForm form = gx_form(M, E, true, false);
    const GxWork w = gx_work(M, K, form.cap, pairs, false);
    if (w.bytes > work_bytes) return scratch_fail(w.bytes, work_bytes);
    GxParams p = gx_params(E, M, N, K, form, type == BW_TYPE_BF16, layout == BW_LAYOUT_KN, swiglu ? kGxGluHalves : kGxPlain,
                           type);
    p.offsets = offsets;
    p.C = C;
    return gx_product(*d, p, form, gx_maps(p, K, ldx, false), X, B, w, static_cast<uint8_t*>(work), pairs, false, st);
}

int dw_check(int E, int M, int N, int K, int out_type)
{
    if (out_type < BW_TYPE_F16 || out_type > BW_TYPE_F32) return BW_ERR_ARG;
    if (!gx_sizes_ok(E, M, N, K) || N % 8 || K % 8) return BW_ERR_SHAPE;
    // tiles and K-blocks within 32-bit indices
    const long long per = (long long)((N + 255) / 256) * ((K + 255) / 256);
    if (per * E >= (1LL << 30) || per * ((long long)M / 64 + E) >= (1LL << 40)) return BW_ERR_SHAPE;
    return BW_OK;
}

size_t dw_work(const DwParams& p, int pairs, size_t* counters)
{
    *counters = up256(gx_work_bytes(pairs, 256));
    return *counters + up256((size_t)dw_counters(p, pairs) * sizeof(int));
}

int gemm_grouped_dw(const void* dY, long long ldy, const void* X, long long ldx, const int* offsets, void* dW, int E, int M,
                    int N, int K, int type, int out_type, void* work, size_t work_bytes, cudaStream_t st)
{
    if (type != BW_TYPE_F16 && type != BW_TYPE_BF16) return BW_ERR_ARG;
    int rc = dw_check(E, M, N, K, out_type);
    if (rc) return rc;
    if (ldy < N || ldy % 8 || ldy > (1LL << 32) || ldx < K || ldx % 8 || ldx > (1LL << 32)) return BW_ERR_SHAPE;
    if (!aligned(dW, 16)) return BW_ERR_ARG;
    cudaError_t e;
    if (M == 0) {  // no rows: every gradient is zero
        e = cudaMemsetAsync(dW, 0, (size_t)E * N * K * (out_type == BW_TYPE_F32 ? 4 : 2), st);
        return e == cudaSuccess ? BW_OK : cuda_fail(e, "cudaMemsetAsync (gradient)");
    }
    if (!aligned(dY, 16) || !aligned(X, 16) || !aligned(offsets, 4) || !aligned(work, 256)) return BW_ERR_ARG;
    DeviceState* d = nullptr;
    int pairs = 0;
    if ((rc = device_state(&d)) || (rc = gx_pairs(*d, &pairs))) return rc;
    DwParams p = dw_params(E, M, N, K, type == BW_TYPE_BF16, out_type);
    size_t at = 0;
    const size_t bytes = dw_work(p, pairs, &at);
    if (bytes > work_bytes) return scratch_fail(bytes, work_bytes);
    p.offsets = offsets;
    p.dW = dW;
    p.work = static_cast<float*>(work);
    p.counters = reinterpret_cast<int*>(static_cast<uint8_t*>(work) + at);
    p.next = p.counters + dw_counters(p, pairs) - 1;
    p.wait_ns = g_wait_ns;
    CUtensorMap my, mx;
    if (!moe_map(&my, dY, 0, (uint64_t)N, (uint64_t)M, 1, (uint64_t)ldy, (uint64_t)ldy * M, 64) ||
        !moe_map(&mx, X, 0, (uint64_t)K, (uint64_t)M, 1, (uint64_t)ldx, (uint64_t)ldx * M, 64)) {
        snprintf(g_errbuf, sizeof g_errbuf, "cuTensorMapEncodeTiled failed");
        return BW_ERR_LAUNCH;
    }
    static std::atomic<bool> limit_set[kMaxDevices];
    if ((rc = zero_counters(p.counters, dw_counters(p, pairs), st))) return rc;
    return launch_pairs(*d, grouped_dw_kernel, limit_set, my, mx, p, pairs, dw_smem(p.ring_bytes, E).bytes, st);
}

int f8_check(int E, int M, int N, int K, int out_type, int swiglu)
{
    if (out_type < BW_TYPE_F16 || out_type > BW_TYPE_F32 || (swiglu != 0 && swiglu != 1)) return BW_ERR_ARG;
    if (E < 0 || !gx_sizes_ok(E ? E : 1, M, N, K) || N % 8 || K % 16 || (swiglu && N % 256)) return BW_ERR_SHAPE;
    return BW_OK;
}

// C = A B^T of e4m3 operands; E 0: one matrix, all rows.
int f8_product(DeviceState& d, int pairs, const GxForm& form, const GxWork& w, const void* A, const float* a_scale, long long lds,
               const void* B, const float* b_scale, const int* offsets, int E, void* C, int M, int N, int K, int out_type,
               int swiglu, uint8_t* work, bool zeroed, cudaStream_t st)
{
    GxParams p = gx_params(E ? E : 1, M, N, K, form, false, false, !swiglu ? kGxPlain : E ? kGxGluHalves : kGxGluBlocks,
                           out_type);
    p.offsets = E ? offsets : nullptr;
    p.C = C;
    p.xs = a_scale;
    p.xs_ld = lds;
    p.ws = b_scale;
    return gx_product(d, p, form, gx_maps(p, K, K, true), A, B, w, work, pairs, zeroed, st);
}

int gemm_f8(const void* A, const void* a_scale, long long lds, const void* B, const void* b_scale, const int* offsets, int E,
            void* C, int M, int N, int K, int out_type, int swiglu, void* work, size_t work_bytes, cudaStream_t st)
{
    int rc = f8_check(E, M, N, K, out_type, swiglu);
    if (rc) return rc;
    if (lds < M) return BW_ERR_SHAPE;
    if (M == 0) return BW_OK;
    if (!aligned(A, 16) || !aligned(B, 16) || !aligned(C, 16) || !aligned(a_scale, 4) || !aligned(b_scale, 4) ||
        !aligned(work, 256) || (E && !aligned(offsets, 4)))
        return BW_ERR_ARG;
    DeviceState* d = nullptr;
    int pairs = 0;
    if ((rc = device_state(&d)) || (rc = gx_pairs(*d, &pairs))) return rc;
    const GxForm form = gx_form(M, E ? E : 1, E > 0, true);
    const GxWork w = gx_work(M, K, form.cap, pairs, false);
    if (w.bytes > work_bytes) return scratch_fail(w.bytes, work_bytes);
    return f8_product(*d, pairs, form, w, A, static_cast<const float*>(a_scale), lds, B, static_cast<const float*>(b_scale),
                      offsets, E, C, M, N, K, out_type, swiglu, static_cast<uint8_t*>(work), false, st);
}

int quant_f8_check(const void* X, int type, long long ld, int rows, int cols)
{
    if (type != BW_TYPE_F16 && type != BW_TYPE_BF16) return BW_ERR_ARG;
    if (rows < 0 || rows > (1 << 30) || cols < 1 || cols % 16 || cols > (1 << 20) || ld < cols || ld % 8) return BW_ERR_SHAPE;
    if ((long long)(rows / kF8Rows + 1) * ((cols + 255) / 256) > 0x7FFFFFFFLL) return BW_ERR_SHAPE;  // blocks of the grid
    if (rows && !aligned(X, 16)) return BW_ERR_ARG;
    return BW_OK;
}

int quant_f8_rows(const void* X, int type, long long ld, void* Q, float* scale, long long lds, int rows, int cols, int* zero,
                  int zero_n, cudaStream_t st)
{
    const QuantF8Params p = {static_cast<const uint16_t*>(X), ld, static_cast<uint8_t*>(Q), scale, lds, rows, cols, zero,
                             zero_n};
    const unsigned grid = (unsigned)((cols + 255) / 256) * (unsigned)((rows + kF8Rows - 1) / kF8Rows);
    if (type == BW_TYPE_BF16)
        quant_f8_rows_kernel<true><<<grid, 256, 0, st>>>(p);
    else
        quant_f8_rows_kernel<false><<<grid, 256, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? BW_OK : cuda_fail(e, "kernel launch (quantiser)");
}

}  // namespace
}  // namespace bw

BW_API int bw_quant_f8(const void* X, int x_type, long long ld, void* Q, void* scale, long long lds, int rows, int cols,
                       void* stream)
{
    using namespace bw;
    int rc = quant_f8_check(X, x_type, ld, rows, cols);
    if (rc) return rc;
    if (lds < rows) return BW_ERR_SHAPE;
    if (rows == 0) return BW_OK;
    if (!aligned(Q, 16) || !aligned(scale, 4)) return BW_ERR_ARG;
    DeviceState* d = nullptr;
    if ((rc = device_state(&d))) return rc;
    return quant_f8_rows(X, x_type, ld, Q, static_cast<float*>(scale), lds, rows, cols, nullptr, 0,
                         static_cast<cudaStream_t>(stream));
}

BW_API int bw_quant_blocks_f8(const void* W, int w_type, void* Q, void* scale, int E, int N, int K, void* stream)
{
    using namespace bw;
    if (w_type != BW_TYPE_F16 && w_type != BW_TYPE_BF16) return BW_ERR_ARG;
    if (E < 0 || E > 65535 || N < 1 || N > (1 << 20) || K < 1 || K > (1 << 20) || K % 16) return BW_ERR_SHAPE;
    if (E == 0) return BW_OK;
    if (!aligned(W, 16) || !aligned(Q, 16) || !aligned(scale, 4)) return BW_ERR_ARG;
    DeviceState* d = nullptr;
    int rc = device_state(&d);
    if (rc) return rc;
    const QuantF8Params p = {static_cast<const uint16_t*>(W), K, static_cast<uint8_t*>(Q), static_cast<float*>(scale), 0, N, K,
                             nullptr, 0};
    const dim3 grid((unsigned)((K + 127) / 128), (unsigned)((N + 127) / 128), (unsigned)E);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (w_type == BW_TYPE_BF16)
        quant_f8_blocks_kernel<true><<<grid, 256, 0, st>>>(p);
    else
        quant_f8_blocks_kernel<false><<<grid, 256, 0, st>>>(p);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? BW_OK : cuda_fail(e, "kernel launch (quantiser)");
}

BW_API int bw_gemm_f8_work_bytes(int E, int M, int N, int K, int out_type, int swiglu, int linear, size_t* bytes)
{
    using namespace bw;
    if (!bytes) return BW_ERR_ARG;
    *bytes = 0;
    int rc = f8_check(E, M, N, K, out_type, swiglu);
    if (rc || M == 0) return rc;
    DeviceState* d = nullptr;
    int pairs = 0;
    if ((rc = device_state(&d)) || (rc = gx_pairs(*d, &pairs))) return rc;
    *bytes = gx_work(M, K, gx_form(M, E ? E : 1, E > 0, true).cap, pairs, linear != 0).bytes;
    return BW_OK;
}

BW_API int bw_gemm_f8(const void* A, const void* a_scale, long long lds, const void* B, const void* b_scale,
                      const void* offsets, int E, void* C, int M, int N, int K, int out_type, int swiglu, void* work,
                      size_t work_bytes, void* stream)
{
    return bw::gemm_f8(A, a_scale, lds, B, b_scale, static_cast<const int*>(offsets), E, C, M, N, K, out_type, swiglu, work,
                       work_bytes, static_cast<cudaStream_t>(stream));
}

BW_API int bw_linear_f8(const void* X, int x_type, long long ld, const void* B, const void* b_scale, const void* offsets,
                        int E, void* C, int M, int N, int K, int swiglu, void* work, size_t work_bytes, void* stream)
{
    using namespace bw;
    int rc = x_type == BW_TYPE_F32 ? BW_ERR_ARG : f8_check(E, M, N, K, x_type, swiglu);
    if (rc || (rc = quant_f8_check(X, x_type, ld, M, K))) return rc;
    if (M == 0) return BW_OK;
    if (!aligned(B, 16) || !aligned(C, 16) || !aligned(b_scale, 4) || !aligned(work, 256) || (E && !aligned(offsets, 4)))
        return BW_ERR_ARG;
    DeviceState* d = nullptr;
    int pairs = 0;
    if ((rc = device_state(&d)) || (rc = gx_pairs(*d, &pairs))) return rc;
    const GxForm form = gx_form(M, E ? E : 1, E > 0, true);
    const GxWork w = gx_work(M, K, form.cap, pairs, true);
    if (w.bytes > work_bytes) return scratch_fail(w.bytes, work_bytes);
    uint8_t* ws = static_cast<uint8_t*>(work);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    float* scale = reinterpret_cast<float*>(ws + w.scale);
    if ((rc = quant_f8_rows(X, x_type, ld, ws + w.q, scale, w.lds, M, K, reinterpret_cast<int*>(ws + w.counters), w.n_counters,
                            st)))
        return rc;
    return f8_product(*d, pairs, form, w, ws + w.q, scale, w.lds, B, static_cast<const float*>(b_scale),
                      static_cast<const int*>(offsets), E, C, M, N, K, x_type, swiglu, ws, true, st);
}

BW_API int bw_gemm_grouped_work_bytes(int E, int M, int N, int K, int layout, int swiglu, size_t* bytes)
{
    using namespace bw;
    if (!bytes) return BW_ERR_ARG;
    *bytes = 0;
    int rc = grouped_check(E, M, N, K, layout, swiglu);
    if (rc || M == 0) return rc;
    DeviceState* d = nullptr;
    int pairs = 0;
    if ((rc = device_state(&d)) || (rc = gx_pairs(*d, &pairs))) return rc;
    *bytes = gx_work(M, K, gx_form(M, E, true, false).cap, pairs, false).bytes;
    return BW_OK;
}

BW_API int bw_gemm_grouped(const void* X, long long ldx, const void* B, const void* offsets, void* C, int E, int M, int N,
                           int K, int type, int layout, int swiglu, void* work, size_t work_bytes, void* stream)
{
    return bw::gemm_grouped(X, ldx, B, static_cast<const int*>(offsets), C, E, M, N, K, type, layout, swiglu, work, work_bytes,
                            static_cast<cudaStream_t>(stream));
}

BW_API int bw_gemm_grouped_dw_work_bytes(int E, int M, int N, int K, int out_type, size_t* bytes)
{
    using namespace bw;
    if (!bytes) return BW_ERR_ARG;
    *bytes = 0;
    int rc = dw_check(E, M, N, K, out_type);
    if (rc || M == 0) return rc;
    DeviceState* d = nullptr;
    int pairs = 0;
    if ((rc = device_state(&d)) || (rc = gx_pairs(*d, &pairs))) return rc;
    size_t at = 0;
    *bytes = dw_work(dw_params(E, M, N, K, false, out_type), pairs, &at);
    return BW_OK;
}

BW_API int bw_gemm_grouped_dw(const void* dY, long long ldy, const void* X, long long ldx, const void* offsets, void* dW,
                              int E, int M, int N, int K, int type, int out_type, void* work, size_t work_bytes, void* stream)
{
    return bw::gemm_grouped_dw(dY, ldy, X, ldx, static_cast<const int*>(offsets), dW, E, M, N, K, type, out_type, work,
                               work_bytes, static_cast<cudaStream_t>(stream));
}
