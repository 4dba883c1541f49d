// gemm_i8.cuh -- host side of the 8-bit integer entries (bw_quant_rows_i8, bw_gemm_i8, bw_gemm_i8_swiglu, bw_linear_i8
// of bwgemm.h), included by bwgemm.cu: argument checks, the plan (plan.h, an int8 row of K planned as an fp16 row of
// K / 2, K rounded up to whole 128-byte stages), the caller's workspace, the launches.
#pragma once
#include "quant_rows.cuh"

namespace bw {
namespace {

// K products of magnitude up to 2^14 (-128 x -128) sum to less than 2^31.
constexpr int kI8MaxK = 131056;

bool i8_shape_ok(int M, int N, int K)
{
    return M >= 0 && N > 0 && K > 0 && N % 64 == 0 && K % 16 == 0 && K <= kI8MaxK;
}
bool aligned(const void* p, uintptr_t a) { return p && reinterpret_cast<uintptr_t>(p) % a == 0; }

// The plan of a call: M x N x K in 8 bits as M x N x K / 2 in fp16.
int i8_plan(DeviceState& d, int M, int N, int K, int epi, bw_plan* q)
{
    std::lock_guard<std::mutex> lock(g_mu);
    int rc = pair_occupancy(d);
    if (rc) return rc;
    // the last plans, by shape (a plan depends on nothing else; making one takes a microsecond of the host's time)
    struct Entry {
        const DeviceState* d;
        int M, N, K, epi;
        bw_plan q;
    };
    static Entry cache[64];
    Entry& at = cache[((unsigned)M * 31u + (unsigned)N / 64u * 7u + (unsigned)K / 16u + (unsigned)epi) % 64u];
    if (at.d == &d && at.M == M && at.N == N && at.K == K && at.epi == epi) {
        *q = at.q;
        return BW_OK;
    }
    const unsigned flags = epi == kEpiI8F32      ? kPlanNoSwap | kPlanI8
                           : epi == kEpiI8SwiGLU ? kPlanGateUp | kPlanI8 | (M > 128 ? kPlanNoSplit : 0u)
                                                 : kPlanI8;
    if ((rc = make_plan(M, N, (K + 127) / 128 * 64, d.sms, d.pairs, 0, q, flags, held_of(d)))) return rc;
    at = {&d, M, N, K, epi, *q};
    return BW_OK;
}

// The workspace of a call: [linear: the quantised rows, their scales][partials of split tiles][their counters].
struct I8Work {
    size_t q_off, scale_off, partial_off, counter_off, bytes;
};
size_t up256(size_t v) { return (v + 255) / 256 * 256; }
I8Work i8_work(const bw_plan& q, int M, int K, bool linear)
{
    I8Work w = {};
    size_t at = 0;
    if (linear) {
        w.q_off = at;
        at = up256(at + (size_t)M * K);
        w.scale_off = at;
        at = up256(at + (size_t)M * sizeof(float));
    }
    w.partial_off = at;
    at = up256(at + q.workspace_bytes);
    w.counter_off = at;
    w.bytes = q.counters || linear ? at + (size_t)q.counters * sizeof(int) : at;
    return w;
}

template <int BN, bool SWAP, bool PAIR, int EPI, int WM = 1>
int i8_launch(DeviceState& d, const bw_plan& q, const CUtensorMap& mx, const CUtensorMap& my, const Params& p,
              cudaStream_t st, bool pdl)
{
    // the instance's shared-memory limit, set once per device (an atomic flag: calls may come from several threads)
    static std::atomic<bool> limit_set[kMaxDevices];
    std::atomic<bool>& done = limit_set[&d - g_dev];
    if (!done.load(std::memory_order_acquire)) {
        cudaError_t e = cudaFuncSetAttribute(gemm_kernel<BN, SWAP, PAIR, EPI, WM>,
                                             cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             KGeom<BN, SWAP, PAIR, EPI, WM>::kSmemBytes);
        if (e != cudaSuccess) return cuda_fail(e, "cudaFuncSetAttribute");
        done.store(true, std::memory_order_release);
    }
    DeviceState attrs_set;  // launch_kernel's own record of the limits: all set
    attrs_set.attrs = ~0ull;
    return launch_kernel<BN, SWAP, PAIR, EPI, WM>(attrs_set, 1ull, q, mx, my, mx, p, st, pdl);
}

template <int EPI, int WM>
int i8_launch_swap(DeviceState& d, const bw_plan& q, const CUtensorMap& mx, const CUtensorMap& my, const Params& p,
                   cudaStream_t st, bool pdl)
{
    switch (q.bn) {
    case 16: return i8_launch<16, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    case 32: return i8_launch<32, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    case 48: return i8_launch<48, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    case 64: return i8_launch<64, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    case 80: return i8_launch<80, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    case 96: return i8_launch<96, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    case 112: return i8_launch<112, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    case 128: return i8_launch<128, true, false, EPI, WM>(d, q, mx, my, p, st, pdl);
    default: return BW_ERR_ARG;
    }
}

int i8_dispatch(DeviceState& d, const bw_plan& q, const CUtensorMap& mx, const CUtensorMap& my, const Params& p,
                cudaStream_t st, int epi, bool pdl)
{
    if (q.kernel == BW_KERNEL_PAIR) {
        if (epi == kEpiI8F32) return i8_launch<256, false, true, kEpiI8F32>(d, q, mx, my, p, st, pdl);
        if (epi == kEpiI8SwiGLU) return i8_launch<256, false, true, kEpiI8SwiGLU>(d, q, mx, my, p, st, pdl);
#if BW_PAIR_WIDE
        if (q.bn == 512) return i8_launch<512, false, true, kEpiI8>(d, q, mx, my, p, st, pdl);
#endif
        return i8_launch<256, false, true, kEpiI8>(d, q, mx, my, p, st, pdl);
    }
    if (q.kernel == BW_KERNEL_TILE && q.bn == 128 && epi == kEpiI8)
        return i8_launch<128, false, false, kEpiI8>(d, q, mx, my, p, st, pdl);
    if (q.kernel != BW_KERNEL_SWAP) {
        snprintf(g_errbuf, sizeof g_errbuf, "this device holds no pairs of SMs");
        return BW_ERR_LAUNCH;
    }
    if (epi == kEpiI8SwiGLU) return i8_launch_swap<kEpiI8SwiGLU, 2>(d, q, mx, my, p, st, pdl);
    return q.wm == 2 ? i8_launch_swap<kEpiI8, 2>(d, q, mx, my, p, st, pdl)
                     : i8_launch_swap<kEpiI8, 1>(d, q, mx, my, p, st, pdl);
}

// C from the quantised rows; zeroed: the counters are already at zero (and the launch may overlap the kernel that
// zeroed them, which it waits for).
int i8_product(DeviceState& d, const bw_plan& q, const I8Work& w, const void* A, const float* a_scale, const void* B,
               const float* b_scale, void* C, int M, int N, int K, int epi, bool bf16, uint8_t* work, bool zeroed,
               cudaStream_t st)
{
    int* counters = reinterpret_cast<int*>(work + w.counter_off);
    if (q.counters && !zeroed) {
        cudaError_t e = cudaMemsetAsync(counters, 0, (size_t)q.counters * sizeof(int), st);
        if (e != cudaSuccess) return cuda_fail(e, "cudaMemsetAsync (counters)");
    }
    CUtensorMap mx, my;
    if (!make_maps(q, A, B, M, N, K / 2, &mx, &my, true)) {
        snprintf(g_errbuf, sizeof g_errbuf, "cuTensorMapEncodeTiled failed");
        return BW_ERR_LAUNCH;
    }
    Params p =
        make_params(q, M, N, q.kblocks * 64, C, reinterpret_cast<float*>(work + w.partial_off), counters, true);
    i8_params(p, a_scale, b_scale, bf16, zeroed);
    return i8_dispatch(d, q, mx, my, p, st, epi, zeroed);
}

int i8_epi(int out_type, int swiglu)
{
    if (swiglu) return out_type == BW_TYPE_F32 ? -1 : kEpiI8SwiGLU;
    return out_type == BW_TYPE_F32 ? kEpiI8F32 : kEpiI8;
}

int i8_check(int M, int N, int K, int out_type, int swiglu)
{
    if (out_type < BW_TYPE_F16 || out_type > BW_TYPE_F32 || (swiglu != 0 && swiglu != 1)) return BW_ERR_ARG;
    if (i8_epi(out_type, swiglu) < 0) return BW_ERR_ARG;
    if (!i8_shape_ok(M, N, K) || (swiglu && N % 256)) return BW_ERR_SHAPE;
    return BW_OK;
}

int scratch_fail(size_t need, size_t have)
{
    snprintf(g_errbuf, sizeof g_errbuf, "the call needs %zu bytes of workspace, %zu given", need, have);
    return BW_ERR_SCRATCH;
}

int i8_gemm(const void* A, const void* a_scale, const void* B, const void* b_scale, void* C, int M, int N, int K,
            int out_type, int swiglu, void* work, size_t work_bytes, cudaStream_t st)
{
    int rc = i8_check(M, N, K, out_type, swiglu);
    if (rc) return rc;
    if (M == 0) return BW_OK;
    if (!aligned(A, 16) || !aligned(B, 16) || !aligned(C, 16) || !aligned(a_scale, 4) || !aligned(b_scale, 16) ||
        (work_bytes && !aligned(work, 256)))
        return BW_ERR_ARG;
    DeviceState* d = nullptr;
    if ((rc = device_state(&d))) return rc;
    const int epi = i8_epi(out_type, swiglu);
    bw_plan q;
    if ((rc = i8_plan(*d, M, N, K, epi, &q))) return rc;
    const I8Work w = i8_work(q, M, K, false);
    if (w.bytes > work_bytes) return scratch_fail(w.bytes, work_bytes);
    return i8_product(*d, q, w, A, static_cast<const float*>(a_scale), B, static_cast<const float*>(b_scale), C, M, N, K,
                      epi, out_type == BW_TYPE_BF16, static_cast<uint8_t*>(work), false, st);
}

// The quantiser's instance: a warp per row up to 2048 elements, else a block whose threads hold 8 of the row's 16-byte
// vectors each: 128 threads up to 8192 elements (more, smaller blocks per SM; many threads with few vectors each lose
// to the blocks' fixed cost: 8192 x 8192 took 62 us with 512 threads where 128 took 50), 512 above.
template <bool BF16>
void quant_launch(const QuantParams& p, cudaStream_t st)
{
    const int nv = p.cols / 8;
    const dim3 warp_rows((p.rows + 7) / 8);
    if (nv <= 64)
        quant_rows_kernel<BF16, 32, 2><<<warp_rows, 256, 0, st>>>(p);
    else if (nv <= 256)
        quant_rows_kernel<BF16, 32, 8><<<warp_rows, 256, 0, st>>>(p);
    else if (nv <= 1024)
        quant_rows_kernel<BF16, 128, 8><<<p.rows, 128, 0, st>>>(p);
    else
        quant_rows_kernel<BF16, 512, 8><<<p.rows, 512, 0, st>>>(p);
}

int quant_rows(const void* X, int x_type, long long ld, void* Q, void* scale, int rows, int cols, int* zero, int zero_n,
               cudaStream_t st)
{
    QuantParams p = {static_cast<const uint16_t*>(X), ld, static_cast<int8_t*>(Q), static_cast<float*>(scale), rows,
                     cols, zero, zero_n};
    if (x_type == BW_TYPE_BF16)
        quant_launch<true>(p, st);
    else
        quant_launch<false>(p, st);
    const cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? BW_OK : cuda_fail(e, "kernel launch (quantiser)");
}

int quant_check(const void* X, int x_type, long long ld, int rows, int cols)
{
    if (x_type != BW_TYPE_F16 && x_type != BW_TYPE_BF16) return BW_ERR_ARG;
    if (rows < 0 || cols <= 0 || cols % 16 || ld < cols || ld % 8) return BW_ERR_SHAPE;
    if (rows > 0 && !aligned(X, 16)) return BW_ERR_ARG;
    return BW_OK;
}

}  // namespace
}  // namespace bw

BW_API int bw_quant_rows_i8(const void* X, int x_type, long long ld, void* Q, void* scale, int rows, int cols,
                            void* stream)
{
    using namespace bw;
    int rc = quant_check(X, x_type, ld, rows, cols);
    if (rc) return rc;
    if (rows == 0) return BW_OK;
    if (!aligned(Q, 16) || !aligned(scale, 4)) return BW_ERR_ARG;
    DeviceState* d = nullptr;
    if ((rc = device_state(&d))) return rc;
    return quant_rows(X, x_type, ld, Q, scale, rows, cols, nullptr, 0, static_cast<cudaStream_t>(stream));
}

BW_API int bw_gemm_i8_work_bytes(int M, int N, int K, int out_type, int swiglu, int linear, size_t* bytes)
{
    using namespace bw;
    if (!bytes) return BW_ERR_ARG;
    *bytes = 0;
    int rc = i8_check(M, N, K, out_type, swiglu);
    if (rc || M == 0) return rc;
    DeviceState* d = nullptr;
    if ((rc = device_state(&d))) return rc;
    bw_plan q;
    if ((rc = i8_plan(*d, M, N, K, i8_epi(out_type, swiglu), &q))) return rc;
    *bytes = i8_work(q, M, K, linear != 0).bytes;
    return BW_OK;
}

BW_API int bw_gemm_i8(const void* A, const void* a_scale, const void* B, const void* b_scale, void* C, int M, int N,
                      int K, int out_type, void* work, size_t work_bytes, void* stream)
{
    return bw::i8_gemm(A, a_scale, B, b_scale, C, M, N, K, out_type, 0, work, work_bytes,
                       static_cast<cudaStream_t>(stream));
}

BW_API int bw_gemm_i8_swiglu(const void* A, const void* a_scale, const void* B, const void* b_scale, void* C, int M,
                             int N, int K, int out_type, void* work, size_t work_bytes, void* stream)
{
    return bw::i8_gemm(A, a_scale, B, b_scale, C, M, N, K, out_type, 1, work, work_bytes,
                       static_cast<cudaStream_t>(stream));
}

BW_API int bw_linear_i8(const void* X, int x_type, long long ld, const void* B, const void* b_scale, void* C, int M,
                        int N, int K, int swiglu, void* work, size_t work_bytes, void* stream)
{
    using namespace bw;
    if (x_type != BW_TYPE_F16 && x_type != BW_TYPE_BF16) return BW_ERR_ARG;
    int rc = i8_check(M, N, K, x_type, swiglu);
    if (rc || (rc = quant_check(X, x_type, ld, M, K))) return rc;
    if (M == 0) return BW_OK;
    if (!aligned(B, 16) || !aligned(C, 16) || !aligned(b_scale, 16) || !aligned(work, 256)) return BW_ERR_ARG;
    DeviceState* d = nullptr;
    if ((rc = device_state(&d))) return rc;
    const int epi = i8_epi(x_type, swiglu);
    bw_plan q;
    if ((rc = i8_plan(*d, M, N, K, epi, &q))) return rc;
    const I8Work w = i8_work(q, M, K, true);
    if (w.bytes > work_bytes) return scratch_fail(w.bytes, work_bytes);
    uint8_t* ws = static_cast<uint8_t*>(work);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if ((rc = quant_rows(X, x_type, ld, ws + w.q_off, ws + w.scale_off, M, K,
                         reinterpret_cast<int*>(ws + w.counter_off), q.counters, st)))
        return rc;
    return i8_product(*d, q, w, ws + w.q_off, reinterpret_cast<const float*>(ws + w.scale_off), B,
                      static_cast<const float*>(b_scale), C, M, N, K, epi, x_type == BW_TYPE_BF16, ws, true, st);
}
