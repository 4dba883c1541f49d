// quant_f8.cuh -- fp16 or bf16 to e4m3 with a scale for each group of 128 of a row, or for each block of 128 x 128.
//
//   a = max |x| of the group,  scale = fl(a / 448),  q = e4m3(fl(x fl(448 / a))), nearest, ties to even
// with fl rounding to fp32 (each quotient and product rounded once, so a result is defined to the bit).  The largest
// magnitude becomes 448, e4m3's largest value.  448 / a leaves fp32 below a = 1.3e-36: a and x are then scaled by 2^100
// first, which rounds nothing.  A group of zeros gets scale 0 and q 0; one that holds an infinity or a NaN gets scale NaN
// and q 0 (its products are NaN, as the unquantised ones' would be).
//
// Bound by its bytes: 2 read and 1 written per element, in one pass, a group held in registers between its maximum and its
// rounding.  10240 x 8192 by blocks: 41 us, 0.94 of the copy bandwidth; 4099 x 7184 by rows: 21 us, 0.65 (14 us of bytes; 3.2
// waves of blocks, their start and the launch).
#pragma once
#include <cuda_fp8.h>

#include "quant_rows.cuh"

namespace bw {

constexpr float kF8Top = 448.0f;

struct QuantF8Params {
    const uint16_t* X;  // rows x cols, ld elements from row to row (16-byte aligned rows)
    long long ld;
    uint8_t* Q;         // rows x cols, contiguous
    float* scale;       // rows: group b of row r at b * lds + r; blocks: [block row][block column]
    long long lds;
    int rows, cols;     // cols % 16 == 0
    int* zero;          // zero_n words set to 0 for the kernel that follows
    int zero_n;
};

struct F8Scale {
    float up, inv, scale;  // q = e4m3((x up) inv)
};
// From the bits of the largest magnitude.
template <bool BF16>
__device__ __forceinline__ F8Scale f8_scale(uint32_t m)
{
    float a, unused;
    unpack2<BF16>(m, a, unused);
    F8Scale s;
    const bool finite = m < (BF16 ? 0x7F80u : 0x7C00u);
    s.up = BF16 && a < 0x1p-100f ? 0x1p100f : 1.0f;
    s.inv = finite && m != 0u ? kF8Top / (a * s.up) : 0.0f;
    s.scale = finite ? a / kF8Top : __uint_as_float(0x7FC00000u);
    return s;
}

// 8 values to e4m3, or 8 zeros where inv is 0 (whatever the values).
template <bool BF16>
__device__ __forceinline__ uint2 f8_pack8(uint4 v, const F8Scale& s)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float a, b;
        unpack2<BF16>(w[i], a, b);
        if (BF16) {
            a *= s.up;
            b *= s.up;
        }
        h[i] = __nv_cvt_float2_to_fp8x2(make_float2(a * s.inv, b * s.inv), __NV_SATFINITE, __NV_E4M3);
    }
    if (s.inv == 0.0f) return make_uint2(0u, 0u);
    return make_uint2(h[0] | h[1] << 16, h[2] | h[3] << 16);
}

constexpr int kF8Rows = 32;  // rows of a block of the row form

// Groups of 128 along a row.  A block takes 32 rows x 256 columns: a warp 4 rows, half a warp a group, and writes the
// groups' 32 scales of a column of groups as one line.
template <bool BF16>
__global__ void __launch_bounds__(256) quant_f8_rows_kernel(const QuantF8Params p)
{
    __shared__ float sc[2][kF8Rows];
    griddep_launch();
    griddep_wait();
    const int across = (p.cols + 255) / 256, bx = blockIdx.x % across, by = blockIdx.x / across;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.zero_n; i += blockDim.x) p.zero[i] = 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r0 = by * kF8Rows + warp * 4, col = bx * 256 + lane * 8;
    uint4 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
        v[i] = r0 + i < p.rows && col < p.cols ? *reinterpret_cast<const uint4*>(p.X + (size_t)(r0 + i) * p.ld + col)
                                               : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t m = max_bits(v[i], 0u);
#pragma unroll
        for (int d = 8; d; d >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xFFFFFFFFu, m, d));
        m = max(m & 0xFFFFu, m >> 16);
        const F8Scale s = f8_scale<BF16>(m);
        if (r0 + i < p.rows && col < p.cols)
            *reinterpret_cast<uint2*>(p.Q + (size_t)(r0 + i) * p.cols + col) = f8_pack8<BF16>(v[i], s);
        if ((lane & 15) == 0) sc[lane >> 4][warp * 4 + i] = s.scale;
    }
    __syncthreads();
    const int t = threadIdx.x;
    const int b = bx * 2 + (t >> 5), r = by * kF8Rows + (t & 31);
    if (t < 64 && r < p.rows && b * 128 < p.cols) p.scale[b * p.lds + r] = sc[t >> 5][t & 31];
}

// Blocks of 128 x 128, a block of 256 threads each: its 2048 16-byte vectors in registers, 8 a thread.  blockIdx.z: the matrix.
template <bool BF16>
__global__ void __launch_bounds__(256) quant_f8_blocks_kernel(const QuantF8Params p)
{
    __shared__ uint32_t warp_max[8];
    const int col = blockIdx.x * 128 + (threadIdx.x & 15) * 8, r0 = blockIdx.y * 128 + (threadIdx.x >> 4);
    const uint16_t* X = p.X + (size_t)blockIdx.z * p.rows * p.ld;
    uint8_t* Q = p.Q + (size_t)blockIdx.z * p.rows * p.cols;
    uint4 v[8];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + 16 * i;
        v[i] = r < p.rows && col < p.cols ? *reinterpret_cast<const uint4*>(X + (size_t)r * p.ld + col)
                                          : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max_bits(v[i], m);
    m = max(m & 0xFFFFu, m >> 16);
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
    __syncthreads();
    m = __reduce_max_sync(0xFFFFFFFFu, warp_max[threadIdx.x & 7]);
    const F8Scale s = f8_scale<BF16>(m);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = r0 + 16 * i;
        if (r < p.rows && col < p.cols) *reinterpret_cast<uint2*>(Q + (size_t)r * p.cols + col) = f8_pack8<BF16>(v[i], s);
    }
    if (threadIdx.x == 0) p.scale[((size_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = s.scale;
}

}  // namespace bw
