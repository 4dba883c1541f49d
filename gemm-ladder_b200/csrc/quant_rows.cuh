// quant_rows.cuh -- rows of fp16 or bf16 to 8-bit signed integers with one scale per row.
//
//   a_m = max_k |x_mk|,  scale_m = a_m / 127,  q_mk = round-half-even(127 x_mk / a_m)   (so |q| <= 127)
// A row of zeros gets scale 0 and q 0; a row holding an infinity or a NaN gets scale NaN and q 0 (its products are NaN,
// as the unquantised ones' would be).
//
// The rounding is that of the exact quotient, whatever computes it.  With r = fl(127 x fl(1 / a)) the quotient is off by
// 3 roundings of 2^-24; x and a have at most 11 significant bits, so a quotient that is not half-way between two
// integers differs from every half-way point by more than 2^-19 of itself, and rint(r) is right.  Half-way quotients
// are settled with the residual 127 x - n a, which is exact in fp32 (both terms are multiples of the same power of two
// and below 2^20 of it): where it is half of a and n is odd, n moves to the other neighbour.  Rows whose a is outside
// [2^-64, 2^64] are scaled by a power of two first, so that neither 1 / a nor 127 x leaves fp32's range.
//
// Bound by its bytes: 2 bytes read and 1 written per element, in one pass, the row kept in registers between its
// maximum and its rounding.  A warp takes a row of up to 2048 elements (8 of them in a block), a block of 512 threads
// a longer one; rows beyond 32768 elements read their tail a second time (from L2).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "ptx.cuh"

namespace bw {

struct QuantParams {
    const uint16_t* X;  // rows x cols, ld elements from row to row (16-byte aligned rows)
    long long ld;
    int8_t* Q;          // rows x cols, contiguous
    float* scale;       // rows
    int rows, cols;     // cols % 16 == 0
    int* zero;          // zero_n words set to 0 for the kernel that follows (its split-tile counters)
    int zero_n;
};

template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t u, float& a, float& b)
{
    if (BF16) {
        a = __uint_as_float(u << 16);
        b = __uint_as_float(u & 0xFFFF0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
        a = f.x;
        b = f.y;
    }
}

// The largest of 2 x 4 packed magnitudes and m (16-bit patterns without the sign order like the values, infinities and
// NaNs above every number).
__device__ __forceinline__ uint32_t max_bits(uint4 v, uint32_t m)
{
    m = __vmaxu2(m, v.x & 0x7FFF7FFFu);
    m = __vmaxu2(m, v.y & 0x7FFF7FFFu);
    m = __vmaxu2(m, v.z & 0x7FFF7FFFu);
    return __vmaxu2(m, v.w & 0x7FFF7FFFu);
}

struct RowScale {
    float mul, inv, a, half_a;  // 127 x 2^e, 1 / (a 2^e), a 2^e, half of it
};

__device__ __forceinline__ int quant1(float x, const RowScale& s)
{
    const float y = x * s.mul;
    const float n = rintf(y * s.inv);
    const float d = fmaf(-n, s.a, y);
    int q = (int)n;
    if (fabsf(d) == s.half_a && (q & 1)) q += d > 0.f ? 1 : -1;
    return q;
}

template <bool BF16>
__device__ __forceinline__ uint2 quant8(uint4 v, const RowScale& s)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float a, b, c, d;
        unpack2<BF16>(w[2 * h], a, b);
        unpack2<BF16>(w[2 * h + 1], c, d);
        const uint32_t ab = __byte_perm((uint32_t)quant1(a, s), (uint32_t)quant1(b, s), 0x0040);
        const uint32_t cd = __byte_perm((uint32_t)quant1(c, s), (uint32_t)quant1(d, s), 0x0040);
        out[h] = __byte_perm(ab, cd, 0x5410);
    }
    return make_uint2(out[0], out[1]);
}

// G threads per row (32: a warp each of 8 rows; 512: the block), VEC 16-byte vectors of the row per thread in registers.
template <bool BF16, int G, int VEC>
__global__ void __launch_bounds__(G == 32 ? 256 : G) quant_rows_kernel(const QuantParams p)
{
    constexpr int kRowsPerBlock = G == 32 ? 8 : 1;
    __shared__ uint32_t warp_max[16];
    griddep_launch();  // the product that follows may set itself up; it waits for this kernel before it reads
    griddep_wait();
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < p.zero_n; i += blockDim.x) p.zero[i] = 0;
    const int t = threadIdx.x % G;
    const int row = blockIdx.x * kRowsPerBlock + threadIdx.x / G;
    if (row >= p.rows) return;  // whole warps; with one row per block, never
    const int nv = p.cols / 8;
    const uint4* x = reinterpret_cast<const uint4*>(p.X + (size_t)row * p.ld);
    uint2* q = reinterpret_cast<uint2*>(p.Q + (size_t)row * p.cols);
    uint4 v[VEC];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = t + i * G;
        v[i] = c < nv ? x[c] : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = max_bits(v[i], m);
    for (int c = t + VEC * G; c < nv; c += G) m = max_bits(x[c], m);
    m = max(m & 0xFFFFu, m >> 16);
    m = __reduce_max_sync(0xFFFFFFFFu, m);
    if (G > 32) {
        if ((threadIdx.x & 31) == 0) warp_max[threadIdx.x >> 5] = m;
        __syncthreads();
        m = __reduce_max_sync(0xFFFFFFFFu, warp_max[threadIdx.x & 15]);
    }
    float a, unused;
    unpack2<BF16>(m, a, unused);
    const bool finite = m < (BF16 ? 0x7F80u : 0x7C00u);
    if (t == 0) p.scale[row] = finite ? a / 127.0f : __uint_as_float(0x7FC00000u);
    if (!finite || m == 0u) {
        for (int c = t; c < nv; c += G) q[c] = make_uint2(0u, 0u);
        return;
    }
    const float e = a < 0x1p-64f ? 0x1p64f : a > 0x1p64f ? 0x1p-64f : 1.0f;
    RowScale s;
    s.a = a * e;
    s.half_a = 0.5f * s.a;
    s.inv = 1.0f / s.a;
    s.mul = 127.0f * e;
#pragma unroll
    for (int i = 0; i < VEC; ++i) {
        const int c = t + i * G;
        if (c < nv) q[c] = quant8<BF16>(v[i], s);
    }
    for (int c = t + VEC * G; c < nv; c += G) q[c] = quant8<BF16>(x[c], s);
}

}  // namespace bw
