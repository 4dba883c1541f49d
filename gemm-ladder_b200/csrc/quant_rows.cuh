// quant_rows.cuh -- rows of fp16 or bf16 to 8-bit signed integers with one scale per row.
//
//   a_m = max_k |x_mk|,  scale_m = a_m / 127,  q_mk = round-half-even(127 x_mk / a_m)   (so |q| <= 127)
// A row of zeros gets scale 0 and q 0; a row holding an infinity or a NaN gets scale NaN and q 0 (its products are NaN,
// as the unquantised ones' would be).
//
// The rounding is that of the exact quotient Q = 127 x / a, whatever computes it.  x = X 2^i and a = A 2^j with integers X
// and A below 2^11, so a Q that is not half-way between two integers is at least 1 / (254 X) > 2^-19 of itself away
// from every half-way point, and any product within 2^-21 of Q rounds to the right integer.  Q is half-way only where
// 254 X 2^(i - j) is an odd multiple 2 n + 1 of A; 127 is prime, so it divides A, or 2 n + 1 is 127 and x is a / 2.
//   - A is no multiple of 127 (and a in [2^-64, 2^64]): q = x c rounded, c = fl(127 / a) (1 + 2^-22); the surplus turns
//     the one half-way case, 63.5, into the even 64.  One multiply-add per element: adding 1.5 x 2^23 leaves the
//     integer in the sum's low bits.
//   - otherwise (8 of 1024 fp16 significands, 1 of 128 bf16 ones): half-way quotients are found by the residual
//     127 x - n a, which is exact in fp32 (both terms are multiples of the same power of two and below 2^20 of it), and
//     rounded to even; a is brought into range by a power of two first, so that neither 1 / a nor 127 x leaves fp32's.
//
// Bound by its bytes where there are many rows: 2 read and 1 written per element, in one pass, the row kept in
// registers between its maximum and its rounding.  (With the residual for every element the kernel was bound by its
// instructions: 8192 x 8192 in 50 us, against 34 us now, 0.91 of the copy bandwidth.)  A warp takes a row of up to 2048 elements (8 of them in a
// block), a block of 128 threads one of up to 8192, of 512 threads a longer one; rows beyond 32768 elements read their
// tail a second time (from L2).
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
    float c;                    // fl(127 / a) (1 + 2^-22)
    float mul, inv, a, half_a;  // 127 x 2^e, 1 / (a 2^e), a 2^e, half of it
};
constexpr float kQuantMagic = 12582912.0f;  // 1.5 x 2^23

// q in the low byte.
template <bool EXACT>
__device__ __forceinline__ uint32_t quant1(float x, const RowScale& s)
{
    if (!EXACT) return __float_as_uint(fmaf(x, s.c, kQuantMagic));
    const float y = x * s.mul;
    const float t = fmaf(y, s.inv, kQuantMagic);
    const float n = t - kQuantMagic;
    const float d = fmaf(-n, s.a, y);
    uint32_t q = __float_as_uint(t);
    if (fabsf(d) == s.half_a && (q & 1u)) q += d > 0.f ? 1u : 0xFFFFFFFFu;
    return q;
}

template <bool BF16, bool EXACT>
__device__ __forceinline__ uint2 quant8(uint4 v, const RowScale& s)
{
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t out[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float a, b, c, d;
        unpack2<BF16>(w[2 * h], a, b);
        unpack2<BF16>(w[2 * h + 1], c, d);
        const uint32_t ab = __byte_perm(quant1<EXACT>(a, s), quant1<EXACT>(b, s), 0x0040);
        const uint32_t cd = __byte_perm(quant1<EXACT>(c, s), quant1<EXACT>(d, s), 0x0040);
        out[h] = __byte_perm(ab, cd, 0x5410);
    }
    return make_uint2(out[0], out[1]);
}

// G threads per row (32: a warp each of 8 rows; more: the block), VEC 16-byte vectors of the row per thread in registers.
template <bool BF16, int G, int VEC>
__global__ void __launch_bounds__(G == 32 ? 256 : G) quant_rows_kernel(const QuantParams p)
{
    constexpr int kRowsPerBlock = G == 32 ? 8 : 1;
    constexpr int kWarps = G / 32;
    __shared__ uint32_t warp_max[kWarps];
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
        m = __reduce_max_sync(0xFFFFFFFFu, warp_max[threadIdx.x % kWarps]);
    }
    float a, unused;
    unpack2<BF16>(m, a, unused);
    const bool finite = m < (BF16 ? 0x7F80u : 0x7C00u);
    if (t == 0) p.scale[row] = finite ? a / 127.0f : __uint_as_float(0x7FC00000u);
    if (!finite || m == 0u) {
        for (int c = t; c < nv; c += G) q[c] = make_uint2(0u, 0u);
        return;
    }
    // A: the significand with its leading bit
    constexpr uint32_t kFrac = BF16 ? 0x7Fu : 0x3FFu;
    const uint32_t A = (m & kFrac) | (m > kFrac ? kFrac + 1u : 0u);
    RowScale s;
    if (A % 127u != 0u && a >= 0x1p-64f && a <= 0x1p64f) {
        s.c = 127.0f / a * (1.0f + 0x1p-22f);
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            const int c = t + i * G;
            if (c < nv) q[c] = quant8<BF16, false>(v[i], s);
        }
        for (int c = t + VEC * G; c < nv; c += G) q[c] = quant8<BF16, false>(x[c], s);
    } else {
        const float e = a < 0x1p-64f ? 0x1p64f : a > 0x1p64f ? 0x1p-64f : 1.0f;
        s.a = a * e;
        s.half_a = 0.5f * s.a;
        s.inv = 1.0f / s.a;
        s.mul = 127.0f * e;
        for (int c = t; c < nv; c += G) q[c] = quant8<BF16, true>(x[c], s);  // (rare: the row again, from L1 or L2)
    }
}

}  // namespace bw
