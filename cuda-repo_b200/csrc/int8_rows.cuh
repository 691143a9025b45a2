// int8_rows.cuh -- the rounding of 16-bit rows to int8 values with one scale
// per row, shared by the token quantiser and the mixture-of-experts kernel.
//
//   a = max_k |x_k|,  scale = a / 127,  q_k = rint(127 x_k / a)  (ties to even)
//
// The rounding is exact: q is what the formula gives in real numbers, although
// a kernel that divides every element would be bound by its arithmetic.  It
// multiplies by RN(127 / a) (relative error 2^-23 after the product's own
// rounding) and then rounds the product p to 20 significant bits.  For p in
// [2^j, 2^(j+1)), j <= 6: a tie k + 1/2 has 8 bits at most, so it lies on that
// grid, and an exact tie's p, 2^(j-22) away at most, rounds onto it.  What is
// not a tie is further from every tie than that can move it: with x = X 2^e,
// a = A 2^f, integers X, A < 2^11 (11 significant bits at most in fp16 and
// bf16), 127 x / a differs from (2k + 1) / 2 by a non-zero multiple of
// 2^(e-f+1) / (2 A) -- more than 2^(j-19), since 127 X 2^(e-f) / A >= 2^j --
// or, for e >= f, of 1 / (2 A); the two roundings move it by 2^(j-20) +
// 2^(j-22).
//
// Rows with an infinity or NaN get that as their scale and zeros as values,
// so a product with them is NaN.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace spmm24 {

__device__ __forceinline__ uint32_t vmaxu2(uint32_t a, uint32_t b) { return __vmaxu2(a, b); }

// The magnitude bits of a 16-bit float order as the magnitudes do, infinities
// above the finite and NaN above those: maxima are taken on them.
__device__ __forceinline__ uint32_t abs_max8(uint4 v) {
    const uint32_t m = 0x7fff7fffu;
    return vmaxu2(vmaxu2(v.x & m, v.y & m), vmaxu2(v.z & m, v.w & m));
}

template <bool BF16>
__device__ __forceinline__ float magnitude(uint32_t bits) {
    if constexpr (BF16) return __uint_as_float(bits << 16);
    return __half2float(__ushort_as_half((unsigned short)bits));
}

struct RowScale {
    float inv;  // RN(127 / (a pre)); 0 for a row of zeros, or one that holds an infinity or NaN
    float pre;  // bf16: 2^64 for a below 2^-60, where 127 / a would overflow; else 1
    bool live;  // some value is not zero and all are finite
};

template <bool BF16>
__device__ __forceinline__ RowScale row_scale(uint32_t top, float* scale) {
    const float a = magnitude<BF16>(top);
    RowScale r;
    r.live = top != 0u && top < (BF16 ? 0x7f80u : 0x7c00u);
    r.pre = BF16 && a < 0x1p-60f ? 0x1p64f : 1.f;
    r.inv = r.live ? __fdiv_rn(127.f, a * r.pre) : 0.f;
    if (scale) *scale = __fdiv_rn(a, 127.f);
    return r;
}

// The low byte is the int8 value; x a finite value of a live row.
template <bool BF16>
__device__ __forceinline__ uint32_t quantize(float x, const RowScale& r) {
    const float p = __fmul_rn(BF16 ? x * r.pre : x, r.inv);
    const float c = __fmul_rn(17.f, p);  // 2^4 + 1: the high 20 of 24 bits, rounded to nearest (Dekker, 1971)
    const float hi = __fsub_rn(c, __fsub_rn(c, p));
    return __float_as_uint(__fadd_rn(hi, 12582912.f));  // 1.5 2^23: the integer, ties to even, in the low bits
}

template <bool BF16>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
    if constexpr (BF16) {
        lo = __uint_as_float(w << 16);
        hi = __uint_as_float(w & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
        lo = f.x;
        hi = f.y;
    }
}

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __byte_perm(__byte_perm(a, b, 0x0040u), __byte_perm(c, d, 0x0040u), 0x5410u);
}

template <bool BF16>
__device__ __forceinline__ uint2 quantize8(uint4 v, const RowScale& r) {
    if (!r.live) return make_uint2(0u, 0u);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t q[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float lo, hi;
        unpack2<BF16>(w[i], lo, hi);
        q[2 * i] = quantize<BF16>(lo, r);
        q[2 * i + 1] = quantize<BF16>(hi, r);
    }
    return make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
}

}  // namespace spmm24
