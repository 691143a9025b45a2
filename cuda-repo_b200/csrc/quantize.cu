// quantize.cu -- 16-bit rows -> int8 rows and one scale per row: the
// activations of spmm24_launch_int8 (a row = a token), and its weights (a row
// = an output channel).
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
//
// Bound by the bytes: 2 read and 1 written for each element, each row read
// once (its elements wait in registers for the row's maximum).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "ptx_sm100.cuh"
#include "spmm24/SpMM_API.h"
#include "spmm24_host.h"

namespace spmm24 {
namespace {

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

// Maximum of `v` over the block (its low and high half-words are candidates);
// every thread gets it.
__device__ __forceinline__ uint32_t block_max(uint32_t v, uint32_t* s) {
    v = __reduce_max_sync(0xffffffffu, max(v & 0xffffu, v >> 16));
    const int warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
    if ((threadIdx.x & 31) == 0) s[warp] = v;
    __syncthreads();
    const int lane = threadIdx.x & 31;
    return __reduce_max_sync(0xffffffffu, lane < warps ? s[lane] : 0u);
}

// Eight elements of a row from element k on; elements past `cols` are zero.
template <bool VEC>
__device__ __forceinline__ uint4 load8(const uint16_t* row, int k, int cols) {
    if constexpr (VEC) {
        return *reinterpret_cast<const uint4*>(row + k);
    } else {
        uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < cols) w[e >> 1] |= (uint32_t)row[k + e] << (16 * (e & 1));
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(int8_t* row, int k, int cols, uint2 q) {
    if constexpr (VEC) {
        *reinterpret_cast<uint2*>(row + k) = q;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (k + e < cols) row[k + e] = (int8_t)((e < 4 ? q.x : q.y) >> (8 * (e & 3)));
    }
}

constexpr int kHeld = 4;  // groups of eight elements that a thread holds in registers

// One row per block.  A thread's groups lie blockDim apart; what does not fit
// in registers (rows of more than 32 blockDim elements) is read again, out of
// L2.
template <bool BF16, bool VEC>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const uint16_t* __restrict__ x, long long ld, int cols,
                                                             int8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ uint32_t warp_max[32];
    ptx::grid_dep_wait();  // launched with programmatic serialization: the previous grid may write the input
    if (threadIdx.x == 0) ptx::grid_dep_launch();
    const uint16_t* row = x + (long long)blockIdx.x * ld;
    int8_t* out = q + (long long)blockIdx.x * cols;
    const int groups = (cols + 7) / 8, step = blockDim.x;
    uint4 v[kHeld];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int g = (int)threadIdx.x + i * step;
        v[i] = g < groups ? load8<VEC>(row, 8 * g, cols) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < kHeld; ++i) m = vmaxu2(m, abs_max8(v[i]));
    for (int g = (int)threadIdx.x + kHeld * step; g < groups; g += step) m = vmaxu2(m, abs_max8(load8<VEC>(row, 8 * g, cols)));
    const RowScale r = row_scale<BF16>(block_max(m, warp_max), threadIdx.x == 0 ? scale + blockIdx.x : nullptr);
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const int g = (int)threadIdx.x + i * step;
        if (g < groups) store8<VEC>(out, 8 * g, cols, quantize8<BF16>(v[i], r));
    }
    for (int g = (int)threadIdx.x + kHeld * step; g < groups; g += step)
        store8<VEC>(out, 8 * g, cols, quantize8<BF16>(load8<VEC>(row, 8 * g, cols), r));
}

// One strip of eight rows (packed B: cols x 8 elements) per block.  A thread
// takes eight consecutive columns of all eight rows: 128 bytes in, eight bytes
// of each row out.  The first such group waits in registers, the others are
// read again, out of L2.
template <bool BF16>
__global__ void __launch_bounds__(1024) quantize_strips_kernel(const uint16_t* __restrict__ x, int rows, int cols,
                                                               int8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ uint32_t part[32][8];
    __shared__ uint32_t top[8];
    ptx::grid_dep_wait();
    if (threadIdx.x == 0) ptx::grid_dep_launch();
    const uint4* strip = reinterpret_cast<const uint4*>(x) + (size_t)blockIdx.x * cols;  // one uint4 per column
    const int groups = cols / 8, row0 = (int)blockIdx.x * 8;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint4 v[8];
    const bool first = (int)threadIdx.x < groups;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = first ? strip[8 * threadIdx.x + i] : make_uint4(0u, 0u, 0u, 0u);
    uint32_t m[4] = {0u, 0u, 0u, 0u};  // rows 2i (low) and 2i + 1 (high)
    auto fold = [&](uint4 w) {
        m[0] = vmaxu2(m[0], w.x & 0x7fff7fffu);
        m[1] = vmaxu2(m[1], w.y & 0x7fff7fffu);
        m[2] = vmaxu2(m[2], w.z & 0x7fff7fffu);
        m[3] = vmaxu2(m[3], w.w & 0x7fff7fffu);
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) fold(v[i]);
    for (int c = 8 * (int)blockDim.x + (int)threadIdx.x; c < cols; c += (int)blockDim.x) fold(strip[c]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = __reduce_max_sync(0xffffffffu, m[i] & 0xffffu);
        const uint32_t hi = __reduce_max_sync(0xffffffffu, m[i] >> 16);
        if (lane == 0) {
            part[warp][2 * i] = lo;
            part[warp][2 * i + 1] = hi;
        }
    }
    __syncthreads();
    if (threadIdx.x < 8) {
        uint32_t t = 0u;
        for (int w = 0; w < (int)(blockDim.x + 31) / 32; ++w) t = max(t, part[w][threadIdx.x]);
        top[threadIdx.x] = t;
        if (row0 + (int)threadIdx.x < rows) row_scale<BF16>(t, scale + row0 + threadIdx.x);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < groups; g += blockDim.x) {
        if (g != (int)threadIdx.x) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = strip[8 * g + i];
        }
#pragma unroll
        for (int pair = 0; pair < 4; ++pair) {
            uint32_t lo[8], hi[8];
            const RowScale r0 = row_scale<BF16>(top[2 * pair], nullptr), r1 = row_scale<BF16>(top[2 * pair + 1], nullptr);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = pair == 0 ? v[i].x : pair == 1 ? v[i].y : pair == 2 ? v[i].z : v[i].w;
                float a, b;
                unpack2<BF16>(w, a, b);
                lo[i] = quantize<BF16>(a, r0);
                hi[i] = quantize<BF16>(b, r1);
            }
            const int row = row0 + 2 * pair;
            if (row < rows)
                *reinterpret_cast<uint2*>(q + (size_t)row * cols + 8 * g) =
                    r0.live ? make_uint2(pack4(lo[0], lo[1], lo[2], lo[3]), pack4(lo[4], lo[5], lo[6], lo[7]))
                            : make_uint2(0u, 0u);
            if (row + 1 < rows)
                *reinterpret_cast<uint2*>(q + (size_t)(row + 1) * cols + 8 * g) =
                    r1.live ? make_uint2(pack4(hi[0], hi[1], hi[2], hi[3]), pack4(hi[4], hi[5], hi[6], hi[7]))
                            : make_uint2(0u, 0u);
        }
    }
}

template <class... KArgs, class... Args>
cudaError_t launch(void (*kern)(KArgs...), unsigned blocks, unsigned threads, cudaStream_t stream, bool pdl, Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
}

}  // namespace
}  // namespace spmm24

extern "C" cudaError_t spmm24_quantize_int8(cudaStream_t stream, const void* x, int rows, int cols, long long ld,
                                            int layout, unsigned flags, void* q, float* scale) {
    using namespace spmm24;
    clear_last_error();
    if (!x || !q || !scale) return record_invalid("null pointer");
    if (rows <= 0 || cols <= 0) return record_invalid("rows and cols must be positive");
    if (flags & ~(unsigned)(SPMM24_BF16 | SPMM24_NO_PDL)) return record_invalid("unknown flag");
    if (layout != SPMM24_OUT_ROW_MAJOR && layout != SPMM24_OUT_PACKED_B) return record_invalid("unknown input layout");
    if ((uintptr_t)x & 1u) return record_invalid("x must be 2-byte aligned");
    if ((uintptr_t)scale & 3u) return record_invalid("scale must be 4-byte aligned");
    const bool bf16 = flags & SPMM24_BF16, pdl = !(flags & SPMM24_NO_PDL);
    const int groups = (cols + 7) / 8;
    const uint16_t* xp = static_cast<const uint16_t*>(x);
    int8_t* qp = static_cast<int8_t*>(q);
    if (layout == SPMM24_OUT_PACKED_B) {
        if (ld != 0) return record_invalid("packed rows have no row stride: ld must be 0");
        if (cols % 8) return record_invalid("packed rows: cols must be a multiple of 8");
        if (((uintptr_t)x & 15u) || ((uintptr_t)q & 7u))
            return record_invalid("packed rows: x must be 16-byte and q 8-byte aligned");
        const unsigned threads = (unsigned)(groups < 512 ? (groups + 31) / 32 * 32 : 512);
        const unsigned blocks = (unsigned)(((long long)rows + 7) / 8);
        return bf16 ? launch(quantize_strips_kernel<true>, blocks, threads, stream, pdl, xp, rows, cols, qp, scale)
                    : launch(quantize_strips_kernel<false>, blocks, threads, stream, pdl, xp, rows, cols, qp, scale);
    }
    if (ld == 0) ld = cols;
    if (ld < cols) return record_invalid("ld must be 0 or at least cols");
    const bool vec = cols % 8 == 0 && ld % 8 == 0 && ((uintptr_t)x & 15u) == 0 && ((uintptr_t)q & 7u) == 0;
    unsigned threads = (unsigned)((groups + 32 * kHeld - 1) / (32 * kHeld) * 32);
    if (threads > 1024) threads = 1024;
    if (bf16)
        return vec ? launch(quantize_rows_kernel<true, true>, (unsigned)rows, threads, stream, pdl, xp, ld, cols, qp, scale)
                   : launch(quantize_rows_kernel<true, false>, (unsigned)rows, threads, stream, pdl, xp, ld, cols, qp, scale);
    return vec ? launch(quantize_rows_kernel<false, true>, (unsigned)rows, threads, stream, pdl, xp, ld, cols, qp, scale)
               : launch(quantize_rows_kernel<false, false>, (unsigned)rows, threads, stream, pdl, xp, ld, cols, qp, scale);
}
