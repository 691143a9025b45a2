// quantize.cu -- 16-bit rows -> int8 rows and one scale per row: the
// activations of spmm24_launch_int8 (a row = a token), and its weights (a row
// = an output channel).
//
//   a = max_k |x_k|,  scale = a / 127,  q_k = rint(127 x_k / a)  (ties to even)
//
// exactly (int8_rows.cuh says how).
//
// Bound by the bytes: 2 read and 1 written for each element, each row read
// once (its elements wait in registers for the row's maximum).
#include <cuda_runtime.h>

#include <cstdint>

#include "int8_rows.cuh"
#include "ptx_sm100.cuh"
#include "spmm24/SpMM_API.h"
#include "spmm24_host.h"

namespace spmm24 {
namespace {

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

// One row per block.  A thread holds HELD groups of eight elements in
// registers, blockDim apart; what does not fit (rows of more than 65536 elements)
// is read again, out of L2.  HELD 4 up to 8192 columns, 8 above: 4096 x 4096 9.9
// and 9.7 us, 148 x 4096 1.5 and 1.9; 4096 x 11008 28.6 and 25.4, 2048 x 28672
// 46.1 and 36.4 (more bytes in flight for a row; fewer warps for a short one).
template <bool BF16, bool VEC, int HELD>
__global__ void __launch_bounds__(1024) quantize_rows_kernel(const uint16_t* __restrict__ x, long long ld, int cols,
                                                             int8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ uint32_t warp_max[32];
    ptx::grid_dep_wait();  // launched with programmatic serialization: the previous grid may write the input
    if (threadIdx.x == 0) ptx::grid_dep_launch();
    const uint16_t* row = x + (long long)blockIdx.x * ld;
    int8_t* out = q + (long long)blockIdx.x * cols;
    const int groups = (cols + 7) / 8, step = blockDim.x;
    uint4 v[HELD];
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int g = (int)threadIdx.x + i * step;
        v[i] = g < groups ? load8<VEC>(row, 8 * g, cols) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i) m = vmaxu2(m, abs_max8(v[i]));
    for (int g = (int)threadIdx.x + HELD * step; g < groups; g += step) m = vmaxu2(m, abs_max8(load8<VEC>(row, 8 * g, cols)));
    const RowScale r = row_scale<BF16>(block_max(m, warp_max), threadIdx.x == 0 ? scale + blockIdx.x : nullptr);
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        const int g = (int)threadIdx.x + i * step;
        if (g < groups) store8<VEC>(out, 8 * g, cols, quantize8<BF16>(v[i], r));
    }
    for (int g = (int)threadIdx.x + HELD * step; g < groups; g += step)
        store8<VEC>(out, 8 * g, cols, quantize8<BF16>(load8<VEC>(row, 8 * g, cols), r));
}

// One strip of eight rows (packed B: cols x 8 elements) per cluster, an equal
// part of its columns per CTA; the CTAs exchange their eight maxima through
// distributed shared memory.  A thread takes eight consecutive columns of all
// eight rows: 128 bytes in, eight bytes of each row out.  The first such group
// waits in registers, the others (more than 4096 columns a CTA) are read again,
// out of L2.  (A column per lane, and a byte transpose across eight lanes for the
// stores, measured the same.)
constexpr int kMaxStripCtas = 8;

template <bool BF16>
__global__ void __launch_bounds__(512, 2) quantize_strips_kernel(const uint16_t* __restrict__ x, int rows, int cols,
                                                              int8_t* __restrict__ q, float* __restrict__ scale) {
    __shared__ uint32_t part[16][8];
    __shared__ uint32_t tops[kMaxStripCtas][8];
    __shared__ RowScale rs[8];
    const int ctas = (int)ptx::cluster_nctarank(), rank = (int)ptx::cluster_ctarank();
    // "This CTA runs", awaited before the first store into another's shared
    // memory; the loads pass meanwhile.  It orders no writes (a releasing arrival cost
    // 3 of 41 us at 4096 x 11008).
    if (ctas > 1) ptx::cluster_arrive_relaxed();
    ptx::grid_dep_wait();
    if (threadIdx.x == 0) ptx::grid_dep_launch();
    const int strip_id = (int)blockIdx.x / ctas, row0 = strip_id * 8;
    const uint4* strip = reinterpret_cast<const uint4*>(x) + (size_t)strip_id * cols;  // one uint4 per column
    const int g0 = (int)((long long)(cols / 8) * rank / ctas), g1 = (int)((long long)(cols / 8) * (rank + 1) / ctas);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint4 v[8];
    uint32_t m[4] = {0u, 0u, 0u, 0u};  // rows 2i (low) and 2i + 1 (high)
    const int mine = g0 + (int)threadIdx.x;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = mine < g1 ? strip[8 * mine + i] : make_uint4(0u, 0u, 0u, 0u);
    auto fold = [&](uint4 w) {
        m[0] = vmaxu2(m[0], w.x & 0x7fff7fffu);
        m[1] = vmaxu2(m[1], w.y & 0x7fff7fffu);
        m[2] = vmaxu2(m[2], w.z & 0x7fff7fffu);
        m[3] = vmaxu2(m[3], w.w & 0x7fff7fffu);
    };
#pragma unroll
    for (int i = 0; i < 8; ++i) fold(v[i]);
    for (int c = 8 * (g0 + (int)blockDim.x) + (int)threadIdx.x; c < 8 * g1; c += (int)blockDim.x) fold(strip[c]);
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
    if (ctas > 1) ptx::cluster_wait_acquire();  // every CTA of the cluster runs
    if ((int)threadIdx.x < 8 * ctas) {  // this CTA's maxima into every CTA's slot of it
        const int j = threadIdx.x & 7, to = threadIdx.x >> 3;
        uint32_t t = 0u;
        for (int w = 0; w < (int)blockDim.x / 32; ++w) t = max(t, part[w][j]);
        ptx::st_cluster_u32(ptx::mapa_shared(ptx::smem_u32(&tops[rank][j]), (uint32_t)to), t);
    }
    ptx::cluster_sync();
    if (threadIdx.x < 8) {
        uint32_t t = 0u;
        for (int c = 0; c < ctas; ++c) t = max(t, tops[c][threadIdx.x]);
        const int row = row0 + (int)threadIdx.x;
        rs[threadIdx.x] = row_scale<BF16>(t, rank == 0 && row < rows ? scale + row : nullptr);
    }
    __syncthreads();
    for (int g = mine; g < g1; g += blockDim.x) {
        if (g != mine) {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = strip[8 * g + i];
        }
#pragma unroll
        for (int pair = 0; pair < 4; ++pair) {
            uint32_t lo[8], hi[8];
            const RowScale r0 = rs[2 * pair], r1 = rs[2 * pair + 1];
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
cudaError_t launch(void (*kern)(KArgs...), unsigned blocks, unsigned threads, unsigned cluster, cudaStream_t stream, bool pdl,
                   Args... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(blocks, 1, 1);
    cfg.blockDim = dim3(threads, 1, 1);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster ? 2 : 1;
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
    if (cols > 1 << 30) return record_invalid("cols must be at most 2^30");  // the kernels' column indices run past it
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
        // CTAs per strip: eight where strips are few (64 elements a thread are 1.2
        // us of arithmetic when one CTA has 4096 columns; up to eight CTAs an SM) or long
        // (registers hold 4096 columns a CTA), else as many as that leaves.  With 1, 2, 4
        // and 8: 16 x 4096 5.9, 4.2, 3.4, 3.1 us; 509 x 4096 6.1, 4.4, 4.1, 4.3; 4096 x
        // 4096 17.7, 16.2, 16.5, 18.9; 4096 x 11008 47, 48, 49, 41.
        const long long strips = ((long long)rows + 7) / 8;
        unsigned ctas = kMaxStripCtas;
        while (ctas > 1 && cols <= 4096 && (strips * ctas > 8LL * current_sms() || groups < 64 * (int)ctas)) ctas /= 2;
        const int each = (groups + (int)ctas - 1) / (int)ctas;
        const unsigned threads = (unsigned)(each < 512 ? (each + 31) / 32 * 32 : 512);
        if (strips * ctas > 0x7fffffffLL) return record_invalid("packed rows: too many rows");
        const unsigned blocks = (unsigned)(strips * ctas);
        return bf16 ? launch(quantize_strips_kernel<true>, blocks, threads, ctas, stream, pdl, xp, rows, cols, qp, scale)
                    : launch(quantize_strips_kernel<false>, blocks, threads, ctas, stream, pdl, xp, rows, cols, qp, scale);
    }
    if (ld == 0) ld = cols;
    if (ld < cols) return record_invalid("ld must be 0 or at least cols");
    const bool vec = cols % 8 == 0 && ld % 8 == 0 && ((uintptr_t)x & 15u) == 0 && ((uintptr_t)q & 7u) == 0;
    const int held = cols > 8192 ? 8 : 4;
    unsigned threads = (unsigned)((groups + 32 * held - 1) / (32 * held) * 32);
    if (threads > 1024) threads = 1024;
    auto go = [&](auto kern) { return launch(kern, (unsigned)rows, threads, 0u, stream, pdl, xp, ld, cols, qp, scale); };
    if (held == 8) {
        if (bf16) return vec ? go(quantize_rows_kernel<true, true, 8>) : go(quantize_rows_kernel<true, false, 8>);
        return vec ? go(quantize_rows_kernel<false, true, 8>) : go(quantize_rows_kernel<false, false, 8>);
    }
    if (bf16) return vec ? go(quantize_rows_kernel<true, true, 4>) : go(quantize_rows_kernel<true, false, 4>);
    return vec ? go(quantize_rows_kernel<false, true, 4>) : go(quantize_rows_kernel<false, false, 4>);
}
