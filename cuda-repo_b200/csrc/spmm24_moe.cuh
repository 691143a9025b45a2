// spmm24_moe.cuh -- a whole mixture-of-experts layer for a few tokens (T <= 32)
// in one persistent launch, 2:4-sparse experts in fp16, bf16 or int8.
//
//   l[t, e] = sum_i router[e, i] x[t, i]              (fp32)
//   E_t     = the k largest l[t, .], ties to the lower expert
//   w[t, j] = softmax(l[t, .])[E_t[j]], optionally divided by their sum
//   h[t, j] = act(Wg_e x_t) * (Wu_e x_t)              e = E_t[j]
//   y[t]    = sum_j w[t, j] Wd_e h[t, j]
//
// int8 experts: x_t is rounded to int8 with its own scale (int8_rows.cuh),
// every h[t, j] likewise with the scale of its own largest value, products are
// exact 32-bit sums times the channel's and the row's scale.  16-bit experts:
// h is rounded once to the operand type, which a 16-bit product needs.
//
// Bound by the chosen experts' weights, each read once: 3 I H values of 9/8
// (16-bit) or 5/8 bytes per expert that some token chose.  So one CTA per SM
// streams weights through a TMA ring without a stop, as the grouped kernel
// does, and everything else is arranged around that:
//
//   - All T tokens are the columns of every product (an expert's other columns
//     are not used): no gather, and the x or h tile is the same for every
//     expert; 16 or 32 columns cost the tensor core nothing beside the stream.
//   - Work is cut into K stages, not tiles: the gate / up phase has (expert,
//     128 rows, stage) units, the down phase (128 rows, expert, stage) ones,
//     and every CTA takes an equal run of them, whatever the routing.  A tile
//     that several CTAs share is summed from their fp32 (int8: integer) partials
//     in the workspace, in the order of the K stages, each of them taking an
//     equal part of its rows, so results do not depend on timing.
//   - h has to be complete (int8: and rounded, which needs each row's largest
//     value first) before a down product reads it: grid barriers (cooperative
//     launch: all CTAs are resident).  The stream does not stop for them: the
//     experts in use go in two groups A and B, gate / up of A, gate / up of B,
//     down of A, down of B, and a group's barriers pass while the other's
//     weights stream; the ring is filled ahead of each.
//   - Routing weights multiply the down products in fp32, expert by expert, as
//     they leave TMEM; h stays unscaled.
//
// Roles (192 threads) as in the grouped kernel: warp 0 TMA producer, warp 1
// MMA issuer, warps 2-5 epilogue; before that all warps compute the router.
// Every wait is bounded; one that gives up records a status bit and its role
// stops, the others then give up in turn, TMEM is freed.
//
// Measured, E = 8, k = 2, 4096 x 11008: 1 token fp16 61 us (304 MB, 5.0 TB/s;
// floor 46.5 at the copy rate), int8 54 (169 MB, 3.1; 25.8), 32 tokens int8 140
// (676 MB, 4.8; 103); E = 64, k = 8, 2048 x 1024, 8 tokens bf16 70 (297 MB, 4.2;
// 45.4); E = 5, k = 2, 1024 x 640, 3 tokens 19 (latency).  The weight stream runs
// at 6.0 TB/s; the rest is the front (routing known after 5 us, int8 6, of many
// experts 8, and a first load of 2), the int8 rows' barriers where a group's stream is
// too short to hide them (a message through L2 takes 1-2 us while it is full),
// and the last partials (3-4 us).
#pragma once
#include <cstddef>

#include "int8_rows.cuh"
#include "spmm24_common.cuh"

namespace spmm24 {

constexpr int kMoeMaxTokens = 32;
constexpr int kMoeMaxExperts = 256;
constexpr int kMoeMaxTopK = 16;
constexpr int kMoeMaxCtas = 160;
constexpr int kMoeMaxTiles = 32768;  // (expert, 128 rows of I) tiles of the gate / up phase
constexpr int kMoeMaxShares = 4;  // K shares of a logit
constexpr int kMoeSplitUnits = 8;  // gate / up units per CTA from which the experts go in two groups
constexpr int kMoeWarps = kThreads / 32;
// Experts of a CTA's gate / up run, one for each epilogue warp: as long as there are at
// most three experts in use a CTA, a run is as long as three experts at most, and meets
// four (the host refuses more; 256 experts need 86 SMs).
constexpr int kMoeRunExperts = kEpiThreads / 32;

struct MoeParams {
    CUtensorMap tmGU, tmGUE;  // gate and up weights of all experts: values, metadata
    CUtensorMap tmD, tmDE;    // down weights
    CUtensorMap tmX, tmH;     // the products' B operands: x (int8: its rounded rows), h
    const uint16_t* x;        // packed strips
    const uint16_t* router;   // E x H, or null: ids and weights are given
    int* ids;                 // T x k
    float* weights;
    const float* gu_scale;    // int8: E x 2I, E x H
    const float* d_scale;
    uint16_t* y;
    Epilogue epi;             // M = H, N = T
    int T, H, I, E, k;
    int strips;               // ceil(T / 8)
    int act, norm, bf16;
    int max_slots;            // min(E, T k): experts that can be in use
    int logit_shares;         // K shares of a logit
    // workspace
    uint32_t* bar;            // arrivals at the grid barrier
    uint32_t* epoch;          // launches so far: the tags of this launch's partials
    float* logits;            // [share][T][E]
    uint64_t* part;           // [CTA][2][32 column pairs][128 rows][2] {value, tag}
    uint32_t* amax;           // int8: [slot][32] largest |h| (bits)
    float* xscale;            // int8: [32]
    int8_t* xq;               // int8: T x H
    float* h32;               // int8: [slot][T][I]
    int8_t* hq;               // int8: [slot][T][I]
    uint16_t* h16;            // 16-bit: [slot][strips][I][8]
    SPMM24_TRACE_FIELD
};

constexpr int kMoeSharedBytes = 6880 + 4 * 768;
constexpr int kMoeKeptLogits = 768;
constexpr int moe_stages(int n_tile, bool i8) { return n_tile == 16 ? 9 : i8 ? 7 : 8; }

template <int N_TILE, bool I8>
struct MoeCfg : Cfg<N_TILE, moe_stages(N_TILE, I8), 4, I8> {
    static constexpr int STAGES = moe_stages(N_TILE, I8);
    using B_ = Cfg<N_TILE, STAGES, 4, I8>;
    static constexpr int BAR_OFFSET = B_::RING_BYTES;
    static constexpr int NUM_BARS = 2 * STAGES + 4;  // full, empty, acc_full[2], acc_empty[2]
    static constexpr int AUX_OFFSET = (BAR_OFFSET + NUM_BARS * 8 + 15) / 16 * 16;
    static constexpr int SMEM_BYTES = AUX_OFFSET + kMoeSharedBytes;
    static constexpr int SMEM_ALLOC = SMEM_BYTES + 1024;  // slack to align the base to 1024 B
    static_assert(SMEM_ALLOC <= 232448, "shared memory overflow");
    static_assert(B_::STAGE_BYTES % 1024 == 0, "stages must stay 1024-byte aligned");
};

// Routing and small state in shared memory.
struct MoeShared {
    int ids[kMoeMaxTokens * kMoeMaxTopK];        // -1: no expert
    float weights[kMoeMaxTokens * kMoeMaxTopK];
    uint32_t mask[kMoeMaxExperts];               // tokens of each expert
    uint16_t list[kMoeMaxExperts];               // experts in use, in increasing order
    uint8_t slot[kMoeMaxExperts];                // an expert's place there
    float xscale[kMoeMaxTokens];
    uint32_t hmax[kMoeRunExperts][kMoeMaxTokens];  // int8: largest |h| (bits) in this CTA's rows, its run's experts
    uint32_t red[kMoeWarps][8];
    uint32_t top[kMoeMaxTokens];
    uint32_t tmem, base, epoch, n_active, last, dead;
    alignas(16) float logits[kMoeKeptLogits];    // the logits, where they fit; read four at a time
};
static_assert(sizeof(MoeShared) <= kMoeSharedBytes, "MoeCfg reserves its bytes");
static_assert(offsetof(MoeShared, logits) % 16 == 0, "read as float4");

// ------------------------------------------------------------ grid barrier
// One word that counts arrivals, `ctas` per barrier, and wraps at a multiple
// of that (so it stays a multiple between launches).  Before a CTA's own first
// arrival the launch's first barrier cannot be over, so the word then read,
// rounded down to a multiple, is the launch's base, and its n-th barrier is
// over once the count has reached base + n ctas.  One atomic and one poll:
// 1.5 us, where a count that the last CTA resets before it publishes a
// generation takes three round trips (2.3 us).
__device__ __forceinline__ uint32_t moe_wrap(uint32_t ctas) { return ctas << 20; }
// One thread, after a barrier of the block's threads: its fence covers their
// writes.
__device__ __forceinline__ void moe_arrive(uint32_t* bar, uint32_t ctas) {
    __threadfence();
    atomicInc(bar, moe_wrap(ctas) - 1u);
}
__device__ __forceinline__ bool moe_wait(const uint32_t* bar, uint32_t base, uint32_t n, uint32_t ctas) {
    const uint32_t wrap = moe_wrap(ctas);
    uint32_t target = base + n * ctas;
    if (target >= wrap) target -= wrap;
    const uint64_t t0 = ptx::globaltimer();
    uint32_t spins = 0;
    while (true) {
        const uint32_t c = ptx::ld_acquire_gpu(bar);
        if ((c >= target ? c - target : c + wrap - target) < wrap / 2) return true;
        if ((++spins & 255u) == 0u && ptx::globaltimer() - t0 > kWaitLimitNs) {
            atomicOr(&g_spmm24_status, kStatusBarrierTimeout);
            return false;
        }
    }
}

// An equal run of the units 0 .. U - 1 for each CTA: q or (the first r CTAs)
// q + 1 of them.
struct MoeRuns {
    int units, ctas, q, r;  // ctas <= units
    __device__ __forceinline__ MoeRuns(int units_, int grid)
        : units(units_), ctas(min(grid, units_)), q(ctas ? units / ctas : 0), r(units - q * ctas) {}
    __device__ __forceinline__ int begin(int cta) const { return cta < ctas ? cta * q + min(cta, r) : units; }
    __device__ __forceinline__ int owner(int unit) const {
        const int big = r * (q + 1);
        return unit < big ? unit / (q + 1) : r + (unit - big) / q;
    }
};

// SiLU y sigmoid(y), and GELU's tanh form 0.5 y (1 + tanh z) as y sigmoid(2 z),
// to a few steps of fp32 beside the value itself: y / (1 + e^-x), and y e^x where x is so
// low that e^-x could overflow (1 + e^x is 1 there).  expf and the division are
// the exact kinds: the few values of this layer are no load, and h, which is rounded
// next, takes another value wherever it crosses a border.  GELU's x has seven
// roundings of its own (2^-24 each), which e^-x sees |x| times.
__device__ __forceinline__ float moe_activate(float y, int act) {
    if (act == kActRelu) return y > 0.f || y != y ? y : 0.f;
    if (act != kActSilu && act != kActGelu) return y;
    const float x = act == kActSilu ? y : 1.5957691216057308f * (y + 0.044715f * y * y * y);
    const bool low = x < -80.f;
    const float e = expf(low ? x : -x);
    return low ? y * e : y / (1.f + e);
}

// int8: h -> rint(127 h / a), ties to even, exactly, for fp32 |h| <= a; inv =
// RN(127 / a).  The product h inv is off by its own rounding and inv's, each
// 2^-24 of at most 127: less than 2^-16 together.  So it names the integer unless it
// lies that near to a tie k + 1/2 (one value in 2^14); there 254 |h| against (2k + 1) a
// decides, products of 24 and 8 bits that doubles hold.
__device__ __forceinline__ uint32_t moe_round_h(float h, float a, float inv) {
    const float p = fabsf(h) * inv;
    float q = rintf(p);
    if (fabsf(fabsf(p - q) - 0.5f) < 0x1p-15f) {
        const float k = floorf(p);
        const double d = 254.0 * (double)fabsf(h) - (2.0 * (double)k + 1.0) * (double)a;
        q = d > 0.0 || (d == 0.0 && ((int)k & 1)) ? k + 1.f : k;
    }
    return (uint32_t)(int)copysignf(q, h);
}

// ------------------------------------------------------------------ router
// Unit (expert, strip of eight tokens, K share): a block, eight partial
// logits.  A lane takes eight consecutive inputs at a time.  Shares of about
// one load per lane, summed over the block's warps here, leave few values to
// add per logit after the grid barrier, where latency counts.
template <bool BF16>
__device__ __forceinline__ void moe_router(const MoeParams& p, MoeShared& sh, int unit0, int step) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int shares = p.logit_shares, groups = p.H / 8, units = p.E * p.strips * shares;
    for (int it = unit0; it < units; it += step) {
        const int ks = it % shares, s = it / shares % p.strips, e = it / shares / p.strips;
        const uint4* wrow = reinterpret_cast<const uint4*>(p.router + (size_t)e * p.H);
        const uint4* xs = reinterpret_cast<const uint4*>(p.x) + (size_t)s * p.H;
        float acc[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) acc[t] = 0.f;
        const int g1 = (int)((long long)groups * (ks + 1) / shares);
        for (int g = (int)((long long)groups * ks / shares) + (int)threadIdx.x; g < g1; g += kThreads) {
            const uint4 w4 = wrow[g];
            uint4 xv[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) xv[i] = xs[8 * g + i];
            const uint32_t w[4] = {w4.x, w4.y, w4.z, w4.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float w0, w1;
                unpack2<BF16>(w[i >> 1], w0, w1);
                const float wi = i & 1 ? w1 : w0;
                const uint32_t xw[4] = {xv[i].x, xv[i].y, xv[i].z, xv[i].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float a, b;
                    unpack2<BF16>(xw[q], a, b);
                    acc[2 * q] = fmaf(wi, a, acc[2 * q]);
                    acc[2 * q + 1] = fmaf(wi, b, acc[2 * q + 1]);
                }
            }
        }
        // eight sums over 32 lanes, halving the values with the lanes: the
        // lane ends with the sum of token 4 (lane / 16) + 2 (lane / 8 % 2) + lane / 4 % 2
#pragma unroll
        for (int n = 4, o = 16; n; n >>= 1, o >>= 1) {
#pragma unroll
            for (int t = 0; t < n; ++t) {
                const float give = lane & o ? acc[t] : acc[t + n], keep = lane & o ? acc[t + n] : acc[t];
                acc[t] = keep + __shfl_xor_sync(0xffffffffu, give, o);
            }
        }
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 2);
        acc[0] += __shfl_xor_sync(0xffffffffu, acc[0], 1);
        if ((lane & 3) == 0) sh.red[warp][lane >> 2] = __float_as_uint(acc[0]);
        __syncthreads();
        const int t = 8 * s + (int)threadIdx.x;
        if (threadIdx.x < 8 && t < p.T) {
            float l = 0.f;
            for (int w = 0; w < kMoeWarps; ++w) l += __uint_as_float(sh.red[w][threadIdx.x]);
            p.logits[((size_t)ks * p.T + t) * p.E + e] = l;
        }
        __syncthreads();  // sh.red is free again
    }
}

// A logit's key: keys order as the logits do, NaN above all (it then makes
// every weight of its token NaN) and below 2^32 - 1; -0 and +0 are a tie.
__device__ __forceinline__ uint32_t moe_key(float v) {
    const uint32_t b = __float_as_uint(v + 0.f);
    return v != v ? 0xfffffffeu : (b & 0x80000000u) ? ~b : b | 0x80000000u;
}

// Top k of every token, by rank: an expert's place is the number of its
// token's experts that come before it, and those of the first k places write
// themselves down.  A thread per (token, expert), each against all: choosing
// one after another is a chain of warp reductions (T = 8, E = 64, k = 8: 6.6 us
// against 1 for this).  l, key: [T][pitch] logits and keys in shared memory,
// padded with -inf and keys 0.  All threads.
__device__ __forceinline__ void moe_top_k(const MoeParams& p, MoeShared& sh, const float* l, const uint32_t* key,
                                          int pitch) {
    const int n = p.T * p.E;
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const int t = i / p.E, e = i - t * p.E;
        const uint4* row = reinterpret_cast<const uint4*>(key + t * pitch);
        const uint32_t mine = key[t * pitch + e];
        int place = 0;
#pragma unroll 4
        for (int g = 0; g < pitch / 4; ++g) {
            const uint4 v = row[g];
            // before this one: the larger, and of the equal those to its left
            place += (v.x >= mine + (4 * g >= e)) + (v.y >= mine + (4 * g + 1 >= e)) + (v.z >= mine + (4 * g + 2 >= e)) +
                     (v.w >= mine + (4 * g + 3 >= e));
        }
        if (place < p.k) {
            sh.ids[t * p.k + place] = e;
            if (place == 0) sh.top[t] = __float_as_uint(l[t * pitch + e]);
            atomicOr(&sh.mask[e], 1u << t);
        }
    }
}

// The chosen experts' weights, a thread for each, out of the logits l (EXP: out
// of exp(l - largest)).  thread, threads: the caller's place among those that
// take part.
template <bool EXP>
__device__ __forceinline__ void moe_weights(const MoeParams& p, MoeShared& sh, const float* l, int pitch, int thread,
                                            int threads, bool publish) {
    for (int i = thread; i < p.T * p.k; i += threads) {
        const int t = i / p.k;
        const float* lt = l + t * pitch;
        const float top = __uint_as_float(sh.top[t]);
        auto e_of = [&](float x) { return EXP ? x : expf(x - top); };
        float sum = 0.f;
        if (p.norm) {
            for (int j = 0; j < p.k; ++j) sum += e_of(lt[sh.ids[t * p.k + j]]);
        } else {
            float4 s4 = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
            for (int e = 0; e < pitch; e += 4) {
                const float4 x = *reinterpret_cast<const float4*>(lt + e);
                s4 = make_float4(s4.x + e_of(x.x), s4.y + e_of(x.y), s4.z + e_of(x.z), s4.w + e_of(x.w));
            }
            sum = (s4.x + s4.y) + (s4.z + s4.w);
        }
        const float w = e_of(lt[sh.ids[i]]) / sum;
        sh.weights[i] = w;
        if (publish) {
            if (p.ids) p.ids[i] = sh.ids[i];
            if (p.weights) p.weights[i] = w;
        }
    }
}

// int8: x -> int8 rows.  Unit (strip, one of `parts` column ranges): a block.
// Every block finds its strip's eight maxima (the strip comes out of L2), then
// rounds its own columns.
template <bool BF16>
__device__ __forceinline__ void moe_quantize_x(const MoeParams& p, MoeShared& sh, int unit, int parts) {
    const int s = unit / parts, part = unit % parts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint4* strip = reinterpret_cast<const uint4*>(p.x) + (size_t)s * p.H;
    const uint32_t abs2 = 0x7fff7fffu;
    uint32_t m[4] = {0u, 0u, 0u, 0u};
    for (int c0 = threadIdx.x; c0 < p.H; c0 += 12 * kThreads) {
        uint4 v[12];  // twelve loads in flight
#pragma unroll
        for (int i = 0; i < 12; ++i)
            v[i] = c0 + i * kThreads < p.H ? strip[c0 + i * kThreads] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
        for (int i = 0; i < 12; ++i) {
            m[0] = vmaxu2(m[0], v[i].x & abs2);
            m[1] = vmaxu2(m[1], v[i].y & abs2);
            m[2] = vmaxu2(m[2], v[i].z & abs2);
            m[3] = vmaxu2(m[3], v[i].w & abs2);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t lo = __reduce_max_sync(0xffffffffu, m[i] & 0xffffu);
        const uint32_t hi = __reduce_max_sync(0xffffffffu, m[i] >> 16);
        if (lane == 0) {
            sh.red[warp][2 * i] = lo;
            sh.red[warp][2 * i + 1] = hi;
        }
    }
    __syncthreads();
    if (threadIdx.x < 8) {
        uint32_t t = 0u;
        for (int w = 0; w < kMoeWarps; ++w) t = max(t, sh.red[w][threadIdx.x]);
        sh.top[threadIdx.x] = t;
        const int row = 8 * s + (int)threadIdx.x;
        if (part == 0 && row < p.T) row_scale<BF16>(t, p.xscale + row);
    }
    __syncthreads();
    const int groups = p.H / 8, g1 = (int)((long long)groups * (part + 1) / parts);
    for (int g = (int)((long long)groups * part / parts) + threadIdx.x; g < g1; g += kThreads) {
        uint4 v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = strip[8 * g + i];
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            if (8 * s + t >= p.T) break;
            const RowScale r = row_scale<BF16>(sh.top[t], nullptr);
            uint32_t q[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t w = t < 2 ? v[i].x : t < 4 ? v[i].y : t < 6 ? v[i].z : v[i].w;
                float a, b;
                unpack2<BF16>(w, a, b);
                q[i] = r.live ? quantize<BF16>(t & 1 ? b : a, r) : 0u;
            }
            *reinterpret_cast<uint2*>(p.xq + (size_t)(8 * s + t) * p.H + 8 * g) =
                make_uint2(pack4(q[0], q[1], q[2], q[3]), pack4(q[4], q[5], q[6], q[7]));
        }
    }
    __syncthreads();  // sh.red and sh.top are free again
}

// ------------------------------------------------------------------ stages
template <class C_>
__device__ __forceinline__ void moe_load_acts(uint8_t* st, uint64_t* bar, const CUtensorMap* tm, int slot, int strips,
                                              int s, uint64_t pol) {
    if constexpr (C_::kFp8) {  // rows [slot][token] of int8: two boxes of 128 bytes x N_TILE rows
        ptx::tma_load_3d(st + C_::A_BYTES, tm, bar, 256 * s, 0, slot, pol);
        ptx::tma_load_3d(st + C_::A_BYTES + C_::B_BYTES / 2, tm, bar, 256 * s + 128, 0, slot, pol);
    } else {
        ptx::tma_load_4d(st + C_::A_BYTES, tm, bar, 0, 2 * s, 0, slot * strips, pol);
    }
}

// The four sparse MMAs of one stage (mma_stage, mma_stage_fp8), with the
// activations of another slot of the ring: the up product reads the gate
// product's.
template <class C_, int N_TILE, bool I8>
__device__ __forceinline__ void moe_mma_stage(uint32_t st, uint32_t st_acts, uint32_t meta_col, uint32_t d_tmem,
                                              uint32_t accumulate, uint32_t fmt) {
    const uint32_t stB = st_acts + C_::A_BYTES, stE = st + C_::A_BYTES + C_::B_BYTES;
    ptx::tmem_cp_128x128b(meta_col, smem_desc(stE, 0, 128));
    if constexpr (I8) {
        constexpr uint32_t idesc = (make_idesc_fp8<N_TILE>() & ~kIdescF32) | kIdescInt8;
        ptx::tmem_cp_128x128b(meta_col + 4, smem_desc(stE + 2048, 0, 128));
#pragma unroll
        for (int j = 0; j < 4; ++j)
            ptx::mma_sp_i8(d_tmem, smem_desc(st + j * 4096, 2048, 128),
                           smem_desc_sw128(stB + (j >> 1) * (C_::B_BYTES / 2) + (j & 1) * 64), meta_col + 2 * j, idesc,
                           j ? 1u : accumulate);
    } else {
        const uint32_t idesc = make_idesc<N_TILE>() | fmt;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            ptx::mma_sp_f16(d_tmem, smem_desc(st + j * 2048, 4 * 2048, 128), smem_desc(stB + j * 512, 128, 2048),
                            meta_col + (j & 2), idesc | (uint32_t)(j & 1), j ? 1u : accumulate);
    }
}

template <int N_TILE>
__device__ __forceinline__ void moe_read_acc(uint32_t taddr, uint32_t (&v)[N_TILE]) {
#pragma unroll
    for (int c = 0; c < N_TILE; c += 16) ptx::tmem_ld_32x32b_x16(taddr + c, *reinterpret_cast<uint32_t(*)[16]>(v + c));
}

template <bool I8>
__device__ __forceinline__ uint32_t moe_add(uint32_t a, uint32_t b) {
    return I8 ? a + b : __float_as_uint(__uint_as_float(a) + __uint_as_float(b));
}

// int8: one warp's largest |h| of a token, to shared memory, for the CTA's run's
// nth expert (kMoeRunExperts of them at most): global atomics stall behind a full
// weight stream (0.5 us each), so there is one per token and expert, at the end of
// the run.
__device__ __forceinline__ void moe_note_max(MoeShared& sh, int nth, int t, float h) {
    // bits order as magnitudes, NaN above all
    const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(h) & 0x7fffffffu);
    if ((threadIdx.x & 31u) == 0u) atomicMax(&sh.hmax[nth][t], m);
}

// Two 64-bit words {value, tag, value, tag}: each word is read as it was
// written, so a word with the right tag holds its value -- the partial needs no
// fence, flag or counter (with those, a shared tile cost 5 us; so 2).
__device__ __forceinline__ void moe_put2(uint64_t* p, uint32_t a, uint32_t b, uint32_t tag) {
    asm volatile("st.relaxed.gpu.global.v2.b64 [%0], {%1, %2};" ::"l"(p), "l"((uint64_t)tag << 32 | a),
                 "l"((uint64_t)tag << 32 | b)
                 : "memory");
}
__device__ __forceinline__ void moe_get2(const uint64_t* p, uint64_t& a, uint64_t& b) {
    asm volatile("ld.relaxed.gpu.global.v2.b64 {%0, %1}, [%2];" : "=l"(a), "=l"(b) : "l"(p) : "memory");
}

// A tile that several CTAs share: every one of them writes its partial (the
// first T columns of every N_TILE of its NV, 32-bit words), and at the end of
// the phase, when all have written at about the same time, finishes an equal
// part of the tile's rows from all partials, added in K order.
struct MoeTile {
    int first, c0, c1;  // the tile's first unit; the CTAs that share it
    __device__ __forceinline__ MoeTile(const MoeRuns& runs, int tile, int stages)
        : first(tile * stages), c0(runs.owner(first)), c1(runs.owner(first + stages - 1)) {}
    // A CTA's run meets a shared tile at its begin (its slot 0) or, the first
    // CTA's where the tile is not the first of its run, at its end (slot 1).
    __device__ __forceinline__ int slot(const MoeRuns& runs, int c) const {
        return 2 * c + (c == c0 && runs.begin(c) < first ? 1 : 0);
    }
};
// 64-bit words of a gate / up partial (a down partial takes half of them).
constexpr size_t kMoeSlotWords = (size_t)kTileM * 2 * kMoeMaxTokens;
// Partials of the first group's down run lie behind those of the others.
constexpr size_t kMoePartWords = (size_t)kMoeMaxCtas * 3 * kMoeSlotWords;

// pairs: bit n, columns 2n and 2n + 1 of every N_TILE are wanted.
template <int N_TILE, int NV>
__device__ __forceinline__ void moe_put_partial(uint64_t* slot, const uint32_t (&v)[NV], int row, uint32_t pairs,
                                                uint32_t tag) {
    uint64_t* at = slot + (size_t)row * 2;
#pragma unroll
    for (int i = 0; i < NV; i += 2)
        if (pairs >> (i % N_TILE / 2) & 1u) moe_put2(at + (size_t)i * kTileM, v[i], v[i + 1], tag);
}
// Pairs of tokens with a member in `mask`.
__device__ __forceinline__ uint32_t moe_pairs(uint32_t mask) {
    uint32_t m = (mask | mask >> 1) & 0x55555555u;  // bit 2n -> bit n
    m = (m | m >> 1) & 0x33333333u;
    m = (m | m >> 2) & 0x0f0f0f0fu;
    m = (m | m >> 4) & 0x00ff00ffu;
    return (m | m >> 8) & 0xffffu;
}

// Sums NP column pairs (the words of columns col[n], col[n] + 1) of one row
// over `count` partials, BATCH of them in flight at once; slot(i): the i-th
// partial's words.  fold: the warp's lanes are 8 rows by 4 parts of the
// partials, whose sums lanes 0-7 then add in order -- for tiles of many
// partials, which each hold few rows of.  The order of the sum depends on the
// sizes and the routing alone.
template <int NP, int BATCH, bool INT, class Slot>
__device__ __forceinline__ void moe_sum_partials(int count, Slot&& slot, const int (&col)[NP], int row, uint32_t tag,
                                                 bool fold, uint32_t (&sum)[2 * NP], bool& ok) {
    const int part = fold ? (int)(threadIdx.x & 31u) >> 3 : 0;
    const int first = fold ? count * part / 4 : 0, last = fold ? count * (part + 1) / 4 : count;
#pragma unroll
    for (int n = 0; n < 2 * NP; ++n) sum[n] = 0u;
    uint64_t t0 = 0;
#pragma unroll 1
    for (int c = first; c < last; c += BATCH) {
        uint64_t x[BATCH][2 * NP];
        for (uint32_t polls = 1;; ++polls) {
            bool there = true;
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                if (c + i >= last) break;
                const uint64_t* at = slot(c + i) + (size_t)row * 2;
#pragma unroll
                for (int n = 0; n < NP; ++n) moe_get2(at + (size_t)col[n] * kTileM, x[i][2 * n], x[i][2 * n + 1]);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
#pragma unroll
                for (int n = 0; n < 2 * NP; ++n)
                    there = there && (c + i >= last || (uint32_t)(x[i][n] >> 32) == tag);
            if (there || !ok) break;
            ptx::nanosleep_ns(100);  // polls of every CTA at once would crowd out what they wait for
            if ((polls & 255u) == 0u) {
                const uint64_t now = ptx::globaltimer();
                if (!t0) t0 = now;
                if (now - t0 > kWaitLimitNs) {
                    atomicOr(&g_spmm24_status, kStatusEpilogueTimeout);
                    ok = false;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i)
            if (c + i < last) {
#pragma unroll
                for (int n = 0; n < 2 * NP; ++n) sum[n] = moe_add<INT>(sum[n], (uint32_t)x[i][n]);
            }
    }
    ok = __all_sync(0xffffffffu, ok);
    if (fold) {
#pragma unroll
        for (int n = 0; n < 2 * NP; ++n) {
            const uint32_t own = sum[n];
#pragma unroll
            for (int i = 1; i < 4; ++i) sum[n] = moe_add<INT>(sum[n], __shfl_down_sync(0xffffffffu, own, 8 * i));
        }
    }
}

template <int N_TILE, bool I8>
__global__ void __launch_bounds__(kThreads, 1) spmm24_moe_kernel(const __grid_constant__ MoeParams p) {
    using C_ = MoeCfg<N_TILE, I8>;
    constexpr int STAGES = C_::STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C_::BAR_OFFSET);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;  // [2]
    uint64_t* acc_empty = acc_full + 2;   // [2]
    MoeShared& sh = *reinterpret_cast<MoeShared*>(smem + C_::AUX_OFFSET);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = (int)blockIdx.x, grid = (int)gridDim.x;

    // The barrier's count before this CTA's first arrival, and the epoch: under
    // way while the router runs.
    uint32_t count0 = 0u, epoch0 = 0u;
    if (threadIdx.x == 0) {
        count0 = ptx::ld_relaxed_gpu(p.bar);
        epoch0 = ptx::ld_relaxed_gpu(p.epoch);
        SPMM24_STAMP(0);
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        for (int b = 0; b < 2; ++b) {
            ptx::mbar_init(&acc_full[b], 1);
            ptx::mbar_init(&acc_empty[b], kEpiThreads / 32);
        }
        ptx::fence_mbarrier_init();
        sh.dead = 0u;
        ptx::prefetch_tmap(&p.tmGU);
        ptx::prefetch_tmap(&p.tmGUE);
        ptx::prefetch_tmap(&p.tmX);
        ptx::prefetch_tmap(&p.tmD);
        ptx::prefetch_tmap(&p.tmDE);
        ptx::prefetch_tmap(&p.tmH);
    }
    if (warp == 1) {
        ptx::tmem_alloc(&sh.tmem, C_::TMEM_COLS);
        ptx::tmem_relinquish();
    }
    for (int e = threadIdx.x; e < kMoeMaxExperts; e += kThreads) sh.mask[e] = 0u;
    ptx::tc_fence_before();

    // ------------------------------------------- router, rounding of x
    int quant_ctas = 0;
    if constexpr (I8) {
        const int parts = min(8, max(1, grid / 2 / p.strips));
        quant_ctas = p.strips * parts;
        for (int u = cta; u < quant_ctas; u += grid) {
            if (p.bf16) moe_quantize_x<true>(p, sh, u, parts);
            else moe_quantize_x<false>(p, sh, u, parts);
        }
        if (cta == grid - 1)  // the largest |h| of this launch starts from zero
            for (int i = threadIdx.x; i < p.max_slots * kMoeMaxTokens; i += kThreads) p.amax[i] = 0u;
    }
    if (p.router) {
        // the CTAs that do not round x come first
        const int unit0 = (cta + grid - quant_ctas % grid) % grid;
        if (p.bf16) moe_router<true>(p, sh, unit0, grid);
        else moe_router<false>(p, sh, unit0, grid);
    }
    if (threadIdx.x == 0) {
        sh.base = count0 - count0 % (uint32_t)grid;
        sh.epoch = epoch0;
    }
    if constexpr (I8) ptx::fence_proxy_async_global();  // xq is read by TMA
    __syncthreads();
    ptx::tc_fence_after();
    const uint32_t tmem_base = sh.tmem;
    const uint32_t base = sh.base, tag = 4u * sh.epoch + 1u;  // zeroed memory holds no tag
    uint32_t barriers = 0;  // of this launch, so far
    if (I8 || p.router) {
        ++barriers;
        if (threadIdx.x == 0) {
            moe_arrive(p.bar, (uint32_t)grid);
            if (!moe_wait(p.bar, base, barriers, (uint32_t)grid)) sh.dead = 1u;
            __threadfence();
        }
        __syncthreads();
    }

    // --------------------------------------------------------- routing
    // The weights are not needed before the down products: where the logits are
    // kept, the epilogue warps compute them behind the first weight stages.
    const int pitch = (p.E + 3) / 4 * 4;
    const bool kept = p.router && p.T * pitch <= kMoeKeptLogits;
    if (p.router) {
        // T x E logits and keys in the ring, which is still idle
        const int n = p.T * pitch, logits = p.T * p.E;
        uint32_t* key = reinterpret_cast<uint32_t*>(smem);
        float* l = kept ? sh.logits : reinterpret_cast<float*>(key + n);
#pragma unroll 2
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const int t = i / pitch, e = i - t * pitch;
            const float* at = p.logits + t * p.E + e;
            float v[kMoeMaxShares];
#pragma unroll
            for (int s = 0; s < kMoeMaxShares; ++s)
                v[s] = e < p.E && s < p.logit_shares ? __ldcg(at + (size_t)s * logits) : 0.f;
            float sum = v[0];
#pragma unroll
            for (int s = 1; s < kMoeMaxShares; ++s)
                if (s < p.logit_shares) sum += v[s];
            key[i] = e < p.E ? moe_key(sum) : 0u;
            l[i] = e < p.E ? sum : -INFINITY;
        }
        __syncthreads();
        moe_top_k(p, sh, l, key, pitch);
        if (!kept) {
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += kThreads) l[i] = expf(l[i] - __uint_as_float(sh.top[i / pitch]));
            __syncthreads();
            moe_weights<true>(p, sh, l, pitch, threadIdx.x, kThreads, cta == 0);
        }
        ptx::fence_proxy_async_smem();  // before TMA writes the ring
    } else {
        for (int i = threadIdx.x; i < p.T * p.k; i += kThreads) {
            const int e = p.ids[i];
            const bool some = e >= 0 && e < p.E;
            sh.ids[i] = some ? e : -1;
            sh.weights[i] = p.weights[i];
            if (some) atomicOr(&sh.mask[e], 1u << (i / p.k));
        }
    }
    __syncthreads();
    if (warp == 0) {
        int n = 0;
        for (int e0 = 0; e0 < p.E; e0 += 32) {
            const bool used = e0 + lane < p.E && sh.mask[e0 + lane] != 0u;
            const uint32_t b = __ballot_sync(0xffffffffu, used);
            if (used) {
                const int place = n + __popc(b & ((1u << lane) - 1u));
                sh.list[place] = (uint16_t)(e0 + lane);
                sh.slot[e0 + lane] = (uint8_t)place;
            }
            n += __popc(b);
        }
        if (lane == 0) sh.n_active = (uint32_t)n;
    }
    __syncthreads();

    if (threadIdx.x == 0) SPMM24_STAMP(3);
    const int n_active = sh.dead ? 0 : (int)sh.n_active;
    const int stage_k = I8 ? 256 : 128;
    const int gu_groups = p.H * 2 / stage_k, d_groups = p.I * 2 / stage_k;  // metadata groups along K
    const int S1 = (gu_groups + 1) / 2, Se = (d_groups + 1) / 2;            // stages of one gate / up, one down product
    const int i_tiles = (p.I + kTileM - 1) / kTileM, h_tiles = (p.H + kTileM - 1) / kTileM;
    // Two groups of experts (the first nA in use, the others), unless there is
    // little work: gate / up of A, of B, down of A, of B.
    const bool split = n_active > 1 && h_tiles <= grid &&
                       (long long)n_active * i_tiles * S1 >= (long long)kMoeSplitUnits * grid;
    // A is the larger: behind B's gate / up (two thirds of an expert's weights)
    // A's barriers pass, behind A's down products B's
    const int nA = split ? (2 * n_active + 1) / 3 : n_active, n_groups = split ? 2 : 1;
    // gate / up units (slot, 128 rows of I, stage), down units (128 rows of H, slot, stage) of one group
    auto first_of = [&](int g) { return g ? nA : 0; };
    auto count_of = [&](int g) { return g ? n_active - nA : nA; };
    auto runs1_of = [&](int g) { return MoeRuns(count_of(g) * i_tiles * S1, grid); };
    auto runs2_of = [&](int g) { return MoeRuns(h_tiles * count_of(g) * Se, grid); };
    auto h_done = [&](int g) { return barriers + (I8 ? 2u * g + 2u : g + 1u); };  // barrier after a group's h is in place

    if (warp == 0) {
        // ------------------------------------------------ TMA producer
        if (lane == 0 && n_active > 0) {
            const uint64_t pol_stream = ptx::policy_evict_first(), pol_keep = ptx::policy_evict_last();
            const uint32_t acts_bytes = I8 ? C_::B_BYTES : (uint32_t)p.strips * 2048u;
            const uint32_t w_bytes = C_::A_BYTES + C_::E_BYTES;
            int it = 0, issued = 0;  // ring slots so far; armed in all
            bool ok = true;
            auto slot_of = [&](int i) { return i % STAGES; };
            auto acquire = [&](int i, uint32_t bytes) {
                const int s = slot_of(i);
                if (i >= STAGES && !ptx::mbar_wait_bounded(&empty[s], (uint32_t)(i / STAGES - 1) & 1u, kWaitLimitNs)) {
                    atomicOr(&g_spmm24_status, kStatusProducerTimeout);
                    return false;
                }
                ptx::mbar_arrive_expect_tx(&full[s], bytes);
                issued = i + 1;
                return true;
            };
            // The walks over units keep their place without divisions: one thread
            // issues every load, and has 0.4 us a stage to keep up with HBM.
#pragma unroll 1
            for (int g = 0; g < n_groups && ok; ++g) {
                const MoeRuns runs = runs1_of(g);
                const int b = runs.begin(cta), e = runs.begin(cta + 1);
                int s = b % S1, i_tile = b / S1 % i_tiles, slot = first_of(g) + b / S1 / i_tiles;
                for (int u = b; u < e && ok; ++u) {
                    const int row0 = sh.list[slot] * 2 * p.I + i_tile * kTileM;
                    for (int half = 0; half < 2; ++half, ++it) {
                        ok = acquire(it, half ? w_bytes : w_bytes + acts_bytes);
                        if (!ok) break;
                        uint8_t* st = smem + slot_of(it) * C_::STAGE_BYTES;
                        load_stage_weights<C_>(st, &full[slot_of(it)], &p.tmGU, &p.tmGUE, (row0 + half * p.I) / 16, 2 * s,
                                               pol_stream);
                        if (!half) moe_load_acts<C_>(st, &full[slot_of(it)], &p.tmX, 0, p.strips, s, pol_keep);
                    }
                    if (++s == S1) {
                        s = 0;
                        if (++i_tile == i_tiles) {
                            i_tile = 0;
                            ++slot;
                        }
                    }
                }
            }
#pragma unroll 1
            for (int g = 0; g < n_groups && ok; ++g) {
                const MoeRuns runs = runs2_of(g);
                const int b = runs.begin(cta), n = runs.begin(cta + 1) - b;
                if (n <= 0) continue;
                const int first = first_of(g), count = count_of(g);
                struct Walk {
                    int tile, slot, s;
                };
                auto step = [&](Walk& w) {
                    if (++w.s < Se) return;
                    w.s = 0;
                    if (++w.slot < first + count) return;
                    w.slot = first;
                    ++w.tile;
                };
                const int in_tile = b % (count * Se);
                Walk ww{b / (count * Se), first + in_tile / Se, in_tile % Se}, wa = ww;  // weights, activations
                auto weights = [&](int i) {
                    load_stage_weights<C_>(smem + slot_of(i) * C_::STAGE_BYTES, &full[slot_of(i)], &p.tmD, &p.tmDE,
                                           (sh.list[ww.slot] * p.H + ww.tile * kTileM) / 16, 2 * ww.s, pol_stream);
                    step(ww);
                };
                auto acts = [&](int i) {
                    moe_load_acts<C_>(smem + slot_of(i) * C_::STAGE_BYTES, &full[slot_of(i)], &p.tmH, wa.slot, p.strips,
                                      wa.s, pol_keep);
                    step(wa);
                };
                // the first stages' weights before the wait for h
                int ahead = 0;
                while (ok && ahead < min(STAGES, n)) {
                    ok = acquire(it + ahead, w_bytes + acts_bytes);
                    if (ok) weights(it + ahead++);
                }
                if (ok) ok = moe_wait(p.bar, base, h_done(g), (uint32_t)grid);
                if (g == 0) SPMM24_STAMP(5);
                for (int i = 0; i < ahead && ok; ++i) acts(it + i);
                for (int i = ahead; i < n && ok; ++i) {
                    if (!(ok = acquire(it + i, w_bytes + acts_bytes))) break;
                    weights(it + i);
                    acts(it + i);
                }
                it += n;
            }
            if (!ok)  // gave up: let the copies in flight land before the block ends
                for (int i = max(0, issued - STAGES); i < issued; ++i)
                    ptx::mbar_wait_bounded(&full[slot_of(i)], (uint32_t)(i / STAGES) & 1u, 10000000ull);
        }
        __syncwarp();
    } else if (warp == 1) {
        // -------------------------------------------------- MMA issuer
        const uint32_t smem_base = ptx::smem_u32(smem), fmt = p.bf16 ? kIdescBf16 : 0u;
        int it = 0, j = 0;
        bool ok = n_active > 0;
        // waits until accumulator pair j & 1 has been read; false: give up
        auto begin_acc = [&]() {
            if (j >= 2) {
                if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&acc_empty[j & 1], (uint32_t)((j >> 1) - 1) & 1u,
                                                                    kWaitLimitNs))) {
                    if (lane == 0) atomicOr(&g_spmm24_status, kStatusMmaTimeout);
                    return false;
                }
                ptx::tc_fence_after();
            }
            return true;
        };
        auto wait_full = [&](int i) {
            if (!__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&full[i % STAGES], (uint32_t)(i / STAGES) & 1u,
                                                                kWaitLimitNs))) {
                if (lane == 0) atomicOr(&g_spmm24_status, kStatusMmaTimeout);
                return false;
            }
            ptx::tc_fence_after();
            return true;
        };
        auto stage = [&](int i, int acts, uint32_t d, uint32_t accumulate) {
            moe_mma_stage<C_, N_TILE, I8>(smem_base + i % STAGES * C_::STAGE_BYTES,
                                          smem_base + acts % STAGES * C_::STAGE_BYTES,
                                          tmem_base + C_::META_COL + C_::META_STRIDE * (i % STAGES), d, accumulate, fmt);
        };
        auto end_acc = [&]() {
            if (lane == 0) ptx::tc_commit(&acc_full[j & 1]);
            __syncwarp();
            ++j;
        };
#pragma unroll 1
        for (int g = 0; g < n_groups && ok; ++g) {
            const MoeRuns runs = runs1_of(g);
            const int e = runs.begin(cta + 1);
            for (int u = runs.begin(cta); u < e && ok;) {
                const int s0 = u % S1, s1 = min(S1, s0 + e - u);
                if (!(ok = begin_acc())) break;
                const uint32_t d = tmem_base + (uint32_t)((j & 1) * 2 * N_TILE);
                for (int s = s0; s < s1 && ok; ++s, it += 2) {
                    for (int half = 0; half < 2; ++half) {
                        if (!(ok = wait_full(it + half))) break;
                        if (lane == 0 && it + half == 0) SPMM24_STAMP(1);
                        if (2 * s + 1 >= gu_groups)
                            patch_tail_metadata<C_>(smem + (it + half) % STAGES * C_::STAGE_BYTES, lane);
                        if (lane == 0) {
                            stage(it + half, it, d + (uint32_t)(half * N_TILE), s > s0);
                            if (half) {  // the up product was the last to read the gate slot's activations
                                ptx::tc_commit(&empty[it % STAGES]);
                                ptx::tc_commit(&empty[(it + 1) % STAGES]);
                            }
                        }
                        __syncwarp();
                    }
                }
                if (!ok) break;
                end_acc();
                u += s1 - s0;
            }
        }
        if (lane == 0) SPMM24_STAMP(2);
#pragma unroll 1
        for (int g = 0; g < n_groups && ok; ++g) {
            const MoeRuns runs = runs2_of(g);
            const int e = runs.begin(cta + 1);
            for (int u = runs.begin(cta); u < e && ok;) {  // a segment ends with its expert: the epilogue weighs each
                const int s0 = u % Se, s1 = min(Se, s0 + e - u);
                if (!(ok = begin_acc())) break;
                const uint32_t d = tmem_base + (uint32_t)((j & 1) * 2 * N_TILE);
                for (int s = s0; s < s1; ++s, ++it) {
                    if (!(ok = wait_full(it))) break;
                    if (2 * s + 1 >= d_groups) patch_tail_metadata<C_>(smem + it % STAGES * C_::STAGE_BYTES, lane);
                    if (lane == 0) {
                        stage(it, it, d, s > s0);
                        ptx::tc_commit(&empty[it % STAGES]);
                    }
                    __syncwarp();
                }
                if (!ok) break;
                end_acc();
                u += s1 - s0;
            }
        }
        if (lane == 0) SPMM24_STAMP(7);
    } else {
        // ---------------------------------------------------- epilogue
        const int quad = warp & 3, row = quad * 32 + lane;  // thread = output row (TMEM lane)
        const uint32_t tmem_row = tmem_base + ((uint32_t)(quad * 32) << 16);
        int j = 0;
        bool ok = true;
        // A warp whose wait gave up goes on without waiting, so that the warps
        // still meet at their barriers (the launch's outputs are then void).
        auto wait_acc = [&]() {
            if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(&acc_full[j & 1], (uint32_t)(j >> 1) & 1u,
                                                                      kWaitLimitNs))) {
                atomicOr(&g_spmm24_status, kStatusEpilogueTimeout);
                ok = false;
            }
            ptx::tc_fence_after();
        };
        auto release_acc = [&]() {
            ptx::tc_fence_before();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive(&acc_empty[j & 1]);
            ++j;
        };
        // all epilogue threads: wait for the launch's n-th grid barrier
        auto wait_grid = [&](uint32_t n) {
            if (threadIdx.x == 64) sh.last = ok && moe_wait(p.bar, base, n, (uint32_t)grid) ? 1u : 0u;
            ptx::named_barrier(kBarEpi, kEpiThreads);
            ok = ok && sh.last != 0u;
            ptx::named_barrier(kBarEpi, kEpiThreads);
            __threadfence();
        };
        // The tiles of a run: finished by the CTAs that share them, an equal
        // part of the rows each.  A warp takes 32 rows and PAIRS pairs of tokens
        // at a time (of many partials 8 rows), the loads of BATCH partials in
        // flight.
        if (I8 && threadIdx.x - 64 < p.T) sh.xscale[threadIdx.x - 64] = __ldcg(p.xscale + threadIdx.x - 64);
        if (kept) moe_weights<false>(p, sh, sh.logits, pitch, threadIdx.x - 64, kEpiThreads, cta == 0);
        ptx::named_barrier(kBarEpi, kEpiThreads);
        constexpr int PAIRS = N_TILE == 16 ? 1 : 4, BATCH1 = N_TILE == 16 ? 8 : 2, BATCH2 = N_TILE == 16 ? 8 : 4;
#pragma unroll 1
        for (int g = 0; g < n_groups && n_active > 0; ++g) {
            const MoeRuns runs = runs1_of(g);
            const int b = runs.begin(cta), end = runs.begin(cta + 1), first = first_of(g);
            const int slot0 = first + b / S1 / i_tiles;  // the run's first expert
            if constexpr (I8) {
                sh.hmax[warp - 2][lane] = 0u;
                ptx::named_barrier(kBarEpi, kEpiThreads);
                // the run's channel scales into L2, ahead of their use under a full stream
                for (int t = b / S1; b < end && t * S1 < end; ++t) {
                    const int r = t % i_tiles * kTileM + (int)(threadIdx.x & 3u) * 32;
                    const float* at = p.gu_scale + (size_t)sh.list[first + t / i_tiles] * 2 * p.I + r;
                    if (threadIdx.x < 64 + 8 && r < p.I) ptx::prefetch_l2(threadIdx.x & 4u ? at + p.I : at);
                }
            }
            for (int u = b; u < end;) {
                const int tile = u / S1, s0 = u % S1, s1 = min(S1, s0 + end - u);
                u += s1 - s0;
                const int slot = first + tile / i_tiles, e = sh.list[slot], r = tile % i_tiles * kTileM + row;
                const bool live = r < p.I;
                float gs = 0.f, us = 0.f;
                if constexpr (I8) {
                    if (live) {
                        gs = p.gu_scale[(size_t)e * 2 * p.I + r];
                        us = p.gu_scale[(size_t)e * 2 * p.I + p.I + r];
                    }
                }
                const uint32_t mask = sh.mask[e];
                uint32_t v[2 * N_TILE];  // gate, up
                wait_acc();
                moe_read_acc<2 * N_TILE>(tmem_row + (uint32_t)((j & 1) * 2 * N_TILE), v);
                ptx::tmem_wait_ld();
                release_acc();
                if (s1 - s0 < S1) {
                    moe_put_partial<N_TILE>(p.part + (size_t)(2 * cta + (b < tile * S1 ? 1 : 0)) * kMoeSlotWords, v, row,
                                            moe_pairs(mask), tag + (uint32_t)g);
                    continue;
                }
                if constexpr (I8) {
#pragma unroll
                    for (int t = 0; t < N_TILE; ++t) {
                        if (!(mask >> t & 1u)) continue;
                        const float xs = sh.xscale[t];
                        const float h = live ? moe_activate(int8_value((int)v[t], gs, xs), p.act) *
                                                   int8_value((int)v[N_TILE + t], us, xs)
                                             : 0.f;
                        if (live) __stcg(p.h32 + ((size_t)slot * p.T + t) * p.I + r, h);
                        moe_note_max(sh, slot - slot0, t, h);
                    }
                } else if (live) {
#pragma unroll
                    for (int s = 0; s < N_TILE / 8; ++s) {
                        if (s >= p.strips) break;
                        uint32_t w[4];
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const int t = 8 * s + 2 * q;
                            w[q] = 0u;  // a pair of tokens that have other experts
                            if (mask >> t & 3u)
                                w[q] = pack2(
                                    moe_activate(__uint_as_float(v[t]), p.act) * __uint_as_float(v[N_TILE + t]),
                                    moe_activate(__uint_as_float(v[t + 1]), p.act) * __uint_as_float(v[N_TILE + t + 1]),
                                    p.bf16);
                        }
                        *reinterpret_cast<uint4*>(p.h16 + (((size_t)slot * p.strips + s) * p.I + r) * 8) =
                            make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
            // shared tiles: the first and the last of the run, their units dealt to the warps in turn
            int dealt = 0;
            for (int t = b / S1; b < end && t * S1 < end; t += max(1, (end - 1) / S1 - t)) {
                if (b <= t * S1 && end >= (t + 1) * S1) continue;
                const MoeTile tile(runs, t, S1);
                const int shares = tile.c1 - tile.c0 + 1, mine = cta - tile.c0;
                const int r0 = kTileM * mine / shares, r1 = kTileM * (mine + 1) / shares;
                const bool fold = shares > 4 && r1 - r0 <= 32 && __popc(moe_pairs(sh.mask[sh.list[first + t / i_tiles]])) < 4 * PAIRS;
                const int rows = fold ? 8 : 32, blocks = (r1 - r0 + rows - 1) / rows;
                const int slot = first + t / i_tiles, e = sh.list[slot];
                const uint32_t mask = sh.mask[e], pairs = moe_pairs(mask);
                const int units = blocks * ((__popc(pairs) + PAIRS - 1) / PAIRS), mine0 = (warp - 2 - dealt) & 3;
                dealt += units;
                for (int w = mine0; w < units; w += kEpiThreads / 32) {
                    const int rt = r0 + w % blocks * rows + lane % rows, r = t % i_tiles * kTileM + rt;  // row of the tile, of I
                    const bool live = lane < rows && rt < r1 && r < p.I;
                    float gs = 0.f, us = 0.f;
                    if constexpr (I8) {
                        if (live) {
                            gs = p.gu_scale[(size_t)e * 2 * p.I + r];
                            us = p.gu_scale[(size_t)e * 2 * p.I + p.I + r];
                        }
                    }
                    uint32_t m = pairs;
                    for (int n = w / blocks * PAIRS; n > 0; --n) m &= m - 1u;
                    int col[2 * PAIRS], tok0[PAIRS];
#pragma unroll
                    for (int n = 0; n < PAIRS; ++n) {
                        tok0[n] = m ? 2 * (__ffs((int)m) - 1) : -1;  // the pair's first token
                        col[n] = m ? tok0[n] : col[0];               // none left: the first one's columns again
                        col[PAIRS + n] = N_TILE + col[n];
                        m &= m - 1u;
                    }
                    uint32_t v[4 * PAIRS];  // gate values, up values
                    moe_sum_partials<2 * PAIRS, BATCH1, I8>(
                        shares, [&](int i) { return p.part + (size_t)tile.slot(runs, tile.c0 + i) * kMoeSlotWords; }, col,
                        min(rt, kTileM - 1), tag + (uint32_t)g, fold, v, ok);
#pragma unroll
                    for (int n = 0; n < PAIRS; ++n) {
                        if (tok0[n] < 0) break;
                        float h[2];
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            const int tok = tok0[n] + i;
                            const uint32_t gv = v[2 * n + i], uv = v[2 * PAIRS + 2 * n + i];
                            if constexpr (I8) {
                                h[i] = 0.f;
                                if (!(mask >> tok & 1u)) continue;
                                const float xs = sh.xscale[tok];
                                if (live) {
                                    h[i] = moe_activate(int8_value((int)gv, gs, xs), p.act) * int8_value((int)uv, us, xs);
                                    __stcg(p.h32 + ((size_t)slot * p.T + tok) * p.I + r, h[i]);
                                }
                                moe_note_max(sh, slot - slot0, tok, h[i]);
                            } else {
                                h[i] = moe_activate(__uint_as_float(gv), p.act) * __uint_as_float(uv);
                            }
                        }
                        if constexpr (!I8) {
                            if (live)
                                *reinterpret_cast<uint32_t*>(
                                    p.h16 + (((size_t)slot * p.strips + tok0[n] / 8) * p.I + r) * 8 + tok0[n] % 8) =
                                    pack2(h[0], h[1], p.bf16);
                        }
                    }
                }
            }
            if (threadIdx.x == 64) SPMM24_STAMP(4);
            // the group's h is in place, this CTA's share of it
            if constexpr (I8) {
                ptx::named_barrier(kBarEpi, kEpiThreads);
                const int slot = slot0 + warp - 2;
                if (slot < first + count_of(g) && sh.hmax[warp - 2][lane])
                    atomicMax(p.amax + slot * kMoeMaxTokens + lane, sh.hmax[warp - 2][lane]);
            } else {
                ptx::fence_proxy_async_global();  // h is read by TMA
            }
            ptx::named_barrier(kBarEpi, kEpiThreads);
            if (threadIdx.x == 64 && ok) moe_arrive(p.bar, (uint32_t)grid);
            if constexpr (I8) {
                // round h, once every row's largest value is known: (token,
                // choice) rows in pieces of 512 values, four pieces in flight
                wait_grid(barriers + 2u * (uint32_t)g + 1u);
                constexpr int AHEAD = 4;
                const int pieces = (p.I + 511) / 512, units = ok ? p.T * p.k * pieces : 0;
                for (int w0 = cta; w0 < units; w0 += AHEAD * grid) {
                    float4 h[AHEAD];
                    float a[AHEAD];
                    size_t at[AHEAD];
#pragma unroll
                    for (int n = 0; n < AHEAD; ++n) {
                        const int w = w0 + n * grid, i = w / pieces, c = w % pieces * 512 + (threadIdx.x - 64) * 4;
                        const int e = w < units ? sh.ids[i] : -1, slot = e < 0 ? 0 : sh.slot[e], t = i / p.k;
                        a[n] = -1.f;
                        if (e < 0 || (slot >= nA) != (g == 1) || c >= p.I) continue;
                        at[n] = ((size_t)slot * p.T + t) * p.I + c;
                        a[n] = __uint_as_float(__ldcg(p.amax + slot * kMoeMaxTokens + t));
                        h[n] = __ldcg(reinterpret_cast<const float4*>(p.h32 + at[n]));
                    }
#pragma unroll
                    for (int n = 0; n < AHEAD; ++n) {
                        if (a[n] == -1.f) continue;
                        // a row of zeros, or one with an infinity or NaN: zeros, times its scale
                        const bool live = a[n] > 0.f && a[n] <= 3.402823466e38f;
                        // far below 1, 127 / a would overflow: both times 2^64, which changes no quotient
                        const float pre = a[n] < 0x1p-60f ? 0x1p64f : 1.f, top = a[n] * pre, inv = 127.f / top;
                        const float hv[4] = {h[n].x, h[n].y, h[n].z, h[n].w};
                        uint32_t q[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) q[i] = live ? moe_round_h(hv[i] * pre, top, inv) : 0u;
                        *reinterpret_cast<uint32_t*>(p.hq + at[n]) = pack4(q[0], q[1], q[2], q[3]);
                    }
                }
                ptx::fence_proxy_async_global();  // hq is read by TMA
                ptx::named_barrier(kBarEpi, kEpiThreads);
                if (threadIdx.x == 64 && ok) moe_arrive(p.bar, (uint32_t)grid);
            } else if (g + 1 < n_groups) {
                wait_grid(h_done(g));  // the next group's partials take the same slots
            }
        }
        const bool vec = (p.T % 8 == 0) && ((reinterpret_cast<uintptr_t>(p.y) & 15u) == 0) &&
                         ((reinterpret_cast<uintptr_t>(p.epi.residual) & 15u) == 0);
        const bool plain = epilogue_is_plain(p.epi);
        auto finish = [&](uint32_t (&y)[N_TILE], int tile) {
            const int gm = tile * kTileM + row;
            if (gm >= p.H) return;
#pragma unroll
            for (int c = 0; c < N_TILE; c += 8) {
                if (c >= p.T) break;
                float f[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(y[c + i]);
                epilogue_store8<true>(p.y, f, p.epi, gm, c, p.H, p.T, vec, plain);
            }
        };
        uint64_t* const part2 = p.part + (size_t)kMoeMaxCtas * 2 * kMoeSlotWords;  // the first group's down partials
#pragma unroll 1
        for (int g = 0; g < n_groups && n_active > 0; ++g) {
            const MoeRuns runs = runs2_of(g);
            const int b = runs.begin(cta), end = runs.begin(cta + 1), first = first_of(g), S2 = count_of(g) * Se;
            for (int u = b; u < end;) {
                const int tile = u / S2, s0 = u % S2, s1 = min(S2, s0 + end - u);
                uint32_t y[N_TILE];
#pragma unroll
                for (int t = 0; t < N_TILE; ++t) y[t] = 0u;
                for (int s = s0; s < s1;) {
                    const int slot = first + s / Se, e = sh.list[slot];
                    // this expert's weight of token `lane` (the same expert twice: the sum)
                    float w = 0.f, scale = 1.f;
                    const uint32_t mask = sh.mask[e];
                    if (lane < p.T)
                        for (int i = 0; i < p.k; ++i)
                            if (sh.ids[lane * p.k + i] == e) w += sh.weights[lane * p.k + i];
                    if constexpr (I8) {
                        if (mask >> lane & 1u) w *= __uint_as_float(__ldcg(p.amax + slot * kMoeMaxTokens + lane)) / 127.f;
                        const int gm = tile * kTileM + row;
                        scale = gm < p.H ? p.d_scale[(size_t)e * p.H + gm] : 0.f;
                    }
                    uint32_t v[N_TILE];
                    wait_acc();
                    moe_read_acc<N_TILE>(tmem_row + (uint32_t)((j & 1) * 2 * N_TILE), v);
                    ptx::tmem_wait_ld();
                    release_acc();
#pragma unroll
                    for (int t = 0; t < N_TILE; ++t) {
                        const float wt = __shfl_sync(0xffffffffu, w, t);
                        const float d = I8 ? (float)(int)v[t] * scale : __uint_as_float(v[t]);
                        if (mask >> t & 1u) y[t] = __float_as_uint(fmaf(wt, d, __uint_as_float(y[t])));
                    }
                    s = min(s1, (s / Se + 1) * Se);
                }
                u += s1 - s0;
                if (n_groups == 1 && s1 - s0 == S2) {
                    finish(y, tile);
                    continue;
                }
                // h_tiles <= grid where there are two groups: a run meets two tiles at most
                const size_t slot = 2 * cta + (b < tile * S2 ? 1 : 0);
                moe_put_partial<N_TILE>(g == 0 ? part2 + slot * (kMoeSlotWords / 2) : p.part + slot * kMoeSlotWords, y, row,
                                        (1u << (p.T + 1) / 2) - 1u, tag + 2u);
            }
        }
        if (n_active > 0) {
            // the last group's run says whose tiles are whose; the first group's
            // partials come first in the sum
            const MoeRuns runs = runs2_of(n_groups - 1), runs_a = runs2_of(0);
            const int b = runs.begin(cta), end = runs.begin(cta + 1), S2 = count_of(n_groups - 1) * Se;
            int dealt = 0;
            for (int t = b / S2; b < end && t * S2 < end; ++t) {
                if (n_groups == 1 && b <= t * S2 && end >= (t + 1) * S2) continue;
                const MoeTile tile(runs, t, S2), tile_a(runs_a, t, nA * Se);
                const int shares = tile.c1 - tile.c0 + 1, mine = cta - tile.c0;
                const int before = n_groups == 2 ? tile_a.c1 - tile_a.c0 + 1 : 0;
                const int r0 = kTileM * mine / shares, r1 = kTileM * (mine + 1) / shares;
                const bool fold = before + shares > 4 && r1 - r0 <= 32 && p.T <= 6 * PAIRS;
                const int rows = fold ? 8 : 32, blocks = (r1 - r0 + rows - 1) / rows;
                const int cols = p.epi.packed ? 8 * p.strips : p.T;
                const int units = blocks * ((cols + 2 * PAIRS - 1) / (2 * PAIRS)), mine0 = (warp - 2 - dealt) & 3;
                dealt += units;
                auto slot = [&](int i) -> const uint64_t* {
                    if (i < before) return part2 + (size_t)tile_a.slot(runs_a, tile_a.c0 + i) * (kMoeSlotWords / 2);
                    const size_t at = tile.slot(runs, tile.c0 + i - before);
                    return n_groups == 1 ? part2 + at * (kMoeSlotWords / 2) : p.part + at * kMoeSlotWords;
                };
                for (int w = mine0; w < units; w += kEpiThreads / 32) {
                    const int rt = r0 + w % blocks * rows + lane % rows, t0 = w / blocks * 2 * PAIRS;
                    const int gm = t * kTileM + rt;
                    int col[PAIRS];
#pragma unroll
                    for (int n = 0; n < PAIRS; ++n) col[n] = t0 + 2 * n < p.T ? t0 + 2 * n : 0;
                    uint32_t v[2 * PAIRS];
                    moe_sum_partials<PAIRS, BATCH2, false>(before + shares, slot, col, min(rt, kTileM - 1), tag + 2u, fold,
                                                           v, ok);
                    if (lane >= rows || rt >= r1 || gm >= p.H) continue;
                    if constexpr (PAIRS == 4) {
                        float y[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) y[i] = __uint_as_float(v[i]);
                        epilogue_store8<true>(p.y, y, p.epi, gm, t0, p.H, p.T, vec, plain);
                    } else {
#pragma unroll
                        for (int i = 0; i < 2 * PAIRS; ++i) {
                            const int tok = t0 + i;
                            if (tok >= cols) break;
                            const size_t at = c_offset(p.epi, gm, tok, p.H, p.T);
                            float y[1] = {__uint_as_float(v[i])};
                            if (!plain) {
                                epilogue_pre<1, true>(y, p.epi, gm);
                                if (p.epi.residual && tok < p.T) y[0] += elem_to_f32(p.epi.residual[at], p.epi.bf16);
                            }
                            p.y[at] = tok < p.T ? f32_to_elem(y[0], p.epi.bf16) : (uint16_t)0;
                        }
                    }
                }
            }
        } else if (!sh.dead) {  // no token has an expert
            uint32_t y[N_TILE];
#pragma unroll
            for (int t = 0; t < N_TILE; ++t) y[t] = 0u;
            for (int tile = cta; tile < h_tiles; tile += grid) finish(y, tile);
        }
        if (threadIdx.x == 64) SPMM24_STAMP(6);
    }

    ptx::tc_fence_before();
    __syncthreads();
    // every CTA that shares a tile has read the epoch before the grid barrier
    if (cta == 0 && threadIdx.x == 0) *p.epoch = sh.epoch + 1u;
    if (warp == 1) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc(tmem_base, C_::TMEM_COLS);
    }
}

}  // namespace spmm24
