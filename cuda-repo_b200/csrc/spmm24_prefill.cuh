// spmm24_prefill.cuh -- the int8 prefill kernel: persistent CTA pairs on
// 512 x 224 tiles, each tile's epilogue behind the next one's main loop.
//
// Tiles, operands and MMAs are those of the two-M-half pair kernel
// (spmm24_pair2_kernel): per stage of 256 K a CTA moves 68 KB for two M = 256
// MMAs sets that share B, and the main loop runs at 0.69 us a stage, 6.3 PFLOP/s
// dense-equivalent over the GPU.  One tile per CTA spends another 8.8 us on
// start, pipeline fill, two accumulators' epilogue and exit: 44 % of a tile of
// 4096 K.  Here a pair walks tiles, the ring of loads runs on across them, and
// eight warps of each CTA do nothing but epilogues.  TMEM is full (two
// accumulators of 224 columns and the metadata), so the next tile's MMAs wait
// until an accumulator has been read: eight epilogue warps take one to registers
// at once, 112 columns of a row for each thread, release it, and only then scale,
// activate, round and store.  The two follow one another: the next tile's first half
// starts on the stages at hand while the first accumulator's values are stored, its
// second half waits until they are and the second accumulator has been read.
//
// Measured: 11008 x 4096 x 4096 (418 tiles, 6 rounds of 74 pairs) 119.5 -> 99 us,
// 8192^3 248 -> 230.  A stage takes 1160 cycles, what the tensor cores' operand
// reads take at 128 bytes a cycle (A 4 KB, B 14 KB a step, eight steps); a tile
// of 16 stages takes 27.7 thousand: 5.2 of them wait for the accumulators (the store
// of the first that the head start does not cover) and 3.6 for loads (60 bytes a cycle
// and SM out of L2).
//
// Row-major C needs N % 8 == 0 and 16-byte alignment, a packed C nothing.  No
// residual.
//
// Roles (384 threads): warps 0-2 TMA producers (A and metadata of each M half,
// B), warp 3 of the leader MMA issuer, warps 4-11 epilogue.  Every wait is
// bounded; an epilogue warp whose wait gave up goes on without waiting, so that
// the warps still meet at their barriers.
#pragma once
#include "spmm24_kernel.cuh"

namespace spmm24 {

constexpr int kPrefillThreads = 384;
constexpr int kPrefillEpiThreads = 256;  // 8 warps: two share a row's columns

template <int STAGES>
struct PrefillCfg : Pair2Cfg<STAGES, true, true> {
    using P_ = Pair2Cfg<STAGES, true, true>;
    static constexpr int COLS = P_::TILE_N / 2;          // columns of an epilogue warp
    static constexpr int BUF_PITCH = 80;                 // bytes: 32 columns and 16 against bank conflicts
    static constexpr int STORE_OFFSET = P_::RING_BYTES;  // [8 warps][32 rows]
    static constexpr int XS_OFFSET = STORE_OFFSET + 8 * 32 * BUF_PITCH;  // [2][TILE_N] column scales
    static constexpr int BAR_OFFSET = XS_OFFSET + 2 * P_::TILE_N * 4;
    static constexpr int NUM_BARS = 2 * STAGES + 3;         // full, empty, acc_full, acc_empty[2]
    static constexpr int HOLDER_OFFSET = BAR_OFFSET + NUM_BARS * 8;
    static constexpr int SMEM_BYTES = HOLDER_OFFSET + 16;
    static constexpr int SMEM_ALLOC = SMEM_BYTES + 1024;
    static_assert(SMEM_ALLOC <= 232448, "shared memory overflow");
    static_assert(COLS % 16 == 0, "whole chunks of 16 columns");
};

template <int STAGES>
__global__ void __launch_bounds__(kPrefillThreads, 1)
spmm24_prefill_int8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                           const __grid_constant__ CUtensorMap tmE,
                           const PairParams p, int m_tiles, int n_tiles) {
    using C_ = PrefillCfg<STAGES>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* full = reinterpret_cast<uint64_t*>(smem + C_::BAR_OFFSET);  // used in the leader only
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + 1;  // [2], used in the leader only
    uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C_::HOLDER_OFFSET);

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const uint32_t rank = ptx::cluster_ctarank();  // 0 = leader (issues the MMAs), 1 = peer
    const bool leader = rank == 0;
    const int pair = (int)blockIdx.x >> 1, pairs = (int)gridDim.x >> 1, tiles = m_tiles * n_tiles;
    const int st_count = p.stages_total;
    // Tile t in rasterisation order, as the other pair kernels': consecutive
    // tiles walk down kPairGroupM tile rows before the next column.
    auto tile_at = [&](int t, int& m_tile, int& n_tile) {
        const int per_group = kPairGroupM * n_tiles;
        const int first_m = t / per_group * kPairGroupM, group_m = min(m_tiles - first_m, kPairGroupM);
        m_tile = first_m + t % per_group % group_m;
        n_tile = t % per_group / group_m;
    };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(&full[s], 1);
            ptx::mbar_init(&empty[s], 1);
        }
        ptx::mbar_init(acc_full, 1);
        for (int h = 0; h < 2; ++h) ptx::mbar_init(&acc_empty[h], 2 * kPrefillEpiThreads / 32);  // both CTAs' warps
        ptx::fence_mbarrier_init();
        ptx::prefetch_tmap(&tmA);
        ptx::prefetch_tmap(&tmB);
        ptx::prefetch_tmap(&tmE);
    }
    if (warp == 3) {
        ptx::tmem_alloc_pair(tmem_holder, C_::TMEM_COLS);
        ptx::tmem_relinquish_pair();
    }
    ptx::tc_fence_before();
    ptx::cluster_sync();  // both CTAs: barriers initialised, TMEM allocated
    ptx::tc_fence_after();
    const uint32_t tmem_base = *tmem_holder;
    if (threadIdx.x == 0) ptx::grid_dep_launch();

    if (warp < 3) {
        // ------------------------------------------------- TMA producers
        // Both CTAs' loads complete on the leader's full barrier, which its
        // warp 0 arms.
        if (lane == 0) {
            const uint64_t pol = ptx::policy_evict_last();
            const uint32_t full0 = ptx::mapa_shared(ptx::smem_u32(&full[0]), 0u);
            const int n = pair < tiles ? ((tiles - 1 - pair) / pairs + 1) * st_count : 0;
            const int pre = p.weights_static && warp < 2 ? min(STAGES, n) : 0;  // weights before the previous grid ends
            int t = pair, s_in = 0, band = 0, row = 0;
            auto place = [&]() {
                int m_tile, n_tile;
                tile_at(t, m_tile, n_tile);
                band = (m_tile * C_::TILE_M + warp * 2 * kTileM + (int)rank * kTileM) / 16;
                row = n_tile * C_::TILE_N + (int)rank * C_::HALF_N;
            };
            if (n > 0) place();
            bool waited = false;
            for (int it = 0; it < n; ++it) {
                if (it >= pre && !waited) {
                    ptx::grid_dep_wait();
                    waited = true;
                }
                const int s = it % STAGES;
                if (it >= STAGES &&
                    !ptx::mbar_wait_bounded(&empty[s], (uint32_t)(it / STAGES - 1) & 1u, kWaitLimitNs)) {
                    atomicOr(&g_spmm24_status, kStatusProducerTimeout);
                    break;
                }
                uint8_t* st = smem + s * C_::STAGE_BYTES;
                const uint32_t bar = full0 + 8u * s;
                if (warp == 2) {
                    ptx::tma_load_2d_pair(st + C_::A_BYTES, &tmB, bar, 256 * s_in, row, pol);
                    ptx::tma_load_2d_pair(st + C_::A_BYTES + C_::B_BYTES / 2, &tmB, bar, 256 * s_in + 128, row, pol);
                } else {
                    if (warp == 0 && leader) ptx::mbar_arrive_expect_tx(&full[s], 2 * C_::STAGE_BYTES);
                    ptx::tma_load_3d_pair(st + warp * C_::A_HALF, &tmA, bar, 0, band, 8 * s_in, pol);
                    ptx::tma_load_3d_pair(st + C_::A_BYTES + C_::B_BYTES + warp * C_::E_HALF, &tmE, bar, 0, band, 2 * s_in,
                                          pol);
                }
                if (++s_in == st_count) {
                    s_in = 0;
                    t += pairs;
                    if (t < tiles) place();
                }
            }
        }
        __syncwarp();
    } else if (warp == 3 && leader) {
        // ---------------------------------- MMA issuer (leader CTA only)
        constexpr uint32_t idesc = (pair_idesc_fp8<C_::TILE_N>() & ~kIdescF32) | kIdescInt8;
        const uint32_t smem_base = ptx::smem_u32(smem);
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t parity) {
            if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(bar, parity & 1u, kWaitLimitNs))) {
                if (lane == 0) atomicOr(&g_spmm24_status, kStatusMmaTimeout);
                ok = false;
            }
            ptx::tc_fence_after();
            return ok;
        };
        // one M half's four MMAs of ring stage `it`
        auto half = [&](int it, int h, bool accumulate) {
            const uint32_t st = smem_base + it % STAGES * C_::STAGE_BYTES, stB = st + C_::A_BYTES;
            const uint32_t stE = stB + C_::B_BYTES + (uint32_t)h * C_::E_HALF;
            const uint32_t meta = tmem_base + (h ? C_::META1_COL : C_::META0_COL) + C_::META_STRIDE * (it % C_::META_SLOTS);
            ptx::tmem_cp_128x128b_pair(meta, smem_desc(stE, 0, 128));
            ptx::tmem_cp_128x128b_pair(meta + 4, smem_desc(stE + 2048, 0, 128));
#pragma unroll
            for (int j = 0; j < 4; ++j)
                ptx::mma_sp_i8_pair(tmem_base + (uint32_t)h * C_::ACC1_COL,
                                    smem_desc(st + (uint32_t)h * C_::A_HALF + j * 4096, 2048, 128),
                                    smem_desc_sw128(stB + (j >> 1) * (C_::B_BYTES / 2) + (j & 1) * 64), meta + 2 * j,
                                    idesc, accumulate || j ? 1u : 0u);
        };
        int it = 0, i = 0;
        for (int t = pair; t < tiles && ok; t += pairs, ++i) {
            const int head = min(STAGES, st_count);
            if (i > 0 && !wait(&acc_empty[0], (uint32_t)(i - 1))) break;
            for (int s = 0; s < head && ok; ++s) {
                if (!wait(&full[(it + s) % STAGES], (uint32_t)((it + s) / STAGES))) break;
                if (lane == 0) half(it + s, 0, s > 0);
                __syncwarp();
            }
            if (!ok || (i > 0 && !wait(&acc_empty[1], (uint32_t)(i - 1)))) break;
            for (int s = 0; s < head; ++s) {
                if (lane == 0) {
                    half(it + s, 1, s > 0);
                    ptx::tc_commit_pair_mc(&empty[(it + s) % STAGES], (uint16_t)0x3);  // frees the slot in both CTAs
                }
                __syncwarp();
            }
            for (int s = head; s < st_count; ++s) {
                if (!wait(&full[(it + s) % STAGES], (uint32_t)((it + s) / STAGES))) break;
                if (lane == 0) {
                    half(it + s, 0, true);
                    half(it + s, 1, true);
                    ptx::tc_commit_pair_mc(&empty[(it + s) % STAGES], (uint16_t)0x3);
                }
                __syncwarp();
            }
            if (!ok) break;
            if (lane == 0) ptx::tc_commit_pair_mc(acc_full, (uint16_t)0x3);
            __syncwarp();
            it += st_count;
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------ epilogue
        const int quad = warp & 3, side = (warp - 4) >> 2;  // TMEM lanes, half of the columns
        const int row = quad * 32 + lane;
        constexpr int PIECES = C_::COLS / 8;  // of eight columns: 16 bytes of output
        uint8_t* buf = smem + C_::STORE_OFFSET + (warp - 4) * 32 * C_::BUF_PITCH;
        float* xs = reinterpret_cast<float*>(smem + C_::XS_OFFSET);
        const uint32_t empty0 = ptx::mapa_shared(ptx::smem_u32(&acc_empty[0]), 0u);
        bool ok = true;
        ptx::grid_dep_wait();  // scales and bias may be written, C read or written by the previous grid
        int i = 0;
        for (int t = pair; t < tiles; t += pairs, ++i) {
            int m_tile, n_tile;
            tile_at(t, m_tile, n_tile);
            const int gn0 = n_tile * C_::TILE_N, gm0 = m_tile * C_::TILE_M + (int)rank * kTileM;
            float* x = xs + (i & 1) * C_::TILE_N;  // the other buffer may still be read for the tile before
            for (int c = (int)threadIdx.x - 128; c < C_::TILE_N; c += kPrefillEpiThreads)
                x[c] = !p.x_scale ? 1.f : gn0 + c < p.N ? p.x_scale[gn0 + c] : 0.f;
            float w[2], bias[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int gm = gm0 + h * 2 * kTileM + row;
                w[h] = p.w_scale && gm < p.M ? p.w_scale[gm] : 1.f;
                bias[h] = p.epi.bias && gm < p.M ? elem_to_f32(p.epi.bias[gm], p.epi.bf16) : 0.f;
            }
            ptx::named_barrier(kBarEpi, kPrefillEpiThreads);
            if (ok && !__all_sync(0xffffffffu, ptx::mbar_wait_bounded(acc_full, (uint32_t)i & 1u, kWaitLimitNs))) {
                atomicOr(&g_spmm24_status, kStatusEpilogueTimeout);
                ok = false;
            }
            ptx::tc_fence_after();
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
                const uint32_t taddr = tmem_base + (uint32_t)(h * C_::ACC1_COL) + ((uint32_t)(quad * 32) << 16) +
                                       (uint32_t)(side * C_::COLS);
                const float wsc = h ? w[1] : w[0], b = h ? bias[1] : bias[0];
                const int gm = gm0 + h * 2 * kTileM + row;
                uint32_t v[C_::COLS];
#pragma unroll
                for (int c = 0; c + 16 <= C_::COLS; c += 16)
                    ptx::tmem_ld_32x32b_x16(taddr + c, *reinterpret_cast<uint32_t(*)[16]>(v + c));
                ptx::tmem_wait_ld();
                ptx::tc_fence_before();  // the half is in registers: the next tile may have it
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive_cluster(empty0 + 8u * h);
                const int gn = gn0 + side * C_::COLS;
                const float* xc = x + side * C_::COLS;
                auto piece = [&](int q, uint32_t (&o)[4]) {  // eight columns, scaled, activated, rounded
                    const float4 s0 = *reinterpret_cast<const float4*>(xc + 8 * q);
                    const float4 s1 = *reinterpret_cast<const float4*>(xc + 8 * q + 4);
                    const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
                    float y[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[e] = int8_value((int)v[8 * q + e], wsc, s[e]);
                    epilogue_pre<8, true>(y, p.epi, gm, &b);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] = pack2(y[2 * e], y[2 * e + 1], p.epi.bf16);
                };
                if (p.epi.packed) {  // consecutive lanes take consecutive rows of a strip
#pragma unroll
                    for (int q = 0; q < PIECES; ++q) {
                        uint32_t o[4];
                        piece(q, o);
                        const int lim = p.N - gn - 8 * q;
                        if (gm >= p.M || lim <= 0) continue;
                        if (lim < 8) {  // pad columns are zero
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[e] = 2 * e >= lim ? 0u : 2 * e + 1 >= lim ? o[e] & 0xffffu : o[e];
                        }
                        *reinterpret_cast<uint4*>(p.C + (((size_t)((gn >> 3) + q) * p.M + gm) << 3)) =
                            make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    continue;
                }
                // Row-major: 32 rows x 32 columns at a time through the warp's
                // buffer, so that four lanes store 64 contiguous bytes of a row.
#pragma unroll
                for (int q0 = 0; q0 < PIECES; q0 += 4) {
                    const int per_row = q0 + 4 <= PIECES ? 4 : PIECES % 4;
#pragma unroll
                    for (int q = 0; q < per_row; ++q) {
                        uint32_t o[4];
                        piece(q0 + q, o);
                        *reinterpret_cast<uint4*>(buf + lane * C_::BUF_PITCH + 16 * q) = make_uint4(o[0], o[1], o[2], o[3]);
                    }
                    __syncwarp();
                    const int rows = 32 / per_row, at = lane % per_row, r0 = lane / per_row, cn = gn + 8 * (q0 + at);
#pragma unroll
                    for (int r = 0; r < 32; r += rows) {
                        const int rm = gm - lane + r + r0;
                        const uint4 o = *reinterpret_cast<const uint4*>(buf + (r + r0) * C_::BUF_PITCH + at * 16);
                        if (rm < p.M && cn < p.N) *reinterpret_cast<uint4*>(p.C + (size_t)rm * p.N + cn) = o;
                    }
                    __syncwarp();
                }
            }
        }
    }

    ptx::tc_fence_before();
    __syncthreads();
    ptx::cluster_sync();  // neither CTA may leave while the pair still shares shared memory / TMEM
    if (warp == 3) {
        ptx::tc_fence_after();
        ptx::tmem_dealloc_pair(tmem_base, C_::TMEM_COLS);
    }
}

}  // namespace spmm24
