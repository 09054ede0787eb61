// CTA-pair variant of the 4-bit GEMM: a cluster of two CTAs on neighbouring SMs owns a 256 x 256 output tile and runs one tcgen05.mma
// (cta_group::2, M = 256, N = 256, K = 64) per K step, persistent over tiles.  Operands, scales and epilogue are those of gemm_fp4.cu.
//
// Roles per CTA (10 warps) as in the 8-bit kernel (gemm_pair.cu):
//   warp 0     TMA producer: its 128 rows of A and of B, its rows' block scales, and the block scales of all 256 columns
//   warp 1     TMEM allocation; in the leader one thread copies a slab's scales to both CTAs' TMEM and issues its four MMAs
//   warps 2-9  epilogue of the CTA's own 128 rows x 256 columns, through shared memory and TMA stores
//
// TMEM has 512 columns, two accumulators and the scales of a slab need 512 + 48.  So the accumulators overlap by 64 columns:
// [0, 256) and [192, 448), scales from 448 on.  The epilogue takes the 64 shared columns of a tile first and gives them back at once; all
// that the next tile's MMAs wait for is those, because the rest of their accumulator was read before the epilogue came to this tile.
//
// What bounds it (clocks of one SM, 6144 x 2048 x 8192 nvfp4): the MMAs of a tile take 4130, 516 a slab of 256, the tile 5600.  Five stages of
// 38 KB just cover the 2000 clocks from a freed stage to its next operands, at 54 bytes a clock and SM, of 64 that the SM can take from L2
// and 74 that the MMAs alone would take; and from a tile's last MMA to the next one's first 700 to 900 pass.  With GELU the epilogue takes
// 6600 of a tile's 7000.  Tried: 16 epilogue warps (a tile's epilogue 4000 and 5600, but it comes in one burst, and the loads suffer: 81.0 ->
// 89.1 thousand clocks in all, with GELU 97.3 -> 96.7); fragments of 16 x 64 through stmatrix and plain stores (88.3, 95.3); A's rows kept in
// shared memory for all tiles of a row block, which halves the loads and leaves three stages for B (95.0, 97.7); scales copied to TMEM one
// K step ahead or to alternate columns (no change).
// 6144 x 8192 x 2048 mxfp4 37.5 us, 5.5 PFLOP/s, 0.84 of four times the measured bf16 rate; 24576 x 2048 x 8192 157 us, nvfp4 171, with GELU
// 205 under the power cap.

#include "gemm_fp4.cuh"

namespace q8k {

constexpr int kFp4PairStages = 5;
constexpr int kFp4PairOverlap = 64;          // columns that both accumulators have
constexpr int kFp4PairScaleCols = 448;       // where the scales begin

template <bool NV>
struct Fp4PairSmem {
    static constexpr int kABytes = kGemmBM * 128, kBBytes = kGemmBM * 128;     // this CTA's rows of A and of B
    static constexpr int kScales = fp4_slab_scales(NV);                        // of 128 rows
    static constexpr int kStageBytes = kABytes + kBBytes + 3 * kScales;        // its rows of A, both row tiles of B
    static constexpr int kStoreBoxBytes = 32 * 64;                             // output staging: per epilogue warp two boxes of 32 rows x 32 columns
    static constexpr int kStoreOffset = kFp4PairStages * kStageBytes;
    static constexpr int kBarOffset = kStoreOffset + (kGemmEpilogueThreads / 32) * 2 * kStoreBoxBytes;
    static constexpr int kNumBars = 2 * kFp4PairStages + 4;
    static constexpr int kTmemPtrOffset = kBarOffset + kNumBars * 8;
    static constexpr int kAbortOffset = kTmemPtrOffset + 4;
    static constexpr int kColumnOffset = (kAbortOffset + 4 + 15) & ~15;        // two tiles' column scales and biases, {s, s, b, b} of a pair
    static constexpr int kTotal = kColumnOffset + 2 * 256 * 8;
    static_assert(kStageBytes % 1024 == 0 && kTotal <= 227 * 1024, "pair GEMM shared memory");
};

struct Fp4PairParams {
    Fp4GemmParams g;
    int n_tiles, total_tiles;                // tiles of 256 x 256
};

template <bool NV, bool GELU, bool F16>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
gemm_fp4_pair_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b,
                     const __grid_constant__ CUtensorMap tmap_as, const __grid_constant__ CUtensorMap tmap_bs,
                     const __grid_constant__ CUtensorMap tmap_c, const Fp4PairParams pp) {
    using L = Fp4PairSmem<NV>;
    constexpr int STAGES = kFp4PairStages, TILES = fp4_slab_tiles(NV);
    const Fp4GemmParams& p = pp.g;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t smem_base = ptx::smem_u32(smem);
    if (smem_base & 1023u) {                                   // same offset in both CTAs: both leave
        pdl_wait();
        if (threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (37 << 8));
        return;
    }
    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto tmem_full_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    auto tmem_free_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };      // the shared columns of accumulator a have been read
    volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(smem + L::kTmemPtrOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOffset);
    float4* columns = reinterpret_cast<float4*>(smem + L::kColumnOffset);      // [2][128]

    const uint32_t rank = ptx::cluster_ctarank();              // 0 = leader, 1 = peer
    const bool leader = rank == 0;
    const int cluster_id = blockIdx.x >> 1;
    const int num_clusters = gridDim.x >> 1;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int slabs = (p.K + kFp4Slab - 1) / kFp4Slab;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 2);                    // one arrive.expect_tx from each CTA's producer
            ptx::mbar_init(empty_bar(s), 1);                   // one commit from the leader's MMA thread
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(tmem_full_bar(a), 1);
            ptx::mbar_init(tmem_free_bar(a), 2 * (kGemmEpilogueThreads / 32));    // every epilogue warp of both CTAs
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
        ptx::prefetch_tensormap(&tmap_as);
        ptx::prefetch_tensormap(&tmap_bs);
        ptx::prefetch_tensormap(&tmap_c);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair<512>(ptx::smem_u32(const_cast<uint32_t*>(tmem_ptr_smem)));
        ptx::tmem_relinquish_alloc_permit_pair();
    }
    pdl_wait();                                                // everything above overlaps the kernel before
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();                                   // both CTAs' barriers exist before anyone signals across
    ptx::tcgen05_fence_after_sync();
    pdl_release();                                             // this CTA holds its TMEM: the next kernel may move in behind it
    const uint32_t tmem_base = *tmem_ptr_smem;
    const uint32_t leader_full0 = ptx::mapa_shared(full_bar(0), 0);

    if (warp == 0) {
        // ------------------------------------------------ TMA producer (both CTAs)
        if (ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 1;                                   // empty_bar phase to wait for: the first round passes
            bool ok = true;
            constexpr int SLAB_ROWS = L::kScales / 256;
            for (int tile = cluster_id; ok && tile < pp.total_tiles; tile += num_clusters) {
                const int m0 = tile / pp.n_tiles * 256, n0 = tile % pp.n_tiles * 256;
                const int a_row = m0 + (int)rank * kGemmBM, b_row = n0 + (int)rank * kGemmBM;
                for (int i = 0; i < slabs; ++i) {
                    if (!ptx::mbar_wait(empty_bar(s), ph, abort_flag)) { ok = false; break; }
                    const uint32_t fb = leader_full0 + 8u * s;
                    ptx::mbar_arrive_expect_tx_cluster(fb, L::kStageBytes);
                    const uint32_t dst = smem_base + s * L::kStageBytes;
                    ptx::tma_load_2d_pair(dst, &tmap_a, fb, i * 128, a_row);
                    ptx::tma_load_2d_pair(dst + L::kABytes, &tmap_b, fb, i * 128, b_row);
                    ptx::tma_load_3d_pair(dst + L::kABytes + L::kBBytes, &tmap_as, fb, 0, i * SLAB_ROWS, a_row / 128);
                    ptx::tma_load_3d_pair(dst + L::kABytes + L::kBBytes + L::kScales, &tmap_bs, fb, 0, i * SLAB_ROWS, n0 / 128);
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (34 << 8));
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer (leader CTA only)
        if (leader && ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            uint32_t tile_i = 0;
            bool ok = true;
            const uint32_t idesc[2] = {ptx::make_idesc_fp4(256, 256, !NV, 0), ptx::make_idesc_fp4(256, 256, !NV, 2)};
            const uint32_t ta = tmem_base + kFp4PairScaleCols, tb = ta + 4 * TILES;
            for (int tile = cluster_id; ok && tile < pp.total_tiles; tile += num_clusters, ++tile_i) {
                const uint32_t acc = tile_i & 1u;
                if (tile_i > 0) {                              // the tile before has given the shared columns back
                    if (!ptx::mbar_wait(tmem_free_bar(acc ^ 1u), ((tile_i - 1) >> 1) & 1u, abort_flag)) { ok = false; break; }
                    ptx::tcgen05_fence_after_sync();
                }
                const uint32_t d_tmem = tmem_base + acc * (256 - kFp4PairOverlap);
                for (int i = 0; i < slabs; ++i) {
                    if (!ptx::mbar_wait(full_bar(s), ph, abort_flag)) { ok = false; break; }
                    ptx::tcgen05_fence_after_sync();
                    const uint32_t src = smem_base + s * L::kStageBytes;
                    const uint64_t as_desc = ptx::make_scales_desc(src + L::kABytes + L::kBBytes);
                    const uint64_t bs_desc = ptx::make_scales_desc(src + L::kABytes + L::kBBytes + L::kScales);
                    const uint64_t a_desc = ptx::make_kmajor_desc(src, 128);
                    const uint64_t b_desc = ptx::make_kmajor_desc(src + L::kABytes, 128);
#pragma unroll
                    for (int t = 0; t < TILES; ++t) {
                        ptx::tmem_copy_scales_pair(ta + 4 * t, as_desc + 32 * t);
                        ptx::tmem_copy_scales_pair(tb + 8 * t, bs_desc + 32 * t);
                        ptx::tmem_copy_scales_pair(tb + 8 * t + 4, bs_desc + L::kScales / 16 + 32 * t);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int t = NV ? k : k / 2;
                        ptx::mma_fp4<NV ? 4 : 2, true>(d_tmem, a_desc + 2 * k, b_desc + 2 * k, idesc[NV ? 0 : k & 1], ta + 4 * t, tb + 8 * t,
                                                       (i > 0 || k > 0) ? 1u : 0u);
                    }
                    // the stage is reusable in BOTH CTAs once these have retired
                    ptx::tcgen05_commit_both(empty_bar(s));
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
                if (ok) ptx::tcgen05_commit_both(tmem_full_bar(acc));
            }
            if (!ok && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (35 << 8));
        }
    } else {
        // ------------------------------------------------ epilogue (warps 2..9) of this CTA's 128 rows
        const int quarter = warp & 3;
        const int half = (warp - 2) >> 2;
        const int epi_tid = threadIdx.x - 64;
        const uint32_t store_base = smem_base + L::kStoreOffset + (uint32_t)(warp - 2) * 2u * L::kStoreBoxBytes;
        uint32_t tile_i = 0;
        uint32_t store_i = 0;                                  // stores issued by this warp: picks the staging box
        // A launch that follows a failed one on the same status word stores nothing.  (Read here and not ahead of everything: 0.4 us of every call.)
        const int prior_failure = p.status != nullptr ? *reinterpret_cast<volatile int*>(p.status) : 0;
        // what the next tile needs from global memory is on its way while this one is worked on
        float next_scale = 0.f, next_bias = 0.f, next_sa = 0.f;
        auto prefetch = [&](int tile) {
            if (tile >= pp.total_tiles) return;
            const int row = tile / pp.n_tiles * 256 + (int)rank * kGemmBM + quarter * 32 + lane, n = tile % pp.n_tiles * 256 + epi_tid;
            next_sa = row >= p.M ? 0.f : p.a_scales != nullptr ? p.a_scales[row] : 1.f;
            next_scale = n >= p.N ? 0.f : p.b_scales != nullptr ? p.b_scales[n] : 1.f;
            next_bias = n < p.N && p.bias != nullptr ? p.bias[n] : 0.f;
        };
        prefetch(cluster_id);
        bool ok = true;
        for (int tile = cluster_id; tile < pp.total_tiles; tile += num_clusters, ++tile_i) {
            const int m0 = tile / pp.n_tiles * 256 + (int)rank * kGemmBM, n0 = tile % pp.n_tiles * 256;
            const uint32_t acc = tile_i & 1u;
            const float4* column = columns + acc * 128;
            {
                float* c = reinterpret_cast<float*>(columns + acc * 128 + epi_tid / 2) + (epi_tid & 1);
                c[0] = next_scale;
                c[2] = next_bias;
            }
            const float2 sa2 = make_float2(next_sa, next_sa);
            // One barrier a tile: who has passed it knows that all have read the columns of two tiles ago.
            asm volatile("bar.sync 1, 256;" ::: "memory");
            prefetch(tile + num_clusters);
            const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * (256 - kFp4PairOverlap);
            // 32-column chunks of this warp: one of the two shared ones first, then three of the six others
            auto chunk = [&](int c) {
                return acc == 0 ? (c == 0 ? 6 + half : 3 * half + c - 1) : (c == 0 ? half : 2 + 3 * half + c - 1);
            };
            if (ok) ok = ptx::mbar_wait(tmem_full_bar(acc), (tile_i >> 1) & 1u, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            ptx::tcgen05_fence_after_sync();

            uint32_t r[2][32];
            __syncwarp();
            ptx::tmem_ld_32x32b_x32(t_row + chunk(0) * 32, r[0]);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                ptx::tmem_wait_ld();
                if (c == 0) {                                  // the leader's MMA thread waits for both CTAs
                    ptx::tcgen05_fence_before_sync();
                    __syncwarp();
                    if (lane == 0) ptx::mbar_arrive_cluster(ptx::mapa_shared(tmem_free_bar(acc), 0));
                }
                if (c + 1 < 4) ptx::tmem_ld_32x32b_x32(t_row + chunk(c + 1) * 32, r[(c + 1) & 1]);
                const int cl = chunk(c) * 32, nc = n0 + cl;
                const uint32_t(&rc)[32] = r[c & 1];
                if (nc < p.N && prior_failure == 0) {          // warp-uniform
                    const uint32_t box = store_base + (store_i & 1u) * L::kStoreBoxBytes;
                    ++store_i;
                    // the store that last used this box (two stores ago) must have read it out
                    if (lane == 0) ptx::bulk_wait_group_read<1>();
                    __syncwarp();
                    // row `lane` of the box, 16-byte pieces XOR-swizzled as the tensor map expects (SWIZZLE_64B: piece ^= (row >> 1) & 3)
                    const uint32_t row_addr = box + (uint32_t)lane * 64u, sw = ((uint32_t)lane >> 1) & 3u;
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = q * 8 + e * 2;
                            const float4 sb = column[(cl + j) / 2];
                            float2 y = ffma2(make_float2(__uint_as_float(rc[j]), __uint_as_float(rc[j + 1])), fmul2(sa2, make_float2(sb.x, sb.y)),
                                             make_float2(sb.z, sb.w));
                            if constexpr (GELU) y = gelu_tanh_fast2(y);
                            w[e] = pack16<F16>(y);
                        }
                        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + (((uint32_t)q ^ sw) << 4)),
                                     "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                                     : "memory");
                    }
                    ptx::fence_proxy_async_smem();
                    __syncwarp();
                    if (lane == 0) {
                        ptx::tma_store_3d(&tmap_c, box, nc * 2, m0 + quarter * 32, 0);
                        ptx::bulk_commit_group();
                    }
                }
                __syncwarp();
            }
        }
        if (lane == 0) ptx::bulk_wait_group<0>();    // this warp's stores are performed before the CTA may exit
        if (!ok && p.status != nullptr && epi_tid == 0) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (36 << 8));
    }

    // ---------------------------------------------------- teardown: neither CTA may leave while the other can still read its shared memory,
    // signal its barriers or write its TMEM
    if (threadIdx.x == 0 && *abort_flag != 0) {
        // a wait was abandoned: give copies still in flight time to land before the CTA gives up its shared memory
        const unsigned long long t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 50000ull) {}
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();
    if (warp == 1) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc_pair<512>(tmem_base);
    }
}

template <bool NV, bool GELU, bool F16>
static int launch_fp4_pair_as(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tas, const CUtensorMap& tbs, const CUtensorMap& tc,
                              const Fp4PairParams& pp, cudaStream_t st) {
    auto kern = gemm_fp4_pair_kernel<NV, GELU, F16>;
    constexpr int SMEM = Fp4PairSmem<NV>::kTotal;
    static std::atomic<uint64_t> smem_done{0};
    if (int rc = allow_dynamic_smem((const void*)kern, SMEM, smem_done)) return rc;
    // how many 2-CTA clusters can be resident at once (cached per kernel variant)
    static int max_clusters = -1;
    if (max_clusters < 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * gemm_num_sms());
        cfg.blockDim = dim3(kGemmThreads);
        cfg.dynamicSmemBytes = SMEM;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
        max_clusters = n;
    }
    if (max_clusters < 8) return Q8K_ERR_UNSUPPORTED;
    const int clusters = pp.total_tiles < max_clusters ? pp.total_tiles : max_clusters;
    Q8K_CUDA_OK(launch_dependent(kern, 2 * clusters, kGemmThreads, SMEM, st, 1, ta, tb, tas, tbs, tc, pp));
    return Q8K_OK;
}

int launch_fp4_pair(bool nv, bool gelu, bool f16, const Fp4Operand& a, const Fp4Operand& b, const Fp4GemmParams& p, cudaStream_t st) {
    const char* op = "fp4_mm";
    Fp4PairParams pp;
    pp.g = p;
    const int64_t m_tiles = ((int64_t)p.M + 255) / 256;
    pp.n_tiles = (p.N + 255) / 256;
    if (m_tiles * pp.n_tiles > 0x7fffffffLL) return Q8K_ERR_UNSUPPORTED;
    pp.total_tiles = (int)(m_tiles * pp.n_tiles);
    CUtensorMap ta, tb, tas, tbs, tc;
    if (int rc = make_values_map(&ta, a.values, p.M, p.K, kGemmBM, op)) return rc;
    if (int rc = make_values_map(&tb, b.values, p.N, p.K, kGemmBM, op)) return rc;
    if (int rc = make_scales_map(&tas, a.block_scales, nv, p.M, p.K, 1, op)) return rc;
    if (int rc = make_scales_map(&tbs, b.block_scales, nv, p.N, p.K, 2, op)) return rc;
    // output rows as bytes, boxes of 32 columns and 32 rows (N % 16 == 0: the pitch is a multiple of 16 bytes)
    {
        const uint64_t dims[3] = {(uint64_t)p.N * 2, (uint64_t)p.M, 1};
        const uint64_t strides[2] = {(uint64_t)p.N * 2, (uint64_t)p.M * (uint64_t)p.N * 2};
        const uint32_t box[3] = {64, 32, 1};
        if (int rc = make_byte_tensor_map(&tc, p.out, 3, dims, strides, box, 64, op)) return rc;
    }
#define Q8K_FP4(NV)                                                                                          \
    do {                                                                                                     \
        if (gelu) return f16 ? launch_fp4_pair_as<NV, true, true>(ta, tb, tas, tbs, tc, pp, st)              \
                             : launch_fp4_pair_as<NV, true, false>(ta, tb, tas, tbs, tc, pp, st);            \
        return f16 ? launch_fp4_pair_as<NV, false, true>(ta, tb, tas, tbs, tc, pp, st)                       \
                   : launch_fp4_pair_as<NV, false, false>(ta, tb, tas, tbs, tc, pp, st);                     \
    } while (0)
    if (nv) Q8K_FP4(true);
    Q8K_FP4(false);
#undef Q8K_FP4
}

}  // namespace q8k
