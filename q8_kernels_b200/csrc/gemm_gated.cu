// Gated 8-bit projection: gate and up projection, activation and product in one kernel,
//   gate = (A . Wg^T) * (sa[m] * sg[n]) + bg[n],  up = (A . Wu^T) * (sa[m] * su[n]) + bu[n],  out = act(gate) * up   (bf16)
// with Wg and Wu the first and the last F rows of one weight W [2F, K].  The backward pass needs gate and up: with SAVE they are stored
// as well, rounded to bf16 as a projection's output would be; `out` is computed from the unrounded values.
//
// A pair of CTAs (cta_group::2) owns 256 rows and `bn` output columns, i.e. 2 bn columns of the product.  The MMA takes the first
// half of its B rows from the even CTA and the second from the odd one: the even CTA loads rows of Wg, the odd one the same rows of
// Wu, so columns [0, bn) of the accumulator are the gate and [bn, 2 bn) the up projection of the same output columns, in the TMEM
// lanes of the same thread.  No weight has to be laid out anew, and neither projection's result leaves the SM.
//
// Roles, barriers and the bounded waits are those of the pair kernel (gemm_pair.cu): warp 0 TMA producer, warp 1 MMA issuer (even CTA)
// and TMEM allocation, warps 2-9 epilogue; two accumulators, so that the epilogue of a tile runs under the products of
// the next.
//
// Bound by the tensor pipe: 6144 x 2048 x 8192 int8 134 us, 3.1 POP/s, pipe 91.3 % busy.  With SAVE 165 us (79.2 %): the 201 MB of gate and
// up cross L2 beside the operands (2.2 GB instead of 1.6); without their stores alone it runs at 135 again.  Tried there: six stages with two
// boxes (no change), boxes of 128 bytes a row (170), stores marked evict-first (164 to 167: DRAM reads 115 -> 90 MB, time within
// the noise).

#include <math.h>

#include "gemm_common.cuh"

namespace q8k {

constexpr int kGatedBN = 128;                // output columns of the widest tile: 256 columns of the product
constexpr int kGatedTmemCols = 512;          // two accumulators of 256 columns

template <bool SAVE>
struct GatedSmemT {
    static constexpr int kStages = SAVE ? 5 : 6;
    static constexpr int kABytes = kGemmBM * kGemmBK;
    static constexpr int kBBytes = kGatedBN * kGemmBK;
    static constexpr int kStageBytes = kABytes + kBBytes;
    // output staging: per epilogue warp a ring of boxes of 32 rows x 64 bytes, one store each
    static constexpr int kRing = SAVE ? 3 : 2;
    static constexpr int kBoxBytes = 32 * 64;
    static constexpr int kStoreOffset = kStages * kStageBytes;
    static constexpr int kStoreBytes = (kGemmEpilogueThreads / 32) * kRing * kBoxBytes;
    static constexpr int kBarOffset = kStoreOffset + kStoreBytes;
    static constexpr int kNumBars = 2 * kStages + 4;
    static constexpr int kTmemPtrOffset = kBarOffset + kNumBars * 8;
    static constexpr int kAbortOffset = kTmemPtrOffset + 4;
    static constexpr int kPriorOffset = kAbortOffset + 4;
    static constexpr int kScaleOffset = (kPriorOffset + 4 + 15) & ~15;         // gate columns, then up columns
    static constexpr int kBiasOffset = kScaleOffset + 2 * kGatedBN * 4;
    static constexpr int kTotal = kBiasOffset + 2 * kGatedBN * 4;
    static_assert(kTotal <= 227 * 1024, "gated GEMM shared memory");
};

struct GatedParams {
    const float* a_scales;
    const float* b_scales;                   // [2F]
    const float* bias;                       // [2F] or null
    int* status;
    int M, F, K;
    int bn;                                  // output columns of a tile: 32, 64, 96 or 128
    int n_tiles, total_tiles;
};

// silu(g) = g / (1 + e^-g); tanh-GELU = g / (1 + e^(-2u)) with u = sqrt(2/pi) (g + 0.044715 g^3): no cancellation anywhere.  The exponent
// v = g or 2u is rounded to fp32 before the exponential, so the result is off by up to (5 |v| + 12) 2^-24 of itself where v is negative (its
// constants and products; ex2 and rcp are good to 2^-22) and by some units of 2^-24 where it is positive: at v = -20 2^-17, far below half a
// step of bf16, 2^-8, which is what it is rounded to.  e^(-v) overflows to infinity for very negative v, and g / infinity is the right 0.
template <bool GELU> __device__ __forceinline__ float gated_act(float g) {
    constexpr float kLog2e = 1.4426950408889634f;
    float t;
    if constexpr (GELU) {
        constexpr float kC0 = -2.0f * 0.7978845608028654f * kLog2e, kC1 = kC0 * 0.044715f;
        t = g * fmaf(kC1, g * g, kC0);
    } else {
        t = -kLog2e * g;
    }
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(e + 1.0f));
    return g * r;
}

template <bool INT8, bool GELU, bool SAVE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kGemmThreads, 1)
gemm_8bit_gated_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                       const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ CUtensorMap tmap_pre, const GatedParams p) {
    using L = GatedSmemT<SAVE>;
    constexpr int STAGES = L::kStages;
    extern __shared__ __align__(1024) uint8_t smem[];
    const uint32_t smem_base = ptx::smem_u32(smem);
    if (smem_base & 1023u) {                                   // same offset in both CTAs: both leave
        pdl_wait();
        if (threadIdx.x == 0 && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (31 << 8));
        return;
    }
    const uint32_t bar_base = smem_base + L::kBarOffset;
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (STAGES + s); };
    auto tmem_full_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
    auto tmem_empty_bar = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
    volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(smem + L::kTmemPtrOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kAbortOffset);
    volatile int* prior_failure = reinterpret_cast<volatile int*>(smem + L::kPriorOffset);
    float* scale_smem = reinterpret_cast<float*>(smem + L::kScaleOffset);
    float* bias_smem = reinterpret_cast<float*>(smem + L::kBiasOffset);

    const uint32_t rank = ptx::cluster_ctarank();              // 0: leader, gate rows; 1: up rows
    const bool leader = rank == 0;
    const int cluster_id = blockIdx.x >> 1;
    const int num_clusters = gridDim.x >> 1;
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int k_iters = (p.K + kGemmBK - 1) / kGemmBK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) {
            ptx::mbar_init(full_bar(s), 2);                    // one arrive.expect_tx from each CTA's producer
            ptx::mbar_init(empty_bar(s), 1);                   // one commit from the leader's MMA thread
        }
        for (int a = 0; a < 2; ++a) {
            ptx::mbar_init(tmem_full_bar(a), 1);
            ptx::mbar_init(tmem_empty_bar(a), 2 * (kGemmEpilogueThreads / 32));   // every epilogue warp of both CTAs
        }
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_w);
        ptx::prefetch_tensormap(&tmap_out);
        if (SAVE) ptx::prefetch_tensormap(&tmap_pre);
    }
    if (warp == 1) {
        ptx::tmem_alloc_pair<kGatedTmemCols>(ptx::smem_u32(const_cast<uint32_t*>(tmem_ptr_smem)));
        ptx::tmem_relinquish_alloc_permit_pair();
    }
    pdl_wait();                                                // everything above overlaps the kernel before
    // A launch that follows a failed one on the same status word does nothing; the leader decides for both CTAs.
    if (threadIdx.x == 0 && leader) {
        const int v = p.status != nullptr ? *reinterpret_cast<volatile int*>(p.status) : 0;
        *prior_failure = v;
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ptx::mapa_shared(smem_base + L::kPriorOffset, 1)), "r"(v)
                     : "memory");
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();                                   // both CTAs' barriers exist before anyone signals across
    ptx::tcgen05_fence_after_sync();
    pdl_release();                                             // this CTA holds its TMEM: the next kernel may move in behind it
    const bool skip = *prior_failure != 0;
    const uint32_t tmem_base = *tmem_ptr_smem;

    const uint32_t leader_full0 = ptx::mapa_shared(full_bar(0), 0);
    auto leader_tmem_empty_bar = [&](int a) { return ptx::mapa_shared(tmem_empty_bar(a), 0); };

    if (skip) {
    } else if (warp == 0) {
        // ------------------------------------------------ TMA producer (both CTAs)
        if (ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 1;                                   // empty_bar phase to wait for: the first round passes
            bool ok = true;
            const uint32_t bytes = L::kABytes + (uint32_t)p.bn * kGemmBK;
            for (int tile = cluster_id; ok && tile < p.total_tiles; tile += num_clusters) {
                const int a_row = tile / p.n_tiles * 2 * kGemmBM + (int)rank * kGemmBM;
                // The gate's last tile may run on into the rows of the up projection, and that one's beyond the weight
                // (zeros): columns from F on, which no store takes.
                const int w_row = tile % p.n_tiles * p.bn + (int)rank * p.F;
                for (int kb = 0; kb < k_iters; ++kb) {
                    if (!ptx::mbar_wait(empty_bar(s), ph, abort_flag)) { ok = false; break; }
                    const uint32_t fb = leader_full0 + 8u * s;
                    ptx::mbar_arrive_expect_tx_cluster(fb, bytes);
                    const uint32_t a_dst = smem_base + s * L::kStageBytes;
                    ptx::tma_load_2d_pair(a_dst, &tmap_a, fb, kb * kGemmBK, a_row);
                    ptx::tma_load_2d_pair(a_dst + L::kABytes, &tmap_w, fb, kb * kGemmBK, w_row);
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (28 << 8));
        }
    } else if (warp == 1) {
        // ------------------------------------------------ MMA issuer (leader CTA only)
        if (leader && ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            uint32_t tile_i = 0;
            bool ok = true;
            const uint32_t idesc = INT8 ? ptx::make_idesc_s8(2 * kGemmBM, 2 * p.bn) : ptx::make_idesc_e4m3(2 * kGemmBM, 2 * p.bn);
            for (int tile = cluster_id; ok && tile < p.total_tiles; tile += num_clusters, ++tile_i) {
                const uint32_t acc = tile_i & 1u;
                const uint32_t acc_ph = (tile_i >> 1) & 1u;
                if (!ptx::mbar_wait(tmem_empty_bar(acc), acc_ph ^ 1u, abort_flag)) { ok = false; break; }
                ptx::tcgen05_fence_after_sync();
                const uint32_t d_tmem = tmem_base + acc * (2 * kGatedBN);
                for (int kb = 0; kb < k_iters; ++kb) {
                    if (!ptx::mbar_wait(full_bar(s), ph, abort_flag)) { ok = false; break; }
                    ptx::tcgen05_fence_after_sync();
                    const uint32_t a_addr = smem_base + s * L::kStageBytes;
                    const uint64_t a_desc = ptx::make_kmajor_desc(a_addr, 128);
                    const uint64_t b_desc = ptx::make_kmajor_desc(a_addr + L::kABytes, 128);
#pragma unroll
                    for (int k = 0; k < kGemmBK / 32; ++k) {
                        const uint32_t accumulate = (kb > 0 || k > 0) ? 1u : 0u;
                        if constexpr (INT8) ptx::mma_i8_pair(d_tmem, a_desc + 2 * k, b_desc + 2 * k, idesc, accumulate);
                        else ptx::mma_f8f6f4_pair(d_tmem, a_desc + 2 * k, b_desc + 2 * k, idesc, accumulate);
                    }
                    ptx::tcgen05_commit_both(empty_bar(s));    // the stage is reusable in both CTAs once these MMAs retire
                    if (++s == STAGES) { s = 0; ph ^= 1u; }
                }
                if (ok) ptx::tcgen05_commit_both(tmem_full_bar(acc));
            }
            if (!ok && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (29 << 8));
        }
    } else {
        // ------------------------------------------------ epilogue (warps 2..9) of this CTA's 128 rows
        const int quarter = warp & 3;
        const int half = (warp - 2) >> 2;
        const int epi_tid = threadIdx.x - 64;
        const uint32_t store_base = smem_base + L::kStoreOffset + (uint32_t)(warp - 2) * L::kRing * L::kBoxBytes;
        const int chunks = p.bn / 32;
        const int c_lo = half == 0 ? 0 : (chunks + 1) / 2;     // warps 2-5 take the first half of the chunks, 6-9 the rest
        const int c_hi = half == 0 ? (chunks + 1) / 2 : chunks;
        uint32_t tile_i = 0;
        uint32_t box_i = 0;                                    // next box of this warp's ring
        bool ok = true;
        for (int tile = cluster_id; tile < p.total_tiles; tile += num_clusters, ++tile_i) {
            const int row0 = tile / p.n_tiles * 2 * kGemmBM + (int)rank * kGemmBM + quarter * 32;
            const int n0 = tile % p.n_tiles * p.bn;
            const uint32_t acc = tile_i & 1u;
            const uint32_t acc_ph = (tile_i >> 1) & 1u;

            asm volatile("bar.sync 1, 256;" ::: "memory");     // the tile before has been read out of the arrays
            for (int c = epi_tid; c < 2 * p.bn; c += kGemmEpilogueThreads) {
                const bool up = c >= p.bn;
                const int n = n0 + (up ? c - p.bn : c);
                const bool in = n < p.F;
                const int at = up ? p.F + n : n;
                scale_smem[c] = in ? p.b_scales[at] : 0.f;
                bias_smem[c] = in && p.bias != nullptr ? p.bias[at] : 0.f;
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");

            const int row = row0 + lane;
            const float sa = row < p.M ? p.a_scales[row] : 0.f;
            const float2 sa2 = make_float2(sa, sa);
            const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16) + acc * (2 * kGatedBN);

            if (ok) ok = ptx::mbar_wait(tmem_full_bar(acc), acc_ph, abort_flag);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) continue;
            ptx::tcgen05_fence_after_sync();

            // row `lane` of the box, 16-byte pieces swizzled as the tensor maps expect (SWIZZLE_64B: piece ^= (row >> 1) & 3)
            const uint32_t sw = ((uint32_t)lane >> 1) & 3u;
            auto store_chunk = [&](const CUtensorMap* map, const uint32_t (&w)[16], int x, int which_or_row, int row_or_zero) {
                const uint32_t box = store_base + box_i * L::kBoxBytes;
                if (++box_i == (uint32_t)L::kRing) box_i = 0;
                if (lane == 0) ptx::bulk_wait_group_read<L::kRing - 1>();      // the store that last used this box has read it out
                __syncwarp();
                const uint32_t row_addr = box + (uint32_t)lane * 64u;
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(row_addr + (((uint32_t)q ^ sw) << 4)),
                                 "r"(w[4 * q]), "r"(w[4 * q + 1]), "r"(w[4 * q + 2]), "r"(w[4 * q + 3])
                                 : "memory");
                ptx::fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) {
                    ptx::tma_store_3d(map, box, x, which_or_row, row_or_zero);
                    ptx::bulk_commit_group();
                }
            };

            for (int c = c_lo; c < c_hi; ++c) {                // (warp-uniform)
                uint32_t rg[32], ru[32];
                ptx::tmem_ld_32x32b_x32(t_row + c * 32, rg);
                ptx::tmem_ld_32x32b_x32(t_row + p.bn + c * 32, ru);
                ptx::tmem_wait_ld();
                const int nc = n0 + c * 32;
                if (nc >= p.F) continue;
                uint32_t wo[16], wg[16], wu[16];
#pragma unroll
                for (int j = 0; j < 32; j += 2) {
                    const float2 g = epilogue_pair<INT8, false>(rg[j], rg[j + 1], sa2, scale_smem + c * 32 + j, bias_smem + c * 32 + j);
                    const float2 u = epilogue_pair<INT8, false>(ru[j], ru[j + 1], sa2, scale_smem + p.bn + c * 32 + j,
                                                                bias_smem + p.bn + c * 32 + j);
                    const __nv_bfloat162 o = __floats2bfloat162_rn(gated_act<GELU>(g.x) * u.x, gated_act<GELU>(g.y) * u.y);
                    wo[j / 2] = *reinterpret_cast<const uint32_t*>(&o);
                    if constexpr (SAVE) {
                        const __nv_bfloat162 g2 = __floats2bfloat162_rn(g.x, g.y), u2 = __floats2bfloat162_rn(u.x, u.y);
                        wg[j / 2] = *reinterpret_cast<const uint32_t*>(&g2);
                        wu[j / 2] = *reinterpret_cast<const uint32_t*>(&u2);
                    }
                }
                store_chunk(&tmap_out, wo, nc * 2, row0, 0);
                if constexpr (SAVE) {                          // [M, 2, F]: the gate's columns end at F, not in the up projection's
                    store_chunk(&tmap_pre, wg, nc * 2, 0, row0);
                    store_chunk(&tmap_pre, wu, nc * 2, 1, row0);
                }
            }
            ptx::tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) ptx::mbar_arrive_cluster(leader_tmem_empty_bar(acc));   // the leader's MMA thread waits for both CTAs
        }
        if (lane == 0) ptx::bulk_wait_group<0>();              // this warp's stores are performed before the CTA may exit
        if (!ok && p.status != nullptr && epi_tid == 0) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (30 << 8));
    }

    // ---------------------------------------------------- teardown: neither CTA may leave while the other can
    // still read its shared memory, signal its barriers or write its TMEM
    if (threadIdx.x == 0 && *abort_flag != 0) {
        // A wait was abandoned: copies issued before that get time to land before the CTA gives its memory up.
        const unsigned long long t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 50000ull) {}
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::cluster_sync_all();
    if (warp == 1) {
        ptx::tcgen05_fence_after_sync();
        ptx::tmem_dealloc_pair<kGatedTmemCols>(tmem_base);
    }
}

// ------------------------------------------------------------------ few rows
// With few rows the weight is all there is to move, and pair tiles leave half of the tensor cores' rows and, with 64 tiles for 8192
// columns, a seventh of the SMs idle.  Here every CTA owns 128 rows x bn columns (bn a multiple of 8, chosen so that the tiles fill the
// device once): the first bn rows of its B operand come from Wg, the last bn from Wu.  Of A only the rows that exist are loaded, into a
// slot of their size, so that the ring holds most of a tile's weights at once; the MMA reads 128 rows from there all the same, which
// brings whatever lies behind into accumulator rows that nobody looks at.
//
// Up to eight rows (FUSED) are rotated and quantised here as well, by the epilogue's warps of every CTA for itself while the weight streams
// in: a kernel less, and what it computes again costs nothing that anybody waits for.  1 x 2048 x 8192 int8 with its quantizer 11.4 ->
// 9.4 us.
//
// With `early` the weight's first loads are issued before the wait for the kernel before this one, which quantises the activation.
// The caller vouches that the weight was complete when that kernel began: it did not let this one start before its own wait.
constexpr int kGatedFewMaxStages = 16;
constexpr int kGatedFewMaxBN = 128;
struct GatedFewTail {                        // behind the operand ring
    static constexpr int kNumBars = 2 * kGatedFewMaxStages + 1;
    static constexpr int kTmemPtrOffset = kNumBars * 8;
    static constexpr int kAbortOffset = kTmemPtrOffset + 4;
    static constexpr int kScaleOffset = (kAbortOffset + 4 + 15) & ~15;
    static constexpr int kBiasOffset = kScaleOffset + 2 * kGatedFewMaxBN * 4;
    static constexpr int kTotal = kBiasOffset + 2 * kGatedFewMaxBN * 4;
};
struct GatedFewParams {
    const float* a_scales;
    const float* b_scales;
    const float* bias;
    __nv_bfloat16* out;                      // [M, F]
    __nv_bfloat16* pre;                      // [M, 2, F] or null
    int* status;
    int M, F, K;
    int bn, n_tiles;
    int stages, a_slot, stage_bytes, load_bytes;
    int early;
    uint32_t idesc;
    // FUSED: the rows of the activation, and where the quantised ones (1 KB per slab of K) and the rotations' buffers lie
    const __nv_bfloat16* x;
    float scale;                             // of the rotation
    int rotate, log_n, groups;               // columns padded to 2^log_n; groups of threads that take a row each
    int a_offset, buf_offset;
};

constexpr int kGatedFusedRows = 8;
// Position of element e in a rotation's buffer: a pad word after every eight, so that runs of eight and their strides spread over the banks.
__device__ __forceinline__ int gated_buf(int e) { return e + (e >> 3); }

// The quantised activation of up to eight rows, into the operand layout of the MMA (rows of 128 bytes, 16-byte pieces XOR the row), by the
// 256 epilogue threads.  The same values and bits as q8k_gated_quant: butterflies in fp32, stride 1 first, then the scale, the
// rounding to bf16 and the row's grid.  A row with NaN has NaN as its maximum and scale: int8 bytes could not hold it.
template <bool INT8>
__device__ __forceinline__ void gated_quant_rows(const GatedFewParams& p, uint8_t* smem, float* a_scales, float* red, int k_iters) {
    const int threads = kGemmEpilogueThreads / p.groups;       // 64, 128 or 256
    const int tid = (int)threadIdx.x - 64;
    const int group = tid / threads, t = tid - group * threads;
    auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(2 + group), "r"(threads) : "memory"); };
    float* buf = reinterpret_cast<float*>(smem + p.buf_offset) + group * gated_buf(1 << p.log_n);
    uint8_t* a = smem + p.a_offset;
    const int n = 1 << p.log_n;
    for (int row = group; row < p.M; row += p.groups) {
        const __nv_bfloat16* xr = p.x + (int64_t)row * p.K;
        float amax = 0.f;
        if (p.rotate) {
            for (int b = t; b < n / 8; b += threads) {         // strides 1, 2, 4 on the way in
                float v[8];
                if (b * 8 < p.K) load_vec<__nv_bfloat16, 8>(xr + b * 8, v);
                else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) v[j] = 0.f;
                }
                butterfly_consecutive<8>(v);
#pragma unroll
                for (int j = 0; j < 8; ++j) buf[gated_buf(b * 8 + j)] = v[j];
            }
            for (int lo = 3; lo < p.log_n; lo += 3) {          // then strides 2^lo, 2^(lo+1), 2^(lo+2), as far as there are
                sync();
                const int bits = p.log_n - lo < 3 ? p.log_n - lo : 3;
                const bool last = lo + 3 >= p.log_n;
                for (int b = t; b < n / 8; b += threads) {
                    // eight elements: one butterfly of eight, or at the last strides 8 >> bits neighbouring ones of 2^bits
                    int e[8];
                    float v[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        e[j] = bits == 3 ? (b >> lo << (lo + 3)) + (b & ((1 << lo) - 1)) + (j << lo)
                                         : b * (8 >> bits) + (j >> bits) + ((j & ((1 << bits) - 1)) << lo);
                        v[j] = buf[gated_buf(e[j])];
                    }
#pragma unroll
                    for (int st = 0; st < 3; ++st) {
                        if (st < bits) {
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const int k = ((h >> st) << (st + 1)) | (h & ((1 << st) - 1));
                                const float f = v[k], g = v[k + (1 << st)];
                                v[k] = __fadd_rn(f, g);
                                v[k + (1 << st)] = __fsub_rn(f, g);
                            }
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        if (last) {
                            v[j] = __bfloat162float(__float2bfloat16_rn(__fmul_rn(v[j], p.scale)));
                            if (e[j] < p.K) amax = max_nan(amax, fabsf(v[j]));
                        }
                        buf[gated_buf(e[j])] = v[j];
                    }
                }
            }
        } else {
            for (int b = t; b < p.K / 8; b += threads) {
                float v[8];
                load_vec<__nv_bfloat16, 8>(xr + b * 8, v);
#pragma unroll
                for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(v[j]));
            }
        }
        amax = warp_max<true>(amax);
        if ((tid & 31) == 0) red[tid >> 5] = amax;
        sync();
        for (int k = 0; k < threads / 32; ++k) amax = max_nan(amax, red[group * (threads / 32) + k]);
        const float f = quant_factor<true>(INT8 ? 127.0f : 448.0f, amax);
        const float mul = amax == 0.f ? 0.f : f;
        if (t == 0) a_scales[row] = __fdiv_rn(1.0f, f);
        for (int c = t; c < k_iters * 8; c += threads) {       // 16 elements each; zeros behind K
            union { uint4 v; uint8_t b[16]; uint16_t h[8]; } o;
            o.v = make_uint4(0, 0, 0, 0);
            if (c * 16 < p.K) {
                float v[16];
                if (p.rotate) {
#pragma unroll
                    for (int j = 0; j < 16; ++j) v[j] = buf[gated_buf(c * 16 + j)];
                } else {
                    load_vec<__nv_bfloat16, 16>(xr + c * 16, v);
                }
#pragma unroll
                for (int j = 0; j < 16; j += 2) {
                    const float y0 = __fmul_rn(v[j], mul), y1 = __fmul_rn(v[j + 1], mul);
                    if constexpr (INT8) {                      // halves away from zero: see tokenwise_quant_kernel
                        o.b[j] = (uint8_t)(int8_t)__float2int_rz(__fadd_rn(y0, copysignf(0.49999997f, y0)));
                        o.b[j + 1] = (uint8_t)(int8_t)__float2int_rz(__fadd_rn(y1, copysignf(0.49999997f, y1)));
                    } else {
                        o.h[j / 2] = float2_to_e4m3x2_sat(y0, y1);
                    }
                }
            }
            *reinterpret_cast<uint4*>(a + (c >> 3) * 1024 + row * 128 + (((c & 7) ^ row) << 4)) = o.v;
        }
        sync();                                                // the buffer and the partial maxima have been read
    }
}

template <int COLS> __device__ __forceinline__ void gated_few_tmem(bool alloc, uint32_t arg) {
    if (alloc) ptx::tmem_alloc<COLS>(arg);
    else ptx::tmem_dealloc<COLS>(arg);
}
__device__ __forceinline__ void gated_few_tmem_any(int bn, bool alloc, uint32_t arg) {   // whole warp, convergent
    if (bn <= 16) gated_few_tmem<32>(alloc, arg);
    else if (bn <= 32) gated_few_tmem<64>(alloc, arg);
    else if (bn <= 64) gated_few_tmem<128>(alloc, arg);
    else gated_few_tmem<256>(alloc, arg);
}

template <bool INT8, bool GELU, bool FUSED>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_8bit_gated_few_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                           const __grid_constant__ GatedFewParams p) {
    using L = GatedFewTail;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t smem_base = ptx::smem_u32(smem);
    uint8_t* tail = smem + p.stages * p.stage_bytes;
    const uint32_t bar_base = ptx::smem_u32(tail);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kGatedFewMaxStages + s); };
    const uint32_t acc_bar = bar_base + 8u * (2 * kGatedFewMaxStages);
    volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(tail + L::kTmemPtrOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + L::kAbortOffset);
    float* scale_smem = reinterpret_cast<float*>(tail + L::kScaleOffset);
    float* bias_smem = reinterpret_cast<float*>(tail + L::kBiasOffset);
    __shared__ int prior_failure;
    __shared__ float fused_scales[FUSED ? kGatedFusedRows : 1], fused_red[FUSED ? kGemmEpilogueThreads / 32 : 1];

    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int m0 = (int)(blockIdx.x / p.n_tiles) * kGemmBM;
    const int n0 = (int)(blockIdx.x % p.n_tiles) * p.bn;
    const int k_iters = (p.K + kGemmBK - 1) / kGemmBK;

    if (threadIdx.x == 0) {
        for (int s = 0; s < p.stages; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
        }
        ptx::mbar_init(acc_bar, 1);
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        ptx::prefetch_tensormap(&tmap_w);
        if (!FUSED) ptx::prefetch_tensormap(&tmap_a);
    }
    if (warp == 1) {
        gated_few_tmem_any(p.bn, true, ptx::smem_u32(const_cast<uint32_t*>(tmem_ptr_smem)));
        ptx::tmem_relinquish_alloc_permit();
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::tcgen05_fence_after_sync();
    const uint32_t tmem_base = *tmem_ptr_smem;
    auto load_weight = [&](int s, int kb) {                    // (columns from F on: see gemm_8bit_gated_kernel; no store takes them)
        const uint32_t dst = smem_base + s * p.stage_bytes + p.a_slot;
        ptx::mbar_arrive_expect_tx(full_bar(s), (uint32_t)p.load_bytes);
        ptx::tma_load_2d(dst, &tmap_w, full_bar(s), kb * kGemmBK, n0);
        ptx::tma_load_2d(dst + p.bn * kGemmBK, &tmap_w, full_bar(s), kb * kGemmBK, p.F + n0);
    };
    const int ahead = p.early ? min(p.stages, k_iters) : 0;
    if (warp == 0 && ahead > 0) {
        if (ptx::elect_one()) {
            for (int s = 0; s < ahead; ++s) load_weight(s, s);
        }
        __syncwarp();
    }
    pdl_wait();
    if (threadIdx.x == 0) prior_failure = p.status != nullptr ? *reinterpret_cast<volatile int*>(p.status) : 0;
    __syncthreads();
    pdl_release();                                             // this CTA holds its TMEM: the next kernel may move in behind it
    // A launch that follows a failed one on the same status word stores nothing (loads that are under way have to land).
    bool ok = true;
    const bool skip = prior_failure != 0;

    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    if (warp == 0) {
        if (ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 1;                                   // empty_bar phase to wait for: the first round passes
            for (int kb = 0; kb < k_iters; ++kb) {
                if (kb >= ahead) {
                    if (!ptx::mbar_wait(empty_bar(s), ph, abort_flag)) { ok = false; break; }
                    load_weight(s, kb);
                }
                if (!FUSED) ptx::tma_load_2d(smem_base + s * p.stage_bytes, &tmap_a, full_bar(s), kb * kGemmBK, m0);
                if (++s == p.stages) { s = 0; ph ^= 1u; }
            }
            if (!ok && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (32 << 8));
        }
        __syncwarp();
    } else if (warp == 1) {
        if (FUSED) asm volatile("bar.sync 6, 288;" ::: "memory");              // the quantised rows are there
        if (ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            for (int kb = 0; kb < k_iters; ++kb) {
                if (!ptx::mbar_wait(full_bar(s), ph, abort_flag)) { ok = false; break; }
                ptx::tcgen05_fence_after_sync();
                const uint32_t stage = smem_base + s * p.stage_bytes;
                const uint64_t a_desc = ptx::make_kmajor_desc(FUSED ? smem_base + p.a_offset + kb * 1024 : stage, 128);
                const uint64_t b_desc = ptx::make_kmajor_desc(stage + p.a_slot, 128);
#pragma unroll
                for (int k = 0; k < kGemmBK / 32; ++k) {
                    const uint32_t accumulate = (kb > 0 || k > 0) ? 1u : 0u;
                    if constexpr (INT8) ptx::mma_i8(tmem_base, a_desc + 2 * k, b_desc + 2 * k, p.idesc, accumulate);
                    else ptx::mma_f8f6f4(tmem_base, a_desc + 2 * k, b_desc + 2 * k, p.idesc, accumulate);
                }
                ptx::tcgen05_commit(empty_bar(s));
                if (++s == p.stages) { s = 0; ph ^= 1u; }
            }
            if (ok) ptx::tcgen05_commit(acc_bar);
            else if (p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (33 << 8));
        }
        __syncwarp();
    } else {
        for (int c = (int)threadIdx.x - 64; c < 2 * p.bn; c += kGemmEpilogueThreads) {
            const bool up = c >= p.bn;
            const int n = n0 + (up ? c - p.bn : c);
            const bool in = n < p.F;
            const int at = up ? p.F + n : n;
            scale_smem[c] = in ? p.b_scales[at] : 0.f;
            bias_smem[c] = in && p.bias != nullptr ? p.bias[at] : 0.f;
        }
        if constexpr (FUSED) {
            gated_quant_rows<INT8>(p, smem, fused_scales, fused_red, k_iters);
            ptx::fence_proxy_async_smem();                     // the MMA reads through the async proxy
            asm volatile("bar.sync 6, 288;" ::: "memory");
        } else {
            asm volatile("bar.sync 1, 256;" ::: "memory");
        }
        const int row = m0 + quarter * 32 + lane;
        const bool row_ok = row < p.M && !skip;
        const float sa = row >= p.M ? 0.f : FUSED ? fused_scales[row & (kGatedFusedRows - 1)] : p.a_scales[row];
        const float2 sa2 = make_float2(sa, sa);
        ok = ptx::mbar_wait(acc_bar, 0, abort_flag);
        ok = __all_sync(0xffffffffu, ok);                      // keep the warp convergent for tcgen05.ld
        ptx::tcgen05_fence_after_sync();
        if (!ok && p.status != nullptr && threadIdx.x == 64) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (34 << 8));
        if (ok && m0 + quarter * 32 < p.M) {                   // (warp-uniform)
            const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
            // groups of eight columns in turn: F % 16 == 0, so eight are all in or all out
#pragma unroll 1
            for (int c = half * 8; c < p.bn && n0 + c < p.F; c += 16) {
                uint32_t rg[8], ru[8];
                ptx::tmem_ld_32x32b_x8(t_row + c, rg);
                ptx::tmem_ld_32x32b_x8(t_row + p.bn + c, ru);
                ptx::tmem_wait_ld();
                uint32_t wo[4], wg[4], wu[4];
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const float2 g = epilogue_pair<INT8, false>(rg[j], rg[j + 1], sa2, scale_smem + c + j, bias_smem + c + j);
                    const float2 u = epilogue_pair<INT8, false>(ru[j], ru[j + 1], sa2, scale_smem + p.bn + c + j, bias_smem + p.bn + c + j);
                    const __nv_bfloat162 o = __floats2bfloat162_rn(gated_act<GELU>(g.x) * u.x, gated_act<GELU>(g.y) * u.y);
                    const __nv_bfloat162 g2 = __floats2bfloat162_rn(g.x, g.y), u2 = __floats2bfloat162_rn(u.x, u.y);
                    wo[j / 2] = *reinterpret_cast<const uint32_t*>(&o);
                    wg[j / 2] = *reinterpret_cast<const uint32_t*>(&g2);
                    wu[j / 2] = *reinterpret_cast<const uint32_t*>(&u2);
                }
                if (row_ok) {
                    *reinterpret_cast<uint4*>(p.out + (int64_t)row * p.F + n0 + c) = make_uint4(wo[0], wo[1], wo[2], wo[3]);
                    if (p.pre != nullptr) {
                        __nv_bfloat16* pr = p.pre + (int64_t)row * 2 * p.F + n0 + c;
                        *reinterpret_cast<uint4*>(pr) = make_uint4(wg[0], wg[1], wg[2], wg[3]);
                        *reinterpret_cast<uint4*>(pr + p.F) = make_uint4(wu[0], wu[1], wu[2], wu[3]);
                    }
                }
                __syncwarp();
            }
        }
    }

    if (threadIdx.x == 0 && *abort_flag != 0) {
        // a wait was abandoned: give copies still in flight time to land before the CTA gives up its shared memory
        const unsigned long long t0 = ptx::globaltimer_ns();
        while (ptx::globaltimer_ns() - t0 < 50000ull) {}
    }
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        ptx::tcgen05_fence_after_sync();
        gated_few_tmem_any(p.bn, false, tmem_base);
    }
}

// ------------------------------------------------------------------ host side
template <bool INT8, bool GELU, bool SAVE>
static int launch_gated_as(const CUtensorMap& ta, const CUtensorMap& tw, const CUtensorMap& to, const CUtensorMap& tp,
                           const GatedParams& p, cudaStream_t st) {
    using L = GatedSmemT<SAVE>;
    auto kern = gemm_8bit_gated_kernel<INT8, GELU, SAVE>;
    static std::atomic<uint64_t> smem_done{0};
    if (int rc = allow_dynamic_smem((const void*)kern, L::kTotal, smem_done)) return rc;
    static std::atomic<int> max_clusters{-1};                  // 2-CTA clusters that can be resident at once
    int most = max_clusters.load(std::memory_order_relaxed);
    if (most < 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(2 * gemm_num_sms());
        cfg.blockDim = dim3(kGemmThreads);
        cfg.dynamicSmemBytes = L::kTotal;
        cudaLaunchAttribute attr;
        attr.id = cudaLaunchAttributeClusterDimension;
        attr.val.clusterDim.x = 2; attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
        cfg.attrs = &attr;
        cfg.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&most, kern, &cfg) != cudaSuccess) { cudaGetLastError(); most = 0; }
        max_clusters.store(most, std::memory_order_relaxed);
    }
    if (most < 1) return Q8K_ERR_UNSUPPORTED;
    const int clusters = p.total_tiles < most ? p.total_tiles : most;
    Q8K_CUDA_OK(launch_dependent(kern, 2 * clusters, kGemmThreads, L::kTotal, st, 1, ta, tw, to, tp, p));
    return Q8K_OK;
}

// Which kernel and tiles: those with the shortest estimate (us).
//   pair: 3.3, and for every round of tiles 1.5 and per 128-byte slab of K 0.165 for the issuing threads or 0.31 at 256 columns
//         of the product
//   few:  where its tiles fill the device at most once (or there are at most 128 rows): 3.3, the epilogue's 1.5e-4 bn^2, and the
//         longer of the slabs, each 0.165 or its bytes at 140 GB/s of one SM's L2 port, and the weight at 5.5 TB/s
// Measured, best tiles of either (pair against few, CUDA graphs, weights from HBM): M = 1, K = 2048, F = 8192 14.1 against 8.8;  M = 77,
// K = 4096, F = 10240 23.5 against 16.9;  M = 128, K = 2048, F = 8192 11.7 against 9.5;  M = 129 11.8 against 12.4;  M = 512 16.4 against
// 22.5;  K = F = 4096, M = 256 12.0 against 11.3, M = 384 15.7 against 13.6;  K = 2048, F = 5504, M = 300 13.4 against 12.0, M = 600 15.8
// against 18.8;  K = 2048, F = 688, M = 1000 7.0 against 6.2;  K = 512, F = 1408, M = 1001 5.9 against 5.3, M = 2002 8.1 against 10.3.
struct GatedPlan { bool few; int bn; };
static GatedPlan gated_plan(int M, int F, int K, int sms) {
    const double slabs = (K + kGemmBK - 1) / kGemmBK;
    const int clusters = sms / 2;
    double best = 1e30;
    GatedPlan plan = {false, kGatedBN};
    for (int c = kGatedBN; c >= 32; c -= 32) {
        const double tiles = (double)((M + 2 * kGemmBM - 1) / (2 * kGemmBM)) * ((F + c - 1) / c);
        const double rounds = (double)(int64_t)((tiles + clusters - 1) / clusters);
        const double slab = 0.31 * c / kGatedBN > 0.165 ? 0.31 * c / kGatedBN : 0.165;
        const double t = 3.3 + rounds * (slabs * slab + 1.5);
        if (t < best) { best = t; plan.bn = c; }
    }
    // the narrowest tiles that fill the device once
    const int64_t m_tiles = (M + kGemmBM - 1) / kGemmBM;
    const int64_t per_row = sms / m_tiles;                     // tiles that 128 rows may have
    int64_t bn = per_row == 0 ? kGatedFewMaxBN + 1 : ((F + per_row - 1) / per_row + 7) / 8 * 8;
    if (bn < 16) bn = 16;
    if (M <= kGemmBM && bn > kGatedFewMaxBN) bn = kGatedFewMaxBN;
    if (bn > kGatedFewMaxBN) return plan;
    const int a_rows = M >= kGemmBM ? kGemmBM : (M + 7) / 8 * 8;
    const double bytes = (double)(a_rows + 2 * bn) * kGemmBK / 140e3;
    const double stream = slabs * (bytes > 0.165 ? bytes : 0.165), weight = 2.0 * F * K / 5.5e6;
    if (M <= kGemmBM || 3.3 + 1.5e-4 * bn * bn + (stream > weight ? stream : weight) < best) {
        plan.few = true;
        plan.bn = (int)bn;
    }
    return plan;
}

// x: with it the rows are quantised in the kernel (`a` and the scales are not looked at).
template <bool INT8, bool GELU, bool FUSED>
static int launch_gated_few(const void* a, const void* w, const GatedParams& g, void* out, void* pre, int bn, bool early, const void* x, bool rotate,
                            cudaStream_t st, const char* op) {
    GatedFewParams p = {};
    p.a_scales = g.a_scales; p.b_scales = g.b_scales; p.bias = g.bias;
    p.out = (__nv_bfloat16*)out; p.pre = (__nv_bfloat16*)pre;
    p.status = g.status;
    p.M = g.M; p.F = g.F; p.K = g.K;
    const int a_rows = g.M >= kGemmBM ? kGemmBM : (g.M + 7) / 8 * 8;
    p.bn = bn;
    p.n_tiles = (g.F + bn - 1) / bn;
    p.a_slot = FUSED ? 0 : a_rows * kGemmBK;
    p.load_bytes = p.a_slot + 2 * bn * kGemmBK;
    p.stage_bytes = p.load_bytes;                              // (a multiple of 1024: a_rows and bn are of 8)
    const int k_iters = (g.K + kGemmBK - 1) / kGemmBK;
    // the MMA of the last slab reads 16 KB from its rows of A on, the shared memory ends there or later
    int extra = kGemmBM * kGemmBK;
    if constexpr (FUSED) {
        p.x = (const __nv_bfloat16*)x;
        p.rotate = rotate;
        p.scale = 1.0f / sqrtf((float)g.K);
        p.log_n = 3;
        while ((1 << p.log_n) < g.K) ++p.log_n;
        const int row_bytes = (1 << p.log_n) / 8 * 9 * (int)sizeof(float);
        p.groups = 4;
        while (p.groups > 1 && (p.groups > g.M || p.groups * row_bytes > 48 * 1024)) p.groups /= 2;
        const int bufs = rotate ? (p.groups * row_bytes + 1023) / 1024 * 1024 : 0;
        extra = k_iters * 1024 + (bufs > extra ? bufs : extra);
    }
    const int budget = 224 * 1024 - GatedFewTail::kTotal - extra;
    p.stages = budget / p.stage_bytes;
    if (p.stages > kGatedFewMaxStages) p.stages = kGatedFewMaxStages;
    if (p.stages > k_iters) p.stages = k_iters;
    Q8K_REQUIRE(p.stages >= 1, Q8K_ERR_UNSUPPORTED, "%s: no room for the operands", op);
    if constexpr (FUSED) {                                     // behind the ring and its barriers
        p.a_offset = (p.stages * p.stage_bytes + GatedFewTail::kTotal + 1023) / 1024 * 1024;
        p.buf_offset = p.a_offset + k_iters * 1024;
    }
    p.early = early ? 1 : 0;
    p.idesc = INT8 ? ptx::make_idesc_s8(kGemmBM, 2 * bn) : ptx::make_idesc_e4m3(kGemmBM, 2 * bn);
    CUtensorMap ta, tw;
    {
        const uint64_t dims[2] = {(uint64_t)g.K, 2 * (uint64_t)g.F};
        const uint64_t strides[1] = {(uint64_t)g.K};
        const uint32_t box[2] = {(uint32_t)kGemmBK, (uint32_t)bn};
        if (int rc = make_byte_tensor_map(&tw, w, 2, dims, strides, box, 128, op)) return rc;
    }
    ta = tw;
    if constexpr (!FUSED) {
        const uint64_t dims[2] = {(uint64_t)g.K, (uint64_t)g.M};
        const uint64_t strides[1] = {(uint64_t)g.K};
        const uint32_t box[2] = {(uint32_t)kGemmBK, (uint32_t)a_rows};
        if (int rc = make_byte_tensor_map(&ta, a, 2, dims, strides, box, 128, op)) return rc;
    }
    auto kern = gemm_8bit_gated_few_kernel<INT8, GELU, FUSED>;
    static std::atomic<uint64_t> smem_done{0};
    if (int rc = allow_dynamic_smem((const void*)kern, 226 * 1024, smem_done)) return rc;
    const int smem = 1024 + (FUSED ? p.a_offset : p.stages * p.stage_bytes + GatedFewTail::kTotal) + extra;
    const int64_t grid = (int64_t)((g.M + kGemmBM - 1) / kGemmBM) * p.n_tiles;
    Q8K_REQUIRE(grid <= 0x7fffffffLL, Q8K_ERR_TOO_LARGE, "%s: too many tiles", op);
    Q8K_CUDA_OK(launch_dependent(kern, (unsigned)grid, kGemmThreads, smem, st, 1, ta, tw, p));
    return Q8K_OK;
}

bool gated_fused_rows(int M, int K) { return M <= kGatedFusedRows && K <= 8192; }

int gated_mm_fused(const char* op, bool int8, const void* x, bool rotate, const void* w, const float* bias, const float* w_scales, void* out,
                   void* pre, int activation, int M, int F, int K, int* dev_status, void* stream) {
    const GatedParams p = {nullptr, w_scales, bias, dev_status, M, F, K, 0, 0, 0};
    const int bn = gated_plan(M, F, K, gemm_num_sms()).bn;
    const bool gelu = activation == Q8K_ACT_GELU_TANH;
    cudaStream_t st = (cudaStream_t)stream;
    return int8 ? (gelu ? launch_gated_few<true, true, true>(nullptr, w, p, out, pre, bn, false, x, rotate, st, op)
                        : launch_gated_few<true, false, true>(nullptr, w, p, out, pre, bn, false, x, rotate, st, op))
                : (gelu ? launch_gated_few<false, true, true>(nullptr, w, p, out, pre, bn, false, x, rotate, st, op)
                        : launch_gated_few<false, false, true>(nullptr, w, p, out, pre, bn, false, x, rotate, st, op));
}

int gated_mm(const char* op, bool weight_ready, int int8, const void* a, const void* w, const float* bias, const float* a_scales,
             const float* w_scales, void* out, void* pre, int activation, int M, int F, int K, int* dev_status, void* stream) {
    Q8K_REQUIRE(M >= 0 && F > 0 && K > 0, Q8K_ERR_INVALID_ARG, "%s: bad shape M=%d F=%d K=%d", op, M, F, K);
    Q8K_REQUIRE(F % 16 == 0 && K % 16 == 0, Q8K_ERR_INVALID_ARG, "%s: F=%d and K=%d must be multiples of 16", op, F, K);
    Q8K_REQUIRE(F <= 0x3fffffff && M <= 0x7fffffff - 2 * kGemmBM, Q8K_ERR_TOO_LARGE, "%s: M=%d or F=%d too large", op, M, F);
    Q8K_REQUIRE(activation == Q8K_ACT_SILU || activation == Q8K_ACT_GELU_TANH, Q8K_ERR_UNSUPPORTED, "%s: activation %d is unknown", op,
                activation);
    if (M == 0) return Q8K_OK;
    Q8K_REQUIRE(a && w && a_scales && w_scales && out, Q8K_ERR_INVALID_ARG, "%s: null pointer", op);
    Q8K_REQUIRE(aligned16(a) && aligned16(w) && aligned16(out) && aligned16(pre), Q8K_ERR_INVALID_ARG,
                "%s: a, w, out and pre must be 16-byte aligned", op);
    GatedParams p = {a_scales, w_scales, bias, dev_status, M, F, K, 0, 0, 0};
    const GatedPlan plan = gated_plan(M, F, K, gemm_num_sms());
    const bool gelu = activation == Q8K_ACT_GELU_TANH;
    cudaStream_t st = (cudaStream_t)stream;
    auto few = [&](int bn) {
        return int8 ? (gelu ? launch_gated_few<true, true, false>(a, w, p, out, pre, bn, weight_ready, nullptr, false, st, op)
                            : launch_gated_few<true, false, false>(a, w, p, out, pre, bn, weight_ready, nullptr, false, st, op))
                    : (gelu ? launch_gated_few<false, true, false>(a, w, p, out, pre, bn, weight_ready, nullptr, false, st, op)
                            : launch_gated_few<false, false, false>(a, w, p, out, pre, bn, weight_ready, nullptr, false, st, op));
    };
    if (plan.few) return few(plan.bn);
    p.bn = plan.bn;
    p.n_tiles = (F + p.bn - 1) / p.bn;
    const int64_t total = (int64_t)((M + 2 * kGemmBM - 1) / (2 * kGemmBM)) * p.n_tiles;
    Q8K_REQUIRE(total <= 0x7fffffffLL, Q8K_ERR_TOO_LARGE, "%s: too many tiles", op);
    p.total_tiles = (int)total;
    CUtensorMap ta, tw, to, tp;
    {
        const uint64_t dims[2] = {(uint64_t)K, (uint64_t)M};
        const uint64_t strides[1] = {(uint64_t)K};
        const uint32_t box[2] = {(uint32_t)kGemmBK, (uint32_t)kGemmBM};
        if (int rc = make_byte_tensor_map(&ta, a, 2, dims, strides, box, 128, op)) return rc;
    }
    {
        const uint64_t dims[2] = {(uint64_t)K, 2 * (uint64_t)F};
        const uint64_t strides[1] = {(uint64_t)K};
        const uint32_t box[2] = {(uint32_t)kGemmBK, (uint32_t)p.bn};
        if (int rc = make_byte_tensor_map(&tw, w, 2, dims, strides, box, 128, op)) return rc;
    }
    {
        const uint64_t dims[3] = {2 * (uint64_t)F, (uint64_t)M, 1};
        const uint64_t strides[2] = {2 * (uint64_t)F, 2 * (uint64_t)F * (uint64_t)M};
        const uint32_t box[3] = {64, 32, 1};
        if (int rc = make_byte_tensor_map(&to, out, 3, dims, strides, box, 64, op)) return rc;
    }
    tp = to;
    if (pre != nullptr) {
        const uint64_t dims[3] = {2 * (uint64_t)F, 2, (uint64_t)M};
        const uint64_t strides[2] = {2 * (uint64_t)F, 4 * (uint64_t)F};
        const uint32_t box[3] = {64, 1, 32};
        if (int rc = make_byte_tensor_map(&tp, pre, 3, dims, strides, box, 64, op)) return rc;
    }
#define Q8K_GATED(I8, SV) (gelu ? launch_gated_as<I8, true, SV>(ta, tw, to, tp, p, st) : launch_gated_as<I8, false, SV>(ta, tw, to, tp, p, st))
    int rc;
    if (pre != nullptr) rc = int8 ? Q8K_GATED(true, true) : Q8K_GATED(false, true);
    else rc = int8 ? Q8K_GATED(true, false) : Q8K_GATED(false, false);
#undef Q8K_GATED
    if (rc != Q8K_ERR_UNSUPPORTED) return rc;
    return few(F < kGatedFewMaxBN ? (F + 7) / 8 * 8 : kGatedFewMaxBN);         // the device cannot co-schedule the pairs
}

}  // namespace q8k

extern "C" int q8k_gated_mm(int int8, const void* a, const void* w, const float* bias, const float* a_scales, const float* w_scales,
                            void* out, void* pre, int activation, int M, int F, int K, int* dev_status, void* stream) {
    return q8k::gated_mm("gated_mm", false, int8, a, w, bias, a_scales, w_scales, out, pre, activation, M, F, K, dev_status, stream);
}

extern "C" int q8k_gated_plan(int M, int F, int K, int plan[2]) {
    using q8k::set_error_detail;
    Q8K_REQUIRE(plan != nullptr && M > 0 && F > 0 && K > 0, Q8K_ERR_INVALID_ARG, "gated_plan: null plan or bad shape");
    const q8k::GatedPlan p = q8k::gated_plan(M, F, K, q8k::gemm_num_sms());
    plan[0] = p.few ? 0 : 1;
    plan[1] = p.bn;
    return Q8K_OK;
}
