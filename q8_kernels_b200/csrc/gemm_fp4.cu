// 4-bit GEMM with block scales: out = act((A . B^T) * (ra[m] * rb[n]) + bias[n]), A [M, K] and B [N, K] both mxfp4 or both nvfp4 (fp4.cuh).
//
// The tensor core multiplies the e2m1 values with their blocks' scales and adds in fp32 (kind::mxf4nvf4); the rows' scales (nvfp4),
// the bias, tanh-GELU and the one rounding to 16 bits are the epilogue's.
//
// 128 x bn tiles, bn of 32, 64, 128 or 192, one a CTA: for products that 256 x 256 tiles on CTA pairs (gemm_fp4_pair.cu) do not spread over the
// device.  Roles (10 warps):
//   warp 0     TMA producer: values, in slabs of 256 along K (128 bytes), and block scales of the tile's rows and columns
//   warp 1     TMEM allocation; one thread issues a slab's four MMAs (K = 64)
//   warps 2-9  block scales from shared memory to TMEM, warps 2-5 those in even stages and 6-9 those in odd ones; then the epilogue
//   FEW        warps 2-9 first quantise the rows of A, up to eight, which then stay in shared memory for all slabs
// All waits are bounded.
//
// Bound by the latency of one short main loop, a few slabs to each of few CTAs.  The tensor core's own copy of scales (tcgen05.cp, 512 bytes)
// stands in the pipe of the MMAs for some 65 clocks, and a slab of nvfp4 needs eight of them.  Registers bring
// the scales past that pipe, every stage to its own columns.  Measured with M = 1 on cold operands, tcgen05.cp -> registers, us:
//   nvfp4 N x K = 2048 x 2048 5.2 -> 4.2, 2048 x 8192 15.2 -> 10.2, 8192 x 2048 6.4 -> 5.9; mxfp4 4.3 -> 4.1, 10.9 -> 9.3, 5.7 -> 5.2.  All that the epilogue needs from global
// memory, the status word too, is read beside the main loop, which before waited for it (5.9 -> 5.4, 5.2 -> 4.9).
//
// What is left of a slab are some 450 clocks of two threads, whose waits (70 clocks each even for what has come) and issues follow one another: two waits,
// four MMAs and a commit of the one, a wait and four copies of the other; the MMAs themselves are not it (one in the place of four: 5 %).  Not kept:
// loads by two or three warps (no change), accumulators of their own for the four MMAs (no change), stages of two slabs, which leave fewer of them
// (16 x 2048 x 8192 9.9 -> 9.1 us, but 128 x 20480 x 4096 15.0 -> 17.6, 77 x 10240 x 4096 9.4 -> 10.3).  With fewer than 128 rows a stage holds those rows only, and there are
// up to 16 of them (1 x 20480 x 4096 13.3 -> 12.3 us): the MMA's other rows are whatever follows in shared memory, other stages' values as they come
// and go, and give rows that nobody reads.
//
// The scales of B can be named from every second column of TMEM only, i.e. from rows n that are multiples of 64.  A tile of 32 columns
// multiplies the 64 from the multiple of 64 below; the rows of B that it does not own are not loaded there, and what stands in their place
// gives columns that nobody reads.

#include "gemm_fp4.cuh"
#include "fp4_quant.cuh"

namespace q8k {

constexpr int kFp4MaxStages = 16;
constexpr int kFp4MaxBN = 192;
constexpr int kFp4ABytes = kGemmBM * 128;
constexpr int kFp4Few = 8;                   // rows that the product quantises itself, one group of the operand's layout
struct Fp4Smem {                             // behind the operand ring
    static constexpr int kNumBars = 3 * kFp4MaxStages + 2;
    static constexpr int kTmemPtrOffset = kNumBars * 8;
    static constexpr int kAbortOffset = kTmemPtrOffset + 4;
    static constexpr int kColScaleOffset = (kAbortOffset + 4 + 15) & ~15;
    static constexpr int kBiasOffset = kColScaleOffset + kFp4MaxBN * 4;
    static constexpr int kRowOffset = kBiasOffset + kFp4MaxBN * 4;             // of few rows: the absmax's bits, the scales
    static constexpr int kTotal = kRowOffset + 2 * kFp4Few * 4;
};
struct Fp4TileParams {
    Fp4GemmParams g;
    int n_tiles;
    int bn;                                  // tile columns: 32, 64, 128 or 192
    int window;                              // columns of the MMA: 64 where bn is 32, see above
    int b_tiles;                             // 128-row tiles of B's scales that a window touches: 1 or 2
    int stages, stage_bytes, a_bytes;        // a_bytes: of A's values in a stage
    int b_ahead;                             // the kernel before on the stream has nothing to do with B and waited for what came before it
    const uint8_t *a_block_scales, *b_block_scales;
    const void* x;                           // FEW: the rows that the kernel quantises, and their type
    int x_f16;
};

// Up to eight rows of x in 4 bits, by 256 threads: values as slabs of eight rows of 128 bytes, swizzled, scales as the first words of the lanes
// that hold the rows, [tile along K][8].  `tops`: zeros.
template <bool NV, typename Tin>
__device__ __forceinline__ void fp4_few_rows(const Tin* __restrict__ x, int rows, int K, int slabs, uint8_t* values, uint8_t* scales, uint32_t* tops,
                                             float* row_scales) {
    constexpr int TILES = fp4_slab_tiles(NV);
    const int warp = (threadIdx.x - 64) >> 5, lane = threadIdx.x & 31;
    const int warps = rows == 1 ? 8 : rows == 2 ? 4 : rows <= 4 ? 2 : 1;       // of a row
    const int row = warp / warps, step = 32 * warps, t0 = warp % warps * 32 + lane;
    const int units = K / kFp4Unit, filled = slabs * (kFp4Slab / kFp4Unit);    // `filled`: a multiple of 16, so half warps leave the loops together
    const bool here = row < rows;
    const Tin* from = x + (int64_t)row * K;
    uint4 first[1][2], r[1][2];
    fp4_load<Tin, 1>(from, t0, 0, units, here, first);
    float g = 0.f, rs = 0.f;
    if constexpr (NV) {
        float top = Fp4In<Tin>::absmax(first[0]);
        for (int u = t0 + step; u < units; u += step) {
            fp4_load<Tin, 1>(from, u, 0, units, here, r);
            top = max_nan(top, Fp4In<Tin>::absmax(r[0]));
        }
        top = warp_max<true>(top);
        if (lane == 0 && here) atomicMax(&tops[row], __float_as_uint(top));    // (NaN has the largest bits)
        asm volatile("bar.sync 1, 256;" ::: "memory");
        fp4_row_factors(here ? __uint_as_float(tops[row]) : 0.f, g, rs);
        if (here && t0 == 0) row_scales[row] = rs;
    }
    for (int base = t0 - lane; base < filled; base += step) {                  // the same for a warp
        const int u = base + lane;
        if (u == t0) { r[0][0] = first[0][0]; r[0][1] = first[0][1]; }
        else fp4_load<Tin, 1>(from, u, 0, units, here, r);
        float factor;
        const uint8_t scale = fp4_block_scale<NV>(Fp4In<Tin>::absmax(r[0]), g, rs, factor);
        if (!here || u >= filled) continue;
        const int slab = u >> 4, b = u & 15;
        if (u < units) *reinterpret_cast<uint2*>(values + slab * 1024 + row * 128 + (((b >> 1) ^ row) << 4) + (b & 1) * 8) = fp4_pack<Tin>(r[0], factor);
        const int block = NV ? b : b >> 1;
        if (NV || (b & 1) == 0) scales[(slab * TILES + (block >> 2)) * (4 * kFp4Few) + row * 4 + (block & 3)] = u < units ? scale : 0;
    }
}

// FEW: A is p.M <= 8 rows of x, which every CTA quantises for itself.
template <bool NV, bool GELU, bool F16, bool FEW>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_fp4_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ Fp4TileParams sp) {
    using L = Fp4Smem;
    constexpr int TILES = fp4_slab_tiles(NV);                  // 512-byte scale tiles a slab
    const Fp4GemmParams& p = sp.g;
    const int bn = sp.bn, stages = sp.stages, nt = sp.b_tiles;

    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t smem_base = ptx::smem_u32(smem);
    const int slabs = (p.K + kFp4Slab - 1) / kFp4Slab;
    uint8_t* few_values = smem + stages * sp.stage_bytes;      // FEW: behind the ring, whose stages hold B alone
    uint8_t* few_scales = few_values + slabs * (kFp4Few * 128);
    uint8_t* tail = FEW ? few_scales + slabs * TILES * (4 * kFp4Few) : few_values;
    const uint32_t bar_base = ptx::smem_u32(tail);
    auto full_bar = [&](int s) { return bar_base + 8u * s; };
    auto empty_bar = [&](int s) { return bar_base + 8u * (kFp4MaxStages + s); };
    auto scaled_bar = [&](int s) { return bar_base + 8u * (2 * kFp4MaxStages + s); };      // its scales are in TMEM
    const uint32_t acc_bar = bar_base + 8u * (3 * kFp4MaxStages), few_bar = acc_bar + 8u;
    volatile uint32_t* tmem_ptr_smem = reinterpret_cast<volatile uint32_t*>(tail + L::kTmemPtrOffset);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tail + L::kAbortOffset);
    float* col_scale_smem = reinterpret_cast<float*>(tail + L::kColScaleOffset);
    float* bias_smem = reinterpret_cast<float*>(tail + L::kBiasOffset);
    uint32_t* few_tops = reinterpret_cast<uint32_t*>(tail + L::kRowOffset);
    float* few_row_scales = reinterpret_cast<float*>(few_tops + kFp4Few);
    const int warp = threadIdx.x >> 5;
    const int lane = threadIdx.x & 31;
    const int n_blk = blockIdx.x % sp.n_tiles;
    const int m_blk = blockIdx.x / sp.n_tiles;
    const int n0 = n_blk * bn, off = n0 % 64, window = sp.window;
    // offsets in a stage: A, B, A's scales, B's scales
    const uint32_t b_at = sp.a_bytes, as_at = b_at + (uint32_t)window * 128u, bs_at = as_at + (FEW ? 0 : fp4_slab_scales(NV));

    if (threadIdx.x == 0) {
        for (int s = 0; s < stages; ++s) {
            ptx::mbar_init(full_bar(s), 1);
            ptx::mbar_init(empty_bar(s), 1);
            ptx::mbar_init(scaled_bar(s), kGemmEpilogueThreads / 64);
        }
        ptx::mbar_init(acc_bar, 1);
        ptx::mbar_init(few_bar, 1);
        if constexpr (FEW)
            for (int i = 0; i < kFp4Few; ++i) few_tops[i] = 0;
        *abort_flag = 0;
        ptx::fence_barrier_init();
        ptx::fence_proxy_async_smem();
        if constexpr (!FEW) ptx::prefetch_tensormap(&tmap_a);
        ptx::prefetch_tensormap(&tmap_b);
    }

    // ---- warp 0's loads.  A slab's scales of one row tile lie together; behind B's last row tile there are none.
    const int row_tile = n0 / 128, b_tiles = min(nt, (p.N + 127) / 128 - row_tile);
    const uint8_t* bs = sp.b_block_scales + (int64_t)row_tile * slabs * fp4_slab_scales(NV);   // (stepped: addresses from i cost 60 clocks a slab)
    auto load_b = [&](int i, int s) {
        const uint32_t dst = smem_base + s * sp.stage_bytes;
        ptx::mbar_arrive_expect_tx(full_bar(s), sp.a_bytes + bn * 128 + ((FEW ? 0 : 1) + b_tiles) * fp4_slab_scales(NV));
        ptx::tma_load_2d(dst + b_at + (uint32_t)off * 128u, &tmap_b, full_bar(s), i * 128, n0);
        ptx::bulk_load(dst + bs_at, bs, fp4_slab_scales(NV), full_bar(s));
        if (b_tiles > 1) ptx::bulk_load(dst + bs_at + fp4_slab_scales(NV), bs + (int64_t)slabs * fp4_slab_scales(NV), fp4_slab_scales(NV), full_bar(s));
        bs += fp4_slab_scales(NV);
    };
    const int ahead = sp.b_ahead ? stages : 0;                 // (stages <= slabs)
    if (warp == 0) {
        __syncwarp();                                          // the barriers exist
        if (ptx::elect_one())
            for (int i = 0; i < ahead; ++i) load_b(i, i);
        bs = sp.b_block_scales + ((int64_t)row_tile * slabs + ahead) * fp4_slab_scales(NV);
    }
    if (warp == 1) {
        ptx::tmem_alloc<512>(ptx::smem_u32(const_cast<uint32_t*>(tmem_ptr_smem)));
        ptx::tmem_relinquish_alloc_permit();
    }
    pdl_wait();
    ptx::tcgen05_fence_before_sync();
    __syncthreads();
    ptx::tcgen05_fence_after_sync();
    pdl_release();
    const uint32_t tmem_base = *tmem_ptr_smem;
    bool ok = true;

    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    // scales in TMEM, of stage s: A's tiles, then B's, tile t of its row tile j at (t nt + j) * 4
    const uint32_t scale_cols = 4u * TILES * (1 + nt);
    auto scales_of = [&](int s) { return tmem_base + window + s * scale_cols; };

    if (warp == 0) {
        if (ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 1;                                   // empty_bar phase to wait for: the first round passes
            const uint8_t* as = sp.a_block_scales + (int64_t)m_blk * slabs * fp4_slab_scales(NV);
            for (int i = 0; i < slabs; ++i) {
                if (!ptx::mbar_wait(empty_bar(s), ph, abort_flag)) { ok = false; break; }
                if (i >= ahead) load_b(i, s);
                if constexpr (!FEW) {
                    const uint32_t dst = smem_base + s * sp.stage_bytes;
                    ptx::tma_load_2d(dst, &tmap_a, full_bar(s), i * 128, m_blk * kGemmBM);
                    ptx::bulk_load(dst + as_at, as, fp4_slab_scales(NV), full_bar(s));
                    as += fp4_slab_scales(NV);
                }
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
            if (!ok && p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (31 << 8));
        }
        __syncwarp();
    } else if (warp == 1) {
        if (ptx::elect_one()) {
            int s = 0;
            uint32_t ph = 0;
            const uint32_t shift = n0 % 128 >= 64 ? 2u : 0u;   // the window may begin in the middle of a tile of scales
            uint32_t idesc[2] = {ptx::make_idesc_fp4(kGemmBM, window, !NV, 0), ptx::make_idesc_fp4(kGemmBM, window, !NV, 2)};
            if (FEW && !ptx::mbar_wait(few_bar, 0, abort_flag)) ok = false;
            for (int i = 0; ok && i < slabs; ++i) {
                if (!ptx::mbar_wait(full_bar(s), ph, abort_flag) || !ptx::mbar_wait(scaled_bar(s), ph, abort_flag)) { ok = false; break; }
                ptx::tcgen05_fence_after_sync();
                const uint32_t src = smem_base + s * sp.stage_bytes;
                const uint32_t ta = scales_of(s), tb = ta + 4 * TILES + shift;
                const uint64_t a_desc = ptx::make_kmajor_desc(FEW ? ptx::smem_u32(few_values) + i * (kFp4Few * 128) : src, 128);
                const uint64_t b_desc = ptx::make_kmajor_desc(src + b_at, 128);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int t = NV ? k : k / 2;
                    ptx::mma_fp4<NV ? 4 : 2, false>(tmem_base, a_desc + 2 * k, b_desc + 2 * k, idesc[NV ? 0 : k & 1], ta + 4 * t, tb + 4 * t * nt,
                                                    (i > 0 || k > 0) ? 1u : 0u);
                }
                ptx::tcgen05_commit(empty_bar(s));
                if (++s == stages) { s = 0; ph ^= 1u; }
            }
            if (ok) ptx::tcgen05_commit(acc_bar);
            else if (p.status != nullptr) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (32 << 8));
        }
        __syncwarp();
    } else {
        // what the epilogue needs is on its way.  A launch that follows a failed one on the same status word stores nothing.
        const int prior_failure = p.status != nullptr ? *reinterpret_cast<volatile int*>(p.status) : 0;
        const int row = m_blk * kGemmBM + quarter * 32 + lane, column = threadIdx.x - 64;
        const bool row_ok = row < p.M, column_ok = column < bn && n0 + column < p.N;
        float sa = !row_ok ? 0.f : p.a_scales != nullptr ? p.a_scales[row] : 1.f;
        const float sb = !column_ok ? 0.f : p.b_scales != nullptr ? p.b_scales[n0 + column] : 1.f;
        const float bias = column_ok && p.bias != nullptr ? p.bias[n0 + column] : 0.f;
        // ------------------------------------------------ scales: warps 2-5 those in even stages, 6-9 those in odd ones; lane l of every lane
        // quarter holds the 16 bytes of rows l, l + 32, l + 64, l + 96 of a tile
        {
            const uint8_t* from = smem + as_at + lane * 16;    // A's tiles, then B's; FEW: B's
            if constexpr (FEW) {
                if (sp.x_f16) fp4_few_rows<NV>(static_cast<const __half*>(sp.x), p.M, p.K, slabs, few_values, few_scales, few_tops, few_row_scales);
                else fp4_few_rows<NV>(static_cast<const __nv_bfloat16*>(sp.x), p.M, p.K, slabs, few_values, few_scales, few_tops, few_row_scales);
                ptx::fence_proxy_async_smem();
                asm volatile("bar.sync 1, 256;" ::: "memory");
                if (threadIdx.x == 64) ptx::mbar_arrive(few_bar);
                if (NV && row_ok) sa = few_row_scales[row];
            }
            const uint32_t to = (uint32_t)(quarter * 32) << 16;
            int s = -1;
            uint32_t ph = 0;
            for (int i = 0; i < slabs; ++i) {
                if (++s == stages) { s = 0; ph ^= 1u; }
                if ((s & 1) != half) continue;                 // a stage's phases are all awaited by the same warps: parity tells two apart
                ok = ptx::mbar_wait(full_bar(s), ph, abort_flag);
                ok = __all_sync(0xffffffffu, ok);              // keep the warp convergent for tcgen05.st
                if (!ok) break;
                ptx::tcgen05_fence_after_sync();
                const uint8_t* src = from + s * sp.stage_bytes;
                const uint32_t at = scales_of(s) + to;
                uint4 w[3][TILES];
                if constexpr (FEW) {                           // row l is the first of lane l's four
#pragma unroll
                    for (int t = 0; t < TILES; ++t)
                        w[0][t] = make_uint4(lane < kFp4Few ? *reinterpret_cast<const uint32_t*>(few_scales + (i * TILES + t) * (4 * kFp4Few) + lane * 4) : 0, 0, 0, 0);
                }
#pragma unroll
                for (int j = FEW ? 1 : 0; j < 3; ++j)
#pragma unroll
                    for (int t = 0; t < TILES; ++t)
                        if (j <= nt) w[j][t] = *reinterpret_cast<const uint4*>(src + ((j - (FEW ? 1 : 0)) * TILES + t) * 512);
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    ptx::tmem_st_32x32b_x4(at + 4 * t, w[0][t]);
                    ptx::tmem_st_32x32b_x4(at + 4 * TILES + 4 * t * nt, w[1][t]);
                    if (nt == 2) ptx::tmem_st_32x32b_x4(at + 4 * TILES + 4 * (2 * t + 1), w[2][t]);
                }
                ptx::tmem_wait_st();
                ptx::tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) ptx::mbar_arrive(scaled_bar(s));
            }
        }
        // ------------------------------------------------ epilogue
        if (column < bn) {                                     // bn <= 192, 256 threads
            col_scale_smem[column] = sb;
            bias_smem[column] = bias;
        }
        asm volatile("bar.sync 1, 256;" ::: "memory");
        if (ok) ok = ptx::mbar_wait(acc_bar, 0, abort_flag);
        ok = __all_sync(0xffffffffu, ok);                      // keep the warp convergent for tcgen05.ld
        ptx::tcgen05_fence_after_sync();
        if (!ok && p.status != nullptr && threadIdx.x == 64) atomicExch(p.status, Q8K_STATUS_TIMEOUT | (33 << 8));
        if (ok && prior_failure == 0) {
            const uint32_t t_row = tmem_base + ((uint32_t)(quarter * 32) << 16);
            uint16_t* out = reinterpret_cast<uint16_t*>(p.out) + (int64_t)row * p.N + n0;
#pragma unroll 1
            for (int cl = half * 16; cl < bn; cl += 32) {
                uint32_t r[16];
                ptx::tmem_ld_32x32b_x16(t_row + off + cl, r);
                ptx::tmem_wait_ld();
                if (row_ok && n0 + cl < p.N) {                 // N % 16 == 0
#pragma unroll
                    for (int g = 0; g < 2; ++g) {
                        uint32_t w[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const int c = g * 8 + 2 * j;
                            w[j] = pack16<F16>(epilogue_pair<false, GELU>(r[c], r[c + 1], make_float2(sa, sa), col_scale_smem + cl + c,
                                                                          bias_smem + cl + c));
                        }
                        *reinterpret_cast<uint4*>(out + cl + g * 8) = make_uint4(w[0], w[1], w[2], w[3]);
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
        ptx::tmem_dealloc<512>(tmem_base);
    }
}

template <bool NV, bool GELU, bool F16, bool FEW>
static int launch_fp4_as(const CUtensorMap& ta, const CUtensorMap& tb, const Fp4TileParams& sp, unsigned grid, int smem, cudaStream_t st) {
    auto kern = gemm_fp4_kernel<NV, GELU, F16, FEW>;
    static std::atomic<uint64_t> smem_done{0};
    if (int rc = allow_dynamic_smem((const void*)kern, 226 * 1024, smem_done)) return rc;
    Q8K_CUDA_OK(launch_dependent(kern, grid, kGemmThreads, smem, st, 1, ta, tb, sp));
    return Q8K_OK;
}

// x: rows for the kernel to quantise, in the place of a; null: none.
static int launch_fp4_tiles(bool nv, bool gelu, bool f16, const Fp4Operand& a, const void* x, bool x_f16, const Fp4Operand& b, const Fp4GemmParams& p,
                            int bn, bool b_ahead, cudaStream_t st) {
    const char* op = "fp4_mm";
    Fp4TileParams sp;
    sp.g = p;
    sp.bn = bn;
    sp.b_ahead = b_ahead;
    sp.window = bn == 32 ? 64 : bn;
    sp.b_tiles = bn == 192 ? 2 : 1;
    const bool few = x != nullptr;
    const int a_rows = few ? 0 : split_a_rows(p.M);
    CUtensorMap ta, tb;
    if (int rc = make_values_map(&tb, b.values, p.N, p.K, bn, op)) return rc;
    ta = tb;                                                   // (not looked at with `few`)
    if (!few) {
        if (int rc = make_values_map(&ta, a.values, p.M, p.K, a_rows, op)) return rc;
    }
    sp.x = x;
    sp.x_f16 = x_f16;
    sp.a_block_scales = static_cast<const uint8_t*>(a.block_scales);
    sp.b_block_scales = static_cast<const uint8_t*>(b.block_scales);
    sp.a_bytes = a_rows * 128;
    sp.stage_bytes = (sp.a_bytes + sp.window * 128 + fp4_slab_scales(nv) * ((few ? 0 : 1) + sp.b_tiles) + 1023) / 1024 * 1024;
    const int64_t m_tiles = (p.M + kGemmBM - 1) / kGemmBM;
    sp.n_tiles = (p.N + bn - 1) / bn;
    Q8K_REQUIRE(m_tiles * sp.n_tiles <= 0x7fffffffLL, Q8K_ERR_TOO_LARGE, "%s: too many tiles", op);
    const int slabs = fp4_slabs(p.K), few_values = few ? slabs * kFp4Few * 128 : 0, few_scales = few ? slabs * fp4_slab_tiles(nv) * 4 * kFp4Few : 0;
    // the MMA takes 128 rows from the last slab of A that is there, wherever they end
    const int behind = few_scales + Fp4Smem::kTotal, last = few ? kFp4Few * 128 : sp.a_bytes;
    const int end = few_values + (behind > kFp4ABytes - last ? behind : kFp4ABytes - last) + 1024;
    // TMEM's 512 columns hold the accumulator and every stage's scales of A and of B
    int stages = (212 * 1024 - end) / sp.stage_bytes;
    const int by_tmem = (512 - sp.window) / (4 * fp4_slab_tiles(nv) * (1 + sp.b_tiles));
    if (stages > by_tmem) stages = by_tmem;
    if (stages > slabs) stages = slabs;
    if (stages > kFp4MaxStages) stages = kFp4MaxStages;
    sp.stages = stages;
    const int smem = stages * sp.stage_bytes + end;
    const unsigned grid = (unsigned)(m_tiles * sp.n_tiles);
#define Q8K_FP4(NV, FEW)                                                                                 \
    do {                                                                                                 \
        if (gelu) return f16 ? launch_fp4_as<NV, true, true, FEW>(ta, tb, sp, grid, smem, st)            \
                             : launch_fp4_as<NV, true, false, FEW>(ta, tb, sp, grid, smem, st);          \
        return f16 ? launch_fp4_as<NV, false, true, FEW>(ta, tb, sp, grid, smem, st)                     \
                   : launch_fp4_as<NV, false, false, FEW>(ta, tb, sp, grid, smem, st);                   \
    } while (0)
    if (few && nv) Q8K_FP4(true, true);
    if (few) Q8K_FP4(false, true);
    if (nv) Q8K_FP4(true, false);
    Q8K_FP4(false, false);
#undef Q8K_FP4
}

// Up to this many values of x, two units a thread, a product of few rows quantises them itself, in every CTA anew, which saves a launch.  Quantizer and
// product against the product alone in a CUDA graph, us, nvfp4 / mxfp4: 1 row of 2048 to N = 8192 6.9 / 6.0 against 5.9 / 5.1, of 8192 to 2048 11.4 / 10.5
// against 11.1 / 10.0; 4 rows of 2048 to 2048 5.7 / 5.4 against 5.7 / 4.8, 8 of them 5.7 / 5.4 against 7.1 / 5.6, 4 of 4096 to 4096 8.7 / 8.1 against
// 9.8 / 8.3.  The host takes 6.6 us for one launch and 9.8 for two and the workspace.
constexpr int kFp4FewValues = 8192;

// The narrowest tile whose grid fits the device once, one CTA an SM; 0 where none does, for the CTA pairs.  Measured, us, nvfp4 / mxfp4 on cold
// operands, a tile against the pairs: M, N, K = 16, 2048, 2048 with 32 columns 4.1 / 3.9 against 7.1 / 7.1; 16, 8192, 2048 with 64 5.3 / 4.8
// against 8.6 / 8.5; 300, 4096, 4096 with 128 9.3 / 8.6 against 10.4 / 10.3; 300, 2048, 8192 with 64 11.0 / 10.2 against 14.9 / 14.7.
// Two rounds of tiles cost twice: 300, 8192, 2048 with 128 12.2 / 10.6 against 8.5 / 8.4; 24576, 128, 2048 13.3 against 11.4.  192 columns are
// worth it for one row tile only, of which the pairs leave half empty (128, 20480, 4096: 15.0 / 14.6 against 18.1 / 17.7); with more rows the
// pairs' grid fits once where theirs does, and is faster (256, 10240, 4096: 13.9 / 13.1 against 11.4 / 11.3).
static int fp4_tile_columns(int M, int N) {
    const int64_t m_tiles = ((int64_t)M + kGemmBM - 1) / kGemmBM;
    for (int bn : {32, 64, 128, 192})
        if (m_tiles * ((N + bn - 1) / bn) <= gemm_num_sms() && (bn < 192 || m_tiles == 1)) return bn;
    return 0;
}

bool fp4_quantises_rows(int M, int N, int K) { return M <= kFp4Few && (int64_t)M * K <= kFp4FewValues && fp4_tile_columns(M, N) != 0; }

int fp4_mm(int format, const void* a, const void* a_block_scales, const float* a_row_scales, const void* b, const void* b_block_scales,
           const float* b_row_scales, const float* bias, void* out, int out_dtype, int M, int N, int K, int fuse_gelu, int* dev_status, bool b_ahead,
           const void* x, bool x_f16, cudaStream_t st) {
    const char* op = "fp4_mm";
    Q8K_REQUIRE(format == Q8K_FP4_MX || format == Q8K_FP4_NV, Q8K_ERR_UNSUPPORTED, "%s: format %d is unknown", op, format);
    const bool nv = format == Q8K_FP4_NV;
    Q8K_REQUIRE(M >= 0 && N > 0 && K > 0 && N % 16 == 0 && K % 32 == 0, Q8K_ERR_INVALID_ARG,
                "%s: M=%d must not be negative, N=%d a multiple of 16 and K=%d of 32", op, M, N, K);
    Q8K_REQUIRE(M <= 0x7fffff00 && N <= kFp4MaxN, Q8K_ERR_TOO_LARGE, "%s: M=%d or N=%d too large", op, M, N);
    Q8K_REQUIRE(out_dtype == Q8K_DT_BF16 || out_dtype == Q8K_DT_F16, Q8K_ERR_UNSUPPORTED, "%s: output dtype %d is not bf16 or fp16", op, out_dtype);
    if (M == 0) return Q8K_OK;
    Q8K_REQUIRE((x || (a && a_block_scales && (!nv || a_row_scales))) && b && b_block_scales && out && (!nv || b_row_scales), Q8K_ERR_INVALID_ARG,
                "%s: null pointer", op);
    Q8K_REQUIRE(aligned16(x) && aligned16(a) && aligned16(a_block_scales) && aligned16(b) && aligned16(b_block_scales) && aligned16(out), Q8K_ERR_INVALID_ARG,
                "%s: values, block scales and out must be 16-byte aligned", op);
    Fp4GemmParams p;
    p.a_scales = nv ? a_row_scales : nullptr;
    p.b_scales = nv ? b_row_scales : nullptr;
    p.bias = bias;
    p.out = out;
    p.status = dev_status;
    p.M = M; p.N = N; p.K = K;
    const Fp4Operand oa = {a, a_block_scales, a_row_scales}, ob = {b, b_block_scales, b_row_scales};
    int bn = fp4_tile_columns(M, N);
    if (bn == 0) {
        const int rc = launch_fp4_pair(nv, fuse_gelu != 0, out_dtype == Q8K_DT_F16, oa, ob, p, st);
        if (rc != Q8K_ERR_UNSUPPORTED) return rc;
        bn = 128;                                              // a device that holds few pairs at once
    }
    return launch_fp4_tiles(nv, fuse_gelu != 0, out_dtype == Q8K_DT_F16, oa, x, x_f16, ob, p, bn, b_ahead, st);
}

}  // namespace q8k

extern "C" int q8k_fp4_mm(int format, const void* a, const void* a_block_scales, const float* a_row_scales, const void* b, const void* b_block_scales,
                          const float* b_row_scales, const float* bias, void* out, int out_dtype, int M, int N, int K, int fuse_gelu,
                          int* dev_status, void* stream) {
    return q8k::fp4_mm(format, a, a_block_scales, a_row_scales, b, b_block_scales, b_row_scales, bias, out, out_dtype, M, N, K, fuse_gelu, dev_status, false,
                       nullptr, false, (cudaStream_t)stream);
}
