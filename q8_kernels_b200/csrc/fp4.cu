// Quantizer of microscaled 4-bit values (fp4.cuh has the formats) and what goes back from them.
//
//   mxfp4   exponent e = max(floor(log2(absmax of the block)) - 2, -127), values x 2^-e rounded to e2m1
//   nvfp4   r = A / 2688 (6 * 448) with A the row's absmax; a block of absmax a gets s = e4m3(a (448 / A)) and its values are rounded
//           from x (1 / (s r)); s = 0 leaves zeros.  All in fp32, each operation rounded.
// A factor that fp32 does not hold (rows whose absmax is below 1.3e-36, blocks below some 1e-37) is FLT_MAX, so that no zero becomes NaN.
// A block of mxfp4 with NaN or an infinity has NaN as its scale, a row of nvfp4 NaN or infinity as its row scale: the row's products are NaN.

#include <type_traits>
#include "fp4_quant.cuh"

namespace q8k {

// Few rows: a CTA for every row, UNITS units a thread.  The row's scales beyond K, up to its last slab, become 0.
template <typename Tin, bool NV, int UNITS>
__global__ void __launch_bounds__(1024)
fp4_quant_row_kernel(const Tin* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ q, uint8_t* __restrict__ block_scales,
                     float* __restrict__ row_scales, int K, int slabs) {
    __shared__ float red[32];
    const int64_t row = blockIdx.x;
    const int t = threadIdx.x, units = K / kFp4Unit;
    pdl_wait();
    pdl_release();
    uint4 r[UNITS][2];
    fp4_load<Tin, UNITS>(x + row * x_stride, t, blockDim.x, units, true, r);
    float a[UNITS];
    float top = 0.f, g = 0.f, rs = 0.f;
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        a[i] = Fp4In<Tin>::absmax(r[i]);
        top = max_nan(top, a[i]);
    }
    if constexpr (NV) {
        top = warp_max<true>(top);
        if (blockDim.x > 32) {
            if ((t & 31) == 0) red[t >> 5] = top;
            __syncthreads();
            top = warp_max<true>((t & 31) < blockDim.x / 32 ? red[t & 31] : 0.f);
        }
        fp4_row_factors(top, g, rs);
        if (t == 0) row_scales[row] = rs;
    }
#pragma unroll
    for (int i = 0; i < UNITS; ++i) {
        const int u = t + i * blockDim.x;
        float factor;
        const uint8_t scale = fp4_block_scale<NV>(a[i], g, rs, factor);
        if (u < units) *reinterpret_cast<uint2*>(q + row * (int64_t)(K / 2) + u * 8) = fp4_pack<Tin>(r[i], factor);
        if (u < slabs * (kFp4Slab / kFp4Unit)) {
            if constexpr (NV) block_scales[fp4_scale_at<true>(row, u, slabs)] = u < units ? scale : 0;
            else if ((u & 1) == 0) block_scales[fp4_scale_at<false>(row, u >> 1, slabs)] = u < units ? scale : 0;
        }
    }
}

// Many rows: a CTA takes the eight rows whose block scales lie side by side, r, r + 1 and those 32, 64 and 96 further on, and stores the scales as
// whole sectors of 32 bytes from shared memory.  (Byte by byte they were a fifth of all accesses to L2.)  T threads a row; where the rows
// are taken in steps, the next ones are on their way while one is quantised.  Scales of rows behind the last one, up to the row tile's end, become 0.
constexpr int kFp4GroupRows = 8;
template <typename Tin, bool NV, int UNITS, int T, int CTA>
__global__ void __launch_bounds__(CTA)
fp4_quant_kernel(const Tin* __restrict__ x, int64_t x_stride, uint8_t* __restrict__ q, uint8_t* __restrict__ block_scales,
                 float* __restrict__ row_scales, int64_t rows, int K, int slabs) {
    constexpr int AT_ONCE = CTA / T, STEPS = kFp4GroupRows / AT_ONCE;
    static_assert(AT_ONCE >= 1 && AT_ONCE <= kFp4GroupRows, "rows at a time");
    static_assert(!NV || T == 32, "a row of nvfp4, whose absmax all of its threads need, is one warp's");
    extern __shared__ __align__(16) uint8_t scales[];          // [tiles along K][32]
    const int group = threadIdx.x / T, t = threadIdx.x % T, units = K / kFp4Unit;
    const int64_t row0 = (int64_t)(blockIdx.x >> 4) * 128 + (blockIdx.x & 15) * 2;
    pdl_wait();
    pdl_release();
    auto row_of = [&](int step, int& local) {
        local = step * AT_ONCE + group;
        return row0 + (local & 1) + 32 * (local >> 1);
    };
    uint4 r[UNITS][2];
    int local;
    int64_t row = row_of(0, local);
    fp4_load<Tin, UNITS>(x + row * x_stride, t, T, units, row < rows, r);
#pragma unroll
    for (int step = 0; step < STEPS; ++step) {
        uint4 next[STEPS > 1 ? UNITS : 1][2];
        int local_next = 0;
        int64_t row_next = rows;
        if constexpr (STEPS > 1) {
            if (step + 1 < STEPS) {
                row_next = row_of(step + 1, local_next);
                fp4_load<Tin, UNITS>(x + row_next * x_stride, t, T, units, row_next < rows, next);
            }
        }
        const bool here = row < rows;
        float a[UNITS];
        float top = 0.f, g = 0.f, rs = 0.f;
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            a[i] = Fp4In<Tin>::absmax(r[i]);
            top = max_nan(top, a[i]);
        }
        if constexpr (NV) {
            top = warp_max<true>(top);
            fp4_row_factors(top, g, rs);
            if (here && t == 0) row_scales[row] = rs;
        }
#pragma unroll
        for (int i = 0; i < UNITS; ++i) {
            const int u = t + i * T;
            float factor;
            const uint8_t scale = fp4_block_scale<NV>(a[i], g, rs, factor);            // (0 for rows and units that are not there)
            if (here && u < units) *reinterpret_cast<uint2*>(q + row * (int64_t)(K / 2) + u * 8) = fp4_pack<Tin>(r[i], factor);
            const int b = NV ? u : u >> 1;
            if (u < slabs * (kFp4Slab / kFp4Unit) && (NV || (u & 1) == 0))
                scales[(b >> 2) * 32 + (local & 1) * 16 + (local >> 1) * 4 + (b & 3)] = scale;
        }
        if constexpr (STEPS > 1) {
#pragma unroll
            for (int i = 0; i < UNITS; ++i) { r[i][0] = next[i][0]; r[i][1] = next[i][1]; }
            row = row_next;
            local = local_next;
        }
    }
    __syncthreads();
    const int tiles = slabs * fp4_slab_tiles(NV);
    uint8_t* to = block_scales + (int64_t)(blockIdx.x >> 4) * tiles * 512 + (blockIdx.x & 15) * 32;
    for (int k = threadIdx.x; k < 2 * tiles; k += CTA)
        *reinterpret_cast<uint4*>(to + (int64_t)(k >> 1) * 512 + (k & 1) * 16) = *reinterpret_cast<const uint4*>(scales + k * 16);
}

// Which of the two, from times of CUDA graphs (us, groups of rows against a CTA a row): rows of 2048 values, 24576 of them nvfp4 21.0 against 26.1,
// mxfp4 19.8 against 26.0, 6144 of them 7.4 against 7.4 and 6.5 against 7.0, 2002 of them 4.2 against 4.2 and 3.6 against 3.2;  6144 rows of
// 4096 15.4 against 11.9 and 12.3 against 10.8, of 8192 25.2 against 22.1 and 24.2 against 19.8 (0.89 and 0.98 of the copy rate): a long
// row fills a CTA, and eight of them one after the other leave a long last round.
// Units of a thread, a CTA a row: one for few or short rows, where latency counts (2002 x 2048 mxfp4 3.2, two 3.7), else two (6144 x 8192 nvfp4 one
// 28.4, two 22.3, four 22.1), and four where 1024 threads need them.
constexpr int kFp4GroupK = 2048, kFp4GroupMinRows = 4096, kFp4FewRows = 1024;
template <typename Tin, bool NV>
static int launch_fp4_quant(const void* x, int64_t stride, void* q, void* bs, float* rs, int64_t rows, int K, cudaStream_t st) {
    const int slabs = fp4_slabs(K), units = slabs * (kFp4Slab / kFp4Unit);
    if (K > kFp4GroupK || rows < kFp4GroupMinRows) {
        auto go = [&](auto kern, int per) {
            const int threads = ((units + per - 1) / per + 31) / 32 * 32;
            Q8K_CUDA_OK(launch_dependent(kern, (unsigned)rows, (unsigned)threads, 0, st, 1, (const Tin*)x, stride, (uint8_t*)q, (uint8_t*)bs, rs, K, slabs));
            return (int)Q8K_OK;
        };
        if (units <= 1024 && (rows < kFp4FewRows || K <= kFp4GroupK)) return go(fp4_quant_row_kernel<Tin, NV, 1>, 1);
        return units <= 2048 ? go(fp4_quant_row_kernel<Tin, NV, 2>, 2) : go(fp4_quant_row_kernel<Tin, NV, 4>, 4);
    }
    auto go = [&](auto kern) {
        Q8K_CUDA_OK(launch_dependent(kern, (unsigned)(fp4_row_tiles(rows) * 16), 256, (size_t)slabs * fp4_slab_tiles(NV) * 32, st, 1, (const Tin*)x, stride,
                                     (uint8_t*)q, (uint8_t*)bs, rs, rows, K, slabs));
        return (int)Q8K_OK;
    };
    if (units <= 32) return go(fp4_quant_kernel<Tin, NV, 1, 32, 256>);
    if (units <= 64) return go(fp4_quant_kernel<Tin, NV, 2, 32, 256>);
    if constexpr (!NV) return go(fp4_quant_kernel<Tin, NV, 2, 64, 256>);       // (no sum over a row: two steps with the next rows on their way)
    return units <= 96 ? go(fp4_quant_kernel<Tin, NV, 3, 32, 256>) : go(fp4_quant_kernel<Tin, NV, 4, 32, 256>);
}

// What the values stand for: value * block scale (exact in fp32) * row scale, rounded, then to Tout.
template <typename Tout, bool NV>
__global__ void __launch_bounds__(256)
fp4_dequant_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ block_scales, const float* __restrict__ row_scales,
                   Tout* __restrict__ y, int64_t rows, int K, int slabs) {
    const int per_row = K / kFp4Unit;
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    pdl_wait();
    pdl_release();
    if (i >= rows * per_row) return;
    const int64_t row = i / per_row;
    const int u = (int)(i - row * per_row);
    const uint2 w = *reinterpret_cast<const uint2*>(q + row * (int64_t)(K / 2) + u * 8);
    const float s = fp4_scale_value<NV>(block_scales[fp4_scale_at<NV>(row, NV ? u : u >> 1, slabs)]);
    const float r = NV ? row_scales[row] : 1.f;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        float v[8];
        e2m1_to_float8(h == 0 ? w.x : w.y, v);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = __fmul_rn(__fmul_rn(v[k], s), r);
        store_vec<Tout, 8>(y + row * (int64_t)K + u * kFp4Unit + h * 8, v);
    }
}

template <typename Tout> static int launch_fp4_dequant(bool nv, const void* q, const void* bs, const float* rs, void* y, int64_t rows, int K,
                                                       cudaStream_t st) {
    const int64_t threads = rows * (K / kFp4Unit);
    auto kern = nv ? fp4_dequant_kernel<Tout, true> : fp4_dequant_kernel<Tout, false>;
    Q8K_CUDA_OK(launch_dependent(kern, (unsigned)((threads + 255) / 256), 256, 0, st, 1, (const uint8_t*)q, (const uint8_t*)bs, rs, (Tout*)y, rows, K,
                                 fp4_slabs(K)));
    return Q8K_OK;
}

// ------------------------------------------------------------------ weight operand of the backward product
// w [N, K] de-quantised (value * block scale, exact, times the row's scale, rounded to fp32), transposed and quantised to e4m3 with one scale
// per input channel, factor 448 / absmax as the 8-bit linears have it, FLT_MAX at most.  Two passes over the weight, which is small: the absmax of the
// columns over chunks of rows; then tiles of 128 x 128, whose CTAs take the maxima over the chunks, are turned in shared memory.
constexpr int kF4Cols = 128;                 // columns of a CTA: 8 groups of 16
constexpr int kF4Rows = 128;                 // rows of a turned tile
constexpr int kF4MaxParts = 32;
constexpr int kF4Threads = 256;

// 16 consecutive values of a row, before their scales
struct Fp4Raw { uint2 q; uint8_t s; float r; };
template <bool NV>
__device__ __forceinline__ Fp4Raw fp4_load16(const uint8_t* __restrict__ w, const uint8_t* __restrict__ bs, const float* __restrict__ rs, int row, int c,
                                             int K, int slabs) {
    return {*reinterpret_cast<const uint2*>(w + (int64_t)row * (K / 2) + c / 2), bs[fp4_scale_at<NV>(row, c / (NV ? 16 : 32), slabs)],
            NV ? rs[row] : 1.f};
}
// and as pairs with them.  A product of an e2m1 and an e4m3 value has six bits and at least 2^-10: fp16 holds it.
template <bool NV> __device__ __forceinline__ void fp4_values16(const Fp4Raw& x, float2 (&v)[8]) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        uint32_t p[4];
        asm("{\n\t"
            ".reg .b8 a, b, c, d;\n\t"
            "mov.b32 {a, b, c, d}, %4;\n\t"
            "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
            "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
            "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
            "cvt.rn.f16x2.e2m1x2 %3, d;\n\t"
            "}"
            : "=r"(p[0]), "=r"(p[1]), "=r"(p[2]), "=r"(p[3])
            : "r"(h == 0 ? x.q.x : x.q.y));
        __half2 s2;
        if constexpr (NV) {
            const __half s = __half(__nv_cvt_fp8_to_halfraw(x.s, __NV_E4M3));
            s2 = __half2(s, s);
        }
        const float scale = NV ? x.r : fp4_scale_value<false>(x.s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            __half2 q = *reinterpret_cast<const __half2*>(&p[i]);
            if constexpr (NV) q = __hmul2(q, s2);
            v[4 * h + i] = fmul2(__half22float2(q), make_float2(scale, scale));
        }
    }
}

// Bound by the latency of its loads: a thread has eight rows of 16 columns on their way at a time.
constexpr int kF4Ahead = 8;
template <bool NV>
__global__ void __launch_bounds__(kF4Threads, 4)
fp4_weight_absmax_kernel(const uint8_t* __restrict__ w, const uint8_t* __restrict__ bs, const float* __restrict__ rs, float* __restrict__ part, int N,
                         int K, int slabs, int rows) {
    __shared__ float red[kF4Threads / 32][kF4Cols];
    pdl_wait();
    pdl_release();
    const int cg = threadIdx.x & 7, rl = threadIdx.x >> 3;     // column group, row of a step of 32
    const int c0 = blockIdx.x * kF4Cols + cg * 16;
    const int r_end = min((int)(blockIdx.y + 1) * rows, N);
    float m[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) m[j] = 0.f;
    if (c0 < K) {
        for (int r0 = blockIdx.y * rows + rl; r0 < r_end; r0 += 32 * kF4Ahead) {
            Fp4Raw x[kF4Ahead];
#pragma unroll
            for (int i = 0; i < kF4Ahead; ++i)
                x[i] = r0 + 32 * i < r_end ? fp4_load16<NV>(w, bs, rs, r0 + 32 * i, c0, K, slabs) : Fp4Raw{make_uint2(0, 0), 0, 0.f};
#pragma unroll
            for (int i = 0; i < kF4Ahead; ++i) {
                float2 v[8];
                fp4_values16<NV>(x[i], v);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    m[2 * j] = fmaxf(m[2 * j], fabsf(v[j].x));
                    m[2 * j + 1] = fmaxf(m[2 * j + 1], fabsf(v[j].y));
                }
            }
        }
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {                             // over the four rows of a warp
        m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], 8));
        m[j] = fmaxf(m[j], __shfl_xor_sync(0xffffffffu, m[j], 16));
        if ((threadIdx.x & 31) < 8) red[threadIdx.x >> 5][cg * 16 + j] = m[j];
    }
    __syncthreads();
    const int c = blockIdx.x * kF4Cols + threadIdx.x;
    if (threadIdx.x < kF4Cols && c < K) {
        float a = red[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < kF4Threads / 32; ++k) a = fmaxf(a, red[k][threadIdx.x]);
        part[(int64_t)blockIdx.y * K + c] = a;
    }
}

// The kernel before this one on the stream read the weight and let it start only once it had waited for the weight's writer, so the weight
// may be loaded before the wait.
template <bool NV>
__global__ void __launch_bounds__(kF4Threads)
fp4_weight_turn_kernel(const uint8_t* __restrict__ w, const uint8_t* __restrict__ bs, const float* __restrict__ rs, const float* __restrict__ part,
                       int parts, uint8_t* __restrict__ q, float* __restrict__ scales, int N, int K, int slabs) {
    __shared__ float top[2][kF4Cols];
    __shared__ __align__(16) float mul[kF4Cols];
    __shared__ __align__(16) uint32_t turned[kF4Cols][kF4Rows / 4];
    const int cb = blockIdx.x * kF4Cols, r0 = blockIdx.y * kF4Rows;
    const int cg = threadIdx.x & 7, rg = threadIdx.x >> 3;     // 16 columns, four rows
    const int c0 = cb + cg * 16;
    const bool in = c0 < K && r0 + rg * 4 < N;                 // N % 16 == 0: all four rows exist, or none
    Fp4Raw x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = in ? fp4_load16<NV>(w, bs, rs, r0 + rg * 4 + i, c0, K, slabs) : Fp4Raw{make_uint2(0, 0), 0, 0.f};
    pdl_wait();
    pdl_release();
    {
        const int c = threadIdx.x & (kF4Cols - 1), half = threadIdx.x / kF4Cols;
        float a = 0.f;
        if (cb + c < K) {
#pragma unroll 8
            for (int k = half; k < parts; k += 2) a = fmaxf(a, part[(int64_t)k * K + cb + c]);
        }
        top[half][c] = a;
        __syncthreads();
        if (half == 0) {
            a = fmaxf(a, top[1][c]);
            // A column of zeros quantises to zeros, its scale is 0.  Below 448 / FLT_MAX the factor is FLT_MAX: an infinite one would make NaN
            // of the column's zeros.
            const float f = fp4_finite(__fdiv_rn(448.0f, a));
            // column group g's k-th four factors lie at (8 k + g) * 4: the eight groups of a warp read 128 bytes in a row
            mul[(c & 15) / 4 * 32 + c / 16 * 4 + (c & 3)] = a == 0.f ? 0.f : f;
            if (blockIdx.y == 0 && cb + c < K) scales[cb + c] = a == 0.f ? 0.f : __fdiv_rn(1.0f, f);
        }
    }
    __syncthreads();
    if (in) {
        float2 v[4][8];
#pragma unroll
        for (int i = 0; i < 4; ++i) fp4_values16<NV>(x[i], v[i]);
        // row group rg of a column goes to word rg + 4 * (column group): the words that a warp stores lie in 32 banks, and four of a
        // column stay together for the 16-byte reads below
        const int at = (rg + 4 * cg) & 31;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float4 f = *reinterpret_cast<const float4*>(mul + k * 32 + cg * 4);
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const float2 f2 = j == 0 ? make_float2(f.x, f.y) : make_float2(f.z, f.w);
                float2 y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = fmul2(v[i][2 * k + j], f2);
                const int c = cg * 16 + k * 4 + 2 * j;
                turned[c][at] = (uint32_t)float2_to_e4m3x2_sat(y[0].x, y[1].x) | ((uint32_t)float2_to_e4m3x2_sat(y[2].x, y[3].x) << 16);
                turned[c + 1][at] = (uint32_t)float2_to_e4m3x2_sat(y[0].y, y[1].y) | ((uint32_t)float2_to_e4m3x2_sat(y[2].y, y[3].y) << 16);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kF4Cols / 32; ++i) {
        const int c = i * 32 + (threadIdx.x >> 3), part16 = threadIdx.x & 7;
        const int n = r0 + part16 * 16;
        if (cb + c < K && n < N)
            *reinterpret_cast<uint4*>(q + (int64_t)(cb + c) * N + n) = *reinterpret_cast<const uint4*>(&turned[c][(part16 * 4 + 4 * (c / 16)) & 31]);
    }
}

template <bool NV>
static int launch_fp4_weight(const void* w, const void* bs, const float* rs, void* q, float* scales, float* part, int N, int K, cudaStream_t st) {
    const unsigned cols = (unsigned)((K + kF4Cols - 1) / kF4Cols);
    const int slabs = fp4_slabs(K);
    // four CTAs an SM, all of one size: rows a CTA by that, in steps of 32
    int parts = (int)((unsigned)(4 * gemm_num_sms()) / cols);
    parts = parts < 1 ? 1 : parts > kF4MaxParts ? kF4MaxParts : parts;
    const int rows = ((N + parts - 1) / parts + 31) / 32 * 32;
    parts = (N + rows - 1) / rows;
    Q8K_CUDA_OK(launch_dependent(fp4_weight_absmax_kernel<NV>, dim3(cols, (unsigned)parts), kF4Threads, 0, st, 1, (const uint8_t*)w, (const uint8_t*)bs, rs,
                                 part, N, K, slabs, rows));
    Q8K_CUDA_OK(launch_dependent(fp4_weight_turn_kernel<NV>, dim3(cols, (unsigned)((N + kF4Rows - 1) / kF4Rows)), kF4Threads, 0, st, 1,
                                 (const uint8_t*)w, (const uint8_t*)bs, rs, part, parts, (uint8_t*)q, scales, N, K, slabs));
    return Q8K_OK;
}

static int fp4_check(const char* op, int format, int64_t rows, int K) {
    Q8K_REQUIRE(format == Q8K_FP4_MX || format == Q8K_FP4_NV, Q8K_ERR_UNSUPPORTED, "%s: format %d is unknown", op, format);
    Q8K_REQUIRE(rows >= 0 && K > 0 && K % 32 == 0, Q8K_ERR_INVALID_ARG, "%s: rows %lld must not be negative and K=%d a positive multiple of 32", op,
                (long long)rows, K);
    Q8K_REQUIRE(K <= 65536, Q8K_ERR_UNSUPPORTED, "%s: K=%d exceeds 65536", op, K);
    Q8K_REQUIRE(rows <= 0x7fffff00LL && rows * (K / 16) <= 0x7fffffffLL * 128, Q8K_ERR_TOO_LARGE, "%s: %lld rows of %d", op, (long long)rows, K);
    return Q8K_OK;
}

}  // namespace q8k

extern "C" size_t q8k_fp4_scale_bytes(int format, int64_t rows, int K) {
    if (rows <= 0 || K <= 0 || (format != Q8K_FP4_MX && format != Q8K_FP4_NV)) return 0;
    return (size_t)q8k::fp4_scale_bytes(format == Q8K_FP4_NV, rows, K);
}

extern "C" int q8k_fp4_quant(const void* x, int x_dtype, int64_t x_row_stride, int format, void* values, void* block_scales, float* row_scales,
                             int64_t rows, int K, void* stream) {
    using namespace q8k;
    const char* op = "fp4_quant";
    if (int rc = fp4_check(op, format, rows, K)) return rc;
    const bool nv = format == Q8K_FP4_NV;
    Q8K_REQUIRE(x_dtype == Q8K_DT_BF16 || x_dtype == Q8K_DT_F16, Q8K_ERR_UNSUPPORTED, "%s: input dtype %d is not bf16 or fp16", op, x_dtype);
    if (rows == 0) return Q8K_OK;
    Q8K_REQUIRE(x && values && block_scales && (row_scales || !nv) && aligned16(x) && aligned16(values) && aligned16(block_scales),
                Q8K_ERR_INVALID_ARG, "%s: null or misaligned pointer", op);
    Q8K_REQUIRE(rows == 1 || (x_row_stride >= K && x_row_stride % 8 == 0), Q8K_ERR_INVALID_ARG,
                "%s: row stride %lld must be at least K and a multiple of 16 bytes", op, (long long)x_row_stride);
    cudaStream_t st = (cudaStream_t)stream;
    if (x_dtype == Q8K_DT_BF16)
        return nv ? launch_fp4_quant<__nv_bfloat16, true>(x, x_row_stride, values, block_scales, row_scales, rows, K, st)
                  : launch_fp4_quant<__nv_bfloat16, false>(x, x_row_stride, values, block_scales, row_scales, rows, K, st);
    return nv ? launch_fp4_quant<__half, true>(x, x_row_stride, values, block_scales, row_scales, rows, K, st)
              : launch_fp4_quant<__half, false>(x, x_row_stride, values, block_scales, row_scales, rows, K, st);
}

extern "C" int q8k_fp4_dequant(const void* values, const void* block_scales, const float* row_scales, int format, void* y, int y_dtype, int64_t rows,
                               int K, void* stream) {
    using namespace q8k;
    const char* op = "fp4_dequant";
    if (int rc = fp4_check(op, format, rows, K)) return rc;
    const bool nv = format == Q8K_FP4_NV;
    Q8K_REQUIRE(y_dtype == Q8K_DT_BF16 || y_dtype == Q8K_DT_F16 || y_dtype == Q8K_DT_F32, Q8K_ERR_UNSUPPORTED,
                "%s: output dtype %d is not bf16, fp16 or fp32", op, y_dtype);
    if (rows == 0) return Q8K_OK;
    Q8K_REQUIRE(y && values && block_scales && (row_scales || !nv) && aligned16(y) && aligned16(values), Q8K_ERR_INVALID_ARG,
                "%s: null or misaligned pointer", op);
    cudaStream_t st = (cudaStream_t)stream;
    if (y_dtype == Q8K_DT_BF16) return launch_fp4_dequant<__nv_bfloat16>(nv, values, block_scales, row_scales, y, rows, K, st);
    if (y_dtype == Q8K_DT_F16) return launch_fp4_dequant<__half>(nv, values, block_scales, row_scales, y, rows, K, st);
    return launch_fp4_dequant<float>(nv, values, block_scales, row_scales, y, rows, K, st);
}

extern "C" size_t q8k_fp4_weight_operand_workspace_bytes(int N, int K) {
    return N <= 0 || K <= 0 ? 0 : (size_t)q8k::kF4MaxParts * (size_t)K * sizeof(float);         // partial maxima
}

extern "C" int q8k_fp4_weight_operand(int format, const void* values, const void* block_scales, const float* row_scales, void* q, float* scales, int N,
                                      int K, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace q8k;
    const char* op = "fp4_weight_operand";
    if (int rc = fp4_check(op, format, N, K)) return rc;
    const bool nv = format == Q8K_FP4_NV;
    Q8K_REQUIRE(N > 0 && N % 16 == 0, Q8K_ERR_INVALID_ARG, "%s: N=%d must be a positive multiple of 16", op, N);
    Q8K_REQUIRE(N <= 65535 * kF4Rows, Q8K_ERR_TOO_LARGE, "%s: N=%d too large", op, N);
    Q8K_REQUIRE(values && block_scales && (row_scales || !nv) && q && scales && workspace && aligned16(values) && aligned16(q) && aligned16(workspace),
                Q8K_ERR_INVALID_ARG, "%s: null or misaligned pointer", op);
    const size_t need = q8k_fp4_weight_operand_workspace_bytes(N, K);
    Q8K_REQUIRE(workspace_bytes >= need, Q8K_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    cudaStream_t st = (cudaStream_t)stream;
    return nv ? launch_fp4_weight<true>(values, block_scales, row_scales, q, scales, (float*)workspace, N, K, st)
              : launch_fp4_weight<false>(values, block_scales, row_scales, q, scales, (float*)workspace, N, K, st);
}

extern "C" int q8k_fp4_backward_quant(const void* grad, int dtype, void* q, float* scales, int64_t rows, int N, void* stream) {
    using namespace q8k;
    const char* op = "fp4_backward_quant";
    Q8K_REQUIRE(dtype == Q8K_DT_BF16 || dtype == Q8K_DT_F16, Q8K_ERR_UNSUPPORTED, "%s: gradient dtype %d is not bf16 or fp16", op, dtype);
    return tokenwise_quant_as<kRowsFinite>(op, grad, dtype, q, Q8K_DT_E4M3, scales, rows, N, N, (cudaStream_t)stream);
}

// Where the parts of the quantised activation lie in the workspace of q8k_fp4_linear.
static void fp4_linear_parts(bool nv, int M, int K, size_t& scales_at, size_t& rows_at, size_t& bytes) {
    scales_at = ((size_t)M * (size_t)(K / 2) + 255) / 256 * 256;
    rows_at = scales_at + (size_t)q8k::fp4_scale_bytes(nv, M, K);          // (a multiple of 512)
    bytes = rows_at + (nv ? (size_t)M * sizeof(float) : 0);
}

extern "C" size_t q8k_fp4_linear_workspace_bytes(int format, int M, int N, int K) {
    if (M <= 0 || N <= 0 || K <= 0 || (format != Q8K_FP4_MX && format != Q8K_FP4_NV)) return 0;
    if (q8k::fp4_quantises_rows(M, N, K)) return 0;
    size_t scales_at, rows_at, bytes;
    fp4_linear_parts(format == Q8K_FP4_NV, M, K, scales_at, rows_at, bytes);
    return bytes;
}

extern "C" int q8k_fp4_linear(int format, const void* x, int x_dtype, const void* w, const void* w_block_scales, const float* w_row_scales,
                              const float* bias, void* out, int out_dtype, int M, int N, int K, int fuse_gelu, void* workspace,
                              size_t workspace_bytes, int* dev_status, void* stream) {
    using namespace q8k;
    const char* op = "fp4_linear";
    if (int rc = fp4_check(op, format, M, K)) return rc;
    const bool nv = format == Q8K_FP4_NV;
    Q8K_REQUIRE(N > 0 && N % 16 == 0, Q8K_ERR_INVALID_ARG, "%s: N=%d must be a positive multiple of 16", op, N);
    Q8K_REQUIRE(N <= kFp4MaxN, Q8K_ERR_TOO_LARGE, "%s: N=%d too large", op, N);
    if (M == 0) return Q8K_OK;
    if (fp4_quantises_rows(M, N, K)) {
        Q8K_REQUIRE(x_dtype == Q8K_DT_BF16 || x_dtype == Q8K_DT_F16, Q8K_ERR_UNSUPPORTED, "%s: input dtype %d is not bf16 or fp16", op, x_dtype);
        Q8K_REQUIRE(x != nullptr, Q8K_ERR_INVALID_ARG, "%s: null pointer", op);
        return fp4_mm(format, nullptr, nullptr, nullptr, w, w_block_scales, w_row_scales, bias, out, out_dtype, M, N, K, fuse_gelu, dev_status, false, x,
                      x_dtype == Q8K_DT_F16, (cudaStream_t)stream);
    }
    Q8K_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0, Q8K_ERR_INVALID_ARG,
                "%s: the workspace must be 256-byte aligned", op);
    size_t scales_at, rows_at, need;
    fp4_linear_parts(nv, M, K, scales_at, rows_at, need);
    Q8K_REQUIRE(workspace_bytes >= need, Q8K_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    uint8_t* values = static_cast<uint8_t*>(workspace);
    uint8_t* blocks = values + scales_at;
    float* rows = nv ? reinterpret_cast<float*>(values + rows_at) : nullptr;
    if (int rc = q8k_fp4_quant(x, x_dtype, K, format, values, blocks, rows, M, K, stream)) return rc;
    return fp4_mm(format, values, blocks, rows, w, w_block_scales, w_row_scales, bias, out, out_dtype, M, N, K, fuse_gelu, dev_status, true,
                  nullptr, false, (cudaStream_t)stream);
}
