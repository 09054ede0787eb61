// The gated projection around its GEMMs (gemm_gated.cu): the activation's quantizer, and the two operands of the backward product.
//
// Backward pass up to the product with the weight: out = act(gate) * up has the gradients
//   dgate = dout * up * act'(gate),  dup = dout * act(gate)
// which the FP8 GEMM takes as one row [dgate | dup] of 2F e4m3 values with one scale.  Bound by HBM: 2 bytes of dout and 4 of gate
// and up are read per column, 2 bytes written; the 2F fp32 values of a row stay in registers between the absmax and the cast, so
// nothing is rounded before it.  CTAs walk over rows and have the next ones on their way to shared memory by cp.async, each thread
// the pieces that it reads itself: 6144 x 8192 66 us, 0.93 of the copy rate (85 with a CTA for every row).

#include <math.h>

#include <type_traits>
#include "common.cuh"

namespace q8k {

constexpr int kGatedItem = 8;
constexpr int kGatedMaxF = 16384;

// act(g) and its derivative of two adjacent columns, both from s = 1 / (1 + e^(-v)):  silu: v = g, act' = s + g s (1 - s);  tanh-GELU:
// v = 2 sqrt(2/pi) (g + c g^3), act' = s + g s (1 - s) v'.  Their errors are those of gated_act in gemm_gated.cu.  Where s (1 - s) is 0 the
// second term is, too, also where g^2 has overflowed.
// Packed pairs: element by element the kernel issued 26 instructions a column, half of its slots.
template <bool GELU> __device__ __forceinline__ void gated_act_grad(float2 g, float2& act, float2& grad) {
    constexpr float kLog2e = 1.4426950408889634f, kA = 2.0f * 0.7978845608028654f, kB = kA * 0.044715f;
    auto pair = [](float v) { return make_float2(v, v); };
    float2 gg, t;                                              // -v log2 e
    if constexpr (GELU) {
        gg = fmul2(g, g);
        t = fmul2(g, ffma2(gg, pair(-kLog2e * kB), pair(-kLog2e * kA)));
    } else {
        t = fmul2(g, pair(-kLog2e));
    }
    float2 e, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.x) : "f"(t.x));
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e.y) : "f"(t.y));
    e = fadd2(e, pair(1.0f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(e.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(e.y));
    act = fmul2(g, s);
    const float2 rest = fsub2(pair(1.0f), s);
    float2 slope = fmul2(act, rest);                           // g s (1 - s)
    if constexpr (GELU) {
        const float2 dv = ffma2(gg, pair(3.0f * kB), pair(kA));
        slope = fmul2(slope, dv);
        slope.x = s.x == 0.f || rest.x == 0.f ? 0.f : slope.x;
        slope.y = s.y == 0.f || rest.y == 0.f ? 0.f : slope.y;
    }
    grad = fadd2(s, slope);
}

__device__ __forceinline__ float2 bf16_pair(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }

__device__ __forceinline__ void gated_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}

// T threads of ITEMS groups of 8 columns, CTAS of them an SM, S rows in the ring (6 bytes a column each).
template <int I, int TT, int C, int SS> struct GatedBackLayout { static constexpr int items = I, threads = TT, ctas = C, slots = SS; };

template <bool GELU, typename L>
__global__ void __launch_bounds__(L::threads, L::ctas)
gated_backward_quant_kernel(const __nv_bfloat16* __restrict__ dout, const __nv_bfloat16* __restrict__ pre, uint8_t* __restrict__ q,
                            float* __restrict__ scales, int M, int F) {
    constexpr int ITEMS = L::items, T = L::threads, S = L::slots;
    extern __shared__ __align__(16) uint8_t gated_smem[];      // [S][dout | gate | up]
    __shared__ float red[2][T / 32];
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(gated_smem);
    const int slot_bytes = 6 * F;
    auto fetch = [&](int row, int slot) {
        if (row < M) {
            const __nv_bfloat16* dr = dout + (int64_t)row * F;
            const __nv_bfloat16* pr = pre + (int64_t)row * 2 * F;
            const uint32_t dst = ring + slot * slot_bytes;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int e = (threadIdx.x + i * T) * kGatedItem;
                if (e < F) {
                    gated_copy16(dst + 2 * e, dr + e);
                    gated_copy16(dst + 2 * F + 2 * e, pr + e);
                    gated_copy16(dst + 4 * F + 2 * e, pr + F + e);
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    pdl_wait();
    pdl_release();
#pragma unroll
    for (int k = 0; k < S - 1; ++k) fetch(blockIdx.x + k * gridDim.x, k);
    int slot = 0, turn = 0;
    for (int row = blockIdx.x; row < M; row += gridDim.x, turn ^= 1) {
        asm volatile("cp.async.wait_group %0;" ::"n"(S - 2) : "memory");
        const uint8_t* in = gated_smem + slot * slot_bytes;
        float2 dg[ITEMS][kGatedItem / 2], du[ITEMS][kGatedItem / 2];
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int e = (threadIdx.x + i * T) * kGatedItem;
            if (e < F) {
                const uint4 d4 = *reinterpret_cast<const uint4*>(in + 2 * e);
                const uint4 g4 = *reinterpret_cast<const uint4*>(in + 2 * F + 2 * e);
                const uint4 u4 = *reinterpret_cast<const uint4*>(in + 4 * F + 2 * e);
                const uint32_t dw[4] = {d4.x, d4.y, d4.z, d4.w}, gw[4] = {g4.x, g4.y, g4.z, g4.w}, uw[4] = {u4.x, u4.y, u4.z, u4.w};
#pragma unroll
                for (int k = 0; k < kGatedItem / 2; ++k) {
                    const float2 d = bf16_pair(dw[k]);
                    float2 act, grad;
                    gated_act_grad<GELU>(bf16_pair(gw[k]), act, grad);
                    dg[i][k] = fmul2(fmul2(d, bf16_pair(uw[k])), grad);
                    du[i][k] = fmul2(d, act);
                    asm("max.f32 %0, %0, %1, %2;" : "+f"(amax) : "f"(fabsf(dg[i][k].x)), "f"(fabsf(dg[i][k].y)));
                    asm("max.f32 %0, %0, %1, %2;" : "+f"(amax) : "f"(fabsf(du[i][k].x)), "f"(fabsf(du[i][k].y)));
                }
            }
        }
        fetch(row + (S - 1) * gridDim.x, slot == 0 ? S - 1 : slot - 1);       // into the slot that this thread read a row ago
        if (++slot == S) slot = 0;
        amax = warp_max(amax);
        if ((threadIdx.x & 31) == 0) red[turn][threadIdx.x >> 5] = amax;
        __syncthreads();                                       // (two arrays: the one before is not written until the next barrier)
        amax = red[turn][0];
#pragma unroll
        for (int w = 1; w < T / 32; ++w) amax = fmaxf(amax, red[turn][w]);
        const float scale = quant_factor<true>(448.0f, amax);  // the saturating cast below: see tokenwise_quant_kernel
        const float mul = amax == 0.f ? 0.f : scale;
        const float2 mul2 = make_float2(mul, mul);
        uint8_t* qr = q + (int64_t)row * 2 * F;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int e = (threadIdx.x + i * T) * kGatedItem;
            if (e < F) {
                union { uint2 v; uint16_t h[4]; } a, b;
#pragma unroll
                for (int k = 0; k < kGatedItem / 2; ++k) {
                    const float2 x = fmul2(dg[i][k], mul2), y = fmul2(du[i][k], mul2);
                    a.h[k] = float2_to_e4m3x2_sat(x.x, x.y);
                    b.h[k] = float2_to_e4m3x2_sat(y.x, y.y);
                }
                *reinterpret_cast<uint2*>(qr + e) = a.v;
                *reinterpret_cast<uint2*>(qr + F + e) = b.v;
            }
        }
        if (threadIdx.x == 0) scales[row] = __fdiv_rn(1.0f, scale);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");       // (the copies behind the last row were empty)
}

template <bool GELU, typename L>
static int launch_gated_backward_as(const void* dout, const void* pre, void* q, float* scales, int M, int F, cudaStream_t st) {
    auto kern = gated_backward_quant_kernel<GELU, L>;
    constexpr int most = L::slots * 6 * L::items * L::threads * kGatedItem;
    static_assert(most * L::ctas <= 224 * 1024, "gated backward ring");
    if (most > 40 * 1024) {
        static std::atomic<uint64_t> smem_done{0};
        if (int rc = allow_dynamic_smem((const void*)kern, most, smem_done)) return rc;
    }
    const int ctas = gemm_num_sms() * L::ctas;
    Q8K_CUDA_OK(launch_dependent(kern, (unsigned)(M < ctas ? M : ctas), L::threads, L::slots * 6 * F, st, 1, (const __nv_bfloat16*)dout,
                                 (const __nv_bfloat16*)pre, (uint8_t*)q, scales, M, F));
    return Q8K_OK;
}

// Both sides of each limit: the layout that is taken at the widest rows it holds | the next one for the same rows.  us of 24 million gates,
// silu and GELU, by F:
//   512  39.3|40.1 41.0|46.4    1024  36.5|35.9 37.8|40.6    2048  35.0|31.3 34.4|35.4    4096  34.4|36.0 33.5|38.0    8192  31.6|36.1 33.0|39.1
template <bool GELU>
static int launch_gated_backward(const void* dout, const void* pre, void* q, float* scales, int M, int F, cudaStream_t st) {
    const int items = F / kGatedItem;
#define Q8K_GB(...) return launch_gated_backward_as<GELU, GatedBackLayout<__VA_ARGS__>>(dout, pre, q, scales, M, F, st)
    if (items <= 64) Q8K_GB(1, 64, 16, 4);
    if (items <= 128) Q8K_GB(1, 128, 8, 4);
    if (items <= 256) Q8K_GB(1, 256, 4, 4);
    if (items <= 512) Q8K_GB(2, 256, 3, 3);
    if (items <= 1024) Q8K_GB(4, 256, 2, 2);
    Q8K_GB(4, 512, 1, 2);
#undef Q8K_GB
}

// The weight operand of the backward product: w [N, K] (int8 or e4m3) times its row scales, transposed and quantised to e4m3 with one
// scale per row of the result, i.e. per column of w.  w is read once and q written once; a column's absmax needs all rows first, so
// there are two passes, the second of which finds w in L2, with a small kernel between them that makes the columns' factors of the
// partial maxima (taken by each CTA of the second pass for itself, 64 dependent loads, they were most of its time: 16384 x 2048
// int8 40.9 us).  Now 22.5 us, where w once in and q once out are 10: bound by instruction issue, every element being widened and scaled twice
// (53 and 58 % of the slots), and by three launches in a row.
//
// Tiles of 128 columns, 16 per thread (one 16-byte load of a row), so a warp reads four rows of 128 bytes.
constexpr int kWtCols = 128;
constexpr int kWtMaxRows = 512;              // rows whose absmax one CTA takes, at most (multiples of 64)
constexpr int kWtRows = 128;                 // rows of a tile that is quantised and turned
constexpr int kWtThreads = 256;

// Four elements times their row's scale, as packed pairs of columns.
template <typename Tw> __device__ __forceinline__ void wt_values(uint32_t w, float s, float2 (&v)[2]) {
    if constexpr (std::is_same_v<Tw, int8_t>) {
        // 2^23 + 128 + b has the byte b + 128 in its last bits: a permutation and an exact difference instead of a conversion,
        // which runs at an eighth of their rate
        const uint32_t u = w ^ 0x80808080u;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const float2 f = make_float2(__uint_as_float(__byte_perm(u, 0x4B000000u, 0x7650 | (2 * j))),
                                         __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7650 | (2 * j + 1))));
            v[j] = fmul2(fsub2(f, make_float2(8388736.0f, 8388736.0f)), make_float2(s, s));
        }
    } else {
        float f[4];
        e4m3x4_to_float(w, f);
#pragma unroll
        for (int j = 0; j < 2; ++j) v[j] = fmul2(make_float2(f[2 * j], f[2 * j + 1]), make_float2(s, s));
    }
}

template <typename Tw>
__global__ void __launch_bounds__(kWtThreads)
gated_weight_absmax_kernel(const Tw* __restrict__ w, const float* __restrict__ row_scales, float* __restrict__ part, int N, int K,
                           int rows) {
    __shared__ float red[kWtThreads / 32][kWtCols];
    pdl_wait();
    pdl_release();
    const int cg = threadIdx.x & 7, rl = threadIdx.x >> 3;     // column group, row within a step of 32
    const int c0 = blockIdx.x * kWtCols + cg * 16;
    const int r0 = blockIdx.y * rows, r_end = min(r0 + rows, N);
    float m[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) m[j] = 0.f;
    if (c0 < K) {
        // two rows at a time into one maximum of three operands; rows beyond N (a multiple of 16, so not pairs of them) have scale 0
#pragma unroll 4
        for (int i = 0; i < kWtMaxRows / 64; ++i) {
            const int r = r0 + i * 64 + rl * 2;
            const bool in = r < r_end;
            uint32_t xw[2][4];
            float s[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint4 x = in ? *reinterpret_cast<const uint4*>(w + (int64_t)(r + h) * K + c0) : make_uint4(0, 0, 0, 0);
                s[h] = in ? row_scales[r + h] : 0.f;
                xw[h][0] = x.x; xw[h][1] = x.y; xw[h][2] = x.z; xw[h][3] = x.w;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                float2 u[2], v[2];
                wt_values<Tw>(xw[0][k], s[0], u);
                wt_values<Tw>(xw[1][k], s[1], v);
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    asm("max.f32 %0, %0, %1, %2;" : "+f"(m[k * 4 + 2 * j]) : "f"(fabsf(u[j].x)), "f"(fabsf(v[j].x)));
                    asm("max.f32 %0, %0, %1, %2;" : "+f"(m[k * 4 + 2 * j + 1]) : "f"(fabsf(u[j].y)), "f"(fabsf(v[j].y)));
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
    const int c = blockIdx.x * kWtCols + threadIdx.x;
    if (threadIdx.x < kWtCols && c < K) {
        float a = red[0][threadIdx.x];
#pragma unroll
        for (int k = 1; k < kWtThreads / 32; ++k) a = fmaxf(a, red[k][threadIdx.x]);
        part[(int64_t)blockIdx.y * K + c] = a;
    }
}

// factors[c] = 448 * (1 / absmax of column c) (0 for a column of zeros), scales[c] = 1 / that: 32 columns a CTA.
constexpr int kWtFactorWarps = 8;
__global__ void __launch_bounds__(32 * kWtFactorWarps)
gated_weight_factor_kernel(const float* __restrict__ part, int parts, float* __restrict__ factors, float* __restrict__ scales, int K) {
    __shared__ float red[kWtFactorWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;
    pdl_wait();
    pdl_release();
    float a = 0.f;
    if (c < K) {
#pragma unroll 8
        for (int k = warp; k < parts; k += kWtFactorWarps) a = fmaxf(a, part[(int64_t)k * K + c]);
    }
    red[warp][lane] = a;
    __syncthreads();
    if (warp == 0 && c < K) {
#pragma unroll
        for (int k = 1; k < kWtFactorWarps; ++k) a = fmaxf(a, red[k][lane]);
        const float f = quant_factor<true>(448.0f, a);
        factors[c] = a == 0.f ? 0.f : f;                       // a column of zeros quantises to zeros
        scales[c] = __fdiv_rn(1.0f, f);
    }
}

// The kernels before this one on the stream read w and let it start only once they had waited for its writer, so w may be loaded
// before the wait.
template <typename Tw>
__global__ void __launch_bounds__(kWtThreads)
gated_weight_quant_kernel(const Tw* __restrict__ w, const float* __restrict__ row_scales, const float* __restrict__ factors,
                          uint8_t* __restrict__ q, int N, int K) {
    __shared__ __align__(16) float mul[kWtCols];
    __shared__ __align__(16) uint32_t turned[kWtCols][kWtRows / 4];
    const int cb = blockIdx.x * kWtCols, r0 = blockIdx.y * kWtRows;
    const int cg = threadIdx.x & 7, rg = threadIdx.x >> 3;     // 16 columns, four rows
    uint4 x[4];
    float s[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {                              // N % 16 == 0: all four rows exist, or none
        const bool in = cb + cg * 16 < K && r0 + rg * 4 < N;
        x[i] = in ? *reinterpret_cast<const uint4*>(w + (int64_t)(r0 + rg * 4 + i) * K + cb + cg * 16) : make_uint4(0, 0, 0, 0);
        s[i] = in ? row_scales[r0 + rg * 4 + i] : 0.f;
    }
    pdl_wait();
    pdl_release();
    // column group g's k-th four factors lie at (8 k + g) * 4: the eight groups of a warp read 128 bytes in a row
    if (threadIdx.x < kWtCols && cb + (int)threadIdx.x < K)
        mul[(threadIdx.x & 15) / 4 * 32 + threadIdx.x / 16 * 4 + (threadIdx.x & 3)] = factors[cb + threadIdx.x];
    __syncthreads();
    if (cb + cg * 16 < K) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float2 v[4][2];                                    // [row][pair of columns]
            const int c = cg * 16 + k * 4;
            const float4 f = *reinterpret_cast<const float4*>(mul + k * 32 + cg * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                wt_values<Tw>(k == 0 ? x[i].x : k == 1 ? x[i].y : k == 2 ? x[i].z : x[i].w, s[i], v[i]);
                v[i][0] = fmul2(v[i][0], make_float2(f.x, f.y));
                v[i][1] = fmul2(v[i][1], make_float2(f.z, f.w));
            }
            // saturating cast: see tokenwise_quant_kernel.  Row group rg of a column goes to word rg + 4 * (column group): the 32
            // words that a warp stores lie in 32 banks, and four of a column stay together for the 16-byte reads below.
            const int at = (rg + 4 * cg) & 31;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                turned[c + 2 * j][at] = (uint32_t)float2_to_e4m3x2_sat(v[0][j].x, v[1][j].x) | ((uint32_t)float2_to_e4m3x2_sat(v[2][j].x, v[3][j].x) << 16);
                turned[c + 2 * j + 1][at] = (uint32_t)float2_to_e4m3x2_sat(v[0][j].y, v[1][j].y) | ((uint32_t)float2_to_e4m3x2_sat(v[2][j].y, v[3][j].y) << 16);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWtCols / 32; ++i) {
        const int c = i * 32 + (threadIdx.x >> 3), part16 = threadIdx.x & 7;
        const int n = r0 + part16 * 16;
        if (cb + c < K && n < N)
            *reinterpret_cast<uint4*>(q + (int64_t)(cb + c) * N + n) =
                *reinterpret_cast<const uint4*>(&turned[c][(part16 * 4 + 4 * (c / 16)) & 31]);
    }
}

template <typename Tw>
static int launch_gated_weight(const void* w, const float* row_scales, void* q, float* scales, float* part, int N, int K, cudaStream_t st) {
    const unsigned cols = (unsigned)((K + kWtCols - 1) / kWtCols);
    // four CTAs an SM, all of one size: rows a CTA by that, in steps of 64
    const unsigned want = (unsigned)(4 * gemm_num_sms()) / cols > 0 ? (unsigned)(4 * gemm_num_sms()) / cols : 1u;
    int rows = (int)((N + want - 1) / want + 63) / 64 * 64;
    if (rows > kWtMaxRows) rows = kWtMaxRows;
    const int parts = (N + rows - 1) / rows;
    Q8K_CUDA_OK(launch_dependent(gated_weight_absmax_kernel<Tw>, dim3(cols, (unsigned)parts), kWtThreads, 0, st, 1, (const Tw*)w, row_scales,
                                 part, N, K, rows));
    float* factors = part + (int64_t)parts * K;
    Q8K_CUDA_OK(launch_dependent(gated_weight_factor_kernel, dim3((unsigned)((K + 31) / 32)), 32 * kWtFactorWarps, 0, st, 1, part, parts, factors,
                                 scales, K));
    Q8K_CUDA_OK(launch_dependent(gated_weight_quant_kernel<Tw>, dim3(cols, (unsigned)((N + kWtRows - 1) / kWtRows)), kWtThreads, 0, st, 1,
                                 (const Tw*)w, row_scales, factors, (uint8_t*)q, N, K));
    return Q8K_OK;
}

}  // namespace q8k

extern "C" int q8k_gated_backward_quant(const void* grad, const void* pre, void* q, float* scales, int activation, int M, int F,
                                        void* stream) {
    using namespace q8k;
    const char* op = "gated_backward_quant";
    Q8K_REQUIRE(M >= 0 && F > 0 && F % 16 == 0, Q8K_ERR_INVALID_ARG, "%s: M=%d must not be negative and F=%d a multiple of 16", op, M, F);
    Q8K_REQUIRE(F <= kGatedMaxF, Q8K_ERR_UNSUPPORTED, "%s: F=%d exceeds %d", op, F, kGatedMaxF);
    Q8K_REQUIRE(M <= 0x7fff0000, Q8K_ERR_TOO_LARGE, "%s: M=%d too large", op, M);
    Q8K_REQUIRE(activation == Q8K_ACT_SILU || activation == Q8K_ACT_GELU_TANH, Q8K_ERR_UNSUPPORTED, "%s: activation %d is unknown", op,
                activation);
    if (M == 0) return Q8K_OK;
    Q8K_REQUIRE(grad && pre && q && scales && aligned16(grad) && aligned16(pre) && aligned16(q), Q8K_ERR_INVALID_ARG,
                "%s: null or misaligned pointer", op);
    cudaStream_t st = (cudaStream_t)stream;
    return activation == Q8K_ACT_GELU_TANH ? launch_gated_backward<true>(grad, pre, q, scales, M, F, st)
                                           : launch_gated_backward<false>(grad, pre, q, scales, M, F, st);
}

extern "C" size_t q8k_gated_weight_operand_workspace_bytes(int F, int K) {
    if (F <= 0 || K <= 0) return 0;
    return ((2 * (size_t)F + 63) / 64 + 1) * (size_t)K * sizeof(float);   // partial maxima of at least 64 rows, factors
}

extern "C" int q8k_gated_weight_operand(const void* w, int w_dtype, const float* w_scales, void* q, float* scales, int F, int K,
                                        void* workspace, size_t workspace_bytes, void* stream) {
    using namespace q8k;
    const char* op = "gated_weight_operand";
    Q8K_REQUIRE(F > 0 && K > 0 && F % 16 == 0 && K % 16 == 0, Q8K_ERR_INVALID_ARG, "%s: F=%d and K=%d must be positive multiples of 16", op,
                F, K);
    Q8K_REQUIRE(F <= 65535 * (kWtRows / 2), Q8K_ERR_TOO_LARGE, "%s: F=%d too large", op, F);
    Q8K_REQUIRE(w && w_scales && q && scales && workspace && aligned16(w) && aligned16(q) && aligned16(workspace), Q8K_ERR_INVALID_ARG,
                "%s: null or misaligned pointer", op);
    const size_t need = q8k_gated_weight_operand_workspace_bytes(F, K);
    Q8K_REQUIRE(workspace_bytes >= need, Q8K_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    cudaStream_t st = (cudaStream_t)stream;
    if (w_dtype == Q8K_DT_I8) return launch_gated_weight<int8_t>(w, w_scales, q, scales, (float*)workspace, 2 * F, K, st);
    if (w_dtype == Q8K_DT_E4M3) return launch_gated_weight<e4m3_t>(w, w_scales, q, scales, (float*)workspace, 2 * F, K, st);
    set_error_detail("%s: weight dtype %d is not int8 or e4m3", op, w_dtype);
    return Q8K_ERR_UNSUPPORTED;
}

extern "C" int q8k_gated_quant(const void* x, int x_dtype, int64_t x_row_stride, void* q, int q_dtype, float* scales, int64_t rows,
                               int dim, int rotate, void* stream) {
    using namespace q8k;
    const char* op = "gated_quant";
    Q8K_REQUIRE(x_dtype == Q8K_DT_BF16 || x_dtype == Q8K_DT_E4M3, Q8K_ERR_UNSUPPORTED, "%s: input dtype %d is not bf16 or e4m3", op, x_dtype);
    cudaStream_t st = (cudaStream_t)stream;
    return rotate ? hadamard_quant_as<true>(op, x, x_dtype, q, q_dtype, scales, rows, dim, x_row_stride, 1.0f / sqrtf((float)dim), st)
                  : tokenwise_quant_as<kRowsGated>(op, x, x_dtype, q, q_dtype, scales, rows, dim, x_row_stride, st);
}

extern "C" size_t q8k_gated_linear_workspace_bytes(int M, int K) {
    if (M <= 0 || K <= 0) return 0;
    return ((size_t)M * (size_t)K + 255) / 256 * 256 + (size_t)M * sizeof(float);
}

extern "C" int q8k_gated_linear(const void* x, int x_dtype, const void* w, int w_dtype, const float* w_scales, const float* bias, void* out,
                                void* pre, int activation, int M, int F, int K, int rotate, void* workspace, size_t workspace_bytes,
                                int* dev_status, void* stream) {
    using namespace q8k;
    const char* op = "gated_linear";
    Q8K_REQUIRE(M >= 0 && F > 0 && K > 0 && F % 16 == 0 && K % 16 == 0, Q8K_ERR_INVALID_ARG,
                "%s: M=%d must not be negative, F=%d and K=%d multiples of 16", op, M, F, K);
    Q8K_REQUIRE(w_dtype == Q8K_DT_I8 || w_dtype == Q8K_DT_E4M3, Q8K_ERR_UNSUPPORTED, "%s: weight dtype %d is not int8 or e4m3", op, w_dtype);
    Q8K_REQUIRE(x_dtype == Q8K_DT_BF16 || x_dtype == Q8K_DT_E4M3, Q8K_ERR_UNSUPPORTED, "%s: input dtype %d is not bf16 or e4m3", op, x_dtype);
    Q8K_REQUIRE(activation == Q8K_ACT_SILU || activation == Q8K_ACT_GELU_TANH, Q8K_ERR_UNSUPPORTED, "%s: activation %d is unknown", op,
                activation);
    if (M == 0) return Q8K_OK;
    Q8K_REQUIRE(x && w && w_scales && out && aligned16(w) && aligned16(out) && aligned16(pre), Q8K_ERR_INVALID_ARG,
                "%s: null or misaligned pointer", op);
    Q8K_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0, Q8K_ERR_INVALID_ARG,
                "%s: the workspace must be 256-byte aligned", op);
    const size_t need = q8k_gated_linear_workspace_bytes(M, K);
    Q8K_REQUIRE(workspace_bytes >= need, Q8K_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
    if (x_dtype == Q8K_DT_BF16 && aligned16(x) && gated_fused_rows(M, K))
        return gated_mm_fused(op, w_dtype == Q8K_DT_I8, x, rotate != 0, w, bias, w_scales, out, pre, activation, M, F, K, dev_status, stream);
    float* scales = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + ((size_t)M * (size_t)K + 255) / 256 * 256);
    if (int rc = q8k_gated_quant(x, x_dtype, K, workspace, w_dtype, scales, M, K, rotate, stream)) return rc;
    // The quantizer waits for everything before it and only then lets its dependents start, or does so by ending: by the time the
    // product may run, the weight is complete.
    return gated_mm(op, true, w_dtype == Q8K_DT_I8, workspace, w, bias, scales, w_scales, out, pre, activation, M, F, K, dev_status, stream);
}
