// Norm of every head of queries and keys, and its rotation by position, in one pass:  y = R(p) (x rstd w),  rstd = 1 / sqrt(mean(x^2) + eps).
// Backward, from x and the gradient g of y:
//   t = R(-p) g,   dw = sum over tokens and heads of t x rstd,   u = t w,   dx = rstd (u - x rstd^2 mean(u x))
// The two sums of a head, of x^2 and of u x, need no statistic of one another, so they are taken together and x and g are read once.
//
// Bound by HBM: forward reads and writes every element once, backward reads two and writes one.  The angles are made in the kernel, once per
// token and pair (rotary.cuh), and shared by the heads through shared memory.
//
// A head lies on as many lanes of one warp as it has units of 16 channels: 2 V channels at a time, one pair of runs of V, so that a lane's
// cosines, sines and weights stay the same for all heads that it takes, and the sums need shuffles only.
// In the half layout the runs of a rotated unit are half a rotation apart; otherwise they follow one another.

#include <type_traits>
#include "rotary.cuh"

namespace q8k {

struct HeadTensor {
    const void *x, *g;                       // g: gradient of the output, backward only
    const float* w;                          // null: 1
    void* out;                               // y, or dx
    int64_t x_batch, x_token, x_head, g_batch, g_token, g_head, out_batch, out_token, out_head;
    int heads;
};

struct HeadNormParams {
    HeadTensor t[2];                         // queries, keys
    RotaryAngles angles;
    float eps;
    float* part;                             // [CTA][2][head_dim] sums for dw; null: not wanted
    int64_t tokens;                          // batch * seq
    int seq, head_dim, rotary_dim, half;     // half: layout
};

constexpr int kHeadMaxDim = 512;
constexpr int kHeadThreads = 128;
constexpr int kHeadChannels = 16;            // channels of a lane
constexpr int kHeadRows = 8;                 // heads of a thread, where there are threads for the others
constexpr int kHeadMaxCtas = 148 * 8;        // of the backward pass with sums

// A warp's lanes are groups of `lanes`, each with a head; a CTA's groups are `tokens` times `head_lanes`.
struct HeadLanes { int lanes, groups, head_lanes, tokens; };

template <int BYTES> struct HeadRaw;
template <> struct HeadRaw<2>  { using type = uint16_t; };
template <> struct HeadRaw<4>  { using type = uint32_t; };
template <> struct HeadRaw<8>  { using type = uint2; };
template <> struct HeadRaw<16> { using type = uint4; };

// Sum over a group's lanes, in each of them; `top` is half the power of two that holds them.
__device__ __forceinline__ float head_sum(float v, int lane, int lanes, int top, bool pow2) {
    if (pow2) {
        for (int o = top; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    }
    const int in = lane % lanes, first = lane - in;
    for (int o = top; o > 0; o >>= 1) {
        const float u = __shfl_down_sync(0xffffffffu, v, o);
        if (in + o < lanes) v += u;
    }
    return __shfl_sync(0xffffffffu, v, first);
}

// V channels an access.  TWO: a pair's channels lie in the two runs of a unit (half layout, or V = 1), else side by side in one.
template <typename T, int V, bool TWO, bool BACK>
__global__ void __launch_bounds__(kHeadThreads, BACK ? 2 : 4)
head_norm_kernel(const __grid_constant__ HeadNormParams p, const HeadLanes l) {
    constexpr int UNITS = kHeadChannels / (2 * V);             // of a lane
    using Raw = typename HeadRaw<V * sizeof(T)>::type;
    union Run { Raw r; T e[V]; };
    struct Head { Run a[UNITS], b[UNITS]; };
    extern __shared__ float smem[];
    float2* turns = reinterpret_cast<float2*>(smem);           // [tokens][rotary_dim / 2] cosine, sine
    const int half_dim = p.rotary_dim / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int group = lane / l.lanes, ul = lane - group * l.lanes;
    const int slot = warp * l.groups + group;
    const int tl = slot / l.head_lanes, h0 = slot - tl * l.head_lanes;
    const bool has_slot = group < l.groups && tl < l.tokens;
    const bool pow2 = (l.lanes & (l.lanes - 1)) == 0;
    int top = 16;                                              // half the power of two that holds the lanes
    while (top >= l.lanes && top > 0) top >>= 1;
    pdl_wait();
    pdl_release();

    // where the runs of this lane's units begin, and whether they exist
    int at_a[UNITS], at_b[UNITS], turn_at[UNITS];
    bool has_a[UNITS], has_b[UNITS], turned[UNITS];
    const int rot_units = TWO ? half_dim / V : 0;
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        const int u = ul + j * l.lanes;
        turned[j] = u < rot_units;
        turn_at[j] = u * V;
        if (TWO && turned[j]) {
            at_a[j] = p.half ? u * V : 2 * u * V;
            at_b[j] = at_a[j] + (p.half ? half_dim : 1);
        } else {
            at_a[j] = 2 * u * V;
            if (TWO) at_a[j] = p.rotary_dim + 2 * (u - rot_units) * V;
            at_b[j] = at_a[j] + V;
        }
        has_a[j] = has_slot && at_a[j] < p.head_dim;
        has_b[j] = has_slot && at_b[j] < p.head_dim;
    }
    float acc[BACK ? 2 : 1][BACK ? kHeadChannels : 1];
    if constexpr (BACK) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < kHeadChannels; ++j) acc[i][j] = 0.f;
    }

    const int64_t blocks = (p.tokens + l.tokens - 1) / l.tokens;
    for (int64_t block = blockIdx.x; block < blocks; block += gridDim.x) {
        const int64_t token = block * l.tokens + tl;
        const bool here = has_slot && token < p.tokens;
        const int64_t batch = token / p.seq, s = token - batch * p.seq;
        if (half_dim > 0) {
            if (block != (int64_t)blockIdx.x) __syncthreads(); // the angles before have been read
            for (int i = threadIdx.x; i < l.tokens * half_dim; i += kHeadThreads) {
                const int k = i / half_dim, pair = i - k * half_dim;
                const int64_t tok = block * l.tokens + k;
                if (tok < p.tokens) {
                    const int64_t b = tok / p.seq, at = tok - b * p.seq;
                    const RotaryAngles& a = p.angles;
                    const int64_t from = b * a.pos_batch + at * a.pos_token;
                    const double pos = a.positions == nullptr ? (double)at : a.axes != nullptr ? rotary_position<true>(a, from, pair)
                                                                                               : rotary_position<false>(a, from, pair);
                    turns[i] = rotary_turn(a, pos, pair);
                }
            }
            __syncthreads();
        }
        // the lane's cosines and sines: (1, 0) for channels that are not rotated
        float2 turn[UNITS][V];
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                bool rot = turned[j];
                int i = turn_at[j] + k;
                if constexpr (!TWO) {                          // pairs k < V / 2 in run a, the others in run b
                    i = (k < V / 2 ? at_a[j] : at_b[j] - V) / 2 + k;
                    rot = i < half_dim;
                }
                turn[j][k] = here && rot ? turns[tl * half_dim + i] : make_float2(1.f, 0.f);
            }
        }
#pragma unroll
        for (int which = 0; which < 2; ++which) {
            const HeadTensor& t = p.t[which];
            if (t.heads == 0) continue;
            float w[UNITS][2][V];
#pragma unroll
            for (int j = 0; j < UNITS; ++j) {
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    w[j][0][k] = t.w == nullptr || !has_a[j] ? 1.f : t.w[at_a[j] + k];
                    w[j][1][k] = t.w == nullptr || !has_b[j] ? 1.f : t.w[at_b[j] + k];
                }
            }
            const T* x = static_cast<const T*>(t.x) + batch * t.x_batch + s * t.x_token;
            const T* g = static_cast<const T*>(t.g) + batch * t.g_batch + s * t.g_token;
            T* out = static_cast<T*>(t.out) + batch * t.out_batch + s * t.out_token;
            const int rounds = (t.heads + l.head_lanes - 1) / l.head_lanes;
            constexpr int AHEAD = 2;                           // heads on their way together
            for (int r0 = 0; r0 < rounds; r0 += AHEAD) {       // (the same for all lanes of a warp)
                Head in[AHEAD], gr[BACK ? AHEAD : 1];
                bool ok[AHEAD];
#pragma unroll
                for (int q = 0; q < AHEAD; ++q) {
                    const int h = h0 + (r0 + q) * l.head_lanes;
                    ok[q] = here && h < t.heads;
#pragma unroll
                    for (int j = 0; j < UNITS; ++j) {
                        in[q].a[j].r = in[q].b[j].r = Raw{};
                        if (ok[q] && has_a[j]) in[q].a[j].r = *reinterpret_cast<const Raw*>(x + h * t.x_head + at_a[j]);
                        if (ok[q] && has_b[j]) in[q].b[j].r = *reinterpret_cast<const Raw*>(x + h * t.x_head + at_b[j]);
                        if constexpr (BACK) {
                            gr[q].a[j].r = gr[q].b[j].r = Raw{};
                            if (ok[q] && has_a[j]) gr[q].a[j].r = *reinterpret_cast<const Raw*>(g + h * t.g_head + at_a[j]);
                            if (ok[q] && has_b[j]) gr[q].b[j].r = *reinterpret_cast<const Raw*>(g + h * t.g_head + at_b[j]);
                        }
                    }
                }
#pragma unroll
                for (int q = 0; q < AHEAD; ++q) {
                    if (r0 + q >= rounds) break;
                    const int h = h0 + (r0 + q) * l.head_lanes;
                    float v[UNITS][2][V], d[BACK ? UNITS : 1][2][V];
                    float sum = 0.f, dot = 0.f;
#pragma unroll
                    for (int j = 0; j < UNITS; ++j) {
#pragma unroll
                        for (int k = 0; k < V; ++k) {
                            v[j][0][k] = to_float<T>(in[q].a[j].e[k]);
                            v[j][1][k] = to_float<T>(in[q].b[j].e[k]);
                            sum = fmaf(v[j][0][k], v[j][0][k], sum);
                            sum = fmaf(v[j][1][k], v[j][1][k], sum);
                        }
                    }
                    // the rotation of a unit's pairs in place
                    auto rotate = [&](float (&y)[2][V], const float2 (&c)[V]) {
#pragma unroll
                        for (int k = 0; k < V; ++k) {
                            float& a = TWO ? y[0][k] : y[2 * k / V][2 * k % V];
                            float& b = TWO ? y[1][k] : y[2 * k / V][2 * k % V + (V > 1 ? 1 : 0)];
                            const float a0 = a, b0 = b;
                            a = a0 * c[k].x - b0 * c[k].y;
                            b = b0 * c[k].x + a0 * c[k].y;
                        }
                    };
                    if constexpr (BACK) {
#pragma unroll
                        for (int j = 0; j < UNITS; ++j) {
#pragma unroll
                            for (int k = 0; k < V; ++k) {
                                d[j][0][k] = to_float<T>(gr[q].a[j].e[k]);
                                d[j][1][k] = to_float<T>(gr[q].b[j].e[k]);
                            }
                            rotate(d[j], turn[j]);             // (the sine is negated)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int k = 0; k < V; ++k) dot = fmaf(d[j][i][k] * w[j][i][k], v[j][i][k], dot);
                        }
                    }
                    sum = head_sum(sum, lane, l.lanes, top, pow2);
                    if constexpr (BACK) dot = head_sum(dot, lane, l.lanes, top, pow2);
                    const float rstd = rsqrtf(sum / (float)p.head_dim + p.eps);
                    const float c = BACK ? rstd * rstd * dot / (float)p.head_dim : 0.f;
#pragma unroll
                    for (int j = 0; j < UNITS; ++j) {
                        if constexpr (BACK) {
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int k = 0; k < V; ++k) {
                                    if (ok[q]) acc[which][(j * 2 + i) * V + k] = fmaf(d[j][i][k], v[j][i][k] * rstd, acc[which][(j * 2 + i) * V + k]);
                                    v[j][i][k] = rstd * (d[j][i][k] * w[j][i][k] - v[j][i][k] * c);
                                }
                        } else {
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int k = 0; k < V; ++k) v[j][i][k] = v[j][i][k] * rstd * w[j][i][k];
                            rotate(v[j], turn[j]);
                        }
#pragma unroll
                        for (int k = 0; k < V; ++k) {
                            in[q].a[j].e[k] = from_float<T>(v[j][0][k]);
                            in[q].b[j].e[k] = from_float<T>(v[j][1][k]);
                        }
                        if (ok[q] && has_a[j]) *reinterpret_cast<Raw*>(out + h * t.out_head + at_a[j]) = in[q].a[j].r;
                        if (ok[q] && has_b[j]) *reinterpret_cast<Raw*>(out + h * t.out_head + at_b[j]) = in[q].b[j].r;
                    }
                }
            }
        }
    }
    if constexpr (BACK) {
        if (p.part == nullptr) return;
        // over the CTA's groups in order, queries then keys
        const int slots = kHeadThreads / 32 * l.groups;
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
            if (group < l.groups) {
#pragma unroll
                for (int j = 0; j < UNITS; ++j)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        if (has_a[j]) smem[slot * p.head_dim + at_a[j] + k] = which == 0 ? acc[0][(j * 2) * V + k] : acc[1][(j * 2) * V + k];
                        if (has_b[j]) smem[slot * p.head_dim + at_b[j] + k] = which == 0 ? acc[0][(j * 2 + 1) * V + k] : acc[1][(j * 2 + 1) * V + k];
                    }
            }
            __syncthreads();
            for (int c = threadIdx.x; c < p.head_dim; c += kHeadThreads) {
                float a = 0.f;
                for (int k = 0; k < slots && k < l.tokens * l.head_lanes; ++k) a += smem[k * p.head_dim + c];
                p.part[((int64_t)blockIdx.x * 2 + which) * p.head_dim + c] = a;
            }
        }
    }
}

// dw of queries and keys from the CTAs' sums, 32 columns a CTA, in a fixed order
constexpr int kHeadSumWarps = 8;
__global__ void __launch_bounds__(32 * kHeadSumWarps)
head_norm_sum_kernel(const float* __restrict__ part, int parts, float* __restrict__ dq, float* __restrict__ dk, int dim) {
    __shared__ float red[kHeadSumWarps][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int c = blockIdx.x * 32 + lane;                      // of 2 dim
    pdl_wait();
    pdl_release();
    float a = 0.f;
    if (c < 2 * dim)
        for (int k = warp; k < parts; k += kHeadSumWarps) a += part[(int64_t)k * 2 * dim + c];
    red[warp][lane] = a;
    __syncthreads();
    if (warp == 0 && c < 2 * dim) {
#pragma unroll
        for (int k = 1; k < kHeadSumWarps; ++k) a += red[k][lane];
        float* out = c < dim ? dq : dk;
        if (out != nullptr) out[c < dim ? c : c - dim] = a;
    }
}

template <typename T, int V, bool TWO, bool BACK>
static int launch_head_norm_as(const HeadNormParams& p, float* dqw, float* dkw, cudaStream_t st) {
    constexpr int UNITS = kHeadChannels / (2 * V);
    // units of a head: those that are rotated, and the rest (TWO); else pairs of runs
    const int units = TWO ? p.rotary_dim / 2 / V + (p.head_dim - p.rotary_dim + 2 * V - 1) / (2 * V) : (p.head_dim + 2 * V - 1) / (2 * V);
    HeadLanes l;
    l.lanes = (units + UNITS - 1) / UNITS;
    l.groups = 32 / l.lanes;
    const int slots = kHeadThreads / 32 * l.groups;
    const int heads = p.t[0].heads > p.t[1].heads ? p.t[0].heads : p.t[1].heads;
    int per_thread = kHeadRows;
    auto lanes = [&](int n) { const int want = (heads + n - 1) / n; return want < slots ? want : slots; };
    while (per_thread > 1 && (p.tokens + slots / lanes(per_thread) - 1) / (slots / lanes(per_thread)) < gemm_num_sms()) --per_thread;
    l.head_lanes = lanes(per_thread);
    l.tokens = slots / l.head_lanes;
    const int room = p.rotary_dim > 0 ? 24 * 1024 / (4 * p.rotary_dim) : l.tokens;
    if (l.tokens > room) l.tokens = room;
    const int64_t blocks = (p.tokens + l.tokens - 1) / l.tokens;
    int64_t grid = blocks;
    size_t smem = (size_t)l.tokens * p.rotary_dim * 4;
    if (BACK && p.part != nullptr) {
        const int64_t most = 4 * gemm_num_sms() < kHeadMaxCtas ? 4 * gemm_num_sms() : kHeadMaxCtas;
        if (grid > most) grid = most;
        const size_t sums = (size_t)slots * p.head_dim * 4;
        if (smem < sums) smem = sums;
    }
    Q8K_CUDA_OK(launch_dependent(head_norm_kernel<T, V, TWO, BACK>, (unsigned)grid, kHeadThreads, smem, st, 1, p, l));
    if (BACK && p.part != nullptr)
        Q8K_CUDA_OK(launch_dependent(head_norm_sum_kernel, (unsigned)((2 * p.head_dim + 31) / 32), 32 * kHeadSumWarps, 0, st, 1, p.part, (int)grid, dqw, dkw,
                                     p.head_dim));
    return Q8K_OK;
}

template <typename T, bool BACK> static int launch_head_norm(const HeadNormParams& p, int v, float* dqw, float* dkw, cudaStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (v == 8) return p.half ? launch_head_norm_as<T, 8, true, BACK>(p, dqw, dkw, st) : launch_head_norm_as<T, 8, false, BACK>(p, dqw, dkw, st);
    }
    if (v >= 4) return p.half ? launch_head_norm_as<T, 4, true, BACK>(p, dqw, dkw, st) : launch_head_norm_as<T, 4, false, BACK>(p, dqw, dkw, st);
    if (v >= 2) return p.half ? launch_head_norm_as<T, 2, true, BACK>(p, dqw, dkw, st) : launch_head_norm_as<T, 2, false, BACK>(p, dqw, dkw, st);
    return launch_head_norm_as<T, 1, true, BACK>(p, dqw, dkw, st);
}

// One call of either direction.  in[i]: x, gradient (backward), output of queries and keys, with their strides.
struct HeadArgs { const void *x, *g; void* out; const int64_t *xs, *gs, *os; const float* w; float* dw; int heads; };
template <bool BACK>
static int head_norm(const char* op, const HeadArgs (&in)[2], int dtype, float eps, const RotaryAngles& angles, int batch, int seq, int head_dim,
                     int rotary_dim, int half_layout, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    Q8K_REQUIRE(batch >= 0 && seq >= 0 && in[0].heads >= 0 && in[1].heads >= 0 && head_dim > 0, Q8K_ERR_INVALID_ARG, "%s: negative size", op);
    Q8K_REQUIRE(rotary_dim >= 0 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, Q8K_ERR_INVALID_ARG,
                "%s: rotary_dim %d must be even and at most the head dim %d", op, rotary_dim, head_dim);
    Q8K_REQUIRE(head_dim <= kHeadMaxDim, Q8K_ERR_UNSUPPORTED, "%s: head dim %d exceeds %d", op, head_dim, kHeadMaxDim);
    Q8K_REQUIRE((int64_t)(in[0].heads + (int64_t)in[1].heads) * head_dim <= (1 << 24), Q8K_ERR_UNSUPPORTED, "%s: %d + %d heads of %d are too many", op,
                in[0].heads, in[1].heads, head_dim);
    Q8K_REQUIRE(dtype == Q8K_DT_F32 || dtype == Q8K_DT_F16 || dtype == Q8K_DT_BF16, Q8K_ERR_UNSUPPORTED,
                "%s: dtype %d is not float32, float16 or bfloat16", op, dtype);
    Q8K_REQUIRE((int64_t)batch * seq <= 0x7fffffffLL, Q8K_ERR_TOO_LARGE, "%s: %lld tokens", op, (long long)batch * seq);
    const int size = dtype_size(dtype);
    HeadNormParams p = {};
    const bool sums = BACK && (in[0].dw != nullptr || in[1].dw != nullptr);
    if (sums) {
        const size_t need = q8k_head_norm_backward_workspace_bytes(head_dim);
        Q8K_REQUIRE(workspace != nullptr && aligned16(workspace), Q8K_ERR_INVALID_ARG, "%s: null or misaligned workspace", op);
        Q8K_REQUIRE(workspace_bytes >= need, Q8K_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, need);
        p.part = static_cast<float*>(workspace);
    }
    if (batch == 0 || seq == 0 || in[0].heads + in[1].heads == 0) {
        for (const HeadArgs& a : in)
            if (sums && a.dw != nullptr) Q8K_CUDA_OK(cudaMemsetAsync(a.dw, 0, (size_t)head_dim * sizeof(float), st));
        return Q8K_OK;
    }
    if (rotary_dim > 0) {
        if (int rc = rotary_check_angles(op, angles)) return rc;
    }
    // the widest access, up to 16 bytes, that divides the channels, strides and addresses of all tensors
    int v = 16 / size;
    auto divides = [&](int64_t n) { while (n % v != 0) v /= 2; };
    divides(head_dim);
    divides(rotary_dim);
    if (half_layout) divides(rotary_dim / 2);
    for (int i = 0; i < 2; ++i) {
        const HeadArgs& a = in[i];
        HeadTensor& t = p.t[i];
        t.heads = a.heads;
        if (a.heads == 0) continue;
        const void* ptrs[3] = {a.x, BACK ? a.g : a.x, a.out};
        const int64_t* strides[3] = {a.xs, BACK ? a.gs : a.xs, a.os};
        const int64_t n[3] = {batch, seq, a.heads};
        for (int k = 0; k < 3; ++k) {
            Q8K_REQUIRE(ptrs[k] != nullptr && strides[k] != nullptr && reinterpret_cast<uintptr_t>(ptrs[k]) % size == 0, Q8K_ERR_INVALID_ARG,
                        "%s: null or misaligned pointer", op);
            divides((int64_t)(reinterpret_cast<uintptr_t>(ptrs[k]) / size));
            for (int j = 0; j < 3; ++j)
                if (n[j] > 1) divides(strides[k][j]);          // a stride over one element does not matter
        }
        Q8K_REQUIRE(reinterpret_cast<uintptr_t>(a.w) % 4 == 0, Q8K_ERR_INVALID_ARG, "%s: misaligned weight", op);
        t.x = a.x; t.g = BACK ? a.g : a.x; t.w = a.w; t.out = a.out;
        t.x_batch = strides[0][0]; t.x_token = strides[0][1]; t.x_head = strides[0][2];
        t.g_batch = strides[1][0]; t.g_token = strides[1][1]; t.g_head = strides[1][2];
        t.out_batch = strides[2][0]; t.out_token = strides[2][1]; t.out_head = strides[2][2];
    }
    p.angles = angles;
    p.angles.sign = BACK ? -1.f : 1.f;
    p.eps = eps;
    p.tokens = (int64_t)batch * seq;
    p.seq = seq; p.head_dim = head_dim; p.rotary_dim = rotary_dim; p.half = half_layout != 0;
    float *dqw = in[0].dw, *dkw = in[1].dw;
    if (dtype == Q8K_DT_BF16) return launch_head_norm<__nv_bfloat16, BACK>(p, v, dqw, dkw, st);
    if (dtype == Q8K_DT_F16) return launch_head_norm<__half, BACK>(p, v, dqw, dkw, st);
    return launch_head_norm<float, BACK>(p, v, dqw, dkw, st);
}

static RotaryAngles head_angles(const void* positions, int type, const int64_t* strides, int n_axes, const int* axes, const double* freq, float amplitude) {
    RotaryAngles a = {positions, type, 0, 0, 0, axes, n_axes, freq, amplitude, 1.f};
    if (positions != nullptr && strides != nullptr) {
        a.pos_batch = strides[0];
        a.pos_token = strides[1];
        a.pos_axis = axes != nullptr ? strides[2] : 0;
    }
    return a;
}

}  // namespace q8k

extern "C" int q8k_head_norm(const void* q, const int64_t q_strides[3], const float* q_weight, void* q_out, const int64_t q_out_strides[3], int q_heads,
                             const void* k, const int64_t k_strides[3], const float* k_weight, void* k_out, const int64_t k_out_strides[3], int k_heads,
                             int dtype, float eps, const void* positions, int position_type, const int64_t position_strides[3], int n_axes,
                             const int* axes, const double* frequencies, float amplitude, int batch, int seq, int head_dim, int rotary_dim,
                             int half_layout, void* stream) {
    using namespace q8k;
    Q8K_REQUIRE(positions == nullptr || position_strides != nullptr, Q8K_ERR_INVALID_ARG, "head_norm: null position strides");
    const HeadArgs in[2] = {{q, nullptr, q_out, q_strides, nullptr, q_out_strides, q_weight, nullptr, q_heads},
                            {k, nullptr, k_out, k_strides, nullptr, k_out_strides, k_weight, nullptr, k_heads}};
    return head_norm<false>("head_norm", in, dtype, eps, head_angles(positions, position_type, position_strides, n_axes, axes, frequencies, amplitude),
                            batch, seq, head_dim, rotary_dim, half_layout, nullptr, 0, (cudaStream_t)stream);
}

extern "C" size_t q8k_head_norm_backward_workspace_bytes(int head_dim) {
    return head_dim <= 0 ? 0 : (size_t)q8k::kHeadMaxCtas * 2 * (size_t)head_dim * sizeof(float);
}

extern "C" int q8k_head_norm_backward(const void* q, const int64_t q_strides[3], const float* q_weight, const void* q_grad,
                                      const int64_t q_grad_strides[3], void* dq, const int64_t dq_strides[3], float* dq_weight, int q_heads,
                                      const void* k, const int64_t k_strides[3], const float* k_weight, const void* k_grad,
                                      const int64_t k_grad_strides[3], void* dk, const int64_t dk_strides[3], float* dk_weight, int k_heads, int dtype,
                                      float eps, const void* positions, int position_type, const int64_t position_strides[3], int n_axes,
                                      const int* axes, const double* frequencies, float amplitude, int batch, int seq, int head_dim,
                                      int rotary_dim, int half_layout, void* workspace, size_t workspace_bytes, void* stream) {
    using namespace q8k;
    Q8K_REQUIRE(positions == nullptr || position_strides != nullptr, Q8K_ERR_INVALID_ARG, "head_norm_backward: null position strides");
    const HeadArgs in[2] = {{q, q_grad, dq, q_strides, q_grad_strides, dq_strides, q_weight, dq_weight, q_heads},
                            {k, k_grad, dk, k_strides, k_grad_strides, dk_strides, k_weight, dk_weight, k_heads}};
    return head_norm<true>("head_norm_backward", in, dtype, eps,
                           head_angles(positions, position_type, position_strides, n_axes, axes, frequencies, amplitude), batch, seq, head_dim,
                           rotary_dim, half_layout, workspace, workspace_bytes, (cudaStream_t)stream);
}
