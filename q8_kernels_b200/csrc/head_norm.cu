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
// The heads that a thread takes one after the other are on their way by cp.async, three ahead: with plain loads two ahead 64 registers more were needed and
// 16384 x 40 x 128 took 86 us forward and 195 backward.  Measured (bf16, CUDA graphs, of the copy rate): 16384 x 40 x 128 forward 55.5 us (0.92), backward
// 95.5 (0.81; without dw 84), 6144 x 64 x 64 17.7 and 33.5; fp32 8192 x 32 x 128 44.5 (0.92) and 67.8 (0.91).  Tried: five and seven, three and five
// CTAs an SM, three stages: all slower.

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
    float* part;                             // [CTA][head_dim] sums for dw; null: not wanted
    unsigned tokens;                         // batch * seq
    unsigned seq;
    int head_dim, rotary_dim, half;          // half: layout
};

constexpr int kHeadMaxDim = 512;
constexpr int kHeadThreads = 128;
constexpr int kHeadChannels = 16;            // channels of a lane: 8 in the first runs of its units, 8 in the second
constexpr int kHeadRows = 8;                 // heads of a thread, where there are threads for the others
// CTAs of the backward pass with sums, four of which an SM holds at once: one that works on, token after token, adds up more before it writes its
// sums, but the last ones leave SMs idle.  16384 x 40 x 128 with 4, 8, 12, 16, 20, 24, 36 an SM: 110, 103, 97, 96.5, 95.5, 98, 103 us.
constexpr int kHeadSumCtas = 20, kHeadMaxCtas = 148 * kHeadSumCtas;

// A warp's lanes are groups of `lanes`, each with a head.  A CTA works for queries or for keys; its groups are `tokens` times `head_lanes`.
// CTAs [0, ctas[0]) are the queries', the ctas[1] behind them the keys'.
struct HeadSplit { int head_lanes, tokens, ctas; };
struct HeadLanes { int lanes, groups; HeadSplit of[2]; };

template <int BYTES> struct HeadRaw;
template <> struct HeadRaw<2>  { using type = uint16_t; };
template <> struct HeadRaw<4>  { using type = uint32_t; };
template <> struct HeadRaw<8>  { using type = uint2; };
template <> struct HeadRaw<16> { using type = uint4; };

// Sums over a group's lanes, in each of them.  LANES 0: any number of them, `top` is half the power of two that holds them.
template <int LANES, int N> __device__ __forceinline__ void head_sum(float (&v)[N], int lane, int lanes, int top) {
    if constexpr (LANES > 0) {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
        }
    } else {
        const int in = lane % lanes, first = lane - in;
#pragma unroll 1
        for (int o = top; o > 0; o >>= 1) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float u = __shfl_down_sync(0xffffffffu, v[i], o);
                if (in + o < lanes) v[i] += u;
            }
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __shfl_sync(0xffffffffu, v[i], first);
    }
}

// Eight values of a lane's runs, widened as packed pairs, and back.
template <typename T> __device__ __forceinline__ void head_widen(const T (&e)[8], float2 (&v)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(to_float<T>(e[2 * i]), to_float<T>(e[2 * i + 1]));
}
template <> __device__ __forceinline__ void head_widen<__nv_bfloat16>(const __nv_bfloat16 (&e)[8], float2 (&v)[4]) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&e);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
}
template <typename T> __device__ __forceinline__ void head_narrow(const float2 (&v)[4], T (&e)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        e[2 * i] = from_float<T>(v[i].x);
        e[2 * i + 1] = from_float<T>(v[i].y);
    }
}
template <> __device__ __forceinline__ void head_narrow<__nv_bfloat16>(const float2 (&v)[4], __nv_bfloat16 (&e)[8]) {
    __nv_bfloat162* w = reinterpret_cast<__nv_bfloat162*>(&e);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __floats2bfloat162_rn(v[i].x, v[i].y);
}
template <> __device__ __forceinline__ void head_narrow<__half>(const float2 (&v)[4], __half (&e)[8]) {
    __half2* w = reinterpret_cast<__half2*>(&e);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = __floats2half2_rn(v[i].x, v[i].y);
}

// Asynchronous copy of BYTES (4, 8 or 16) to shared memory, zeros where `there` is false.
template <int BYTES> __device__ __forceinline__ void head_copy(uint32_t dst, const void* src, bool there) {
    const int n = there ? BYTES : 0;
    if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(dst), "l"(src), "n"(BYTES), "r"(n) : "memory");
}

// V channels an access.  TWO: a pair's channels lie in the two runs of a unit (half layout, or V = 1), else side by side in one.
// A lane has 8 / V units; their first runs are its channels a[0..8), their second ones b[0..8).
//
// A thread's heads are on their way to its own slots of a ring in shared memory, STAGES of them, the first while the angles are made and the
// next token's while this one's are worked on.
template <typename T, bool BACK> struct HeadRing {
    static constexpr int stages = BACK && sizeof(T) == 4 ? 3 : 4;         // (three of 16 KB leave room for four CTAs an SM)
    static constexpr int pieces = 8 * (int)sizeof(T) / 16;     // 16-byte pieces of a run
    static constexpr int runs = BACK ? 4 : 2;                  // x: a, b; gradient: a, b
    static constexpr int stage_bytes = runs * pieces * kHeadThreads * 16;
    static constexpr int bytes = stages * stage_bytes;
};
//
// LANES: heads of 16 LANES channels, all of whose lanes and, in every round, heads exist, and weights of 16-byte alignment; 0: any.  (The
// checks, the sums' loops and the index arithmetic of the general form are half of its instructions.)
template <typename T, int V, bool TWO, bool BACK, int LANES>
__global__ void __launch_bounds__(kHeadThreads, BACK ? 4 : 6)
head_norm_kernel(const __grid_constant__ HeadNormParams p, const __grid_constant__ HeadLanes l) {
    using Ring = HeadRing<T, BACK>;
    constexpr int UNITS = 8 / V;
    using Raw = typename HeadRaw<V * sizeof(T)>::type;
    extern __shared__ __align__(16) uint8_t smem[];
    float2* turns = reinterpret_cast<float2*>(smem + Ring::bytes);             // [tokens][rotary_dim / 2] cosine, sine
    const bool keys = (int)blockIdx.x >= l.of[0].ctas;
    const HeadSplit& sp = l.of[keys];
    const HeadTensor& t = p.t[keys];
    const unsigned cta = blockIdx.x - (keys ? l.of[0].ctas : 0);
    const int half_dim = p.rotary_dim / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int lanes = LANES > 0 ? LANES : l.lanes, groups = LANES > 0 ? 32 / LANES : l.groups;
    const int group = lane / lanes, ul = lane - group * lanes;
    const int slot = warp * groups + group;
    const int tl = slot / sp.head_lanes, h0 = slot - tl * sp.head_lanes;
    const bool has_slot = (LANES > 0 || group < groups) && tl < sp.tokens;
    int top = 16;                                              // half the power of two that holds the lanes
    while (top >= lanes) top >>= 1;
    pdl_wait();
    pdl_release();

    // where the runs of this lane's units begin, and whether they exist
    int at_a[UNITS], at_b[UNITS];
    bool has_a[UNITS], has_b[UNITS];
    // (neighbouring lanes' runs follow one another: with both runs of a unit side by side, every access would take half of each sector, and
    // 16384 x 40 x 128 interleaved took 84 us in the place of 64)
    const int rot_units = TWO ? half_dim / V : 0;
    const int rest_units = TWO ? (p.head_dim - p.rotary_dim + 2 * V - 1) / (2 * V) : 0;
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        const int u = ul + j * lanes;
        if (!TWO) {
            at_a[j] = (ul + 2 * j * lanes) * V;
            at_b[j] = at_a[j] + lanes * V;
        } else if (u < rot_units) {
            at_a[j] = p.half ? u * V : 2 * u * V;
            at_b[j] = at_a[j] + (p.half ? half_dim : 1);
        } else {                                               // a unit of channels that are not rotated
            at_a[j] = u - rot_units < rest_units ? p.rotary_dim + (u - rot_units) * V : p.head_dim;
            at_b[j] = at_a[j] + rest_units * V;
        }
        has_a[j] = LANES > 0 || (has_slot && at_a[j] < p.head_dim);
        has_b[j] = LANES > 0 || (has_slot && at_b[j] < p.head_dim);
    }
    const unsigned blocks = (p.tokens + sp.tokens - 1) / sp.tokens;
    const int rounds = (t.heads + sp.head_lanes - 1) / sp.head_lanes;          // the same for all threads

    // ---- the ring
    const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
    // a run's unit j of a stage: bytes j V sizeof(T) of it, in pieces of 16
    auto place = [](int stage, int run, int j) {
        const int at = j * V * (int)sizeof(T);
        return stage * Ring::stage_bytes + (run * Ring::pieces + at / 16) * kHeadThreads * 16 + at % 16;
    };
    auto bring = [&](int stage, int run, const T* from, const int (&at)[UNITS], const bool (&has)[UNITS], bool ok) {
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
            const bool there = ok && has[j];
            const T* src = from + at[j];                       // (not read unless it is there)
            if constexpr (V * sizeof(T) >= 4) {
                head_copy<V * (int)sizeof(T)>(ring + place(stage, run, j), src, there);
            } else {
                *reinterpret_cast<Raw*>(smem + threadIdx.x * 16 + place(stage, run, j)) = there ? *reinterpret_cast<const Raw*>(src) : Raw{};
            }
        }
    };
    unsigned f_block = cta;
    int f_round = 0, f_stage = 0;
    const T *fx = static_cast<const T*>(t.x), *fg = static_cast<const T*>(t.g);
    bool f_here = false;
    auto fetch_token = [&]() {                                 // f_block's token
        const unsigned token = f_block * sp.tokens + tl;
        f_here = has_slot && f_block < blocks && token < p.tokens;
        const unsigned batch = f_here ? token / p.seq : 0, s = f_here ? token - batch * p.seq : 0;
        fx = static_cast<const T*>(t.x) + batch * t.x_batch + s * t.x_token + h0 * t.x_head;
        if constexpr (BACK) fg = static_cast<const T*>(t.g) + batch * t.g_batch + s * t.g_token + h0 * t.g_head;
    };
    auto fetch = [&]() {
        const bool ok = f_here && (LANES > 0 || h0 + f_round * sp.head_lanes < t.heads);
        bring(f_stage, 0, fx, at_a, has_a, ok);
        bring(f_stage, 1, fx, at_b, has_b, ok);
        if constexpr (BACK) {
            bring(f_stage, 2, fg, at_a, has_a, ok);
            bring(f_stage, 3, fg, at_b, has_b, ok);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        fx += sp.head_lanes * t.x_head;
        if constexpr (BACK) fg += sp.head_lanes * t.g_head;
        f_stage = f_stage + 1 == Ring::stages ? 0 : f_stage + 1;
        if (++f_round == rounds) {
            f_round = 0;
            f_block += sp.ctas;
            fetch_token();
        }
    };
    fetch_token();
#pragma unroll
    for (int i = 0; i + 1 < Ring::stages; ++i) fetch();

    float2 w[2][4], acc[2][BACK ? 4 : 1];
#pragma unroll
    for (int j = 0; j < UNITS; ++j) {
        if constexpr (LANES > 0) {
#pragma unroll
            for (int k = 0; k < V; k += 4) {
                const float4 one = make_float4(1.f, 1.f, 1.f, 1.f);
                const float4 wa = t.w == nullptr ? one : *reinterpret_cast<const float4*>(t.w + at_a[j] + k);
                const float4 wb = t.w == nullptr ? one : *reinterpret_cast<const float4*>(t.w + at_b[j] + k);
                const int i = (j * V + k) / 2;
                w[0][i] = make_float2(wa.x, wa.y); w[0][i + 1] = make_float2(wa.z, wa.w);
                w[1][i] = make_float2(wb.x, wb.y); w[1][i + 1] = make_float2(wb.z, wb.w);
            }
        } else {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int i = j * V + k;
                (i % 2 ? w[0][i / 2].y : w[0][i / 2].x) = t.w == nullptr || !has_a[j] ? 1.f : t.w[at_a[j] + k];
                (i % 2 ? w[1][i / 2].y : w[1][i / 2].x) = t.w == nullptr || !has_b[j] ? 1.f : t.w[at_b[j] + k];
            }
        }
    }
#pragma unroll
    for (int i = 0; i < (BACK ? 4 : 1); ++i) acc[0][i] = acc[1][i] = make_float2(0.f, 0.f);
    const float inv_dim = 1.0f / (float)p.head_dim;

    int stage = 0;
    for (unsigned block = cta; block < blocks; block += sp.ctas) {
        const unsigned token = block * sp.tokens + tl;
        const bool here = has_slot && token < p.tokens;
        const unsigned batch = here ? token / p.seq : 0, s = here ? token - batch * p.seq : 0;
        T* out = static_cast<T*>(t.out) + batch * t.out_batch + s * t.out_token + h0 * t.out_head;
        if (half_dim > 0) {
            if (block != cta) __syncthreads();                 // the angles before have been read
            for (int i = threadIdx.x; i < sp.tokens * half_dim; i += kHeadThreads) {
                const int k = i / half_dim, pair = i - k * half_dim;
                const unsigned tok = block * sp.tokens + k;
                if (tok < p.tokens) {
                    const unsigned b = tok / p.seq, at = tok - b * p.seq;
                    const RotaryAngles& a = p.angles;
                    const int64_t from = b * a.pos_batch + at * a.pos_token;
                    const double pos = a.positions == nullptr ? (double)at : a.axes != nullptr ? rotary_position<true>(a, from, pair)
                                                                                               : rotary_position<false>(a, from, pair);
                    turns[i] = rotary_turn(a, pos, pair);
                }
            }
            __syncthreads();
        }
        // What the rotation multiplies a channel and its partner with: a' = a c - b s, b' = b c + a s.  Forward with the weights in it.
        // (1, 0) for channels that are not rotated.
        float2 own[2][4], other[2][4];
#pragma unroll
        for (int j = 0; j < UNITS; ++j) {
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const int i = j * V + k;
                auto at = [](float2 (&v)[4], int n) -> float& { return n % 2 ? v[n / 2].y : v[n / 2].x; };
                if constexpr (TWO) {                           // pair i: a[i] with b[i]
                    const int u = ul + j * lanes;
                    const float2 c = here && u < rot_units ? turns[tl * half_dim + u * V + k] : make_float2(1.f, 0.f);
                    at(own[0], i) = at(own[1], i) = c.x;
                    at(other[0], i) = -c.y;
                    at(other[1], i) = c.y;
                } else if (k % 2 == 0) {                       // channel i with i + 1, in both runs
#pragma unroll
                    for (int run = 0; run < 2; ++run) {
                        const int pair = ((run ? at_b[j] : at_a[j]) + k) / 2;
                        const float2 c = here && pair < half_dim ? turns[tl * half_dim + pair] : make_float2(1.f, 0.f);
                        own[run][i / 2] = make_float2(c.x, c.x);
                        other[run][i / 2] = make_float2(-c.y, c.y);
                    }
                }
            }
        }
        if constexpr (!BACK) {
#pragma unroll
            for (int run = 0; run < 2; ++run)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    own[run][i] = fmul2(own[run][i], w[run][i]);
                    other[run][i] = fmul2(other[run][i], TWO ? w[1 - run][i] : make_float2(w[run][i].y, w[run][i].x));
                }
        }
        auto rotate = [&](float2 (&y)[2][4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float2 a = y[0][i], b = y[1][i];
                y[0][i] = ffma2(a, own[0][i], fmul2(TWO ? b : make_float2(a.y, a.x), other[0][i]));
                y[1][i] = ffma2(b, own[1][i], fmul2(TWO ? a : make_float2(b.y, b.x), other[1][i]));
            }
        };
        auto read = [&](int run, float2 (&v)[4]) {
            alignas(16) T e[8];
#pragma unroll
            for (int k = 0; k < Ring::pieces; ++k)
                reinterpret_cast<uint4*>(e)[k] =
                    *reinterpret_cast<const uint4*>(smem + threadIdx.x * 16 + stage * Ring::stage_bytes + (run * Ring::pieces + k) * kHeadThreads * 16);
            head_widen<T>(e, v);
        };
        for (int r = 0; r < rounds; ++r) {
            asm volatile("cp.async.wait_group %0;" ::"n"(Ring::stages - 2) : "memory");
            float2 v[2][4], d[2][BACK ? 4 : 1], tx[2][BACK ? 4 : 1];
            float sums[BACK ? 2 : 1];                          // of x^2, of u x
            read(0, v[0]);
            read(1, v[1]);
            float2 sq = fmul2(v[0][0], v[0][0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) sq = ffma2(v[0][i], v[0][i], sq);
#pragma unroll
            for (int i = 0; i < 4; ++i) sq = ffma2(v[1][i], v[1][i], sq);
            sums[0] = sq.x + sq.y;
            if constexpr (BACK) {
                read(2, d[0]);
                read(3, d[1]);
                rotate(d);                                     // (the sine is negated)
                float2 dot = make_float2(0.f, 0.f);
#pragma unroll
                for (int run = 0; run < 2; ++run)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        tx[run][i] = fmul2(d[run][i], v[run][i]);
                        dot = ffma2(tx[run][i], w[run][i], dot);
                    }
                sums[1] = dot.x + dot.y;
            }
            stage = stage + 1 == Ring::stages ? 0 : stage + 1;
            fetch();                                           // into the slot that the round before has read
            head_sum<LANES>(sums, lane, lanes, top);
            const float rstd = rsqrtf(fmaf(sums[0], inv_dim, p.eps));
            const float2 r2 = make_float2(rstd, rstd);
            const bool ok = here && (LANES > 0 || h0 + r * sp.head_lanes < t.heads);
            if constexpr (BACK) {
                // A head that is not there is zeros, and with eps = 0 its rstd an infinity: it adds 0 * 0, not 0 * inf.
                const float there = ok ? rstd : 0.f;
                const float2 there2 = make_float2(there, there);
                const float c = -rstd * (rstd * rstd * (sums[1] * inv_dim));
                const float2 c2 = make_float2(c, c);
#pragma unroll
                for (int run = 0; run < 2; ++run)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        acc[run][i] = ffma2(tx[run][i], there2, acc[run][i]);
                        v[run][i] = ffma2(d[run][i], fmul2(w[run][i], r2), fmul2(v[run][i], c2));
                    }
            } else {
#pragma unroll
                for (int run = 0; run < 2; ++run)
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[run][i] = fmul2(v[run][i], r2);
                rotate(v);
            }
            alignas(16) T a[8], b[8];
            head_narrow<T>(v[0], a);
            head_narrow<T>(v[1], b);
#pragma unroll
            for (int j = 0; j < UNITS; ++j) {
                if (ok && has_a[j]) *reinterpret_cast<Raw*>(out + at_a[j]) = *reinterpret_cast<const Raw*>(a + j * V);
                if (ok && has_b[j]) *reinterpret_cast<Raw*>(out + at_b[j]) = *reinterpret_cast<const Raw*>(b + j * V);
            }
            out += sp.head_lanes * t.out_head;
        }
        if constexpr (!BACK) break;                            // (one block a CTA)
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    if constexpr (BACK) {
        if (p.part == nullptr) return;
        // over the CTA's groups in order
        float* sum = reinterpret_cast<float*>(smem);
        __syncthreads();
        if (group < groups) {
#pragma unroll
            for (int j = 0; j < UNITS; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    const int i = j * V + k;
                    if (has_a[j]) sum[slot * p.head_dim + at_a[j] + k] = i % 2 ? acc[0][i / 2].y : acc[0][i / 2].x;
                    if (has_b[j]) sum[slot * p.head_dim + at_b[j] + k] = i % 2 ? acc[1][i / 2].y : acc[1][i / 2].x;
                }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < p.head_dim; c += kHeadThreads) {
            float a = 0.f;
            for (int k = 0; k < sp.tokens * sp.head_lanes; ++k) a += sum[k * p.head_dim + c];
            p.part[(int64_t)blockIdx.x * p.head_dim + c] = a;
        }
    }
}

// dw from the CTAs' sums, 8 columns (a sector) a CTA, in a fixed order; blockIdx.y: queries, keys
constexpr int kHeadSumThreads = 512, kHeadSumColumns = 8;
__global__ void __launch_bounds__(kHeadSumThreads)
head_norm_sum_kernel(const float* __restrict__ part, int q_parts, int k_parts, float* __restrict__ dq, float* __restrict__ dk, int dim) {
    constexpr int ROWS = kHeadSumThreads / kHeadSumColumns;
    __shared__ float red[kHeadSumThreads / 32][kHeadSumColumns];
    const int col = threadIdx.x % kHeadSumColumns, row = threadIdx.x / kHeadSumColumns;
    const int c = blockIdx.x * kHeadSumColumns + col;
    float* out = blockIdx.y == 0 ? dq : dk;
    pdl_wait();
    pdl_release();
    if (out == nullptr) return;
    const int first = blockIdx.y == 0 ? 0 : q_parts, last = blockIdx.y == 0 ? q_parts : q_parts + k_parts;
    float a = 0.f;
    if (c < dim) {
#pragma unroll 8
        for (int k = first + row; k < last; k += ROWS) a += part[(int64_t)k * dim + c];
    }
#pragma unroll
    for (int o = 16; o >= kHeadSumColumns; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    if ((threadIdx.x & 31) < kHeadSumColumns) red[threadIdx.x >> 5][col] = a;
    __syncthreads();
    if (threadIdx.x < kHeadSumColumns && c < dim) {
#pragma unroll
        for (int k = 1; k < kHeadSumThreads / 32; ++k) a += red[k][col];
        out[c] = a;
    }
}

template <typename T, int V, bool TWO, bool BACK>
static int launch_head_norm_as(const HeadNormParams& p, float* dqw, float* dkw, cudaStream_t st) {
    constexpr int UNITS = 8 / V;
    // units of a head: those that are rotated, and the rest (TWO); else pairs of runs
    const int units = TWO ? p.rotary_dim / 2 / V + (p.head_dim - p.rotary_dim + 2 * V - 1) / (2 * V) : (p.head_dim + 2 * V - 1) / (2 * V);
    HeadLanes l;
    l.lanes = (units + UNITS - 1) / UNITS;
    l.groups = 32 / l.lanes;
    const int slots = kHeadThreads / 32 * l.groups;
    const int room = p.rotary_dim > 0 ? 24 * 1024 / (4 * p.rotary_dim) : slots;
    const bool sums = BACK && p.part != nullptr;
    const int all = p.t[0].heads + p.t[1].heads;
    const int most = kHeadSumCtas * gemm_num_sms() < kHeadMaxCtas ? kHeadSumCtas * gemm_num_sms() : kHeadMaxCtas;
    size_t smem = 0;                                           // angles; the sums take the ring's place (at most 8 KB)
    for (int i = 0; i < 2; ++i) {
        const int heads = p.t[i].heads;
        HeadSplit& sp = l.of[i];
        sp = {1, 1, 0};
        if (heads == 0) continue;
        int per_thread = kHeadRows;
        auto lanes = [&](int n) { const int want = (heads + n - 1) / n; return want < slots ? want : slots; };
        while (per_thread > 1 && (p.tokens + slots / lanes(per_thread) - 1) / (slots / lanes(per_thread)) < (unsigned)gemm_num_sms()) --per_thread;
        // A number of heads a thread near that one which leaves no thread without a head in the last round: the forms for whole heads need it, and
        // it saves the idle ones.  6144 tokens, forward and backward, us: 40 heads of 128 28.6 -> 22.5 and 54.7 -> 48.1, 72 of 64 24.4 -> 21.3 and
        // 47.7 -> 43.8, 44 of 64 18.6 -> 14.9 and 34.1 -> 27.4, 26 of 128 20.6 -> 18.1 and 39.6 -> 34.7; none near 17 heads.
        auto whole = [&](int n) { return heads % lanes(n) == 0; };
        int near = per_thread;
        while (near > 1 && near > per_thread / 2 && !whole(near)) --near;
        if (!whole(near)) {
            for (near = per_thread; near < 2 * per_thread && !whole(near);) ++near;
            if (!whole(near) || (p.tokens + slots / lanes(near) - 1) / (slots / lanes(near)) < (unsigned)gemm_num_sms()) near = per_thread;
        }
        sp.head_lanes = lanes(near);
        sp.tokens = slots / sp.head_lanes;
        if (sp.tokens > room) sp.tokens = room;
        const unsigned blocks = (p.tokens + sp.tokens - 1) / sp.tokens;
        const unsigned share = (unsigned)((int64_t)most * heads / all);        // of the CTAs that the sums allow
        sp.ctas = (int)(sums && blocks > share ? (share > 0 ? share : 1) : blocks);
        const size_t angles = (size_t)sp.tokens * p.rotary_dim * 4;
        if (smem < angles) smem = angles;
    }
    const unsigned grid = (unsigned)(l.of[0].ctas + l.of[1].ctas);
    auto kern = head_norm_kernel<T, V, TWO, BACK, 0>;
    int form = 0;
    if constexpr (V * sizeof(T) == 16) {                       // the common heads of 64, 128 and 256 channels
        bool whole = p.head_dim == kHeadChannels * l.lanes;
        for (int i = 0; i < 2; ++i)
            whole = whole && (p.t[i].heads == 0 || (p.t[i].heads % l.of[i].head_lanes == 0 && aligned16(p.t[i].w)));
        if (whole && l.lanes == 4) { kern = head_norm_kernel<T, V, TWO, BACK, 4>; form = 1; }
        if (whole && l.lanes == 8) { kern = head_norm_kernel<T, V, TWO, BACK, 8>; form = 2; }
        if (whole && l.lanes == 16) { kern = head_norm_kernel<T, V, TWO, BACK, 16>; form = 3; }
    }
    // All of these kernels ask for the whole of an SM's shared memory, since an SM keeps what it set aside for a kernel until that has left:
    // a backward pass that came in beside the last CTAs of the forward pass (1/6 of an SM each) had room for fewer CTAs until its
    // own end, and both together took 192 us in the place of 166 (16384 x 40 x 128).
    static std::atomic<uint64_t> smem_done[4] = {};
    if (int rc = allow_dynamic_smem((const void*)kern, HeadRing<T, BACK>::bytes + 24 * 1024, smem_done[form], true)) return rc;
    Q8K_CUDA_OK(launch_dependent(kern, grid, kHeadThreads, HeadRing<T, BACK>::bytes + smem, st, 1, p, l));
    if (sums) {
        static std::atomic<uint64_t> sum_done{0};
        if (int rc = allow_dynamic_smem((const void*)head_norm_sum_kernel, 0, sum_done, true)) return rc;
        Q8K_CUDA_OK(launch_dependent(head_norm_sum_kernel, dim3((unsigned)((p.head_dim + kHeadSumColumns - 1) / kHeadSumColumns), 2), kHeadSumThreads, 0, st, 1, p.part, l.of[0].ctas,
                                     l.of[1].ctas, dqw, dkw, p.head_dim));
    }
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
    p.tokens = (unsigned)batch * (unsigned)seq;
    p.seq = (unsigned)seq; p.head_dim = head_dim; p.rotary_dim = rotary_dim; p.half = half_layout != 0;
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
    return head_dim <= 0 ? 0 : ((size_t)q8k::kHeadMaxCtas + 2) * (size_t)head_dim * sizeof(float);
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
