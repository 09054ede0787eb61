// Rotary embedding of queries and keys from positions: pair i of a head's first `rotary_dim` channels is turned by the angle
// position * freq[i] and scaled by `amplitude`; the other channels are copied.
//   a' = amplitude (a cos - b sin),  b' = amplitude (b cos + a sin)
// with (a, b) = channels (2i, 2i + 1) in the interleaved layout and (i, i + rotary_dim / 2) in the half layout.  The backward pass is the
// same kernel with the angle negated.
//
// Bound by HBM: every element of q and k is read and written once, in one launch, and no table is read.  The angles are
// computed here, once per token and pair, and shared by all heads through shared memory.  A position of a million radians has
// no correct digit in fp32 after its reduction, so position * freq / (2 pi) is formed in fp64, the whole turns are dropped there, and
// sine and cosine are taken of the rest, at most half a turn, in fp32.

#include <math_constants.h>
#include "common.cuh"

namespace q8k {

struct RotaryTensor {
    const void* in;
    void* out;
    int64_t in_batch, in_token, in_head, out_batch, out_token, out_head;       // strides in elements; channels are contiguous
    int heads;
};

struct RotaryParams {
    RotaryTensor q, k;
    const void* positions;                   // null: 0, 1, ... of each batch entry
    int positions64;                         // int64 rather than int32
    int64_t pos_batch, pos_token;
    const double* freq;
    float amplitude, sign;
    int64_t tokens;                          // batch * seq
    int seq, head_dim, rotary_dim, half;     // half: layout
};

constexpr int kRotaryThreads = 256;
constexpr int kRotaryMaxDim = 4096;

// V channels at a time where everything is 16-byte aligned (VEC), one pair at a time otherwise.  A CTA takes `tpc` consecutive tokens.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kRotaryThreads)
rotary_kernel(const __grid_constant__ RotaryParams p, int tpc) {
    extern __shared__ float2 turns[];                          // [tpc][rotary_dim / 2] cosine, sine
    constexpr int V = VEC ? 16 / sizeof(T) : 1;
    const int half_dim = p.rotary_dim / 2;
    const int64_t token0 = (int64_t)blockIdx.x * tpc;
    const int nt = (int)(p.tokens - token0 < tpc ? p.tokens - token0 : tpc);
    pdl_wait();
    pdl_release();

    for (int i = threadIdx.x; i < nt * half_dim; i += kRotaryThreads) {
        const int tl = i / half_dim, pair = i - tl * half_dim;
        const int64_t token = token0 + tl;
        const int64_t batch = token / p.seq, s = token - batch * p.seq;
        int64_t pos = s;
        if (p.positions != nullptr) {
            const int64_t at = batch * p.pos_batch + s * p.pos_token;
            pos = p.positions64 ? static_cast<const int64_t*>(p.positions)[at] : (int64_t)static_cast<const int32_t*>(p.positions)[at];
        }
        const double t = (double)pos * (p.freq[pair] * 0.15915494309189535);   // 1 / (2 pi)
        float sn, cs;
        sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
        turns[i] = make_float2(cs * p.amplitude, sn * p.amplitude * p.sign);
    }
    __syncthreads();

    // units of a head: in the half layout V pairs (two runs of V channels), in the interleaved one V / 2 pairs (one run;
    // VEC = false: the pair); then the channels behind the rotated ones, V at a time
    const int rot_units = p.half || !VEC ? half_dim / V : p.rotary_dim / V;
    const int units = rot_units + (p.head_dim - p.rotary_dim) / V;
    const int heads = p.q.heads + p.k.heads;
    const int per_token = heads * units;
    for (int i = threadIdx.x; i < nt * per_token; i += kRotaryThreads) {
        const int tl = i / per_token;
        const int r = i - tl * per_token;
        const int h = r / units, u = r - h * units;
        const int64_t token = token0 + tl;
        const int64_t batch = token / p.seq, s = token - batch * p.seq;
        const bool is_q = h < p.q.heads;
        const RotaryTensor& a = is_q ? p.q : p.k;
        const int hl = is_q ? h : h - p.q.heads;
        const T* in = static_cast<const T*>(a.in) + batch * a.in_batch + s * a.in_token + hl * a.in_head;
        T* out = static_cast<T*>(a.out) + batch * a.out_batch + s * a.out_token + hl * a.out_head;
        const float2* cs = turns + tl * half_dim;
        if (u >= rot_units) {
            const int c = p.rotary_dim + (u - rot_units) * V;
            if constexpr (VEC) *reinterpret_cast<uint4*>(out + c) = *reinterpret_cast<const uint4*>(in + c);
            else out[c] = in[c];
        } else if constexpr (!VEC) {
            const int c0 = p.half ? u : 2 * u, c1 = p.half ? u + half_dim : 2 * u + 1;
            const float x = to_float<T>(in[c0]), y = to_float<T>(in[c1]);
            out[c0] = from_float<T>(x * cs[u].x - y * cs[u].y);
            out[c1] = from_float<T>(y * cs[u].x + x * cs[u].y);
        } else if (p.half) {
            const int c = u * V;
            float x[V], y[V], ox[V], oy[V];
            load_vec<T, V>(in + c, x);
            load_vec<T, V>(in + c + half_dim, y);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 w = cs[c + j];
                ox[j] = x[j] * w.x - y[j] * w.y;
                oy[j] = y[j] * w.x + x[j] * w.y;
            }
            store_vec<T, V>(out + c, ox);
            store_vec<T, V>(out + c + half_dim, oy);
        } else {
            const int c = u * V;
            float x[V], o[V];
            load_vec<T, V>(in + c, x);
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 w = cs[(c + j) / 2];
                o[j] = x[j] * w.x - x[j + 1] * w.y;
                o[j + 1] = x[j + 1] * w.x + x[j] * w.y;
            }
            store_vec<T, V>(out + c, o);
        }
    }
}

template <typename T> static int launch_rotary(const RotaryParams& p, bool vec, cudaStream_t st) {
    // tokens per CTA: about four units of work a thread, but no fewer CTAs than SMs
    const int v = vec ? (int)(16 / sizeof(T)) : 1;
    const int64_t per_token = (int64_t)(p.q.heads + p.k.heads) * (p.head_dim / v);
    int64_t tpc = (4 * kRotaryThreads + per_token - 1) / per_token;
    const int64_t spread = (p.tokens + gemm_num_sms() - 1) / gemm_num_sms();
    if (tpc > spread) tpc = spread;
    const int64_t room = 32 * 1024 / (4 * p.rotary_dim);      // shared memory: 4 bytes times rotary_dim per token, up to 32 KB
    if (tpc > room) tpc = room;
    if (tpc < 1) tpc = 1;
    const int64_t grid = (p.tokens + tpc - 1) / tpc;
    Q8K_REQUIRE(grid <= 0x7fffffffLL, Q8K_ERR_TOO_LARGE, "rotary: %lld tokens", (long long)p.tokens);
    auto kern = vec ? rotary_kernel<T, true> : rotary_kernel<T, false>;
    Q8K_CUDA_OK(launch_dependent(kern, (unsigned)grid, kRotaryThreads, (size_t)tpc * p.rotary_dim * 4, st, 1, p, (int)tpc));
    return Q8K_OK;
}

}  // namespace q8k

using namespace q8k;

extern "C" int q8k_rotary(const void* q, const int64_t q_strides[3], void* q_out, const int64_t q_out_strides[3], int q_heads,
                          const void* k, const int64_t k_strides[3], void* k_out, const int64_t k_out_strides[3], int k_heads,
                          int dtype, const void* positions, int positions_int64, int64_t position_batch_stride,
                          int64_t position_token_stride, const double* frequencies, float amplitude, int batch, int seq, int head_dim,
                          int rotary_dim, int half_layout, int backward, void* stream) {
    const char* op = "rotary";
    Q8K_REQUIRE(batch >= 0 && seq >= 0 && q_heads >= 0 && k_heads >= 0, Q8K_ERR_INVALID_ARG, "%s: negative size", op);
    Q8K_REQUIRE(rotary_dim >= 2 && rotary_dim % 2 == 0 && rotary_dim <= head_dim, Q8K_ERR_INVALID_ARG,
                "%s: rotary_dim %d must be even and between 2 and the head dim %d", op, rotary_dim, head_dim);
    Q8K_REQUIRE(head_dim <= kRotaryMaxDim, Q8K_ERR_UNSUPPORTED, "%s: head dim %d exceeds %d", op, head_dim, kRotaryMaxDim);
    Q8K_REQUIRE((int64_t)(q_heads + (int64_t)k_heads) * head_dim <= (1 << 24), Q8K_ERR_UNSUPPORTED, "%s: %d + %d heads of %d are too many",
                op, q_heads, k_heads, head_dim);
    const int size = dtype_size(dtype);
    Q8K_REQUIRE(dtype == Q8K_DT_F32 || dtype == Q8K_DT_F16 || dtype == Q8K_DT_BF16, Q8K_ERR_UNSUPPORTED,
                "%s: dtype %d is not float32, float16 or bfloat16", op, dtype);
    if (batch == 0 || seq == 0 || q_heads + k_heads == 0) return Q8K_OK;
    Q8K_REQUIRE(frequencies != nullptr && reinterpret_cast<uintptr_t>(frequencies) % 8 == 0, Q8K_ERR_INVALID_ARG,
                "%s: null or misaligned frequencies", op);
    Q8K_REQUIRE(reinterpret_cast<uintptr_t>(positions) % (positions_int64 ? 8 : 4) == 0, Q8K_ERR_INVALID_ARG,
                "%s: misaligned positions", op);
    RotaryParams p = {};
    const int v = 16 / size;
    bool vec = head_dim % v == 0 && rotary_dim % v == 0 && (!half_layout || (rotary_dim / 2) % v == 0);
    auto tensor = [&](RotaryTensor& t, const void* in, const int64_t* is, void* out, const int64_t* os, int heads) {
        t.heads = heads;
        if (heads == 0) return true;
        if (in == nullptr || out == nullptr || is == nullptr || os == nullptr || reinterpret_cast<uintptr_t>(in) % size ||
            reinterpret_cast<uintptr_t>(out) % size)
            return false;
        t.in = in; t.out = out;
        t.in_batch = is[0]; t.in_token = is[1]; t.in_head = is[2];
        t.out_batch = os[0]; t.out_token = os[1]; t.out_head = os[2];
        vec = vec && aligned16(in) && aligned16(out);
        const int64_t n[3] = {batch, seq, heads};              // a stride over one element does not matter
        for (int i = 0; i < 3; ++i) vec = vec && (n[i] == 1 || (is[i] % v == 0 && os[i] % v == 0));
        return true;
    };
    Q8K_REQUIRE(tensor(p.q, q, q_strides, q_out, q_out_strides, q_heads) && tensor(p.k, k, k_strides, k_out, k_out_strides, k_heads),
                Q8K_ERR_INVALID_ARG, "%s: null or misaligned pointer", op);
    p.positions = positions;
    p.positions64 = positions_int64 != 0;
    p.pos_batch = position_batch_stride;
    p.pos_token = position_token_stride;
    p.freq = frequencies;
    p.amplitude = amplitude;
    p.sign = backward ? -1.f : 1.f;
    p.tokens = (int64_t)batch * seq;
    p.seq = seq; p.head_dim = head_dim; p.rotary_dim = rotary_dim; p.half = half_layout != 0;
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == Q8K_DT_BF16) return launch_rotary<__nv_bfloat16>(p, vec, st);
    if (dtype == Q8K_DT_F16) return launch_rotary<__half>(p, vec, st);
    return launch_rotary<float>(p, vec, st);
}
