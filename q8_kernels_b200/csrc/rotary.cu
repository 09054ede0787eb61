// Rotary embedding of queries and keys from positions: pair i of a head's first `rotary_dim` channels is turned by the angle
// position * freq[i] and scaled by `amplitude`; the other channels are copied.
//   a' = amplitude (a cos - b sin),  b' = amplitude (b cos + a sin)
// with (a, b) = channels (2i, 2i + 1) in the interleaved layout and (i, i + rotary_dim / 2) in the half layout.  The backward pass is the
// same kernel with the angle negated.  With several axes a pair takes the position of its own one.
//
// Bound by HBM: every element of q and k is read and written once, in one launch, and no table is read.  The angles are
// computed here, once per token and pair (rotary.cuh), and shared by the heads through shared memory.
//
// What is left to save are instructions: at the copy rate an SM has some 15 for an element.  So a thread takes the same channels of
// eight heads of one token, up to sixteen where that leaves fewer threads idle (launch_rotary_as), fewer in short calls: its cosines and
// sines come from shared memory once, and its addresses advance by the head's stride.
// CTAs of 128 threads, eight an SM: the chain from position to sine hides behind the first loads and behind other CTAs' stores, and the
// last ones to finish are short.  Measured (bf16, CUDA graphs): 6144 tokens x 64 heads x 64 interleaved 16.3 us (0.94 of the copy rate),
// 16384 x 40 x 128 half 53.7 us (0.95), interleaved 52.3 (0.98).  Tried, when these took 17.5 and 61.6: six CTAs without spills (17.9, 64.3), one head's loads at a
// time (19.8, 65.2), a thread for one unit with the next token's elements on their way meanwhile (30.9, 103).

#include <type_traits>
#include "rotary.cuh"

namespace q8k {

struct RotaryTensor {
    const void* in;
    void* out;
    int64_t in_batch, in_token, in_head, out_batch, out_token, out_head;       // strides in elements; channels are contiguous
    int heads;
};

struct RotaryParams {
    RotaryTensor q, k;
    RotaryAngles angles;
    int64_t tokens;                          // batch * seq
    int seq, head_dim, rotary_dim, half;     // half: layout
};

constexpr int kRotaryMaxDim = 4096;
constexpr int kRotaryThreads = 128;
constexpr int kRotaryWave = 4;               // CTAs an SM that more heads a thread have to leave, half of what it holds at once
constexpr int kRotaryHeads = 8;              // heads of a thread, where there are threads for the others

// How a CTA's threads are laid out over its tokens: unit_lanes threads for the units of a head, head_lanes for the heads.
struct RotaryLanes { int units, unit_lanes, head_lanes, tokens; };

template <int BYTES> struct RotaryRaw;
template <> struct RotaryRaw<2>  { using type = uint16_t; };
template <> struct RotaryRaw<4>  { using type = uint32_t; };
template <> struct RotaryRaw<8>  { using type = uint2; };
template <> struct RotaryRaw<16> { using type = uint4; };

// V channels at a time, all accesses aligned to them.  TWO: a pair's channels lie apart (half layout, or V = 1), so a unit is V pairs in
// two runs of V channels; otherwise V / 2 pairs in one.  PART: there are channels behind the rotated ones, whose units copy one or two
// runs.  AXES: positions with several axes.
template <typename T, int V, bool TWO, bool PART, bool AXES>
__global__ void __launch_bounds__(kRotaryThreads, TWO && PART ? 6 : 8)
rotary_kernel(const __grid_constant__ RotaryParams p, const RotaryLanes l) {
    constexpr int PAIRS = TWO ? V : V / 2;
    constexpr int AHEAD = TWO ? 2 : 4;                         // heads whose loads are on their way together
    using Raw = typename RotaryRaw<V * sizeof(T)>::type;
    union Elems { Raw r; T e[V]; };
    extern __shared__ float2 turns[];                          // [tokens][rotary_dim / 2] cosine, sine
    const int half_dim = p.rotary_dim / 2;
    const int per_token = l.unit_lanes * l.head_lanes;
    const int tl = threadIdx.x / per_token, rest = threadIdx.x - tl * per_token;
    const unsigned token = blockIdx.x * (unsigned)l.tokens + (unsigned)tl;
    const unsigned batch = token / (unsigned)p.seq, s = token - batch * (unsigned)p.seq;
    const bool here = tl < l.tokens && token < (unsigned)p.tokens;
    pdl_wait();
    pdl_release();

    const int h0 = rest / l.unit_lanes;
    const int rot_units = half_dim / PAIRS;
    using Batch = Elems[AHEAD];
    auto fetch = [](Batch& x, Batch& y, const T*& in, int64_t step, int n, int next, bool second) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            if (k < n) {
                x[k].r = *reinterpret_cast<const Raw*>(in);
                if (second) y[k].r = *reinterpret_cast<const Raw*>(in + next);
                in += step;
            }
        }
    };
    auto left = [&](const RotaryTensor& a, int h) { return (a.heads - h + l.head_lanes - 1) / l.head_lanes; };
    auto start_of = [&](const RotaryTensor& a, int h, int c) {
        return static_cast<const T*>(a.in) + batch * a.in_batch + s * a.in_token + h * a.in_head + c;
    };
    // The first heads of q are on their way while the angles are made: 61.6 -> 55.5 and 17.5 -> 16.3 us; 6144 x 64 x 128 with 64 channels
    // rotated 41.9 -> 36.5 half, 41.1 -> 33.1 interleaved.  (Behind: 6164 tokens, 6 heads of 192 in 4-byte accesses 12.4 -> 13.4.)
    const int u0 = rest - h0 * l.unit_lanes;
    Batch x, y;
    const bool early = here && u0 < l.units && h0 < p.q.heads;
    if (early) {
        const bool copy = TWO && PART && u0 >= rot_units;
        const int c = V == 1 && !p.half ? 2 * u0 : copy ? 2 * u0 * V : u0 * V;
        const T* in = start_of(p.q, h0, c);
        fetch(x, y, in, l.head_lanes * p.q.in_head, left(p.q, h0), copy ? V : p.half ? half_dim : 1, TWO && (!copy || c + V < p.head_dim));
    }
    if (here) {                                                // a token's threads make its angles
        const RotaryAngles& a = p.angles;
        const int64_t at = batch * a.pos_batch + s * a.pos_token;
        double pos = (double)s;
        if (!AXES && a.positions != nullptr) pos = rotary_position<false>(a, at, 0);
        for (int i = rest; i < half_dim; i += per_token) {
            if constexpr (AXES) pos = rotary_position<true>(a, at, i);
            turns[tl * half_dim + i] = rotary_turn(a, pos, i);
        }
    }
    __syncthreads();
    if (!here) return;

    for (int u = u0; u < l.units; u += l.unit_lanes) {
        const bool copy = PART && u >= rot_units;
        const int c = TWO && copy ? 2 * u * V : V == 1 && !p.half ? 2 * u : u * V;
        const int next = copy ? V : p.half ? half_dim : 1;     // from a unit's first run to its second
        const bool second = TWO && (!copy || c + V < p.head_dim);
        float2 w[PAIRS];
#pragma unroll
        for (int j = 0; j < PAIRS; ++j) w[j] = copy ? make_float2(1.f, 0.f) : turns[tl * half_dim + u * PAIRS + j];
        auto walk = [&](const RotaryTensor& a, int h, bool there) {      // heads h, h + head_lanes, ... of q or k
            const T* in = start_of(a, h, c);
            T* out = static_cast<T*>(a.out) + batch * a.out_batch + s * a.out_token + h * a.out_head + c;
            const int64_t in_step = l.head_lanes * a.in_head, out_step = l.head_lanes * a.out_head;
            while (h < a.heads) {
                const int n = left(a, h);                      // heads left
                if (there) in += AHEAD * in_step;
                else fetch(x, y, in, in_step, n, next, second);
                there = false;
#pragma unroll
                for (int k = 0; k < AHEAD; ++k) {
                    if (k >= n) break;
                    if (!copy) {
#pragma unroll
                        for (int j = 0; j < PAIRS; ++j) {
                            T& a0 = x[k].e[TWO ? j : 2 * j];
                            T& b0 = TWO ? y[k].e[j] : x[k].e[TWO ? 0 : 2 * j + 1];
                            const float f = to_float<T>(a0), g = to_float<T>(b0);
                            a0 = from_float<T>(f * w[j].x - g * w[j].y);
                            b0 = from_float<T>(g * w[j].x + f * w[j].y);
                        }
                    }
                    *reinterpret_cast<Raw*>(out) = x[k].r;
                    if (second) *reinterpret_cast<Raw*>(out + next) = y[k].r;
                    out += out_step;
                }
                h += AHEAD * l.head_lanes;
            }
        };
        // heads of k go on where those of q end, so that every lane has as many
        const int after = p.q.heads > h0 ? (p.q.heads - h0 + l.head_lanes - 1) / l.head_lanes * l.head_lanes + h0 : h0;
        walk(p.q, h0, early && u == u0);
        walk(p.k, after - p.q.heads, false);
    }
}

template <typename T, int V, bool TWO> static int launch_rotary_as(const RotaryParams& p, cudaStream_t st) {
    const int heads = p.q.heads + p.k.heads;
    RotaryLanes l;
    constexpr int run = TWO ? 2 * V : V;
    l.units = p.rotary_dim / 2 / (TWO ? V : V / 2) + (p.head_dim - p.rotary_dim + run - 1) / run;
    l.unit_lanes = l.units < kRotaryThreads ? l.units : kRotaryThreads;
    // kRotaryHeads heads a thread, up to twice as many where that leaves fewer threads idle and enough CTAs, fewer while
    // there are SMs without a CTA; then as many tokens as threads are left for.  (More heads, us: 16384 x 40 x 128 interleaved 62.7 -> 52.4, half
    // 56.0 -> 53.9, 8192 x 32 x 96 19.0 -> 17.9, 4096 x 48 x 128 half 19.2 -> 16.1; but 1023 x 32 x 72 in fewer CTAs 4.2 -> 5.6.)
    const int rest = kRotaryThreads / l.unit_lanes;
    int per_thread = kRotaryHeads;
    auto lanes = [&](int n) { const int want = (heads + n - 1) / n; return want < rest ? want : rest; };
    auto used = [&](int n) { return lanes(n) * (rest / lanes(n)); };
    for (int n = kRotaryHeads + 1; n <= 2 * kRotaryHeads; ++n)
        if (used(n) > used(per_thread) && p.tokens >= (int64_t)kRotaryWave * gemm_num_sms() * (rest / lanes(n))) per_thread = n;
    while (per_thread > 1 && (p.tokens + rest / lanes(per_thread) - 1) / (rest / lanes(per_thread)) < gemm_num_sms()) --per_thread;
    l.head_lanes = lanes(per_thread);
    l.tokens = rest / l.head_lanes;
    const int room = 24 * 1024 / (4 * p.rotary_dim);           // shared memory: 4 bytes times rotary_dim per token, up to 24 KB
    if (l.tokens > room) l.tokens = room;
    const int64_t grid = (p.tokens + l.tokens - 1) / l.tokens;
    const unsigned threads = (unsigned)((l.tokens * l.unit_lanes * l.head_lanes + 31) / 32 * 32);
    const bool part = p.rotary_dim < p.head_dim;
    auto kern = p.angles.axes != nullptr ? (part ? rotary_kernel<T, V, TWO, true, true> : rotary_kernel<T, V, TWO, false, true>)
                                         : (part ? rotary_kernel<T, V, TWO, true, false> : rotary_kernel<T, V, TWO, false, false>);
    Q8K_CUDA_OK(launch_dependent(kern, (unsigned)grid, threads, (size_t)l.tokens * p.rotary_dim * 4, st, 1, p, l));
    return Q8K_OK;
}

// v: channels that all accesses are aligned to, a power of two
template <typename T> static int launch_rotary(const RotaryParams& p, int v, cudaStream_t st) {
    if constexpr (sizeof(T) == 2) {
        if (v == 8) return p.half ? launch_rotary_as<T, 8, true>(p, st) : launch_rotary_as<T, 8, false>(p, st);
    }
    if (v >= 4) return p.half ? launch_rotary_as<T, 4, true>(p, st) : launch_rotary_as<T, 4, false>(p, st);
    if (v >= 2) return p.half ? launch_rotary_as<T, 2, true>(p, st) : launch_rotary_as<T, 2, false>(p, st);
    return launch_rotary_as<T, 1, true>(p, st);
}

// Whether a tensor may be rotated in its own place: one layout, whose heads do not overlap.  Every element is then read and written by
// one thread; with shared elements a thread would load what another has rotated already.
static bool rotary_in_place(const int64_t* in, const int64_t* out, const int64_t (&count)[3], int64_t head_dim) {
    int64_t extent = head_dim;
    int order[3], n = 0;
    for (int i = 0; i < 3; ++i) {
        if (count[i] == 1) continue;                           // a stride over one element does not matter
        if (in[i] != out[i]) return false;
        int at = n++;
        for (; at > 0 && in[order[at - 1]] > in[i]; --at) order[at] = order[at - 1];
        order[at] = i;
    }
    for (int k = 0; k < n; ++k) {                              // from the innermost out: each step beyond all that lies inside it
        const int64_t step = in[order[k]];
        if (step < extent) return false;
        extent += step * (count[order[k]] - 1);
    }
    return true;
}

static int rotary(const char* op, const void* q, const int64_t* q_strides, void* q_out, const int64_t* q_out_strides, int q_heads, const void* k,
                  const int64_t* k_strides, void* k_out, const int64_t* k_out_strides, int k_heads, int dtype, const RotaryAngles& angles,
                  int batch, int seq, int head_dim, int rotary_dim, int half_layout, cudaStream_t st) {
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
    for (int i = 0; i < 2; ++i) {
        const void *in = i ? k : q, *out = i ? k_out : q_out;
        const int64_t *is = i ? k_strides : q_strides, *os = i ? k_out_strides : q_out_strides;
        const int64_t count[3] = {batch, seq, i ? k_heads : q_heads};
        Q8K_REQUIRE(count[2] == 0 || in == nullptr || in != out || is == nullptr || os == nullptr || rotary_in_place(is, os, count, head_dim),
                    Q8K_ERR_INVALID_ARG, "%s: in place, %s needs the input's strides and heads that do not overlap", op, i ? "k" : "q");
    }
    if (int rc = rotary_check_angles(op, angles)) return rc;
    Q8K_REQUIRE((int64_t)batch * seq <= 0x7fffffffLL, Q8K_ERR_TOO_LARGE, "%s: %lld tokens", op, (long long)batch * seq);
    RotaryParams p = {};
    // the widest access, up to 16 bytes, that divides the channels, strides and addresses of all four tensors
    int v = 16 / size;
    auto divides = [&](int64_t n) { while (n % v != 0) v /= 2; };
    divides(head_dim);
    divides(rotary_dim);
    if (half_layout) divides(rotary_dim / 2);
    auto tensor = [&](RotaryTensor& t, const void* in, const int64_t* is, void* out, const int64_t* os, int heads) {
        t.heads = heads;
        if (heads == 0) return true;
        if (in == nullptr || out == nullptr || is == nullptr || os == nullptr || reinterpret_cast<uintptr_t>(in) % size ||
            reinterpret_cast<uintptr_t>(out) % size)
            return false;
        t.in = in; t.out = out;
        t.in_batch = is[0]; t.in_token = is[1]; t.in_head = is[2];
        t.out_batch = os[0]; t.out_token = os[1]; t.out_head = os[2];
        divides((int64_t)(reinterpret_cast<uintptr_t>(in) / size));
        divides((int64_t)(reinterpret_cast<uintptr_t>(out) / size));
        const int64_t n[3] = {batch, seq, heads};              // a stride over one element does not matter
        for (int i = 0; i < 3; ++i) {
            if (n[i] == 1) continue;
            divides(is[i]);
            divides(os[i]);
        }
        return true;
    };
    Q8K_REQUIRE(tensor(p.q, q, q_strides, q_out, q_out_strides, q_heads) && tensor(p.k, k, k_strides, k_out, k_out_strides, k_heads),
                Q8K_ERR_INVALID_ARG, "%s: null or misaligned pointer", op);
    p.angles = angles;
    p.tokens = (int64_t)batch * seq;
    p.seq = seq; p.head_dim = head_dim; p.rotary_dim = rotary_dim; p.half = half_layout != 0;
    if (dtype == Q8K_DT_BF16) return launch_rotary<__nv_bfloat16>(p, v, st);
    if (dtype == Q8K_DT_F16) return launch_rotary<__half>(p, v, st);
    return launch_rotary<float>(p, v, st);
}

}  // namespace q8k

extern "C" int q8k_rotary(const void* q, const int64_t q_strides[3], void* q_out, const int64_t q_out_strides[3], int q_heads,
                          const void* k, const int64_t k_strides[3], void* k_out, const int64_t k_out_strides[3], int k_heads,
                          int dtype, const void* positions, int positions_int64, int64_t position_batch_stride,
                          int64_t position_token_stride, const double* frequencies, float amplitude, int batch, int seq, int head_dim,
                          int rotary_dim, int half_layout, int backward, void* stream) {
    const q8k::RotaryAngles angles = {positions, positions_int64 ? Q8K_POS_I64 : Q8K_POS_I32, position_batch_stride, position_token_stride, 0,
                                      nullptr, 1, frequencies, amplitude, backward ? -1.f : 1.f};
    return q8k::rotary("rotary", q, q_strides, q_out, q_out_strides, q_heads, k, k_strides, k_out, k_out_strides, k_heads, dtype, angles, batch, seq,
                       head_dim, rotary_dim, half_layout, (cudaStream_t)stream);
}

extern "C" int q8k_axial_rotary(const void* q, const int64_t q_strides[3], void* q_out, const int64_t q_out_strides[3], int q_heads,
                                const void* k, const int64_t k_strides[3], void* k_out, const int64_t k_out_strides[3], int k_heads, int dtype,
                                const void* positions, int position_type, const int64_t position_strides[3], int n_axes, const int* axes,
                                const double* frequencies, float amplitude, int batch, int seq, int head_dim, int rotary_dim,
                                int half_layout, int backward, void* stream) {
    Q8K_REQUIRE(axes != nullptr && position_strides != nullptr, Q8K_ERR_INVALID_ARG, "axial_rotary: null axes or position strides");
    const q8k::RotaryAngles angles = {positions, position_type, position_strides[0], position_strides[1], position_strides[2],
                                      axes, n_axes, frequencies, amplitude, backward ? -1.f : 1.f};
    return q8k::rotary("axial_rotary", q, q_strides, q_out, q_out_strides, q_heads, k, k_strides, k_out, k_out_strides, k_heads, dtype, angles, batch,
                       seq, head_dim, rotary_dim, half_layout, (cudaStream_t)stream);
}
