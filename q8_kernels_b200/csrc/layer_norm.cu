// Layer norm over the last dim, forward and backward:
//   z = (x - mean) * rstd,  rstd = 1 / sqrt(mean((x - mean)^2) + eps),  y = z * w + b
//   dx = rstd * (g w - mean(g w) - z mean(g w z)),  dw = sum_rows g z,  db = sum_rows g
//
// Both passes are bound by HBM: the forward reads x and writes y, the backward reads x and g and writes dx.  Groups of T threads walk
// over rows, with w, b and the sums of dw and db in registers; G groups make a CTA.  A row has to be complete before its first output,
// so what keeps HBM busy are the next rows: they come by cp.async into a ring of S - 1 rows ahead in shared memory, where bytes on
// their way cost no registers.  What every thread does once a row (the exchange of the sums, addresses) is some 150 instructions, the
// rest 5 to 8 an element, so a thread has many elements of a row: 24 or 32, which few warps with many registers each allow; arithmetic
// is on packed pairs for the same reason.  24576 x 2048 bf16: forward 33.1 us (0.93 of the copy rate; with 16 elements a thread 36.5,
// with 64, w and b from L1, 46 to 51), backward 47.0 (0.98), with dw and db 54.8;  16384 x 1536 16.8, 25.0, 33.4 (16 elements: 22.6,
// 28.3, 38.3);  8192 x 1537 18.0, 19.7, 28.4 (20.2, 21.9, 29.8): single elements cost twice the instructions.
//
// The variance is taken from the differences to the mean, not E[x^2] - mean^2, which loses all digits of a row whose mean is large
// against its spread.  Sums, statistics and the gradients of w and b are fp32.
//
// Columns of a thread: VEC (dim a multiple of 8, all rows 16-byte aligned): items of 8 consecutive elements, which the thread copies
// and reads back itself, with no barrier.  Otherwise single elements T apart, the same in every row wherever the rows start (which the
// sums over rows need): the group copies the row in the 16-byte pieces of memory that it lies in, and reads elements after a barrier.

#include <type_traits>
#include "common.cuh"

namespace q8k {

constexpr int kLnItem = 8;
constexpr int kLnMaxDim = 16384;

// What thread `t` of a row's T threads owns in its item i: column of element j, and whether it exists.
template <int T, bool VEC> __device__ __forceinline__ int ln_col(int t, int i, int j) {
    return VEC ? (t + i * T) * kLnItem + j : t + (i * kLnItem + j) * T;
}
template <int T, bool VEC> __device__ __forceinline__ bool ln_has(int t, int i, int j, int dim) {
    return ln_col<T, VEC>(t, i, VEC ? 0 : j) < dim;
}

// An item as four packed pairs; columns that do not exist read as 0.
struct LnItem { float2 v[kLnItem / 2]; };

template <typename E, int T, bool VEC>
__device__ __forceinline__ LnItem ln_load(const E* row, int dim, int t, int i) {
    LnItem r;
    float v[kLnItem];
    if constexpr (VEC) {
        if (ln_has<T, VEC>(t, i, 0, dim)) load_vec<E, kLnItem>(row + ln_col<T, VEC>(t, i, 0), v);
        else {
#pragma unroll
            for (int j = 0; j < kLnItem; ++j) v[j] = 0.f;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kLnItem; ++j) v[j] = ln_has<T, VEC>(t, i, j, dim) ? to_float<E>(row[ln_col<T, VEC>(t, i, j)]) : 0.f;
    }
#pragma unroll
    for (int k = 0; k < kLnItem / 2; ++k) r.v[k] = make_float2(v[2 * k], v[2 * k + 1]);
    return r;
}

template <typename E, int T, bool VEC>
__device__ __forceinline__ void ln_store(E* row, int dim, int t, int i, const LnItem& r) {
    float v[kLnItem];
#pragma unroll
    for (int k = 0; k < kLnItem / 2; ++k) { v[2 * k] = r.v[k].x; v[2 * k + 1] = r.v[k].y; }
    if constexpr (VEC) {
        if (ln_has<T, VEC>(t, i, 0, dim)) store_vec<E, kLnItem>(row + ln_col<T, VEC>(t, i, 0), v);
    } else {
#pragma unroll
        for (int j = 0; j < kLnItem; ++j)
            if (ln_has<T, VEC>(t, i, j, dim)) row[ln_col<T, VEC>(t, i, j)] = from_float<E>(v[j]);
    }
}
__device__ __forceinline__ float2 pair_of(float v) { return make_float2(v, v); }

// Barrier of the T threads of one row group: its own named barrier where a CTA has several.
template <int T, int G> __device__ __forceinline__ void ln_group_sync(int group) {
    if constexpr (T <= 32) __syncwarp();
    else if constexpr (G == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(T) : "memory");
}

// Sum over the first WARPS (at most 32) lanes, in every lane of that power-of-two block.
template <int WARPS> __device__ __forceinline__ float ln_lane_sum(float v) {
#pragma unroll
    for (int o = WARPS / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

__device__ __forceinline__ void ln_copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void ln_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void ln_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Start the copy of a row into its slot of the ring.  [lo, hi) are the addresses of the tensor's first and behind its last element: a
// piece that reaches beyond them is copied by the element.
template <typename E, int ITEMS, int T, bool VEC>
__device__ __forceinline__ void ln_fetch(const E* row, int dim, int t, char* slot, const char* lo, const char* hi) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(slot);
    if constexpr (VEC) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int c = ln_col<T, VEC>(t, i, 0);
            if (c < dim) {
#pragma unroll
                for (int k = 0; k < (int)(kLnItem * sizeof(E) / 16); ++k)
                    ln_copy16(dst + c * (int)sizeof(E) + 16 * k, reinterpret_cast<const char*>(row + c) + 16 * k);
            }
        }
    } else {
        const char* first = reinterpret_cast<const char*>(row);
        const char* from = first - (reinterpret_cast<uintptr_t>(first) & 15);
        const int bytes = (int)(first - from) + dim * (int)sizeof(E);
        for (int k = t * 16; k < bytes; k += T * 16) {
            const char* p = from + k;
            if (p >= lo && p + 16 <= hi) {
                ln_copy16(dst + k, p);
            } else {
                for (int e = 0; e < 16; e += (int)sizeof(E))
                    if (p + e >= first && p + e < first + (int64_t)dim * (int)sizeof(E))
                        *reinterpret_cast<E*>(slot + k + e) = *reinterpret_cast<const E*>(p + e);
            }
        }
    }
}
// Where the row's first element lies in its slot.
template <typename E, bool VEC> __device__ __forceinline__ const E* ln_slot_row(const char* slot, const E* row) {
    return reinterpret_cast<const E*>(slot + (VEC ? 0 : reinterpret_cast<uintptr_t>(row) & 15));
}

// Threads of a CTA, CTAs an SM holds by registers, rows of the ring: as many as the SM's 227 KB leave for all of them, up to four.
template <int I, int T, int G> struct LnLayout { static constexpr int items = I, threads = T, rows = G, cta = T * G; };
// keep: w and b (backward: also z and g w) stay in registers; else, for rows of more than 8192 columns, they are read again, from L1 or
// from the ring, so that two such rows fit an SM at a time (forward), or one with the sums of dw and db (backward).  The ring has two
// rows then, which leaves L1 the room for w and b: with all that fit they came from L2, twice the bytes of the row itself.
template <typename L> struct LnForward {
    static constexpr bool keep = L::items <= 4;                // w and b in registers
    static constexpr int ctas = L::cta == 128 ? (L::items == 4 ? 3 : 4) : L::cta > 256 ? 1 : L::items <= 2 ? 3 : 2;
};
template <typename L> struct LnBackward {
    static constexpr bool keep = L::items <= 2 || L::cta <= 384;
    static constexpr int ctas = L::cta == 128 ? (L::items == 4 ? 3 : 4) : L::cta <= 256 && L::items <= 2 ? 2 : 1;
};
template <typename L, int CTAS, int BYTES> struct LnRing {
    static constexpr int row = L::rows * (L::threads * L::items * kLnItem * BYTES + 64);
    static constexpr int fit = 224 * 1024 / CTAS / row;
    static constexpr int most = L::items <= 2 || (L::cta <= 384 && L::items <= 4) ? 4 : 2;
    static constexpr int slots = fit > most ? most : fit < 1 ? 1 : fit;
};

// Mean and variance in one exchange between warps: each warp takes the mean of its own elements and the squares of their
// differences to that (shuffles), and with n_w elements, sum s_w and squares q_w the row has
//   mean = sum s_w / n,  n var = sum (q_w + n_w (s_w / n_w - mean)^2),
// all terms positive.
template <typename Tx, typename Ty, typename L, bool VEC>
__global__ void __launch_bounds__(L::cta, LnForward<L>::ctas)
layer_norm_kernel(const Tx* __restrict__ x, int64_t x_stride, const float* __restrict__ w, const float* __restrict__ b,
                  Ty* __restrict__ y, float* __restrict__ mean_out, float* __restrict__ rstd_out, int64_t rows, int dim, float eps,
                  int slot_bytes) {
    constexpr int ITEMS = L::items, T = L::threads, G = L::rows, WARPS = T / 32;
    constexpr int S = LnRing<L, LnForward<L>::ctas, sizeof(Tx)>::slots;
    constexpr bool KEEP = LnForward<L>::keep;
    extern __shared__ __align__(16) char ln_smem[];
    __shared__ float2 red[2][G][WARPS];
    const int group = threadIdx.x / T, t = threadIdx.x % T;
    char* ring = ln_smem + group * S * slot_bytes;
    const int64_t step = (int64_t)gridDim.x * G;
    const int64_t row0 = (int64_t)blockIdx.x * G + group;
    const char* lo = reinterpret_cast<const char*>(x);
    const char* hi = reinterpret_cast<const char*>(x + (rows - 1) * x_stride + dim);
    auto fetch = [&](int64_t row, int slot) {
        if (row < rows) ln_fetch<Tx, ITEMS, T, VEC>(x + row * x_stride, dim, t, ring + slot * slot_bytes, lo, hi);
        ln_commit();
    };
    auto weight = [&](int i) {
        LnItem r;
#pragma unroll
        for (int k = 0; k < kLnItem / 2; ++k) r.v[k] = pair_of(1.f);
        return w != nullptr ? ln_load<float, T, VEC>(w, dim, t, i) : r;
    };
    auto bias = [&](int i) {
        LnItem r;
#pragma unroll
        for (int k = 0; k < kLnItem / 2; ++k) r.v[k] = pair_of(0.f);
        return b != nullptr ? ln_load<float, T, VEC>(b, dim, t, i) : r;
    };
    pdl_wait();
    pdl_release();
#pragma unroll
    for (int k = 0; k < S - 1; ++k) fetch(row0 + k * step, k);
    LnItem wv[KEEP ? ITEMS : 1], bv[KEEP ? ITEMS : 1];
    if constexpr (KEEP) {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) { wv[i] = weight(i); bv[i] = bias(i); }
    }
    // elements of a warp: those of its threads (VEC: runs of 8 each, 256 from (warp * 32 + i * T) * 8 on; else 32 from warp * 32 on, T apart)
    auto count = [&](int wp) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if constexpr (VEC) {
                n += max(0, min(32 * kLnItem, dim - (wp * 32 + i * T) * kLnItem));
            } else {
#pragma unroll
                for (int j = 0; j < kLnItem; ++j) n += max(0, min(32, dim - wp * 32 - (i * kLnItem + j) * T));
            }
        }
        return (float)n;
    };
    const float inv = 1.0f / (float)dim;
    const float own_inv = 1.0f / fmaxf(1.f, count(t >> 5));
    const float lane_n = count((t & 31) % WARPS), lane_inv = 1.0f / fmaxf(1.f, lane_n);
    int slot = 0, turn = 0;
    for (int64_t row = row0; row < rows; row += step, turn ^= 1) {
        if constexpr (S == 1) {
            if (!VEC) ln_group_sync<T, G>(group);              // the row before has been read
            fetch(row, 0);
            ln_wait<0>();
        } else {
            ln_wait<S - 2>();
        }
        if (!VEC) ln_group_sync<T, G>(group);                  // everyone's pieces have landed; the slot before has been read
        const Tx* xr = ln_slot_row<Tx, VEC>(ring + slot * slot_bytes, x + row * x_stride);
        LnItem v[ITEMS];
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) v[i] = ln_load<Tx, T, VEC>(xr, dim, t, i);
        if constexpr (S > 1) fetch(row + (S - 1) * step, slot == 0 ? S - 1 : slot - 1);
        if (++slot == S) slot = 0;
        float2 s2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
#pragma unroll
            for (int k = 0; k < kLnItem / 2; ++k) s2 = fadd2(s2, v[i].v[k]);
        }
        const float s = warp_sum(s2.x + s2.y);
        float mean = s * (WARPS == 1 ? inv : own_inv);
        float2 q2 = make_float2(0.f, 0.f);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (!VEC || ln_has<T, VEC>(t, i, 0, dim)) {
#pragma unroll
                for (int k = 0; k < kLnItem / 2; ++k) {
                    float2 d = fsub2(v[i].v[k], pair_of(mean));
                    if constexpr (!VEC) {
                        if (!ln_has<T, VEC>(t, i, 2 * k, dim)) d.x = 0.f;
                        if (!ln_has<T, VEC>(t, i, 2 * k + 1, dim)) d.y = 0.f;
                    }
                    q2 = ffma2(d, d, q2);
                }
            }
        }
        float q = warp_sum(q2.x + q2.y);
        if constexpr (WARPS > 1) {
            if ((t & 31) == 0) red[turn][group][t >> 5] = make_float2(s, q);
            ln_group_sync<T, G>(group);                        // (two buffers: the one before is not written until the next barrier)
            const float2 p = red[turn][group][(t & 31) % WARPS];          // lane k, k + WARPS, ... take warp k's part
            mean = ln_lane_sum<WARPS>(p.x) * inv;
            const float d = fmaf(p.x, lane_inv, -mean);        // (a warp without elements has lane_n = 0)
            q = ln_lane_sum<WARPS>(fmaf(lane_n * d, d, p.y));
        }
        const float rstd = rsqrtf(fmaf(q, inv, eps));
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            if (!KEEP) { wv[0] = weight(i); bv[0] = bias(i); }
            LnItem o;
#pragma unroll
            for (int k = 0; k < kLnItem / 2; ++k)
                o.v[k] = ffma2(fmul2(fsub2(v[i].v[k], pair_of(mean)), pair_of(rstd)), wv[KEEP ? i : 0].v[k], bv[KEEP ? i : 0].v[k]);
            ln_store<Ty, T, VEC>(y + row * (int64_t)dim, dim, t, i, o);
        }
        if (t == 0) {
            if (mean_out != nullptr) mean_out[row] = mean;
            if (rstd_out != nullptr) rstd_out[row] = rstd;
        }
    }
    ln_wait<0>();                                              // (the copies behind the last row were empty)
}

// The groups of a CTA add their sums of g z and g in shared memory at the end, and part[CTA][2][dim] is summed over the CTAs by
// layer_norm_wgrad_kernel: fixed orders, no atomics, the same bits in every run.
template <typename Tx, typename Tg, typename L, bool VEC, bool WGRAD>
__global__ void __launch_bounds__(L::cta, LnBackward<L>::ctas)
layer_norm_backward_kernel(const Tx* __restrict__ x, int64_t x_stride, const Tg* __restrict__ g, const float* __restrict__ mean,
                           const float* __restrict__ rstd, const float* __restrict__ w, Tx* __restrict__ dx, float* __restrict__ part,
                           int64_t rows, int dim, int x_slot_bytes, int g_slot_bytes) {
    constexpr int ITEMS = L::items, T = L::threads, G = L::rows, WARPS = T / 32;
    constexpr int S = LnRing<L, LnBackward<L>::ctas, sizeof(Tx) + sizeof(Tg)>::slots;
    constexpr bool KEEP = LnBackward<L>::keep;
    extern __shared__ __align__(16) char ln_smem[];
    __shared__ float2 red[2][G][WARPS];
    const int group = threadIdx.x / T, t = threadIdx.x % T;
    char* x_ring = ln_smem + group * S * (x_slot_bytes + g_slot_bytes);
    char* g_ring = x_ring + S * x_slot_bytes;
    const int64_t step = (int64_t)gridDim.x * G;
    const int64_t row0 = (int64_t)blockIdx.x * G + group;
    const char* x_lo = reinterpret_cast<const char*>(x);
    const char* x_hi = reinterpret_cast<const char*>(x + (rows - 1) * x_stride + dim);
    const char* g_lo = reinterpret_cast<const char*>(g);
    const char* g_hi = reinterpret_cast<const char*>(g + rows * dim);
    auto fetch = [&](int64_t row, int slot) {
        if (row < rows) {
            ln_fetch<Tx, ITEMS, T, VEC>(x + row * x_stride, dim, t, x_ring + slot * x_slot_bytes, x_lo, x_hi);
            ln_fetch<Tg, ITEMS, T, VEC>(g + row * (int64_t)dim, dim, t, g_ring + slot * g_slot_bytes, g_lo, g_hi);
        }
        ln_commit();
    };
    auto weight = [&](int i) {
        LnItem r;
#pragma unroll
        for (int k = 0; k < kLnItem / 2; ++k) r.v[k] = pair_of(1.f);
        return w != nullptr ? ln_load<float, T, VEC>(w, dim, t, i) : r;
    };
    pdl_wait();
    pdl_release();
#pragma unroll
    for (int k = 0; k < S - 1; ++k) fetch(row0 + k * step, k);
    float m_next = 0.f, r_next = 0.f;
    if (row0 < rows) { m_next = mean[row0]; r_next = rstd[row0]; }
    LnItem wv[KEEP ? ITEMS : 1];
    LnItem dw[WGRAD ? ITEMS : 1], db[WGRAD ? ITEMS : 1];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
        if constexpr (WGRAD) {
#pragma unroll
            for (int k = 0; k < kLnItem / 2; ++k) dw[i].v[k] = db[i].v[k] = make_float2(0.f, 0.f);
        }
        if constexpr (KEEP) wv[i] = weight(i);
    }
    const float inv = 1.0f / (float)dim;
    int slot = 0, turn = 0;
    for (int64_t row = row0; row < rows; row += step, turn ^= 1) {
        if constexpr (S == 1) {
            if (!VEC) ln_group_sync<T, G>(group);              // the row before has been read
            fetch(row, 0);
            ln_wait<0>();
        } else {
            ln_wait<S - 2>();
        }
        if (!VEC) ln_group_sync<T, G>(group);                  // everyone's pieces have landed; the slot before has been read
        const Tx* xr = ln_slot_row<Tx, VEC>(x_ring + slot * x_slot_bytes, x + row * x_stride);
        const Tg* gr = ln_slot_row<Tg, VEC>(g_ring + slot * g_slot_bytes, g + row * (int64_t)dim);
        const float m = m_next, r = r_next;
        if (row + step < rows) { m_next = mean[row + step]; r_next = rstd[row + step]; }
        // z = x r - m r, one rounding more than (x - m) r would have only where x and m cancel: the difference is taken first
        auto normalised = [&](int i) {
            LnItem z = ln_load<Tx, T, VEC>(xr, dim, t, i);
#pragma unroll
            for (int k = 0; k < kLnItem / 2; ++k) z.v[k] = fmul2(fsub2(z.v[k], pair_of(m)), pair_of(r));
            return z;
        };
        LnItem z[KEEP ? ITEMS : 1], gw[KEEP ? ITEMS : 1];
        float2 s0 = make_float2(0.f, 0.f), s1 = s0;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int at = KEEP ? i : 0;
            z[at] = normalised(i);
            gw[at] = ln_load<Tg, T, VEC>(gr, dim, t, i);
            if (!KEEP) wv[0] = weight(i);
#pragma unroll
            for (int k = 0; k < kLnItem / 2; ++k) {            // columns that do not exist have g = 0: they add nothing
                if constexpr (WGRAD) {
                    dw[i].v[k] = ffma2(gw[at].v[k], z[at].v[k], dw[i].v[k]);
                    db[i].v[k] = fadd2(db[i].v[k], gw[at].v[k]);
                }
                gw[at].v[k] = fmul2(gw[at].v[k], wv[at].v[k]);
                s0 = fadd2(s0, gw[at].v[k]);
                s1 = ffma2(gw[at].v[k], z[at].v[k], s1);
            }
        }
        if constexpr (S > 1) fetch(row + (S - 1) * step, slot == 0 ? S - 1 : slot - 1);
        if (++slot == S) slot = 0;
        if (dx == nullptr) continue;                           // only the sums over rows are wanted
        float a = warp_sum(s0.x + s0.y), c = warp_sum(s1.x + s1.y);
        if constexpr (WARPS > 1) {
            if ((t & 31) == 0) red[turn][group][t >> 5] = make_float2(a, c);
            ln_group_sync<T, G>(group);                        // (two buffers: the one before is not written until the next barrier)
            const float2 p = red[turn][group][(t & 31) % WARPS];
            a = ln_lane_sum<WARPS>(p.x);
            c = ln_lane_sum<WARPS>(p.y);
        }
        a *= inv;
        c *= inv;
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int at = KEEP ? i : 0;
            if (!KEEP) {                                       // the slot is not refilled before the next row
                z[0] = normalised(i);
                gw[0] = ln_load<Tg, T, VEC>(gr, dim, t, i);
                wv[0] = weight(i);
#pragma unroll
                for (int k = 0; k < kLnItem / 2; ++k) gw[0].v[k] = fmul2(gw[0].v[k], wv[0].v[k]);
            }
            LnItem o;
#pragma unroll
            for (int k = 0; k < kLnItem / 2; ++k)
                o.v[k] = fmul2(fsub2(gw[at].v[k], ffma2(z[at].v[k], pair_of(c), pair_of(a))), pair_of(r));
            ln_store<Tx, T, VEC>(dx + row * (int64_t)dim, dim, t, i, o);
        }
    }
    ln_wait<0>();                                              // (the copies behind the last row were empty)
    if constexpr (WGRAD) {
        float* p = part + (int64_t)blockIdx.x * 2 * dim;
        if constexpr (G == 1) {
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                ln_store<float, T, VEC>(p, dim, t, i, dw[i]);
                ln_store<float, T, VEC>(p + dim, dim, t, i, db[i]);
            }
        } else {
            constexpr int W = T * kLnItem * ITEMS;             // columns of the layout, at least dim
            float* sums = reinterpret_cast<float*>(ln_smem);   // in the ring's place
            __syncthreads();
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                ln_store<float, T, VEC>(sums + group * 2 * W, W, t, i, dw[i]);
                ln_store<float, T, VEC>(sums + group * 2 * W + W, W, t, i, db[i]);
            }
            __syncthreads();
            for (int k = threadIdx.x; k < 2 * W; k += T * G) {
                const int which = k / W, c = k - which * W;
                if (c < dim) {
                    float s = sums[k];
#pragma unroll
                    for (int o = 1; o < G; ++o) s += sums[o * 2 * W + k];
                    p[which * dim + c] = s;
                }
            }
        }
    }
}

// dw[c] = sum over CTAs of part[CTA][0][c], db[c] likewise of part[CTA][1][c]: a CTA takes 32 of the 2 * dim columns, warp k the parts
// k, k + 32, ..., and the 32 sums are added by shuffles.
constexpr int kLnSumWarps = 32;
__global__ void __launch_bounds__(32 * kLnSumWarps)
layer_norm_wgrad_kernel(const float* __restrict__ part, int parts, float* __restrict__ dw, float* __restrict__ db, int dim) {
    __shared__ float sums[kLnSumWarps][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;
    pdl_wait();
    pdl_release();
    float s = 0.f;
    if (c < 2 * (int64_t)dim) {
#pragma unroll 10
        for (int k = warp; k < parts; k += kLnSumWarps) s += part[k * 2 * (int64_t)dim + c];
    }
    sums[warp][lane] = s;
    __syncthreads();
    s = warp_sum(sums[lane][warp]);                            // column `warp` of the 32
    const int64_t cw = (int64_t)blockIdx.x * 32 + warp;
    if (lane == 0 && cw < 2 * (int64_t)dim) {
        float* out = cw < dim ? dw : db;
        if (out != nullptr) out[cw < dim ? cw : cw - dim] = s;
    }
}

// ------------------------------------------------------------------ host side
// Layouts.  fp32 rows have twice the bytes for the same instructions, and above 768 columns 16 elements a thread do better with them
// (6144 x 2048: forward 17.7 us against 20.4 with 32, backward 24.7 against 29.7).
// Both sides of each limit: the layout that is taken at the widest rows it holds | the next one for the same rows.  us of the forward pass, of
// dx, and of dx with the sums, by columns; 24 million elements of bf16, 12 million of fp32:
//   bf16   256  20.8|22.4 31.3|31.7 34.9|38.1     512  15.7|18.0 25.1|24.7 29.8|33.4     768  15.1|17.5 23.1|24.4 29.9|33.1
//         1024  15.3|19.6 23.3|25.6 30.2|37.9    1536  15.9|18.7 24.2|25.5 32.5|34.7    2048  16.1|19.2 24.3|26.4 30.7|40.4
//         3000  16.8|19.2 25.5|27.1 36.2|40.0    4096  16.3|20.3 24.5|36.4 32.0|45.0    6144  16.6|24.1 (backward: no limit)
//         8192  19.9|30.0 26.6|44.9 35.6|64.2
//   fp32   256  18.5|16.0 24.7|24.8 28.2|28.7     512  15.7|14.7 22.9|21.7 26.9|27.1     768  16.0|16.3 22.0|23.4 27.4|27.8
//         1024  16.4|18.2 23.0|24.7 27.1|29.3    2048  17.4|19.1 23.4|27.2 27.1|33.8    4096  18.7|18.3 24.9|29.1 30.3|34.6
//         8192  20.8|26.4 26.5|45.3 35.4|52.9
// Behind the next one: narrow rows of fp32, by up to a seventh in the forward pass.
enum : int { kLnForward, kLnDx, kLnSums };   // backward pass without and with dw and db
template <int PASS, bool FP32, typename F> static int ln_layout(int dim, F&& f) {
    const int items = (dim + kLnItem - 1) / kLnItem;
    constexpr int B = PASS == kLnForward ? 1 : 2;
    constexpr int S = PASS == kLnSums ? 2 : 1;                 // CTAs of twice the size leave half the sums behind
    if (items <= 32) return f(LnLayout<1, 32, 8 * B>());
    if (items <= 64) return f(LnLayout<2, 32, 8 * B>());
    if (items <= 96) return f(LnLayout<3, 32, PASS == kLnSums ? 12 : 4>());
    if constexpr (FP32) {
        if (items <= 128) return f(LnLayout<2, 64, 4 * B>());
        if (items <= 256) return f(LnLayout<2, 128, 2 * B>());
        if (items <= 512) return f(LnLayout<2, 256, B>());
    } else {
        if (items <= 128) return f(LnLayout<4, 32, 4 * S>());
        if (items <= 192) return f(LnLayout<3, 64, 2 * S>());
        if (items <= 256) return f(LnLayout<4, 64, 2 * S>());
        if (items <= 384) return f(LnLayout<3, 128, S>());
        if (items <= 512) return f(LnLayout<4, 128, S>());
    }
    if constexpr (PASS == kLnForward) {
        if (items <= 768) return f(LnLayout<3, 256, 1>());
        if (items <= 1024) return f(LnLayout<2, 512, 1>());
        return f(LnLayout<8, 256, 1>());
    } else {
        if (items <= 1024) return f(LnLayout<2, 512, 1>());
        return f(LnLayout<4, 512, 1>());
    }
}

// CTAs of a pass: as many as the device holds, or what the rows need.  With sums over rows a CTA leaves 8 dim bytes of them behind,
// as much as two to four rows are, so it should have four rows a group, unless that leaves SMs idle (1001 x 1537 fp16, backward:
// 10.5 us with a CTA for every row group).
template <typename L> static int ln_grid(int64_t rows, int ctas, bool sums) {
    const int64_t most = (int64_t)gemm_num_sms() * ctas;
    int64_t need = (rows + L::rows - 1) / L::rows;
    if (sums && need > gemm_num_sms()) {
        const int64_t fewer = (need + 3) / 4;
        need = fewer > gemm_num_sms() ? fewer : gemm_num_sms();
    }
    return (int)(need < most ? need : most);
}
template <bool FP32> static int ln_sums_ctas(int64_t rows, int dim) {
    return ln_layout<kLnSums, FP32>(dim, [&](auto l) { return ln_grid<decltype(l)>(rows, LnBackward<decltype(l)>::ctas, true); });
}

// Bytes of a row in the ring.
static int ln_slot(int dim, int size, bool vec) { return (dim * size + 15) / 16 * 16 + (vec ? 0 : 16); }

static int check_ln(const char* op, int64_t rows, int dim, int64_t x_stride) {
    Q8K_REQUIRE(rows >= 0 && rows <= 0x7fffffffLL, Q8K_ERR_INVALID_ARG, "%s: rows %lld out of range", op, (long long)rows);
    Q8K_REQUIRE(dim > 0, Q8K_ERR_INVALID_ARG, "%s: dim %d must be positive", op, dim);
    Q8K_REQUIRE(dim <= kLnMaxDim, Q8K_ERR_UNSUPPORTED, "%s: dim %d exceeds %d", op, dim, kLnMaxDim);
    Q8K_REQUIRE(x_stride >= 0, Q8K_ERR_INVALID_ARG, "%s: negative row stride", op);
    return Q8K_OK;
}

static bool ln_aligned(const void* p, int dtype) {
    const int size = dtype_size(dtype);
    return size > 0 && reinterpret_cast<uintptr_t>(p) % size == 0;
}

template <typename Tx, typename Ty, typename L, bool VEC>
static int launch_ln_as(const void* x, int64_t x_stride, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t rows,
                        int dim, float eps, cudaStream_t st) {
    auto kern = layer_norm_kernel<Tx, Ty, L, VEC>;
    using Ring = LnRing<L, LnForward<L>::ctas, sizeof(Tx)>;
    constexpr int S = Ring::slots, most = S * Ring::row;
    const int slot = ln_slot(dim, sizeof(Tx), VEC);
    if (most > 40 * 1024) {
        static std::atomic<uint64_t> smem_done{0};
        if (int rc = allow_dynamic_smem((const void*)kern, most, smem_done)) return rc;
    }
    Q8K_CUDA_OK(launch_dependent(kern, (unsigned)ln_grid<L>(rows, LnForward<L>::ctas, false), L::cta, L::rows * S * slot, st, 1, (const Tx*)x, x_stride,
                                 w, b, (Ty*)y, mean, rstd, rows, dim, eps, slot));
    return Q8K_OK;
}

template <typename Tx, typename Ty>
static int launch_ln(const void* x, int64_t x_stride, const float* w, const float* b, void* y, float* mean, float* rstd, int64_t rows,
                     int dim, float eps, bool vec, cudaStream_t st) {
    auto launch = [&](auto l) {
        using L = decltype(l);
        return vec ? launch_ln_as<Tx, Ty, L, true>(x, x_stride, w, b, y, mean, rstd, rows, dim, eps, st)
                   : launch_ln_as<Tx, Ty, L, false>(x, x_stride, w, b, y, mean, rstd, rows, dim, eps, st);
    };
    return ln_layout<kLnForward, sizeof(Tx) == 4>(dim, launch);
}

template <typename Tx, typename Tg, typename L, bool VEC, bool WGRAD>
static int launch_ln_backward_as(const void* x, int64_t x_stride, const void* g, const float* mean, const float* rstd, const float* w, void* dx,
                                 float* part, int64_t rows, int dim, cudaStream_t st) {
    auto kern = layer_norm_backward_kernel<Tx, Tg, L, VEC, WGRAD>;
    using Ring = LnRing<L, LnBackward<L>::ctas, sizeof(Tx) + sizeof(Tg)>;
    constexpr int S = Ring::slots;
    constexpr int sums = WGRAD && L::rows > 1 ? L::cta * 2 * L::items * kLnItem * (int)sizeof(float) : 0;
    constexpr int most = S * Ring::row > sums ? S * Ring::row : sums;
    static_assert(most <= 226 * 1024, "layer norm ring");
    const int x_slot = ln_slot(dim, sizeof(Tx), VEC), g_slot = ln_slot(dim, sizeof(Tg), VEC);
    if (most > 40 * 1024) {
        static std::atomic<uint64_t> smem_done{0};
        if (int rc = allow_dynamic_smem((const void*)kern, most, smem_done)) return rc;
    }
    const int bytes = L::rows * S * (x_slot + g_slot);
    Q8K_CUDA_OK(launch_dependent(kern, (unsigned)ln_grid<L>(rows, LnBackward<L>::ctas, WGRAD), L::cta, bytes > sums ? bytes : sums, st, 1, (const Tx*)x,
                                 x_stride, (const Tg*)g, mean, rstd, w, (Tx*)dx, part, rows, dim, x_slot, g_slot));
    return Q8K_OK;
}

template <typename Tx, typename Tg>
static int launch_ln_backward(const void* x, int64_t x_stride, const void* g, const float* mean, const float* rstd, const float* w,
                              void* dx, float* part, int64_t rows, int dim, bool vec, cudaStream_t st) {
    if (part != nullptr)
        return ln_layout<kLnSums, sizeof(Tx) == 4>(dim, [&](auto l) {
            using L = decltype(l);
            return vec ? launch_ln_backward_as<Tx, Tg, L, true, true>(x, x_stride, g, mean, rstd, w, dx, part, rows, dim, st)
                       : launch_ln_backward_as<Tx, Tg, L, false, true>(x, x_stride, g, mean, rstd, w, dx, part, rows, dim, st);
        });
    return ln_layout<kLnDx, sizeof(Tx) == 4>(dim, [&](auto l) {
        using L = decltype(l);
        return vec ? launch_ln_backward_as<Tx, Tg, L, true, false>(x, x_stride, g, mean, rstd, w, dx, part, rows, dim, st)
                   : launch_ln_backward_as<Tx, Tg, L, false, false>(x, x_stride, g, mean, rstd, w, dx, part, rows, dim, st);
    });
}

}  // namespace q8k

using namespace q8k;

extern "C" int q8k_layer_norm(const void* x, int x_dtype, int64_t x_row_stride, const float* weight, const float* bias, void* y,
                              int y_dtype, float* mean, float* rstd, int64_t rows, int dim, float eps, void* stream) {
    const char* op = "layer_norm";
    if (int rc = check_ln(op, rows, dim, x_row_stride)) return rc;
    if (rows == 0) return Q8K_OK;
    Q8K_REQUIRE(x && y, Q8K_ERR_INVALID_ARG, "%s: null pointer", op);
    Q8K_REQUIRE(ln_aligned(x, x_dtype) && ln_aligned(y, y_dtype) && ln_aligned(weight, Q8K_DT_F32) && ln_aligned(bias, Q8K_DT_F32),
                Q8K_ERR_INVALID_ARG, "%s: a pointer is not aligned to its element, or an unknown type", op);
    const bool vec = dim % kLnItem == 0 && aligned16(x) && (x_row_stride * dtype_size(x_dtype)) % 16 == 0 && aligned16(y) &&
                     aligned16(weight) && aligned16(bias);
    cudaStream_t st = (cudaStream_t)stream;
#define Q8K_LN_FWD(DX, DY)                                                                       \
    if (x_dtype == DX && y_dtype == DY)                                                          \
        return launch_ln<DType<DX>::type, DType<DY>::type>(x, x_row_stride, weight, bias, y, mean, rstd, rows, dim, eps, vec, st)
    Q8K_LN_FWD(Q8K_DT_BF16, Q8K_DT_BF16);
    Q8K_LN_FWD(Q8K_DT_BF16, Q8K_DT_E4M3);
    Q8K_LN_FWD(Q8K_DT_F16, Q8K_DT_F16);
    Q8K_LN_FWD(Q8K_DT_F32, Q8K_DT_F32);
    Q8K_LN_FWD(Q8K_DT_F32, Q8K_DT_BF16);
    Q8K_LN_FWD(Q8K_DT_F32, Q8K_DT_F16);
#undef Q8K_LN_FWD
    set_error_detail("%s: dtype pair (%d -> %d) not supported", op, x_dtype, y_dtype);
    return Q8K_ERR_UNSUPPORTED;
}

extern "C" size_t q8k_layer_norm_backward_workspace_bytes(int64_t rows, int dim) {
    if (rows <= 0 || dim <= 0 || dim > kLnMaxDim) return 0;
    const int a = ln_sums_ctas<false>(rows, dim), b = ln_sums_ctas<true>(rows, dim);       // whatever x's type
    return (size_t)(a > b ? a : b) * 2 * (size_t)dim * sizeof(float);
}

extern "C" int q8k_layer_norm_backward(const void* x, int x_dtype, int64_t x_row_stride, const void* grad, int grad_dtype,
                                       const float* mean, const float* rstd, const float* weight, void* dx, float* dweight,
                                       float* dbias, int64_t rows, int dim, void* workspace, size_t workspace_bytes, void* stream) {
    const char* op = "layer_norm_backward";
    if (int rc = check_ln(op, rows, dim, x_row_stride)) return rc;
    cudaStream_t st = (cudaStream_t)stream;
    const bool sums = dweight != nullptr || dbias != nullptr;
    Q8K_REQUIRE(ln_aligned(dweight, Q8K_DT_F32) && ln_aligned(dbias, Q8K_DT_F32), Q8K_ERR_INVALID_ARG, "%s: misaligned gradient", op);
    if (rows == 0) {                                           // sums over no rows
        if (dweight != nullptr) Q8K_CUDA_OK(cudaMemsetAsync(dweight, 0, (size_t)dim * sizeof(float), st));
        if (dbias != nullptr) Q8K_CUDA_OK(cudaMemsetAsync(dbias, 0, (size_t)dim * sizeof(float), st));
        return Q8K_OK;
    }
    if (dx == nullptr && !sums) return Q8K_OK;
    Q8K_REQUIRE(x && grad && mean && rstd, Q8K_ERR_INVALID_ARG, "%s: null pointer", op);
    Q8K_REQUIRE(ln_aligned(x, x_dtype) && ln_aligned(dx, x_dtype) && ln_aligned(grad, grad_dtype) && ln_aligned(weight, Q8K_DT_F32),
                Q8K_ERR_INVALID_ARG, "%s: a pointer is not aligned to its element, or an unknown type", op);
    float* part = nullptr;
    if (sums) {
        Q8K_REQUIRE(workspace != nullptr && aligned16(workspace), Q8K_ERR_INVALID_ARG, "%s: null or misaligned workspace", op);
        Q8K_REQUIRE(workspace_bytes >= q8k_layer_norm_backward_workspace_bytes(rows, dim), Q8K_ERR_WORKSPACE,
                    "%s: workspace of %zu bytes, %zu needed", op, workspace_bytes, q8k_layer_norm_backward_workspace_bytes(rows, dim));
        part = (float*)workspace;
    }
    const bool vec = dim % kLnItem == 0 && aligned16(x) && (x_row_stride * dtype_size(x_dtype)) % 16 == 0 && aligned16(grad) &&
                     aligned16(dx) && aligned16(weight);
    int rc = Q8K_ERR_UNSUPPORTED;
#define Q8K_LN_BWD(DX, DG)                                                                       \
    if (x_dtype == DX && grad_dtype == DG)                                                       \
        rc = launch_ln_backward<DType<DX>::type, DType<DG>::type>(x, x_row_stride, grad, mean, rstd, weight, dx, part, rows, dim, vec, st)
    Q8K_LN_BWD(Q8K_DT_BF16, Q8K_DT_BF16);
    else Q8K_LN_BWD(Q8K_DT_F16, Q8K_DT_F16);
    else Q8K_LN_BWD(Q8K_DT_F32, Q8K_DT_F32);
    else Q8K_LN_BWD(Q8K_DT_F32, Q8K_DT_BF16);
    else Q8K_LN_BWD(Q8K_DT_F32, Q8K_DT_F16);
    else set_error_detail("%s: dtype pair (%d, gradient %d) not supported", op, x_dtype, grad_dtype);
#undef Q8K_LN_BWD
    if (rc != Q8K_OK || !sums) return rc;
    Q8K_CUDA_OK(launch_dependent(layer_norm_wgrad_kernel, (unsigned)((2 * (int64_t)dim + 31) / 32), 32 * kLnSumWarps, 0, st, 1, part,
                                 x_dtype == Q8K_DT_F32 ? ln_sums_ctas<true>(rows, dim) : ln_sums_ctas<false>(rows, dim), dweight, dbias, dim));
    return Q8K_OK;
}
