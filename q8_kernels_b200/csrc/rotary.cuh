// The angles of rotary embeddings, shared by the kernels that turn heads: pair i of a token turns by position[axis(i)] * freq[i].
//
// A position of a million radians has no correct digit in fp32 after its reduction, so position * freq / (2 pi) is formed in fp64, the whole
// turns are dropped there, and sine and cosine are taken of the rest, at most half a turn, in fp32.
#pragma once

#include "common.cuh"

namespace q8k {

struct RotaryAngles {
    const void* positions;                   // null: 0, 1, ... of each batch entry
    int kind;                                // Q8K_POS_*
    int64_t pos_batch, pos_token, pos_axis;  // strides in elements
    const int* axes;                         // axis of each pair; null: one axis
    int n_axes;
    const double* freq;
    float amplitude, sign;
};

// AXES: there is an axis for each pair.  (An axis beyond the last one is taken as the last.)
template <bool AXES> __device__ __forceinline__ double rotary_position(const RotaryAngles& a, int64_t at, int i) {
    if constexpr (AXES) {
        const unsigned axis = min((unsigned)a.axes[i], (unsigned)(a.n_axes - 1));
        at += (int64_t)axis * a.pos_axis;
    }
    switch (a.kind) {
        case Q8K_POS_I64: return (double)static_cast<const int64_t*>(a.positions)[at];
        case Q8K_POS_I32: return (double)static_cast<const int32_t*>(a.positions)[at];
        case Q8K_POS_F32: return (double)static_cast<const float*>(a.positions)[at];
        default: return static_cast<const double*>(a.positions)[at];
    }
}
__device__ __forceinline__ float2 rotary_turn(const RotaryAngles& a, double pos, int i) {
    const double t = pos * (a.freq[i] * 0.15915494309189535);  // 1 / (2 pi)
    float sn, cs;
    sincospif(2.0f * (float)(t - rint(t)), &sn, &cs);
    return make_float2(cs * a.amplitude, sn * a.amplitude * a.sign);
}

// What positions, frequencies and axes have to fulfil.
inline int rotary_check_angles(const char* op, const RotaryAngles& a) {
    Q8K_REQUIRE(a.freq != nullptr && reinterpret_cast<uintptr_t>(a.freq) % 8 == 0, Q8K_ERR_INVALID_ARG, "%s: null or misaligned frequencies", op);
    Q8K_REQUIRE(a.kind >= Q8K_POS_I32 && a.kind <= Q8K_POS_F64, Q8K_ERR_INVALID_ARG, "%s: position type %d is unknown", op, a.kind);
    const int size = a.kind == Q8K_POS_I64 || a.kind == Q8K_POS_F64 ? 8 : 4;
    Q8K_REQUIRE(reinterpret_cast<uintptr_t>(a.positions) % size == 0, Q8K_ERR_INVALID_ARG, "%s: misaligned positions", op);
    if (a.axes != nullptr) {
        Q8K_REQUIRE(a.n_axes >= 1 && a.positions != nullptr && reinterpret_cast<uintptr_t>(a.axes) % 4 == 0, Q8K_ERR_INVALID_ARG,
                    "%s: several axes need positions, %d axes of them", op, a.n_axes);
    }
    return Q8K_OK;
}

}  // namespace q8k
