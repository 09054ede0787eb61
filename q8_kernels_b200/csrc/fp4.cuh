// Microscaled 4-bit values: what their quantizer and their products share.
//
// A row of K values (a multiple of 32) is K / 2 bytes, the lower nibble first, and one scale a block:
//   mxfp4   blocks of 32, e8m0 (a power of two)
//   nvfp4   blocks of 16, e4m3, and one fp32 scale a row
// The block scales lie as the tensor core's copy wants them: tiles of 128 rows x 4 blocks are 512 bytes, row r's four scales at
// (r % 32) * 16 + (r / 32) * 4; tiles follow one another along K, then along the rows, and K is filled up to slabs of 256 values
// (128 bytes of them), 2 tiles or 4.
#pragma once

#include "common.cuh"

namespace q8k {

constexpr int kFp4Slab = 256;                                  // values
constexpr int kFp4MaxN = (1 << 30) - 16;                       // columns of a product: its stores name them by byte, in 32 bits
constexpr int fp4_block(bool nv) { return nv ? 16 : 32; }
constexpr int fp4_slab_tiles(bool nv) { return nv ? 4 : 2; }
constexpr int fp4_slab_scales(bool nv) { return 512 * fp4_slab_tiles(nv); }   // bytes for 128 rows
inline int fp4_slabs(int K) { return (K + kFp4Slab - 1) / kFp4Slab; }
inline int64_t fp4_row_tiles(int64_t rows) { return (rows + 127) / 128; }
inline int64_t fp4_scale_bytes(bool nv, int64_t rows, int K) { return fp4_row_tiles(rows) * fp4_slabs(K) * (int64_t)fp4_slab_scales(nv); }

// Where the scale of block b (along K) of a row lies.
template <bool NV> __host__ __device__ __forceinline__ int64_t fp4_scale_at(int64_t row, int b, int slabs) {
    constexpr int TILES = NV ? 4 : 2;
    return ((row >> 7) * slabs * TILES + (b >> 2)) * 512 + (row & 31) * 16 + ((row >> 5) & 3) * 4 + (b & 3);
}

// Eight fp32 values to four bytes of e2m1: nearest, halves to even, beyond 6 to 6.
__device__ __forceinline__ uint32_t float8_to_e2m1(const float (&v)[8]) {
    uint32_t w;
    asm("{\n\t"
        ".reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t"
        "}"
        : "=r"(w)
        : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
    return w;
}
// Eight values of four bytes, exact.
__device__ __forceinline__ void e2m1_to_float8(uint32_t w, float (&v)[8]) {
    uint32_t h[4];
    asm("{\n\t"
        ".reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t"
        "}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(w));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[i]));
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
// What a block's scale byte stands for; e8m0's 255 is NaN, its 0 the subnormal 2^-127.
template <bool NV> __device__ __forceinline__ float fp4_scale_value(uint8_t b) {
    if constexpr (NV) return e4m3_to_float(b);
    return b == 255 ? __int_as_float(0x7fffffff) : b == 0 ? __int_as_float(0x00400000) : __int_as_float((int)b << 23);
}

// An operand of a product.
struct Fp4Operand {
    const void* values;                      // [rows, K / 2]
    const void* block_scales;
    const float* row_scales;                 // nvfp4 only
};

// q8k_fp4_mm.  b_ahead: the kernel before it on the stream is the quantizer of A, which has waited for everything before it, so B can be loaded at once.
// x: 16-bit rows for the product to quantise, in the place of a (null), where fp4_quantises_rows; else null.
int fp4_mm(int format, const void* a, const void* a_block_scales, const float* a_row_scales, const void* b, const void* b_block_scales,
           const float* b_row_scales, const float* bias, void* out, int out_dtype, int M, int N, int K, int fuse_gelu, int* dev_status, bool b_ahead,
           const void* x, bool x_f16, cudaStream_t st);
bool fp4_quantises_rows(int M, int N, int K);

}  // namespace q8k
