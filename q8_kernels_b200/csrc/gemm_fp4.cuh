// Pieces shared by the 4-bit GEMM kernels.
#pragma once

#include "fp4.cuh"
#include "gemm_common.cuh"

namespace q8k {

struct Fp4GemmParams {
    const float* a_scales;                   // fp32 row scales; null for mxfp4
    const float* b_scales;
    const float* bias;                       // may be null
    void* out;
    int* status;
    int M, N, K;
};

// 256 x 256 tiles on CTA pairs; Q8K_ERR_UNSUPPORTED (without touching the error detail) when the device cannot co-schedule the clusters.
int launch_fp4_pair(bool nv, bool gelu, bool f16, const Fp4Operand& a, const Fp4Operand& b, const Fp4GemmParams& p, cudaStream_t st);

// Tensor map of an operand's block scales: [row tiles][slabs][bytes of a slab], in rows of 256 bytes, boxes of one slab of `tiles` row tiles.
inline int make_scales_map(CUtensorMap* map, const void* scales, bool nv, int64_t rows, int K, int tiles, const char* op) {
    const uint64_t per_slab = (uint64_t)fp4_slab_scales(nv) / 256, per_tile = per_slab * (uint64_t)fp4_slabs(K);
    const uint64_t dims[3] = {256, per_tile, (uint64_t)fp4_row_tiles(rows)};
    const uint64_t strides[2] = {256, 256 * per_tile};
    const uint32_t box[3] = {256, (uint32_t)per_slab, (uint32_t)tiles};
    return make_byte_tensor_map(map, scales, 3, dims, strides, box, 0, op);
}
// Tensor map of an operand's values: boxes of one slab (128 bytes) of `rows` rows.
inline int make_values_map(CUtensorMap* map, const void* values, int64_t rows, int K, int box_rows, const char* op) {
    const uint64_t dims[2] = {(uint64_t)K / 2, (uint64_t)rows};
    const uint64_t strides[1] = {(uint64_t)K / 2};
    const uint32_t box[2] = {128, (uint32_t)box_rows};
    return make_byte_tensor_map(map, values, 2, dims, strides, box, 128, op);
}

}  // namespace q8k
