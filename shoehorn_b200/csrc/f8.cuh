// Launch interface of the block-scaled 8-bit operators (f8.cu, f8_mm.cu).
//
// The format: E4M3 codes with one f32 scale for each block of kF8Block
// columns (of one row, or of kF8Block rows), value = code * scale.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"

namespace shc {

constexpr int kF8Block = 128;
// Largest E4M3 magnitude, and the block maximum below which a block's scale
// stays at 2^-126: scale and inverse are then normal f32 numbers for any
// input, an all-zero block's among them.
constexpr float kF8Top = 448.0f;
constexpr float kF8Least = 448.0f * 1.17549435e-38f;

// n_mats matrices of n_rows x ne0.  Strides count elements (bytes for codes).
struct F8Codec {
    const void *src;  // encode: rows of src_type
    int type;         // encode: source type; decode: destination type (SHC_SRC_*)
    int64_t src_row_stride, src_mat_stride;
    uint8_t *codes;  // 16-byte aligned, strides multiples of 16
    int64_t code_row_stride, code_mat_stride;
    float *scales;  // [n_mats, ceil(n_rows / block_rows), ceil(ne0 / kF8Block)]
    void *dst;      // decode: [n_mats, n_rows, ne0]
    int64_t n_mats, n_rows, ne0;
    int block_rows;  // 1 or kF8Block
};
cudaError_t launch_f8_encode(const F8Codec &c, cudaStream_t st);
cudaError_t launch_f8_decode(const F8Codec &c, cudaStream_t st);

// D = A W^T (W [n, k], A [rows, k]) or, transposed, D = A W (A [rows, n]).
struct F8Product {
    const uint8_t *a;
    const float *a_scales;
    int64_t a_row_stride, a_scale_stride, n_rows;
    const uint8_t *w;
    const float *w_scales;  // [n_experts, ceil(n / 128), ceil(k / 128)]
    int64_t w_row_stride, w_mat_stride, n_experts, n, k;
    const void *offsets;  // null: one expert takes every row
    int offsets_64;
    int transposed;
    int dst_type;
    void *dst;
    int64_t dst_row_stride;
    int *status;
};
// SHC_* status
int launch_f8_product(const F8Product &p, int num_sms, cudaStream_t st);

}  // namespace shc
