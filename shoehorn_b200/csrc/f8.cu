// Block-scaled 8-bit codes: E4M3 with one scale for each block of 128
// columns (block_rows = 1, activations) or of 128 x 128 elements (block_rows
// = 128, weights).
//
//   top   = max(max |x| over the block's finite elements, 448 * 2^-126)
//   scale = top / 448,  code = e4m3(x * (448 / top)),  value = code * scale
//
// The quotient 448 / top is rounded once per block and the product once per
// element, so a code's value before its rounding to E4M3 is within 2^-23 of
// x / scale.  NaN and infinite elements become the NaN code and leave the
// block's scale to the finite ones.
#include "f8.cuh"

namespace shc {
namespace {

constexpr int kLanes = 16;  // lanes of one 128-column block, 8 columns each

// Two E4M3 codes, lo in the low byte; NaN gives 0x7F, magnitudes above 448
// give 448 (reached only by the rounding of x * (448 / top)).
__device__ __forceinline__ uint16_t e4m3x2(float lo, float hi) {
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 e4m3x2_val(uint16_t c) {
    uint32_t h;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(c));
    return __half22float2(*reinterpret_cast<__half2 *>(&h));
}

__device__ __forceinline__ float inf_f() { return __uint_as_float(0x7f800000u); }

// Eight columns of a row from `col`, columns at or past ne0 as zeros.
template <bool VEC>
__device__ __forceinline__ void load_cols(const RowSrc &s, int64_t row, int64_t col, float v[8]) {
    if (VEC && col + 8 <= s.ne0) {
        load8(s, row, col, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = col + i < s.ne0 ? load1(s, row, col + i) : 0.0f;
    }
}

// Largest magnitude, NaN ignored; infinite if any element is.
__device__ __forceinline__ float top8(const float v[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) m = fmaxf(m, fabsf(v[i]));
    return m;
}
// Infinite elements to NaN (the NaN code); returns the finite ones' maximum.
__device__ __forceinline__ float drop_inf8(float v[8]) {
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; i++) {
        if (fabsf(v[i]) == inf_f()) v[i] = __uint_as_float(0x7fffffffu);
        else m = fmaxf(m, fabsf(v[i]));
    }
    return m;
}

// Codes of eight columns; a whole group is one 8-byte store (codes rows start
// on 16-byte boundaries), the row's ragged end single bytes.
__device__ __forceinline__ void store_codes(uint8_t *row, int64_t col, int64_t ne0, const float v[8], float inv) {
    if (col >= ne0) return;
    uint32_t w[2];
#pragma unroll
    for (int i = 0; i < 2; i++)
        w[i] = (uint32_t)e4m3x2(v[4 * i] * inv, v[4 * i + 1] * inv) |
               ((uint32_t)e4m3x2(v[4 * i + 2] * inv, v[4 * i + 3] * inv) << 16);
    if (col + 8 <= ne0) {
        *reinterpret_cast<uint2 *>(row + col) = make_uint2(w[0], w[1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (col + i < ne0) row[col + i] = (uint8_t)(w[i >> 2] >> (8 * (i & 3)));
    }
}

// One 16-lane half-warp per (row, block).
template <bool VEC>
__global__ void __launch_bounds__(256) f8_encode_rows_kernel(F8Codec c) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, total = c.n_mats * c.n_rows * nb;
    const int lane = threadIdx.x & (kLanes - 1);
    const int64_t step = (int64_t)gridDim.x * (256 / kLanes);
    const int64_t rounds = (total + step - 1) / step;  // whole warps stay together for the shuffles
    int64_t u = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    for (int64_t i = 0; i < rounds; i++, u += step) {
        const bool on = u < total;
        const int64_t row = on ? u / nb : 0, b = on ? u - row * nb : 0;
        const int64_t mat = row / c.n_rows, r = row - mat * c.n_rows;
        const int64_t col = b * kF8Block + lane * 8;
        const size_t esz = c.type == SHC_SRC_F32 ? 4 : 2;
        const RowSrc s{static_cast<const uint8_t *>(c.src) + mat * c.src_mat_stride * (int64_t)esz, c.type,
                       on ? c.ne0 : 0, c.src_row_stride};
        float v[8];
        load_cols<VEC>(s, r, col, v);
        float m = top8(v);
#pragma unroll
        for (int o = kLanes / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if (__any_sync(~0u, m == inf_f())) {
            m = drop_inf8(v);
#pragma unroll
            for (int o = kLanes / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        }
        m = fmaxf(m, kF8Least);
        if (!on) continue;
        store_codes(c.codes + mat * c.code_mat_stride + r * c.code_row_stride, col, c.ne0, v, kF8Top / m);
        if (lane == 0) c.scales[u] = m / kF8Top;
    }
}

// One thread block per 128 x 128 tile, held in registers between the maximum
// and the codes: thread t has columns 8 (t % 16).. of rows t / 16 + 16 i.
template <bool VEC>
__global__ void __launch_bounds__(256) f8_encode_tiles_kernel(F8Codec c) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, rb = (c.n_rows + kF8Block - 1) / kF8Block;
    const int lane = threadIdx.x & (kLanes - 1), r16 = threadIdx.x / kLanes;
    __shared__ float s_top[2][8];
    int turn = 0;
    for (int64_t tile = blockIdx.x; tile < c.n_mats * rb * nb; tile += gridDim.x) {
        const int64_t b = tile % nb, rest = tile / nb, mat = rest / rb, row0 = (rest - mat * rb) * kF8Block;
        const int64_t col = b * kF8Block + lane * 8;
        const size_t esz = c.type == SHC_SRC_F32 ? 4 : 2;
        const RowSrc s{static_cast<const uint8_t *>(c.src) + mat * c.src_mat_stride * (int64_t)esz, c.type, c.ne0,
                       c.src_row_stride};
        float v[8][8];
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int64_t r = row0 + r16 + 16 * i;
            if (r < c.n_rows) {
                load_cols<VEC>(s, r, col, v[i]);
            } else {
#pragma unroll
                for (int j = 0; j < 8; j++) v[i][j] = 0.0f;
            }
            m = fmaxf(m, top8(v[i]));
        }
        // Block-wide maximum; the second pass only where an element is infinite.
        for (int pass = 0; pass < 2; pass++) {
            for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
            if ((threadIdx.x & 31) == 0) s_top[turn][threadIdx.x / 32] = m;
            __syncthreads();
#pragma unroll
            for (int w = 0; w < 8; w++) m = fmaxf(m, s_top[turn][w]);
            turn ^= 1;  // the next maximum does not overwrite one still being read
            if (m != inf_f()) break;
            m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; i++) m = fmaxf(m, drop_inf8(v[i]));
        }
        m = fmaxf(m, kF8Least);
        const float inv = kF8Top / m;
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const int64_t r = row0 + r16 + 16 * i;
            if (r < c.n_rows)
                store_codes(c.codes + mat * c.code_mat_stride + r * c.code_row_stride, col, c.ne0, v[i], inv);
        }
        if (threadIdx.x == 0) c.scales[tile] = m / kF8Top;
    }
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// One thread per eight codes of a row.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) f8_decode_kernel(F8Codec c) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, rb = (c.n_rows + c.block_rows - 1) / c.block_rows;
    const int64_t ng = (c.ne0 + 7) / 8, total = c.n_mats * c.n_rows * ng;
    for (int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x; u < total; u += (int64_t)gridDim.x * 256) {
        const int64_t row = u / ng, col = (u - row * ng) * 8;
        const int64_t mat = row / c.n_rows, r = row - mat * c.n_rows;
        const float s = __ldg(c.scales + (mat * rb + r / c.block_rows) * nb + col / kF8Block);
        const uint8_t *p = c.codes + mat * c.code_mat_stride + r * c.code_row_stride + col;
        const int n = c.ne0 - col < 8 ? (int)(c.ne0 - col) : 8;
        uint16_t q[4] = {0, 0, 0, 0};
        if (n == 8) {
            const uint2 w = __ldg(reinterpret_cast<const uint2 *>(p));
            q[0] = (uint16_t)w.x;
            q[1] = (uint16_t)(w.x >> 16);
            q[2] = (uint16_t)w.y;
            q[3] = (uint16_t)(w.y >> 16);
        } else {
            for (int i = 0; i < n; i++) q[i >> 1] |= (uint16_t)((uint16_t)p[i] << (8 * (i & 1)));
        }
        __align__(16) T y[8];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 f = e4m3x2_val(q[i]);
            y[2 * i] = from_f32<T>(f.x * s);
            y[2 * i + 1] = from_f32<T>(f.y * s);
        }
        T *o = static_cast<T *>(c.dst) + row * c.ne0 + col;
        if (VEC && n == 8) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; i++)
                reinterpret_cast<uint4 *>(o)[i] = reinterpret_cast<const uint4 *>(y)[i];
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (i < n) o[i] = y[i];
        }
    }
}

unsigned grid_for(int64_t items, int64_t per_block, int num_sms, int waves) {
    int64_t b = (items + per_block - 1) / per_block;
    const int64_t most = (int64_t)num_sms * waves;
    return (unsigned)(b < 1 ? 1 : b > most ? most : b);
}

}  // namespace

cudaError_t launch_f8_encode(const F8Codec &c, int num_sms, cudaStream_t st) {
    const int64_t esz = c.type == SHC_SRC_F32 ? 4 : 2;
    // 128-bit loads where every row starts on a 16-byte boundary
    const bool vec = ((uintptr_t)c.src & 15) == 0 && c.src_row_stride * esz % 16 == 0 &&
                     c.src_mat_stride * esz % 16 == 0;
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block;
    if (c.block_rows == 1) {
        const unsigned g = grid_for(c.n_mats * c.n_rows * nb, 256 / kLanes, num_sms, 64);
        if (vec) f8_encode_rows_kernel<true><<<g, 256, 0, st>>>(c);
        else f8_encode_rows_kernel<false><<<g, 256, 0, st>>>(c);
    } else {
        const unsigned g = grid_for(c.n_mats * ((c.n_rows + kF8Block - 1) / kF8Block) * nb, 1, num_sms, 64);
        if (vec) f8_encode_tiles_kernel<true><<<g, 256, 0, st>>>(c);
        else f8_encode_tiles_kernel<false><<<g, 256, 0, st>>>(c);
    }
    return cudaGetLastError();
}

cudaError_t launch_f8_decode(const F8Codec &c, int num_sms, cudaStream_t st) {
    const int64_t esz = c.type == SHC_SRC_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)c.dst & 15) == 0 && c.ne0 * esz % 16 == 0;
    const unsigned g = grid_for(c.n_mats * c.n_rows * ((c.ne0 + 7) / 8), 256, num_sms, 64);
    if (c.type == SHC_SRC_F32) {
        if (vec) f8_decode_kernel<float, true><<<g, 256, 0, st>>>(c);
        else f8_decode_kernel<float, false><<<g, 256, 0, st>>>(c);
    } else if (c.type == SHC_SRC_F16) {
        if (vec) f8_decode_kernel<__half, true><<<g, 256, 0, st>>>(c);
        else f8_decode_kernel<__half, false><<<g, 256, 0, st>>>(c);
    } else {
        if (vec) f8_decode_kernel<__nv_bfloat16, true><<<g, 256, 0, st>>>(c);
        else f8_decode_kernel<__nv_bfloat16, false><<<g, 256, 0, st>>>(c);
    }
    return cudaGetLastError();
}

}  // namespace shc
