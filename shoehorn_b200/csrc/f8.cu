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

constexpr int kLanes = 8;   // lanes of one 128-column block
constexpr int kElems = 16;  // columns of one lane: one 16-byte store of codes

// Two E4M3 codes, lo in the low byte; NaN gives 0x7F, magnitudes above 448
// give 448 (reached only by the rounding of x * (448 / top)).
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
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

// A lane's 16 source elements as they lie in memory.  16-bit types stay
// packed: half the registers, and the magnitudes' maximum takes two elements
// per instruction.
template <int ST>
struct Raw {
    static constexpr int kWords = ST == SHC_SRC_F32 ? 16 : 8;
    uint32_t w[kWords];

    // Columns col.. of the row at p (on a 16-byte boundary), zeros from ne0 on.
    __device__ __forceinline__ void load(const uint8_t *p, int64_t col, int64_t ne0) {
        constexpr int esz = ST == SHC_SRC_F32 ? 4 : 2;
        if (col + kElems <= ne0) {
            const uint4 *q = reinterpret_cast<const uint4 *>(p + col * esz);
#pragma unroll
            for (int i = 0; i < kWords / 4; i++) {
                const uint4 v = __ldcs(q + i);  // read once
                w[4 * i] = v.x;
                w[4 * i + 1] = v.y;
                w[4 * i + 2] = v.z;
                w[4 * i + 3] = v.w;
            }
        } else if (ST == SHC_SRC_F32) {
#pragma unroll
            for (int i = 0; i < kWords; i++)
                w[i] = col + i < ne0 ? __ldg(reinterpret_cast<const uint32_t *>(p) + col + i) : 0u;
        } else {
            const uint16_t *q = reinterpret_cast<const uint16_t *>(p) + col;
#pragma unroll
            for (int i = 0; i < kWords; i++) {
                const uint32_t lo = col + 2 * i < ne0 ? __ldg(q + 2 * i) : 0u;
                const uint32_t hi = col + 2 * i + 1 < ne0 ? __ldg(q + 2 * i + 1) : 0u;
                w[i] = lo | hi << 16;
            }
        }
    }
    __device__ __forceinline__ void zero() {
#pragma unroll
        for (int i = 0; i < kWords; i++) w[i] = 0;
    }
    __device__ __forceinline__ float at(int i) const {
        if (ST == SHC_SRC_F32) return __uint_as_float(w[i % kWords]);
        const uint32_t v = w[(i >> 1) % kWords];
        if (ST == SHC_SRC_BF16) return __uint_as_float(i & 1 ? v & 0xFFFF0000u : v << 16);
        return f16_val((uint16_t)(i & 1 ? v >> 16 : v));
    }
    // Largest magnitude, NaN ignored; infinite if any element is.
    __device__ __forceinline__ float top() const {
        if (ST == SHC_SRC_F32) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < kWords; i++) m = fmaxf(m, fabsf(__uint_as_float(w[i])));
            return m;
        }
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kWords; i++) {
            const uint32_t v = w[i] & 0x7FFF7FFFu;
            if (ST == SHC_SRC_BF16) asm("max.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(v));
            else asm("max.f16x2 %0, %0, %1;" : "+r"(m) : "r"(v));
        }
        if (ST == SHC_SRC_BF16) return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xFFFF0000u));
        return fmaxf(f16_val((uint16_t)m), f16_val((uint16_t)(m >> 16)));
    }
    // Infinite elements to NaN (the NaN code); returns the finite ones' maximum.
    __device__ __forceinline__ float drop_inf() {
        float m = 0.0f;
#pragma unroll
        for (int i = 0; i < kElems; i++) {
            const float x = fabsf(at(i));
            if (x != inf_f()) {
                m = fmaxf(m, x);
            } else if (ST == SHC_SRC_F32) {
                w[i % kWords] = 0x7FFFFFFFu;
            } else {
                w[(i >> 1) % kWords] |= i & 1 ? 0x7FFF0000u : 0x00007FFFu;
            }
        }
        return m;
    }
    // Codes to a row that starts on a 16-byte boundary: one 16-byte store,
    // the row's ragged end in single bytes.
    __device__ __forceinline__ void store(uint8_t *row, int64_t col, int64_t ne0, float inv) const {
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; i++)
            q[i] = e4m3x2(at(4 * i) * inv, at(4 * i + 1) * inv) | e4m3x2(at(4 * i + 2) * inv, at(4 * i + 3) * inv) << 16;
        if (col + kElems <= ne0) {
            *reinterpret_cast<uint4 *>(row + col) = make_uint4(q[0], q[1], q[2], q[3]);
        } else {
#pragma unroll
            for (int i = 0; i < kElems; i++)
                if (col + i < ne0) row[col + i] = (uint8_t)(q[i >> 2] >> (8 * (i & 3)));
        }
    }
};

template <int ST>
__device__ __forceinline__ const uint8_t *src_row(const F8Codec &c, int64_t mat, int64_t r) {
    return static_cast<const uint8_t *>(c.src) + (mat * c.src_mat_stride + r * c.src_row_stride) * (ST == SHC_SRC_F32 ? 4 : 2);
}

// Activations: eight lanes per (row, block), kUnits of them at once so that a
// warp has kUnits x 4 blocks' loads in flight.  I: unit index type, 32 bits
// wherever the units can be counted in them (a division by the row's blocks
// per unit).
template <int ST>
__host__ __device__ constexpr int units() { return ST == SHC_SRC_F32 ? 2 : 4; }

template <int ST, typename I>
__global__ void __launch_bounds__(256) f8_encode_rows_kernel(F8Codec c) {
    constexpr int kUnits = units<ST>(), kPerBlock = 256 / kLanes;
    const I nb = (I)((c.ne0 + kF8Block - 1) / kF8Block), total = (I)(c.n_mats * c.n_rows) * nb, rows = (I)c.n_rows;
    const int lane = threadIdx.x & (kLanes - 1);
    const I u0 = (I)blockIdx.x * (kPerBlock * kUnits) + threadIdx.x / kLanes;
    Raw<ST> v[kUnits];
    uint8_t *row[kUnits];
    int64_t col[kUnits];
    float m[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const I u = u0 + (I)(k * kPerBlock);
        const I g = u < total ? u / nb : 0, b = u < total ? u - g * nb : 0;
        const I mat = c.n_mats > 1 ? g / rows : 0, r = g - mat * rows;
        col[k] = (int64_t)b * kF8Block + lane * kElems;
        if (u >= total) col[k] = c.ne0;
        row[k] = c.codes + (int64_t)mat * c.code_mat_stride + (int64_t)r * c.code_row_stride;
        v[k].load(src_row<ST>(c, mat, r), col[k], c.ne0);
    }
    bool inf = false;
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        m[k] = v[k].top();
#pragma unroll
        for (int o = kLanes / 2; o; o >>= 1) m[k] = fmaxf(m[k], __shfl_xor_sync(~0u, m[k], o));
        inf |= m[k] == inf_f();
    }
    if (__any_sync(~0u, inf)) {
#pragma unroll
        for (int k = 0; k < kUnits; k++) {
            m[k] = v[k].drop_inf();
#pragma unroll
            for (int o = kLanes / 2; o; o >>= 1) m[k] = fmaxf(m[k], __shfl_xor_sync(~0u, m[k], o));
        }
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const I u = u0 + (I)(k * kPerBlock);
        const float t = fmaxf(m[k], kF8Least);
        if (col[k] < c.ne0) v[k].store(row[k], col[k], c.ne0, kF8Top / t);
        if (u < total && lane == 0) c.scales[u] = t / kF8Top;
    }
}

// Weights: one thread block per 128 x 128 tile, held in registers between the
// maximum and the codes; thread t has 16 columns of rows t / 8 + 32 i.
template <int ST>
__global__ void __launch_bounds__(256) f8_encode_tiles_kernel(F8Codec c) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, rb = (c.n_rows + kF8Block - 1) / kF8Block;
    const int64_t tile = blockIdx.x, b = tile % nb, rest = tile / nb, mat = rest / rb;
    const int64_t row0 = (rest - mat * rb) * kF8Block + threadIdx.x / kLanes;
    const int64_t col = b * kF8Block + (threadIdx.x & (kLanes - 1)) * kElems;
    __shared__ float s_top[2][8];
    Raw<ST> v[4];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t r = row0 + 32 * i;
        if (r < c.n_rows) v[i].load(src_row<ST>(c, mat, r), col, c.ne0);
        else v[i].zero();
    }
#pragma unroll
    for (int i = 0; i < 4; i++) m = fmaxf(m, v[i].top());
    // Block-wide maximum; a second pass only where an element is infinite.
    for (int pass = 0; pass < 2; pass++) {
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
        if ((threadIdx.x & 31) == 0) s_top[pass][threadIdx.x / 32] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) m = fmaxf(m, s_top[pass][w]);
        if (m != inf_f()) break;
        m = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) m = fmaxf(m, v[i].drop_inf());
    }
    m = fmaxf(m, kF8Least);
    const float inv = kF8Top / m;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t r = row0 + 32 * i;
        if (r < c.n_rows) v[i].store(c.codes + mat * c.code_mat_stride + r * c.code_row_stride, col, c.ne0, inv);
    }
    if (threadIdx.x == 0) c.scales[tile] = m / kF8Top;
}

// Rows that start at any element: a warp per (row, block), lane l on columns l,
// l + 32, l + 64 and l + 96, so that loads and code bytes of a warp are
// adjacent whatever the alignment (16 columns a lane as above took 4 times as
// long: 8192 x 14330 bf16 250 us).
template <int ST>
__device__ __forceinline__ float load_any(const uint8_t *row, int64_t col) {
    if (ST == SHC_SRC_F32) return __ldg(reinterpret_cast<const float *>(row) + col);
    const uint16_t h = __ldg(reinterpret_cast<const uint16_t *>(row) + col);
    return ST == SHC_SRC_BF16 ? bf16_bits_to_f32(h) : f16_val(h);
}
// The block's largest finite magnitude over a warp's v; infinite elements become NaN.
template <int N>
__device__ __forceinline__ float warp_top(float v[N], bool &inf) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++) m = fmaxf(m, fabsf(v[j]));
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    inf = m == inf_f();
    return m;
}
template <int N>
__device__ __forceinline__ float warp_top_finite(float v[N]) {
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < N; j++) {
        if (fabsf(v[j]) == inf_f()) v[j] = __uint_as_float(0x7FFFFFFFu);
        else m = fmaxf(m, fabsf(v[j]));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    return m;
}
__device__ __forceinline__ void store_any(uint8_t *row, int64_t col, int64_t ne0, const float v[4], float inv) {
    const uint32_t lo = e4m3x2(v[0] * inv, v[1] * inv), hi = e4m3x2(v[2] * inv, v[3] * inv);
    if (col < ne0) row[col] = (uint8_t)lo;
    if (col + 32 < ne0) row[col + 32] = (uint8_t)(lo >> 8);
    if (col + 64 < ne0) row[col + 64] = (uint8_t)hi;
    if (col + 96 < ne0) row[col + 96] = (uint8_t)(hi >> 8);
}

template <int ST, typename I>
__global__ void __launch_bounds__(256) f8_encode_rows_any_kernel(F8Codec c) {
    constexpr int kUnits = 4;
    const I nb = (I)((c.ne0 + kF8Block - 1) / kF8Block), total = (I)(c.n_mats * c.n_rows) * nb, rows = (I)c.n_rows;
    const int lane = threadIdx.x & 31;
    const I u0 = (I)blockIdx.x * (8 * kUnits) + threadIdx.x / 32;
    float v[kUnits][4];
    uint8_t *row[kUnits];
    int64_t col[kUnits];
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const I u = u0 + (I)(k * 8);
        const I g = u < total ? u / nb : 0, b = u < total ? u - g * nb : 0;
        const I mat = c.n_mats > 1 ? g / rows : 0, r = g - mat * rows;
        col[k] = u < total ? (int64_t)b * kF8Block + lane : c.ne0;
        row[k] = c.codes + (int64_t)mat * c.code_mat_stride + (int64_t)r * c.code_row_stride;
        const uint8_t *src = src_row<ST>(c, mat, r);
#pragma unroll
        for (int j = 0; j < 4; j++) v[k][j] = col[k] + 32 * j < c.ne0 ? load_any<ST>(src, col[k] + 32 * j) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < kUnits; k++) {
        const I u = u0 + (I)(k * 8);
        bool inf;
        float m = warp_top<4>(v[k], inf);
        if (inf) m = warp_top_finite<4>(v[k]);
        m = fmaxf(m, kF8Least);
        store_any(row[k], col[k], c.ne0, v[k], kF8Top / m);
        if (u < total && lane == 0) c.scales[u] = m / kF8Top;
    }
}

// The same for a 128 x 128 tile: warp w on rows w + 8 i.
template <int ST>
__global__ void __launch_bounds__(256) f8_encode_tiles_any_kernel(F8Codec c) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, rb = (c.n_rows + kF8Block - 1) / kF8Block;
    const int64_t tile = blockIdx.x, b = tile % nb, rest = tile / nb, mat = rest / rb;
    const int64_t row0 = (rest - mat * rb) * kF8Block + threadIdx.x / 32;
    const int64_t col = b * kF8Block + (threadIdx.x & 31);
    __shared__ float s_top[2][8];
    float v[64];
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int64_t r = row0 + 8 * i;
        const uint8_t *src = src_row<ST>(c, mat, r < c.n_rows ? r : 0);
#pragma unroll
        for (int j = 0; j < 4; j++)
            v[4 * i + j] = r < c.n_rows && col + 32 * j < c.ne0 ? load_any<ST>(src, col + 32 * j) : 0.0f;
    }
    bool inf;
    float m = warp_top<64>(v, inf);
    for (int pass = 0; pass < 2; pass++) {
        if ((threadIdx.x & 31) == 0) s_top[pass][threadIdx.x / 32] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < 8; w++) m = fmaxf(m, s_top[pass][w]);
        if (m != inf_f()) break;
        m = warp_top_finite<64>(v);
    }
    m = fmaxf(m, kF8Least);
    const float inv = kF8Top / m;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        const int64_t r = row0 + 8 * i;
        if (r < c.n_rows)
            store_any(c.codes + mat * c.code_mat_stride + r * c.code_row_stride, col, c.ne0, v + 4 * i, inv);
    }
    if (threadIdx.x == 0) c.scales[tile] = m / kF8Top;
}

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A warp per run of a row's columns, kEach adjacent ones a lane and step: 16
// bytes of output where rows of the output start on 16-byte boundaries (so a
// warp's stores are adjacent; 16 codes a lane left 64-byte strides between
// f32 stores, 127 us for 8192 x 14336), else one.
template <typename T, bool VEC, typename I>
__global__ void __launch_bounds__(256) f8_decode_kernel(F8Codec c) {
    constexpr int kEach = VEC ? 16 / (int)sizeof(T) : 1, kSteps = VEC ? 32 / kEach : 16, kRun = 32 * kEach * kSteps;
    const I runs = (I)((c.ne0 + kRun - 1) / kRun), rows = (I)c.n_rows;
    const I u = (I)blockIdx.x * 8 + threadIdx.x / 32, g = u / runs;
    if (g >= (I)(c.n_mats * c.n_rows)) return;
    const I mat = c.n_mats > 1 ? g / rows : 0, r = g - mat * rows;
    const int64_t col0 = (int64_t)(u - g * runs) * kRun + (threadIdx.x & 31) * kEach;
    const int shift = c.block_rows == 1 ? 0 : 7;
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, rb = (c.n_rows + c.block_rows - 1) / c.block_rows;
    const float *scales = c.scales + ((int64_t)mat * rb + (int64_t)(r >> shift)) * nb;
    const uint8_t *codes = c.codes + (int64_t)mat * c.code_mat_stride + (int64_t)r * c.code_row_stride;
    T *out = static_cast<T *>(c.dst) + (int64_t)g * c.ne0;
    uint32_t q[kSteps][kEach > 4 ? 2 : 1];
    float s[kSteps];
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
        const int64_t col = col0 + k * 32 * kEach;
        if (col >= c.ne0) continue;
        s[k] = __ldg(scales + (col >> 7));
        if (kEach == 8) {
            const uint2 w = __ldcs(reinterpret_cast<const uint2 *>(codes + col));
            q[k][0] = w.x;
            q[k][kEach > 4 ? 1 : 0] = w.y;
        } else if (kEach == 4) {
            q[k][0] = __ldcs(reinterpret_cast<const uint32_t *>(codes + col));
        } else {
            q[k][0] = __ldcs(codes + col);
        }
    }
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
        const int64_t col = col0 + k * 32 * kEach;
        if (col >= c.ne0) continue;
        __align__(16) T y[kEach > 1 ? kEach : 2];
#pragma unroll
        for (int i = 0; i < (kEach + 1) / 2; i++) {
            const float2 f = e4m3x2_val((uint16_t)(q[k][i >> 1] >> (16 * (i & 1))));
            y[2 * i] = from_f32<T>(f.x * s[k]);
            y[2 * i + 1] = from_f32<T>(f.y * s[k]);
        }
        if (kEach == 1) out[col] = y[0];
        else *reinterpret_cast<uint4 *>(out + col) = *reinterpret_cast<const uint4 *>(y);
    }
}

// Thread blocks for `items` of `per_block`; 0 where no grid holds them.
unsigned grid_for(int64_t items, int64_t per_block) {
    const int64_t b = (items + per_block - 1) / per_block;
    return b > INT32_MAX ? 0 : (unsigned)b;
}

template <int ST>
cudaError_t encode(const F8Codec &c, bool vec, cudaStream_t st) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block;
    if (c.block_rows != 1) {
        const unsigned g = grid_for(c.n_mats * ((c.n_rows + kF8Block - 1) / kF8Block) * nb, 1);
        if (!g) return cudaErrorInvalidValue;
        if (vec) f8_encode_tiles_kernel<ST><<<g, 256, 0, st>>>(c);
        else f8_encode_tiles_any_kernel<ST><<<g, 256, 0, st>>>(c);
        return cudaGetLastError();
    }
    const int64_t total = c.n_mats * c.n_rows * nb;
    const unsigned g = grid_for(total, vec ? 256 / kLanes * units<ST>() : 32);
    if (!g) return cudaErrorInvalidValue;
    const bool wide = total >= INT32_MAX;
    if (vec && !wide) f8_encode_rows_kernel<ST, uint32_t><<<g, 256, 0, st>>>(c);
    else if (vec) f8_encode_rows_kernel<ST, uint64_t><<<g, 256, 0, st>>>(c);
    else if (!wide) f8_encode_rows_any_kernel<ST, uint32_t><<<g, 256, 0, st>>>(c);
    else f8_encode_rows_any_kernel<ST, uint64_t><<<g, 256, 0, st>>>(c);
    return cudaGetLastError();
}

template <typename T>
cudaError_t decode(const F8Codec &c, bool vec, cudaStream_t st) {
    const int64_t run = vec ? 1024 : 512, units = c.n_mats * c.n_rows * ((c.ne0 + run - 1) / run);
    const unsigned g = grid_for(units, 8);
    if (!g) return cudaErrorInvalidValue;
    const bool wide = units >= INT32_MAX;
    if (vec && !wide) f8_decode_kernel<T, true, uint32_t><<<g, 256, 0, st>>>(c);
    else if (vec) f8_decode_kernel<T, true, uint64_t><<<g, 256, 0, st>>>(c);
    else if (!wide) f8_decode_kernel<T, false, uint32_t><<<g, 256, 0, st>>>(c);
    else f8_decode_kernel<T, false, uint64_t><<<g, 256, 0, st>>>(c);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_f8_encode(const F8Codec &c, cudaStream_t st) {
    const int64_t esz = c.type == SHC_SRC_F32 ? 4 : 2;
    // 128-bit loads where every row starts on a 16-byte boundary
    const bool vec = ((uintptr_t)c.src & 15) == 0 && c.src_row_stride * esz % 16 == 0 &&
                     c.src_mat_stride * esz % 16 == 0;
    if (c.type == SHC_SRC_F32) return encode<SHC_SRC_F32>(c, vec, st);
    if (c.type == SHC_SRC_F16) return encode<SHC_SRC_F16>(c, vec, st);
    return encode<SHC_SRC_BF16>(c, vec, st);
}

cudaError_t launch_f8_decode(const F8Codec &c, cudaStream_t st) {
    const int64_t esz = c.type == SHC_SRC_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)c.dst & 15) == 0 && c.ne0 * esz % 16 == 0;
    if (c.type == SHC_SRC_F32) return decode<float>(c, vec, st);
    if (c.type == SHC_SRC_F16) return decode<__half>(c, vec, st);
    return decode<__nv_bfloat16>(c, vec, st);
}

}  // namespace shc
