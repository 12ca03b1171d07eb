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
//
// An element is read once and its code written once (the tile kernel holds its
// tile in registers between the maximum and the codes); with rows on 16-byte
// boundaries all three kernels are bound by HBM.  8192 x 14336 bf16 to 1 x 128 blocks 63.2 us (5.63
// TB/s, 0.86 of the measured copy), to tiles 60.8, f32 87-91 us (6.5-6.8
// TB/s); 14336 x 4096 tiles decoded to bf16 28.6 us (6.16 TB/s, 0.94).  Rows
// that start off 16-byte boundaries take longer (8192 x 14330 bf16 97 us, 0.55
// of the copy; f32 101; 4096 x 14331 decoded to bf16 45.8), by what was not
// profiled.
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

    // Columns col.. of the row at p, zeros from ne0 on.  VEC: the row starts
    // on a 16-byte boundary.  Otherwise the aligned 16-byte words around the
    // columns are loaded and shifted into place (elements one by one took 3
    // times as long), as long as they lie within [lo, hi), the source's bytes.
    template <bool VEC>
    __device__ __forceinline__ void load(const uint8_t *p, int64_t col, int64_t ne0, const uint8_t *lo, const uint8_t *hi) {
        constexpr int esz = ST == SHC_SRC_F32 ? 4 : 2;
        const uint8_t *from = p + col * esz;
        const int off = VEC ? 0 : (int)((uintptr_t)from & 15);
        if (col >= ne0) {
            zero();
        } else if (VEC ? col + kElems <= ne0 : from - off >= lo && from - off + 4 * kWords + 16 <= hi) {
            const uint4 *q = reinterpret_cast<const uint4 *>(from - off);
            uint32_t x[kWords + 4];
#pragma unroll
            for (int i = 0; i < kWords / 4 + (VEC ? 0 : 1); i++) {
                const uint4 v = VEC ? __ldcs(q + i) : __ldg(q + i);  // aligned words are read once, others by two lanes
                x[4 * i] = v.x;
                x[4 * i + 1] = v.y;
                x[4 * i + 2] = v.z;
                x[4 * i + 3] = v.w;
            }
            if (!VEC) {
#pragma unroll
                for (int i = 0; i < kWords + 2; i++) x[i] = off & 8 ? x[i + 2] : x[i];
#pragma unroll
                for (int i = 0; i < kWords + 1; i++) x[i] = off & 4 ? x[i + 1] : x[i];
            }
#pragma unroll
            for (int i = 0; i < kWords; i++) w[i] = !VEC && esz == 2 && off & 2 ? __funnelshift_r(x[i], x[i + 1], 16) : x[i];
            if (!VEC && col + kElems > ne0) {
                const int n = (int)(ne0 - col);
#pragma unroll
                for (int i = 0; i < kWords; i++) {
                    if (esz == 4) w[i] = i < n ? w[i] : 0u;
                    else w[i] = 2 * i + 1 < n ? w[i] : 2 * i < n ? w[i] & 0xFFFFu : 0u;
                }
            }
        } else if (ST == SHC_SRC_F32) {
#pragma unroll
            for (int i = 0; i < kWords; i++)
                w[i] = col + i < ne0 ? __ldg(reinterpret_cast<const uint32_t *>(p) + col + i) : 0u;
        } else {
            const uint16_t *q = reinterpret_cast<const uint16_t *>(p) + col;
#pragma unroll
            for (int i = 0; i < kWords; i++) {
                const uint32_t a = col + 2 * i < ne0 ? __ldg(q + 2 * i) : 0u;
                const uint32_t b = col + 2 * i + 1 < ne0 ? __ldg(q + 2 * i + 1) : 0u;
                w[i] = a | b << 16;
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

template <int ST>
__device__ __forceinline__ const uint8_t *src_end(const F8Codec &c) {
    return src_row<ST>(c, c.n_mats - 1, c.n_rows - 1) + c.ne0 * (ST == SHC_SRC_F32 ? 4 : 2);
}

// Activations: eight lanes per (row, block), kUnits of them at once so that a
// warp has kUnits x 4 blocks' loads in flight.  I: unit index type, 32 bits
// wherever the units can be counted in them (a division by the row's blocks
// per unit).
template <int ST>
__host__ __device__ constexpr int units() { return ST == SHC_SRC_F32 ? 2 : 4; }

template <int ST, bool VEC, typename I>
__global__ void __launch_bounds__(256) f8_encode_rows_kernel(F8Codec c) {
    constexpr int kUnits = units<ST>(), kPerBlock = 256 / kLanes;
    const I nb = (I)((c.ne0 + kF8Block - 1) / kF8Block), total = (I)(c.n_mats * c.n_rows) * nb, rows = (I)c.n_rows;
    const int lane = threadIdx.x & (kLanes - 1);
    const I u0 = (I)blockIdx.x * (kPerBlock * kUnits) + threadIdx.x / kLanes;
    const uint8_t *const lo = src_row<ST>(c, 0, 0), *const hi = src_end<ST>(c);
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
        v[k].template load<VEC>(src_row<ST>(c, mat, r), col[k], c.ne0, lo, hi);
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
template <int ST, bool VEC>
__global__ void __launch_bounds__(256) f8_encode_tiles_kernel(F8Codec c) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, rb = (c.n_rows + kF8Block - 1) / kF8Block;
    const int64_t tile = blockIdx.x, b = tile % nb, rest = tile / nb, mat = rest / rb;
    const int64_t row0 = (rest - mat * rb) * kF8Block + threadIdx.x / kLanes;
    const int64_t col = b * kF8Block + (threadIdx.x & (kLanes - 1)) * kElems;
    __shared__ float s_top[2][8];
    const uint8_t *const lo = src_row<ST>(c, 0, 0), *const hi = src_end<ST>(c);
    Raw<ST> v[4];
    float m = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const int64_t r = row0 + 32 * i;
        if (r < c.n_rows) v[i].template load<VEC>(src_row<ST>(c, mat, r), col, c.ne0, lo, hi);
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

template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// A warp per run of a row's columns, 16 bytes of output a lane and step, so
// that a warp's stores are adjacent (16 codes a lane left 64-byte strides
// between f32 stores: 127 us for 8192 x 14336, 90 so).  Where rows of the
// output do not all start on 16-byte boundaries (VEC false) a row's steps
// start at its first one, their codes are shifted into place, and the few
// elements before and after are written one by one by the run at hand.
template <typename T, bool VEC, typename I>
__global__ void __launch_bounds__(256) f8_decode_kernel(F8Codec c) {
    constexpr int kEach = 16 / (int)sizeof(T), kSteps = 32 / kEach, kRun = 32 * kEach * kSteps, kCodes = kEach / 4;
    const I runs = (I)((c.ne0 + kRun - 1) / kRun), rows = (I)c.n_rows;
    const I u = (I)blockIdx.x * 8 + threadIdx.x / 32, g = u / runs;
    if (g >= (I)(c.n_mats * c.n_rows)) return;
    const I mat = c.n_mats > 1 ? g / rows : 0, r = g - mat * rows, run = u - g * runs;
    const int lane = threadIdx.x & 31;
    const int shift = c.block_rows == 1 ? 0 : 7;
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block, rb = (c.n_rows + c.block_rows - 1) / c.block_rows;
    const float *scales = c.scales + ((int64_t)mat * rb + (int64_t)(r >> shift)) * nb;
    const uint8_t *codes = c.codes + (int64_t)mat * c.code_mat_stride + (int64_t)r * c.code_row_stride;
    T *out = static_cast<T *>(c.dst) + (int64_t)g * c.ne0;
    // elements before the row's first 16-byte boundary
    const int head = VEC ? 0 : (int)((16 - ((uintptr_t)out & 15) & 15) / sizeof(T));
    const int64_t col0 = head + (int64_t)run * kRun + lane * kEach;
    uint32_t q[kSteps][kCodes];
    float s[kSteps][2];
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
        const int64_t col = col0 + k * 32 * kEach;
        if (col + kEach > c.ne0) continue;
        s[k][0] = __ldg(scales + (col >> 7));
        if (!VEC) s[k][1] = __ldg(scales + (col + kEach - 1 >> 7));
        // whole words of codes up to the last's
        const uint32_t *w = reinterpret_cast<const uint32_t *>(codes + (col & ~(int64_t)3));
        if (VEC && kCodes == 2) {
            const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(w));
            q[k][0] = v.x;
            q[k][kCodes - 1] = v.y;
        } else {
            uint32_t x[kCodes + 1];
#pragma unroll
            for (int i = 0; i < kCodes; i++) x[i] = VEC ? __ldcs(w + i) : __ldg(w + i);
            x[kCodes] = 0;
            if (!VEC && (head & 3)) {
                const int64_t at = (col & ~(int64_t)3) + 4 * kCodes;
                if (at + 4 <= c.ne0) {
                    x[kCodes] = __ldg(w + kCodes);
                } else {  // nothing past the row's last code is touched
#pragma unroll
                    for (int i = 0; i < 3; i++)
                        if (at + i < c.ne0) x[kCodes] |= (uint32_t)codes[at + i] << (8 * i);
                }
            }
#pragma unroll
            for (int i = 0; i < kCodes; i++) q[k][i] = VEC ? x[i] : __funnelshift_r(x[i], x[i + 1], 8 * (head & 3));
        }
    }
#pragma unroll
    for (int k = 0; k < kSteps; k++) {
        const int64_t col = col0 + k * 32 * kEach;
        if (col + kEach > c.ne0) continue;
        const int in0 = VEC ? kEach : kF8Block - (int)(col & (kF8Block - 1));  // elements in the first block
        __align__(16) T y[kEach];
#pragma unroll
        for (int i = 0; i < kEach; i += 2) {
            const float2 f = e4m3x2_val((uint16_t)(q[k][i >> 2] >> (8 * (i & 2))));
            y[i] = from_f32<T>(f.x * (VEC || i < in0 ? s[k][0] : s[k][1]));
            y[i + 1] = from_f32<T>(f.y * (VEC || i + 1 < in0 ? s[k][0] : s[k][1]));
        }
        *reinterpret_cast<uint4 *>(out + col) = *reinterpret_cast<const uint4 *>(y);
    }
    if (!VEC && run == 0) {
        const int64_t body = (c.ne0 - head) / kEach * kEach, after = c.ne0 > head ? head + body : c.ne0;
        // lanes 0-15: the head; 16-31: what whole steps leave of the row
        const int64_t col = lane < 16 ? lane : after + lane - 16;
        if (lane < 16 ? lane < head && col < c.ne0 : col < c.ne0)
            out[col] = from_f32<T>(e4m3x2_val(codes[col]).x * __ldg(scales + (col >> 7)));
    }
}

// Thread blocks for `items` of `per_block`; 0 where no grid holds them.
unsigned grid_for(int64_t items, int64_t per_block) {
    const int64_t b = (items + per_block - 1) / per_block;
    return b > INT32_MAX ? 0 : (unsigned)b;
}

template <int ST, bool VEC>
cudaError_t encode(const F8Codec &c, cudaStream_t st) {
    const int64_t nb = (c.ne0 + kF8Block - 1) / kF8Block;
    if (c.block_rows != 1) {
        const unsigned g = grid_for(c.n_mats * ((c.n_rows + kF8Block - 1) / kF8Block) * nb, 1);
        if (!g) return cudaErrorInvalidValue;
        f8_encode_tiles_kernel<ST, VEC><<<g, 256, 0, st>>>(c);
        return cudaGetLastError();
    }
    const int64_t total = c.n_mats * c.n_rows * nb;
    const unsigned g = grid_for(total, 256 / kLanes * units<ST>());
    if (!g) return cudaErrorInvalidValue;
    if (total < INT32_MAX) f8_encode_rows_kernel<ST, VEC, uint32_t><<<g, 256, 0, st>>>(c);
    else f8_encode_rows_kernel<ST, VEC, uint64_t><<<g, 256, 0, st>>>(c);
    return cudaGetLastError();
}

template <typename T>
cudaError_t decode(const F8Codec &c, bool vec, cudaStream_t st) {
    const int64_t run = 1024, units = c.n_mats * c.n_rows * ((c.ne0 + run - 1) / run);
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
    if (c.type == SHC_SRC_F32) return vec ? encode<SHC_SRC_F32, true>(c, st) : encode<SHC_SRC_F32, false>(c, st);
    if (c.type == SHC_SRC_F16) return vec ? encode<SHC_SRC_F16, true>(c, st) : encode<SHC_SRC_F16, false>(c, st);
    return vec ? encode<SHC_SRC_BF16, true>(c, st) : encode<SHC_SRC_BF16, false>(c, st);
}

cudaError_t launch_f8_decode(const F8Codec &c, cudaStream_t st) {
    const int64_t esz = c.type == SHC_SRC_F32 ? 4 : 2;
    const bool vec = ((uintptr_t)c.dst & 15) == 0 && c.ne0 * esz % 16 == 0;
    if (c.type == SHC_SRC_F32) return decode<float>(c, vec, st);
    if (c.type == SHC_SRC_F16) return decode<__half>(c, vec, st);
    return decode<__nv_bfloat16>(c, vec, st);
}

}  // namespace shc
