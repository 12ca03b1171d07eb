// Products of block-scaled 8-bit matrices, plain or grouped by expert.
//
//   D[m, o] = sum_c  sa[m, c] * sb[c, o / 128] * sum_{i in block c} A[m, i] B[i, o]
//
// A is rows of E4M3 codes with a scale per 128 columns; B is W^T (or W itself
// for the transposed product, the gradient with respect to A's rows) with a
// scale per 128 x 128 tile, so over one 128-long block c of the contraction
// and one 128-wide block of outputs the scale of an output row is one number.
// The tensor cores sum a block's 128 products into TMEM (f32); the epilogue
// warps read that partial sum, and one fused multiply-add per element folds
// it, scaled, into f32 registers.  Nothing is rounded below f32 before the
// final conversion to the output type.
//
// A CTA computes 128 rows x BN columns at a time.  One warp keeps a ring of
// shared-memory stages filled by TMA (128 contraction bytes per row, 128-byte
// swizzle), one thread issues the tcgen05 products of a stage into one of two
// TMEM accumulators, and BN / 32 epilogue warps drain the other.  W is read
// in the same boxes for both products; only its descriptor differs (K-major
// for W^T, MN-major for W).
//
// Rows of an expert (or of the whole matrix) that lie past its end are loaded
// as zeros or as the next expert's rows, and not stored: rows of D depend on
// their own row of A only.
//
// Every wait is bounded (kWaitNs, then SHC_ETIMEOUT in the status word): all
// roles leave their loops, the copies and products in flight are waited for,
// TMEM is freed and the kernel returns.
#include <cuda.h>

#include "f8.cuh"
#include "fuse.cuh"

namespace shc {
namespace {

constexpr int kTileM = 128;
constexpr int kTileK = kF8Block;  // bytes of one stage row, the swizzle's width
constexpr unsigned long long kWaitNs = 4000000000ull;
constexpr int kMmaK = 32;  // contraction length of one tcgen05 product of 8-bit operands

template <int BN>
struct Shape {
    static constexpr int kStages = BN == 128 ? 6 : 4;
    static constexpr int kABytes = kTileM * kTileK, kBBytes = BN * kTileK;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kEpiWarps = BN / 32;  // four per 128 columns, one per 32 TMEM lanes
    static constexpr int kThreads = (kEpiWarps + 2) * 32;
    static constexpr size_t kSmem = (size_t)kStages * kStageBytes + 1024;  // + alignment of the ring
    static constexpr uint32_t kTmemCols = 2 * BN;
};

struct MmArgs {
    const float *a_scales;
    const float *w_scales;
    const void *offsets;
    int offsets_64;
    int64_t n_rows, n_experts;
    int64_t a_scale_stride;
    int64_t w_scale_expert, w_scale_out, w_scale_in;  // strides of a tile's scale: expert, output block, contraction block
    int out;       // output columns
    int blocks_c;  // contraction blocks
    int a_box;     // rows of one box of A
    void *dst;
    int64_t dst_row_stride;
    int dst_type;
    int vec;  // 16-byte stores of whole 8-column groups
    int *status;
};

struct Control {
    unsigned long long full[8], empty[8];
    unsigned long long acc_full[2], acc_empty[2];
    unsigned long long drain;
    uint32_t tmem;
    int abort;
};

// ---------------------------------------------------------------- waits

// True when the phase completed, false after kWaitNs or once another warp gave up.
__device__ __noinline__ bool wait_slow(unsigned long long *b, uint32_t parity, volatile int *abort, int *status) {
    const unsigned long long t0 = global_ns();
    while (!mbar_test(b, parity)) {
        if (*abort) return false;
        if (global_ns() - t0 > kWaitNs) {
            *abort = 1;
            set_status(status, SHC_ETIMEOUT);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool bar_wait(unsigned long long *b, uint32_t parity, volatile int *abort, int *status) {
    return mbar_test(b, parity) || wait_slow(b, parity, abort, status);
}
// After a give-up: wait, bounded, for work that is still in flight.
__device__ __noinline__ void wait_drain(unsigned long long *b, uint32_t parity) {
    const unsigned long long t0 = global_ns();
    while (!mbar_test(b, parity) && global_ns() - t0 < kWaitNs) {
    }
}
__device__ __forceinline__ void expect_tx(unsigned long long *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}

// ---------------------------------------------------------------- TMA, tcgen05

__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, unsigned long long *bar, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, unsigned long long *bar, int x, int y, int z) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// Shared-memory descriptor of a 128-byte-swizzled operand tile.  stride: from
// one group of eight rows to the next; lead (MN-major only): from one 128-byte
// wide group of columns to the next.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: E4M3 operands, f32 accumulator, A K-major.
__host__ __device__ constexpr uint32_t instr_desc(int n, bool b_mn_major) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
}
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
        : "memory");
}
__device__ __forceinline__ void mma_commit(unsigned long long *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 32 consecutive f32 columns of the warp's 32 TMEM lanes, one lane per thread.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t r[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
// Waits for this thread's TMEM loads; r is tied to the wait so that no use of
// it moves ahead.
__device__ __forceinline__ void tmem_wait_ld(uint32_t r[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]),
                   "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]),
                   "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27])
                 :
                 : "memory");
    asm volatile("" : "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31]));
}

// acc += part * (s, s), two f32 fused multiply-adds per instruction.
__device__ __forceinline__ void fma2(uint64_t &acc, uint32_t p0, uint32_t p1, uint64_t s2) {
    asm("{\n .reg .b64 t;\n mov.b64 t, {%1, %2};\n fma.rn.f32x2 %0, t, %3, %0;\n}" : "+l"(acc) : "r"(p0), "r"(p1), "l"(s2));
}

// ---------------------------------------------------------------- tiles

struct Tile {
    int64_t expert, row0, row_end;  // rows [row0, min(row0 + 128, row_end)) of A and D
    int col0;                       // first output column
};

// Hands out the tiles of the grid's CTAs in turn: expert by expert, within an
// expert a column of row tiles before the next column (so CTAs running
// together share W's tiles in L2).  Called by whole warps; experts are looked
// up 32 at a time.  Offsets are clamped to the rows there are, so no tile
// reaches outside A and D whatever they hold.
struct Tiles {
    int64_t t, base, e0;  // base: tiles before expert e0
    int64_t n_out, step;
    const MmArgs &p;
    __device__ Tiles(const MmArgs &args, int bn)
        : t(blockIdx.x), base(0), e0(0), n_out((args.out + bn - 1) / bn), step(gridDim.x), p(args) {}
    __device__ __forceinline__ int64_t offset(int64_t e) const {
        const int64_t v = p.offsets_64 ? static_cast<const int64_t *>(p.offsets)[e]
                                       : (int64_t) static_cast<const int32_t *>(p.offsets)[e];
        return v < 0 ? 0 : v > p.n_rows ? p.n_rows : v;
    }
    __device__ bool next(Tile &o, int bn) {
        const int lane = threadIdx.x & 31;
        for (;;) {
            if (e0 >= p.n_experts) return false;
            int64_t lo = 0, hi = p.n_rows;
            const int64_t e = e0 + lane;
            if (p.offsets) {
                lo = e < p.n_experts ? offset(e) : 0;
                hi = e < p.n_experts ? offset(e + 1) : 0;
            } else if (lane) {
                hi = 0;
            }
            if (hi < lo) hi = lo;
            const int64_t mine = (hi - lo + kTileM - 1) / kTileM * n_out;
            int64_t sum = mine;  // inclusive prefix sum over the lanes
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t v = __shfl_up_sync(~0u, sum, d);
                if (lane >= d) sum += v;
            }
            const unsigned in = __ballot_sync(~0u, t < base + sum);
            if (in) {
                const int l = __ffs(in) - 1;
                const int64_t first = base + __shfl_sync(~0u, sum - mine, l);
                const int64_t elo = __shfl_sync(~0u, lo, l), ehi = __shfl_sync(~0u, hi, l);
                const int64_t at = t - first, mt = (ehi - elo + kTileM - 1) / kTileM;
                o.expert = e0 + l;
                o.col0 = (int)(at / mt) * bn;
                o.row0 = elo + at % mt * kTileM;
                o.row_end = ehi;
                t += step;
                return true;
            }
            base += __shfl_sync(~0u, sum, 31);
            e0 += 32;
        }
    }
};

// ---------------------------------------------------------------- epilogue stores

__device__ __forceinline__ uint32_t pack_f16(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Eight consecutive columns of one row of D.
__device__ __forceinline__ void store8(const MmArgs &p, int64_t row, int col, const float v[8]) {
    const int64_t at = row * p.dst_row_stride + col;
    if (p.dst_type == SHC_SRC_F32) {
        float *d = static_cast<float *>(p.dst) + at;
        if (p.vec && col + 8 <= p.out) {
            reinterpret_cast<float4 *>(d)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4 *>(d)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++)
                if (col + i < p.out) d[i] = v[i];
        }
        return;
    }
    uint16_t *d = static_cast<uint16_t *>(p.dst) + at;
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; i++)
        w[i] = p.dst_type == SHC_SRC_F16 ? pack_f16(v[2 * i], v[2 * i + 1]) : pack_bf16(v[2 * i], v[2 * i + 1]);
    if (p.vec && col + 8 <= p.out) {
        *reinterpret_cast<uint4 *>(d) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (col + i < p.out) d[i] = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
    }
}

// ---------------------------------------------------------------- kernel

template <int BN, bool TRANS>
__global__ void __launch_bounds__(Shape<BN>::kThreads, 1)
    f8_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                      const __grid_constant__ MmArgs p) {
    using S = Shape<BN>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Control ctl;
    const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;  // the swizzle's pattern repeats every 1024 bytes
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; s++) {
            mbar_init(&ctl.full[s], 1);
            mbar_init(&ctl.empty[s], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&ctl.acc_full[i], 1);
            mbar_init(&ctl.acc_empty[i], S::kEpiWarps);
        }
        mbar_init(&ctl.drain, 1);
        ctl.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == S::kEpiWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)),
                     "n"(S::kTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&ctl.tmem);
    volatile int *abort = &ctl.abort;

    Tiles tiles(p, BN);
    Tile tile;
    if (warp == S::kEpiWarps) {
        // ------------------------------------------------ loads
        uint32_t it = 0;
        bool ok = true;
        while (ok && tiles.next(tile, BN)) {
            const int64_t rows = tile.row_end - tile.row0 < kTileM ? tile.row_end - tile.row0 : kTileM;
            const int boxes = (int)((rows + p.a_box - 1) / p.a_box);
            if (lane == 0) {
                for (int c = 0; ok && c < p.blocks_c; c++) {
                    const uint32_t s = it % S::kStages, round = it / S::kStages;
                    if (!bar_wait(&ctl.empty[s], (round & 1) ^ 1, abort, p.status)) {
                        ok = false;
                        break;
                    }
                    const uint32_t a = ring + s * S::kStageBytes, b = a + S::kABytes;
                    expect_tx(&ctl.full[s], boxes * p.a_box * kTileK + S::kBBytes);
                    for (int i = 0; i < boxes; i++)
                        tma_2d(a + i * p.a_box * kTileK, &map_a, &ctl.full[s], c * kTileK, (int)tile.row0 + i * p.a_box);
#pragma unroll
                    for (int j = 0; j < BN / 128; j++) {
                        const int o = tile.col0 + j * 128, x = c * kTileK;
                        tma_3d(b + j * 128 * kTileK, &map_w, &ctl.full[s], TRANS ? o : x, TRANS ? x : o, (int)tile.expert);
                    }
                    it++;
                }
            }
            ok = __shfl_sync(~0u, (int)ok, 0);
        }
        if (lane == 0 && !ok)  // copies still in flight land before the CTA ends
            for (uint32_t k = it > S::kStages ? it - S::kStages : 0; k < it; k++)
                wait_drain(&ctl.full[k % S::kStages], (k / S::kStages) & 1);
    } else if (warp == S::kEpiWarps + 1) {
        // ------------------------------------------------ products
        constexpr uint32_t idesc = instr_desc(BN, TRANS);
        uint32_t it = 0;
        bool ok = true;
        while (ok && tiles.next(tile, BN)) {
            if (lane == 0) {
                for (int c = 0; ok && c < p.blocks_c; c++, it++) {
                    const uint32_t s = it % S::kStages, buf = it & 1;
                    if (!bar_wait(&ctl.acc_empty[buf], ((it >> 1) & 1) ^ 1, abort, p.status) ||
                        !bar_wait(&ctl.full[s], (it / S::kStages) & 1, abort, p.status)) {
                        ok = false;
                        break;
                    }
                    fence_after();
                    const uint32_t a = ring + s * S::kStageBytes, b = a + S::kABytes;
#pragma unroll
                    for (int k = 0; k < kTileK / kMmaK; k++) {
                        const uint64_t da = smem_desc(a + k * kMmaK, 16, 1024);
                        // MN-major: 32 rows of 128 columns further; K-major: 32 bytes along the row
                        const uint64_t db = TRANS ? smem_desc(b + k * kMmaK * 128, 128 * kTileK, 1024)
                                                  : smem_desc(b + k * kMmaK, 16, 1024);
                        mma_f8(tmem + buf * BN, da, db, idesc, k > 0);
                    }
                    mma_commit(&ctl.empty[s]);
                    mma_commit(&ctl.acc_full[buf]);
                }
            }
            ok = __shfl_sync(~0u, (int)ok, 0);
        }
        if (lane == 0 && !ok) {  // products still in flight end before TMEM is freed
            mma_commit(&ctl.drain);
            wait_drain(&ctl.drain, 0);
        }
    } else {
        // ------------------------------------------------ scaling and stores
        const int lanes0 = (warp & 3) * 32, half = warp >> 2;  // TMEM lanes of this warp; its 128 columns
        uint32_t it = 0;
        bool ok = true;
        while (ok && tiles.next(tile, BN)) {
            const int64_t row = tile.row0 + lanes0 + lane;
            const bool mine = row < tile.row_end;
            const int col0 = tile.col0 + half * 128;
            const float *sa = p.a_scales + (mine ? row * p.a_scale_stride : 0);
            // a block of columns wholly past the end has no scale
            const float *sb = p.w_scales + tile.expert * p.w_scale_expert +
                              (col0 < p.out ? (int64_t)(col0 / 128) * p.w_scale_out : 0);
            uint64_t acc[64];
#pragma unroll
            for (int i = 0; i < 64; i++) acc[i] = 0;
            float na = mine ? __ldg(sa) : 0.0f, nb = __ldg(sb);
            for (int c = 0; c < p.blocks_c; c++, it++) {
                const float s = na * nb;
                if (c + 1 < p.blocks_c) {  // the next block's scales, ahead of its sums
                    na = mine ? __ldg(sa + c + 1) : 0.0f;
                    nb = __ldg(sb + (int64_t)(c + 1) * p.w_scale_in);
                }
                const uint32_t buf = it & 1;
                ok = __all_sync(~0u, bar_wait(&ctl.acc_full[buf], (it >> 1) & 1, abort, p.status));
                if (!ok) break;  // the whole warp
                fence_after();
                const uint32_t from = tmem + ((uint32_t)lanes0 << 16) + buf * BN + half * 128;
                uint64_t s2;
                asm("mov.b64 %0, {%1, %1};" : "=l"(s2) : "f"(s));
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    uint32_t r[32];
                    tmem_ld32(from + q * 32, r);
                    tmem_wait_ld(r);
#pragma unroll
                    for (int i = 0; i < 16; i++) fma2(acc[q * 16 + i], r[2 * i], r[2 * i + 1], s2);
                }
                fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ctl.acc_empty[buf]);
            }
            if (ok && mine) {
#pragma unroll
                for (int g = 0; g < 16; g++) {
                    if (col0 + g * 8 >= p.out) break;
                    float v[8];
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        asm("mov.b64 {%0, %1}, %2;" : "=f"(v[2 * i]), "=f"(v[2 * i + 1]) : "l"(acc[g * 4 + i]));
                    store8(p, row, col0 + g * 8, v);
                }
            }
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    if (warp == S::kEpiWarps)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(S::kTmemCols));
}

// ---------------------------------------------------------------- host

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled fn = [] {
        void *f = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess)
            f = nullptr;
        return reinterpret_cast<EncodeTiled>(f);
    }();
    return fn;
}

// Codes [depth][rows][cols] read in boxes of box_rows rows x 128 columns;
// whatever lies outside reads as zero.
bool code_map(CUtensorMap *map, const uint8_t *p, int64_t cols, int64_t rows, int64_t depth, int64_t row_stride,
              int64_t mat_stride, int box_rows, int rank) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)depth};
    const cuuint64_t strides[2] = {(cuuint64_t)row_stride, (cuuint64_t)mat_stride};
    const cuuint32_t box[3] = {kTileK, (cuuint32_t)box_rows, 1}, steps[3] = {1, 1, 1};
    const EncodeTiled f = encode_tiled();
    return f && f(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, (cuuint32_t)rank, const_cast<uint8_t *>(p), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, bool TRANS>
cudaError_t launch(const CUtensorMap &ma, const CUtensorMap &mw, const MmArgs &a, unsigned grid, cudaStream_t st) {
    using S = Shape<BN>;
    int per_sm;
    const cudaError_t e = resident_blocks((const void *)f8_product_kernel<BN, TRANS>, S::kThreads, S::kSmem, &per_sm);
    if (e != cudaSuccess) return e;
    f8_product_kernel<BN, TRANS><<<grid, S::kThreads, S::kSmem, st>>>(ma, mw, a);
    return cudaGetLastError();
}

}  // namespace

int launch_f8_product(const F8Product &p, int num_sms, cudaStream_t st) {
    constexpr int BN = 128;
    const int64_t inner = p.transposed ? p.n : p.k, out = p.transposed ? p.k : p.n;
    MmArgs a{};
    a.a_scales = p.a_scales;
    a.w_scales = p.w_scales;
    a.offsets = p.offsets;
    a.offsets_64 = p.offsets_64;
    a.n_rows = p.n_rows;
    a.n_experts = p.n_experts;
    a.a_scale_stride = p.a_scale_stride;
    const int64_t nb = (p.n + kF8Block - 1) / kF8Block, kb = (p.k + kF8Block - 1) / kF8Block;
    a.w_scale_expert = nb * kb;
    a.w_scale_out = p.transposed ? 1 : kb;
    a.w_scale_in = p.transposed ? kb : 1;
    a.out = (int)out;
    a.blocks_c = (int)((inner + kTileK - 1) / kTileK);
    a.dst = p.dst;
    a.dst_row_stride = p.dst_row_stride;
    a.dst_type = p.dst_type;
    const int64_t esz = p.dst_type == SHC_SRC_F32 ? 4 : 2;
    a.vec = ((uintptr_t)p.dst & 15) == 0 && p.dst_row_stride * esz % 16 == 0;
    a.status = p.status;
    a.a_box = p.n_rows / (p.n_experts > 0 ? p.n_experts : 1) >= kTileM ? kTileM : 32;

    CUtensorMap ma, mw;
    if (!code_map(&ma, p.a, inner, p.n_rows, 1, p.a_row_stride, 0, a.a_box, 2) ||
        !code_map(&mw, p.w, p.k, p.n, p.n_experts, p.w_row_stride, p.w_mat_stride, 128, 3))
        return SHC_EINVAL;
    // Tiles there can be at most: every expert with rows may end in a part tile.
    const int64_t some = p.n_experts < p.n_rows ? p.n_experts : p.n_rows;
    const int64_t most = ((p.n_rows + kTileM - 1) / kTileM + (p.offsets ? some : 0)) * ((out + BN - 1) / BN);
    const unsigned grid = (unsigned)(most < num_sms ? most : num_sms);
    const cudaError_t e = p.transposed ? launch<BN, true>(ma, mw, a, grid, st) : launch<BN, false>(ma, mw, a, grid, st);
    if (e == cudaSuccess) return SHC_OK;
    return e == cudaErrorMemoryAllocation ? SHC_ENOMEM : SHC_ECUDA;
}

}  // namespace shc
