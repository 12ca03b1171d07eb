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
// final conversion to the output type.  Where the two scales multiply to a
// number outside f32's normal range, the sum is multiplied by a power of two
// first and the rest of the product follows, so that a result in f32's range
// does not depend on theirs (see apart).
//
// Twelve warps, each with one job:
//   loads     TMA into a ring of stages: 128 contraction bytes of A's and B's
//             rows, 128-byte swizzle.  W is read in the same boxes for both
//             products; only its descriptor differs (K-major for W^T, MN-major
//             for W).
//   products  two warps issue the even and the odd blocks (tcgen05.mma,
//             kind::f8f6f4), every block into an accumulator of its own.
//   scales    one warp multiplies sa by sb for four blocks at a time and hands
//             them to the epilogue through shared memory, with the tile's
//             place (scales loaded by the epilogue itself stalled it: 401
//             against 309 us for 4096 x 14336 x 4096).
//   epilogue  eight warps drain the accumulators (two per 128 columns, so one
//             fills while the other is read) and store the tile through TMA.
// Tiles are 128 x 128, 128 x 256, or 256 x 256 by a pair of CTAs (each holds
// its own 128 rows of A and half of B, so a block takes 32 KB from L2 per CTA
// where a single one takes 48); plan_for says when.  Where few tiles leave
// SMs idle, a cluster shares a tile's contraction and joins its sums through
// distributed shared memory, in rank order: no atomics, no workspace.
//
// What bounds it (4096 x 14336 x 4096, a pair's 256 x 256 tiles, 218-253 us,
// 1.90-2.21 PFLOP/s, with the clock that the power limit leaves; the parts were
// timed where the whole took 227): the products alone take 138 us (514 cycles
// a block, their rate), the loads alone 113 us (17 TB/s from L2), but a block passes in 865 cycles, because
// an epilogue warp needs that long to wait for, read and scale its 128
// columns.  With one multiply-add in eight it took 202 us, without the stores
// 217, without either 164 (where the whole took 227).  Sixteen
// narrower epilogue warps took 247 us (more instructions), 32-column TMEM
// loads 290 (spilled), a single warp issuing products and acknowledging on
// two barriers a block 301.
//
// Rows of a tile that lie past the end of their expert (or of the whole
// matrix) are loaded as zeros or as the next expert's rows, or, behind the last
// box that holds a row, not at all (the stage keeps what was there).  They are
// not stored: rows of D depend on their own row of A only.
//
// Every wait is bounded (kWaitNs, then SHC_ETIMEOUT in the status word): all
// roles of all CTAs of the cluster leave their loops, and the kernel returns.
// Whether it finished or gave up, no CTA ends before what can still reach it
// has: the loading thread waits for its stages' products, or after a give-up
// for the copies themselves, the product warps for their last products, and
// the loading threads of a pair, whose copies all signal the leader, tell one
// another how many blocks they issued, so that the one behind can issue the
// copies that the other's barrier phases wait for.
#include <cuda.h>

#include "f8.cuh"
#include "fuse.cuh"

#include <type_traits>

namespace shc {
namespace {

constexpr int kTileM = 128;           // rows of one CTA's tile
constexpr int kTileK = kF8Block;      // bytes of one stage row, the swizzle's width
constexpr int kMmaK = 32;             // contraction length of one tcgen05 product of 8-bit operands
constexpr int kSlotBlocks = 4;        // contraction blocks whose scales share a slot
constexpr int kSlots = 3;             // of scales on their way
constexpr int kPieceBytes = 32 * 64;  // a warp's staging of 32 output rows x 64 bytes
// Registers: 384 threads start with 168 each, three warps to a scheduler (504
// of its 512 x 32).  The eight epilogue warps hold up to 128 sums a thread and
// take 216, the other four keep 72: 2 x 216 + 72 = 504.
constexpr int kEpiRegs = 216, kOtherRegs = 72;
constexpr unsigned long long kWaitNs = 4000000000ull;

// BN output columns per tile; PAIR CTAs (a cluster of one or two) work on one
// tile of PAIR x 128 rows.
template <int BN, int PAIR>
struct Shape {
    static constexpr int kBRows = BN / PAIR;  // rows of B that one CTA holds
    static constexpr int kABytes = kTileM * kTileK, kBBytes = kBRows * kTileK;
    static constexpr int kStageBytes = kABytes + kBBytes;
    static constexpr int kStages = 163840 / kStageBytes;  // 160 KB
    static constexpr int kEpiWarps = 8;                   // two for each 32 TMEM lanes
    static constexpr int kThreads = (kEpiWarps + 4) * 32;
    // All of TMEM: each 128-column half of the tile has accumulators of its
    // own, so the epilogue drains one half while the other is summed.
    static constexpr int kHalves = BN / 128;
    static constexpr int kBufs = 512 / BN;
    static_assert(kBufs < kStages, "see the order of the product warps' waits");
    static constexpr int kGroups = BN / 128;  // groups of 64 columns that one epilogue warp drains
    // [block][BN / 128][128 rows], of products of scales; behind them as many powers of two (see kFar)
    static constexpr int kScales = kSlotBlocks * BN, kSlotBytes = 2 * kScales * 4;
    static constexpr size_t kSmem =
        (size_t)kStages * kStageBytes + kEpiWarps * kPieceBytes + kSlots * kSlotBytes + 1024;  // + alignment
};

struct MmArgs {
    const float *a_scales;
    const float *w_scales;
    const void *offsets;
    int offsets_64;
    int n_rows, n_experts;
    int64_t a_scale_stride;
    int64_t w_scale_expert, w_scale_out, w_scale_in;  // strides of a tile's scale: expert, output block, contraction block
    int out;       // output columns
    int blocks_c;  // contraction blocks
    int a_box;     // rows of one box of A
    int split;     // CTAs (a cluster of them) that share a tile's contraction
    void *dst;
    int64_t dst_row_stride;
    int dst_type;
    int align;      // bytes that every row of dst starts on a multiple of: 16, 8 or fewer
    int tma_store;  // map_d describes dst
    int *status;
};

struct Control {
    unsigned long long full[5];    // a stage's bytes have landed
    unsigned long long done[5];    // its products are done: it is free
    struct {
        unsigned long long full, empty;  // an accumulator holds a block's sums; they have been read
    } acc[2][4];  // [half][buffer]
    unsigned long long slot_full[kSlots], slot_empty[kSlots];
    unsigned long long drain[2];  // a product warp's products are done, all of them
    unsigned long long met;       // the other CTA of the pair has written `issued`
    int4 slot[kSlots];  // what a slot's scales are for: first row of this CTA, end of rows, first column, blocks (see kLast)
    int4 joined;  // SPLIT: first row, rows and first column of the tile whose sums are in the ring
    uint32_t tmem;
    uint32_t issued;  // blocks that the other CTA of the pair has issued copies for
    int abort;
};
constexpr int kLast = 256;  // added to a slot's blocks where they are the tile's last ones
constexpr int kFar = 512;   // added where the products of scales go with powers of two

// ---------------------------------------------------------------- waits

// To a shared address of another CTA of the cluster (or of this one).
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t rank, uint32_t v) {
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n st.shared::cluster.u32 [a], %2;\n}" ::"r"(addr),
                 "r"(rank), "r"(v)
                 : "memory");
}
__device__ __forceinline__ bool bar_test(unsigned long long *b, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
        : "=r"(ok)
        : "r"(smem_u32(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
// Ends the waits of every CTA of the cluster (of this one, where there is none).
__device__ __forceinline__ void give_up(volatile int *abort, int *status) {
    uint32_t n;
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(n));
#pragma unroll 1
    for (uint32_t r = 0; r < n; r++) st_cluster(smem_u32(const_cast<const int *>(abort)), r, 1);
    set_status(status, SHC_ETIMEOUT);
}
// True when the phase completed, false after kWaitNs or once a warp of the
// cluster gave up.  The clock is read on every 256th try only: reading it takes longer than
// most waits.  (Inline: a call would spill the epilogue's sums.)
__device__ __forceinline__ bool bar_wait(unsigned long long *b, uint32_t parity, volatile int *abort, int *status) {
    unsigned long long t0 = 0;
#pragma unroll 1
    for (uint32_t i = 1;; i++) {
        if (bar_test(b, parity)) return true;
        if (i % 256) continue;
        if (*abort) return false;
        const unsigned long long t = global_ns();
        if (t0 == 0) t0 = t;
        if (t - t0 > kWaitNs) {
            give_up(abort, status);
            return false;
        }
    }
}
// One lane of a converged warp, known to the compiler to be one (so that what
// it alone executes can be kept in uniform registers, which tcgen05 needs).
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(one));
    return one != 0;
}
// For a whole warp: one try by all lanes, then one lane waits for all (32
// pollers a barrier slow the others down).  The lanes that did not see the
// phase complete themselves are ordered behind the one that did by
// __syncwarp; the shuffle alone orders no memory.
__device__ __forceinline__ bool warp_wait(unsigned long long *b, uint32_t parity, volatile int *abort, int *status) {
    if (__all_sync(~0u, bar_test(b, parity))) return true;
    int ok = 1;
    if ((threadIdx.x & 31) == 0) ok = bar_wait(b, parity, abort, status);
    ok = __shfl_sync(~0u, ok, 0);
    __syncwarp();
    return ok;
}
// For work in flight, which ends whether or not the kernel gave up: bounded by time alone.
__device__ __forceinline__ void wait_drain(unsigned long long *b, uint32_t parity) {
    const unsigned long long t0 = global_ns();
    while (!bar_test(b, parity) && global_ns() - t0 < kWaitNs) {
    }
}
__device__ __forceinline__ void expect_tx(unsigned long long *b, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}

__device__ __forceinline__ void st_shared(uint32_t addr, float v) {
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// ---------------------------------------------------------------- TMA, tcgen05

// Loads signal `bar`, an address in the cluster's shared window: the CTA's
// own barrier, or in a pair the leader's.
template <int PAIR>
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y) {
    if (PAIR == 2)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
            "l"(map), "r"(bar), "r"(x), "r"(y)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
            "l"(map), "r"(bar), "r"(x), "r"(y)
            : "memory");
}
template <int PAIR>
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z) {
    if (PAIR == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
            "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
            "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
            : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap *map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src),
                 "r"(x), "r"(y)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// This thread's stores have read their shared memory / are complete.
__device__ __forceinline__ void store_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void store_wait() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// f32 at a shared address of another CTA of the cluster.
__device__ __forceinline__ float ld_cluster(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.f32 %0, [a];\n}"
        : "=f"(v)
        : "r"(addr), "r"(rank)
        : "memory");
    return v;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
// The same shared address in the leader CTA of the pair.
__device__ __forceinline__ uint32_t in_leader(uint32_t addr) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}
// Arrives on a barrier of this CTA or, in a pair, of the leader.  (What is
// handed over is TMEM, ordered by tcgen05.fence; a release at cluster scope
// would wait for the warp's outstanding memory operations: 1150 cycles a
// block.)
template <int PAIR>
__device__ __forceinline__ void arrive_cluster(uint32_t bar) {
    if (PAIR == 2) asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
    else asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// The loading threads of a pair meet, each once, and tell one another how many
// blocks they have issued copies for.  Returns the other's (0 if it did not come).
__device__ __forceinline__ uint32_t meet(Control &ctl, uint32_t rank, uint32_t issued) {
    st_cluster(smem_u32(&ctl.issued), rank ^ 1, issued);
    asm volatile(
        "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n}" ::"r"(
            smem_u32(&ctl.met)),
        "r"(rank ^ 1)
        : "memory");
    uint32_t ok = 0;
    const unsigned long long t0 = global_ns();
    while (!ok && global_ns() - t0 < kWaitNs)
        asm volatile(
            "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], 0;\n selp.u32 %0, 1, 0, p;\n}"
            : "=r"(ok)
            : "r"(smem_u32(&ctl.met))
            : "memory");
    return ok ? *reinterpret_cast<volatile uint32_t *>(&ctl.issued) : 0;
}
template <bool CLUSTER>
__device__ __forceinline__ void sync_all() {
    if (CLUSTER) {
        asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    } else {
        __syncthreads();
    }
}

// Shared-memory descriptor of a 128-byte-swizzled operand tile.  stride: from
// one group of eight rows to the next; lead (MN-major only): from one 128-byte
// wide group of columns to the next.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) |
           (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: E4M3 operands, f32 accumulator, A K-major.
__host__ __device__ constexpr uint32_t instr_desc(int m, int n, bool b_mn_major) {
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
template <int PAIR>
__device__ __forceinline__ void mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    if (PAIR == 2)
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
    else
        asm volatile(
            "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
            " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d),
            "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)add)
            : "memory");
}
// Arrives on the barrier (in a pair: on both CTAs' barriers at this address)
// when the products issued so far are done.
template <int PAIR>
__device__ __forceinline__ void mma_commit(unsigned long long *bar) {
    if (PAIR == 2)
        asm volatile(
            "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                smem_u32(bar)),
            "h"((uint16_t)3)
            : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                     : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// 16 consecutive f32 columns of the warp's 32 TMEM lanes, one lane per thread.
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t r[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
}
// Waits for this thread's TMEM loads; r is tied to the wait so that no use of
// it moves ahead.
__device__ __forceinline__ void tmem_wait_ld(uint32_t r[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// ---------------------------------------------------------------- tiles

struct Tile {
    int expert, row0, row_end;  // rows [row0, min(row0 + TM, row_end)) of A and D
    int col0;                   // first output column
};

// Hands out tiles of TM x BN to the grid's CTAs (or pairs) in turn: expert by expert, within an
// expert a column of row tiles before the next column (so CTAs running
// together share W's tiles in L2).  Called by whole warps; experts are looked
// up 32 at a time.  Offsets are clamped to the rows there are and to the
// largest one before them, so that whatever they hold no tile reaches outside
// A and D, no row is in two tiles, and there are most_tiles at most (a cluster
// that shares a contraction takes one tile only: its sums lie in the ring).
template <int BN, int PAIR>
struct Tiles {
    static constexpr int TM = kTileM * PAIR;
    int64_t t, base;  // base: tiles before expert e0
    int e0, least;   // least: the largest offset before e0's
    const MmArgs &p;
    __device__ __forceinline__ Tiles(const MmArgs &args) : t(blockIdx.x / (PAIR * args.split)), base(0), e0(0), least(0), p(args) {}
    __device__ __forceinline__ int offset(int e) const {
        const int64_t v = p.offsets_64 ? static_cast<const int64_t *>(p.offsets)[e]
                                       : (int64_t) static_cast<const int32_t *>(p.offsets)[e];
        return v < 0 ? 0 : v > p.n_rows ? p.n_rows : (int)v;
    }
    __device__ __forceinline__ bool next(Tile &o) {
        const int lane = threadIdx.x & 31;
        const int n_out = (p.out + BN - 1) / BN;
        for (;;) {
            if (e0 >= p.n_experts) return false;
            int lo = 0, hi = lane ? 0 : p.n_rows;
            if (p.offsets) {
                const int e = e0 + lane;
                lo = e < p.n_experts ? offset(e) : 0;
                hi = e < p.n_experts ? offset(e + 1) : 0;
                if (__any_sync(~0u, e < p.n_experts && (lo < least || hi < lo))) {  // offsets that decrease
                    lo = lo < least ? least : lo;
                    for (int d = 1; d < 32; d <<= 1) {
                        const int v = __shfl_up_sync(~0u, lo, d);
                        if (lane >= d && v > lo) lo = v;
                    }
                    if (hi < lo) hi = lo;
                }
            }
            const int64_t mine = (int64_t)(((uint32_t)(hi - lo) + TM - 1) / TM) * n_out;
            int64_t sum = mine;  // inclusive prefix sum over the lanes
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t v = __shfl_up_sync(~0u, sum, d);
                if (lane >= d) sum += v;
            }
            const unsigned in = __ballot_sync(~0u, t < base + sum);
            if (in) {
                const int l = __ffs(in) - 1;
                const uint32_t at = (uint32_t)(t - base - __shfl_sync(~0u, sum - mine, l));  // below 2^31: one expert's tiles
                lo = __shfl_sync(~0u, lo, l);
                hi = __shfl_sync(~0u, hi, l);
                const uint32_t mt = ((uint32_t)(hi - lo) + TM - 1) / TM, ct = at / mt;
                o.expert = e0 + l;
                o.col0 = (int)ct * BN;
                o.row0 = lo + (int)(at - ct * mt) * TM;
                o.row_end = hi;
                t += gridDim.x / (PAIR * p.split);
                return true;
            }
            base += __shfl_sync(~0u, sum, 31);
            least = __shfl_sync(~0u, hi, 31);  // of 32 experts; with fewer this was the last look
            e0 += 32;
        }
    }
};

// ---------------------------------------------------------------- epilogue stores

__device__ __forceinline__ uint32_t pack_f16(float2 v) {
    const __half2 h = __floats2half2_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float2 v) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// A warp's 32 x 64 sums (lane = row) to D, 64 bytes of each row at a time
// through `stage` (32 rows x 64 bytes, 16-byte pieces swizzled as TMA's
// 64-byte mode does, so both sides are free of bank conflicts): by one TMA
// store where all 32 rows may be written, else row by row.
template <int DT>
__device__ __forceinline__ void store_rows(const MmArgs &p, const CUtensorMap *map_d, uint32_t stage, const float2 acc[32],
                                           int row0, int row_end, int col0) {
    constexpr int esz = DT == SHC_SRC_F32 ? 4 : 2;
    constexpr int kCols = 64 / esz;  // columns of 64 bytes
    constexpr int kPer = 16 / esz;   // columns of 16 bytes
    const int lane = threadIdx.x & 31;
    // rows past the end may be written only where TMA clips them
    const bool tma = p.tma_store && (row0 + 32 <= row_end || row_end == p.n_rows);
#pragma unroll
    for (int q = 0; q < 64 / kCols; q++) {
        const int col = col0 + q * kCols;
        if (col >= p.out) break;
        if (lane == 0) store_wait_read();  // the piece before this one has left the stage
        __syncwarp();
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float2 *v = acc + (q * kCols + k * kPer) / 2;
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                if (DT == SHC_SRC_F32) w[i] = __float_as_uint(i & 1 ? v[i / 2].y : v[i / 2].x);
                else w[i] = DT == SHC_SRC_F16 ? pack_f16(v[i % (kPer / 2)]) : pack_bf16(v[i % (kPer / 2)]);
            }
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 64 + ((k ^ (lane >> 1 & 3)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
        }
        if (tma) {
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) tma_store_2d(map_d, stage, col, row0);
            continue;
        }
        __syncwarp();
        const int rows = row_end - row0 < 32 ? row_end - row0 : 32;
        uint8_t *d = static_cast<uint8_t *>(p.dst) + ((int64_t)row0 * p.dst_row_stride + col) * esz;
        const int64_t pitch = p.dst_row_stride * esz;
        // Rows of the piece: 16 bytes a lane where rows of D start on 16-byte
        // boundaries, 8 where they start on 8-byte ones, else single elements.
        if (p.align >= 16 && col + kCols <= p.out) {
            for (int r = lane >> 2; r < rows; r += 8) {
                uint32_t w[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                             : "r"(stage + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) << 4)));
                *reinterpret_cast<uint4 *>(d + r * pitch + (lane & 3) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
            }
        } else if (p.align == 8 && col + kCols <= p.out) {
            const int k = lane & 7;
            for (int r = lane >> 3; r < rows; r += 4) {
                uint32_t w[2];
                asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];"
                             : "=r"(w[0]), "=r"(w[1])
                             : "r"(stage + r * 64 + (((k >> 1) ^ (r >> 1 & 3)) << 4) + (k & 1) * 8));
                *reinterpret_cast<uint2 *>(d + r * pitch + k * 8) = make_uint2(w[0], w[1]);
            }
        } else {
            // kCols columns of 32 / kCols rows at once
            const int c = lane % kCols;
            if (col + c < p.out) {
                for (int r = lane / kCols; r < rows; r += 32 / kCols) {
                    const uint32_t at = stage + r * 64 + ((((c / kPer) ^ (r >> 1 & 3)) << 4) | (c % kPer) * esz);
                    if (DT == SHC_SRC_F32) {
                        uint32_t v;
                        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
                        *reinterpret_cast<uint32_t *>(d + r * pitch + c * 4) = v;
                    } else {
                        uint16_t v;
                        asm volatile("ld.shared.b16 %0, [%1];" : "=h"(v) : "r"(at));
                        *reinterpret_cast<uint16_t *>(d + r * pitch + c * 2) = v;
                    }
                }
            }
        }
        __syncwarp();
    }
}

// ---------------------------------------------------------------- scales

// m passes the span where a scale looked at lies outside a range: rows' from
// 2^-100 to 2^100, weights' from 2^-26 to 2^26, negative ones and NaN outside.
// Within, their product is a normal number for certain.  (A look at every
// product took twice the operations and 2 to 3 % of the large products' time,
// this takes 1 %.)
__device__ __forceinline__ void look(uint32_t &m, float scale, uint32_t least) {
    const uint32_t v = __float_as_uint(scale) - least;
    m = m > v ? m : v;
}
constexpr uint32_t kLeastA = (127u - 100) << 23, kSpanA = 200u << 23, kLeastW = (127u - 26) << 23, kSpanW = 52u << 23;

// The product of two scales as .x times .y, a power of two: the f32 product
// and 1 where that is a normal number.  A block's sum is 0 or between 2^-18
// and 2^25 and is multiplied by .y first, which is exact for 2^-96 and 2^96.
// .x is then a normal number wherever the result can lie in f32's range: it
// falls under 2^-126 for products under 2^-222, and would be infinite for
// products over 2^224, which no sum but 0 brings back (so it is the largest
// number instead, and a sum of 0 gives 0).
__device__ __forceinline__ float2 apart(float x, float y) {
    const bool less = fabsf(x) < fabsf(y);
    const float small = less ? x : y, large = less ? y : x, product = x * y;
    constexpr float kTiny = 0x1p-126f, kHuge = 0x1.fffffep127f, kDown = 0x1p-96f, kUp = 0x1p96f;
    if (fabsf(product) < kTiny) return make_float2(small * kUp * large, kDown);
    if (fabsf(product) > kHuge && fabsf(large) <= kHuge) {
        const float v = large * kDown * small;
        return make_float2(copysignf(fminf(fabsf(v), kHuge), v), kUp);
    }
    return make_float2(product, 1.0f);
}

// ---------------------------------------------------------------- kernel

// Four columns of one row of D, for the joined parts of a split tile.
__device__ __forceinline__ void store4(const MmArgs &p, int row, int col, const float v[4]) {
    const int64_t at = (int64_t)row * p.dst_row_stride + col;
    const bool whole = p.align >= 16 && col + 4 <= p.out;
    if (p.dst_type == SHC_SRC_F32) {
        float *d = static_cast<float *>(p.dst) + at;
        if (whole) {
            *reinterpret_cast<float4 *>(d) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 4; i++)
                if (col + i < p.out) d[i] = v[i];
        }
        return;
    }
    uint16_t *d = static_cast<uint16_t *>(p.dst) + at;
    const float2 lo = make_float2(v[0], v[1]), hi = make_float2(v[2], v[3]);
    const uint2 w = p.dst_type == SHC_SRC_F16 ? make_uint2(pack_f16(lo), pack_f16(hi)) : make_uint2(pack_bf16(lo), pack_bf16(hi));
    if (whole) {
        *reinterpret_cast<uint2 *>(d) = w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (col + i < p.out) d[i] = (uint16_t)((i < 2 ? w.x : w.y) >> (16 * (i & 1)));
    }
}

// SPLIT (with BN = 128, PAIR = 1): a cluster of p.split CTAs shares one tile,
// each taking an equal run of its contraction blocks.  They leave their sums
// in their rings, which nothing else uses by then, and each adds up (always
// in rank order) and stores its share of the columns.
template <int BN, int PAIR, bool TRANS, bool SPLIT>
__global__ void __launch_bounds__(Shape<BN, PAIR>::kThreads, 1)
    f8_product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_w,
                      const __grid_constant__ CUtensorMap map_d, const __grid_constant__ MmArgs p) {
    using S = Shape<BN, PAIR>;
    extern __shared__ uint8_t smem_raw[];
    __shared__ Control ctl;
    const uint32_t ring = (smem_u32(smem_raw) + 1023) & ~1023u;  // the swizzle's pattern repeats every 1024 bytes
    const int warp = threadIdx.x / 32, lane = threadIdx.x & 31;
    const int rank = PAIR == 2 ? (int)cluster_rank() : 0;
    const int part = SPLIT ? (int)cluster_rank() : 0;
    const int c_begin = SPLIT ? p.blocks_c * part / p.split : 0;  // this CTA's contraction blocks
    const int blocks = SPLIT ? p.blocks_c * (part + 1) / p.split - c_begin : p.blocks_c;

    if (threadIdx.x == 0) {
        for (int s = 0; s < S::kStages; s++) {
            mbar_init(&ctl.full[s], 1);
            mbar_init(&ctl.done[s], 1);
        }
        for (int h = 0; h < S::kHalves; h++)
            for (int i = 0; i < S::kBufs; i++) {
                mbar_init(&ctl.acc[h][i].full, 1);
                mbar_init(&ctl.acc[h][i].empty, S::kEpiWarps / S::kHalves * PAIR);
            }
        for (int i = 0; i < kSlots; i++) {
            mbar_init(&ctl.slot_full[i], 1);
            mbar_init(&ctl.slot_empty[i], S::kEpiWarps);
        }
        for (int i = 0; i < 2; i++) mbar_init(&ctl.drain[i], 1);
        mbar_init(&ctl.met, 1);
        ctl.abort = 0;
        ctl.joined = make_int4(0, 0, 0, 0);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == S::kEpiWarps) {
        if (PAIR == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)), "n"(512)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&ctl.tmem)), "n"(512)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    }
    fence_before();
    __syncthreads();
    if (PAIR == 2) sync_all<true>();  // both CTAs' barriers are set up
    fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(&ctl.tmem);
    volatile int *abort = &ctl.abort;

    const uint32_t stages = ring + S::kStages * S::kStageBytes;  // of the epilogue, then the slots of scales
    float *const slots = reinterpret_cast<float *>(smem_raw + (stages - smem_u32(smem_raw)) + S::kEpiWarps * kPieceBytes);
    if (warp >= S::kEpiWarps) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        Tiles<BN, PAIR> tiles(p);
        Tile tile;
        if (warp == S::kEpiWarps) {
            // ------------------------------------------------ loads
            struct Boxes {
                int mine;        // boxes of A for this CTA
                uint32_t bytes;  // of a block, both CTAs'
            };
            const auto boxes_of = [&](const Tile &tile) {
                int boxes[PAIR];  // of A, for each CTA
#pragma unroll
                for (int r = 0; r < PAIR; r++) {
                    int rows = tile.row_end - tile.row0 - r * kTileM;
                    rows = rows < 0 ? 0 : rows > kTileM ? kTileM : rows;
                    boxes[r] = (rows + p.a_box - 1) / p.a_box;
                }
                Boxes b{PAIR == 2 && rank ? boxes[PAIR - 1] : boxes[0], 0};
#pragma unroll
                for (int r = 0; r < PAIR; r++) b.bytes += boxes[r] * p.a_box * kTileK + S::kBBytes;
                return b;
            };
            const auto issue = [&](const Tile &tile, const Boxes &boxes, uint32_t s, int c) {
                const uint32_t a = ring + s * S::kStageBytes, b = a + S::kABytes;
                uint32_t bar = smem_u32(&ctl.full[s]);
                if (rank == 0) expect_tx(&ctl.full[s], boxes.bytes);  // the leader counts both CTAs' bytes
                if (PAIR == 2) bar = in_leader(bar);
                for (int i = 0; i < boxes.mine; i++)
                    tma_2d<PAIR>(a + i * p.a_box * kTileK, &map_a, bar, c * kTileK, tile.row0 + rank * kTileM + i * p.a_box);
#pragma unroll
                for (int j = 0; j < S::kBRows / 128; j++) {
                    const int o = tile.col0 + rank * S::kBRows + j * 128, x = c * kTileK;
                    tma_3d<PAIR>(b + j * 128 * kTileK, &map_w, bar, TRANS ? o : x, TRANS ? x : o, tile.expert);
                }
            };
            uint32_t it = 0;
            bool ok = true;
            while (ok && tiles.next(tile)) {
                const Boxes boxes = boxes_of(tile);
                if (elect_one()) {
                    for (int c = c_begin; c < c_begin + blocks; c++) {
                        const uint32_t s = it % S::kStages, round = it / S::kStages;
                        if (!bar_wait(&ctl.done[s], (round & 1) ^ 1, abort, p.status)) {
                            ok = false;
                            break;
                        }
                        issue(tile, boxes, s, c);
                        it++;
                    }
                }
                ok = __all_sync(~0u, (int)ok);
            }
            // From here on to the end of what is in flight for this CTA.
            it = __reduce_max_sync(~0u, it);
            if (PAIR == 2) {
                uint32_t other = 0;
                if (elect_one()) other = meet(ctl, rank, it);
                other = __reduce_max_sync(~0u, other);
                if (it < other) {
                    // After a give-up: the other CTA has loaded into stages, so they were free in both, and the
                    // copies that complete their phases can be issued without a wait.
                    Tiles<BN, PAIR> again(p);
                    for (uint32_t k = 0; k < other && again.next(tile); k += blocks) {
                        const Boxes boxes = boxes_of(tile);
                        if (elect_one())
                            for (uint32_t c = k < it ? it - k : 0; c < (uint32_t)blocks && k + c < other; c++)
                                issue(tile, boxes, (k + c) % S::kStages, (int)c);
                    }
                    it = other;
                }
            }
            if (elect_one()) {
                const uint32_t last = it > S::kStages ? it - S::kStages : 0;
                for (uint32_t k = last; k < it && ok; k++)
                    ok = bar_wait(&ctl.done[k % S::kStages], (k / S::kStages) & 1, abort, p.status);
                if (rank == 0) {
                    for (uint32_t k = last; k < it && !ok; k++) wait_drain(&ctl.full[k % S::kStages], (k / S::kStages) & 1);
                } else {  // its copies signal the leader, which waits for them; the leader's products signal here
                    wait_drain(&ctl.drain[0], 0);
                    wait_drain(&ctl.drain[1], 0);
                }
            }
        } else if (warp < S::kEpiWarps + 3) {
            // ------------------------------------------------ products (of a pair: issued by its leader)
            // Every block's sum starts afresh in its own accumulator, so two
            // warps issue the even and the odd blocks without regard to one
            // another; one thread's waits and issues take longer than a
            // block's products.
            const uint32_t me = warp - (S::kEpiWarps + 1);
            constexpr uint32_t idesc = instr_desc(kTileM * PAIR, 128, TRANS);
            const uint64_t da0 = smem_desc(ring, 16, 1024);
            const uint64_t db0 = TRANS ? smem_desc(ring + S::kABytes, 128 * kTileK, 1024) : smem_desc(ring + S::kABytes, 16, 1024);
            // the next 32 of the contraction: MN-major 32 rows of 128 columns further, K-major 32 bytes along the row
            constexpr uint64_t kStepA = kMmaK >> 4, kStepB = (TRANS ? kMmaK * 128 : kMmaK) >> 4;
            // The half's columns of B.  A CTA of a pair holds 128 adjacent columns, 64 of either half.
            constexpr uint64_t kHalfB = (TRANS && PAIR == 2 ? 64 : 128 / PAIR * kTileK) >> 4;
            uint32_t it = me, s = me, phase = 0;  // this warp's block, counted over all tiles; its stage
            uint32_t first = me;                  // its first block in the tile
            bool ok = rank == 0;
            while (ok && tiles.next(tile)) {
                if (elect_one()) {
                    for (uint32_t c = first; c < (uint32_t)blocks; c += 2, it += 2) {
                        const uint32_t buf = it % S::kBufs, acc_phase = ((it / S::kBufs) & 1) ^ 1;
                        const uint64_t da = da0 + (uint64_t)(s * (S::kStageBytes >> 4)), db = db0 + (uint64_t)(s * (S::kStageBytes >> 4));
#pragma unroll
                        for (int h = 0; h < S::kHalves; h++) {
                            ok = bar_wait(&ctl.acc[h][buf].empty, acc_phase, abort, p.status);
                            // After the first of those: it says that block it - kBufs was drained, so block
                            // it - kStages before it has landed and `phase` cannot mean the one before that
                            // (the other warp's block, which this one never waited for).
                            if (h == 0) ok = ok && bar_wait(&ctl.full[s], phase, abort, p.status);
                            if (!ok) break;
                            fence_after();
#pragma unroll
                            for (int k = 0; k < kTileK / kMmaK; k++)
                                mma_f8<PAIR>(tmem + (h * S::kBufs + buf) * 128, da + k * kStepA, db + h * kHalfB + k * kStepB,
                                             idesc, k > 0);
                            mma_commit<PAIR>(&ctl.acc[h][buf].full);
                        }
                        if (!ok) break;
                        mma_commit<PAIR>(&ctl.done[s]);
                        s += 2;
                        if (s >= S::kStages) s -= S::kStages, phase ^= 1;
                    }
                }
                first = (first + blocks) & 1;
                ok = __all_sync(~0u, (int)ok);
            }
            if (rank == 0 && elect_one()) {  // its products end before TMEM is freed
                mma_commit<PAIR>(&ctl.drain[me]);
                wait_drain(&ctl.drain[me], 0);
            }
        } else {
            // ------------------------------------------------ tiles and their scales for the epilogue
            constexpr int kHalves = BN / 128;
            uint32_t slot = 0, phase = 1;
            bool ok = true;
            while (ok && tiles.next(tile)) {
                const int row0 = tile.row0 + rank * kTileM;
                const float *sa[4];
                const float *sb[kHalves];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int row = row0 + i * 32 + lane;
                    sa[i] = row < tile.row_end ? p.a_scales + (int64_t)row * p.a_scale_stride : nullptr;
                }
#pragma unroll
                for (int h = 0; h < kHalves; h++) {
                    // a block of columns wholly past the end has no scale of its own
                    const int col = tile.col0 + h * 128;
                    sb[h] = p.w_scales + (int64_t)tile.expert * p.w_scale_expert +
                            (col < p.out ? (int64_t)(col / 128) * p.w_scale_out : 0);
                }
                for (int c0 = 0; c0 < blocks; c0 += kSlotBlocks) {
                    const int n = blocks - c0 < kSlotBlocks ? blocks - c0 : kSlotBlocks;
                    float va[kSlotBlocks][4], vb[kSlotBlocks][kHalves];
#pragma unroll
                    for (int c = 0; c < kSlotBlocks; c++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) va[c][i] = c < n && sa[i] ? __ldg(sa[i] + c_begin + c0 + c) : 1.0f;
#pragma unroll
                        for (int h = 0; h < kHalves; h++)
                            vb[c][h] = c < n ? __ldg(sb[h] + (int64_t)(c_begin + c0 + c) * p.w_scale_in) : 1.0f;
                    }
                    uint32_t seen_a = 0, seen_w = 0;
#pragma unroll
                    for (int c = 0; c < kSlotBlocks; c++) {
#pragma unroll
                        for (int i = 0; i < 4; i++) look(seen_a, va[c][i], kLeastA);
#pragma unroll
                        for (int h = 0; h < kHalves; h++) look(seen_w, vb[c][h], kLeastW);
                    }
                    const bool far = __any_sync(~0u, seen_a > kSpanA || seen_w > kSpanW);
                    ok = warp_wait(&ctl.slot_empty[slot], phase, abort, p.status);
                    if (!ok) break;
                    float *const to = slots + slot * (S::kSlotBytes / 4) + lane;
                    if (!far) {
#pragma unroll
                        for (int c = 0; c < kSlotBlocks; c++)
#pragma unroll
                            for (int h = 0; h < kHalves; h++)
#pragma unroll
                                for (int i = 0; i < 4; i++) to[(c * kHalves + h) * 128 + i * 32] = va[c][i] * vb[c][h];
                    } else {
#pragma unroll
                        for (int c = 0; c < kSlotBlocks; c++)
#pragma unroll
                            for (int h = 0; h < kHalves; h++)
#pragma unroll
                                for (int i = 0; i < 4; i++) {
                                    const float2 v = apart(va[c][i], vb[c][h]);
                                    to[(c * kHalves + h) * 128 + i * 32] = v.x;
                                    to[S::kScales + (c * kHalves + h) * 128 + i * 32] = v.y;
                                }
                    }
                    if (lane == 0)
                        ctl.slot[slot] = make_int4(row0, tile.row_end, tile.col0,
                                                   n + (c0 + n == blocks ? kLast : 0) + (far ? kFar : 0));
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ctl.slot_full[slot]);
                    if (++slot == kSlots) slot = 0, phase ^= 1;
                }
            }
            if (ok && warp_wait(&ctl.slot_empty[slot], phase, abort, p.status) && lane == 0) {  // no more
                ctl.slot[slot] = make_int4(0, 0, 0, 0);
                mbar_arrive(&ctl.slot_full[slot]);
            }
        }
    } else {
        // ------------------------------------------------ scaling and stores
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kEpiRegs));
        // TMEM lanes of this warp, the half it drains, its 64-column groups
        // there, and where those are in the tile: in a pair, a half's two
        // groups are 64 columns of either CTA's 128.
        const int lanes0 = (warp & 3) * 32, half = S::kHalves == 2 ? warp >> 2 : 0, group0 = S::kHalves == 2 ? 0 : warp >> 2;
        const auto block_of = [&](int u) { return PAIR == 2 ? u : half; };
        const auto col_of = [&](int u) { return PAIR == 2 ? u * 128 + half * 64 : half * 128 + (group0 + u) * 64; };
        const uint32_t stage = stages + warp * kPieceBytes;
        const uint32_t from = tmem + ((uint32_t)lanes0 << 16) + half * S::kBufs * 128 + group0 * 64;
        const uint32_t empty0 = PAIR == 2 ? in_leader(smem_u32(&ctl.acc[half][0].empty)) : smem_u32(&ctl.acc[half][0].empty);
        uint32_t slot = 0, phase = 0;
        uint32_t g = 0;  // blocks so far
        bool fresh = true;
        float2 acc[S::kGroups][32];
        while (warp_wait(&ctl.slot_full[slot], phase, abort, p.status)) {
            const int4 t = ctl.slot[slot];
            const int n = t.w & (kLast - 1), row0 = t.x + lanes0;
            if (n == 0) break;
            if (fresh) {
#pragma unroll
                for (int u = 0; u < S::kGroups; u++)
#pragma unroll
                    for (int i = 0; i < 32; i++) acc[u][i] = make_float2(0.0f, 0.0f);
            }
            // The slot's blocks; with_twos: their sums are multiplied by powers of two first.  (Two loops: the
            // choice within one took the prompt's product from 236 to 252 us.  All-zero blocks have the least
            // scale and come here too: 93 zero rows among 4096 take 5 % more, a zero row in every tile half as much again.)
            const auto blocks_of_slot = [&](auto with_twos) {
                constexpr bool kTwos = decltype(with_twos)::value;
                const float *scales = slots + slot * (S::kSlotBytes / 4) + lanes0 + lane;
#pragma unroll 1
                for (int c = 0; c < n; c++, g++, scales += BN) {
                    const uint32_t buf = g % S::kBufs;
                    float2 scale[S::kGroups];
                    float two[S::kGroups];
#pragma unroll
                    for (int u = 0; u < S::kGroups; u++) {
                        scale[u].x = scale[u].y = scales[block_of(u) * 128];
                        if (kTwos) two[u] = scales[S::kScales + block_of(u) * 128];
                    }
                    if (!warp_wait(&ctl.acc[half][buf].full, g / S::kBufs & 1, abort, p.status)) return false;
                    fence_after();
                    if (row0 < t.y) {  // else no row of this warp is anyone's
                        uint32_t r[2][16];
                        tmem_ld16(from + buf * 128, r[0]);
#pragma unroll
                        for (int q = 0; q < 4 * S::kGroups; q++) {
                            tmem_wait_ld(r[q & 1]);
                            if (q + 1 < 4 * S::kGroups) tmem_ld16(from + buf * 128 + (q + 1) * 16, r[(q + 1) & 1]);
#pragma unroll
                            for (int k = 0; k < 8; k++) {
                                float2 &a = acc[q / 4][q % 4 * 8 + k];
                                float2 v = make_float2(__uint_as_float(r[q & 1][2 * k]), __uint_as_float(r[q & 1][2 * k + 1]));
                                if (kTwos) v = __fmul2_rn(v, make_float2(two[q / 4], two[q / 4]));
                                a = __ffma2_rn(v, scale[q / 4], a);
                            }
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_cluster<PAIR>(empty0 + buf * (uint32_t)sizeof(ctl.acc[0][0]));
                }
                return true;
            };
            const bool ok = t.w & kFar ? blocks_of_slot(std::true_type()) : blocks_of_slot(std::false_type());
            if (!ok) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl.slot_empty[slot]);
            if (++slot == kSlots) slot = 0, phase ^= 1;
            fresh = t.w & kLast;
            if (SPLIT && fresh) {
                if (threadIdx.x == 0) ctl.joined = make_int4(t.x, t.y - t.x < kTileM ? t.y - t.x : kTileM, t.z, 0);
                if (row0 < t.y) {
#pragma unroll
                    for (int i = 0; i < 32; i++) {
                        const uint32_t at = ring + ((group0 * 64 + 2 * i) * kTileM + lanes0 + lane) * 4;
                        st_shared(at, acc[0][i].x);
                        st_shared(at + kTileM * 4, acc[0][i].y);
                    }
                }
            } else if (fresh && row0 < t.y) {
#pragma unroll
                for (int u = 0; u < S::kGroups; u++) {
                    const int col0 = t.z + col_of(u);
                    if (p.dst_type == SHC_SRC_BF16) store_rows<SHC_SRC_BF16>(p, &map_d, stage, acc[u], row0, t.y, col0);
                    else if (p.dst_type == SHC_SRC_F16) store_rows<SHC_SRC_F16>(p, &map_d, stage, acc[u], row0, t.y, col0);
                    else store_rows<SHC_SRC_F32>(p, &map_d, stage, acc[u], row0, t.y, col0);
                }
            }
        }
        if (lane == 0) store_wait();
    }
    __syncwarp();
    if (SPLIT) {
        sync_all<true>();  // every part's sums are in its ring
        const int4 joined = ctl.joined;
        // Items of one row x four columns; all parts' sums of an item are on their way at once.
        const int wide = kTileM / p.split;  // columns of this CTA
        for (int at = threadIdx.x; at < joined.y * (wide / 4); at += S::kThreads) {
            const int c = at / joined.y, row = at - c * joined.y, col = part * wide + c * 4;
            float v[8][4];
#pragma unroll
            for (int q = 0; q < 8; q++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    v[q][i] = q < p.split ? ld_cluster(ring + ((col + i) * kTileM + row) * 4, q) : 0.0f;
#pragma unroll
            for (int q = 1; q < 8; q++)
#pragma unroll
                for (int i = 0; i < 4; i++) v[0][i] += v[q][i];
            store4(p, joined.x + row, joined.z + col, v[0]);
        }
        __syncwarp();
    }
    fence_before();
    sync_all<PAIR == 2 || SPLIT>();  // nothing reaches into a CTA that has ended
    fence_after();
    if (warp == S::kEpiWarps) {
        if (PAIR == 2) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512));
    }
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

// Rows of D in pieces of 32 rows x 64 bytes.
bool out_map(CUtensorMap *map, void *p, int64_t cols, int64_t rows, int64_t row_stride, int dst_type) {
    const int esz = dst_type == SHC_SRC_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(row_stride * esz)};
    const cuuint32_t box[2] = {(cuuint32_t)(64 / esz), 32}, steps[2] = {1, 1};
    const CUtensorMapDataType t = dst_type == SHC_SRC_F32   ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                  : dst_type == SHC_SRC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                            : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const EncodeTiled f = encode_tiled();
    return f && f(map, t, 2, p, dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                  CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int BN, int PAIR, bool TRANS, bool SPLIT>
cudaError_t launch(const CUtensorMap maps[3], const MmArgs &a, unsigned grid, cudaStream_t st) {
    using S = Shape<BN, PAIR>;
    auto *fn = f8_product_kernel<BN, PAIR, TRANS, SPLIT>;
    int per_sm;
    const cudaError_t e = resident_blocks((const void *)fn, S::kThreads, S::kSmem, &per_sm);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid * PAIR * a.split;
    cfg.blockDim = S::kThreads;
    cfg.dynamicSmemBytes = S::kSmem;
    cfg.stream = st;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {(unsigned)(PAIR * a.split), 1, 1};
    cfg.attrs = &attr;
    cfg.numAttrs = PAIR * a.split > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, fn, maps[0], maps[1], maps[2], a);
}

// Tiles there can be at most: every expert with rows may end in a part tile.
int64_t most_tiles(const MmArgs &a, int tm, int bn) {
    const int64_t some = a.n_experts < a.n_rows ? a.n_experts : a.n_rows;
    return (((int64_t)a.n_rows + tm - 1) / tm + (a.offsets ? some : 0)) * ((a.out + bn - 1) / bn);
}

// Which tiles to use: the least of the times below, in units of 10 ns, fitted
// to 60 products of 1 to 8192 rows, 1024 to 14336 columns and 8 to 112 blocks
// with 16-bit results in rows on 16-byte boundaries (within 20 % of all but
// those that HBM bounds, where the shapes tie).  It knows neither wider results
// nor rows off those boundaries nor how many experts have rows, and is off
// there: 7.5 us for 1037 x 2008 x 1030 to f32 (9.7-11.9 measured), 15.0 for the
// gradient of 3001 rows and 16 experts, 1000 x 2050 to f32 (24-32), 242 for 4096
// rows of 8 uneven experts, 14336 x 4096 (270-330), 27.1 for 96 rows over 64
// experts, 2048 x 1024 (23).
//
//   tile                    start   each wave of tiles        4096 cubed, measured
//   128 x 128               3.9 us  1.0 us + 0.29 x blocks    79 us
//   128 x 256               3.5     2.0    + 0.47             71
//   256 x 256, CTA pair     3.0     3.4    + 0.41             70
//
// A grouped product has row tiles for whole tiles' rows and half a tile more
// for each expert, or one for each expert with rows.  Where 128 x 128 tiles
// leave most SMs idle, a cluster of CTAs shares a tile's contraction: 4.9 us + 0.29
// x a part's blocks, and joining two parts takes 1.7 us + 3.5 x rows / 128 and
// four or eight 1.3 + 2.8 x rows / 128, whatever the number of blocks, so that
// one row through 4096 x 4096 takes 8.8 us in four parts (13.2 in one) and 128
// rows through 2048 x 1024 6.1 in one (8.1 in four).  Clusters of eight do not all run at once beyond 64
// CTAs (16 of them take twice as long as 8).
struct Plan {
    int bn, pair, split;
};
Plan plan_for(const MmArgs &a, int num_sms) {
    const auto waves = [&](int tm, int bn, int at_once) {
        int64_t down = ((int64_t)a.n_rows + tm - 1) / tm;
        if (a.offsets) {
            const int64_t some = a.n_experts < a.n_rows ? a.n_experts : a.n_rows;
            down = down + some / 2 > some ? down + some / 2 : some;
        }
        return (down * ((a.out + bn - 1) / bn) + at_once - 1) / at_once;
    };
    const int64_t c = a.blocks_c;
    Plan best{128, 1, 1};
    int64_t least = 390 + waves(128, 128, num_sms) * (100 + 29 * c);
    const auto offer = [&](int64_t time, Plan plan) {
        if (time < least) least = time, best = plan;
    };
    offer(350 + waves(128, 256, num_sms) * (200 + 47 * c), Plan{256, 1, 1});
    if (num_sms >= 2) offer(300 + waves(256, 256, num_sms / 2) * (340 + 41 * c), Plan{256, 2, 1});
    const int64_t tiles = most_tiles(a, kTileM, 128), each = a.n_rows / a.n_experts, rows = each < kTileM ? each : kTileM;
    for (int z = 2; z <= 8; z *= 2) {
        if (tiles * z > (z == 8 ? 64 : num_sms) || c < 2 * z) break;
        offer(490 + 29 * c / z + (z == 2 ? 170 + 350 * rows / 128 : 130 + 280 * rows / 128), Plan{128, 1, z});
    }
    return best;
}

template <int BN, int PAIR, bool SPLIT = false>
cudaError_t launch_shape(const CUtensorMap maps[3], const MmArgs &a, bool transposed, int num_sms, cudaStream_t st) {
    const int64_t most = most_tiles(a, kTileM * PAIR, BN);
    const unsigned grid = (unsigned)(most < num_sms / PAIR ? most : num_sms / PAIR);
    return transposed ? launch<BN, PAIR, true, SPLIT>(maps, a, grid, st) : launch<BN, PAIR, false, SPLIT>(maps, a, grid, st);
}

}  // namespace

int launch_f8_product(const F8Product &p, int num_sms, cudaStream_t st) {
    const int64_t inner = p.transposed ? p.n : p.k, out = p.transposed ? p.k : p.n;
    MmArgs a{};
    a.a_scales = p.a_scales;
    a.w_scales = p.w_scales;
    a.offsets = p.offsets;
    a.offsets_64 = p.offsets_64;
    a.n_rows = (int)p.n_rows;
    a.n_experts = (int)p.n_experts;
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
    const uint64_t starts = (uintptr_t)p.dst | (uint64_t)(p.dst_row_stride * esz);
    a.align = starts % 16 == 0 ? 16 : starts % 8 == 0 ? 8 : 1;
    a.status = p.status;
    a.a_box = p.n_rows / p.n_experts >= kTileM ? kTileM : 32;  // short experts: no more rows than there are, nearly

    CUtensorMap maps[3];
    if (!code_map(&maps[0], p.a, inner, p.n_rows, 1, p.a_row_stride, 0, a.a_box, 2) ||
        !code_map(&maps[1], p.w, p.k, p.n, p.n_experts, p.w_row_stride, p.w_mat_stride, 128, 3))
        return SHC_EINVAL;
    a.tma_store = a.align == 16 && p.dst_row_stride * esz < ((int64_t)1 << 40) &&
                  out_map(&maps[2], p.dst, out, p.n_rows, p.dst_row_stride, p.dst_type);
    if (!a.tma_store) maps[2] = maps[0];
    const Plan plan = plan_for(a, num_sms);
    a.split = plan.split;
    cudaError_t e;
    if (plan.pair == 2) e = launch_shape<256, 2>(maps, a, p.transposed, num_sms, st);
    else if (plan.bn == 256) e = launch_shape<256, 1>(maps, a, p.transposed, num_sms, st);
    else if (plan.split > 1) e = launch_shape<128, 1, true>(maps, a, p.transposed, num_sms, st);
    else e = launch_shape<128, 1>(maps, a, p.transposed, num_sms, st);
    if (e == cudaSuccess) return SHC_OK;
    cudaGetLastError();  // reported here; the next call's launch check starts clean
    return e == cudaErrorMemoryAllocation ? SHC_ENOMEM : SHC_ECUDA;
}

}  // namespace shc
