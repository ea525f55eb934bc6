// grouped_dense.cu -- the grouped products (grouped.h) of bf16 operands on the
// 5th-generation tensor cores.
//
// A CTA pair (cluster of 2, tcgen05.mma.cta_group::2, M = 256, N <= 256)
// computes a 256 x N tile with float32 accumulators in tensor memory:
//
//                  M (256)    N            K (sum)   A                  B
//   kProduct       outputs    group rows   inputs    W_g   (K-major)    X  (K-major)
//   kInputGrad     inputs     group rows   outputs   W_g   (M-major)    dY (K-major)
//   kWeightGrad    outputs    inputs       rows      dY    (M-major)    X  (N-major)
//
// The rows are the MMA's N in the first two: N may be any multiple of 32, so
// that a group's last rows, or a group of a few rows, cost tensor time only
// for the rows that are there, and a group of a few rows streams its weights
// without padding them to a tile.  No operand is transposed in memory: the
// M- and N-major ones are read so by the MMA (descriptor LBO = 64 columns,
// SBO = 8 rows of the sum).
//
// Each CTA stages its 128 rows of A and its half of B in shared memory by TMA
// (64 terms of the sum per stage, 128-byte swizzle), each operand by a warp of
// its own and in one TMA instruction: a thread issues one per about 200 clocks
// whatever its size, so that a stage of four 8 KB boxes from one thread took
// 826 clocks where the MMAs need 512.  An M- or N-major operand is therefore
// viewed as 64-column chunks x rows, two chunks to a box, except where a chunk
// is cut by the operand's last column.  Terms past
// the end of the sum's axis are read as zeros by TMA, from a view of the
// weights with an axis for the groups, so that the next group's weights are
// never multiplied.  The sum over rows ends inside a stage: there a warp of
// each CTA zeroes the rows past the group's end of both operands before the MMA
// (0 * NaN is NaN, so one operand would not do).
//
// The tensor cores cut every addition to an accumulator towards zero, so that a
// sum made in one accumulator comes out short, by more the longer it is.
// Measured: float32 results of normal values 4.0e-7 over 512 terms and 6.2e-7
// over 768 (a float32 sum with rounding errs by 2e-7 to 4e-7, to both sides);
// values of one sign 3e-6 over 2048 terms, 2.4e-5 over 8192, 6.6e-5 over 65536,
// 1.6e-3 over 262144, 7.0e-3 over 1048576 (bf16's half step is 3.9e-3).  Sums
// are therefore made in runs of stages, which the epilogue adds in registers,
// with rounding, while the next run is multiplied.  Float32 results in runs of 512 terms: of
// 768 they took 1.5 % less time and erred by 6.8e-7 instead of 4.5e-7; of 256
// they took 14 % more, as the epilogue needs about five stages to add a run up.
// Results in bf16 in runs of 1024 terms: of 2048 terms they took up to 2 % less
// time (8192 rows in 16 groups, 2048 -> 1024: 47.1 and 48.0 us) and 1.1e-3 of
// the values were rounded to another bf16 number than the exact sum, instead of
// 6.2e-4; of 512 terms 3 % more, and 3.2e-4 (a float32 sum with rounding:
// 2.5e-4).  Products whose sums have one run at most have a kernel without the
// registers for more.
// Every 16 runs join a total in local memory, and what that addition rounds off
// is carried on (fold(), grouped.h): equal rows would otherwise be rounded
// alike every time (1.6e-4 over 16777216 rows).
//
// Persistent kernel, one CTA per SM; warp 0 loads A, warp 1 issues the MMAs
// (leader), warps 2-9 epilogue (TMEM -> bf16 / float32 -> shared memory ->
// coalesced rows), warp 10 loads B, warp 11 zeroes row tails.  Two accumulators: the epilogue of a tile
// overlaps the next tile's products.  Every wait is bounded as in tc.cu.
//
// Measured (B200, in loops of most of a second, at the power cap): 8192^3 1260
// TF/s (cuBLAS 1340); 64 groups of 1536 rows, 2048 x 2048, product and input
// gradient 1193 TF/s (cuBLAS's batched product 1219), float32 weight gradient
// 1056; 384 rows in 64 groups, 2048 -> 1408, 72.3 us = 5.1 TB/s of weights.
#include <atomic>

#include "grouped.h"
#include "sm100.cuh"

namespace gtmoe {
namespace {

__device__ int g_dense_error;

constexpr int kStageK = 64;              // terms of the sum per stage
constexpr int kStages = 5;
constexpr int kHalf = 128;               // rows of A, and most rows of B, per CTA
constexpr int kTileM = 2 * kHalf, kTileN = 2 * kHalf;
constexpr int kOperandBytes = kHalf * kStageK * 2;  // 16 KB
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kRunStages = 8;            // stages per run of a float32 weight gradient's sums (512 rows)
constexpr int kLongRunStages = 16;       // and of sums rounded to bf16 (1024 terms)
constexpr int kFoldRuns = 16;            // runs added up in a register before they join the total
constexpr int kPartStep = 768;           // rows of a part of a group: a multiple of this
constexpr int kChunkBytes = kStageK * 128;  // 64 columns x 64 terms of an M- or N-major operand
constexpr int kEpiWarps = 8;             // two groups of four (one per TMEM lane quadrant), half the columns each
constexpr int kThreads = (4 + kEpiWarps) * 32;
constexpr int kTmemCols = 512;
constexpr int kBandTiles = 8;            // row tiles per band of the unit order
// epilogue staging, per group of warps two buffers of 16 rows x 128 bf16
// (pitch 272 bytes), or per warp 32 rows x 32 float32 (pitch 144 bytes), or per
// warp 32 rows x 128 bytes for a TMA store (128-byte swizzle)
constexpr int kChunkRows = 16;
constexpr int kRowPitch = 272;
constexpr int kRowBuf = kChunkRows * kRowPitch;
constexpr int kGradPitch = 36;
constexpr int kWarpBuf = 5 * 1024;  // swizzled tiles start on 1024 bytes
constexpr int kEpiBytes = kEpiWarps * kWarpBuf;
static_assert(4 * kRowBuf <= kEpiBytes && 32 * kGradPitch * 4 <= kWarpBuf, "epilogue staging");
constexpr int kBarBytes = 256;
constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kEpiBytes + kBarBytes + (2 * (kMaxGroups + 1) + kThreads / 32) * 4;
static_assert(kSmemBytes <= 232448, "shared memory per CTA");

struct DenseArgs {
    const int64_t *counts;
    int groups;
    int64_t rows;
    int inputs, outputs;
    void *out;
    int out_f32, accumulate;
    int sum_runs;   // kWeightGrad: float32 sums over runs of stages (else for long groups only)
    int part_rows;  // kWeightGrad: rows of a group per unit
    float *parts;   // and where the sums of a group's parts go if it has several
};

// D f32, A and B bf16, M = 256, N in bits 17-22; A or B M/N-major in bits 15, 16
template <GroupedOp OP>
__device__ __forceinline__ uint32_t instr_desc(int n) {
    return (1u << 4) | (1u << 7) | (1u << 10) | ((OP == kProduct ? 0u : 1u) << 15) |
           ((OP == kWeightGrad ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(kTileM >> 4) << 24);
}
// M- or N-major operand, 128-byte swizzle: 64 columns x 64 terms per chunk
__device__ __forceinline__ uint64_t column_major_desc(uint32_t saddr) {
    return (uint64_t)((saddr & 0x3FFFFu) >> 4) | (uint64_t)(kChunkBytes >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}

__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_pair(uint32_t dst, const CUtensorMap *map, int x, int y, int z, int w,
                                         uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4, %5}], [%6];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void tma_store(const CUtensorMap *map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%1, %2, %3}], [%4];" ::"l"((uint64_t)map),
                 "r"(x), "r"(y), "r"(z), "r"(src)
                 : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// One lane of a converged warp.  The loading and issuing warps stay converged
// and let one lane issue: with a branch on the lane number around the loop the
// compiler cannot keep addresses and descriptors in uniform registers, and a
// stage's four MMAs took 498 clocks to issue instead of fewer than the 512 that
// they run (577 -> 514 clocks per stage).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}\n"
        : "=r"(r));
    return r != 0;
}

// The four MMAs of a stage: 16 terms each, a_step and b_step apart in the
// operands' descriptors.
template <int A_STEP, int B_STEP>
__device__ __forceinline__ void mma_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p, t;\n\t"
        "setp.ne.b32 p, %10, 0;\n\t"
        "setp.eq.b32 t, 0, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %9, p;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %3, %4, %9, t;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %5, %6, %9, t;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %7, %8, %9, t;\n\t}\n" ::"r"(d),
        "l"(a), "l"(b), "l"(a + A_STEP), "l"(b + B_STEP), "l"(a + 2 * A_STEP), "l"(b + 2 * B_STEP),
        "l"(a + 3 * A_STEP), "l"(b + 3 * B_STEP), "r"(idesc), "r"((uint32_t)accumulate));
}
static_assert(kStageK == 64, "four MMAs per stage");

// Barriers 1 and 2: the epilogue's groups of four warps.
__device__ __forceinline__ void epi_bar(int group) { asm volatile("bar.sync %0, 128;" ::"r"(1 + group) : "memory"); }
// A group's warps take a tile together or stop together.
__device__ __forceinline__ bool epi_vote(int group, bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, %2, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(r)
        : "r"((uint32_t)ok), "r"(1 + group)
        : "memory");
    return r != 0;
}

// What the waits of one CTA share: its own and its peer's abort flag.
struct Aborts {
    volatile int *own;
    uint32_t peer;
};
// Bounded wait with cluster-scope acquire; false when it gave up.  progress: a
// count that others move before the barrier's turn comes; the limit runs from
// its last change.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, const Aborts &ab, int code,
                                         const volatile uint32_t *progress = nullptr) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    uint32_t seen = progress ? *progress : 0;
    uint64_t t0 = global_timer_ns();
    while (true) {
        for (int i = 0; i < 32; i++)
            if (mbar_try_wait_cluster(bar, parity)) return true;
        if (*ab.own) return false;
        if (progress && *progress != seen) {
            seen = *progress;
            t0 = global_timer_ns();
        }
        if (global_timer_ns() - t0 > kWaitLimitNs) {
            atomicCAS(&g_dense_error, 0, code);
            *ab.own = 1;
            asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(ab.peer), "r"(1) : "memory");
            return false;
        }
    }
}
// What was issued before an abort lands before the CTA can leave.
__device__ __forceinline__ void settle() {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 1000000ull) {
    }
}

// One tile: group, its first row of A in its operand (m0), first row of B in
// the group or first column (n0), columns of the tile (n_valid, and n: the next
// multiple of 32), stages of the sum, and the rows row0 .. row0 + rows that it
// reads (the group's, or a part of them).  part < 0: the unit has all of the
// group's rows.
struct Unit {
    int g, m0, n0, n_valid, n, stages, row0, rows, part;
};

// Unit u of the launch.  A group's (a part's) units run in bands of kBandTiles
// column tiles of D: within a band the A tile is the outer index, so that the
// units at work together, about 8 x 9 tiles, share operands through L2.  Every
// role walks its units in increasing order.
template <GroupedOp OP>
struct Units {
    const int *start, *tiles;
    int groups, m_tiles, inputs, outputs, part_rows;
    int g = 0;
    __device__ __forceinline__ int64_t total() const {
        return OP == kWeightGrad ? (int64_t)tiles[groups] : (int64_t)tiles[groups] * m_tiles;
    }
    __device__ __forceinline__ Unit at(int64_t u) {
        const int64_t per = OP == kWeightGrad ? 1 : m_tiles;
        while (tiles[g + 1] * per <= u) g++;
        int r = (int)(u - tiles[g] * per);
        Unit w;
        w.g = g;
        w.row0 = start[g];
        w.rows = start[g + 1] - start[g];
        w.part = -1;
        int n_tiles = tiles[g + 1] - tiles[g];
        if (OP == kWeightGrad) {
            n_tiles = (inputs + kTileN - 1) / kTileN;
            if (w.rows > part_rows) {
                const int area = m_tiles * n_tiles, part = r / area;
                r -= part * area;
                w.part = tiles[g] / area + part;
                w.row0 += part * part_rows;
                w.rows = min(part_rows, w.rows - part * part_rows);
            }
        }
        const int band = r / (kBandTiles * m_tiles);
        const int first = band * kBandTiles, in_band = min(kBandTiles, n_tiles - first);
        const int q = r - band * kBandTiles * m_tiles;
        w.m0 = q / in_band * kTileM;
        w.n0 = (first + q % in_band) * kTileN;
        w.n_valid = min(kTileN, (OP == kWeightGrad ? inputs : w.rows) - w.n0);
        w.n = (w.n_valid + 31) & ~31;
        const int sum = OP == kProduct ? inputs : OP == kInputGrad ? outputs : w.rows;
        w.stages = (sum + kStageK - 1) / kStageK;
        return w;
    }
};

// Stages of a unit's sum between two additions in registers.
template <GroupedOp OP, bool RUNS>
__device__ __forceinline__ int run_stages_of(const DenseArgs &a, const Unit &w) {
    return !RUNS ? w.stages : OP == kWeightGrad && a.sum_runs ? kRunStages : kLongRunStages;
}

// The tensor maps of a launch.  a, b: the whole boxes (two 64-column chunks of
// an M- or N-major operand); a_edge, b_edge: one chunk; b_rows: rows of a
// K-major B in boxes of 32 and 64 rows.
// out: dW, and parts the sums of a group's parts, 32 rows x 128 bytes.
struct Maps {
    CUtensorMap a, b, a_edge, b_edge, b_rows[2], out, parts;
};

// RUNS: sums may have several runs of stages (always so for kWeightGrad).
template <GroupedOp OP, bool RUNS>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_dense_kernel(const __grid_constant__ Maps maps, const DenseArgs a) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint8_t *epi = smem + kStages * kStageBytes;
    uint64_t *bars = (uint64_t *)(epi + kEpiBytes);
    uint64_t *full = bars;                    // [kStages] stage loaded in both CTAs (leader)
    uint64_t *empty = bars + kStages;         // [kStages] stage's MMAs done (both CTAs)
    uint64_t *tail = bars + 2 * kStages;      // [kStages] this CTA's part of a sum's last stage loaded
    uint64_t *tmem_full = bars + 3 * kStages; // [2] accumulator ready (both CTAs)
    uint64_t *tmem_empty = tmem_full + 2;     // [2] both epilogues done (leader)
    uint32_t *tmem_slot = (uint32_t *)(tmem_full + 4);
    volatile uint32_t *loaded = tmem_slot + 2;  // stages that the warp that loads A has issued
    static_assert((3 * kStages + 4) * 8 + 12 <= kBarBytes, "barrier area");
    int *start = (int *)((uint8_t *)bars + kBarBytes);
    int *tiles = start + kMaxGroups + 1;
    int *scratch = tiles + kMaxGroups + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    const int cluster = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;
    Aborts ab;
    ab.own = (volatile int *)(tmem_slot + 1);
    ab.peer = mapa_shared(smem_u32((const void *)ab.own), rank ^ 1u);

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; s++) {
            // the leader's producer (twice), or each CTA's tail warp once
            mbar_init(&full[s], 2);
            mbar_init(&empty[s], 1);
            mbar_init(&tail[s], 1);
        }
        for (int b = 0; b < 2; b++) {
            mbar_init(&tmem_full[b], 1);
            mbar_init(&tmem_empty[b], 2 * kEpiWarps);
        }
        *ab.own = 0;
        *loaded = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                     "r"(kTmemCols));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    }
    const int m_size = OP == kInputGrad ? a.inputs : a.outputs;
    const int m_tiles = (m_size + kTileM - 1) / kTileM;
    const bool counts_ok =
        OP == kWeightGrad ? group_ranges(a.counts, a.groups, a.rows, a.part_rows, 1,
                                         m_tiles * ((a.inputs + kTileN - 1) / kTileN), start, tiles, scratch)
                          : group_ranges(a.counts, a.groups, a.rows, kTileN, 0, 1, start, tiles, scratch);
    if (!counts_ok && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(&g_dense_error, 0, kErrBadCounts);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers are initialised before any remote operation
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    Units<OP> units{start, tiles, a.groups, m_tiles, a.inputs, a.outputs, a.part_rows};
    const int64_t total = units.total();

    if (warp == 0 || warp == 2 + kEpiWarps) {
        // ---------------- TMA: A, and the arrival for both operands, or B
        const bool loads_a = warp == 0;
        const bool issuer = elect_one();
        uint32_t j = 0;  // stages issued by this CTA
        bool ok = true;
        for (int64_t u = cluster; u < total && ok; u += n_clusters) {
            const Unit w = units.at(u);
            const int half_n = w.n >> 1;  // this CTA's rows (columns) of B
            const int am = w.m0 + (int)rank * kHalf;
            const int bn = w.n0 + (int)rank * half_n + (OP == kWeightGrad ? 0 : w.row0);
            // an M- or N-major operand's two chunks in one box unless its last column cuts one
            const int a_cols = OP == kInputGrad ? a.inputs : a.outputs;
            const bool a_whole = OP == kProduct || am + kHalf <= (a_cols & ~63);
            const bool b_whole = OP != kWeightGrad || (w.n == kTileN && bn + kHalf <= (a.inputs & ~63));
            const int b_chunks = OP == kWeightGrad ? (half_n + 63) / 64 : 0;
            // a K-major B by the smallest box that holds its rows
            const CUtensorMap *b_map = OP == kWeightGrad || half_n > 64 ? &maps.b : &maps.b_rows[half_n > 32];
            const uint32_t bytes =
                kOperandBytes + (OP == kWeightGrad ? b_chunks * kChunkBytes
                                 : half_n > 64     ? kOperandBytes
                                                   : (half_n > 32 ? 64 : 32) * 128);
            for (int s = 0; s < w.stages; s++, j++) {
                const int sb = (int)(j % kStages);
                ok = __all_sync(0xffffffffu, wait_for(&empty[sb], ((j / kStages) & 1) ^ 1, ab, 1));
                if (!ok) break;
                const int k0 = s * kStageK;
                // B's bytes may land before the arrival below: the phase waits for it
                const bool cut = OP == kWeightGrad && k0 + kStageK > w.rows;
                if (loads_a && issuer) {
                    if (cut) {
                        mbar_arrive_expect_tx(&tail[sb], bytes);
                    } else if (leader) {
                        mbar_arrive_expect_tx(&full[sb], 2 * bytes);
                        mbar_arrive(&full[sb]);
                    }
                }
                const uint32_t bar = cut ? mapa_shared(smem_u32(&tail[sb]), rank) : mapa_shared(smem_u32(&full[sb]), 0);
                const uint32_t sa = smem_u32(smem + sb * kStageBytes), sbb = sa + kOperandBytes;
                if (!issuer) {
                } else if (!loads_a) {
                    if (OP != kWeightGrad) {
                        tma_pair(sbb, b_map, k0, bn, bar);
                    } else if (b_whole) {
                        tma_pair(sbb, b_map, 0, w.row0 + k0, bn / 64, bar);
                    } else {
                        for (int i = 0; i < b_chunks; i++)
                            tma_pair(sbb + i * kChunkBytes, &maps.b_edge, bn + 64 * i, w.row0 + k0, bar);
                    }
                } else if (OP == kProduct) {
                    tma_pair(sa, &maps.a, k0, am, w.g, bar);
                } else if (a_whole) {
                    if (OP == kInputGrad) tma_pair(sa, &maps.a, 0, k0, am / 64, w.g, bar);
                    else tma_pair(sa, &maps.a, 0, w.row0 + k0, am / 64, bar);
                } else {
                    for (int i = 0; i < 2; i++) {
                        if (OP == kInputGrad) tma_pair(sa + i * kChunkBytes, &maps.a_edge, am + 64 * i, k0, w.g, bar);
                        else tma_pair(sa + i * kChunkBytes, &maps.a_edge, am + 64 * i, w.row0 + k0, bar);
                    }
                }
                if (OP == kWeightGrad && loads_a && issuer) *loaded = j + 1;
                __syncwarp();
            }
        }
        if (*ab.own) settle();
    } else if (warp == 1) {
        // ---------------- MMA issue (leader)
        if (leader) {
            const bool issuer = elect_one();
            uint32_t j = 0, run = 0;  // stages, and accumulators filled
            bool ok = true;
            for (int64_t u = cluster; u < total && ok; u += n_clusters) {
                const Unit w = units.at(u);
                const uint32_t idesc = instr_desc<OP>(w.n);
                const int run_stages = run_stages_of<OP, RUNS>(a, w);
                for (int s0 = 0; s0 < w.stages && ok; s0 += run_stages, run++) {
                    const uint32_t acc = run & 1, d = tmem_base + acc * kTileN;
                    ok = __all_sync(0xffffffffu, wait_for(&tmem_empty[acc], ((run >> 1) & 1) ^ 1, ab, 2));
                    if (!ok) break;
                    tc_fence_after();
                    const int s1 = min(w.stages, s0 + run_stages);
                    for (int s = s0; s < s1; s++, j++) {
                        const int sb = (int)(j % kStages);
                        ok = __all_sync(0xffffffffu, wait_for(&full[sb], (j / kStages) & 1, ab, 3));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t sa = smem_u32(smem + sb * kStageBytes), sbb = sa + kOperandBytes;
                        const uint64_t ad = OP == kProduct ? sw128_desc(sa) : column_major_desc(sa);
                        const uint64_t bd = OP == kWeightGrad ? column_major_desc(sbb) : sw128_desc(sbb);
                        if (issuer) {
                            // 16 terms: 32 bytes of a K-major row, 16 rows of the others
                            mma_stage<OP == kProduct ? 2 : 128, OP == kWeightGrad ? 128 : 2>(d, ad, bd, idesc, s > s0);
                            umma2_commit_mc(&empty[sb], 0x3);
                        }
                        __syncwarp();
                    }
                    if (ok && issuer) umma2_commit_mc(&tmem_full[acc], 0x3);
                    __syncwarp();
                }
            }
            if (*ab.own) settle();
        }
    } else if (warp < 2 + kEpiWarps) {
        // ---------------- epilogue: this warp has 32 lanes and half the columns of D
        const int quad = warp & 3;  // TMEM lanes 32 * quad ..
        const int group = (warp - 2) >> 2, et = (threadIdx.x - 64) & 127;
        const uint32_t tmem_empty_leader = mapa_shared(smem_u32(&tmem_empty[0]), 0);
        const uint32_t t_warp = tmem_base + ((uint32_t)(quad * 32) << 16) + group * kHalf;
        uint32_t run = 0, buf = 0;
        // the accumulator is in registers: the next tile or run may have it
        auto release = [&](uint32_t acc) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive_remote(tmem_empty_leader + acc * (uint32_t)sizeof(uint64_t));
        };
        // this warp's part of a unit's D, its runs added up with rounding; false when a wait gave up
        auto add_runs = [&](const Unit &w, int left, float (&sum)[kHalf]) {
            const int run_stages = run_stages_of<OP, RUNS>(a, w);
            // in local memory, which units of at most kFoldRuns runs do not touch: at is 0, but the compiler does not see
            // that and so keeps the registers for the sums
            float folded[kHalf];
            const int at = (int)(a.rows >> 40);
            int runs = 0;
#pragma unroll
            for (int i = 0; i < kHalf; i++) sum[i] = 0.f;
            for (int s0 = 0; s0 < w.stages; s0 += run_stages, run++, runs++) {
                if (runs && runs % kFoldRuns == 0) {
                    if (runs == kFoldRuns)
#pragma unroll
                        for (int i = 0; i < kHalf; i++) folded[at + i] = 0.f;
#pragma unroll
                    for (int i = 0; i < kHalf; i++) {
                        fold(folded[at + i], sum[i]);
                        if (i % 4 == 3) asm volatile("" ::: "memory");  // few loads at once: the registers are taken
                    }
                }
                const uint32_t acc = run & 1;
                const bool ready = wait_for(&tmem_full[acc], (run >> 1) & 1, ab, 4);
                if (!epi_vote(group, ready)) return false;
                tc_fence_after();
#pragma unroll
                for (int c = 0; c < kHalf / 16; c++)
                    if (c * 16 < left) {
                        uint32_t v[16];
                        tmem_ld16(t_warp + acc * kTileN + c * 16, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 16; i++) sum[c * 16 + i] += __uint_as_float(v[i]);
                    }
                release(acc);
            }
            if (runs > kFoldRuns)
#pragma unroll
                for (int i = 0; i < kHalf; i++) {
                    sum[i] += folded[at + i];
                    if (i % 4 == 3) asm volatile("" ::: "memory");
                }
            return true;
        };
        // 16 rows of bf16 outputs: a lane has one output feature, value(i) that of row i of the chunk
        auto store_rows = [&](const Unit &w, int c, int m_first, int left, auto value) {
            uint8_t *stage = epi + (group * 2 + buf) * kRowBuf;
            __nv_bfloat16 *col = reinterpret_cast<__nv_bfloat16 *>(stage) + quad * 32 + lane;
#pragma unroll
            for (int i = 0; i < kChunkRows; i++) col[i * (kRowPitch / 2)] = __float2bfloat16(value(i));
            epi_bar(group);
            const int first = c * kChunkRows;
            const int64_t row0 = (int64_t)w.row0 + w.n0 + group * kHalf + first;
            __nv_bfloat16 *out = (__nv_bfloat16 *)a.out + row0 * m_size + m_first;
#pragma unroll
            for (int q = 0; q < kChunkRows / 8; q++) {
                const int r = q * 8 + (et >> 4), seg = et & 15;
                if (first + r < left && m_first + seg * 8 < m_size)
                    *reinterpret_cast<uint4 *>(out + (int64_t)r * m_size + seg * 8) =
                        *reinterpret_cast<const uint4 *>(stage + r * kRowPitch + seg * 16);
            }
            buf ^= 1;  // the next chunk's barrier separates this buffer's reads from its next writes
        };
        for (int64_t u = cluster; u < total; u += n_clusters) {
            const Unit w = units.at(u);
            const int m_first = w.m0 + (int)rank * kHalf;
            const int left = w.n_valid - group * kHalf;  // columns for this group
            if constexpr (OP != kWeightGrad && RUNS) {
                float sum[kHalf];
                if (!add_runs(w, left, sum)) break;
#pragma unroll
                for (int c = 0; c < kHalf / kChunkRows; c++)
                    if (c * kChunkRows < left)
                        store_rows(w, c, m_first, left, [&](int i) { return sum[c * kChunkRows + i]; });
            } else if constexpr (OP != kWeightGrad) {
                const uint32_t acc = run & 1;
                const bool ready = wait_for(&tmem_full[acc], (run >> 1) & 1, ab, 4);
                if (!epi_vote(group, ready)) break;
                tc_fence_after();
                run++;
                const int chunks = left <= 0 ? 0 : left >= kHalf ? kHalf / kChunkRows : (left + kChunkRows - 1) / kChunkRows;
                if (chunks == 0) release(acc);
                for (int c = 0; c < chunks; c++) {
                    // lanes are output features, v[i] row i of the chunk
                    uint32_t v[kChunkRows];
                    tmem_ld16(t_warp + acc * kTileN + c * kChunkRows, v);
                    tmem_ld_wait();
                    if (c == chunks - 1) release(acc);
                    store_rows(w, c, m_first, left, [&](int i) { return __uint_as_float(v[i]); });
                }
            } else {
                // lanes are rows of dW
                float sum[kHalf];
                if (!add_runs(w, left, sum)) break;
                const bool f32 = a.out_f32 || w.part >= 0, add = a.accumulate && w.part < 0;
                if (!add) {
                    // TMA writes the rows out, and leaves out what lies past the last row and column: the LSU path
                    // below costs the shared memory that feeds the MMAs twice the traffic
                    const uint32_t buf_addr = smem_u32(epi) + (warp - 2) * kWarpBuf;
                    const int m0 = m_first + quad * 32, n0 = w.n0 + group * kHalf;
                    const int per = f32 ? 32 : 64;  // columns in 128 bytes
#pragma unroll
                    for (int c = 0; c < kHalf / 32; c++) {
                        if (c * per >= left || c * per >= kHalf || m0 >= a.outputs) break;
                        // the last store has read the buffer
                        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
#pragma unroll
                        for (int i = 0; i < 8; i++) {
                            uint32_t x[4];
                            if (f32) {
#pragma unroll
                                for (int q = 0; q < 4; q++) x[q] = __float_as_uint(sum[c * 32 + i * 4 + q]);
                            } else {
                                const int e = (c & 1) * 64 + i * 8;
#pragma unroll
                                for (int q = 0; q < 4; q++) x[q] = pack_bf16(sum[e + 2 * q], sum[e + 2 * q + 1]);
                            }
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(buf_addr + lane * 128 +
                                                                                         ((i ^ (lane & 7)) << 4)),
                                         "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3])
                                         : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (elect_one())
                            tma_store(w.part >= 0 ? &maps.parts : &maps.out, buf_addr, n0 + c * per, m0,
                                      w.part >= 0 ? w.part : w.g);
                    }
                    continue;
                }
                // added to what is there: coalesced reads and writes by way of shared memory
                float *stage = reinterpret_cast<float *>(epi + (warp - 2) * kWarpBuf);
                // a unit before, of a group that was split, may have left a store that still reads the buffer
                asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                __syncwarp();
                const int64_t o0 = ((int64_t)w.g * a.outputs + m_first + quad * 32) * a.inputs + w.n0 + group * kHalf;
                const int rows = a.outputs - m_first - quad * 32;  // of dW for this warp
#pragma unroll
                for (int c = 0; c < kHalf / 32; c++) {
                    if (c * 32 >= left) break;
                    float4 *mine = reinterpret_cast<float4 *>(stage + lane * kGradPitch);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        mine[i] = make_float4(sum[c * 32 + 4 * i], sum[c * 32 + 4 * i + 1], sum[c * 32 + 4 * i + 2],
                                              sum[c * 32 + 4 * i + 3]);
                    __syncwarp();
                    if (f32) {
                        const int cc = (lane & 7) * 4;
                        float *out = (float *)a.out + o0 + c * 32 + cc;
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            const int r = q * 4 + (lane >> 3);
                            if (r < rows && c * 32 + cc < left) {
                                float4 *p = reinterpret_cast<float4 *>(out + (int64_t)r * a.inputs);
                                const float4 x = *reinterpret_cast<const float4 *>(stage + r * kGradPitch + cc), b = *p;
                                *p = make_float4(x.x + b.x, x.y + b.y, x.z + b.z, x.w + b.w);
                            }
                        }
                    } else {
                        using Io = VecIO<__nv_bfloat16, float, 8>;
                        const int cc = (lane & 3) * 8;
                        __nv_bfloat16 *out = (__nv_bfloat16 *)a.out + o0 + c * 32 + cc;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const int r = q * 8 + (lane >> 2);
                            if (r < rows && c * 32 + cc < left) {
                                __nv_bfloat16 *p = out + (int64_t)r * a.inputs;
                                float b[8];
                                Io::unpack(Io::load(p), b);
#pragma unroll
                                for (int i = 0; i < 8; i++) b[i] += stage[r * kGradPitch + cc + i];
                                Io::store(p, b);
                            }
                        }
                    }
                }
            }
        }
        if (OP == kWeightGrad) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    } else if (OP == kWeightGrad) {
        // ---------------- rows past a group's end, in the sum's last stage, become zeros
        uint32_t j = 0, phases = 0;  // stages passed; per stage of the ring, the parity of its next tail
        bool ok = true;
        for (int64_t u = cluster; u < total && ok; u += n_clusters) {
            const Unit w = units.at(u);
            const int valid = w.rows % kStageK;
            j += w.stages;
            if (w.stages == 0 || valid == 0) continue;
            const int sb = (int)((j - 1) % kStages);
            // from here on the ring may go around millions of times before that stage's turn
            ok = wait_for(&tail[sb], (phases >> sb) & 1, ab, 5, loaded);
            phases ^= 1u << sb;
            if (!__all_sync(0xffffffffu, ok)) break;
            uint8_t *tile = smem + sb * kStageBytes;
            const int chunks = 2 + ((w.n >> 1) + 63) / 64;  // of A, then of B
            for (int i = lane; i < (kStageK - valid) * 8; i += 32)
                for (int q = 0; q < chunks; q++)
                    *reinterpret_cast<uint4 *>(tile + q * kChunkBytes + valid * 128 + i * 16) = make_uint4(0, 0, 0, 0);
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            // the peer's tensor core reads this CTA's zeros on the leader's word: cluster-scope release
            if (lane == 0)
                asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(
                                 mapa_shared(smem_u32(&full[sb]), 0))
                             : "memory");
        }
    }

    tc_fence_before();
    __syncthreads();
    cluster_sync();  // no CTA leaves while its peer may still signal it
    tc_fence_after();
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
    }
}

// A bf16 (float32) view of `base` with 128-byte swizzle: axis i has size[i] elements
// stride[i] elements apart (axis 0 one) and box[i] of them per box; what lies
// outside the sizes reads as zeros.
struct View {
    int axes;
    int64_t size[4], stride[4];
    int box[4];
};
int encode_view(CUtensorMap *map, const void *base, const View &v, bool f32 = false) {
    static const auto enc = tensor_map_encoder();  // looked up once, whichever thread comes first
    if (!enc) return fail(GTMOE_ECUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[4], strides[3];
    cuuint32_t boxes[4], ones[4] = {1, 1, 1, 1};
    for (int i = 0; i < v.axes; i++) {
        dims[i] = (cuuint64_t)v.size[i];
        boxes[i] = (cuuint32_t)v.box[i];
        if (i) strides[i - 1] = (cuuint64_t)v.stride[i] * (f32 ? 4 : 2);
    }
    const CUresult r = enc(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                           (cuuint32_t)v.axes, const_cast<void *>(base), dims, strides, boxes, ones,
                           CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GTMOE_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return 0;
}
// rows x columns, `cols` per row, in boxes of box_rows rows x 64 columns
View matrix(int64_t rows, int64_t cols, int box_rows) { return {2, {cols, rows}, {1, cols}, {64, box_rows}}; }
// the same as chunks of 64 columns, two to a box; only whole chunks
View chunks(int64_t rows, int64_t cols) {
    return {3, {64, rows, cols / 64 ? cols / 64 : 1}, {1, cols, 64}, {64, kStageK, 2}};
}

// Rows of a group per unit of the weight gradient.  With tiles for every CTA
// pair a unit has all of a group's rows; with fewer the groups are split, into
// about two units per pair, and the parts' sums added by a second kernel
// (1 group of 65536 rows, 512 x 512: 467 -> 53 us).  Short groups are not:
// their units end before the second kernel would.
int part_rows(int64_t rows, int64_t inputs, int64_t outputs, int groups) {
    const int64_t area = ((outputs + kTileM - 1) / kTileM) * ((inputs + kTileN - 1) / kTileN);
    if (area * groups >= 74 || rows < (int64_t)groups * 2048) return kAnyRows;
    const int64_t want = (rows * area / 148 + kPartStep - 1) / kPartStep * kPartStep;
    return (int)(want < kPartStep ? kPartStep : want);
}

// Adds the parts' sums of every group that was split, in order, four values
// per thread.
__global__ void __launch_bounds__(256) add_parts_kernel(const DenseArgs a) {
    __shared__ int start[kMaxGroups + 1], first[kMaxGroups + 1], scratch[8];
    group_ranges(a.counts, a.groups, a.rows, a.part_rows, 1, 1, start, first, scratch);
    const int64_t area = (int64_t)a.outputs * a.inputs;
    for (int g = 0; g < a.groups; g++) {
        const int parts = first[g + 1] - first[g];
        if (parts < 2) continue;
        for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < area; i += (int64_t)gridDim.x * 1024) {
            const float *p = a.parts + first[g] * area + i;
            float4 s = *reinterpret_cast<const float4 *>(p);
            for (int q = 1; q < parts; q++) {
                const float4 v = *reinterpret_cast<const float4 *>(p + q * area);
                s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
            }
            const int64_t o = g * area + i;
            if (a.out_f32) {
                float4 *out = reinterpret_cast<float4 *>((float *)a.out + o);
                if (a.accumulate) {
                    const float4 b = *out;
                    s.x += b.x, s.y += b.y, s.z += b.z, s.w += b.w;
                }
                *out = s;
            } else {
                __nv_bfloat162 *out = reinterpret_cast<__nv_bfloat162 *>((__nv_bfloat16 *)a.out + o);
                if (a.accumulate) {
                    const float2 b0 = __bfloat1622float2(out[0]), b1 = __bfloat1622float2(out[1]);
                    s.x += b0.x, s.y += b0.y, s.z += b1.x, s.w += b1.y;
                }
                out[0] = __floats2bfloat162_rn(s.x, s.y);
                out[1] = __floats2bfloat162_rn(s.z, s.w);
            }
        }
    }
}

template <GroupedOp OP, bool RUNS>
int launch(const GroupedProduct &p, int device, cudaStream_t st) {
    auto kern = grouped_dense_kernel<OP, RUNS>;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    // CTA pairs that are resident at once on this device
    static std::atomic<int> resident[64];
    int pairs = device < 64 ? resident[device].load() : 0;
    if (!pairs) {
        GT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
        int sms = 0;
        GT_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
        cfg.gridDim = dim3(2 * ((sms + 1) / 2));
        GT_CUDA(cudaOccupancyMaxActiveClusters(&pairs, kern, &cfg));
        if (pairs < 1) return fail(GTMOE_ECUDA, "no CTA pair of the grouped product fits on this device");
        if (device < 64) resident[device].store(pairs);
    }
    Maps m;
    const int64_t in = p.inputs, out = p.outputs, rows = p.rows;
    if (OP == kWeightGrad) {
        GT_CHECK(encode_view(&m.a, p.a, chunks(rows, out)));
        GT_CHECK(encode_view(&m.a_edge, p.a, matrix(rows, out, kStageK)));
        GT_CHECK(encode_view(&m.b, p.b, chunks(rows, in)));
        GT_CHECK(encode_view(&m.b_edge, p.b, matrix(rows, in, kStageK)));
        m.b_rows[0] = m.b_rows[1] = m.b_edge;
        const bool f32 = p.out_dtype == GTMOE_DTYPE_F32;
        GT_CHECK(encode_view(&m.out, p.c, {3, {in, out, p.groups}, {1, in, in * out}, {f32 ? 32 : 64, 32, 1}}, f32));
        m.parts = m.out;
        const int part = part_rows(rows, in, out, p.groups);
        if (part != kAnyRows)
            GT_CHECK(encode_view(&m.parts, p.workspace,
                                 {3, {in, out, rows / part + p.groups}, {1, in, in * out}, {32, 32, 1}}, true));
    } else {
        const int64_t sum = OP == kProduct ? in : out, group = in * out;
        if (OP == kProduct) {
            GT_CHECK(encode_view(&m.a, p.b, {3, {in, out, p.groups}, {1, in, group}, {kStageK, kHalf, 1}}));
            m.a_edge = m.a;
        } else {
            GT_CHECK(encode_view(&m.a, p.b,
                                 {4, {64, out, in / 64 ? in / 64 : 1, p.groups}, {1, in, 64, group}, {64, kStageK, 2, 1}}));
            GT_CHECK(encode_view(&m.a_edge, p.b, {3, {in, out, p.groups}, {1, in, group}, {64, kStageK, 1}}));
        }
        GT_CHECK(encode_view(&m.b, p.a, matrix(rows, sum, kHalf)));
        GT_CHECK(encode_view(&m.b_rows[0], p.a, matrix(rows, sum, 32)));
        GT_CHECK(encode_view(&m.b_rows[1], p.a, matrix(rows, sum, 64)));
        m.b_edge = m.out = m.parts = m.b;
    }
    DenseArgs a;
    a.counts = p.counts;
    a.groups = p.groups;
    a.rows = p.rows;
    a.inputs = (int)p.inputs;
    a.outputs = (int)p.outputs;
    a.out = p.c;
    a.out_f32 = p.out_dtype == GTMOE_DTYPE_F32;
    a.accumulate = p.accumulate;
    a.part_rows = OP == kWeightGrad ? part_rows(rows, in, out, p.groups) : kAnyRows;
    a.parts = (float *)p.workspace;
    a.sum_runs = a.out_f32 || a.part_rows != kAnyRows;
    // at most this many tiles: the rows of a group end inside a tile or part
    const int64_t m_tiles = ((OP == kInputGrad ? in : out) + kTileM - 1) / kTileM;
    const int64_t some = rows < p.groups ? rows : p.groups;
    const int64_t n_tiles = OP == kWeightGrad ? (p.groups + rows / a.part_rows) * ((in + kTileN - 1) / kTileN)
                                              : rows / kTileN + some;
    const int64_t most = m_tiles * n_tiles;
    cfg.gridDim = dim3(2 * (unsigned)(most < pairs ? most : pairs));
    GT_CUDA(cudaLaunchKernelEx(&cfg, kern, m, a));
    note_launches(1);
    if (OP == kWeightGrad && a.part_rows != kAnyRows) {
        const int64_t blocks = (in * out / 4 + 255) / 256;
        add_parts_kernel<<<(unsigned)(blocks < 148 * 8 ? blocks : 148 * 8), 256, 0, st>>>(a);
        GT_CUDA(cudaGetLastError());
        note_launches(1);
    }
    return 0;
}

}  // namespace

bool grouped_dense_usable(const GroupedProduct &p) {
    // TMA: rows and bases on 16 bytes; the epilogue stores 16 bytes.  A sum
    // over no rows at all has nothing to map.  A launch's tiles are counted in 31 bits.
    const int64_t m_tiles = (p.outputs + kTileM - 1) / kTileM, n_tiles = (p.inputs + kTileN - 1) / kTileN;
    return p.dtype == GTMOE_DTYPE_BF16 && p.rows > 0 && p.inputs % 8 == 0 && p.outputs % 8 == 0 && aligned16(p.a) &&
           aligned16(p.b) && aligned16(p.c) && m_tiles * n_tiles < 0x7ffffffe / p.groups;
}

int launch_grouped_dense(const GroupedProduct &p, int device, cudaStream_t st) {
    if (p.op == kWeightGrad) return launch<kWeightGrad, true>(p, device, st);
    const int64_t terms = p.op == kProduct ? p.inputs : p.outputs;
    if (terms > kLongRunStages * kStageK)
        return p.op == kProduct ? launch<kProduct, true>(p, device, st) : launch<kInputGrad, true>(p, device, st);
    return p.op == kProduct ? launch<kProduct, false>(p, device, st) : launch<kInputGrad, false>(p, device, st);
}

int64_t grouped_dense_workspace(int64_t rows, int64_t inputs, int64_t outputs, int groups) {
    const int64_t part = part_rows(rows, inputs, outputs, groups);
    return part == kAnyRows ? 0 : (rows / part + groups) * inputs * outputs * 4;
}

int grouped_dense_take_error(int *code) {
    const int zero = 0;
    GT_CUDA(cudaMemcpyFromSymbol(code, g_dense_error, sizeof(int)));
    if (*code) GT_CUDA(cudaMemcpyToSymbol(g_dense_error, &zero, sizeof(int)));
    return 0;
}

}  // namespace gtmoe
