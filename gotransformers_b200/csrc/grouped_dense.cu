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
// (64 terms of the sum per stage, 128-byte swizzle).  Terms past the end of
// the sum's axis are read as zeros by TMA, from a three-dimensional view of
// the weights, so that the next group's weights are never multiplied.  The
// sum over rows ends inside a stage: there a warp of each CTA zeroes the rows
// past the group's end of both operands before the MMA (0 * NaN is NaN, so
// one operand would not do).
//
// Persistent kernel, one CTA per SM; warp 0 TMA, warp 1 MMA issue (leader),
// warps 2-5 epilogue (TMEM -> bf16 / float32 -> shared memory -> coalesced
// rows), warp 6 zeroes row tails.  Two accumulators: the epilogue of a tile
// overlaps the next tile's products.  Every wait is bounded as in tc.cu.
#include <atomic>

#include "grouped.h"
#include "sm100.cuh"

namespace gtmoe {
namespace {

__device__ int g_dense_error;

constexpr int kStageK = 64;              // terms of the sum per stage
constexpr int kStages = 6;
constexpr int kHalf = 128;               // rows of A, and most rows of B, per CTA
constexpr int kTileM = 2 * kHalf, kTileN = 2 * kHalf;
constexpr int kOperandBytes = kHalf * kStageK * 2;  // 16 KB
constexpr int kStageBytes = 2 * kOperandBytes;
constexpr int kSmallBox = 32;            // rows of a TMA box of a partial tile of B
constexpr int kChunkBytes = kStageK * 128;  // 64 columns x 64 terms of an M- or N-major operand
constexpr int kEpiWarps = 4;
constexpr int kThreads = 7 * 32;
constexpr int kTmemCols = 512;
constexpr int kBandTiles = 16;           // row tiles per band of the unit order
// epilogue staging: two buffers of 32 rows x 128 bf16 (pitch 272 bytes), or
// per warp 32 rows x 32 float32 (pitch 144 bytes)
constexpr int kRowPitch = 272;
constexpr int kRowBuf = 32 * kRowPitch;
constexpr int kGradPitch = 36;
constexpr int kEpiBytes = kEpiWarps * 32 * kGradPitch * 4;
static_assert(2 * kRowBuf <= kEpiBytes, "epilogue staging");
constexpr int kBarBytes = 256;
constexpr int kSmemBytes = 1024 + kStages * kStageBytes + kEpiBytes + kBarBytes + (2 * (kMaxGroups + 1) + kThreads) * 4;
static_assert(kSmemBytes <= 232448, "shared memory per CTA");

struct DenseArgs {
    const int64_t *counts;
    int groups;
    int64_t rows;
    int inputs, outputs;
    void *out;
    int out_f32, accumulate;
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

__device__ __forceinline__ void tma_pair_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3}], [%4];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_pair_3d(uint32_t dst, const CUtensorMap *map, int x, int y, int z, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, "
        "%3, %4}], [%5];" ::"r"(dst),
        "l"((uint64_t)map), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

__device__ __forceinline__ void epi_bar() { asm volatile("bar.sync 1, %0;" ::"n"(kEpiWarps * 32) : "memory"); }
// The epilogue warps take a tile together or stop together.
__device__ __forceinline__ bool epi_vote(bool ok) {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.and.pred q, 1, %2, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}\n"
        : "=r"(r)
        : "r"((uint32_t)ok), "n"(kEpiWarps * 32)
        : "memory");
    return r != 0;
}

// What the waits of one CTA share: its own and its peer's abort flag.
struct Aborts {
    volatile int *own;
    uint32_t peer;
};
// Bounded wait with cluster-scope acquire; false when it gave up.
__device__ __forceinline__ bool wait_for(uint64_t *bar, uint32_t parity, const Aborts &ab, int code) {
    if (mbar_try_wait_cluster(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    while (true) {
        for (int i = 0; i < 32; i++)
            if (mbar_try_wait_cluster(bar, parity)) return true;
        if (*ab.own) return false;
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

// One tile: group, first row of A in its operand (m0), first row of B in the
// group or first column (n0), columns of the tile (n_valid, and n: the next
// multiple of 32), stages of the sum.
struct Unit {
    int g, m0, n0, n_valid, n, stages;
};

// Unit u of the launch.  A group's units run in bands of kBandTiles row tiles
// (column tiles of the weight gradient): within a band the A tile is the
// outer index, so that units at work together share operands through L2.
// Every role walks its units in increasing order.
template <GroupedOp OP>
struct Units {
    const int *start, *tiles;
    int groups, m_tiles, inputs, outputs;
    int g = 0;
    __device__ __forceinline__ int64_t total() const {
        return OP == kWeightGrad ? (int64_t)tiles[groups] : (int64_t)tiles[groups] * m_tiles;
    }
    __device__ __forceinline__ Unit at(int64_t u) {
        const int64_t per = OP == kWeightGrad ? 1 : m_tiles;
        while (tiles[g + 1] * per <= u) g++;
        const int64_t r = u - tiles[g] * per;
        Unit w;
        w.g = g;
        const int rows = start[g + 1] - start[g];
        int mt, nt;
        if (OP == kWeightGrad) {
            mt = (int)(r % m_tiles);
            nt = (int)(r / m_tiles);
        } else {
            const int n_tiles = tiles[g + 1] - tiles[g];
            const int64_t band = r / ((int64_t)kBandTiles * m_tiles);
            const int first = (int)band * kBandTiles, in_band = min(kBandTiles, n_tiles - first);
            const int q = (int)(r - band * kBandTiles * m_tiles);
            mt = q / in_band;
            nt = first + q % in_band;
        }
        w.m0 = mt * kTileM;
        w.n0 = nt * kTileN;
        w.n_valid = min(kTileN, (OP == kWeightGrad ? inputs : rows) - w.n0);
        w.n = (w.n_valid + 31) & ~31;
        const int sum = OP == kProduct ? inputs : OP == kInputGrad ? outputs : rows;
        w.stages = (sum + kStageK - 1) / kStageK;
        return w;
    }
};

template <GroupedOp OP>
__global__ void __launch_bounds__(kThreads, 1)
    grouped_dense_kernel(const __grid_constant__ CUtensorMap amap, const __grid_constant__ CUtensorMap bmap,
                         const __grid_constant__ CUtensorMap bsmall, const DenseArgs a) {
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
    static_assert((3 * kStages + 4) * 8 + 8 <= kBarBytes, "barrier area");
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
        group_ranges(a.counts, a.groups, a.rows, OP == kWeightGrad ? 0 : kTileN,
                     OP == kWeightGrad ? m_tiles * ((a.inputs + kTileN - 1) / kTileN) : 0, start, tiles, scratch);
    if (!counts_ok && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(&g_dense_error, 0, kErrBadCounts);
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer's barriers are initialised before any remote operation
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    Units<OP> units{start, tiles, a.groups, m_tiles, a.inputs, a.outputs};
    const int64_t total = units.total();

    if (warp == 0) {
        // ---------------- TMA
        if (lane == 0) {
            uint32_t j = 0;  // stages issued by this CTA
            bool ok = true;
            for (int64_t u = cluster; u < total && ok; u += n_clusters) {
                const Unit w = units.at(u);
                const int half_n = w.n >> 1;  // this CTA's rows (columns) of B
                const int am = w.m0 + (int)rank * kHalf;
                const int bn = w.n0 + (int)rank * half_n + (OP == kWeightGrad ? 0 : start[w.g]);
                const bool small = OP != kWeightGrad && w.n < kTileN;
                const int boxes = OP == kWeightGrad ? (half_n + 63) / 64 : small ? (half_n + kSmallBox - 1) / kSmallBox : 1;
                const uint32_t bytes = kOperandBytes + boxes * (OP == kWeightGrad ? kChunkBytes
                                                                : small           ? kSmallBox * 128
                                                                                  : kOperandBytes);
                const int rows_end = start[w.g + 1] - start[w.g];
                for (int s = 0; s < w.stages; s++, j++) {
                    const int sb = (int)(j % kStages);
                    if (!wait_for(&empty[sb], ((j / kStages) & 1) ^ 1, ab, 1)) {
                        ok = false;
                        break;
                    }
                    const bool cut = OP == kWeightGrad && (s + 1) * kStageK > rows_end;
                    uint32_t bar;
                    if (cut) {
                        mbar_arrive_expect_tx(&tail[sb], bytes);
                        bar = smem_u32(&tail[sb]);
                    } else {
                        if (leader) {
                            mbar_arrive_expect_tx(&full[sb], 2 * bytes);
                            mbar_arrive(&full[sb]);
                        }
                        bar = mapa_shared(smem_u32(&full[sb]), 0);
                    }
                    if (cut) bar = mapa_shared(bar, rank);
                    const uint32_t sa = smem_u32(smem + sb * kStageBytes), sbb = sa + kOperandBytes;
                    const int k0 = s * kStageK;
                    if (OP == kProduct) {
                        tma_pair_3d(sa, &amap, k0, am, w.g, bar);
                    } else if (OP == kInputGrad) {
                        tma_pair_3d(sa, &amap, am, k0, w.g, bar);
                        tma_pair_3d(sa + kChunkBytes, &amap, am + 64, k0, w.g, bar);
                    } else {
                        tma_pair_2d(sa, &amap, am, start[w.g] + k0, bar);
                        tma_pair_2d(sa + kChunkBytes, &amap, am + 64, start[w.g] + k0, bar);
                    }
                    if (OP == kWeightGrad) {
                        for (int i = 0; i < boxes; i++)
                            tma_pair_2d(sbb + i * kChunkBytes, &bmap, bn + 64 * i, start[w.g] + k0, bar);
                    } else if (!small) {
                        tma_pair_2d(sbb, &bmap, k0, bn, bar);
                    } else {
                        for (int i = 0; i < boxes; i++)
                            tma_pair_2d(sbb + i * kSmallBox * 128, &bsmall, k0, bn + i * kSmallBox, bar);
                    }
                }
            }
            if (*ab.own) settle();
        }
    } else if (warp == 1) {
        // ---------------- MMA issue (leader)
        if (leader && lane == 0) {
            uint32_t j = 0, tile = 0;
            bool ok = true;
            for (int64_t u = cluster; u < total && ok; u += n_clusters) {
                const Unit w = units.at(u);
                if (w.stages == 0) continue;  // no rows: the epilogue writes zeros
                const uint32_t acc = tile & 1;
                if (!wait_for(&tmem_empty[acc], ((tile >> 1) & 1) ^ 1, ab, 2)) break;
                tc_fence_after();
                const uint32_t d = tmem_base + acc * kTileN, idesc = instr_desc<OP>(w.n);
                for (int s = 0; s < w.stages; s++, j++) {
                    const int sb = (int)(j % kStages);
                    if (!wait_for(&full[sb], (j / kStages) & 1, ab, 3)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    const uint32_t sa = smem_u32(smem + sb * kStageBytes), sbb = sa + kOperandBytes;
                    const uint64_t ad = OP == kProduct ? sw128_desc(sa) : column_major_desc(sa);
                    const uint64_t bd = OP == kWeightGrad ? column_major_desc(sbb) : sw128_desc(sbb);
#pragma unroll
                    for (int k = 0; k < kStageK / 16; k++)
                        // 16 terms: 32 bytes of a K-major row, 16 rows of the others
                        umma2_bf16(d, ad + k * (OP == kProduct ? 2 : 128), bd + k * (OP == kWeightGrad ? 128 : 2), idesc,
                                   (s | k) != 0);
                    umma2_commit_mc(&empty[sb], 0x3);
                }
                if (!ok) break;
                umma2_commit_mc(&tmem_full[acc], 0x3);
                tile++;
            }
            if (*ab.own) settle();
        }
    } else if (warp < 2 + kEpiWarps) {
        // ---------------- epilogue
        const int quad = warp & 3;  // TMEM lanes 32 * quad ..
        const int et = threadIdx.x - 64;
        const uint32_t tmem_empty_leader = mapa_shared(smem_u32(&tmem_empty[0]), 0);
        uint32_t tile = 0, buf = 0;
        for (int64_t u = cluster; u < total; u += n_clusters) {
            const Unit w = units.at(u);
            const uint32_t acc = tile & 1;
            if (w.stages) {
                const bool ready = wait_for(&tmem_full[acc], (tile >> 1) & 1, ab, 4);
                if (!epi_vote(ready)) break;
                tc_fence_after();
            }
            const uint32_t t_row = tmem_base + ((uint32_t)(quad * 32) << 16) + acc * kTileN;
            const int chunks = (w.n_valid + 31) / 32;
            const int m_first = w.m0 + (int)rank * kHalf;
            for (int c = 0; c < chunks; c++) {
                uint32_t v[32];
                if (w.stages) {
                    tmem_ld16(t_row + c * 32, *reinterpret_cast<uint32_t(*)[16]>(v));
                    tmem_ld16(t_row + c * 32 + 16, *reinterpret_cast<uint32_t(*)[16]>(v + 16));
                    tmem_ld_wait();
                    if (c == chunks - 1) {
                        // the accumulator is in registers: the next tile may have it
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_remote(tmem_empty_leader + acc * (uint32_t)sizeof(uint64_t));
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = 0;
                }
                if (OP != kWeightGrad) {
                    // lanes are output features, v[i] row i of the chunk
                    uint8_t *stage = epi + buf * kRowBuf;
                    __nv_bfloat16 *col = reinterpret_cast<__nv_bfloat16 *>(stage) + quad * 32 + lane;
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        col[i * (kRowPitch / 2)] = __float2bfloat16(__uint_as_float(v[i]));
                    epi_bar();
                    const int64_t row0 = (int64_t)start[w.g] + w.n0 + c * 32;
                    __nv_bfloat16 *out = (__nv_bfloat16 *)a.out + row0 * m_size + m_first;
#pragma unroll
                    for (int q = 0; q < 4; q++) {
                        const int r = q * 8 + (et >> 4), seg = et & 15;
                        if (c * 32 + r < w.n_valid && m_first + seg * 8 < m_size)
                            *reinterpret_cast<uint4 *>(out + (int64_t)r * m_size + seg * 8) =
                                *reinterpret_cast<const uint4 *>(stage + r * kRowPitch + seg * 16);
                    }
                    buf ^= 1;  // the next chunk's barrier separates this buffer's reads from its next writes
                } else {
                    // lanes are rows of dW, v[i] column i of the chunk
                    float *stage = reinterpret_cast<float *>(epi) + quad * 32 * kGradPitch;
                    float4 *mine = reinterpret_cast<float4 *>(stage + lane * kGradPitch);
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        mine[i] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                              __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                    __syncwarp();
                    const int col0 = w.n0 + c * 32;
                    const int64_t o0 = ((int64_t)w.g * a.outputs + m_first + quad * 32) * a.inputs + col0;
                    if (a.out_f32) {
                        float *out = (float *)a.out + o0;
                        const int cc = (lane & 7) * 4;
#pragma unroll
                        for (int q = 0; q < 8; q++) {
                            const int r = q * 4 + (lane >> 3);
                            if (m_first + quad * 32 + r < a.outputs && col0 + cc < a.inputs) {
                                float4 *p = reinterpret_cast<float4 *>(out + (int64_t)r * a.inputs + cc);
                                float4 x = *reinterpret_cast<const float4 *>(stage + r * kGradPitch + cc);
                                if (a.accumulate) {
                                    const float4 b = *p;
                                    x.x += b.x, x.y += b.y, x.z += b.z, x.w += b.w;
                                }
                                *p = x;
                            }
                        }
                    } else {
                        __nv_bfloat16 *out = (__nv_bfloat16 *)a.out + o0;
                        const int cc = (lane & 3) * 8;
#pragma unroll
                        for (int q = 0; q < 4; q++) {
                            const int r = q * 8 + (lane >> 2);
                            if (m_first + quad * 32 + r < a.outputs && col0 + cc < a.inputs) {
                                __nv_bfloat16 *p = out + (int64_t)r * a.inputs + cc;
                                float x[8], b[8];
#pragma unroll
                                for (int i = 0; i < 8; i++) x[i] = stage[r * kGradPitch + cc + i];
                                if (a.accumulate) {
                                    VecIO<__nv_bfloat16, float, 8>::unpack(VecIO<__nv_bfloat16, float, 8>::load(p), b);
#pragma unroll
                                    for (int i = 0; i < 8; i++) x[i] += b[i];
                                }
                                VecIO<__nv_bfloat16, float, 8>::store(p, x);
                            }
                        }
                    }
                }
            }
            if (w.stages) tile++;
        }
    } else if (OP == kWeightGrad) {
        // ---------------- rows past a group's end, in the sum's last stage, become zeros
        uint32_t j = 0, phases = 0;  // stages passed; per stage of the ring, the parity of its next tail
        bool ok = true;
        for (int64_t u = cluster; u < total && ok; u += n_clusters) {
            const Unit w = units.at(u);
            const int rows = start[w.g + 1] - start[w.g];
            const int valid = rows % kStageK;
            j += w.stages;
            if (w.stages == 0 || valid == 0) continue;
            const int sb = (int)((j - 1) % kStages);
            ok = wait_for(&tail[sb], (phases >> sb) & 1, ab, 5);
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

// A bf16 view with `dims` (innermost first; each further one dense) and the
// given box, 128-byte swizzle; what lies outside reads as zeros.
int encode_view(CUtensorMap *map, const void *base, int n_dims, const int64_t *size, const int *box) {
    auto enc = tensor_map_encoder();
    if (!enc) return fail(GTMOE_ECUDA, "cuTensorMapEncodeTiled is not available");
    cuuint64_t dims[3], strides[2];
    cuuint32_t boxes[3], ones[3] = {1, 1, 1};
    cuuint64_t bytes = 2;
    for (int i = 0; i < n_dims; i++) {
        dims[i] = (cuuint64_t)size[i];
        boxes[i] = (cuuint32_t)box[i];
        if (i) strides[i - 1] = bytes;
        bytes *= dims[i];
    }
    const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)n_dims, const_cast<void *>(base), dims,
                           strides, boxes, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                           CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(GTMOE_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return 0;
}

template <GroupedOp OP>
int launch(const GroupedProduct &p, int device, cudaStream_t st) {
    auto kern = grouped_dense_kernel<OP>;
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
    CUtensorMap amap, bmap, bsmall;
    const int64_t wdims[3] = {p.inputs, p.outputs, p.groups}, xdims[2] = {p.inputs, p.rows}, ydims[2] = {p.outputs, p.rows};
    const int rows_box[2] = {kStageK, kHalf}, small_box[2] = {kStageK, kSmallBox}, sum_box[2] = {64, kStageK};
    const int w_box[3] = {kStageK, kHalf, 1}, wt_box[3] = {64, kStageK, 1};
    if (OP == kProduct) {
        GT_CHECK(encode_view(&amap, p.b, 3, wdims, w_box));
        GT_CHECK(encode_view(&bmap, p.a, 2, xdims, rows_box));
        GT_CHECK(encode_view(&bsmall, p.a, 2, xdims, small_box));
    } else if (OP == kInputGrad) {
        GT_CHECK(encode_view(&amap, p.b, 3, wdims, wt_box));
        GT_CHECK(encode_view(&bmap, p.a, 2, ydims, rows_box));
        GT_CHECK(encode_view(&bsmall, p.a, 2, ydims, small_box));
    } else {
        GT_CHECK(encode_view(&amap, p.a, 2, ydims, sum_box));
        GT_CHECK(encode_view(&bmap, p.b, 2, xdims, sum_box));
        bsmall = bmap;
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
    // at most this many tiles: the rows of a group end inside a tile
    const int64_t m_tiles = ((OP == kInputGrad ? p.inputs : p.outputs) + kTileM - 1) / kTileM;
    const int64_t n_tiles = OP == kWeightGrad ? p.groups * ((p.inputs + kTileN - 1) / kTileN)
                                              : p.rows / kTileN + (p.rows < p.groups ? p.rows : p.groups);
    const int64_t most = m_tiles * n_tiles;
    cfg.gridDim = dim3(2 * (unsigned)(most < pairs ? most : pairs));
    GT_CUDA(cudaLaunchKernelEx(&cfg, kern, amap, bmap, bsmall, a));
    note_launches(1);
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
    if (p.op == kProduct) return launch<kProduct>(p, device, st);
    if (p.op == kInputGrad) return launch<kInputGrad>(p, device, st);
    return launch<kWeightGrad>(p, device, st);
}

int grouped_dense_take_error(int *code) {
    const int zero = 0;
    GT_CUDA(cudaMemcpyFromSymbol(code, g_dense_error, sizeof(int)));
    if (*code) GT_CUDA(cudaMemcpyToSymbol(g_dense_error, &zero, sizeof(int)));
    return 0;
}

}  // namespace gtmoe
