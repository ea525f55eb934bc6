// layer_norm.cu -- layer norm of rows and its backward pass.
//
//   m = mean(x), v = mean((x - m)^2), r = 1 / sqrt(v + eps), xh = (x - m) r
//   y = xh w + b
//   g = dy w,  dx = r (g - mean(g) - xh mean(g xh)) [+ residual gradient]
//   dw = sum over rows of dy xh,  db = sum over rows of dy
//
// Float32 sums for float32 and bf16 rows, float64 for float64 ones; every
// output is rounded once.  The variance is taken around the mean (two passes
// over the row, which stays in registers), so that rows far from zero keep
// their digits.  All sums have a fixed order: results repeat bit for bit.
#include <math.h>

#include <atomic>
#include <type_traits>

#include "operators.h"
#include "sm100.cuh"

namespace gtmoe {
namespace {

constexpr int kWideThreads = 256;
constexpr int kRingThreads = 256;
// Blocks of the backward, each of which leaves one row of partial weight and
// bias gradients: two per SM of a B200.
constexpr int kBwdBlocks = 2 * 148;
// A ring's mbarriers and abort flag come before its stages in shared memory.
constexpr int kMaxStages = 8;
constexpr int kRingHeader = 512;
// Shared memory for the stages of a backward's block of 256 threads (of 512:
// twice this): two blocks per SM.
constexpr int kBwdStageBytes = 98304;
// The forward: most warps per block, most tiles in a warp's ring, and shared
// memory for a block's rings and parameters.
constexpr int kFwdMostWarps = 16;
constexpr int kFwdStages = 3;
constexpr int kFwdMostBytes = 224 * 1024;
static_assert(2 * kMaxStages * 8 + 4 <= kRingHeader && kFwdMostWarps * (kFwdStages * 8 + 4) <= kRingHeader, "ring header");

__device__ int g_norm_error;  // a bounded wait's code (gtmoe_operators_check)

template <typename ACC>
__device__ __forceinline__ ACC rsqrt_acc(ACC v);
template <>
__device__ __forceinline__ float rsqrt_acc<float>(float v) { return 1.f / sqrtf(v); }
template <>
__device__ __forceinline__ double rsqrt_acc<double>(double v) { return 1.0 / sqrt(v); }

// Sums N values over a team of `team` threads (a multiple of 32 up to the
// block; teams are runs of threads with a named barrier each).  `red` holds
// N values per warp of the block and is not read by an earlier call's
// stragglers: callers alternate between two.
template <int N, typename ACC>
__device__ __forceinline__ void team_sum(ACC (&v)[N], int team, int team_id, ACC (*red)[N]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (team == 32) return;
    const int warp = threadIdx.x >> 5, warps = team >> 5;
    if ((threadIdx.x & 31) == 0)
#pragma unroll
        for (int i = 0; i < N; i++) red[warp][i] = v[i];
    asm volatile("bar.sync %0, %1;" ::"r"(1 + team_id), "r"(team) : "memory");
    // (constant trip counts: the loads then overlap)
    ACC (*mine)[N] = red + team_id * warps;
    auto add_up = [&](auto count) {
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = mine[0][i];
#pragma unroll
        for (int w = 1; w < decltype(count)::value; w++)
#pragma unroll
            for (int i = 0; i < N; i++) v[i] += mine[w][i];
    };
    if (warps == 8) add_up(std::integral_constant<int, 8>());
    else if (warps == 4) add_up(std::integral_constant<int, 4>());
    else if (warps == 2) add_up(std::integral_constant<int, 2>());
    else add_up(std::integral_constant<int, 16>());
}

struct NormArgs {
    const void *x, *weight, *bias;
    void *y, *mean, *rstd;
    int64_t rows;
    int width;
    double eps;
    int team, stages;   // threads per row of the backward; tiles in a ring
    int shared_params;  // bytes of the forward's copy of its parameters
    // backward
    const void *dy, *dres;
    void *dx;
    void *partial;  // blocks x 2 x width
    int want_params;
};

// ---- Rows on 16 bytes: tiles of consecutive rows stream through a ring of
// shared-memory stages, filled by bulk copies a few tiles ahead, so that the
// bytes in flight do not depend on how many registers the sums leave for
// occupancy (the same kernels with rows loaded into registers reached 62 % of
// the copy bandwidth).  A team of threads per row, NV vectors per thread.

// Stage s of a block's ring: a tile's rows of each input one after another.
template <typename T, int INPUTS>
struct Ring {
    uint8_t *data;
    uint64_t *full, *empty;  // [stages]
    int *abort_flag;
    int stages, tile_rows, warps;
    int given;  // inputs that are there: the first ones
    int64_t rows, tiles;
    int64_t row_bytes;
    const void *in[INPUTS];

    __device__ __forceinline__ const T *row(int stage, int input, int r) const {
        return (const T *)(data + ((int64_t)(stage * given + input) * tile_rows + r) * row_bytes);
    }
    __device__ __forceinline__ void init() {
        if (threadIdx.x == 0) {
            for (int s = 0; s < stages; s++) {
                mbar_init(&full[s], 1);
                mbar_init(&empty[s], warps);
            }
            *abort_flag = 0;
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        __syncthreads();
    }
    // Thread 0: copies of tile `t` into its stage.
    __device__ __forceinline__ void fill(int64_t t, int stage) {
        const int64_t r0 = t * tile_rows;
        const int64_t n = rows - r0 < tile_rows ? rows - r0 : tile_rows;
        const uint32_t bytes = (uint32_t)(n * row_bytes);
        mbar_arrive_expect_tx(&full[stage], bytes * given);
#pragma unroll
        for (int i = 0; i < INPUTS; i++)
            if (i < given)
                asm volatile(
                    "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                        smem_u32(row(stage, i, 0))),
                    "l"((const uint8_t *)in[i] + r0 * row_bytes), "r"(bytes), "r"(smem_u32(&full[stage]))
                    : "memory");
    }
    __device__ __forceinline__ bool wait(uint64_t *bar, uint32_t parity, int code) {
        return mbar_wait(bar, parity, (volatile int *)abort_flag, &g_norm_error, code);
    }
};

// Walks the block's tiles: body(stage, tile) by every thread, the stage's data
// ready.  After a wait that ran out the others no longer wait: every warp still
// walks all tiles (on whatever the stages hold), so that the teams' barriers
// stay matched.
// Thread 0 refills a stage one tile after it was read, so that it rarely waits
// for a slower warp.
template <typename R, typename F>
__device__ __forceinline__ void walk_tiles(R &ring, F body) {
    const int64_t first = blockIdx.x, step = gridDim.x;
    if (threadIdx.x == 0)
        for (int s = 0; s < ring.stages && first + s * step < ring.tiles; s++) ring.fill(first + s * step, s);
    int stage = 0;
    uint32_t phase = 0;
    int64_t i = 0;
    for (int64_t t = first; t < ring.tiles; t += step, i++) {
        if (threadIdx.x == 0 && i > 0) {
            const int64_t next = first + (i - 1 + ring.stages) * step;
            if (next < ring.tiles) {
                const int before = stage == 0 ? ring.stages - 1 : stage - 1;
                if (ring.wait(&ring.empty[before], stage == 0 ? phase ^ 1 : phase, 2)) ring.fill(next, before);
            }
        }
        ring.wait(&ring.full[stage], phase, 1);
        __syncwarp();
        body(stage, t);
        __syncwarp();
        if ((threadIdx.x & 31) == 0) mbar_arrive(&ring.empty[stage]);
        if (++stage == ring.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    if (*(volatile int *)ring.abort_flag && threadIdx.x == 0) {
        // copies in flight land before the block can leave
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {
        }
    }
}

template <typename T, int INPUTS>
__device__ __forceinline__ Ring<T, INPUTS> make_ring(const NormArgs &a, uint8_t *smem) {
    Ring<T, INPUTS> r;
    r.stages = a.stages;
    r.tile_rows = (int)blockDim.x / a.team;
    r.warps = (int)blockDim.x >> 5;
    r.rows = a.rows;
    r.tiles = (a.rows + r.tile_rows - 1) / r.tile_rows;
    r.row_bytes = (int64_t)a.width * (int64_t)sizeof(T);
    r.full = (uint64_t *)smem;
    r.empty = r.full + kMaxStages;
    r.abort_flag = (int *)(r.empty + kMaxStages);
    r.data = smem + kRingHeader;
    return r;
}

// A warp per tile of RP rows, with a ring of its own: no warp waits for another
// (a team of four warps per row spent more time in its two sums' barriers than
// a warp on the row), and the bytes in flight are those of the ring.  The RP
// rows share each read of the weights and their sums' latencies overlap.  The
// row is read from shared memory for each of the three passes.  65536 x 4096
// bf16: 201 us = 5.3 TB/s (83 % of the copy bandwidth); 16384 x 2048 with float32
// parameters 32 us; what it waits for is its own instructions' latency (8 to 12
// warps per SM).
template <typename T, typename W, typename ACC, int VEC, int RP>
__global__ void __launch_bounds__(kFwdMostWarps * 32) norm_forward_kernel(const NormArgs a) {
    using X = VecIO<T, ACC, VEC>;
    using P = VecIO<W, ACC, VEC>;
    constexpr int H = VEC / 2;
    extern __shared__ __align__(128) uint8_t smem[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, n = a.width;
    const int64_t row_bytes = (int64_t)n * (int64_t)sizeof(T), tile_bytes = row_bytes * RP;
    uint64_t *full = (uint64_t *)smem + warp * kFwdStages;
    int *abort_flag = (int *)((uint64_t *)smem + kFwdMostWarps * kFwdStages) + warp;
    uint8_t *data = smem + kRingHeader + a.shared_params + warp * a.stages * tile_bytes;
    const int64_t tiles = (a.rows + RP - 1) / RP, step = (int64_t)gridDim.x * warps;
    const int64_t first = (int64_t)blockIdx.x * warps + warp;
    auto fill = [&](int64_t t, int stage) {
        const int64_t r0 = t * RP;
        const uint32_t bytes = (uint32_t)((a.rows - r0 < RP ? a.rows - r0 : RP) * row_bytes);
        mbar_arrive_expect_tx(&full[stage], bytes);
        asm volatile(
            "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                smem_u32(data + stage * tile_bytes)),
            "l"((const uint8_t *)a.x + r0 * row_bytes), "r"(bytes), "r"(smem_u32(&full[stage]))
            : "memory");
    };
    if (lane == 0) {
        for (int s = 0; s < a.stages; s++) mbar_init(&full[s], 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int s = 0; s < a.stages; s++)
            if (first + s * step < tiles) fill(first + s * step, s);
    }
    __syncwarp();
    const W *w = (const W *)a.weight, *b = (const W *)a.bias;
    if (a.shared_params) {
        // the rings leave L1 too small to keep the parameters: one copy for the block's warps
        W *sw = (W *)(smem + kRingHeader), *sb = w ? sw + n : sw;
        for (int c = threadIdx.x * VEC; c < n; c += blockDim.x * VEC) {
            if (w) *reinterpret_cast<typename P::Raw *>(sw + c) = P::load_ro(w + c);
            if (b) *reinterpret_cast<typename P::Raw *>(sb + c) = P::load_ro(b + c);
        }
        __syncthreads();
        if (w) w = sw;
        if (b) b = sb;
    }
    int stage = 0;
    uint32_t phase = 0;
    for (int64_t t = first; t < tiles; t += step) {
        if (!__all_sync(0xffffffffu, mbar_wait(&full[stage], phase, (volatile int *)abort_flag, &g_norm_error, 1))) break;
        const int64_t row = t * RP;
        // past the last row the stage holds an earlier tile, or nothing yet: worked on, not written
        const int there = (int)min((int64_t)RP, a.rows - row);
        const T *x = (const T *)(data + stage * tile_bytes);
        Pair<ACC> v[H], s2[RP];
        ACC s[RP], mean[RP], rstd[RP];
        auto row_sums = [&]() {
#pragma unroll
            for (int r = 0; r < RP; r++) s[r] = s2[r].x + s2[r].y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int r = 0; r < RP; r++) s[r] += __shfl_xor_sync(0xffffffffu, s[r], o);
        };
#pragma unroll
        for (int r = 0; r < RP; r++) s2[r] = both(ACC(0));
#pragma unroll (16 / RP)
        for (int c = lane * VEC; c < n; c += 32 * VEC)
#pragma unroll
            for (int r = 0; r < RP; r++) {
                X::unpack(X::load(x + r * n + c), &v[0].x);
#pragma unroll
                for (int q = 0; q < H; q++) s2[r] = add2(s2[r], v[q]);
            }
        row_sums();
#pragma unroll
        for (int r = 0; r < RP; r++) {
            mean[r] = s[r] / (ACC)n;  // exact for a constant row whose sum is
            s2[r] = both(ACC(0));
        }
#pragma unroll (16 / RP)
        for (int c = lane * VEC; c < n; c += 32 * VEC)
#pragma unroll
            for (int r = 0; r < RP; r++) {
                X::unpack(X::load(x + r * n + c), &v[0].x);
#pragma unroll
                for (int q = 0; q < H; q++) {
                    const Pair<ACC> d = add2(v[q], both(-mean[r]));
                    s2[r] = fma2(d, d, s2[r]);
                }
            }
        row_sums();
#pragma unroll
        for (int r = 0; r < RP; r++) rstd[r] = rsqrt_acc<ACC>(s[r] / (ACC)n + (ACC)a.eps);
        T *y = (T *)a.y + row * n;
#pragma unroll 4
        for (int c = lane * VEC; c < n; c += 32 * VEC) {
            Pair<ACC> pw[H], pb[H];
            if (w) P::unpack(P::load(w + c), &pw[0].x);
            if (b) P::unpack(P::load(b + c), &pb[0].x);
#pragma unroll
            for (int r = 0; r < RP; r++) {
                X::unpack(X::load(x + r * n + c), &v[0].x);
#pragma unroll
                for (int q = 0; q < H; q++) {
                    v[q] = mul2(add2(v[q], both(-mean[r])), both(rstd[r]));
                    if (w && b) v[q] = fma2(v[q], pw[q], pb[q]);
                    else if (w) v[q] = mul2(v[q], pw[q]);
                    else if (b) v[q] = add2(v[q], pb[q]);
                }
                if (r < there) X::store(y + (int64_t)r * n + c, &v[0].x);
            }
        }
        if (lane < there) {
            ACC m = mean[0], rs = rstd[0];
#pragma unroll
            for (int r = 1; r < RP; r++)
                if (lane == r) m = mean[r], rs = rstd[r];
            if (a.mean) ((ACC *)a.mean)[row + lane] = m;
            if (a.rstd) ((ACC *)a.rstd)[row + lane] = rs;
        }
        __syncwarp();  // the stage has been read
        if (lane == 0 && t + a.stages * step < tiles) fill(t + a.stages * step, stage);
        if (++stage == a.stages) {
            stage = 0;
            phase ^= 1;
        }
    }
    if (*(volatile int *)abort_flag && lane == 0) {
        // copies in flight land before the warp leaves
        const uint64_t t0 = global_timer_ns();
        while (global_timer_ns() - t0 < 1000000ull) {
        }
    }
}

// Every thread has the same columns of each of its rows, so that the weight
// and bias gradients add up in registers; each block leaves one partial row of
// both.  65536 x 4096 bf16 with residual gradients: 345 us = 6.2 TB/s (96 %),
// and 9 us for the parameters' sums; 16384 x 2048: 47 and 8 us.
template <typename T, typename W, typename ACC, int VEC, int NV, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 256 ? 2 : 1) norm_backward_kernel(const NormArgs a) {
    using X = VecIO<T, ACC, VEC>;
    using P = VecIO<W, ACC, VEC>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ ACC red[2][THREADS / 32][2];
    const int team = a.team, team_id = threadIdx.x / team, tl = threadIdx.x - team_id * team, n = a.width;
    const ACC inv_n = ACC(1) / (ACC)n;
    Ring<T, 3> ring = make_ring<T, 3>(a, smem);
    ring.in[0] = a.dy;
    ring.in[1] = a.x;
    ring.in[2] = a.dres;
    ring.given = a.dres ? 3 : 2;
    ring.init();
    const W *w = (const W *)a.weight;
    constexpr int H = VEC / 2;
    Pair<ACC> aw2[NV * H], ab2[NV * H], pw[NV * H];
#pragma unroll
    for (int i = 0; i < NV * H; i++) aw2[i] = ab2[i] = both(ACC(0)), pw[i] = both(ACC(1));
#pragma unroll
    for (int i = 0; i < NV; i++) {
        const int c = (i * team + tl) * VEC;
        if (w && c < n) P::unpack(P::load(w + c), &pw[i * H].x);
    }
    int it = 0;
    // the next row's statistics are on their way while a row is worked on
    const int64_t first = (int64_t)blockIdx.x * ring.tile_rows + team_id, row_step = (int64_t)gridDim.x * ring.tile_rows;
    ACC next_mean = ACC(0), next_rstd = ACC(0);
    if (first < a.rows) next_mean = ((const ACC *)a.mean)[first], next_rstd = ((const ACC *)a.rstd)[first];
    walk_tiles(ring, [&](int stage, int64_t t) {
        const int64_t row = t * ring.tile_rows + team_id;
        if (row >= a.rows) return;
        const T *dy = ring.row(stage, 0, team_id), *x = ring.row(stage, 1, team_id), *dres = ring.row(stage, 2, team_id);
        const ACC rs = next_rstd, mean = next_mean;
        if (row + row_step < a.rows) {
            next_mean = ((const ACC *)a.mean)[row + row_step];
            next_rstd = ((const ACC *)a.rstd)[row + row_step];
        }
        Pair<ACC> s1 = both(ACC(0)), s2 = both(ACC(0)), g[NV * H], xh[NV * H];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                X::unpack(X::load(x + c), &xh[i * H].x);
                X::unpack(X::load(dy + c), &g[i * H].x);
#pragma unroll
                for (int e = i * H; e < (i + 1) * H; e++) {
                    xh[e] = mul2(add2(xh[e], both(-mean)), both(rs));
                    aw2[e] = fma2(g[e], xh[e], aw2[e]);
                    ab2[e] = add2(ab2[e], g[e]);
                    g[e] = mul2(g[e], pw[e]);
                    s1 = add2(s1, g[e]);
                    s2 = fma2(g[e], xh[e], s2);
                }
            }
        }
        ACC s[2] = {s1.x + s1.y, s2.x + s2.y};
        team_sum<2, ACC>(s, team, team_id, red[it]);
        it ^= 1;
        // dx = rs g - rs m1 - xh rs m2 (+ dres)
        const ACC c1 = -rs * (s[0] * inv_n), c2 = -rs * (s[1] * inv_n);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                Pair<ACC> v[H];
                if (a.dres) X::unpack(X::load(dres + c), &v[0].x);
#pragma unroll
                for (int q = 0; q < H; q++) {
                    const int e = i * H + q;
                    const Pair<ACC> d = fma2(both(rs), g[e], fma2(xh[e], both(c2), both(c1)));
                    v[q] = a.dres ? add2(v[q], d) : d;
                }
                X::store((T *)a.dx + row * n + c, &v[0].x);
            }
        }
    });
    const ACC *aw = &aw2[0].x, *ab = &ab2[0].x;
    if (!a.want_params) return;
    ACC *out = (ACC *)a.partial + (int64_t)blockIdx.x * 2 * n;
    // the teams' sums in team order, in the ring's memory (its copies have all been waited for)
    ACC *total = (ACC *)(smem + kRingHeader);
    const int teams = (int)blockDim.x / team;
    for (int t = 0; t < teams; t++) {
        __syncthreads();
        if (team_id == t) {
#pragma unroll
            for (int i = 0; i < NV; i++)
#pragma unroll
                for (int q = 0; q < VEC; q++) {
                    const int c = (i * team + tl) * VEC + q, e = i * VEC + q;
                    if (c < n) {
                        const ACC sw = t ? total[c] + aw[e] : aw[e], sb = t ? total[n + c] + ab[e] : ab[e];
                        if (t == teams - 1) {
                            out[c] = sw;
                            out[n + c] = sb;
                        } else {
                            total[c] = sw;
                            total[n + c] = sb;
                        }
                    }
                }
        }
    }
}

// ---- Any other row: a block per row reads it three times (the second and
// third time mostly from L1 and L2).
template <typename T, typename W, typename ACC, int VEC>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(const NormArgs a) {
    using X = VecIO<T, ACC, VEC>;
    using P = VecIO<W, ACC, VEC>;
    __shared__ ACC red[2][kWideThreads / 32][1];
    const int n = a.width;
    const W *w = (const W *)a.weight, *b = (const W *)a.bias;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *xr = (const T *)a.x + row * n;
        ACC s[1] = {ACC(0)}, v[VEC];
#pragma unroll 4
        for (int64_t c = threadIdx.x * VEC; c < n; c += kWideThreads * VEC) {
            X::unpack(X::load(xr + c), v);
#pragma unroll
            for (int q = 0; q < VEC; q++) s[0] += v[q];
        }
        team_sum<1, ACC>(s, kWideThreads, 0, red[0]);
        const ACC mean = s[0] / (ACC)n;
        s[0] = ACC(0);
#pragma unroll 4
        for (int64_t c = threadIdx.x * VEC; c < n; c += kWideThreads * VEC) {
            X::unpack(X::load(xr + c), v);
#pragma unroll
            for (int q = 0; q < VEC; q++) s[0] += (v[q] - mean) * (v[q] - mean);
        }
        team_sum<1, ACC>(s, kWideThreads, 0, red[1]);
        const ACC rstd = rsqrt_acc<ACC>(s[0] / (ACC)n + (ACC)a.eps);
        for (int64_t c = threadIdx.x * VEC; c < n; c += kWideThreads * VEC) {
            ACC pw[VEC], pb[VEC];
            X::unpack(X::load(xr + c), v);
            if (w) P::unpack(P::load(w + c), pw);
            if (b) P::unpack(P::load(b + c), pb);
#pragma unroll
            for (int q = 0; q < VEC; q++) {
                v[q] = (v[q] - mean) * rstd;
                if (w) v[q] *= pw[q];
                if (b) v[q] += pb[q];
            }
            X::store((T *)a.y + row * n + c, v);
        }
        if (threadIdx.x == 0) {
            if (a.mean) ((ACC *)a.mean)[row] = mean;
            if (a.rstd) ((ACC *)a.rstd)[row] = rstd;
        }
    }
}

// The backward of any other row: read twice; a thread adds its columns'
// gradients into the block's partial row in memory, or for narrow rows
// (width <= NV * kWideThreads, VEC 1) in registers.
template <typename T, typename W, typename ACC, int VEC, int NV>
__global__ void __launch_bounds__(kWideThreads) norm_backward_wide_kernel(const NormArgs a) {
    using X = VecIO<T, ACC, VEC>;
    using P = VecIO<W, ACC, VEC>;
    __shared__ ACC red[2][kWideThreads / 32][2];
    const int n = a.width;
    const ACC inv_n = ACC(1) / (ACC)n;
    const W *w = (const W *)a.weight;
    ACC *out = (ACC *)a.partial + (int64_t)blockIdx.x * 2 * n;
    ACC aw[NV ? NV : 1] = {}, ab[NV ? NV : 1] = {};
    int it = 0;
    bool first = true;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, it ^= 1) {
        const T *x = (const T *)a.x + row * n, *dy = (const T *)a.dy + row * n;
        T *dx = (T *)a.dx + row * n;
        const ACC mean = ((const ACC *)a.mean)[row], rs = ((const ACC *)a.rstd)[row];
        ACC s[2] = {ACC(0), ACC(0)};
        auto sums = [&](int64_t c, ACC *g, ACC *xh) {
            ACC pw[VEC];
            X::unpack(X::load(x + c), xh);
            X::unpack(X::load(dy + c), g);
            if (w) P::unpack(P::load(w + c), pw);
#pragma unroll
            for (int q = 0; q < VEC; q++) {
                xh[q] = (xh[q] - mean) * rs;
                if (w) g[q] *= pw[q];
                s[0] += g[q];
                s[1] += g[q] * xh[q];
            }
        };
        if constexpr (NV > 0) {
            // VEC 1: the row's values stay in registers
            ACC g[NV], xh[NV], d[NV];
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int64_t c = threadIdx.x + i * kWideThreads;
                if (c < n) {
                    d[i] = (ACC)dy[c];
                    sums(c, g + i, xh + i);
                    aw[i] += d[i] * xh[i];
                    ab[i] += d[i];
                }
            }
            team_sum<2, ACC>(s, kWideThreads, 0, red[it]);
            const ACC c1 = -rs * (s[0] * inv_n), c2 = -rs * (s[1] * inv_n);
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int64_t c = threadIdx.x + i * kWideThreads;
                if (c < n) {
                    ACC v = rs * g[i] + (xh[i] * c2 + c1);
                    if (a.dres) v = (ACC)((const T *)a.dres)[row * n + c] + v;
                    dx[c] = (T)v;
                }
            }
        } else {
            ACC g[VEC], xh[VEC], v[VEC], o[VEC];
#pragma unroll 2
            for (int64_t c = threadIdx.x * VEC; c < n; c += kWideThreads * VEC) sums(c, g, xh);
            team_sum<2, ACC>(s, kWideThreads, 0, red[it]);
            const ACC c1 = -rs * (s[0] * inv_n), c2 = -rs * (s[1] * inv_n);
            for (int64_t c = threadIdx.x * VEC; c < n; c += kWideThreads * VEC) {
                ACC d[VEC], pw[VEC];
                X::unpack(X::load(x + c), xh);
                X::unpack(X::load(dy + c), d);
                if (w) P::unpack(P::load(w + c), pw);
                if (a.dres) X::unpack(X::load((const T *)a.dres + row * n + c), o);
#pragma unroll
                for (int q = 0; q < VEC; q++) {
                    xh[q] = (xh[q] - mean) * rs;
                    v[q] = rs * (w ? d[q] * pw[q] : d[q]) + (xh[q] * c2 + c1);
                    if (a.dres) v[q] = o[q] + v[q];
                }
                X::store(dx + c, v);
                if (a.want_params)
#pragma unroll
                    for (int q = 0; q < VEC; q++) {
                        out[c + q] = (first ? ACC(0) : out[c + q]) + d[q] * xh[q];
                        out[n + c + q] = (first ? ACC(0) : out[n + c + q]) + d[q];
                    }
            }
        }
        first = false;
    }
    if (NV > 0 && a.want_params)
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int64_t c = threadIdx.x + i * kWideThreads;
            if (c < n) {
                out[c] = aw[i];
                out[n + c] = ab[i];
            }
        }
}

// The blocks' partial rows to the weight (blockIdx.y 0) and bias gradients: 32
// columns per block, 32 runs of partial rows side by side, added in a fixed
// order.  The backward gives no earlier sign than its end, so this launch only
// hides its own set-up behind the last blocks (a sign sooner changed nothing).
template <typename W, typename ACC>
__global__ void __launch_bounds__(1024) norm_params_kernel(const ACC *__restrict__ partial, int blocks, int n,
                                                           void *dweight, void *dbias, int accumulate) {
    __shared__ ACC sum[32][33];
    const int c = blockIdx.x * 32 + threadIdx.x, run = threadIdx.y;
    W *dst = (W *)(blockIdx.y == 0 ? dweight : dbias);
    const ACC *src = partial + blockIdx.y * (int64_t)n + c;
    cudaGridDependencySynchronize();
    ACC s = ACC(0);
    if (c < n && dst) {
#pragma unroll 5
        for (int p = run; p < blocks; p += 32) s += src[(int64_t)p * 2 * n];
    }
    sum[run][threadIdx.x] = s;
    __syncthreads();
    // warp `run` now adds column run of the block
    s = sum[threadIdx.x][run];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int column = blockIdx.x * 32 + run;
    if (threadIdx.x == 0 && column < n && dst) {
        if (accumulate) s += (ACC)dst[column];
        dst[column] = (W)s;
    }
}

// How a ring kernel runs: threads per row (the fewest, a power of two from 32
// on, that hold the row in nv vectors each), rows per tile, stages.
struct RingPlan {
    int team, threads, stages, nv, smem;
};
// bytes: of a row, all inputs together; budget: shared memory for the stages
// of a block of 256 threads
bool ring_plan(int64_t vectors, int nv, int64_t bytes, int most_threads, int64_t budget, RingPlan *p) {
    p->nv = nv;
    p->team = 32;
    while ((int64_t)p->team * nv < vectors) p->team *= 2;
    if (p->team > most_threads) return false;
    // two teams of 256 in one block leave half as many partial rows as two blocks (65536 x 4096: 371 -> 354 us);
    // smaller teams lose that again to adding up more of them
    p->threads = p->team >= kRingThreads ? 2 * kRingThreads : kRingThreads;
    const int64_t stage = bytes * (p->threads / p->team);
    const int64_t fit = budget * (p->threads / kRingThreads) / stage;
    p->stages = (int)(fit < kMaxStages ? fit : kMaxStages);
    p->smem = (int)(kRingHeader + p->stages * stage);
    return p->stages >= 2;
}

// Blocks of `kern` that fit on the device at once; `known` keeps the last
// answer (device, shared memory, blocks).
int resident_blocks(const void *kern, int threads, int smem, int most_smem, int device, std::atomic<uint64_t> &known,
                    int64_t *blocks) {
    const uint64_t key = ((uint64_t)(device + 1) << 52) | ((uint64_t)smem << 32);
    const uint64_t v = known.load(std::memory_order_relaxed);
    if ((v & ~(uint64_t)0xffffffffu) == key) {
        *blocks = (int64_t)(v & 0xffffffffu);
        return 0;
    }
    int per = 0, sms = 0;
    GT_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem));
    GT_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per, kern, threads, smem));
    GT_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    if (per < 1) return fail(GTMOE_ECUDA, "layer norm: no block fits on this device");
    *blocks = (int64_t)per * sms;
    known.store(key | (uint64_t)*blocks, std::memory_order_relaxed);
    return 0;
}

template <typename T, typename W, typename ACC, int VEC>
int forward_vec(NormArgs a, int device, cudaStream_t st) {
    if constexpr (VEC > 1) {
        const int64_t bytes = (int64_t)a.width * sizeof(T);
        // rows per warp: tiles of up to 8 KB, as long as every SM's warps get one
        int rp = bytes <= 2048 ? 4 : bytes <= 4096 ? 2 : 1;
        while (rp > 1 && a.rows < (int64_t)rp * 148 * 12) rp /= 2;
        // rows above 4 KB: one block per SM of as many warps as have room for rings of three tiles (two, where that
        // leaves fewer than eight warps), the parameters beside them (65536 x 4096 bf16: 217 -> 201 us); shorter or few
        // rows: blocks of four warps with rings of two, and L1 keeps the parameters
        const int64_t tile = bytes * rp, tiles = (a.rows + rp - 1) / rp;
        const int64_t params = ((a.weight ? 1 : 0) + (a.bias ? 1 : 0)) * (int64_t)a.width * sizeof(W);
        int64_t stages = kFwdMostBytes - params >= 8 * 3 * tile ? 3 : 2, warps = (kFwdMostBytes - params) / (stages * tile);
        if (warps > kFwdMostWarps) warps = kFwdMostWarps;
        const bool share = bytes > 4096 && warps >= 2 && tiles >= 148 * 2 * warps;
        if (!share) {
            stages = 2;
            warps = kFwdMostBytes / (stages * tile);
            if (warps > 4) warps = 4;
        }
        if (warps >= 2) {
            static std::atomic<uint64_t> known[3];
            auto kern = rp == 4   ? norm_forward_kernel<T, W, ACC, VEC, 4>
                        : rp == 2 ? norm_forward_kernel<T, W, ACC, VEC, 2>
                                  : norm_forward_kernel<T, W, ACC, VEC, 1>;
            a.stages = (int)stages;
            a.shared_params = share ? (int)params : 0;
            const int smem = (int)(kRingHeader + a.shared_params + stages * tile * warps);
            const int64_t want = (tiles + warps - 1) / warps;
            int64_t blocks = 0;
            GT_CHECK(resident_blocks((const void *)kern, (int)warps * 32, smem, kRingHeader + kFwdMostBytes, device,
                                     known[rp / 2], &blocks));
            kern<<<(unsigned)(want < blocks ? want : blocks), (int)warps * 32, smem, st>>>(a);
            GT_CUDA(cudaGetLastError());
            note_launches(1);
            return 0;
        }
    }
    norm_forward_wide_kernel<T, W, ACC, VEC><<<(unsigned)(a.rows < 148 * 64 ? a.rows : 148 * 64), kWideThreads, 0, st>>>(a);
    GT_CUDA(cudaGetLastError());
    note_launches(1);
    return 0;
}

template <typename T, typename W, typename ACC, int VEC>
int backward_vec(NormArgs a, void *dweight, void *dbias, int accumulate, int device, cudaStream_t st) {
    int64_t blocks = 0;
    if (a.rows > 0) {
        RingPlan p;
        bool ring = false;
        if constexpr (VEC > 1) {
            const int64_t vectors = a.width / VEC, bytes = (int64_t)a.width * sizeof(T) * (a.dres ? 3 : 2);
            static std::atomic<uint64_t> known[3];
            ring = ring_plan(vectors, vectors <= 32 ? 1 : 2, bytes, 512, kBwdStageBytes, &p);
            if (ring) {
                auto kern = p.nv == 1          ? norm_backward_kernel<T, W, ACC, VEC, 1, 256>
                            : p.threads == 256 ? norm_backward_kernel<T, W, ACC, VEC, 2, 256>
                                               : norm_backward_kernel<T, W, ACC, VEC, 2, 512>;
                a.team = p.team;
                a.stages = p.stages;
                const int64_t rows = p.threads / p.team, tiles = (a.rows + rows - 1) / rows;
                GT_CHECK(resident_blocks((const void *)kern, p.threads, p.smem, kRingHeader + 2 * kBwdStageBytes, device,
                                         known[p.threads > 256 ? 2 : p.nv - 1], &blocks));
                if (blocks > kBwdBlocks) blocks = kBwdBlocks;
                if (blocks > tiles) blocks = tiles;
                kern<<<(unsigned)blocks, p.threads, p.smem, st>>>(a);
            }
        }
        if (!ring) {
            blocks = a.rows < kBwdBlocks ? a.rows : kBwdBlocks;
            if (VEC == 1 && a.width <= 4 * kWideThreads)
                norm_backward_wide_kernel<T, W, ACC, 1, 4><<<(unsigned)blocks, kWideThreads, 0, st>>>(a);
            else norm_backward_wide_kernel<T, W, ACC, VEC, 0><<<(unsigned)blocks, kWideThreads, 0, st>>>(a);
        }
        GT_CUDA(cudaGetLastError());
        note_launches(1);
    }
    if (!a.want_params) return 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((a.width + 31) / 32), 2);
    cfg.blockDim = dim3(32, 32);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = blocks ? 1 : 0;
    GT_CUDA(cudaLaunchKernelEx(&cfg, norm_params_kernel<W, ACC>, (const ACC *)a.partial, (int)blocks, (int)a.width,
                               dweight, dbias, accumulate));
    note_launches(1);
    return 0;
}

int check_norm(int dtype, int64_t rows, int64_t width, int weight_dtype) {
    if (!known_dtype(dtype) || !known_dtype(weight_dtype)) return fail(GTMOE_EINVAL, "layer norm: unknown dtype");
    if (weight_dtype != dtype && !(dtype == GTMOE_DTYPE_BF16 && weight_dtype == GTMOE_DTYPE_F32))
        return fail(GTMOE_EINVAL, "layer norm: weights have the rows' dtype, or float32 beside bfloat16 rows");
    if (rows < 0) return fail(GTMOE_EINVAL, "layer norm: negative number of rows %lld", (long long)rows);
    if (width < 1 || width > 0x7fffff00)
        return fail(GTMOE_EINVAL, "layer norm: width must be between 1 and 2^31 - 256, got %lld", (long long)width);
    if (!countable(rows, width)) return fail(GTMOE_EINVAL, "layer norm: rows * width is too large");
    return 0;
}

int64_t norm_workspace(int dtype, int64_t rows, int64_t width) {
    const int64_t blocks = rows < kBwdBlocks ? rows : kBwdBlocks;
    return blocks * 2 * width * (int64_t)(dtype == GTMOE_DTYPE_F64 ? 8 : 4);
}

}  // namespace

int norm_take_error(int *code) {
    const int zero = 0;
    GT_CUDA(cudaMemcpyFromSymbol(code, g_norm_error, sizeof(int)));
    if (*code) GT_CUDA(cudaMemcpyToSymbol(g_norm_error, &zero, sizeof(int)));
    return 0;
}

}  // namespace gtmoe

using namespace gtmoe;

extern "C" {

int gtmoe_layer_norm(const void *x, int dtype, int64_t rows, int64_t width, const void *weight, const void *bias,
                     int weight_dtype, double epsilon, void *y, void *mean, void *rstd, void *stream) {
    GT_CHECK(check_norm(dtype, rows, width, weight_dtype));
    if (!(epsilon >= 0) || isinf(epsilon)) return fail(GTMOE_EINVAL, "layer norm: epsilon must be finite and not negative");
    if (rows == 0) return 0;
    if (!x || !y) return fail(GTMOE_EINVAL, "layer norm: x and y must be given");
    const int64_t bytes = rows * width * (int64_t)dtype_size(dtype);
    const int64_t pbytes = width * (int64_t)dtype_size(weight_dtype);
    const int64_t sbytes = rows * (int64_t)(dtype == GTMOE_DTYPE_F64 ? 8 : 4);
    if (overlaps_shifted(x, bytes, y, bytes) || ranges_overlap(weight, pbytes, y, bytes) ||
        ranges_overlap(bias, pbytes, y, bytes) || ranges_overlap(mean, sbytes, y, bytes) ||
        ranges_overlap(rstd, sbytes, y, bytes) || ranges_overlap(mean, sbytes, x, bytes) ||
        ranges_overlap(rstd, sbytes, x, bytes) || ranges_overlap(mean, sbytes, rstd, sbytes) ||
        ranges_overlap(mean, sbytes, weight, pbytes) || ranges_overlap(mean, sbytes, bias, pbytes) ||
        ranges_overlap(rstd, sbytes, weight, pbytes) || ranges_overlap(rstd, sbytes, bias, pbytes))
        return fail(GTMOE_EINVAL, "layer norm: an output overlaps another argument (y may be x itself)");
    DeviceScope scope;
    const size_t es = dtype_size(dtype), ws = dtype_size(weight_dtype), ss = dtype == GTMOE_DTYPE_F64 ? 8 : 4;
    GT_CHECK(scope.enter({{x, "x", es}, {weight, "weight", ws}, {bias, "bias", ws}, {y, "y", es}, {mean, "mean", ss},
                          {rstd, "rstd", ss}}));
    NormArgs a = {};
    a.x = x, a.weight = weight, a.bias = bias, a.y = y, a.mean = mean, a.rstd = rstd;
    a.rows = rows, a.width = (int)width, a.eps = epsilon;
    cudaStream_t st = (cudaStream_t)stream;
    // 16-byte accesses where every row and parameter starts on 16 bytes
    const int vec = 16 / (int)dtype_size(dtype);
    const bool wide = width % vec == 0 && aligned16(x) && aligned16(y) && aligned16(weight) && aligned16(bias);
    if (dtype == GTMOE_DTYPE_F64)
        return wide ? forward_vec<double, double, double, 2>(a, scope.device(), st)
                    : forward_vec<double, double, double, 1>(a, scope.device(), st);
    if (dtype == GTMOE_DTYPE_F32)
        return wide ? forward_vec<float, float, float, 4>(a, scope.device(), st)
                    : forward_vec<float, float, float, 1>(a, scope.device(), st);
    if (weight_dtype == GTMOE_DTYPE_F32)
        return wide ? forward_vec<__nv_bfloat16, float, float, 8>(a, scope.device(), st)
                    : forward_vec<__nv_bfloat16, float, float, 1>(a, scope.device(), st);
    return wide ? forward_vec<__nv_bfloat16, __nv_bfloat16, float, 8>(a, scope.device(), st)
                : forward_vec<__nv_bfloat16, __nv_bfloat16, float, 1>(a, scope.device(), st);
}

int gtmoe_layer_norm_workspace(int dtype, int64_t rows, int64_t width, int64_t *bytes) {
    GT_CHECK(check_norm(dtype, rows, width, dtype));
    if (!bytes) return fail(GTMOE_EINVAL, "layer norm: bytes is NULL");
    *bytes = norm_workspace(dtype, rows, width);
    return 0;
}

int gtmoe_layer_norm_backward(const void *dy, const void *x, int dtype, int64_t rows, int64_t width,
                              const void *weight, int weight_dtype, const void *mean, const void *rstd,
                              const void *dresidual, void *dx, void *dweight, void *dbias, int accumulate,
                              void *workspace, int64_t workspace_bytes, void *stream) {
    GT_CHECK(check_norm(dtype, rows, width, weight_dtype));
    if (rows > 0 && (!dy || !x || !mean || !rstd || !dx))
        return fail(GTMOE_EINVAL, "layer norm: dy, x, mean, rstd and dx must be given");
    const int want = dweight || dbias;
    if (rows == 0 && !want) return 0;
    const int64_t need = norm_workspace(dtype, rows, width);
    if (want && need && (!workspace || workspace_bytes < need))
        return fail(GTMOE_EINVAL, "layer norm: the weight gradients need %lld bytes of workspace, got %lld",
                    (long long)need, (long long)(workspace ? workspace_bytes : 0));
    const int64_t bytes = rows * width * (int64_t)dtype_size(dtype);
    const int64_t pbytes = width * (int64_t)dtype_size(weight_dtype);
    const int64_t sbytes = rows * (int64_t)(dtype == GTMOE_DTYPE_F64 ? 8 : 4);
    const int64_t wbytes = want ? need : 0;
    bool bad = overlaps_shifted(dy, bytes, dx, bytes) || overlaps_shifted(x, bytes, dx, bytes) ||
               overlaps_shifted(dresidual, bytes, dx, bytes);
    const void *small[] = {weight, dweight, dbias};
    const void *large[] = {dy, x, dresidual, dx};
    for (const void *s : small)
        bad |= ranges_overlap(s, pbytes, dx, bytes) || ranges_overlap(s, pbytes, workspace, wbytes);
    for (const void *l : large)
        bad |= ranges_overlap(dweight, pbytes, l, bytes) || ranges_overlap(dbias, pbytes, l, bytes) ||
               ranges_overlap(workspace, wbytes, l, bytes);
    for (const void *s : {mean, rstd})
        bad |= ranges_overlap(s, sbytes, dx, bytes) || ranges_overlap(s, sbytes, dweight, pbytes) ||
               ranges_overlap(s, sbytes, dbias, pbytes) || ranges_overlap(s, sbytes, workspace, wbytes);
    bad |= ranges_overlap(dweight, pbytes, dbias, pbytes) || ranges_overlap(weight, pbytes, dweight, pbytes) ||
           ranges_overlap(weight, pbytes, dbias, pbytes);
    if (bad) return fail(GTMOE_EINVAL, "layer norm: an output overlaps another argument (dx may be dy, x or dresidual itself)");
    DeviceScope scope;
    const size_t es = dtype_size(dtype), ws = dtype_size(weight_dtype), ss = dtype == GTMOE_DTYPE_F64 ? 8 : 4;
    GT_CHECK(scope.enter({{rows ? dy : nullptr, "dy", es}, {rows ? x : nullptr, "x", es}, {weight, "weight", ws},
                          {rows ? mean : nullptr, "mean", ss}, {rows ? rstd : nullptr, "rstd", ss},
                          {rows ? dresidual : nullptr, "dresidual", es}, {rows ? dx : nullptr, "dx", es},
                          {dweight, "dweight", ws}, {dbias, "dbias", ws},
                          {wbytes ? workspace : nullptr, "workspace", 16}}));
    NormArgs a = {};
    a.x = x, a.dy = dy, a.weight = weight, a.mean = (void *)mean, a.rstd = (void *)rstd, a.dres = dresidual, a.dx = dx;
    a.rows = rows, a.width = (int)width, a.partial = workspace, a.want_params = want;
    cudaStream_t st = (cudaStream_t)stream;
    const int vec = 16 / (int)dtype_size(dtype);
    const bool wide = width % vec == 0 && aligned16(x) && aligned16(dy) && aligned16(dresidual) && aligned16(dx) &&
                      aligned16(weight);
    if (dtype == GTMOE_DTYPE_F64)
        return wide ? backward_vec<double, double, double, 2>(a, dweight, dbias, accumulate, scope.device(), st)
                    : backward_vec<double, double, double, 1>(a, dweight, dbias, accumulate, scope.device(), st);
    if (dtype == GTMOE_DTYPE_F32)
        return wide ? backward_vec<float, float, float, 4>(a, dweight, dbias, accumulate, scope.device(), st)
                    : backward_vec<float, float, float, 1>(a, dweight, dbias, accumulate, scope.device(), st);
    if (weight_dtype == GTMOE_DTYPE_F32)
        return wide ? backward_vec<__nv_bfloat16, float, float, 8>(a, dweight, dbias, accumulate, scope.device(), st)
                    : backward_vec<__nv_bfloat16, float, float, 1>(a, dweight, dbias, accumulate, scope.device(), st);
    return wide ? backward_vec<__nv_bfloat16, __nv_bfloat16, float, 8>(a, dweight, dbias, accumulate, scope.device(), st)
                : backward_vec<__nv_bfloat16, __nv_bfloat16, float, 1>(a, dweight, dbias, accumulate, scope.device(), st);
}

}  // extern "C"
