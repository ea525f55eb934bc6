// grouped_product.cu -- matrix products of rows grouped by expert, and the
// gradients of both factors: the C entries, and the kernel on the SIMT cores
// that takes every type, size and alignment.  bf16 operands that tile go to
// the tensor cores (grouped_dense.cu).
#include "grouped.h"

namespace gtmoe {
namespace {

__device__ int g_error;  // first code a kernel recorded since the last check

constexpr int kThreads = 256;
constexpr int kRunTerms = 256;      // terms of a long float32 sum per run
constexpr int kOneRunTerms = 1024;  // and how many a sum may have that is made in one

// One operand of a tile: TILE values along the tile's axis by STEP terms.
// KMAJOR: the terms are contiguous in memory, else the tile's axis is.
// Consecutive threads load along the contiguous axis, into registers while the
// step before is multiplied, then into shared memory as [term][value].
template <typename T, typename ACC, int TILE, int STEP, bool KMAJOR>
struct Operand {
    static constexpr int kLoads = TILE * STEP / kThreads;
    const T *p;      // this thread's first value of step 0
    int64_t q_step, k_step;
    int at, term;    // its place in the tile
    int64_t n, terms;
    ACC v[kLoads];

    // base: value 0, term 0; ld: distance of the outer axis
    __device__ __forceinline__ void begin(const T *base, int64_t ld, int64_t n_values, int64_t n_terms) {
        const int t = threadIdx.x;
        term = KMAJOR ? t % STEP : t / TILE;
        at = KMAJOR ? t / STEP : t % TILE;
        p = base + (KMAJOR ? at * ld + term : term * ld + at);
        q_step = (KMAJOR ? kThreads / STEP : kThreads / TILE) * ld;
        k_step = KMAJOR ? STEP : STEP * ld;
        n = n_values;
        terms = n_terms;
    }
    __device__ __forceinline__ void load(int64_t k0) {
#pragma unroll
        for (int q = 0; q < kLoads; q++) {
            const int i = KMAJOR ? at + q * (kThreads / STEP) : at;
            const int64_t k = k0 + (KMAJOR ? term : term + q * (kThreads / TILE));
            v[q] = i < n && k < terms ? (ACC)p[q * q_step] : ACC(0);
        }
        p += k_step;
    }
    __device__ __forceinline__ void store(ACC (*s)[TILE + 4]) const {
#pragma unroll
        for (int q = 0; q < kLoads; q++) {
            if (KMAJOR) s[term][at + q * (kThreads / STEP)] = v[q];
            else s[term + q * (kThreads / TILE)][at] = v[q];
        }
    }
};

// C[i][j] = sum over p of A(i, p) B(j, p):
//   kProduct     i row, j output, p input:   A = X[i][p],  B = W_g[j][p]
//   kInputGrad   i row, j input,  p output:  A = dY[i][p], B = W_g[p][j]
//   kWeightGrad  i output, j input, p row:   A = dY[p][i], B = X[p][j]
// TI x TJ outputs per block, (TI / 16) x (TJ / 16) per thread, each one sum in
// ascending p, STEP terms per shared-memory step.  Two buffers: one barrier per
// step.  RUNS: a long float32 sum is made in runs of kRunTerms terms, which join
// a total in local memory, and what that addition rounds off is carried on
// (fold()).  One sum was off by 2.1e-5 after 1536 equal terms, 5.9e-5 after
// 65536, and stopped growing at 2^24 ones.  The runs take 7 % more time at most
// (4096 rows in 8 groups, 4096 -> 1024: 842 -> 891 us; weight gradient of 16384
// rows in 8 groups, 1024 x 1024: 927 -> 910 us).  FFMA-bound: 16384 rows in 8 groups, 1024 x 1024, float32
// 45 TF/s (cuBLAS's float32 product of this size of sums 57).
template <typename T, typename ACC, typename OUT, GroupedOp OP, bool RUNS, int TI, int TJ, int STEP>
__global__ void __launch_bounds__(kThreads, TI == 128 && RUNS ? 2 : 0) grouped_simt_product_kernel(const GroupedProduct a) {
    // outputs per thread and axis, in runs of VI and VJ
    constexpr int RI = TI / 16, VI = RI < 4 ? RI : 4, RJ = TJ / 16, VJ = RJ < 4 ? RJ : 4;
    __shared__ __align__(16) ACC sa[2][STEP][TI + 4], sb[2][STEP][TJ + 4];
    __shared__ int start[kMaxGroups + 1], tiles[kMaxGroups + 1], scratch[kThreads / 32];
    const int64_t n_j = OP == kProduct ? a.outputs : a.inputs;
    const int64_t j_tiles = (n_j + TJ - 1) / TJ;
    const bool ok = OP == kWeightGrad ? group_ranges(a.counts, a.groups, a.rows, kAnyRows, 1,
                                                     (int)((a.outputs + TI - 1) / TI), start, tiles, scratch)
                                      : group_ranges(a.counts, a.groups, a.rows, TI, 0, 1, start, tiles, scratch);
    if (!ok && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(&g_error, 0, kErrBadCounts);
    const int64_t total = (int64_t)tiles[a.groups] * j_tiles;
    const T *A = (const T *)a.a, *B = (const T *)a.b;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int g = 0;
    for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
        const int it = (int)(u / j_tiles);
        while (tiles[g + 1] <= it) g++;
        const int64_t i0 = (int64_t)(it - tiles[g]) * TI, j0 = (u % j_tiles) * TJ;
        const int64_t r0 = start[g], m = start[g + 1] - start[g];
        const int64_t i_end = OP == kWeightGrad ? a.outputs : m;
        const int64_t p_end = OP == kProduct ? a.inputs : OP == kInputGrad ? a.outputs : m;
        const T *Wg = B + (int64_t)g * a.outputs * a.inputs;
        Operand<T, ACC, TI, STEP, OP != kWeightGrad> oa;
        Operand<T, ACC, TJ, STEP, OP == kProduct> ob;
        if (OP == kWeightGrad) oa.begin(A + r0 * a.outputs + i0, a.outputs, i_end - i0, p_end);
        else oa.begin(A + (r0 + i0) * p_end, p_end, i_end - i0, p_end);
        if (OP == kProduct) ob.begin(Wg + j0 * a.inputs, a.inputs, n_j - j0, p_end);
        else if (OP == kInputGrad) ob.begin(Wg + j0, a.inputs, n_j - j0, p_end);
        else ob.begin(B + r0 * a.inputs + j0, a.inputs, n_j - j0, p_end);
        ACC acc[RI][RJ] = {};
        oa.load(0);
        ob.load(0);
        // in local memory, which sums of one run do not touch: at is 0, but the compiler does not see that and so
        // keeps the registers for the products
        float total[RI * RJ];
        const int at = (int)(a.rows >> 40);
        int buf = 0;
        for (int64_t p0 = 0; p0 < p_end; p0 += STEP, buf ^= 1) {
            oa.store(sa[buf]);
            ob.store(sb[buf]);
            __syncthreads();  // also: the step before last has been multiplied by every thread
            if (p0 + STEP < p_end) {
                oa.load(p0 + STEP);
                ob.load(p0 + STEP);
            }
#pragma unroll
            for (int p = 0; p < STEP; p++) {
                ACC ra[RI], rb[RJ];
#pragma unroll
                for (int x = 0; x < RI; x++) ra[x] = sa[buf][p][x / VI * 16 * VI + ty * VI + x % VI];
#pragma unroll
                for (int y = 0; y < RJ; y++) rb[y] = sb[buf][p][y / VJ * 16 * VJ + tx * VJ + y % VJ];
#pragma unroll
                for (int x = 0; x < RI; x++)
#pragma unroll
                    for (int y = 0; y < RJ; y++) acc[x][y] += ra[x] * rb[y];
            }
            if constexpr (RUNS)
                if ((p0 + STEP) % kRunTerms == 0 && p0 + STEP < p_end) {
                    const bool first = p0 + STEP == kRunTerms;
#pragma unroll
                    for (int x = 0; x < RI; x++)
#pragma unroll
                        for (int y = 0; y < RJ; y++) {
                            float &t = total[at + x * RJ + y];
                            if (first) t = 0.f;
                            fold(t, acc[x][y]);
                        }
                }
        }
        if constexpr (RUNS)
            if (p_end > kRunTerms)
#pragma unroll
                for (int x = 0; x < RI; x++)
#pragma unroll
                    for (int y = 0; y < RJ; y++) acc[x][y] += total[at + x * RJ + y];
        __syncthreads();  // the buffers are free for the next tile
        OUT *C = (OUT *)a.c;
        const int64_t base = OP == kWeightGrad ? (int64_t)g * a.outputs * a.inputs : r0 * n_j;
#pragma unroll
        for (int x = 0; x < RI; x++)
#pragma unroll
            for (int y = 0; y < RJ; y++) {
                const int64_t i = i0 + x / VI * 16 * VI + ty * VI + x % VI, j = j0 + y / VJ * 16 * VJ + tx * VJ + y % VJ;
                if (i < i_end && j < n_j) {
                    OUT &o = C[base + i * n_j + j];
                    o = (OUT)(OP == kWeightGrad && a.accumulate ? (ACC)o + acc[x][y] : acc[x][y]);
                }
            }
    }
}

// At most this many tiles: the rows of a group end inside a tile.
template <GroupedOp OP>
int64_t most_tiles(const GroupedProduct &p, int ti, int tj) {
    const int64_t n_j = OP == kProduct ? p.outputs : p.inputs;
    const int64_t i_tiles = OP == kWeightGrad ? (int64_t)p.groups * ((p.outputs + ti - 1) / ti)
                                              : p.rows / ti + (p.rows < p.groups ? p.rows : p.groups);
    return i_tiles * ((n_j + tj - 1) / tj);
}

template <typename T, typename ACC, typename OUT, GroupedOp OP, bool RUNS, int TI, int TJ, int STEP>
int launch_simt_tile(const GroupedProduct &p, cudaStream_t st) {
    const int64_t most = most_tiles<OP>(p, TI, TJ);
    const unsigned grid = (unsigned)(most < 148 * 16 ? most : 148 * 16);
    grouped_simt_product_kernel<T, ACC, OUT, OP, RUNS, TI, TJ, STEP><<<grid, kThreads, 0, st>>>(p);
    GT_CUDA(cudaGetLastError());
    note_launches(1);
    return 0;
}

// Groups of few rows on average: tiles of 32 rows, and twice the terms per
// step, since the steps' latencies are what a block then waits for.  Else tiles
// of 128 x 128 (64 products per 16 values read) once they are enough for every
// SM and the groups fill them, else of 64 x 64; float64 has shared memory for
// the latter only.
template <typename T, typename ACC, typename OUT, GroupedOp OP, bool RUNS>
int launch_simt_tiles(const GroupedProduct &p, cudaStream_t st) {
    if constexpr (sizeof(ACC) == 4) {
        const int64_t average = p.rows / p.groups;
        if constexpr (OP != kWeightGrad)
            if (average < 48) return launch_simt_tile<T, ACC, OUT, OP, RUNS, 32, 64, 32>(p, st);
        if ((OP == kWeightGrad || average >= 96) && most_tiles<OP>(p, 128, 128) >= 2 * 148)
            return launch_simt_tile<T, ACC, OUT, OP, RUNS, 128, 128, 16>(p, st);
    }
    return launch_simt_tile<T, ACC, OUT, OP, RUNS, 64, 64, 16>(p, st);
}

// Float32 sums that may have more than kOneRunTerms terms are made in runs.
template <typename T, typename ACC, typename OUT, GroupedOp OP>
int launch_simt(const GroupedProduct &p, cudaStream_t st) {
    if constexpr (sizeof(ACC) == 4)
        if ((OP == kProduct ? p.inputs : OP == kInputGrad ? p.outputs : p.rows) > kOneRunTerms)
            return launch_simt_tiles<T, ACC, OUT, OP, true>(p, st);
    return launch_simt_tiles<T, ACC, OUT, OP, false>(p, st);
}

template <typename T, typename ACC>
int launch_simt_op(const GroupedProduct &p, cudaStream_t st) {
    if (p.op == kProduct) return launch_simt<T, ACC, T, kProduct>(p, st);
    if (p.op == kInputGrad) return launch_simt<T, ACC, T, kInputGrad>(p, st);
    if (p.out_dtype == p.dtype) return launch_simt<T, ACC, T, kWeightGrad>(p, st);
    return launch_simt<T, ACC, float, kWeightGrad>(p, st);
}

int check_sizes(const GroupedProduct &p) {
    if (!known_dtype(p.dtype) || !known_dtype(p.out_dtype)) return fail(GTMOE_EINVAL, "grouped product: unknown dtype");
    if (p.out_dtype != p.dtype && !(p.dtype == GTMOE_DTYPE_BF16 && p.out_dtype == GTMOE_DTYPE_F32))
        return fail(GTMOE_EINVAL, "grouped product: weight gradients have the operands' dtype, or float32 beside bfloat16");
    if (p.rows < 0 || p.rows > 0x7fffff00)
        return fail(GTMOE_EINVAL, "grouped product: rows must be between 0 and 2^31 - 256, got %lld", (long long)p.rows);
    if (p.inputs < 1 || p.outputs < 1 || p.inputs > 0x7fffff00 || p.outputs > 0x7fffff00)
        return fail(GTMOE_EINVAL, "grouped product: inputs and outputs must be between 1 and 2^31 - 256, got %lld and %lld",
                    (long long)p.inputs, (long long)p.outputs);
    if (p.groups < 1 || p.groups > kMaxGroups)
        return fail(GTMOE_EINVAL, "grouped product: needs 1 to %d groups, got %d", kMaxGroups, p.groups);
    if (!countable(p.rows, p.inputs) || !countable(p.rows, p.outputs) || !countable(p.inputs * p.groups, p.outputs))
        return fail(GTMOE_EINVAL, "grouped product: an operand is too large");
    if ((p.outputs + 63) / 64 * p.groups > 0x7fffffff)
        return fail(GTMOE_EINVAL, "grouped product: too many outputs for %d groups", p.groups);
    return 0;
}

int run_grouped(const GroupedProduct &p, const char *a_name, const char *b_name, const char *c_name,
                int64_t workspace_bytes, void *stream) {
    GT_CHECK(check_sizes(p));
    if (p.rows == 0 && p.op != kWeightGrad) return 0;
    if (p.rows == 0 && p.accumulate) return 0;
    if ((p.rows > 0 && (!p.a || !p.b)) || !p.c || !p.counts)
        return fail(GTMOE_EINVAL, "grouped product: %s, %s, counts and %s must be given", a_name, b_name, c_name);
    const int64_t es = (int64_t)dtype_size(p.dtype);
    const int64_t xb = p.rows * p.inputs * es, yb = p.rows * p.outputs * es;
    const int64_t wn = p.groups * p.inputs * p.outputs;
    const int64_t ab = p.op == kProduct ? xb : yb, bb = p.op == kWeightGrad ? xb : wn * es;
    const int64_t cb = p.op == kProduct     ? yb
                       : p.op == kInputGrad ? xb
                                            : wn * (int64_t)dtype_size(p.out_dtype);
    if (ranges_overlap(p.c, cb, p.a, ab) || ranges_overlap(p.c, cb, p.b, bb) || ranges_overlap(p.c, cb, p.counts, 8 * (int64_t)p.groups))
        return fail(GTMOE_EINVAL, "grouped product: %s overlaps another argument", c_name);
    const int64_t need = p.op == kWeightGrad && grouped_dense_usable(p)
                             ? grouped_dense_workspace(p.rows, p.inputs, p.outputs, p.groups)
                             : 0;
    if (need && (!p.workspace || workspace_bytes < need))
        return fail(GTMOE_EINVAL, "grouped product: the weight gradients need %lld bytes of workspace, got %lld",
                    (long long)need, (long long)(p.workspace ? workspace_bytes : 0));
    if (ranges_overlap(p.workspace, need, p.a, ab) || ranges_overlap(p.workspace, need, p.b, bb) ||
        ranges_overlap(p.workspace, need, p.c, cb) || ranges_overlap(p.workspace, need, p.counts, 8 * (int64_t)p.groups))
        return fail(GTMOE_EINVAL, "grouped product: workspace overlaps another argument");
    DeviceScope scope;
    GT_CHECK(scope.enter({{p.c, c_name, dtype_size(p.out_dtype)}, {ab ? p.a : nullptr, a_name, (size_t)es},
                          {bb ? p.b : nullptr, b_name, (size_t)es}, {p.counts, "counts", 8},
                          {need ? p.workspace : nullptr, "workspace", 16}}));
    cudaStream_t st = (cudaStream_t)stream;
    if (grouped_dense_usable(p)) return launch_grouped_dense(p, scope.device(), st);
    if (p.dtype == GTMOE_DTYPE_F64) return launch_simt_op<double, double>(p, st);
    if (p.dtype == GTMOE_DTYPE_F32) return launch_simt_op<float, float>(p, st);
    return launch_simt_op<__nv_bfloat16, float>(p, st);
}

}  // namespace

int grouped_take_error(int *code) {
    GT_CUDA(cudaDeviceSynchronize());
    int simt = 0, dense = 0;
    const int zero = 0;
    GT_CUDA(cudaMemcpyFromSymbol(&simt, g_error, sizeof(int)));
    if (simt) GT_CUDA(cudaMemcpyToSymbol(g_error, &zero, sizeof(int)));
    GT_CHECK(grouped_dense_take_error(&dense));
    // an expired wait before refused counts
    *code = dense && dense != kErrBadCounts ? dense : simt ? simt : dense;
    return 0;
}

}  // namespace gtmoe

using namespace gtmoe;

extern "C" {

int gtmoe_grouped_product(const void *x, const void *w, int dtype, int64_t rows, int64_t inputs, int64_t outputs,
                          int groups, const int64_t *counts, void *y, void *stream) {
    const GroupedProduct p = {kProduct, dtype, dtype, 0, rows, inputs, outputs, groups, counts, x, w, y, nullptr};
    return run_grouped(p, "x", "w", "y", 0, stream);
}

int gtmoe_grouped_product_input_grad(const void *dy, const void *w, int dtype, int64_t rows, int64_t inputs,
                                     int64_t outputs, int groups, const int64_t *counts, void *dx, void *stream) {
    const GroupedProduct p = {kInputGrad, dtype, dtype, 0, rows, inputs, outputs, groups, counts, dy, w, dx, nullptr};
    return run_grouped(p, "dy", "w", "dx", 0, stream);
}

int gtmoe_grouped_product_workspace(int dtype, int64_t rows, int64_t inputs, int64_t outputs, int groups,
                                    int64_t *bytes) {
    const GroupedProduct p = {kWeightGrad, dtype, dtype, 0, rows, inputs, outputs, groups, nullptr, nullptr, nullptr, nullptr, nullptr};
    GT_CHECK(check_sizes(p));
    if (!bytes) return fail(GTMOE_EINVAL, "grouped product: bytes is NULL");
    // whether the operands' addresses suit the tensor cores is not known here
    *bytes = grouped_dense_usable(p) ? grouped_dense_workspace(rows, inputs, outputs, groups) : 0;
    return 0;
}

int gtmoe_grouped_product_weight_grad(const void *dy, const void *x, int dtype, int64_t rows, int64_t inputs,
                                      int64_t outputs, int groups, const int64_t *counts, void *dw, int dw_dtype,
                                      int accumulate, void *workspace, int64_t workspace_bytes, void *stream) {
    const GroupedProduct p = {kWeightGrad, dtype, dw_dtype, accumulate, rows, inputs, outputs,
                              groups,      counts, dy,      x,          dw,   workspace};
    return run_grouped(p, "dy", "x", "dw", workspace_bytes, stream);
}

}  // extern "C"
