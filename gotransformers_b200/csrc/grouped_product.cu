// grouped_product.cu -- matrix products of rows grouped by expert, and the
// gradients of both factors: the C entries, and the kernel on the SIMT cores
// that takes every type, size and alignment.  bf16 operands that tile go to
// the tensor cores (grouped_dense.cu).
#include "grouped.h"

namespace gtmoe {
namespace {

__device__ int g_error;  // first code a kernel recorded since the last check

constexpr int kTile = 64;   // rows and columns of a block's tile
constexpr int kStep = 16;   // terms of the sums per shared-memory step
constexpr int kThreads = 256;

// C[i][j] = sum over p of A(i, p) B(j, p):
//   kProduct     i row, j output, p input:   A = X[i][p],  B = W_g[j][p]
//   kInputGrad   i row, j input,  p output:  A = dY[i][p], B = W_g[p][j]
//   kWeightGrad  i output, j input, p row:   A = dY[p][i], B = X[p][j]
// 4 x 4 outputs per thread, each one sum in ascending p in ACC.
template <typename T, typename ACC, typename OUT, GroupedOp OP>
__global__ void __launch_bounds__(kThreads) grouped_simt_product_kernel(const GroupedProduct a) {
    __shared__ ACC sa[kStep][kTile + 4], sb[kStep][kTile + 4];
    __shared__ int start[kMaxGroups + 1], tiles[kMaxGroups + 1], scratch[kThreads];
    const int64_t n_j = OP == kProduct ? a.outputs : a.inputs;
    const int64_t j_tiles = (n_j + kTile - 1) / kTile;
    const bool ok = OP == kWeightGrad ? group_ranges(a.counts, a.groups, a.rows, kAnyRows, 1,
                                                     (int)((a.outputs + kTile - 1) / kTile), start, tiles, scratch)
                                      : group_ranges(a.counts, a.groups, a.rows, kTile, 0, 1, start, tiles, scratch);
    if (!ok && blockIdx.x == 0 && threadIdx.x == 0) atomicCAS(&g_error, 0, kErrBadCounts);
    const int64_t total = (int64_t)tiles[a.groups] * j_tiles;
    const T *A = (const T *)a.a, *B = (const T *)a.b;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    int g = 0;
    for (int64_t u = blockIdx.x; u < total; u += gridDim.x) {
        const int it = (int)(u / j_tiles);
        while (tiles[g + 1] <= it) g++;
        const int64_t i0 = (int64_t)(it - tiles[g]) * kTile, j0 = (u % j_tiles) * kTile;
        const int64_t r0 = start[g], m = start[g + 1] - start[g];
        const int64_t i_end = OP == kWeightGrad ? a.outputs : m;
        const int64_t p_end = OP == kProduct ? a.inputs : OP == kInputGrad ? a.outputs : m;
        const T *Wg = B + (int64_t)g * a.outputs * a.inputs;
        ACC acc[4][4] = {};
        for (int64_t p0 = 0; p0 < p_end; p0 += kStep) {
            // consecutive threads along the operand's contiguous axis
#pragma unroll
            for (int q = 0; q < kTile * kStep / kThreads; q++) {
                const int e = q * kThreads + threadIdx.x;
                const int ap = OP == kWeightGrad ? e / kTile : e % kStep, ai = OP == kWeightGrad ? e % kTile : e / kStep;
                const int bp = OP == kProduct ? e % kStep : e / kTile, bj = OP == kProduct ? e / kStep : e % kTile;
                ACC va = ACC(0), vb = ACC(0);
                if (i0 + ai < i_end && p0 + ap < p_end)
                    va = (ACC)(OP == kWeightGrad ? A[(r0 + p0 + ap) * a.outputs + i0 + ai]
                                                 : A[(r0 + i0 + ai) * (OP == kProduct ? a.inputs : a.outputs) + p0 + ap]);
                if (j0 + bj < n_j && p0 + bp < p_end)
                    vb = (ACC)(OP == kProduct      ? Wg[(j0 + bj) * a.inputs + p0 + bp]
                               : OP == kInputGrad ? Wg[(p0 + bp) * a.inputs + j0 + bj]
                                                  : B[(r0 + p0 + bp) * a.inputs + j0 + bj]);
                sa[ap][ai] = va;
                sb[bp][bj] = vb;
            }
            __syncthreads();
#pragma unroll
            for (int p = 0; p < kStep; p++) {
                ACC ra[4], rb[4];
#pragma unroll
                for (int q = 0; q < 4; q++) {
                    ra[q] = sa[p][ty * 4 + q];
                    rb[q] = sb[p][tx * 4 + q];
                }
#pragma unroll
                for (int x = 0; x < 4; x++)
#pragma unroll
                    for (int y = 0; y < 4; y++) acc[x][y] += ra[x] * rb[y];
            }
            __syncthreads();
        }
        OUT *C = (OUT *)a.c;
        const int64_t base = OP == kWeightGrad ? (int64_t)g * a.outputs * a.inputs : r0 * n_j;
#pragma unroll
        for (int x = 0; x < 4; x++)
#pragma unroll
            for (int y = 0; y < 4; y++) {
                const int64_t i = i0 + ty * 4 + x, j = j0 + tx * 4 + y;
                if (i < i_end && j < n_j) {
                    OUT &o = C[base + i * n_j + j];
                    o = (OUT)(OP == kWeightGrad && a.accumulate ? (ACC)o + acc[x][y] : acc[x][y]);
                }
            }
    }
}

template <typename T, typename ACC, typename OUT, GroupedOp OP>
int launch_simt(const GroupedProduct &p, cudaStream_t st) {
    const int64_t n_j = OP == kProduct ? p.outputs : p.inputs;
    // at most this many tiles: the rows of a group end inside a tile
    const int64_t i_tiles = OP == kWeightGrad ? (int64_t)p.groups * ((p.outputs + kTile - 1) / kTile)
                                              : p.rows / kTile + (p.rows < p.groups ? p.rows : p.groups);
    const int64_t most = i_tiles * ((n_j + kTile - 1) / kTile);
    const unsigned grid = (unsigned)(most < 148 * 16 ? most : 148 * 16);
    grouped_simt_product_kernel<T, ACC, OUT, OP><<<grid, kThreads, 0, st>>>(p);
    GT_CUDA(cudaGetLastError());
    note_launches(1);
    return 0;
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
    if ((p.outputs + kTile - 1) / kTile * p.groups > 0x7fffffff)
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
