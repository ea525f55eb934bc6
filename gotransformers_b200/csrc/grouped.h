// grouped.h -- the dense products of rows grouped by expert
// (grouped_product.cu on the SIMT cores, grouped_dense.cu on the tensor
// cores): the three products, and the groups' row ranges.
#pragma once

#include "operators.h"

namespace gtmoe {

// With rows r of group g, X rows x inputs, W groups x outputs x inputs, dY
// rows x outputs:
//   kProduct     Y[r]  = X[r] W_g^T
//   kInputGrad   dX[r] = dY[r] W_g
//   kWeightGrad  dW_g  = sum over r of dY[r]^T X[r]
enum GroupedOp { kProduct = 0, kInputGrad = 1, kWeightGrad = 2 };

struct GroupedProduct {
    GroupedOp op;
    int dtype;        // of X, W, dY and of Y, dX
    int out_dtype;    // of dW: dtype, or float32 beside bf16
    int accumulate;   // dW is added to
    int64_t rows, inputs, outputs;
    int groups;
    const int64_t *counts;  // rows per group (device)
    const void *a;    // X, dY, dY
    const void *b;    // W, W, X
    void *c;          // Y, dX, dW
    void *workspace;  // kWeightGrad: grouped_dense_workspace() bytes
};

constexpr int kMaxGroups = kMaxRoutedExperts;
constexpr int kAnyRows = 0x7fffffff;  // a tile_rows that no group fills

// The sum of the threads' values before this one's, cut at `most` (< 2^31;
// cutting a sum of non-negative values early or late gives the same).  Every
// thread of the block calls it; `scratch` is one word per warp, free again when
// it returns.
__device__ __forceinline__ int64_t block_scan(int64_t own, int64_t most, int *scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    auto cut = [&](int64_t v) { return (int)(v < most ? v : most); };
    auto warp_scan = [&](int v) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, v, o);
            if (lane >= o) v = cut((int64_t)v + u);
        }
        return v;
    };
    const int sum = warp_scan(cut(own));
    if (lane == 31) scratch[warp] = sum;
    __syncthreads();
    // every warp scans the warps' sums for itself
    const int all = warp_scan(lane < warps ? scratch[lane] : 0);
    const int before = __shfl_sync(0xffffffffu, all, (warp + 31) & 31);
    const int mine = __shfl_up_sync(0xffffffffu, sum, 1);
    __syncthreads();
    return cut((int64_t)(warp ? before : 0) + (lane ? mine : 0));
}

// Group g's rows are start[g] .. start[g + 1], cut at `rows`; a negative
// count is no rows.  tiles[g] is the number of tiles before group g: `per` for
// each run of tile_rows rows that it has begun, of which it has at least
// `least`.  Every thread of the block calls it; start and tiles are groups + 1
// words of shared memory, scratch one word per warp.  True when the counts were
// as they should be.
__device__ __forceinline__ bool group_ranges(const int64_t *__restrict__ counts, int groups, int64_t rows,
                                             int tile_rows, int least, int per, int *start, int *tiles,
                                             int *scratch) {
    const int threads = blockDim.x, t = threadIdx.x;
    const int run = (groups + threads - 1) / threads;
    const int g0 = min(groups, t * run), g1 = min(groups, g0 + run);
    int64_t sum = 0;
    bool ok = true;
    for (int g = g0; g < g1; g++) {
        int64_t c = counts[g];
        ok = ok && c >= 0 && c <= rows;
        c = c < 0 ? 0 : c < rows ? c : rows;
        sum += c;
        start[g + 1] = (int)c;
    }
    // one more than `rows` still tells a sum that is too large
    int64_t at = block_scan(sum, rows + 1, scratch);
    ok = ok && at + sum <= rows;
    int64_t n_tiles = 0;
    for (int g = g0; g < g1; g++) {
        const int64_t first = at < rows ? at : rows;
        at += start[g + 1];
        const int64_t last = at < rows ? at : rows;
        start[g + 1] = (int)last;
        const int64_t begun = (last - first + tile_rows - 1) / tile_rows;
        const int64_t n = per * (begun < least ? least : begun);
        n_tiles += n;
        tiles[g + 1] = (int)n;
    }
    at = block_scan(n_tiles, 0x7ffffffe, scratch);
    for (int g = g0; g < g1; g++) {
        at += tiles[g + 1];
        tiles[g + 1] = (int)at;
    }
    if (t == 0) start[0] = tiles[0] = 0;
    return __syncthreads_and(ok);
}

// Adds `part`, the sum of a run of terms, to `total`; what the addition rounds
// off is where the next run starts from (Knuth's two-sum), so that a sum's
// error is that of its runs however many they are.
__device__ __forceinline__ void fold(float &total, float &part) {
    const float t = __fadd_rn(total, part), b = __fsub_rn(t, total);
    const float off = __fadd_rn(__fsub_rn(total, __fsub_rn(t, b)), __fsub_rn(part, b));
    total = t;
    part = isfinite(t) ? off : 0.f;  // an infinite sum has no remainder
}

// The tensor-core kernel, and whether it takes these sizes, types and
// addresses.
bool grouped_dense_usable(const GroupedProduct &p);
int launch_grouped_dense(const GroupedProduct &p, int device, cudaStream_t st);
// Reads and clears the code that kernel recorded on the current device.
int grouped_dense_take_error(int *code);
// Bytes of workspace of its weight gradient (0 unless the sums are split).
int64_t grouped_dense_workspace(int64_t rows, int64_t inputs, int64_t outputs, int groups);

}  // namespace gtmoe
