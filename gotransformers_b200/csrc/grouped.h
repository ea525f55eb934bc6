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
};

constexpr int kMaxGroups = kMaxRoutedExperts;

// Group g's rows are start[g] .. start[g + 1], cut at `rows`; a negative
// count is no rows.  Every thread of the block calls it; `start` is groups + 1
// words of shared memory and `scratch` one word per thread.  True when the
// counts were as they should be.
__device__ __forceinline__ bool group_starts(const int64_t *__restrict__ counts, int groups, int64_t rows, int *start,
                                             int *scratch) {
    const int threads = blockDim.x, t = threadIdx.x;
    const int per = (groups + threads - 1) / threads;
    const int g0 = t * per, g1 = min(groups, g0 + per);
    int64_t sum = 0;
    bool ok = true;
    for (int g = g0; g < g1; g++) {
        int64_t c = counts[g];
        if (c < 0 || c > rows) {
            ok = false;
            c = c < 0 ? 0 : rows;
        }
        sum += c;
        if (sum > rows) {
            ok = false;
            sum = rows;
        }
        start[g + 1] = (int)c;
    }
    scratch[t] = (int)sum;
    __syncthreads();
    // inclusive scan over the threads, saturating at `rows` (< 2^31)
    for (int o = 1; o < threads; o <<= 1) {
        const int64_t add = t >= o ? (int64_t)scratch[t - o] : 0;
        __syncthreads();
        const int64_t v = (int64_t)scratch[t] + add;
        if (v > rows) ok = false;
        scratch[t] = (int)(v > rows ? rows : v);
        __syncthreads();
    }
    int64_t at = t ? scratch[t - 1] : 0;
    for (int g = g0; g < g1; g++) {
        at += start[g + 1];
        if (at > rows) at = rows;
        start[g + 1] = (int)at;
    }
    if (t == 0) start[0] = 0;
    return __syncthreads_and(ok);
}

// The tensor-core kernel, and whether it takes these sizes, types and
// addresses.
bool grouped_dense_usable(const GroupedProduct &p);
int launch_grouped_dense(const GroupedProduct &p, int *err, cudaStream_t st);

}  // namespace gtmoe
