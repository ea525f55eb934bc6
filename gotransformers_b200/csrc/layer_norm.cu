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

#include "operators.h"

namespace gtmoe {
namespace {

constexpr int kFwdThreads = 256;
constexpr int kBwdThreads = 512;
// Blocks of the backward, each of which leaves one row of partial weight and
// bias gradients: two per SM of a B200.
constexpr int kBwdBlocks = 2 * 148;

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
#pragma unroll
    for (int i = 0; i < N; i++) v[i] = red[team_id * warps][i];
    for (int w = 1; w < warps; w++)
#pragma unroll
        for (int i = 0; i < N; i++) v[i] += red[team_id * warps + w][i];
}

struct NormArgs {
    const void *x, *weight, *bias;
    void *y, *mean, *rstd;
    int64_t rows;
    int width;
    double eps;
    int team;
    // backward
    const void *dy, *dres;
    void *dx;
    void *partial;  // blocks x 2 x width
    int want_params;
};

// A team per row; the row stays in NV vectors per thread.
template <typename T, typename W, typename ACC, int VEC, int NV>
__global__ void __launch_bounds__(kFwdThreads) norm_forward_kernel(const NormArgs a) {
    using X = VecIO<T, ACC, VEC>;
    using P = VecIO<W, ACC, VEC>;
    __shared__ ACC red[2][kFwdThreads / 32][1];
    const int team = a.team, team_id = threadIdx.x / team, tl = threadIdx.x - team_id * team;
    const int teams = kFwdThreads / team, n = a.width;
    const T *x = (const T *)a.x;
    const W *w = (const W *)a.weight, *b = (const W *)a.bias;
    for (int64_t row = (int64_t)blockIdx.x * teams + team_id; row < a.rows; row += (int64_t)gridDim.x * teams) {
        const T *xr = x + row * n;
        typename X::Raw raw[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) raw[i] = X::load(xr + c);
        }
        ACC s[1] = {ACC(0)};
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                ACC v[VEC];
                X::unpack(raw[i], v);
#pragma unroll
                for (int q = 0; q < VEC; q++) s[0] += v[q];
            }
        }
        team_sum<1, ACC>(s, team, team_id, red[0]);
        const ACC mean = s[0] / (ACC)n;
        s[0] = ACC(0);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                ACC v[VEC];
                X::unpack(raw[i], v);
#pragma unroll
                for (int q = 0; q < VEC; q++) s[0] += (v[q] - mean) * (v[q] - mean);
            }
        }
        team_sum<1, ACC>(s, team, team_id, red[1]);
        const ACC rstd = rsqrt_acc<ACC>(s[0] / (ACC)n + (ACC)a.eps);
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                ACC v[VEC], pw[VEC], pb[VEC];
                X::unpack(raw[i], v);
                if (w) P::unpack(P::load(w + c), pw);
                if (b) P::unpack(P::load(b + c), pb);
#pragma unroll
                for (int q = 0; q < VEC; q++) {
                    ACC r = (v[q] - mean) * rstd;
                    if (w) r *= pw[q];
                    if (b) r += pb[q];
                    v[q] = r;
                }
                X::store((T *)a.y + row * n + c, v);
            }
        }
        if (tl == 0) {
            if (a.mean) ((ACC *)a.mean)[row] = mean;
            if (a.rstd) ((ACC *)a.rstd)[row] = rstd;
        }
    }
}

// Rows too wide for registers: a block per row reads it three times (the
// second and third time mostly from L2).
template <typename T, typename W, typename ACC>
__global__ void __launch_bounds__(kFwdThreads) norm_forward_wide_kernel(const NormArgs a) {
    __shared__ ACC red[2][kFwdThreads / 32][1];
    const int n = a.width;
    const W *w = (const W *)a.weight, *b = (const W *)a.bias;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *xr = (const T *)a.x + row * n;
        ACC s[1] = {ACC(0)};
        for (int c = threadIdx.x; c < n; c += kFwdThreads) s[0] += (ACC)xr[c];
        team_sum<1, ACC>(s, kFwdThreads, 0, red[0]);
        const ACC mean = s[0] / (ACC)n;
        s[0] = ACC(0);
        for (int c = threadIdx.x; c < n; c += kFwdThreads) {
            const ACC v = (ACC)xr[c] - mean;
            s[0] += v * v;
        }
        team_sum<1, ACC>(s, kFwdThreads, 0, red[1]);
        const ACC rstd = rsqrt_acc<ACC>(s[0] / (ACC)n + (ACC)a.eps);
        for (int c = threadIdx.x; c < n; c += kFwdThreads) {
            ACC r = ((ACC)xr[c] - mean) * rstd;
            if (w) r *= (ACC)w[c];
            if (b) r += (ACC)b[c];
            ((T *)a.y)[row * n + c] = (T)r;
        }
        if (threadIdx.x == 0) {
            if (a.mean) ((ACC *)a.mean)[row] = mean;
            if (a.rstd) ((ACC *)a.rstd)[row] = rstd;
        }
    }
}

// One team per row, every thread the same columns of each of its rows, so
// that the weight and bias gradients add up in registers; each block leaves
// one partial row of both.
template <typename T, typename W, typename ACC, int VEC, int NV>
__global__ void __launch_bounds__(kBwdThreads) norm_backward_kernel(const NormArgs a) {
    using X = VecIO<T, ACC, VEC>;
    using P = VecIO<W, ACC, VEC>;
    __shared__ ACC red[2][kBwdThreads / 32][2];
    __shared__ ACC total[2][kBwdThreads / 2 * VEC * (VEC == 1 ? NV : 1)];
    const int team = a.team, team_id = threadIdx.x / team, tl = threadIdx.x - team_id * team;
    const int teams = kBwdThreads / team, n = a.width;
    const ACC inv_n = ACC(1) / (ACC)n;
    const T *x = (const T *)a.x, *dy = (const T *)a.dy, *dres = (const T *)a.dres;
    const W *w = (const W *)a.weight;
    ACC aw[NV * VEC], ab[NV * VEC];
#pragma unroll
    for (int i = 0; i < NV * VEC; i++) aw[i] = ab[i] = ACC(0);
    const int64_t step = (int64_t)gridDim.x * teams;
    int64_t row = (int64_t)blockIdx.x * teams + team_id;
    typename X::Raw nx[NV], ng[NV];
    ACC mean = ACC(0), rstd = ACC(0);
    auto fetch = [&](int64_t r) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                nx[i] = X::load(x + r * n + c);
                ng[i] = X::load(dy + r * n + c);
            }
        }
        mean = ((const ACC *)a.mean)[r];
        rstd = ((const ACC *)a.rstd)[r];
    };
    if (row < a.rows) fetch(row);
    for (int it = 0; row < a.rows; row += step, it ^= 1) {
        ACC g[NV * VEC], xh[NV * VEC];
        const ACC rs = rstd;
        ACC s[2] = {ACC(0), ACC(0)};
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                ACC pw[VEC];
                X::unpack(nx[i], xh + i * VEC);
                X::unpack(ng[i], g + i * VEC);
                if (w) P::unpack(P::load(w + c), pw);
#pragma unroll
                for (int q = 0; q < VEC; q++) {
                    const int e = i * VEC + q;
                    xh[e] = (xh[e] - mean) * rs;
                    aw[e] += g[e] * xh[e];
                    ab[e] += g[e];
                    if (w) g[e] *= pw[q];
                    s[0] += g[e];
                    s[1] += g[e] * xh[e];
                }
            }
        }
        if (row + step < a.rows) fetch(row + step);  // in flight while the team's sums are made
        typename X::Raw rr[NV];
        if (dres) {
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const int c = (i * team + tl) * VEC;
                if (c < n) rr[i] = X::load(dres + row * n + c);
            }
        }
        team_sum<2, ACC>(s, team, team_id, red[it]);
        const ACC m1 = s[0] * inv_n, m2 = s[1] * inv_n;
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const int c = (i * team + tl) * VEC;
            if (c < n) {
                ACC v[VEC];
                if (dres) X::unpack(rr[i], v);
#pragma unroll
                for (int q = 0; q < VEC; q++) {
                    const int e = i * VEC + q;
                    const ACC d = rs * (g[e] - m1 - xh[e] * m2);
                    v[q] = dres ? v[q] + d : d;
                }
                X::store((T *)a.dx + row * n + c, v);
            }
        }
    }
    if (!a.want_params) return;
    ACC *out = (ACC *)a.partial + (int64_t)blockIdx.x * 2 * n;
    if (teams == 1) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int q = 0; q < VEC; q++) {
                const int c = (i * team + tl) * VEC + q;
                if (c < n) {
                    out[c] = aw[i * VEC + q];
                    out[n + c] = ab[i * VEC + q];
                }
            }
        return;
    }
    // several teams (so at most half the block each): their sums in team order
    for (int t = 0; t < teams; t++) {
        if (team_id == t) {
#pragma unroll
            for (int i = 0; i < (VEC == 1 ? NV : 1); i++)
#pragma unroll
                for (int q = 0; q < VEC; q++) {
                    const int c = (i * team + tl) * VEC + q;
                    if (c < n) {
                        total[0][c] = t ? total[0][c] + aw[i * VEC + q] : aw[i * VEC + q];
                        total[1][c] = t ? total[1][c] + ab[i * VEC + q] : ab[i * VEC + q];
                    }
                }
        }
        __syncthreads();
    }
    for (int c = threadIdx.x; c < n; c += kBwdThreads) {
        out[c] = total[0][c];
        out[n + c] = total[1][c];
    }
}

// Rows too wide for registers: a block per row, read twice; a thread adds its
// columns' gradients into the block's partial row in memory.
template <typename T, typename W, typename ACC>
__global__ void __launch_bounds__(kBwdThreads) norm_backward_wide_kernel(const NormArgs a) {
    __shared__ ACC red[2][kBwdThreads / 32][2];
    const int n = a.width;
    const ACC inv_n = ACC(1) / (ACC)n;
    const W *w = (const W *)a.weight;
    ACC *out = (ACC *)a.partial + (int64_t)blockIdx.x * 2 * n;
    int it = 0;
    bool first = true;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x, it ^= 1) {
        const T *x = (const T *)a.x + row * n, *dy = (const T *)a.dy + row * n;
        const ACC mean = ((const ACC *)a.mean)[row], rs = ((const ACC *)a.rstd)[row];
        ACC s[2] = {ACC(0), ACC(0)};
        for (int c = threadIdx.x; c < n; c += kBwdThreads) {
            const ACC g = w ? (ACC)dy[c] * (ACC)w[c] : (ACC)dy[c];
            s[0] += g;
            s[1] += g * (((ACC)x[c] - mean) * rs);
        }
        team_sum<2, ACC>(s, kBwdThreads, 0, red[it]);
        const ACC m1 = s[0] * inv_n, m2 = s[1] * inv_n;
        for (int c = threadIdx.x; c < n; c += kBwdThreads) {
            const ACC d = (ACC)dy[c], xh = ((ACC)x[c] - mean) * rs;
            const ACC g = w ? d * (ACC)w[c] : d;
            ACC v = rs * (g - m1 - xh * m2);
            if (a.dres) v = (ACC)((const T *)a.dres)[row * n + c] + v;
            ((T *)a.dx)[row * n + c] = (T)v;
            if (a.want_params) {
                out[c] = (first ? ACC(0) : out[c]) + d * xh;
                out[n + c] = (first ? ACC(0) : out[n + c]) + d;
            }
        }
        first = false;
    }
}

// The blocks' partial rows to the weight and bias gradients: 32 columns per
// block, 16 runs of partial rows side by side, added in a fixed order.
template <typename W, typename ACC>
__global__ void __launch_bounds__(512) norm_params_kernel(const ACC *__restrict__ partial, int blocks, int n,
                                                          void *dweight, void *dbias, int accumulate) {
    __shared__ ACC sum[2][16][32];
    const int c = blockIdx.x * 32 + threadIdx.x, run = threadIdx.y;
    ACC s0 = ACC(0), s1 = ACC(0);
    if (c < n)
        for (int p = run; p < blocks; p += 16) {
            s0 += partial[(int64_t)p * 2 * n + c];
            s1 += partial[(int64_t)p * 2 * n + n + c];
        }
    sum[0][run][threadIdx.x] = s0;
    sum[1][run][threadIdx.x] = s1;
    __syncthreads();
    if (run >= 2 || c >= n) return;
    W *dst = (W *)(run == 0 ? dweight : dbias);
    if (!dst) return;
    ACC s = sum[run][0][threadIdx.x];
    for (int r = 1; r < 16; r++) s += sum[run][r][threadIdx.x];
    if (accumulate) s += (ACC)dst[c];
    dst[c] = (W)s;
}

// Threads per row: the fewest (a power of two from 32 on) that hold the row
// in nv vectors each.
int team_for(int64_t vectors, int nv, int most) {
    int team = 32;
    while (team < most && (int64_t)team * nv < vectors) team *= 2;
    return team;
}

template <typename T, typename W, typename ACC, int VEC>
int forward_vec(NormArgs a, cudaStream_t st) {
    const int64_t vectors = ((int64_t)a.width + VEC - 1) / VEC;
    // a row in one warp as far as 8 vectors per lane go (no barrier), in a
    // larger team beyond
    const int nv = vectors <= 64 ? 2 : 8;
    if (vectors > (int64_t)kFwdThreads * 8) {
        norm_forward_wide_kernel<T, W, ACC>
            <<<(unsigned)(a.rows < 65535 ? a.rows : 65535), kFwdThreads, 0, st>>>(a);
    } else {
        a.team = team_for(vectors, nv, kFwdThreads);
        const int64_t teams = kFwdThreads / a.team;
        const int64_t want = (a.rows + teams - 1) / teams;
        const unsigned grid = (unsigned)(want < 0x7fffffff ? want : 0x7fffffff);
        if (nv == 2) norm_forward_kernel<T, W, ACC, VEC, 2><<<grid, kFwdThreads, 0, st>>>(a);
        else norm_forward_kernel<T, W, ACC, VEC, 8><<<grid, kFwdThreads, 0, st>>>(a);
    }
    GT_CUDA(cudaGetLastError());
    note_launches(1);
    return 0;
}

template <typename T, typename W, typename ACC, int VEC>
int backward_vec(NormArgs a, void *dweight, void *dbias, int accumulate, cudaStream_t st) {
    const int64_t vectors = ((int64_t)a.width + VEC - 1) / VEC;
    int64_t blocks;
    if (a.rows == 0) {
        blocks = 0;
    } else if (vectors > (int64_t)kBwdThreads * (VEC == 1 ? 8 : 4)) {
        blocks = a.rows < kBwdBlocks ? a.rows : kBwdBlocks;
        norm_backward_wide_kernel<T, W, ACC><<<(unsigned)blocks, kBwdThreads, 0, st>>>(a);
    } else {
        const int most = VEC == 1 ? 2 : 1;  // vectors per thread below a whole block per row
        a.team = team_for(vectors, most, kBwdThreads);
        const int64_t teams = kBwdThreads / a.team, want = (a.rows + teams - 1) / teams;
        blocks = want < kBwdBlocks ? want : kBwdBlocks;
        const int64_t nv = (vectors + a.team - 1) / a.team;
        const unsigned grid = (unsigned)blocks;
        if constexpr (VEC == 1) {
            if (nv <= 2) norm_backward_kernel<T, W, ACC, 1, 2><<<grid, kBwdThreads, 0, st>>>(a);
            else norm_backward_kernel<T, W, ACC, 1, 8><<<grid, kBwdThreads, 0, st>>>(a);
        } else {
            if (nv <= 1) norm_backward_kernel<T, W, ACC, VEC, 1><<<grid, kBwdThreads, 0, st>>>(a);
            else if (nv <= 2) norm_backward_kernel<T, W, ACC, VEC, 2><<<grid, kBwdThreads, 0, st>>>(a);
            else norm_backward_kernel<T, W, ACC, VEC, 4><<<grid, kBwdThreads, 0, st>>>(a);
        }
    }
    if (blocks) {
        GT_CUDA(cudaGetLastError());
        note_launches(1);
    }
    if (!a.want_params) return 0;
    norm_params_kernel<W, ACC><<<(unsigned)((a.width + 31) / 32), dim3(32, 16), 0, st>>>(
        (const ACC *)a.partial, (int)blocks, a.width, dweight, dbias, accumulate);
    GT_CUDA(cudaGetLastError());
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
        ranges_overlap(rstd, sbytes, x, bytes) || ranges_overlap(mean, sbytes, rstd, sbytes))
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
        return wide ? forward_vec<double, double, double, 2>(a, st) : forward_vec<double, double, double, 1>(a, st);
    if (dtype == GTMOE_DTYPE_F32)
        return wide ? forward_vec<float, float, float, 4>(a, st) : forward_vec<float, float, float, 1>(a, st);
    if (weight_dtype == GTMOE_DTYPE_F32)
        return wide ? forward_vec<__nv_bfloat16, float, float, 8>(a, st)
                    : forward_vec<__nv_bfloat16, float, float, 1>(a, st);
    return wide ? forward_vec<__nv_bfloat16, __nv_bfloat16, float, 8>(a, st)
                : forward_vec<__nv_bfloat16, __nv_bfloat16, float, 1>(a, st);
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
        return wide ? backward_vec<double, double, double, 2>(a, dweight, dbias, accumulate, st)
                    : backward_vec<double, double, double, 1>(a, dweight, dbias, accumulate, st);
    if (dtype == GTMOE_DTYPE_F32)
        return wide ? backward_vec<float, float, float, 4>(a, dweight, dbias, accumulate, st)
                    : backward_vec<float, float, float, 1>(a, dweight, dbias, accumulate, st);
    if (weight_dtype == GTMOE_DTYPE_F32)
        return wide ? backward_vec<__nv_bfloat16, float, float, 8>(a, dweight, dbias, accumulate, st)
                    : backward_vec<__nv_bfloat16, float, float, 1>(a, dweight, dbias, accumulate, st);
    return wide ? backward_vec<__nv_bfloat16, __nv_bfloat16, float, 8>(a, dweight, dbias, accumulate, st)
                : backward_vec<__nv_bfloat16, __nv_bfloat16, float, 1>(a, dweight, dbias, accumulate, st);
}

}  // extern "C"
