// dropout.cu -- dropout from a counter-based generator, with the block's
// residual, and its backward pass.
//
//   out_i = residual_i + (keep_i ? x_i / (1 - rate) : 0)
//   dx_i  = keep_i ? dout_i / (1 - rate) : 0
//
// keep_i is a function of (seed, stream, i) alone and is never stored: word j
// of the stream is SplitMix64(key + j), the generator and the key of the
// library's synthetic inputs (quantize.cu, synthetic.py), element i owns half
// i % 2 of word i / 2 (the low half first), and is kept when that half is at
// least rate * 2^32.  The product and the sum are float32 (float64 for float64
// rows) and rounded once.
//
// A word costs about 20 instructions for two elements, which bounds the
// backward pass: 65536 x 4096 bf16 in 194 us, 5.5 TB/s (86 % of the copy
// bandwidth); the forward with a residual moves 6 bytes per element instead of
// 4 and reaches 226 us, 7.1 TB/s.  Four vectors of 16 bytes per thread are
// loaded before the first word is made; four blocks per SM (64 registers) hide
// them better than three of 76 or six of 40 (205 and 227 us).  Multiplications
// in place of the shifts of 64-bit words were slower (229 us).
#include <math.h>

#include "operators.h"

namespace gtmoe {
namespace {

constexpr int kThreads = 256;
constexpr int kUnroll = 4;  // vectors in flight per thread and input

__host__ __device__ __forceinline__ uint64_t split_mix64(uint64_t z) {
    z += 0x9E3779B97F4A7C15ull;
    z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
    z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
    return z ^ (z >> 31);
}

// r + x * scale where bits >= threshold, else r: a predicated multiply-add, no
// selection.
__device__ __forceinline__ float keep_add(uint32_t bits, uint32_t threshold, float x, float scale, float r) {
    asm("{\n\t.reg .pred p;\n\t"
        "setp.ge.u32 p, %1, %2;\n\t"
        "@p fma.rn.f32 %0, %3, %4, %0;\n\t}\n"
        : "+f"(r)
        : "r"(bits), "r"(threshold), "f"(x), "f"(scale));
    return r;
}
__device__ __forceinline__ double keep_add(uint32_t bits, uint32_t threshold, double x, double scale, double r) {
    return bits >= threshold ? fma(x, scale, r) : r;
}

struct DropoutArgs {
    const void *x, *residual;
    void *out;
    int64_t n;
    uint64_t key;     // of word 0
    uint64_t offset;  // the generator's element of x[0]
    uint32_t threshold;
    double scale;
};

// ODD: x[0] owns the high half of its word, so a vector's elements lie in
// VEC / 2 + 1 words.
template <typename T, typename ACC, int VEC, bool ODD>
__global__ void __launch_bounds__(kThreads, 4) dropout_kernel(const DropoutArgs a) {
    using X = VecIO<T, ACC, VEC>;
    const T *x = (const T *)a.x, *res = (const T *)a.residual;
    T *out = (T *)a.out;
    const ACC scale = (ACC)a.scale;
    const int64_t vectors = a.n / VEC;
    for (int64_t v0 = (int64_t)blockIdx.x * (kThreads * kUnroll) + threadIdx.x; v0 < vectors;
         v0 += (int64_t)gridDim.x * (kThreads * kUnroll)) {
        typename X::Raw rx[kUnroll], rr[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int64_t v = v0 + u * kThreads;
            if (v < vectors) {
                rx[u] = X::load(x + v * VEC);
                if (res) rr[u] = X::load(res + v * VEC);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnroll; u++) {
            const int64_t v = v0 + u * kThreads;
            if (v >= vectors) break;
            const uint64_t first = a.offset + (uint64_t)v * VEC;
            uint32_t half[VEC + 2];
            if constexpr (VEC == 1) {
                const uint64_t w = split_mix64(a.key + (first >> 1));
                half[0] = (first & 1) ? (uint32_t)(w >> 32) : (uint32_t)w;
            } else {
#pragma unroll
                for (int q = 0; q < VEC / 2 + (ODD ? 1 : 0); q++) {
                    const uint64_t w = split_mix64(a.key + (first >> 1) + q);
                    half[2 * q] = (uint32_t)w;
                    half[2 * q + 1] = (uint32_t)(w >> 32);
                }
            }
            ACC vx[VEC], vr[VEC];
            X::unpack(rx[u], vx);
            if (res) X::unpack(rr[u], vr);
#pragma unroll
            for (int q = 0; q < VEC; q++)
                vx[q] = keep_add(half[q + (ODD ? 1 : 0)], a.threshold, vx[q], scale, res ? vr[q] : ACC(0));
            X::store(out + v * VEC, vx);
        }
    }
}

template <typename T, typename ACC, int VEC>
int launch_vec(const DropoutArgs &a, cudaStream_t st) {
    const int64_t per = (int64_t)VEC * kThreads * kUnroll;
    const int64_t blocks = (a.n + per - 1) / per;
    const unsigned grid = (unsigned)(blocks < 0x7fffffff ? blocks : 0x7fffffff);
    if (VEC > 1 && (a.offset & 1)) dropout_kernel<T, ACC, VEC, true><<<grid, kThreads, 0, st>>>(a);
    else dropout_kernel<T, ACC, VEC, false><<<grid, kThreads, 0, st>>>(a);
    GT_CUDA(cudaGetLastError());
    note_launches(1);
    return 0;
}

template <typename T, typename ACC, int VEC>
int launch(DropoutArgs a, cudaStream_t st) {
    if (!aligned16(a.x) || !aligned16(a.residual) || !aligned16(a.out)) return launch_vec<T, ACC, 1>(a, st);
    const int64_t head = a.n / VEC * VEC, tail = a.n - head;
    DropoutArgs b = a;
    b.n = head;
    if (head) GT_CHECK((launch_vec<T, ACC, VEC>(b, st)));
    if (!tail) return 0;
    // the last elements of a count that is not a whole number of vectors
    b.n = tail;
    b.x = (const T *)a.x + head;
    if (a.residual) b.residual = (const T *)a.residual + head;
    b.out = (T *)a.out + head;
    b.offset = a.offset + (uint64_t)head;
    return launch_vec<T, ACC, 1>(b, st);
}

}  // namespace

int check_dropout_rate(double rate) {
    if (!(rate >= 0 && rate < 1)) return fail(GTMOE_EINVAL, "dropout: the rate must be at least 0 and below 1, got %g", rate);
    return 0;
}

int launch_dropout(const void *x, const void *residual, int dtype, int64_t n, double rate, uint64_t seed,
                   uint64_t stream_id, int64_t offset, void *out, cudaStream_t st) {
    if (n == 0) return 0;
    DropoutArgs a;
    a.x = x, a.residual = residual, a.out = out, a.n = n;
    a.key = split_mix64(seed ^ (stream_id * 0xD1B54A32D192ED03ull));
    a.offset = (uint64_t)offset;
    a.threshold = (uint32_t)floor(rate * 4294967296.0);
    a.scale = 1.0 / (1.0 - rate);
    if (dtype == GTMOE_DTYPE_F64) return launch<double, double, 2>(a, st);
    if (dtype == GTMOE_DTYPE_F32) return launch<float, float, 4>(a, st);
    return launch<__nv_bfloat16, float, 8>(a, st);
}

}  // namespace gtmoe

using namespace gtmoe;

static int dropout_call(const void *x, const void *residual, int dtype, int64_t n, double rate, uint64_t seed,
                        uint64_t stream_id, int64_t offset, void *out, void *stream, const char *in_name,
                        const char *out_name) {
    if (!known_dtype(dtype)) return fail(GTMOE_EINVAL, "dropout: unknown dtype");
    if (n < 0 || n > (INT64_MAX >> 4)) return fail(GTMOE_EINVAL, "dropout: bad number of values %lld", (long long)n);
    if (offset < 0 || offset > INT64_MAX - n) return fail(GTMOE_EINVAL, "dropout: bad offset %lld", (long long)offset);
    GT_CHECK(check_dropout_rate(rate));
    if (n == 0) return 0;
    if (!x || !out) return fail(GTMOE_EINVAL, "dropout: %s and %s must be given", in_name, out_name);
    const int64_t bytes = n * (int64_t)dtype_size(dtype);
    if (overlaps_shifted(x, bytes, out, bytes) || overlaps_shifted(residual, bytes, out, bytes))
        return fail(GTMOE_EINVAL, "dropout: %s overlaps an input (it may be one itself)", out_name);
    DeviceScope scope;
    const size_t es = dtype_size(dtype);
    GT_CHECK(scope.enter({{x, in_name, es}, {residual, "residual", es}, {out, out_name, es}}));
    return launch_dropout(x, residual, dtype, n, rate, seed, stream_id, offset, out, (cudaStream_t)stream);
}

extern "C" {

int gtmoe_dropout(const void *x, const void *residual, int dtype, int64_t n, double rate, uint64_t seed,
                  uint64_t stream_id, int64_t offset, void *out, void *stream) {
    return dropout_call(x, residual, dtype, n, rate, seed, stream_id, offset, out, stream, "x", "out");
}

int gtmoe_dropout_backward(const void *dout, int dtype, int64_t n, double rate, uint64_t seed, uint64_t stream_id,
                           int64_t offset, void *dx, void *stream) {
    return dropout_call(dout, nullptr, dtype, n, rate, seed, stream_id, offset, dx, stream, "dout", "dx");
}

}  // extern "C"
