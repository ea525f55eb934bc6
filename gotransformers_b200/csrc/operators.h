// operators.h -- what the handle-less operators (layer_norm.cu, dropout.cu,
// grouped_product.cu, grouped_dense.cu) share: argument checks, the device a
// call runs on, and 16-byte vectors of the activation types.
#pragma once

#include <initializer_list>

#include "common.cuh"
#include "internal.h"

namespace gtmoe {

// A pointer argument of an operator, the name its errors use and the size of
// its elements, on which it has to start; NULL ones are skipped.
struct DevArg {
    const void *p;
    const char *name;
    size_t align = 1;
};

// The device that holds an operator's arguments, current for the call; the
// thread's own device is current again afterwards.
class DeviceScope {
   public:
    DeviceScope() = default;
    DeviceScope(const DeviceScope &) = delete;
    DeviceScope &operator=(const DeviceScope &) = delete;
    ~DeviceScope() {
        if (previous_ >= 0) cudaSetDevice(previous_);
    }
    // GTMOE_EINVAL unless every argument is aligned memory of one device,
    // GTMOE_ENODEVICE unless that device is an sm_100
    int enter(std::initializer_list<DevArg> args);
    int device() const { return device_; }

   private:
    int previous_ = -1, device_ = -1;
};

// Whether byte ranges [a, a + na) and [b, b + nb) share a byte.
inline bool ranges_overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && na > 0 && nb > 0 && x < y + (uintptr_t)nb && y < x + (uintptr_t)na;
}
// An output may be an input (each element is read before the thread that read
// it writes it) but not overlap it in another way.
inline bool overlaps_shifted(const void *a, int64_t na, const void *b, int64_t nb) {
    return a != b && ranges_overlap(a, na, b, nb);
}
inline bool aligned16(const void *p) { return ((uintptr_t)p & 15) == 0; }
inline bool known_dtype(int t) { return t >= GTMOE_DTYPE_F64 && t <= GTMOE_DTYPE_BF16; }
// rows x width elements of 8 bytes have to be countable in 63 bits
inline bool countable(int64_t rows, int64_t width) { return width <= 0 || rows <= (INT64_MAX >> 4) / width; }

// Bounded waits that ran out, and refused counts, leave a code in a word of the
// device per source file; gtmoe_operators_check reads them.
constexpr int kErrBadCounts = 101;
// Each reads its words on the current device and clears them; the first waits
// for the device.
int grouped_take_error(int *code);
int norm_take_error(int *code);

// dropout.cu, for the block step (block.cu): device pointers, no checks.
int check_dropout_rate(double rate);
int launch_dropout(const void *x, const void *residual, int dtype, int64_t n, double rate, uint64_t seed,
                   uint64_t stream_id, int64_t offset, void *out, cudaStream_t st);

// Two accumulators side by side: sm_100 multiplies and adds pairs of float32 in
// one instruction.
template <typename ACC>
struct Pair {
    ACC x, y;
};
__device__ __forceinline__ Pair<float> add2(Pair<float> a, Pair<float> b) {
    const float2 r = __fadd2_rn(make_float2(a.x, a.y), make_float2(b.x, b.y));
    return {r.x, r.y};
}
__device__ __forceinline__ Pair<float> mul2(Pair<float> a, Pair<float> b) {
    const float2 r = __fmul2_rn(make_float2(a.x, a.y), make_float2(b.x, b.y));
    return {r.x, r.y};
}
__device__ __forceinline__ Pair<float> fma2(Pair<float> a, Pair<float> b, Pair<float> c) {
    const float2 r = __ffma2_rn(make_float2(a.x, a.y), make_float2(b.x, b.y), make_float2(c.x, c.y));
    return {r.x, r.y};
}
__device__ __forceinline__ Pair<double> add2(Pair<double> a, Pair<double> b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ Pair<double> mul2(Pair<double> a, Pair<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Pair<double> fma2(Pair<double> a, Pair<double> b, Pair<double> c) {
    return {fma(a.x, b.x, c.x), fma(a.y, b.y, c.y)};
}
template <typename ACC>
__device__ __forceinline__ Pair<ACC> both(ACC v) {
    return {v, v};
}

// Read-only data: the compiler may move these loads across stores.
__device__ __forceinline__ uint4 load_const(const uint4 *p) { return __ldg(p); }
__device__ __forceinline__ float4 load_const(const float4 *p) { return __ldg(p); }
__device__ __forceinline__ double2 load_const(const double2 *p) { return __ldg(p); }

// VEC consecutive values of T as ACC: one 16-byte access, or a plain one for VEC = 1.
template <typename T, typename ACC, int VEC>
struct VecIO;
template <typename ACC>
struct VecIO<__nv_bfloat16, ACC, 8> {
    using Raw = uint4;
    static __device__ __forceinline__ Raw load(const __nv_bfloat16 *p) { return *reinterpret_cast<const uint4 *>(p); }
    static __device__ __forceinline__ Raw load_ro(const __nv_bfloat16 *p) {
        return load_const(reinterpret_cast<const uint4 *>(p));
    }
    static __device__ __forceinline__ void unpack(const Raw &r, ACC *v) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ void store(__nv_bfloat16 *p, const ACC *v) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <>
struct VecIO<float, float, 4> {
    using Raw = float4;
    static __device__ __forceinline__ Raw load(const float *p) { return *reinterpret_cast<const float4 *>(p); }
    static __device__ __forceinline__ Raw load_ro(const float *p) {
        return load_const(reinterpret_cast<const float4 *>(p));
    }
    static __device__ __forceinline__ void unpack(const Raw &r, float *v) {
        v[0] = r.x, v[1] = r.y, v[2] = r.z, v[3] = r.w;
    }
    static __device__ __forceinline__ void store(float *p, const float *v) {
        *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
    }
};
// float32 parameters beside 8 bf16 activations: two 16-byte accesses
template <>
struct VecIO<float, float, 8> {
    struct Raw {
        float4 a, b;
    };
    static __device__ __forceinline__ Raw load(const float *p) {
        return {reinterpret_cast<const float4 *>(p)[0], reinterpret_cast<const float4 *>(p)[1]};
    }
    static __device__ __forceinline__ Raw load_ro(const float *p) {
        return {load_const(reinterpret_cast<const float4 *>(p)), load_const(reinterpret_cast<const float4 *>(p) + 1)};
    }
    static __device__ __forceinline__ void unpack(const Raw &r, float *v) {
        v[0] = r.a.x, v[1] = r.a.y, v[2] = r.a.z, v[3] = r.a.w;
        v[4] = r.b.x, v[5] = r.b.y, v[6] = r.b.z, v[7] = r.b.w;
    }
};
template <>
struct VecIO<double, double, 2> {
    using Raw = double2;
    static __device__ __forceinline__ Raw load(const double *p) { return *reinterpret_cast<const double2 *>(p); }
    static __device__ __forceinline__ Raw load_ro(const double *p) {
        return load_const(reinterpret_cast<const double2 *>(p));
    }
    static __device__ __forceinline__ void unpack(const Raw &r, double *v) { v[0] = r.x, v[1] = r.y; }
    static __device__ __forceinline__ void store(double *p, const double *v) {
        *reinterpret_cast<double2 *>(p) = make_double2(v[0], v[1]);
    }
};
template <typename T, typename ACC>
struct VecIO<T, ACC, 1> {
    using Raw = T;
    static __device__ __forceinline__ Raw load(const T *p) { return *p; }
    static __device__ __forceinline__ void unpack(const Raw &r, ACC *v) { v[0] = (ACC)r; }
    static __device__ __forceinline__ void store(T *p, const ACC *v) { *p = (T)v[0]; }
};

}  // namespace gtmoe
