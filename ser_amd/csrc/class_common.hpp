// What the class / vocabulary kernels (kernels_distill.hpp, kernels_embed.hpp, kernels_sample.hpp) share: element
// types, 16-byte vectors at element alignment, wave64 and workgroup reductions.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

namespace serhip {

typedef __bf16 bf16_t;
typedef _Float16 f16_t;

// A 16-byte vector of T that may start at any element: rows of an odd number of classes leave most vectors off
// 16-byte boundaries, and gfx950's global loads and stores take dwords at any byte address, so one form serves both.
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec16 {
    static constexpr int kLen = 16 / sizeof(T);
    T v[kLen];
};

template <typename T>
__device__ __forceinline__ Vec16<T> load16(const T* p) {
    return *reinterpret_cast<const Vec16<T>*>(p);
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const Vec16<T>& x) {
    *reinterpret_cast<Vec16<T>*>(p) = x;
}

__device__ __forceinline__ int64_t load_index(const void* p, int is_i64, int64_t i) {
    return is_i64 ? static_cast<const int64_t*>(p)[i] : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

// element type codes of the C ABI (SERHIP_DTYPE_*)
__device__ __forceinline__ float load_float(const void* p, int dtype, int64_t i) {
    if (dtype == 0) return static_cast<const float*>(p)[i];
    if (dtype == 1) return static_cast<float>(static_cast<const bf16_t*>(p)[i]);
    return static_cast<float>(static_cast<const f16_t*>(p)[i]);
}

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x = fmaxf(x, __shfl_xor(x, o));
    return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}
__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int o = 32; o; o >>= 1) x += __shfl_xor(x, o);
    return x;
}

// 2^x; the hardware instruction (1 ulp), without the denormal-result fix-up of exp2f: weights below 2^-126 of the
// largest are zero
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace serhip
