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
// the same at element `at` (below 2^30) of a row whose address is uniform: a 32-bit offset to scalar registers
template <typename T>
__device__ __forceinline__ Vec16<T> load16_at(const T* p, int at) {
    return *reinterpret_cast<const Vec16<T>*>(reinterpret_cast<const char*>(p) + static_cast<uint32_t>(at) * static_cast<uint32_t>(sizeof(T)));
}
template <typename T>
__device__ __forceinline__ void store16_at(T* p, int at, const Vec16<T>& x) {
    *reinterpret_cast<Vec16<T>*>(reinterpret_cast<char*>(p) + static_cast<uint32_t>(at) * static_cast<uint32_t>(sizeof(T))) = x;
}
template <typename T>
__device__ __forceinline__ void store16(T* p, const Vec16<T>& x) {
    *reinterpret_cast<Vec16<T>*>(p) = x;
}

// The four registers of a 16-byte vector, for rows that stay in registers, and its elements as f32.
typedef uint32_t Quad __attribute__((ext_vector_type(4)));
template <typename T>
__device__ __forceinline__ float quad_element(const Quad& q, int e);
template <>
__device__ __forceinline__ float quad_element<float>(const Quad& q, int e) {
    return __uint_as_float(q[e]);
}
template <>
__device__ __forceinline__ float quad_element<bf16_t>(const Quad& q, int e) {
    return __uint_as_float(e & 1 ? q[e >> 1] & 0xffff0000u : q[e >> 1] << 16);
}
template <>
__device__ __forceinline__ float quad_element<f16_t>(const Quad& q, int e) {
    return static_cast<float>(__builtin_bit_cast(f16_t, static_cast<uint16_t>(e & 1 ? q[e >> 1] >> 16 : q[e >> 1])));
}
template <typename T>
__device__ __forceinline__ constexpr uint32_t minus_infinity_bits() {   // in every element of a register
    return sizeof(T) == 4 ? 0xff800000u : static_cast<T>(1.0f + 0x1p-9f) == static_cast<T>(1.0f) ? 0xff80ff80u : 0xfc00fc00u;
}
// Makes the compiler take the registers for new: what it has unpacked of 16-bit elements it would otherwise keep, at twice
// the registers, from one pass over them to the next.
__device__ __forceinline__ void forget(Quad& q) { asm volatile("" : "+v"(q)); }

// Makes the compiler work out again what it derives from `x` (addresses of every vector, otherwise kept through a kernel).
__device__ __forceinline__ int fresh(int x) {
    asm volatile("" : "+v"(x));
    return x;
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

// Scans and reductions of a whole wave (all 64 lanes active) by data-parallel-primitive moves: within rows of 16 lanes,
// then the last lane of a row into the next rows.  A move is part of an ALU instruction, where a shuffle is a round trip
// through the LDS unit (six steps of it some 600 cycles).  Lanes that receive nothing take `none`, the operation's
// neutral element.
template <int kCtrl, int kRows, typename V>
__device__ __forceinline__ V dpp_move(V none, V x) {
    static_assert(sizeof(V) == 4 || sizeof(V) == 8, "one or two registers");
    V y;
    int n[sizeof(V) / 4], a[sizeof(V) / 4];
    __builtin_memcpy(n, &none, sizeof(V));
    __builtin_memcpy(a, &x, sizeof(V));
#pragma unroll
    for (unsigned i = 0; i < sizeof(V) / 4; ++i) a[i] = __builtin_amdgcn_update_dpp(n[i], a[i], kCtrl, kRows, 0xf, false);
    __builtin_memcpy(&y, a, sizeof(V));
    return y;
}
template <typename V, typename Op>
__device__ __forceinline__ V wave_scan(V x, V none, Op op) {   // inclusive
    x = op(x, dpp_move<0x111, 0xf>(none, x));   // row_shr 1
    x = op(x, dpp_move<0x112, 0xf>(none, x));
    x = op(x, dpp_move<0x114, 0xf>(none, x));
    x = op(x, dpp_move<0x118, 0xf>(none, x));
    x = op(x, dpp_move<0x142, 0xa>(none, x));   // row_bcast 15 into rows 1 and 3
    return op(x, dpp_move<0x143, 0xc>(none, x));   // row_bcast 31 into rows 2 and 3
}
// for use where all lanes are active: in a branch that lane 63 does not take, its `x` may not have been worked out
template <typename V>
__device__ __forceinline__ V last_lane(V x) {
    V y;
    int a[sizeof(V) / 4];
    __builtin_memcpy(a, &x, sizeof(V));
#pragma unroll
    for (unsigned i = 0; i < sizeof(V) / 4; ++i) a[i] = __builtin_amdgcn_readlane(a[i], 63);
    __builtin_memcpy(&y, a, sizeof(V));
    return y;
}
template <typename V>
__device__ __forceinline__ V wave_scan_sum(V x) {
    return wave_scan(x, V(0), [](V a, V b) { return a + b; });
}
template <typename V>
__device__ __forceinline__ V wave_sum(V x) {
    return last_lane(wave_scan_sum(x));
}
// of the first 16 lanes, to all: for one value of each of a workgroup's 16 waves (all lanes active, as above)
template <typename Op>
__device__ __forceinline__ float row_total(float x, float none, Op op) {
    x = op(x, dpp_move<0x111, 0xf>(none, x));
    x = op(x, dpp_move<0x112, 0xf>(none, x));
    x = op(x, dpp_move<0x114, 0xf>(none, x));
    x = op(x, dpp_move<0x118, 0xf>(none, x));
    return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), 15));
}
__device__ __forceinline__ float wave_max(float x) {
    return last_lane(wave_scan(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); }));
}

// 2^x; the hardware instruction (1 ulp), without the denormal-result fix-up of exp2f: weights below 2^-126 of the
// largest are zero
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

}  // namespace serhip
