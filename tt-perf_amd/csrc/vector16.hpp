// vector16.hpp — the operators' 16-byte accesses to bf16 and fp32 rows, and their exponential.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device.hpp"

namespace ttp {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// 2^x by the hardware's instruction: one unit in the last place, results below 2^-126 flushed
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// 16 bytes at any address their element type is aligned to: rows of an odd length start anywhere,
// and gfx950 takes unaligned vector accesses.
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <class T>
constexpr int kPer = 16 / (int)sizeof(T);  // elements per 16 bytes

__device__ __forceinline__ void unpack(u32x4 w, float (&v)[8], const uint16_t*) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        v[2 * k] = bf16_lo(w[k]);
        v[2 * k + 1] = bf16_hi(w[k]);
    }
}
__device__ __forceinline__ void unpack(u32x4 w, float (&v)[4], const float*) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]);
}
__device__ __forceinline__ u32x4 pack(const float (&v)[8], const uint16_t*) {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const f32x2 two = {v[2 * k], v[2 * k + 1]};
        w[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
    }
    return w;
}
__device__ __forceinline__ u32x4 pack(const float (&v)[4], const float*) {
    u32x4 w;
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = __float_as_uint(v[k]);
    return w;
}
__device__ __forceinline__ float widen(uint16_t x) { return bf16_lo(x); }
__device__ __forceinline__ float widen(float x) { return x; }
__device__ __forceinline__ void narrow(float x, uint16_t* p) { *p = (uint16_t)bf16_rne(x); }
__device__ __forceinline__ void narrow(float x, float* p) { *p = x; }

template <class T>
__device__ __forceinline__ u32x4 load16(const T* p) {
    return *reinterpret_cast<const u32x4_any*>(p);
}
template <class T>
__device__ __forceinline__ void store16(T* p, u32x4 w) {
    *reinterpret_cast<u32x4_any*>(p) = w;
}
// the same for what is read once, or not read again soon
template <class T>
__device__ __forceinline__ u32x4 load16_once(const T* p) {
    return __builtin_nontemporal_load(reinterpret_cast<const u32x4_any*>(p));
}
template <class T>
__device__ __forceinline__ void store16_once(T* p, u32x4 w) {
    __builtin_nontemporal_store(static_cast<u32x4_any>(w), reinterpret_cast<u32x4_any*>(p));
}

}  // namespace
}  // namespace ttp
