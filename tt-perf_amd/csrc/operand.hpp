// operand.hpp — what the matrix products share: the order of blocks on the XCDs, chunks of 8 elements
// on their way from memory to the LDS, and the matrix instructions' operands back from it.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vector16.hpp"

namespace ttp {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// Blocks go to the 8 XCDs in turn: neighbours in this order are on one XCD, and share its L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t n) {
    const uint32_t x = b % 8, q = n / 8, r = n % 8;
    return x * q + min(x, r) + b / 8;
}

// x as the sum of three bf16 (pairs packed): each takes the leading 8 bits of what is left.  (Cut
// off, not rounded: the largest numbers would round to infinity.)  Exact but for bits below bf16's
// least number, 2^-133, which an x below 2^-110 can have.  What is left of an infinity is taken
// from the largest number: inf - inf would make it NaN, and a part of its sign, finite, changes
// nothing beside it.  (A clamp, one operation, 1% of a gradient's time; a comparison and a choice
// took 4%.  A NaN stays one by its first part; a signalling one without a bit there, which no
// arithmetic makes, counts as an infinity.)
__device__ __forceinline__ void split3(float a, float b, uint32_t (&p)[3]) {
    constexpr float kMost = 3.4028234663852886e38f;
    p[0] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    a = __builtin_amdgcn_fmed3f(a, -kMost, kMost);
    b = __builtin_amdgcn_fmed3f(b, -kMost, kMost);
    a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
    b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
#pragma unroll
    for (int k = 1; k < 3; ++k) {
        p[k] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
        a -= bf16_lo(p[k]);
        b -= bf16_hi(p[k]);
    }
}

// 8 columns of a row
template <class G>
struct Chunk8;
template <>
struct Chunk8<uint16_t> {
    u32x4 w;
    __device__ __forceinline__ void load(const uint16_t* p) { w = load16(p); }
    __device__ __forceinline__ void clear() { w = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void keep(int n) {  // the first n, then 0
#pragma unroll
        for (int k = 0; k < 4; ++k)
            w[k] = 2 * k + 1 < n ? w[k] : 2 * k < n ? w[k] & 0xFFFFu : 0u;
    }
    __device__ __forceinline__ void load_some(const uint16_t* p, int n) {  // the first n, then 0
        w = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (k < n) w[k / 2] |= (uint32_t)p[k] << (16 * (k % 2));
    }
    __device__ __forceinline__ float value(int k) const {
        return k % 2 ? bf16_hi(w[k / 2]) : bf16_lo(w[k / 2]);
    }
    __device__ __forceinline__ void planes(u32x4 (&p)[1]) const { p[0] = w; }
};
template <>
struct Chunk8<float> {
    u32x4 w[2];
    __device__ __forceinline__ void load(const float* p) {
        w[0] = load16(p);
        w[1] = load16(p + 4);
    }
    __device__ __forceinline__ void clear() { w[0] = w[1] = u32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void keep(int n) {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k / 4][k % 4] = k < n ? w[k / 4][k % 4] : 0u;
    }
    __device__ __forceinline__ void load_some(const float* p, int n) {
#pragma unroll
        for (int k = 0; k < 8; ++k) w[k / 4][k % 4] = k < n ? __float_as_uint(p[k]) : 0u;
    }
    __device__ __forceinline__ float value(int k) const { return __uint_as_float(w[k / 4][k % 4]); }
    __device__ __forceinline__ void planes(u32x4 (&p)[3]) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t three[3];
            split3(value(2 * k), value(2 * k + 1), three);
#pragma unroll
            for (int j = 0; j < 3; ++j) p[j][k] = three[j];
        }
    }
};

// 8 consecutive rows of this lane's column: rows n .. n + 15 of the tile by lane / 32, columns
// f .. f + 31.  Each 16 lanes transpose 4 rows of 16 columns: a lane gives the address of four
// columns of one row and gets four rows of one column.
__device__ __forceinline__ bf16x8 fragment(const short* lds, int pitch, int n, int f) {
    const int lane = threadIdx.x & 63, g = lane >> 4, i = lane & 15;
    const short* p = lds + (n + (g >> 1) * 8 + (i >> 2)) * pitch + f + (g & 1) * 16 + (i & 3) * 4;
    union {
        s16x4 h[2];
        bf16x8 v;
    } u;
    u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
    u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * pitch));
    return u.v;
}

}  // namespace
}  // namespace ttp
