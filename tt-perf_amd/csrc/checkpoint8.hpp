// checkpoint8.hpp — the 8-bit format of kept activations (see ttp_checkpoint8) on the device, and
// its checks on the host.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device.hpp"
#include "matrix.hpp"

namespace ttp {
namespace {

__host__ __device__ __forceinline__ uint64_t kept_width(uint64_t cols) {
    return (cols + TTP_CHECKPOINT_BLOCK - 1) / TTP_CHECKPOINT_BLOCK * TTP_CHECKPOINT_BLOCK;
}

// The scale's byte, of the largest magnitude's bits.  127 = 1.984375 x 2^6 and 448 = 1.75 x 2^8: a
// larger mantissa takes the next power.  The least e4m3 value is 2^-9 of the scale, which from
// the byte 10 on is a normal number.
template <int kFormat>
__device__ __forceinline__ uint32_t block_scale(uint32_t top) {
    constexpr bool kInt8 = kFormat == TTP_CHECKPOINT_INT8;
    constexpr uint32_t kMost = kInt8 ? 0x7E0000u : 0x600000u;
    const int e = (int)(top >> 23) - (kInt8 ? 6 : 8) + ((top & 0x7FFFFFu) > kMost ? 1 : 0);
    return top >= 0x7F800000u ? 255u : (uint32_t)max(e, kInt8 ? 1 : 10);
}

// 8 values on the block's grid.  A block that is not finite (scale 255): zeros, which decode to
// 0 x inf = NaN.
template <int kFormat>
__device__ __forceinline__ u32x2 encode8(const float (&x)[8], uint32_t scale) {
    if (scale == 255u) return u32x2{0, 0};
    const float inv = __uint_as_float((254u - scale) << 23);  // 2^-s, exact
    u32x2 w;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (kFormat == TTP_CHECKPOINT_INT8) {
            uint32_t b[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                b[k] = (uint32_t)(int)__builtin_rintf(x[4 * h + k] * inv) & 0xFFu;
            w[h] = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
        } else {
            int r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h] * inv, x[4 * h + 1] * inv, 0, false);
            r = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * h + 2] * inv, x[4 * h + 3] * inv, r, true);
            w[h] = (uint32_t)r;
        }
    }
    return w;
}

template <int kFormat>
__device__ __forceinline__ void decode8(u32x2 w, uint32_t scale, float (&x)[8]) {
    const float s = __uint_as_float(scale << 23);  // 255: infinity, and the values are 0
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if constexpr (kFormat == TTP_CHECKPOINT_INT8) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                x[4 * h + k] = (float)((int)(w[h] << (24 - 8 * k)) >> 24) * s;
        } else {
            const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], false);
            const f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[h], true);
            x[4 * h] = a.x * s;
            x[4 * h + 1] = a.y * s;
            x[4 * h + 2] = b.x * s;
            x[4 * h + 3] = b.y * s;
        }
    }
}

// A call's kept activation: its fields, its two arrays.
inline int check_kept(ttpi::Buffers& b, const ttp_checkpoint8* k, uint64_t rows, uint64_t cols,
                      bool written) {
    if (!k) return ttpi::fail(TTP_ERR_INVALID, "null checkpoint");
    if (k->format != TTP_CHECKPOINT_INT8 && k->format != TTP_CHECKPOINT_E4M3)
        return ttpi::fail(TTP_ERR_INVALID,
                          "the checkpoint's format must be TTP_CHECKPOINT_INT8 or _E4M3");
    if (k->reserved) return ttpi::fail(TTP_ERR_INVALID, "the checkpoint: reserved must be 0");
    if (k->rows != rows || k->cols != cols)
        return ttpi::fail(TTP_ERR_RANGE, "the checkpoint is of " + std::to_string(k->rows) +
                                             " x " + std::to_string(k->cols) + ", not " +
                                             std::to_string(rows) + " x " + std::to_string(cols));
    if ((uintptr_t)k->values % 16)
        return ttpi::fail(TTP_ERR_INVALID, "the checkpoint's values are not 16-byte aligned");
    const uint64_t width = kept_width(cols);
    const int rc = b.array(k->values, rows * width, 1, "the checkpoint's values", written);
    if (rc) return rc;
    return b.array(k->scales, rows * (width / TTP_CHECKPOINT_BLOCK), 1, "the checkpoint's scales",
                   written);
}

}  // namespace
}  // namespace ttp
