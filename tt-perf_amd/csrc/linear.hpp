// linear.hpp — a linear product's arguments, and what follows the product on the device.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "columns8.hpp"
#include "dropout.hpp"
#include "gelu.hpp"
#include "linear_cut.hpp"
#include "operand.hpp"
#include "vector16.hpp"

namespace ttp {

struct LinearArgs {
    const void *x, *w;
    uint64_t x_stride, w_stride;
    uint32_t rows, cols, outs;
    uint32_t tiles_m, tiles_n;
    // the summed index in parts of `per` (a whole number of steps): each part's sums go to
    // `partial`, rows x outs with a row every `pitch` elements; one part: on to y at once
    uint32_t parts, per;
    float* partial;
    uint32_t pitch;
    // what follows the product
    const void* bias;  // or null, of x's type
    int activation;
    bool has_dropout;
    Dropout dropout;
    const void* residual;  // or null, of y's type
    void* y;
    uint64_t residual_stride, y_stride;
};

// Launches linear_direct_kernel in `shape` on tiles and parts that the arguments name.
__attribute__((visibility("hidden"))) void launch_direct_to_bf16(LinearShape shape, bool transposed,
                                                                 uint32_t blocks, hipStream_t stream,
                                                                 const LinearArgs& a);
__attribute__((visibility("hidden"))) void launch_direct_to_fp32(LinearShape shape, bool transposed,
                                                                 uint32_t blocks, hipStream_t stream,
                                                                 const LinearArgs& a);

namespace {

template <class G>
__device__ __forceinline__ void load_upto8(Chunk8<G>& c, const G* p, int n) {  // then 0
    if (n >= 8)
        c.load(p);
    else if (n > 0)
        c.load_some(p, n);
    else
        c.clear();
}

// The residual's 8 elements from column c on, to be asked for ahead of their use.
template <class Y>
__device__ __forceinline__ void load_residual(const LinearArgs& a, uint32_t row, uint32_t c,
                                              Chunk8<Y>& r) {
    if (a.residual && row < a.rows && c < a.outs)
        load_upto8(r, (const Y*)a.residual + row * a.residual_stride + c, (int)min(a.outs - c, 8u));
}

template <class G>
__device__ __forceinline__ void add_bias8(const LinearArgs& a, uint32_t c, float (&v)[8]) {
    if (!a.bias) return;
    float b[8];
    load_cols((const G*)a.bias, c, a.outs, b);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] += b[j];
}

// 8 neighbouring sums of a row with their bias (column c a multiple of 8), on to y.
template <class Y>
__device__ __forceinline__ void finish8(const LinearArgs& a, uint64_t seed, uint32_t row, uint32_t c,
                                        float (&v)[8], const Chunk8<Y>& r) {
    if (a.activation == TTP_ACTIVATION_RELU) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];  // (NaN stays NaN)
    } else if (a.activation == TTP_ACTIVATION_GELU_ERF) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = gelu<false>(v[j]);
    } else if (a.activation == TTP_ACTIVATION_GELU_TANH) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = gelu<true>(v[j]);
    }
    if (a.has_dropout) {
        const uint32_t groups = (a.outs + 7) / 8;
        const u32x4 w = philox(seed, a.dropout.stream, (uint64_t)row * groups + c / 8);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool keep = keeps(w, j, a.dropout.threshold);
            const float kept = v[j] * a.dropout.factor;
            if (a.residual)
                v[j] = keep ? r.value(j) + kept : r.value(j);
            else
                v[j] = keep ? kept : 0.0f;
        }
    } else if (a.residual) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = r.value(j) + v[j];
    }
    store_cols((Y*)a.y + row * a.y_stride, c, a.outs, v);
}

// A part's 8 sums.
__device__ __forceinline__ void put_part8(const LinearArgs& a, uint32_t part, uint32_t row,
                                          uint32_t c, const float (&v)[8]) {
    float* p = a.partial + ((uint64_t)part * a.rows + row) * a.pitch;  // (whole groups of 8)
    store_cols(p, c, a.pitch, v);
}

}  // namespace
}  // namespace ttp
