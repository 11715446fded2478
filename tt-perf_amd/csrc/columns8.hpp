// columns8.hpp — the operators' work on rows by groups of 8 columns, and which row a group is in.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "vector16.hpp"

namespace ttp {
namespace {

// n / d for n < 2^31 by a multiplication: with l = ceil(log2 d) and M = floor(2^(31 + l) / d) + 1,
// n M / 2^(31 + l) exceeds n / d by less than n / 2^31 / d, too little to reach the next integer.
struct Divider {
    uint64_t m;
    uint32_t shift;
};
inline Divider divider(uint32_t d) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    return {((1ull << (31 + l)) / d) + 1, 31 + l};
}
__device__ __forceinline__ uint32_t divide(uint32_t n, Divider d) {
    return (uint32_t)((n * d.m) >> d.shift);
}

// 8 columns of a row from column c on, those past the row's end as 0
template <class T>
__device__ __forceinline__ void load_cols(const T* row, uint32_t c, uint32_t cols, float (&v)[8]) {
    constexpr int P = kPer<T>;
    if (c + 8 <= cols) {
#pragma unroll
        for (int k = 0; k < 8 / P; ++k) {
            float w[P];
            unpack(load16(row + c + k * P), w, row);
#pragma unroll
            for (int j = 0; j < P; ++j) v[k * P + j] = w[j];
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = c + k < cols ? widen(row[c + k]) : 0.0f;
    }
}
template <class T>
__device__ __forceinline__ void store_cols(T* row, uint32_t c, uint32_t cols, const float (&v)[8]) {
    constexpr int P = kPer<T>;
    if (c + 8 <= cols) {
#pragma unroll
        for (int k = 0; k < 8 / P; ++k) {
            float w[P];
#pragma unroll
            for (int j = 0; j < P; ++j) w[j] = v[k * P + j];
            store16(row + c + k * P, pack(w, row));
        }
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if (c + k < cols) narrow(v[k], row + c + k);
    }
}

}  // namespace
}  // namespace ttp
