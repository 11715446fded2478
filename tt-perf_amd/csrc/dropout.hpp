// dropout.hpp — which elements dropout keeps (see ttp_dropout), on the device, and its checks on the
// host.
//
// Philox 4x32 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy as 1, 2, 3", 2011):
// ten rounds of two 32 x 32 -> 64 bit products each.  An element takes 16 of a group's 128 bits: the
// products are quarter-rate instructions, and 32 bits an element would make them the bound of a
// bf16 activation's dropout (30 lane operations an element against the 23 that a CU has for the
// 4 bytes it moves).  p is therefore a multiple of 2^-16, and the factor is the rounded p's, so
// that the mean stays.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "context.hpp"
#include "device.hpp"

namespace ttp {

struct Dropout {
    uint64_t seed, stream;
    const uint64_t* device_seed;
    uint32_t threshold;  // of 2^16
    float factor;
};

namespace {

__device__ __forceinline__ u32x4 philox(uint64_t seed, uint64_t stream, uint64_t group) {
    uint32_t c0 = (uint32_t)group, c1 = (uint32_t)(group >> 32);
    uint32_t c2 = (uint32_t)stream, c3 = (uint32_t)(stream >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int r = 0; r < 10; ++r) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)a;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return u32x4{c0, c1, c2, c3};
}

// Of a group's words: whether element j (0 to 7) is kept.
__device__ __forceinline__ bool keeps(u32x4 w, int j, uint32_t threshold) {
    return (j % 2 ? w[j / 2] >> 16 : w[j / 2] & 0xFFFFu) >= threshold;
}

__device__ __forceinline__ uint64_t seed_of(const Dropout& d) {
    return d.device_seed ? *d.device_seed : d.seed;
}

inline int check_dropout(const ttp_dropout* d) {
    if (!d) return ttpi::fail(TTP_ERR_INVALID, "null dropout");
    if (!(d->p >= 0.0 && d->p < 1.0))
        return ttpi::fail(TTP_ERR_INVALID, "dropout's p must be in [0, 1)");
    return TTP_OK;
}

inline Dropout dropout_of(const ttp_dropout& d) {
    const uint32_t t = (uint32_t)std::min(std::nearbyint(d.p * 65536.0), 65535.0);
    return {d.seed, d.stream, d.device_seed, t, (float)(65536.0 / (65536.0 - t))};
}

}  // namespace
}  // namespace ttp
