// device.hpp — device code that the library's kernels share: bf16 conversion, the block sum of
// doubles, and the last block of a launch.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ttp {

constexpr int kBlock = 256;  // 4 wave64s: norm pass, its decisions and helper kernels

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------------------------
// bf16
// ------------------------------------------------------------------------------------
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// round-to-nearest-even; NaN -> canonical 0x7FC0
__device__ __forceinline__ uint32_t bf16_rne(float x) {
    const uint32_t u = __float_as_uint(x);
    const uint32_t r = (u + 0x7FFFu + ((u >> 16) & 1u)) >> 16;
    return ((u & 0x7FFFFFFFu) > 0x7F800000u) ? 0x7FC0u : r;
}

__device__ __forceinline__ uint32_t bf16_pack(float a, float b) {
    return bf16_rne(a) | (bf16_rne(b) << 16);
}

// ------------------------------------------------------------------------------------
// block reduction of a double (fixed shape: deterministic)
// ------------------------------------------------------------------------------------
// x of the lane that a DPP control names (both 32-bit halves)
template <int kCtrl>
__device__ __forceinline__ double dpp(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, kCtrl, 0xF, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), kCtrl, 0xF, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)lo | ((uint64_t)hi << 32));
}

// The wave's sum in every lane, as the butterfly x += x[lane ^ off] for off = 32, 16, 8, 4, 2, 1
// gives it (bit for bit), without LDS permutes: a swap of the wave's halves, then of its 16-lane
// rows; within a row a rotation by 8, then by 4 (the values repeat every 8 lanes by then, so lane
// + 4 holds what lane ^ 4 does), then quad permutes.  Each LDS permute waited ~100 cycles, twelve
// of them in a chain at the end of every block: nanoGPT-char's AdamW step took 53.6 us with them
// and takes 53.2, the last of 8 GPT-2 124M shards 74.3 and 74.0.
__device__ __forceinline__ double wave_sum(double x) {
    const uint64_t u = __builtin_bit_cast(uint64_t, x);
    {
        const auto lo = __builtin_amdgcn_permlane32_swap((uint32_t)u, (uint32_t)u, false, false);
        const auto hi =
            __builtin_amdgcn_permlane32_swap((uint32_t)(u >> 32), (uint32_t)(u >> 32), false, false);
        x = __builtin_bit_cast(double, (uint64_t)lo[0] | ((uint64_t)hi[0] << 32)) +
            __builtin_bit_cast(double, (uint64_t)lo[1] | ((uint64_t)hi[1] << 32));
    }
    {
        const uint64_t w = __builtin_bit_cast(uint64_t, x);
        const auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)w, (uint32_t)w, false, false);
        const auto hi =
            __builtin_amdgcn_permlane16_swap((uint32_t)(w >> 32), (uint32_t)(w >> 32), false, false);
        x = __builtin_bit_cast(double, (uint64_t)lo[0] | ((uint64_t)hi[0] << 32)) +
            __builtin_bit_cast(double, (uint64_t)lo[1] | ((uint64_t)hi[1] << 32));
    }
    x += dpp<0x128>(x);  // row_ror:8
    x += dpp<0x124>(x);  // row_ror:4
    x += dpp<0x4E>(x);   // quad_perm:[2,3,0,1]
    x += dpp<0xB1>(x);   // quad_perm:[1,0,3,2]
    return x;
}

__device__ __forceinline__ double block_sum(double x, double* lds) {
    x = wave_sum(x);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if (lane == 0) lds[wave] = x;
    __syncthreads();
    double r = 0.0;
    if (threadIdx.x == 0) {
#pragma unroll
        for (int w = 0; w < kBlock / 64; ++w) r += lds[w];
    }
    __syncthreads();
    return r;  // valid in thread 0
}

// ------------------------------------------------------------------------------------
// the last block of a launch
// ------------------------------------------------------------------------------------
// A value that the launch's last block reads: stored and loaded as a relaxed atomic of device
// scope, past the caches that other XCDs do not share.
__device__ __forceinline__ void st_device(double* p, double x) {
    __hip_atomic_store(p, x, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double ld_device(const double* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Tickets: kTicketGroups counters 128 B apart, which block b takes from counter b modulo
// kTicketGroups, and one more that the last block of each group takes from.  One counter for a
// whole launch made 2,048 blocks wait in line for the same word.  All are zero between
// launches: the block that takes a counter's last ticket sets it back.
constexpr uint32_t kTicketGroups = 32, kTicketPitch = 32;
constexpr uint32_t kTicketWords = (kTicketGroups + 1) * kTicketPitch;
__device__ __forceinline__ bool last_ticket(uint32_t* p, uint32_t of) {
    const bool last =
        __hip_atomic_fetch_add(p, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of - 1;
    if (last) __hip_atomic_store(p, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return last;
}

// Whether this block is the launch's last to get here; every block of the launch calls it, with
// all its lanes, after thread 0's st_device() stores, which the last block may then read with
// ld_device().  Thread 0 waits until its stores have been acknowledged (device-scope stores
// write through, so that is at memory) before it takes its ticket.  That wait takes the place of
// a release fence: a device-scope fence per block also writes the XCD's L2 back and costs
// ~50 ns per block, one block after another.
// Measured (MLP AdamW with clipping, fp32): the step 9.0-9.5 us in two launches against 12.7 with
// a launch of one block for the decisions; the norm kernel's tail takes about as long as that
// launch did where the GPU is the bound (nanoGPT-char 53.7 against 53.6 us).
__device__ __forceinline__ bool is_last_block(uint32_t* tickets, uint32_t* lds_flag) {
    if (threadIdx.x == 0) {
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0);
        asm volatile("" ::: "memory");
        const uint32_t g = blockIdx.x % kTicketGroups;
        const uint32_t size = (gridDim.x - g + kTicketGroups - 1) / kTicketGroups;
        const uint32_t groups = min(gridDim.x, kTicketGroups);
        *lds_flag = last_ticket(tickets + g * kTicketPitch, size) &&
                    last_ticket(tickets + kTicketGroups * kTicketPitch, groups);
    }
    __syncthreads();
    return *lds_flag != 0;
}

}  // namespace ttp
