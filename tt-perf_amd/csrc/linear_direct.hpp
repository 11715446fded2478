// linear_direct.hpp — products of bf16 operands on the 16-byte grid, which go from memory straight
// into the LDS.
//
// kM x 32 F of y per block of four waves, kK of the summed index per step, through kStages LDS
// buffers that the loads fill without passing through registers.
//
// What bounds it: in the steps, power.  The clock falls to 1.7 GHz, and the matrix instructions alone, on
// random operands in registers, reach 2.0 PFLOP/s as 16 x 16 x 32 and 1.7 as 32 x 32 x 16, which is why
// the former are used; steps go at 1.3 PFLOP/s in 128 x 256 tiles and 1.47 in 256 x 160.  The rest is
// what lies before a tile's first step and behind its last, and uneven rounds of tiles: 8192 x 1280 x
// 5120 with GELU takes 118 us (0.91 PFLOP/s), two rounds of 128 x 256 tiles and a half one, 10.8 us of
// each round's 44 outside the steps; 8192 x 5120 x 1280 with dropout and a residual 103 (1.04), one
// round of 256 x 160, 13 us outside; 8192 x 768 x 50257 transposed 850 (0.74), with 24 steps to a
// tile (the library's product alone 575).  A token's 768 x 50257 is bound by W's 77 MB: 14.5 us, 5.3
// TB/s.
//
// Four shapes, since no tile is best for every grid of 256 CUs (linear_cut.hpp has the choice and the
// figures): 256 x 160 moves the fewest bytes through the LDS for a product, one block to a CU; 128 x 256
// and 128 x 128 run two, whose beginnings and ends overlap; 32 x 64 in four buffers keeps what a matrix
// read for few rows needs under way.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "linear.hpp"

namespace ttp {
namespace {

// where loads behind the summed index's end read
__device__ const uint4 kZeros[1] = {};

typedef __attribute__((address_space(3))) void* lds_ptr;

__device__ __forceinline__ void barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
template <int kLeft>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kLeft) : "memory");
}

// 16 bytes per lane from memory to the LDS, a wave's 1024 in the order of its lanes from `to` on.
// (Inline: behind the builtin, which does the same, the compiler waits for every load before it
// reads any of the LDS.  Nothing comes back to a register; who reads the buffer waits by vmcnt.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // (m0 is no register that the compiler keeps)
__device__ __forceinline__ void load_to_lds(uint32_t to, const char* base, uint32_t offset) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2"
                 ::"s"(to), "v"(offset), "s"(base)
                 : "memory", "m0");
}
__device__ __forceinline__ void load_to_lds(uint32_t to, const char* from) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off"
                 ::"s"(to), "v"(from)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// Where 16 bytes lie in a buffer.  Rows along the summed index have kK / 8 chunks, chunk c of a row
// at c ^ (row / (16 / chunks)): 16 rows' chunks c are in different banks.  Rows across it (W as it
// is) have 2 F pieces of 32 bytes.  A transposing load takes a piece of rows 0 to 3, 8 to 11, 16 to
// 19 and 24 to 27 (or those four on), and a row's pieces are turned by turn(row), which spreads
// these over the banks whatever F is.
template <int F>
__device__ __forceinline__ uint32_t turn(uint32_t row) {
    if constexpr (F % 4 == 0) return (row & 3) + (row >> 3 & 1) * 4;
    if constexpr (F % 4 == 2) return (row >> 1 & 1) + (row >> 3 & 1) * 2;
    return row >> 3 & 1;
}

// blocks of a shape that a CU's 160 KB hold
constexpr uint32_t blocks_per_cu(uint32_t m, uint32_t n, uint32_t k, uint32_t stages) {
    return 160 * 1024 / ((m + n) * k * 2 * stages);
}

template <uint32_t kM, int F, int WM, uint32_t kK, uint32_t kStages, class Y, bool kTransposed>
__global__ __launch_bounds__(256, blocks_per_cu(kM, 32 * F, kK, kStages))
void linear_direct_kernel(LinearArgs a) {
    constexpr uint32_t kN = 32 * F;
    constexpr int WN = 4 / WM;
    constexpr int FA = kM / WM / 16, FB = kN / WN / 16;  // 16 x 16 fragments of a wave
    static_assert(FA % 2 == 0 && FB * 16 * WN == (int)kN);
    constexpr uint32_t kBytesA = kM * kK * 2, kBytesB = kN * kK * 2, kBuffer = kBytesA + kBytesB;
    constexpr int kOutPitch = 16 * FB + 4;  // floats; 32 rows of a wave on their way out
    constexpr uint32_t kOut = 4 * 32 * kOutPitch * 4;
    __shared__ __align__(1024) char lds[kStages * kBuffer > kOut ? kStages * kBuffer : kOut];

    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = wave / WN * (kM / WM), wn = wave % WN * (kN / WN);
    uint32_t m0, n0, part;
    {  // neighbours on an XCD: eight tiles of rows by the tiles of columns
        uint32_t id = xcd_order(blockIdx.x, gridDim.x);
        part = id / (a.tiles_m * a.tiles_n);
        id -= part * (a.tiles_m * a.tiles_n);
        const uint32_t group = id / (8 * a.tiles_n), first = group * 8;
        const uint32_t high = min(8u, a.tiles_m - first), in = id - group * 8 * a.tiles_n;
        m0 = (first + in % high) * kM;
        n0 = in / high * kN;
    }

    const uint32_t k0 = part * a.per, cols = min(a.per, a.cols - k0);

    // this lane's chunks, as bytes from the tile's first row: x's rows t / kChunks + kRows j, ...
    constexpr uint32_t kChunks = kK / 8, kRows = 256 / kChunks;  // of a row; rows of a load
    constexpr uint32_t kFillsA = kM / kRows, kFillsB = kN / kRows, kFills = kFillsA + kFillsB;
    static_assert(kFillsB * kRows == kN);
    uint32_t off_a[kFillsA], off_b[kFillsB];
    // the chunk of its row that goes to its place
    const uint32_t ck = t % kChunks ^ (t / kChunks / (16 / kChunks) % kChunks);
#pragma unroll
    for (uint32_t j = 0; j < kFillsA; ++j) {
        const uint32_t row = min(m0 + t / kChunks + kRows * j, a.rows - 1) - m0;
        off_a[j] = (row * (uint32_t)a.x_stride + ck * 8) * 2;
    }
#pragma unroll
    for (uint32_t j = 0; j < kFillsB; ++j) {
        if constexpr (kTransposed) {
            const uint32_t row = min(n0 + t / kChunks + kRows * j, a.outs - 1) - n0;
            off_b[j] = (row * (uint32_t)a.w_stride + ck * 8) * 2;
        } else {
            const uint32_t q = t + 256 * j, row = q / (4 * F), at = q % (4 * F);
            const uint32_t piece = (at / 2 + 2 * F - turn<F>(row)) % (2 * F);
            const uint32_t col = min(n0 + piece * 16 + at % 2 * 8, a.outs - 8) - n0;
            off_b[j] = (row * (uint32_t)a.w_stride + col) * 2;
        }
    }
    const char* xs = (const char*)a.x + (m0 * a.x_stride + k0) * 2;
    const char* ws = (const char*)a.w + (kTransposed ? n0 * a.w_stride + k0 : k0 * a.w_stride + n0) * 2;
    const uint32_t ws_step = kTransposed ? kK * 2 : kK * (uint32_t)a.w_stride * 2;

    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_ptr)lds + wave * 1024;
    const auto fill_one = [&](uint32_t buffer, uint32_t j) {  // load j of a whole step
        const uint32_t to = lds0 + buffer + j * 4096;
        if (j < kFillsA)
            load_to_lds(to, xs, off_a[j < kFillsA ? j : 0]);
        else
            load_to_lds(to, ws, off_b[j < kFillsA ? 0 : j - kFillsA]);
    };
    const auto forward = [&]() {
        xs += kK * 2;
        ws += ws_step;
    };
    const auto fill = [&](uint32_t s, uint32_t buffer) {  // any step: zeros behind the last
        const uint32_t left = cols - s * kK;
        if (left >= kK) {
#pragma unroll
            for (uint32_t j = 0; j < kFills; ++j) fill_one(buffer, j);
            forward();
            return;
        }
        const char* zeros = (const char*)kZeros;
#pragma unroll
        for (uint32_t j = 0; j < kFills; ++j) {
            const uint32_t jb = j < kFillsA ? 0 : j - kFillsA;
            const uint32_t k = j < kFillsA || kTransposed ? ck * 8 : (t + 256 * jb) / (4 * F);
            const char* from = j < kFillsA ? xs + off_a[j < kFillsA ? j : 0] : ws + off_b[jb];
            load_to_lds(lds0 + buffer + j * 4096, k < left ? from : zeros);
        }
    };

    // operands of 32 of the summed index, two sets in turn
    struct Operands {
        bf16x8 a[FA], b[FB];
    } ops[2];
    constexpr uint32_t kRow = kK * 2;  // bytes
    const uint32_t row_at = (lane & 15) * kRow, swz = (lane & 15) / (16 / kChunks) % kChunks;
    constexpr int kReads = FA + FB;
    constexpr int kEach = (kReads + FA * FB - 1) / (FA * FB);  // of them behind a product
    // read n of a set: b0, then the others of b between those of a
    const auto fetch_one = [&](Operands& o, uint32_t at_buffer, int kk, int n) {
        const char* buffer = lds + at_buffer;
        const uint32_t at = row_at + ((kk * 4 + (lane >> 4)) ^ swz) * 16;
        constexpr int kPairs = 2 * (FA < FB ? FA : FB);
        const bool is_a = n < kPairs ? n % 2 == 1 : FA > FB;
        const int i = n < kPairs ? n / 2 : n - kPairs / 2;
        if (is_a) {
            o.a[i < FA ? i : 0] =
                *reinterpret_cast<const bf16x8*>(buffer + (wm + 16 * i) * kRow + at);
            return;
        }
        buffer += kBytesA;
        if constexpr (kTransposed) {
            o.b[i < FB ? i : 0] =
                *reinterpret_cast<const bf16x8*>(buffer + (wn + 16 * i) * kRow + at);
        } else {
            const int l = lane & 15;
            const uint32_t row = kk * 32 + (lane >> 4) * 8 + (l >> 2);  // and 4 rows on: turn is
            const uint32_t piece = (wn / 16 + i + turn<F>(row)) % (2 * F);  // the same there
            const char* p = buffer + row * (64 * F) + piece * 32 + (l & 3) * 8;
            union {
                s16x4 h[2];
                bf16x8 v;
            } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(p + 4 * 64 * F));
            o.b[i < FB ? i : 0] = u.v;
        }
    };
    float bias[FB];  // of this lane's columns
#pragma unroll
    for (int j = 0; j < FB; ++j) {
        const uint32_t c = n0 + wn + 16 * j + (lane & 15);
        bias[j] = a.bias && a.parts == 1 && c < a.outs ? widen(((const uint16_t*)a.bias)[c]) : 0.0f;
    }
    f32x4 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = f32x4{};
    // the products of a set, and what is to be issued behind each
    const auto multiply = [&](const Operands& o, auto&& between) {
#pragma unroll
        for (int n = 0; n < FA * FB; ++n) {
            const int i = n / FB, j = n % FB;
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(o.a[i], o.b[j], acc[i][j], 0, 0, 0);
            between(n);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    const uint32_t steps = (cols + kK - 1) / kK;
    constexpr int kSub = kK / 32;
    static_assert(kSub == 1 || kSub == 2);
    // Waits until at most `later` steps' loads of this wave are still on their way.
    const auto arrived = [&](uint32_t later) {
        static_assert(kStages >= 2 && kStages <= 4 && (kStages - 1) * kFills < 64);
        if (later == 0) wait_loads<0>();
        if (later == 1) wait_loads<kFills>();
        if constexpr (kStages > 2)
            if (later == 2) wait_loads<2 * kFills>();
        if constexpr (kStages > 3)
            if (later == 3) wait_loads<3 * kFills>();
    };
    uint32_t s = 0, here = 0, last = (kStages - 1) * kBuffer;  // the step, its buffer, the one before
    const auto turn_on = [&]() {
        last = here;
        here = here + kBuffer == kStages * kBuffer ? 0 : here + kBuffer;
        ++s;
    };
    // whether step n from here is there, whole
    const auto whole = [&](uint32_t n) { return (uint64_t)(s + n + 1) * kK <= cols; };
    // A step's share of a whole step's loads behind product n of `of` (issued at once they wait in
    // line, and the matrix instructions behind them).
    const auto spread = [&](uint32_t buffer, uint32_t n, uint32_t of) {
#pragma unroll
        for (uint32_t j = 0; j < kFills; ++j)
            if (j * of / kFills == n) fill_one(buffer, j);
        if (n == of - 1) forward();
    };
    if constexpr (kSub == 1) {
        // Blocks share the CU: what one waits for, another's products fill.  A step waits for its
        // buffer, reads it, and multiplies; the buffer of the step before is filled meanwhile.
        const auto step = [&](uint32_t later, auto&& between) {
            arrived(later);
            barrier();
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int n = 0; n < kReads; ++n) fetch_one(ops[0], here, 0, n);
            __builtin_amdgcn_sched_barrier(0);
            multiply(ops[0], between);
            // (every operand is in registers: the next barrier frees the buffer)
            turn_on();
        };
        for (uint32_t k = 0; k < kStages - 1 && k < steps; ++k) fill(k, k * kBuffer);
        while (whole(kStages - 1)) step(kStages - 2, [&](int n) { spread(last, n, FA * FB); });
        while (s < steps)
            step(min(steps - s - 1, kStages - 2), [&](int n) {
                if (n == 0 && s + kStages - 1 < steps) fill(s + kStages - 1, last);
            });
    } else {
        // A step begins with the operands of its first half in registers and reads the second's
        // behind that one's products, then the next step's first behind the second's.  In between
        // every wave has the step's operands and its own loads of the next one: a barrier, behind
        // which the step's buffer is filled again, up to the next barrier.
        const auto step = [&](auto&& first, auto&& second, uint32_t later, bool more) {
            const uint32_t next = here + kBuffer == kStages * kBuffer ? 0 : here + kBuffer;
            multiply(ops[0], [&](int n) {
#pragma unroll
                for (int r = n * kEach; r < (n + 1) * kEach; ++r)
                    if (r < kReads) fetch_one(ops[1], here, 1, r);
                first(n);
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            arrived(later);
            barrier();
            __builtin_amdgcn_sched_barrier(0);
            multiply(ops[1], [&](int n) {
#pragma unroll
                for (int r = n * kEach; r < (n + 1) * kEach; ++r)
                    if (r < kReads && more) fetch_one(ops[0], next, 0, r);
                second(n);
            });
            turn_on();
        };
        const uint32_t ahead = min(steps, kStages);
        for (uint32_t k = 0; k < ahead; ++k) fill(k, k * kBuffer);
        arrived(ahead - 1);
        barrier();
#pragma unroll
        for (int n = 0; n < kReads; ++n) fetch_one(ops[0], 0, 0, n);
        __builtin_amdgcn_sched_barrier(0);
        constexpr uint32_t kHalf = FA * FB;
        const auto none = [](int) {};
        const auto begin = [&](int n) { spread(here, n, 2 * kHalf); };
        const auto rest = [&](int n) { spread(last, kHalf + n, 2 * kHalf); };
        const auto at_once = [&](int n) {
            if (n == 0 && s + kStages < steps) fill(s + kStages, here);
        };
        if (whole(kStages)) {
            step(none, begin, kStages - 2, true);
            while (whole(kStages)) step(rest, begin, kStages - 2, true);
            step(rest, at_once, kStages - 2, true);
        }
        while (s < steps) {
            const bool more = s + 1 < steps;
            step(none, at_once, more ? min(steps - s - 2, kStages - 2) : 0, more);
        }
    }
    barrier();

    // out, 32 rows of this wave at a time through the LDS; the residual is asked for 32 rows ahead
    const uint64_t seed = a.has_dropout ? seed_of(a.dropout) : 0;
    float* out = reinterpret_cast<float*>(lds) + wave * 32 * kOutPitch;
    const auto place = [&](int i, int it) {  // of this lane's 8 columns, of 32 x 2 FB groups
        const uint32_t q = lane + 64 * it;
        struct {
            uint32_t r, c, row, col;
        } p{q / (2 * FB), q % (2 * FB) * 8, 0, 0};
        p.row = m0 + wm + 16 * i + p.r;
        p.col = n0 + wn + p.c;
        return p;
    };
    constexpr bool kAhead = sizeof(Y) == 2;  // (fp32 would take too many registers)
    Chunk8<Y> res[FB], next_res[kAhead ? FB : 1];
    const auto ask = [&](int i, Chunk8<Y>* r) {
        if (a.parts > 1) return;
#pragma unroll
        for (int it = 0; it < FB; ++it) {
            const auto p = place(i, it);
            load_residual(a, p.row, p.col, r[it]);
        }
    };
    if constexpr (kAhead) ask(0, res);
    // (one copy of what follows the product: four of them ran out of the instruction cache and took
    // 40% of an 8192 x 1280 x 5120 product's time)
#pragma unroll 1
    for (int i = 0; i < FA; i += 2) {
#pragma unroll
        for (int ii = 0; ii < FA; ii += 2)
            if (ii == i)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int j = 0; j < FB; ++j)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            out[(16 * h + 4 * (lane >> 4) + k) * kOutPitch + 16 * j +
                                (lane & 15)] = acc[ii + h][j][k] + bias[j];
        __builtin_amdgcn_wave_barrier();
        if constexpr (!kAhead)
            ask(i, res);
        else if (i + 2 < FA)
            ask(i + 2, next_res);
#pragma unroll
        for (int it = 0; it < FB; ++it) {
            const auto p = place(i, it);
            float v[8];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 w =
                    *reinterpret_cast<const f32x4*>(out + p.r * kOutPitch + p.c + 4 * h);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[4 * h + k] = w[k];
            }
            if (p.row < a.rows && p.col < a.outs) {
                if (a.parts > 1)
                    put_part8(a, part, p.row, p.col, v);
                else
                    finish8<Y>(a, seed, p.row, p.col, v, res[it]);
            }
            if constexpr (kAhead) res[it] = next_res[it];
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <uint32_t kM, int F, int WM, uint32_t kK, uint32_t kStages, class Y>
void launch_shape(bool transposed, uint32_t blocks, hipStream_t stream, const LinearArgs& a) {
    if (transposed)
        hipLaunchKernelGGL((linear_direct_kernel<kM, F, WM, kK, kStages, Y, true>), dim3(blocks),
                           dim3(256), 0, stream, a);
    else
        hipLaunchKernelGGL((linear_direct_kernel<kM, F, WM, kK, kStages, Y, false>), dim3(blocks),
                           dim3(256), 0, stream, a);
}

template <class Y>
void launch_direct(LinearShape shape, bool transposed, uint32_t blocks, hipStream_t stream,
                   const LinearArgs& a) {
    switch (shape) {  // (rows, outputs and step of linear_cut.hpp)
        case LinearShape::kThin:
            return launch_shape<32, 2, 1, 64, 4, Y>(transposed, blocks, stream, a);
        case LinearShape::kSmall:
            return launch_shape<128, 4, 2, 64, 2, Y>(transposed, blocks, stream, a);
        case LinearShape::kWide:
            return launch_shape<128, 8, 2, 32, 3, Y>(transposed, blocks, stream, a);
        case LinearShape::kLarge:
            return launch_shape<256, 5, 2, 64, 3, Y>(transposed, blocks, stream, a);
        case LinearShape::kThinAny:
        case LinearShape::kAny: break;
    }
}

}  // namespace
}  // namespace ttp
