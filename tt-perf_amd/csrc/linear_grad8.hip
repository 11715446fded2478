// linear_grad8.hip — a linear layer's weight and bias gradients from its input kept in 8 bits.
//
//   dW[i, o] = sum_t xhat[t, i] dy[t, o]      db[o] = sum_t dy[t, o]
//
// over the rows t (tokens), added to the store's gradients with one rounding.  xhat = v 2^s is
// exact in bf16, so bf16 output gradients go through the bf16 matrix instructions with exact
// products and fp32 sums; an fp32 dy is the sum of three bf16 parts (8 + 8 + 8 bits of its 24),
// three instructions each.  Bound by the matrix instructions at 2 rows cols outs operations.
//
// Both operands have the summed index as their row, and a matrix instruction wants 8 consecutive
// rows of one column in each lane: tiles go to LDS as they lie in memory (kept values widened to
// bf16 once on the way) and come back through the transposing LDS load.  A block has a tile of
// kA columns of xhat by kB of dy, kN rows at a time in two LDS buffers: the next rows' loads are
// in flight while the matrix instructions run.  Few tiles split the rows: each part writes its
// fp32 tile to scratch memory and join_parts_kernel adds them up in order.
//
// Measured, bf16 8192 x 1280 x 5120 (256 x 256 tiles, two parts: 200 blocks for 256 CUs) 116 to
// 131 us by the card's clock, 820 to 925 TFLOP/s, and the join 11; on a CU with a block the matrix
// pipe is busy half of the time, the LDS 0.4; the rest are waits at the steps' barriers.
// fp32 3585 x 384 x 1536 (128 x 128 tiles, seven parts of 512 rows): 28 us, three products each;
// the matrix pipe is busy a quarter of the time, 16 steps are too few to hide the first and the
// last.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "checkpoint8.hpp"
#include "context.hpp"
#include "linear_tiles.hpp"
#include "matrix.hpp"
#include "operand.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

// kA x kB of the gradient per block, kN rows per step, kWA x kWB waves over the tile, kDepth steps'
// loads from memory in flight.
template <int A, int B, int N, int WA, int WB, int D>
struct Tile {
    static constexpr int kA = A, kB = B, kN = N, kWA = WA, kWB = WB, kDepth = D;
    static constexpr int kThreads = 64 * WA * WB;
    static constexpr int kFA = A / WA / 32, kFB = B / WB / 32;  // 32 x 32 fragments of a wave
    // LDS rows are 64 bytes longer than the tile: the four rows that a transposing load takes at
    // once lie in different banks
    static constexpr int kPad = 32;
    static constexpr int kPitchA = A + kPad, kPitchB = B + kPad;  // bf16 elements
};

struct LinearArgs {
    const uint8_t *values, *scales;
    const void* dy;
    uint64_t rows, per;  // rows in all, and of a part (a whole number of steps)
    uint64_t dy_stride;
    uint32_t width, cols, outs;  // width: a kept row's bytes
    uint32_t tiles_a, tiles_b, parts;
    int transposed;  // the weight is outs x cols
    // one part: the gradients (bf16 or fp32; `first`: assigned).  More: parts of the sums
    void *dw, *db;
    int bf16, dw_first, db_first;
    float *dw_parts, *db_parts;
};

// 16 kept values as bf16
template <int kFormat>
__device__ __forceinline__ void widen16(u32x4 w, uint32_t scale, u32x4 (&out)[2]) {
    const float s = __uint_as_float(scale << 23);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        if constexpr (kFormat == TTP_CHECKPOINT_INT8) {
            float v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = (float)((int)(w[k] << (24 - 8 * j)) >> 24) * s;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const f32x2 two = {v[2 * j], v[2 * j + 1]};
                out[k / 2][k % 2 * 2 + j] =
                    __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
            }
        } else {
            const uint32_t u = scale == 255u ? 0x7F7F7F7Fu : w[k];  // NaN
            out[k / 2][k % 2 * 2] = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, s, false));
            out[k / 2][k % 2 * 2 + 1] = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(u, s, true));
        }
    }
}

// Writes n of 16 consecutive elements of a gradient's row.
__device__ __forceinline__ void put(const LinearArgs& a, uint64_t at, uint32_t n,
                                    const float (&v)[16]) {
    if (a.bf16) {
        uint16_t* p = (uint16_t*)a.dw + at;
        if (n == 16) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                float w[8], old[8];
                if (!a.dw_first) unpack(load16(p + 8 * h), old, p);
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    w[k] = a.dw_first ? v[8 * h + k] : old[k] + v[8 * h + k];
                store16(p + 8 * h, pack(w, p));
            }
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (k < (int)n) narrow(a.dw_first ? v[k] : widen(p[k]) + v[k], p + k);
        }
    } else {
        float* p = (float*)a.dw + at;
        if (n == 16) {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                float w[4], old[4];
                if (!a.dw_first) unpack(load16(p + 4 * h), old, p);
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    w[k] = a.dw_first ? v[4 * h + k] : old[k] + v[4 * h + k];
                store16(p + 4 * h, pack(w, p));
            }
        } else {
#pragma unroll
            for (int k = 0; k < 16; ++k)
                if (k < (int)n) p[k] = a.dw_first ? v[k] : p[k] + v[k];
        }
    }
}
__device__ __forceinline__ void put_bias(const LinearArgs& a, uint32_t o, float v) {
    if (a.bf16) {
        uint16_t* p = (uint16_t*)a.db + o;
        narrow(a.db_first ? v : widen(*p) + v, p);
    } else {
        float* p = (float*)a.db + o;
        *p = a.db_first ? v : *p + v;
    }
}

template <class G, int kFormat, class T>
__global__ __launch_bounds__(T::kThreads, T::kThreads == 512 ? 1 : 2) void linear_grad_kernel(
    LinearArgs a) {
    constexpr int kPlanes = sizeof(G) == 2 ? 1 : 3;
    constexpr int kSizeA = T::kN * T::kPitchA, kSizeB = T::kN * T::kPitchB;
    constexpr int kBuffer = kSizeA + kPlanes * kSizeB;
    constexpr int kChunksA = T::kN * T::kA / 16 / T::kThreads;  // per lane and step
    constexpr int kChunksB = T::kN * T::kB / 8 / T::kThreads;
    static_assert(kChunksA >= 1 && kChunksB >= 1 && T::kThreads % (T::kB / 8) == 0 &&
                  T::kThreads % (T::kA / 16) == 0);
    constexpr int kRowsA = T::kThreads / (T::kA / 16), kRowsB = T::kThreads / (T::kB / 8);
    constexpr int kOutPitch = 36;  // floats; a wave's 32 x 32 of the gradient on its way out
    constexpr int kOut = T::kThreads / 64 * 32 * kOutPitch * 2;
    __shared__ __align__(16) short lds[2 * kBuffer > kOut ? 2 * kBuffer : kOut];

    const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
    const uint32_t part = id / (a.tiles_a * a.tiles_b), tile = id % (a.tiles_a * a.tiles_b);
    const uint32_t a0 = tile % a.tiles_a * T::kA, b0 = tile / a.tiles_a * T::kB;
    const uint64_t row0 = part * a.per;
    const uint32_t rows = (uint32_t)(row0 >= a.rows ? 0 : min(a.per, a.rows - row0));
    const bool bias = a.db && a0 == 0;

    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wa = wave / T::kWB * (T::kA / T::kWA), wb = wave % T::kWB * (T::kB / T::kWB);

    // this lane's chunks: columns ca of xhat (of the tile), rows ta + k kRowsA; and of dy
    const uint32_t ca = t % (T::kA / 16) * 16, ta = t / (T::kA / 16);
    const uint32_t cb = t % (T::kB / 8) * 8, tb = t / (T::kB / 8);
    // (columns past the end: any there are, as they only reach sums that are not written)
    const uint32_t column_a = min(a0 + ca, a.width - 16), column_b = b0 + cb < a.outs ? b0 + cb : 0;
    const uint8_t* pa = a.values + (row0 + ta) * a.width + column_a;
    const uint8_t* ps = a.scales + (row0 + ta) * (a.width / 32) + column_a / 32;
    const G* pb = (const G*)a.dy + (row0 + tb) * a.dy_stride + column_b;
    const uint64_t next_a = (uint64_t)T::kN * a.width, next_b = (uint64_t)T::kN * a.dy_stride;
    // The steps whose rows are whole chunks: a row's last chunk reaches into the next row, where
    // there is one (of 8 columns or more).
    const uint32_t whole =
        a.outs < 8 ? 0 : (rows - (a.outs % 8 && rows && row0 + rows == a.rows ? 1 : 0)) / T::kN;
    const int some_b = b0 + cb >= a.outs ? 0 : (int)min(a.outs - b0 - cb, 8u);
    struct Loads {
        u32x4 a[kChunksA];
        uint32_t s[kChunksA];
        Chunk8<G> b[kChunksB];
    };
    const auto forward = [&]() {
        pa += next_a;
        ps += next_a / 32;
        pb += next_b;
    };
    const auto load_whole = [&](Loads& r) {
#pragma unroll
        for (int k = 0; k < kChunksB; ++k) r.b[k].load(pb + (uint64_t)(k * kRowsB) * a.dy_stride);
#pragma unroll
        for (int k = 0; k < kChunksA; ++k) {
            r.a[k] = *reinterpret_cast<const u32x4*>(pa + (uint64_t)(k * kRowsA) * a.width);
            r.s[k] = ps[(uint64_t)(k * kRowsA) * (a.width / 32)];
        }
        forward();
    };
    const auto load = [&](Loads& r, uint32_t step) {
        const uint32_t left = rows - step * T::kN;
        if (step < whole) {
            load_whole(r);
        } else {  // rows past the end count 0
#pragma unroll
            for (int k = 0; k < kChunksB; ++k) {
                const G* p = pb + (uint64_t)(k * kRowsB) * a.dy_stride;
                const int n = tb + k * kRowsB < left ? some_b : 0;
                const uint64_t row = row0 + step * T::kN + tb + k * kRowsB;
                const bool spill = a.outs >= 8 && row + 1 < a.rows;
                if (n == 8 || (n && spill)) {
                    r.b[k].load(p);
                    if (n < 8) r.b[k].keep(n);
                } else if (n) {
                    r.b[k].load_some(p, n);
                } else {
                    r.b[k].clear();
                }
            }
#pragma unroll
            for (int k = 0; k < kChunksA; ++k) {
                r.a[k] = u32x4{0, 0, 0, 0};
                r.s[k] = 1;
                if (ta + k * kRowsA < left && a0 + ca < a.width) {
                    r.a[k] =
                        *reinterpret_cast<const u32x4*>(pa + (uint64_t)(k * kRowsA) * a.width);
                    r.s[k] = ps[(uint64_t)(k * kRowsA) * (a.width / 32)];
                }
            }
            forward();
        }
    };
    const auto store = [&](const Loads& r, short* buffer) {
#pragma unroll
        for (int k = 0; k < kChunksA; ++k) {
            u32x4 w[2];
            widen16<kFormat>(r.a[k], r.s[k], w);
            short* p = buffer + (ta + k * kRowsA) * T::kPitchA + ca;
            *reinterpret_cast<u32x4*>(p) = w[0];
            *reinterpret_cast<u32x4*>(p + 8) = w[1];
        }
#pragma unroll
        for (int k = 0; k < kChunksB; ++k) {
            u32x4 w[kPlanes];
            r.b[k].planes(w);
#pragma unroll
            for (int j = 0; j < kPlanes; ++j)
                *reinterpret_cast<u32x4*>(buffer + kSizeA + j * kSizeB +
                                          (tb + k * kRowsB) * T::kPitchB + cb) = w[j];
        }
    };

    f32x16 acc[T::kFA][T::kFB];
#pragma unroll
    for (int i = 0; i < T::kFA; ++i)
#pragma unroll
        for (int j = 0; j < T::kFB; ++j) acc[i][j] = f32x16{};
    // the bias: this lane's rows of its columns, in two levels (sums of many steps by themselves)
    float near[8] = {}, far[8] = {};
    const auto sum_bias = [&](const Loads& r, uint32_t s) {
#pragma unroll
        for (int k = 0; k < kChunksB; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) near[j] += r.b[k].value(j);
        if ((s & 15) == 15)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                far[j] += near[j];
                near[j] = 0.0f;
            }
    };

    // A step is two rounds of 16 rows, whose operands are in registers before the step begins: step
    // s + 1 goes to the other LDS buffer behind round 0's instructions, its rounds' operands come
    // back behind round 1's, and step s + 2's loads from memory are in flight meanwhile.
    static_assert(T::kN == 32);
    struct Round {
        bf16x8 a[T::kFA], b[kPlanes][T::kFB];
    } round[2];
    const auto fetch = [&](const short* buffer, int r) {
        const int n = r * 16;
#pragma unroll
        for (int i = 0; i < T::kFA; ++i)
            round[r].a[i] = fragment(buffer, T::kPitchA, n, wa + 32 * i);
#pragma unroll
        for (int p = 0; p < kPlanes; ++p)
#pragma unroll
            for (int j = 0; j < T::kFB; ++j)
                round[r].b[p][j] =
                    fragment(buffer + kSizeA + p * kSizeB, T::kPitchB, n, wb + 32 * j);
    };
    const auto multiply = [&](int r) {
#pragma unroll
        for (int p = 0; p < kPlanes; ++p)
#pragma unroll
            for (int i = 0; i < T::kFA; ++i)
#pragma unroll
                for (int j = 0; j < T::kFB; ++j)
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                        round[r].a[i], round[r].b[p][j], acc[i][j], 0, 0, 0);
    };
    const uint32_t steps = (rows + T::kN - 1) / T::kN;
    // kDepth sets of loads in flight: step s uses set s % kDepth, and step s + kDepth's follow it
    Loads loads[T::kDepth];
    const auto advance = [&](Loads& r, uint32_t s, auto&& load_next) {
        short* next = lds + (s & 1) * kBuffer;  // step s: loaded, now into LDS
        multiply(0);
        store(r, next);
        // the next step's conversions between the matrix instructions, not behind them
#pragma unroll
        for (int k = 0; k < T::kFA * T::kFB; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, kPlanes, 0);  // matrix
            __builtin_amdgcn_sched_group_barrier(0x002, 6 * kPlanes, 0);  // vector
            __builtin_amdgcn_sched_group_barrier(0x200, kPlanes, 0);  // LDS writes
        }
        if (bias) sum_bias(r, s);
        load_next(r, s + T::kDepth);
        __syncthreads();
        fetch(next, 0);
        multiply(1);
        fetch(next, 1);
    };
    if (steps) {
#pragma unroll
        for (int d = 0; d < T::kDepth; ++d)
            if ((uint32_t)d < steps) load(loads[d], d);
        store(loads[0], lds);
        if (bias) sum_bias(loads[0], 0);
        if (T::kDepth < steps) load(loads[0], T::kDepth);
        __syncthreads();
        fetch(lds, 0);
        fetch(lds, 1);
        // As long as the loads are of whole tiles they are issued without a branch: what is waited
        // for is then counted, and the younger loads stay in flight.  A step's loads leave before
        // its barrier, and no later step's conversions, which wait for older loads, move in front
        // of them.  (8192 x 1280 x 5120 bf16: 140 us without these loops, 132 with them.  The
        // barrier behind the loads makes an fp32 dy a little slower.)
        uint32_t s = 1;
        for (; s + 2 * T::kDepth <= whole; s += T::kDepth)
#pragma unroll
            for (int d = 1; d <= T::kDepth; ++d) {
                advance(loads[d % T::kDepth], s + d - 1, [&](Loads& r, uint32_t) {
                    load_whole(r);
                    if constexpr (kPlanes == 1) __builtin_amdgcn_sched_barrier(0);
                });
                __builtin_amdgcn_sched_barrier(0);
            }
        for (; s < steps; s += T::kDepth)
#pragma unroll
            for (int d = 1; d <= T::kDepth; ++d)
                if (s + d - 1 < steps)
                    advance(loads[d % T::kDepth], s + d - 1, [&](Loads& r, uint32_t next) {
                        if (next < steps) load(r, next);
                    });
        multiply(0);
        multiply(1);
    }
    __syncthreads();

    // out, 32 x 32 at a time through this wave's LDS: the gradient's rows are columns of xhat,
    // or of dy where the weight is transposed
    float* out = reinterpret_cast<float*>(lds) + wave * 32 * kOutPitch;
    const uint32_t rows_out = a.transposed ? a.outs : a.cols;
    const uint32_t cols_out = a.transposed ? a.cols : a.outs;
#pragma unroll
    for (int i = 0; i < T::kFA; ++i)
#pragma unroll
        for (int j = 0; j < T::kFB; ++j) {
            // lane: column lane % 32 of dy, rows 8 (k / 4) + 4 (lane / 32) + k % 4 of xhat
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int x = 8 * (k / 4) + 4 * (lane >> 5) + k % 4, y = lane & 31;
                out[(a.transposed ? y : x) * kOutPitch + (a.transposed ? x : y)] = acc[i][j][k];
            }
            __builtin_amdgcn_wave_barrier();
            const uint32_t xa = a0 + wa + 32 * i, yb = b0 + wb + 32 * j;
            const uint32_t r = (a.transposed ? yb : xa) + lane / 2;
            const uint32_t c = (a.transposed ? xa : yb) + lane % 2 * 16;
            float v[16];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const f32x4 q = *reinterpret_cast<const f32x4*>(out + lane / 2 * kOutPitch +
                                                                lane % 2 * 16 + 4 * k);
#pragma unroll
                for (int m = 0; m < 4; ++m) v[4 * k + m] = q[m];
            }
            __builtin_amdgcn_wave_barrier();
            if (r < rows_out && c < cols_out) {
                const uint64_t at = (uint64_t)r * cols_out + c;
                const uint32_t n = min(16u, cols_out - c);
                if (a.parts == 1) {
                    put(a, at, n, v);
                } else {
                    float* p = a.dw_parts + (uint64_t)part * rows_out * cols_out + at;
                    if (n == 16) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const float w[4] = {v[4 * k], v[4 * k + 1], v[4 * k + 2],
                                                v[4 * k + 3]};
                            store16(p + 4 * k, pack(w, p));
                        }
                    } else {
#pragma unroll
                        for (int k = 0; k < 16; ++k)
                            if (k < (int)n) p[k] = v[k];
                    }
                }
            }
        }
    if (!bias) return;
    __syncthreads();
    // the lanes that share columns, in order
    float* sums = reinterpret_cast<float*>(lds);  // kRowsB x kB
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[tb * T::kB + cb + j] = far[j] + near[j];
    __syncthreads();
    for (int c = t; c < T::kB; c += T::kThreads) {
        if (b0 + c >= a.outs) break;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kRowsB; ++k) v += sums[k * T::kB + c];
        if (a.parts == 1)
            put_bias(a, b0 + c, v);
        else
            a.db_parts[(uint64_t)part * a.outs + b0 + c] = v;
    }
}

// The parts' sums, in order, into the gradients: four neighbouring elements of the weight per lane,
// then the bias.  Bound by reading the parts.
constexpr int kJoinBlock = 256;
template <class O>
__global__ __launch_bounds__(kJoinBlock) void join_parts_kernel(LinearArgs a) {
    const uint64_t n = (uint64_t)a.cols * a.outs, quads = n / 4;
    const uint64_t rest = n - quads * 4, total = quads + rest + (a.db ? a.outs : 0);
    O* dw = (O*)a.dw;
    for (uint64_t i = (uint64_t)blockIdx.x * kJoinBlock + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * kJoinBlock) {
        if (i < quads) {
            const float* p = a.dw_parts + 4 * i;
            float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
            for (uint32_t k = 0; k < a.parts; ++k) {
                float w[4];
                unpack(load16_once(p + k * n), w, p);
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] += w[j];
            }
            O* g = dw + 4 * i;  // (tensors start on 64 elements)
            if (!a.dw_first)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = widen(g[j]) + v[j];
            if constexpr (sizeof(O) == 2) {
                u32x2 w;
                w.x = bf16_pack(v[0], v[1]);
                w.y = bf16_pack(v[2], v[3]);
                *reinterpret_cast<u32x2*>(g) = w;
            } else {
                *reinterpret_cast<f32x4*>(g) = f32x4{v[0], v[1], v[2], v[3]};
            }
        } else if (i < quads + rest) {
            const uint64_t at = 4 * quads + (i - quads);
            float v = 0.0f;
            for (uint32_t k = 0; k < a.parts; ++k) v += a.dw_parts[k * n + at];
            narrow(a.dw_first ? v : widen(dw[at]) + v, dw + at);
        } else {
            const uint32_t o = (uint32_t)(i - quads - rest);
            float v = 0.0f;
            for (uint32_t k = 0; k < a.parts; ++k) v += a.db_parts[(uint64_t)k * a.outs + o];
            put_bias(a, o, v);
        }
    }
}

// ---- launches -----------------------------------------------------------------------------------
using Wide = Tile<kWideTile, kWideTile, kStepRows, 2, 4, 2>;        // one block per CU
using Narrow = Tile<kNarrowTile, kNarrowTile, kStepRows, 2, 2, 1>;  // two
using Planes = Narrow;  // an fp32 dy: three products each

template <class G, int kFormat, class T>
int launch_tiles(const ttpi::Op& op, const LinearArgs& a) {
    const uint64_t blocks = (uint64_t)a.tiles_a * a.tiles_b * a.parts;
    if (blocks * T::kThreads >= (1ull << 32))
        return ttpi::fail(TTP_ERR_RANGE, "the weight has too many tiles for one launch");
    (void)hipGetLastError();
    hipLaunchKernelGGL((linear_grad_kernel<G, kFormat, T>), dim3((uint32_t)blocks),
                       dim3(T::kThreads), 0, op.stream, a);
    TTPI_HIP(hipGetLastError());
    return TTP_OK;
}

}  // namespace
}  // namespace ttp

using namespace ttp;
using ttpi::fail;

extern "C" int ttp_accumulate_linear_grad8(ttp_ctx* ctx, uint32_t weight, uint32_t bias,
                                           const ttp_checkpoint8* kept, const ttp_matrix* dy,
                                           int transposed) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = ttpi::check_matrix(dy, "the output's gradient"))) return rc;
        if (!kept) return fail(TTP_ERR_INVALID, "null checkpoint");
        if (transposed != 0 && transposed != 1)
            return fail(TTP_ERR_INVALID, "transposed must be 0 or 1");
        const uint64_t rows = dy->rows, outs = dy->cols, cols = kept->cols;
        if (!cols || cols >= (1ull << 31))
            return fail(TTP_ERR_RANGE, "the checkpoint has " + std::to_string(cols) + " columns");
        const bool has_bias = bias != TTP_NO_TENSOR;
        if (has_bias && bias == weight)
            return fail(TTP_ERR_INVALID, "the weight and the bias are the same tensor");
        ttpi::GradTarget w{}, b{};
        if ((rc = ttpi::grad_target(ctx, weight, &w))) return rc;
        if (has_bias && (rc = ttpi::grad_target(ctx, bias, &b))) return rc;
        if (w.numel != cols * outs)
            return fail(TTP_ERR_RANGE, "tensor " + std::to_string(weight) + " has " +
                                           std::to_string(w.numel) + " elements, not " +
                                           std::to_string(cols) + " x " + std::to_string(outs));
        if (has_bias && b.numel != outs)
            return fail(TTP_ERR_RANGE, "tensor " + std::to_string(bias) + " has " +
                                           std::to_string(b.numel) + " elements, not " +
                                           std::to_string(outs));
        ttpi::Buffers buf(ctx);
        if ((rc = check_kept(buf, kept, rows, cols, false))) return rc;
        if ((rc = buf.matrix(dy, rows, outs, "the output's gradient", false))) return rc;
        const uint64_t size = w.bf16 ? 2 : 4;
        if ((rc = buf.array(w.data, w.numel, size, "the weight's gradient", true))) return rc;
        if (has_bias && (rc = buf.array(b.data, outs, size, "the bias's gradient", true)))
            return rc;

        LinearArgs a{};
        a.values = (const uint8_t*)kept->values;
        a.scales = (const uint8_t*)kept->scales;
        a.dy = dy->data;
        a.rows = rows;
        a.dy_stride = dy->stride;
        a.width = (uint32_t)kept_width(cols);
        a.cols = (uint32_t)cols;
        a.outs = (uint32_t)outs;
        a.transposed = transposed;
        a.dw = w.data;
        a.db = has_bias ? b.data : nullptr;
        a.bf16 = w.bf16;
        a.dw_first = w.first;
        a.db_first = b.first;
        const bool bf16 = dy->dtype == TTP_DTYPE_BF16;
        const uint64_t cus = (uint64_t)op.num_cus;
        const Cut cut = choose_cut(rows, a.cols, a.outs, bf16, cus);
        a.tiles_a = cut.tiles_a;
        a.tiles_b = cut.tiles_b;
        a.parts = cut.parts;
        a.per = cut.per;
        if (a.parts > 1) {
            void* ws;
            const uint64_t n = (uint64_t)a.parts * cols * outs;
            if ((rc = ttpi::workspace(ctx, (n + (uint64_t)a.parts * outs) * 4, &ws))) return rc;
            a.dw_parts = (float*)ws;
            a.db_parts = a.dw_parts + n;
        }
        const bool int8 = kept->format == TTP_CHECKPOINT_INT8;
        if (bf16 && cut.wide)
            rc = int8 ? launch_tiles<uint16_t, TTP_CHECKPOINT_INT8, Wide>(op, a)
                      : launch_tiles<uint16_t, TTP_CHECKPOINT_E4M3, Wide>(op, a);
        else if (bf16)
            rc = int8 ? launch_tiles<uint16_t, TTP_CHECKPOINT_INT8, Narrow>(op, a)
                      : launch_tiles<uint16_t, TTP_CHECKPOINT_E4M3, Narrow>(op, a);
        else
            rc = int8 ? launch_tiles<float, TTP_CHECKPOINT_INT8, Planes>(op, a)
                      : launch_tiles<float, TTP_CHECKPOINT_E4M3, Planes>(op, a);
        if (rc) return rc;
        if (a.parts > 1) {
            const uint64_t n = cols * outs / 4 + 3 + outs;
            const dim3 block(kJoinBlock),
                grid((uint32_t)std::min<uint64_t>((n + kJoinBlock - 1) / kJoinBlock, cus * 16));
            (void)hipGetLastError();
            if (a.bf16)
                hipLaunchKernelGGL(join_parts_kernel<uint16_t>, grid, block, 0, op.stream, a);
            else
                hipLaunchKernelGGL(join_parts_kernel<float>, grid, block, 0, op.stream, a);
            TTPI_HIP(hipGetLastError());
        }
        ttpi::grad_written(ctx, weight);
        if (has_bias) ttpi::grad_written(ctx, bias);
        return TTP_OK;
    });
}
