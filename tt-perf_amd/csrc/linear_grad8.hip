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
#include <hip/hip_runtime.h>

#include <algorithm>

#include "checkpoint8.hpp"
#include "context.hpp"
#include "matrix.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// kA x kB of the gradient per block, kN rows per step, kWA x kWB waves
template <int A, int B, int N, int WA, int WB>
struct Tile {
    static constexpr int kA = A, kB = B, kN = N, kWA = WA, kWB = WB;
    static constexpr int kThreads = 64 * WA * WB;
    static constexpr int kFA = A / WA / 32, kFB = B / WB / 32;  // 32 x 32 fragments of a wave
    // LDS rows are 64 bytes longer than the tile: the four rows that a transposing load takes at
    // once lie in different banks
    static constexpr int kPitchA = A + 32, kPitchB = B + 32;  // bf16 elements
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

// Blocks go to the 8 XCDs in turn: neighbours in this order are on one XCD, and share its L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t n) {
    const uint32_t x = b % 8, q = n / 8, r = n % 8;
    return x * q + min(x, r) + b / 8;
}

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

// x as the sum of three bf16 (pairs packed)
__device__ __forceinline__ void split3(float a, float b, uint32_t (&p)[3]) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const f32x2 two = {a, b};
        p[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
        a -= bf16_lo(p[k]);
        b -= bf16_hi(p[k]);
    }
}

// Columns c .. c + 7 of a row, past the end 0
template <class G>
struct Chunk8;
template <>
struct Chunk8<uint16_t> {
    u32x4 w;
    __device__ __forceinline__ void load(const uint16_t* row, uint32_t c, uint32_t cols, bool live) {
        w = u32x4{0, 0, 0, 0};
        if (!live || c >= cols) return;
        if (c + 8 <= cols) {
            w = load16(row + c);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k < cols) w[k / 2] |= (uint32_t)row[c + k] << (16 * (k % 2));
        }
    }
    __device__ __forceinline__ float value(int k) const {
        return k % 2 ? bf16_hi(w[k / 2]) : bf16_lo(w[k / 2]);
    }
    __device__ __forceinline__ void planes(u32x4 (&p)[1]) const { p[0] = w; }
};
template <>
struct Chunk8<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* row, uint32_t c, uint32_t cols, bool live) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = 0.0f;
        if (!live || c >= cols) return;
        if (c + 8 <= cols) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const u32x4 w = load16(row + c + 4 * h);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[4 * h + k] = __uint_as_float(w[k]);
            }
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (c + k < cols) v[k] = row[c + k];
        }
    }
    __device__ __forceinline__ float value(int k) const { return v[k]; }
    __device__ __forceinline__ void planes(u32x4 (&p)[3]) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t three[3];
            split3(v[2 * k], v[2 * k + 1], three);
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

// Writes 16 consecutive elements of a gradient's row (those before `cols`).
__device__ __forceinline__ void put(const LinearArgs& a, uint64_t at, uint32_t n,
                                    const float (&v)[16]) {
    if (a.parts > 1) return;
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
__global__ __launch_bounds__(T::kThreads, 2) void linear_grad_kernel(LinearArgs a) {
    constexpr int kPlanes = sizeof(G) == 2 ? 1 : 3;
    constexpr int kSizeA = T::kN * T::kPitchA, kSizeB = T::kN * T::kPitchB;
    constexpr int kBuffer = kSizeA + kPlanes * kSizeB;
    constexpr int kChunksA = T::kN * T::kA / 16 / T::kThreads;  // per lane and step
    constexpr int kChunksB = T::kN * T::kB / 8 / T::kThreads;
    static_assert(kChunksA >= 1 && kChunksB >= 1 && T::kThreads % (T::kB / 8) == 0);
    constexpr int kOutPitch = 36;  // floats; a wave's 32 x 32 of the gradient on its way out
    constexpr int kOut = T::kWA * T::kWB * 32 * kOutPitch * 2;
    __shared__ __align__(16) short lds[2 * kBuffer > kOut ? 2 * kBuffer : kOut];

    const uint32_t id = xcd_order(blockIdx.x, gridDim.x);
    const uint32_t part = id / (a.tiles_a * a.tiles_b), tile = id % (a.tiles_a * a.tiles_b);
    const uint32_t a0 = tile % a.tiles_a * T::kA, b0 = tile / a.tiles_a * T::kB;
    const uint64_t row0 = part * a.per;
    const uint32_t rows = (uint32_t)(row0 >= a.rows ? 0 : min(a.per, a.rows - row0));
    const bool bias = a.db && a0 == 0;

    const int t = threadIdx.x, wave = t >> 6, lane = t & 63;
    const int wa = wave / T::kWB * (T::kA / T::kWA), wb = wave % T::kWB * (T::kB / T::kWB);

    const uint32_t colb = t % (T::kB / 8) * 8;  // this lane's columns of dy, of the tile
    u32x4 ra[kChunksA];
    uint32_t rs[kChunksA];
    Chunk8<G> rb[kChunksB];
    const auto load = [&](uint32_t step) {
        const uint32_t n0 = step * T::kN;
#pragma unroll
        for (int k = 0; k < kChunksA; ++k) {
            const uint32_t e = t + k * T::kThreads;
            const uint32_t n = n0 + e / (T::kA / 16), c = a0 + e % (T::kA / 16) * 16;
            ra[k] = u32x4{0, 0, 0, 0};
            rs[k] = 1;
            if (n < rows && c < a.width) {
                const uint64_t at = (row0 + n) * a.width + c;
                ra[k] = *reinterpret_cast<const u32x4*>(a.values + at);
                rs[k] = a.scales[at / 32];
            }
        }
#pragma unroll
        for (int k = 0; k < kChunksB; ++k) {
            const uint32_t n = n0 + (t + k * T::kThreads) / (T::kB / 8);
            rb[k].load((const G*)a.dy + (row0 + n) * a.dy_stride, b0 + colb, a.outs, n < rows);
        }
    };
    const auto store = [&](short* buffer) {
#pragma unroll
        for (int k = 0; k < kChunksA; ++k) {
            const uint32_t e = t + k * T::kThreads;
            u32x4 w[2];
            widen16<kFormat>(ra[k], rs[k], w);
            short* p = buffer + e / (T::kA / 16) * T::kPitchA + e % (T::kA / 16) * 16;
            *reinterpret_cast<u32x4*>(p) = w[0];
            *reinterpret_cast<u32x4*>(p + 8) = w[1];
        }
#pragma unroll
        for (int k = 0; k < kChunksB; ++k) {
            const uint32_t e = t + k * T::kThreads;
            u32x4 w[kPlanes];
            rb[k].planes(w);
#pragma unroll
            for (int j = 0; j < kPlanes; ++j)
                *reinterpret_cast<u32x4*>(buffer + kSizeA + j * kSizeB +
                                          e / (T::kB / 8) * T::kPitchB + colb) = w[j];
        }
    };

    f32x16 acc[T::kFA][T::kFB];
#pragma unroll
    for (int i = 0; i < T::kFA; ++i)
#pragma unroll
        for (int j = 0; j < T::kFB; ++j) acc[i][j] = f32x16{};
    // the bias: this lane's rows of its columns, in two levels (sums of many steps by themselves)
    float near[8] = {}, far[8] = {};

    const uint32_t steps = (rows + T::kN - 1) / T::kN;
    if (steps) {
        load(0);
        store(lds);
    }
    for (uint32_t s = 0; s < steps; ++s) {
        __syncthreads();
        if (bias) {
#pragma unroll
            for (int k = 0; k < kChunksB; ++k)
#pragma unroll
                for (int j = 0; j < 8; ++j) near[j] += rb[k].value(j);
            if ((s & 15) == 15)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    far[j] += near[j];
                    near[j] = 0.0f;
                }
        }
        if (s + 1 < steps) load(s + 1);
        const short* buffer = lds + (s & 1) * kBuffer;
#pragma unroll
        for (int n = 0; n < T::kN; n += 16) {
            bf16x8 fa[T::kFA];
#pragma unroll
            for (int i = 0; i < T::kFA; ++i)
                fa[i] = fragment(buffer, T::kPitchA, n, wa + 32 * i);
#pragma unroll
            for (int p = 0; p < kPlanes; ++p) {
                bf16x8 fb[T::kFB];
#pragma unroll
                for (int j = 0; j < T::kFB; ++j)
                    fb[j] = fragment(buffer + kSizeA + p * kSizeB, T::kPitchB, n, wb + 32 * j);
#pragma unroll
                for (int i = 0; i < T::kFA; ++i)
#pragma unroll
                    for (int j = 0; j < T::kFB; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[j],
                                                                            acc[i][j], 0, 0, 0);
            }
        }
        if (s + 1 < steps) store(lds + ((s + 1) & 1) * kBuffer);
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
#pragma unroll
                    for (int k = 0; k < 16; ++k)
                        if (k < (int)n) p[k] = v[k];
                }
            }
        }
    if (!bias) return;
    __syncthreads();
    // the lanes that share columns, in order
    constexpr int kLanes = T::kThreads / (T::kB / 8);
    float* sums = reinterpret_cast<float*>(lds);  // kLanes x kB
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[t / (T::kB / 8) * T::kB + colb + j] = far[j] + near[j];
    __syncthreads();
    for (int c = t; c < T::kB; c += T::kThreads) {
        if (b0 + c >= a.outs) break;
        float v = 0.0f;
#pragma unroll
        for (int k = 0; k < kLanes; ++k) v += sums[k * T::kB + c];
        if (a.parts == 1)
            put_bias(a, b0 + c, v);
        else
            a.db_parts[(uint64_t)part * a.outs + b0 + c] = v;
    }
}

// The parts' sums, in order, into the gradients: four elements of the weight per lane, then the
// bias.
constexpr int kJoinBlock = 256;
__global__ __launch_bounds__(kJoinBlock) void join_parts_kernel(LinearArgs a) {
    const uint64_t n = (uint64_t)a.cols * a.outs, total = n + (a.db ? a.outs : 0);
    for (uint64_t i = (uint64_t)blockIdx.x * kJoinBlock + threadIdx.x; i < total;
         i += (uint64_t)gridDim.x * kJoinBlock) {
        const bool weight = i < n;
        const float* p = weight ? a.dw_parts + i : a.db_parts + (i - n);
        const uint64_t pitch = weight ? n : a.outs;
        float v = 0.0f;
        for (uint32_t k = 0; k < a.parts; ++k) v += p[k * pitch];
        if (!weight) {
            put_bias(a, (uint32_t)(i - n), v);
        } else if (a.bf16) {
            uint16_t* g = (uint16_t*)a.dw + i;
            narrow(a.dw_first ? v : widen(*g) + v, g);
        } else {
            float* g = (float*)a.dw + i;
            *g = a.dw_first ? v : *g + v;
        }
    }
}

// ---- launches -----------------------------------------------------------------------------------
using Wide = Tile<128, 128, 32, 2, 2>;

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

// Tiles below the launch's room (two blocks per CU) split the rows, at least 256 to a part.
template <class T>
void set_tiles(LinearArgs& a, int cus) {
    a.tiles_a = (a.cols + T::kA - 1) / T::kA;
    a.tiles_b = (a.outs + T::kB - 1) / T::kB;
    const uint64_t tiles = (uint64_t)a.tiles_a * a.tiles_b, room = 2 * (uint64_t)cus;
    const uint64_t parts =
        std::max<uint64_t>(std::min<uint64_t>(room / std::min(tiles, room), a.rows / 256), 1);
    a.per = ((a.rows + parts - 1) / parts + T::kN - 1) / T::kN * T::kN;
    a.parts = a.per ? (uint32_t)std::max<uint64_t>((a.rows + a.per - 1) / a.per, 1) : 1;
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
        set_tiles<Wide>(a, op.num_cus);
        if (a.parts > 1) {
            void* ws;
            const uint64_t n = (uint64_t)a.parts * cols * outs;
            if ((rc = ttpi::workspace(ctx, (n + (uint64_t)a.parts * outs) * 4, &ws))) return rc;
            a.dw_parts = (float*)ws;
            a.db_parts = a.dw_parts + n;
        }
        const bool int8 = kept->format == TTP_CHECKPOINT_INT8;
        if (dy->dtype == TTP_DTYPE_BF16)
            rc = int8 ? launch_tiles<uint16_t, TTP_CHECKPOINT_INT8, Wide>(op, a)
                      : launch_tiles<uint16_t, TTP_CHECKPOINT_E4M3, Wide>(op, a);
        else
            rc = int8 ? launch_tiles<float, TTP_CHECKPOINT_INT8, Wide>(op, a)
                      : launch_tiles<float, TTP_CHECKPOINT_E4M3, Wide>(op, a);
        if (rc) return rc;
        if (a.parts > 1) {
            const uint64_t n = cols * outs + outs;
            const uint32_t grid = (uint32_t)std::min<uint64_t>((n + kJoinBlock - 1) / kJoinBlock,
                                                               (uint64_t)op.num_cus * 16);
            (void)hipGetLastError();
            hipLaunchKernelGGL(join_parts_kernel, dim3(grid), dim3(kJoinBlock), 0, op.stream, a);
            TTPI_HIP(hipGetLastError());
        }
        ttpi::grad_written(ctx, weight);
        if (has_bias) ttpi::grad_written(ctx, bias);
        return TTP_OK;
    });
}
