// linear.hip — y = residual + dropout(activation(x W + bias)).
//
// Bound by the matrix instructions at 2 rows cols outs operations.  bf16 products are exact, sums are
// fp32.  An fp32 operand is the sum of three bf16 parts (8 bits each), and of the nine products of
// two operands the six largest are taken.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "context.hpp"
#include "linear.hpp"
#include "matrix.hpp"
#include "operand.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

// ---- operands ---------------------------------------------------------------------------------
// a and b as sums of three bf16 each (pairs packed): the first cut off, so that infinities and the
// largest numbers stay what they are, the others to nearest.  What is left of an infinity is taken
// from the largest number.  (See split3 for numbers below 2^-110 and NaN.)
__device__ __forceinline__ void split3_nearest(float a, float b, uint32_t (&p)[3]) {
    constexpr float kMost = 3.4028234663852886e38f;
    p[0] = __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u);
    a = __builtin_amdgcn_fmed3f(a, -kMost, kMost);
    b = __builtin_amdgcn_fmed3f(b, -kMost, kMost);
    a -= __uint_as_float(__float_as_uint(a) & 0xFFFF0000u);
    b -= __uint_as_float(__float_as_uint(b) & 0xFFFF0000u);
#pragma unroll
    for (int k = 1; k < 3; ++k) {
        const f32x2 two = {a, b};
        p[k] = __builtin_bit_cast(uint32_t, __builtin_convertvector(two, bf16x2));
        a -= bf16_lo(p[k]);
        b -= bf16_hi(p[k]);
    }
}
template <class G>
__device__ __forceinline__ void planes_of(const Chunk8<G>& c, u32x4 (&p)[sizeof(G) == 2 ? 1 : 3]) {
    if constexpr (sizeof(G) == 2) {
        c.planes(p);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            uint32_t three[3];
            split3_nearest(c.value(2 * k), c.value(2 * k + 1), three);
#pragma unroll
            for (int j = 0; j < 3; ++j) p[j][k] = three[j];
        }
    }
}

// The first parts with infinities as the largest number, for the products with another operand's
// second and third part, which may be 0 where the operand is not.
__device__ __forceinline__ bf16x8 finite(bf16x8 v) {
    typedef short i16x8 __attribute__((ext_vector_type(8)));
    typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
    const i16x8 most = (i16x8)(short)0x7F7F;
    const u16x8 least = (u16x8)(unsigned short)0xFF7F;
    const u16x8 u = __builtin_elementwise_min(__builtin_bit_cast(u16x8, v), least);
    return __builtin_bit_cast(bf16x8,
                              __builtin_elementwise_min(__builtin_bit_cast(i16x8, u), most));
}

// ---- operands of any alignment, through registers ---------------------------------------------
// 128 x 128 of y per block of four waves, or 32 x 128 where rows are few and W is what is read (a
// token's 768 x 50257 fp32: 35 us, of 30 for its 154 MB, instead of 64); 32 of the summed index per
// step; bf16 through two LDS buffers, the three parts of fp32 through one, so that blocks share a CU
// and one's products run beside another's splitting (3585 x 384 x 1536: 56 us with two buffers and one
// block, 44 so; 53 with eight waves, half of which split while the others multiply).  bf16 comes here
// where an operand is off the 16-byte grid: the gradient through a table of 50257 tokens, 8192 x 50257 x
// 768, takes 1170 us, in rows padded to a multiple of 8 1090 (the library's product 655 and 585).
constexpr uint32_t kTile = 128, kStep = 32;
constexpr int kPitchK = kStep + 8;  // LDS rows along the summed index, padded against conflicts
constexpr int kPitchN = kTile + 32;

// 8 consecutive elements of the summed index of row f + lane % 32, from n + 8 (lane / 32) on
__device__ __forceinline__ bf16x8 row_fragment(const short* lds, int n, int f) {
    const int lane = threadIdx.x & 63;
    return *reinterpret_cast<const bf16x8*>(lds + (f + (lane & 31)) * kPitchK + n + (lane >> 5) * 8);
}

constexpr int kAnyThreads = 256;
template <class G, class Y, bool kTransposed, uint32_t kM>
__global__ __launch_bounds__(kAnyThreads, kM == kTile ? 2 : 4) void linear_kernel(LinearArgs a) {
    constexpr int kPlanes = sizeof(G) == 2 ? 1 : 3, kBuffers = kPlanes == 1 ? 2 : 1;
    constexpr int FA = kM == kTile ? 2 : 1, FB = FA;  // 32 x 32 fragments of a wave
    constexpr int kChunks = 2;  // of W, that a lane loads in a step
    constexpr int kChunksA = kM == kTile ? 2 : 1;  // of x (kM 32: the first 128 lanes)
    constexpr uint32_t kRows = kTile / kChunks, kRowsN = kStep / kChunks;  // that a load covers
    constexpr int kSizeA = kM * kPitchK;
    constexpr int kSizeB = kTransposed ? kTile * kPitchK : kStep * kPitchN;
    constexpr int kBuffer = kPlanes * (kSizeA + kSizeB);
    constexpr int kOutPitch = 36;  // floats; a wave's 32 x 32 of y on its way out
    static_assert(kBuffers * kBuffer * 2 >= 4 * 32 * kOutPitch * 4);
    __shared__ __align__(16) short lds[kBuffers * kBuffer];

    uint32_t id = xcd_order(blockIdx.x, gridDim.x);
    const uint32_t part = id / (a.tiles_m * a.tiles_n);
    id -= part * (a.tiles_m * a.tiles_n);
    const uint32_t m0 = id % a.tiles_m * kM, n0 = id / a.tiles_m * kTile;
    const uint32_t end = min((part + 1) * a.per, a.cols);  // of the summed index
    const int t = threadIdx.x, lane = t & 63;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wm = kM == kTile ? wave / 2 * 64 : 0, wn = kM == kTile ? wave % 2 * 64 : wave * 32;
    const bool has_a = kM == kTile || wave < 2;

    // this lane's chunks of a step: of x (rows along the summed index), of W
    const uint32_t rk = t % 4 * 8, rr = t / 4;    // of 32 columns x 128 rows
    const uint32_t nn = t % 16 * 8, nk = t / 16;  // of 128 columns x 32 rows
    struct Loads {
        Chunk8<G> a[kChunksA], b[kChunks];
    };
    // Whole steps load without a branch: rows and columns past the end are any there are, as they only
    // reach sums that are not written; a row's last chunk of W as it is reaches into the next row,
    // where there is one.  (With a branch for each chunk of the tiles at the edges, whose loads then
    // wait for each other, 500 x 2176 x 4726 bf16 took 163 us, now 44.)
    const auto whole = [&](uint32_t k0) {
        return k0 + kStep <= end &&
               (kTransposed || a.outs % 8 == 0 || (a.outs >= 8 && k0 + kStep < a.cols));
    };
    const uint32_t column = n0 + nn < a.outs ? n0 + nn : 0;
    const auto load = [&](Loads& l, uint32_t k0) {
        if (whole(k0)) {
            if (has_a)
#pragma unroll
                for (int h = 0; h < kChunksA; ++h) {
                    const uint32_t m = min(m0 + rr + kRows * h, a.rows - 1);
                    l.a[h].load((const G*)a.x + m * a.x_stride + k0 + rk);
                }
#pragma unroll
            for (int h = 0; h < kChunks; ++h) {
                if constexpr (kTransposed)
                    l.b[h].load((const G*)a.w + min(n0 + rr + kRows * h, a.outs - 1) * a.w_stride +
                                k0 + rk);
                else
                    l.b[h].load((const G*)a.w + (k0 + nk + kRowsN * h) * a.w_stride + column);
            }
            return;
        }
        const uint32_t k = k0 + rk;
#pragma unroll
        for (int h = 0; h < kChunksA; ++h) {
            const uint32_t m = m0 + rr + kRows * h;
            load_upto8(l.a[h], (const G*)a.x + m * a.x_stride + k,
                       has_a && m < a.rows && k < end ? (int)min(end - k, 8u) : 0);
        }
#pragma unroll
        for (int h = 0; h < kChunks; ++h) {
            if constexpr (kTransposed) {
                const uint32_t n = n0 + rr + kRows * h;
                load_upto8(l.b[h], (const G*)a.w + n * a.w_stride + k,
                           n < a.outs && k < end ? (int)min(end - k, 8u) : 0);
            } else {
                const uint32_t n = n0 + nn, kb = k0 + nk + kRowsN * h;
                load_upto8(l.b[h], (const G*)a.w + kb * a.w_stride + n,
                           kb < end && n < a.outs ? (int)min(a.outs - n, 8u) : 0);
            }
        }
    };
    const auto store = [&](const Loads& l, short* buffer) {
        if (has_a)
#pragma unroll
            for (int h = 0; h < kChunksA; ++h) {
                u32x4 w[kPlanes];
                planes_of(l.a[h], w);
#pragma unroll
                for (int p = 0; p < kPlanes; ++p)
                    *reinterpret_cast<u32x4*>(buffer + p * kSizeA + (rr + kRows * h) * kPitchK +
                                              rk) = w[p];
            }
#pragma unroll
        for (int h = 0; h < kChunks; ++h) {
            u32x4 w[kPlanes];
            planes_of(l.b[h], w);
            short* b = buffer + kPlanes * kSizeA;
#pragma unroll
            for (int p = 0; p < kPlanes; ++p)
                *reinterpret_cast<u32x4*>(
                    b + p * kSizeB + (kTransposed ? (rr + kRows * h) * kPitchK + rk
                                                  : (nk + kRowsN * h) * kPitchN + nn)) = w[p];
        }
    };

    f32x16 acc[FA][FB];
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) acc[i][j] = f32x16{};
    const auto multiply = [&](const short* buffer) {
#pragma unroll
        for (int k = 0; k < (int)kStep; k += 16) {
            bf16x8 fa[kPlanes][FA], fb[kPlanes][FB];
#pragma unroll
            for (int p = 0; p < kPlanes; ++p) {
                const short* b = buffer + kPlanes * kSizeA + p * kSizeB;
#pragma unroll
                for (int i = 0; i < FA; ++i)
                    fa[p][i] = row_fragment(buffer + p * kSizeA, k, wm + 32 * i);
#pragma unroll
                for (int j = 0; j < FB; ++j)
                    fb[p][j] = kTransposed ? row_fragment(b, k, wn + 32 * j)
                                           : fragment(b, kPitchN, k, wn + 32 * j);
            }
            const auto products = [&](const bf16x8(&u)[FA], const bf16x8(&v)[FB]) {
#pragma unroll
                for (int i = 0; i < FA; ++i)
#pragma unroll
                    for (int j = 0; j < FB; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(u[i], v[j], acc[i][j],
                                                                            0, 0, 0);
            };
            products(fa[0], fb[0]);
            if constexpr (kPlanes == 3) {
#pragma unroll
                for (int i = 0; i < FA; ++i) fa[0][i] = finite(fa[0][i]);
#pragma unroll
                for (int j = 0; j < FB; ++j) fb[0][j] = finite(fb[0][j]);
                products(fa[0], fb[1]);
                products(fa[1], fb[0]);
                products(fa[0], fb[2]);
                products(fa[1], fb[1]);
                products(fa[2], fb[0]);
            }
        }
    };
    const uint32_t first = part * a.per, steps = (end - first + kStep - 1) / kStep;
    Loads l;
    load(l, first);
    if constexpr (kBuffers == 2) {
        store(l, lds);
        if (steps > 1) load(l, first + kStep);
        __syncthreads();
        for (uint32_t s = 0; s < steps; ++s) {
            multiply(lds + (s & 1) * kBuffer);
            if (s + 1 < steps) store(l, lds + ((s + 1) & 1) * kBuffer);
            if (s + 2 < steps) load(l, first + (s + 2) * kStep);
            __syncthreads();
        }
    } else {
        for (uint32_t s = 0; s < steps; ++s) {
            __syncthreads();  // the step before has been read
            store(l, lds);
            __syncthreads();
            if (s + 1 < steps) load(l, first + (s + 1) * kStep);
            multiply(lds);
        }
        __syncthreads();
    }

    // out, 32 x 32 at a time through this wave's LDS
    const uint64_t seed = a.has_dropout ? seed_of(a.dropout) : 0;
    float* out = reinterpret_cast<float*>(lds) + wave * 32 * kOutPitch;
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
        for (int j = 0; j < FB; ++j) {
#pragma unroll
            for (int k = 0; k < 16; ++k)
                out[(8 * (k / 4) + 4 * (lane >> 5) + k % 4) * kOutPitch + (lane & 31)] =
                    acc[i][j][k];
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int h = 0; h < 2; ++h) {
                const uint32_t r = lane / 4 + 16 * h, c = lane % 4 * 8;
                float v[8];
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const f32x4 w = *reinterpret_cast<const f32x4*>(out + r * kOutPitch + c + 4 * q);
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[4 * q + k] = w[k];
                }
                const uint32_t row = m0 + wm + 32 * i + r, col = n0 + wn + 32 * j + c;
                if (row >= a.rows || col >= a.outs) continue;
                if (a.parts > 1) {
                    put_part8(a, part, row, col, v);
                } else {
                    Chunk8<Y> res;
                    load_residual(a, row, col, res);
                    add_bias8<G>(a, col, v);
                    finish8<Y>(a, seed, row, col, v, res);
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
}

// ---- parts ------------------------------------------------------------------------------------
// The parts' sums in order, and what follows: a lane has 8 columns of a row.
constexpr int kJoinBlock = 256;
template <class G, class Y>
__global__ __launch_bounds__(kJoinBlock) void join_parts_kernel(LinearArgs a, uint32_t groups,
                                                                Divider by_groups) {
    const uint32_t i = blockIdx.x * kJoinBlock + threadIdx.x;
    if (i >= a.rows * groups) return;
    const uint32_t row = divide(i, by_groups), c = (i - row * groups) * 8;
    Chunk8<Y> res;
    load_residual(a, row, c, res);
    const uint64_t seed = a.has_dropout ? seed_of(a.dropout) : 0;
    const float* p = a.partial + (uint64_t)row * a.pitch + c;
    float v[8] = {};
#pragma unroll 4
    for (uint32_t k = 0; k < a.parts; ++k) {
        float w[8];
        load_cols(p + (uint64_t)k * a.rows * a.pitch, 0, 8, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] += w[j];
    }
    add_bias8<G>(a, c, v);
    finish8<Y>(a, seed, row, c, v, res);
}

// ---- launches ---------------------------------------------------------------------------------
int check_blocks(uint64_t blocks) {
    if (blocks < (1ull << 23)) return TTP_OK;  // (fewer than 2^32 work-items)
    return ttpi::fail(TTP_ERR_RANGE, "the product has too many tiles for one launch");
}

// f(blocks) launches the tiles of a product whose arguments are complete but for the parts' memory.
template <class G, class Y, class F>
int launch_parts(ttp_ctx* ctx, const ttpi::Op& op, LinearArgs& a, F&& f) {
    const uint64_t blocks = (uint64_t)a.tiles_m * a.tiles_n * a.parts;
    int rc = check_blocks(blocks);
    if (rc) return rc;
    if (a.parts > 1) {
        a.pitch = (a.outs + 7) / 8 * 8;
        void* ws;
        if ((rc = ttpi::workspace(ctx, (uint64_t)a.parts * a.rows * a.pitch * 4, &ws))) return rc;
        a.partial = (float*)ws;
    }
    (void)hipGetLastError();
    f((uint32_t)blocks);
    TTPI_HIP(hipGetLastError());
    if (a.parts > 1) {
        const uint32_t groups = (a.outs + 7) / 8, n = a.rows * groups;  // (parts: of few tiles)
        hipLaunchKernelGGL((join_parts_kernel<G, Y>), dim3((n + kJoinBlock - 1) / kJoinBlock),
                           dim3(kJoinBlock), 0, op.stream, a, groups, divider(groups));
        TTPI_HIP(hipGetLastError());
    }
    return TTP_OK;
}

// Whether the loads that go straight into the LDS may be used: whole 16-byte chunks on their grid,
// and a tile's rows within 31 bits of bytes.
bool on_grid(const LinearArgs& a, bool transposed) {
    return ((uintptr_t)a.x | (uintptr_t)a.w) % 16 == 0 && a.x_stride % 8 == 0 &&
           a.w_stride % 8 == 0 && a.cols % 8 == 0 && (transposed || a.outs % 8 == 0) &&
           a.x_stride < (1u << 22) && a.w_stride < (1u << 22);
}

template <class G, class Y, uint32_t kM>
void launch_any(bool transposed, uint32_t blocks, hipStream_t stream, const LinearArgs& a) {
    if (transposed)
        hipLaunchKernelGGL((linear_kernel<G, Y, true, kM>), dim3(blocks), dim3(kAnyThreads), 0, stream,
                           a);
    else
        hipLaunchKernelGGL((linear_kernel<G, Y, false, kM>), dim3(blocks), dim3(kAnyThreads), 0,
                           stream, a);
}

template <class G, class Y>
int multiply(ttp_ctx* ctx, const ttpi::Op& op, LinearArgs a, bool transposed) {
    constexpr bool kBf16 = sizeof(G) == 2;
    const bool direct = kBf16 && on_grid(a, transposed);
    const LinearCut cut = choose_linear_cut(a.rows, a.cols, a.outs, direct, kBf16, transposed,
                                            (uint64_t)op.num_cus);
    a.tiles_m = (uint32_t)(((uint64_t)a.rows + cut.tile_rows - 1) / cut.tile_rows);
    a.tiles_n = (uint32_t)(((uint64_t)a.outs + cut.tile_outs - 1) / cut.tile_outs);
    a.parts = cut.parts;
    a.per = cut.per;
    return launch_parts<G, Y>(ctx, op, a, [&](uint32_t blocks) {
        if (direct) {
            if (sizeof(Y) == 2)
                launch_direct_to_bf16(cut.shape, transposed, blocks, op.stream, a);
            else
                launch_direct_to_fp32(cut.shape, transposed, blocks, op.stream, a);
        } else if (cut.shape == LinearShape::kThinAny) {
            launch_any<G, Y, kThinRows>(transposed, blocks, op.stream, a);
        } else {
            launch_any<G, Y, kTile>(transposed, blocks, op.stream, a);
        }
    });
}

}  // namespace
}  // namespace ttp

using namespace ttp;
using ttpi::fail;

extern "C" int ttp_linear(ttp_ctx* ctx, const ttp_linear_args* args) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if (!args) return fail(TTP_ERR_INVALID, "null arguments");
        const ttp_matrix *x = args->x, *y = args->y, *res = args->residual;
        if (args->transposed != 0 && args->transposed != 1)
            return fail(TTP_ERR_INVALID, "transposed must be 0 or 1");
        if (args->activation < TTP_ACTIVATION_NONE || args->activation > TTP_ACTIVATION_GELU_TANH)
            return fail(TTP_ERR_INVALID, "activation must be a TTP_ACTIVATION_*");
        if (args->dropout && (rc = check_dropout(args->dropout))) return rc;
        if ((rc = ttpi::check_matrix(x, "the input"))) return rc;
        if ((rc = ttpi::check_matrix(y, "the output"))) return rc;
        const uint64_t rows = x->rows, cols = x->cols, outs = y->cols;
        const bool has_bias = args->bias != TTP_NO_TENSOR;
        ttpi::Param w{}, bias{};
        if ((rc = ttpi::param(ctx, args->weight, &w))) return rc;
        if (has_bias && (rc = ttpi::param(ctx, args->bias, &bias))) return rc;
        if (w.numel != cols * outs)
            return fail(TTP_ERR_RANGE, "tensor " + std::to_string(args->weight) + " has " +
                                           std::to_string(w.numel) + " elements, not " +
                                           std::to_string(cols) + " x " + std::to_string(outs));
        if (has_bias && bias.numel != outs)
            return fail(TTP_ERR_RANGE, "tensor " + std::to_string(args->bias) + " has " +
                                           std::to_string(bias.numel) + " elements, not " +
                                           std::to_string(outs));
        const bool bf16 = x->dtype == TTP_DTYPE_BF16;
        if (bf16 != w.bf16)
            return fail(TTP_ERR_INVALID, std::string("the input has another type than the weight (") +
                                             (w.bf16 ? "bfloat16" : "float32") + ")");
        ttpi::Buffers b(ctx);
        // (y may be the residual, but never what x is: other tiles read x's rows when one is written)
        if ((rc = b.matrix(x, rows, cols, "the input", false, nullptr, true))) return rc;
        if ((rc = b.own(w.data, w.numel, bf16 ? 2 : 4, "the weight", false))) return rc;
        if (has_bias && (rc = b.own(bias.data, outs, bf16 ? 2 : 4, "the bias", false))) return rc;
        if (res && (rc = b.matrix(res, rows, outs, "the residual", false))) return rc;
        if (args->dropout && args->dropout->device_seed &&
            (rc = b.array(args->dropout->device_seed, 1, 8, "the seed", false)))
            return rc;
        if ((rc = b.matrix(y, rows, outs, "the output", true, res))) return rc;
        if (res && res->dtype != y->dtype)
            return fail(TTP_ERR_INVALID, "the residual and the output have different types");
        if (!rows) return TTP_OK;
        LinearArgs a{};
        a.x = x->data;
        a.w = w.data;
        a.x_stride = x->stride;
        a.w_stride = args->transposed ? cols : outs;
        a.rows = (uint32_t)rows;
        a.cols = (uint32_t)cols;
        a.outs = (uint32_t)outs;
        a.bias = bias.data;
        a.activation = args->activation;
        a.has_dropout = args->dropout != nullptr;
        if (a.has_dropout) a.dropout = dropout_of(*args->dropout);
        a.residual = res ? res->data : nullptr;
        a.residual_stride = res ? res->stride : 0;
        a.y = y->data;
        a.y_stride = y->stride;
        const bool y16 = y->dtype == TTP_DTYPE_BF16;
        if (bf16)
            return y16 ? multiply<uint16_t, uint16_t>(ctx, op, a, args->transposed)
                       : multiply<uint16_t, float>(ctx, op, a, args->transposed);
        return y16 ? multiply<float, uint16_t>(ctx, op, a, args->transposed)
                   : multiply<float, float>(ctx, op, a, args->transposed);
    });
}
