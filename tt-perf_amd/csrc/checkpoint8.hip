// checkpoint8.hip — activations kept in 8 bits, restored, and GELU on them.
//
// A block of 32 columns of one row shares the scale 2^s, the least power of two with
// max |x| <= 127 2^s (int8) or 448 2^s (fp8 e4m3); v = x 2^-s is rounded to the grid of 8 bits.
// The power of two costs up to one bit of int8's range against a free scale, and buys that v 2^s
// is exact in bf16: the weight gradient's products take it without another rounding.
//
// All of it is bound by memory: 2 or 4 bytes read and 1.03 written per element (and back).  A
// lane has 8 columns, four lanes a block; the block's largest magnitude is an integer maximum of
// the bits without the sign (infinities and NaN are the largest of all) over the four lanes by
// two lane swaps.  Kept rows are padded to whole blocks, so their accesses are aligned and the
// backward's need no bounds within a block.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "checkpoint8.hpp"
#include "columns8.hpp"
#include "context.hpp"
#include "gelu.hpp"
#include "matrix.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

constexpr int kBlock8 = 256;

struct KeptArgs {
    uint8_t *values, *scales;
    uint32_t rows, cols, groups;  // groups of 8 columns per row (4 to a block)
    Divider by_groups;
};
struct Place {
    uint32_t row, col;
};
__device__ __forceinline__ Place place(const KeptArgs& a, uint32_t i) {
    const uint32_t row = divide(i, a.by_groups);
    return {row, (i - row * a.groups) * 8};
}

// ---- kernels ----------------------------------------------------------------------------------
enum Forward { kPack, kGeluErf, kGeluTanh };

// Lane i: 8 columns.  The four lanes of a block are neighbours (a row is whole blocks).  No loop: a
// launch has as many lanes as there are groups, so that every load of the launch can be in flight.
// Measured: 16384 x 1600 bf16 14.8 us, 5.4 TB/s; with GELU 8192 x 5120 bf16 34 us, 6.2 TB/s.
template <class T, int kFormat, Forward kWhat>
__global__ __launch_bounds__(kBlock8) void pack_kernel(const T* x, uint64_t x_stride, T* y,
                                                       uint64_t y_stride, KeptArgs a) {
    const uint32_t n = a.rows * a.groups, i = blockIdx.x * kBlock8 + threadIdx.x;
    if (i >= n) return;  // (n is a multiple of 4: whole blocks leave)
    const Place p = place(a, i);
    float v[8];
    load_cols(x + p.row * x_stride, p.col, a.cols, v);
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = max(top, __float_as_uint(v[k]) & 0x7FFFFFFFu);
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, true));
    top = max(top, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, true));
    const uint32_t scale = block_scale<kFormat>(top);
    const uint64_t at = (uint64_t)p.row * a.groups * 8 + p.col;
    *reinterpret_cast<u32x2*>(a.values + at) = encode8<kFormat>(v, scale);
    if ((i & 3) == 0) a.scales[at / 32] = (uint8_t)scale;
    if constexpr (kWhat != kPack) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = gelu<kWhat == kGeluTanh>(v[k]);
        store_cols(y + p.row * y_stride, p.col, a.cols, v);
    }
}

enum Backward { kRestore, kSlopeErf, kSlopeTanh };

// Lane i: 8 columns, as above.  Measured: 16384 x 1600 bf16 13.6 us, 5.8 TB/s; the GELU backward of
// 8192 x 5120 bf16 36.6 us, 5.8 TB/s.
template <class T, int kFormat, Backward kWhat>
__global__ __launch_bounds__(kBlock8) void unpack_kernel(KeptArgs a, const T* dy,
                                                         uint64_t dy_stride, T* dx,
                                                         uint64_t dx_stride) {
    const uint32_t n = a.rows * a.groups, i = blockIdx.x * kBlock8 + threadIdx.x;
    if (i >= n) return;
    const Place p = place(a, i);
    if (p.col >= a.cols) return;  // padding alone
    const uint64_t at = (uint64_t)p.row * a.groups * 8 + p.col;
    float v[8];
    decode8<kFormat>(*reinterpret_cast<const u32x2*>(a.values + at), a.scales[at / 32], v);
    if constexpr (kWhat != kRestore) {
        float g[8];
        load_cols(dy + p.row * dy_stride, p.col, a.cols, g);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = g[k] * gelu_slope<kWhat == kSlopeTanh>(v[k]);
    }
    store_cols(dx + p.row * dx_stride, p.col, a.cols, v);
}

// ---- launches ---------------------------------------------------------------------------------
// A launch covers fewer than 2^30 groups (Divider's range, and 2^32 work-items); longer ones are
// split by rows.  f(first row, rows' KeptArgs, grid)
template <class F>
int for_row_ranges(const ttp_checkpoint8& k, F&& f) {
    const uint32_t groups = (uint32_t)(kept_width(k.cols) / 8);
    const uint64_t most = std::max<uint64_t>((1u << 30) / groups, 1);
    for (uint64_t r = 0; r < k.rows; r += most) {
        const uint32_t rows = (uint32_t)std::min<uint64_t>(most, k.rows - r);
        KeptArgs a{(uint8_t*)k.values + r * groups * 8, (uint8_t*)k.scales + r * (groups / 4), rows,
                   (uint32_t)k.cols, groups, divider(groups)};
        const uint32_t grid = (rows * groups + kBlock8 - 1) / kBlock8;
        (void)hipGetLastError();
        f(r, a, dim3(grid));
        TTPI_HIP(hipGetLastError());
    }
    return TTP_OK;
}

template <class T, Forward kWhat>
int pack_rows(hipStream_t stream, const ttp_matrix& x, const ttp_matrix* y,
              const ttp_checkpoint8& k) {
    return for_row_ranges(k, [&](uint64_t r, const KeptArgs& a, dim3 grid) {
        const T* px = (const T*)x.data + r * x.stride;
        T* py = y ? (T*)y->data + r * y->stride : nullptr;
        const uint64_t ys = y ? y->stride : 0;
        if (k.format == TTP_CHECKPOINT_INT8)
            hipLaunchKernelGGL((pack_kernel<T, TTP_CHECKPOINT_INT8, kWhat>), grid, dim3(kBlock8),
                               0, stream, px, x.stride, py, ys, a);
        else
            hipLaunchKernelGGL((pack_kernel<T, TTP_CHECKPOINT_E4M3, kWhat>), grid, dim3(kBlock8),
                               0, stream, px, x.stride, py, ys, a);
    });
}

template <class T, Backward kWhat>
int unpack_rows(hipStream_t stream, const ttp_checkpoint8& k, const ttp_matrix* dy,
                const ttp_matrix& dx) {
    return for_row_ranges(k, [&](uint64_t r, const KeptArgs& a, dim3 grid) {
        const T* pg = dy ? (const T*)dy->data + r * dy->stride : nullptr;
        const uint64_t gs = dy ? dy->stride : 0;
        T* px = (T*)dx.data + r * dx.stride;
        if (k.format == TTP_CHECKPOINT_INT8)
            hipLaunchKernelGGL((unpack_kernel<T, TTP_CHECKPOINT_INT8, kWhat>), grid, dim3(kBlock8),
                               0, stream, a, pg, gs, px, dx.stride);
        else
            hipLaunchKernelGGL((unpack_kernel<T, TTP_CHECKPOINT_E4M3, kWhat>), grid, dim3(kBlock8),
                               0, stream, a, pg, gs, px, dx.stride);
    });
}

int check_approximate(int approximate) {
    if (approximate == TTP_GELU_ERF || approximate == TTP_GELU_TANH) return TTP_OK;
    return ttpi::fail(TTP_ERR_INVALID, "approximate must be TTP_GELU_ERF or TTP_GELU_TANH");
}
int check_same_type(const ttp_matrix* a, const ttp_matrix* b, const char* what) {
    if (a->dtype == b->dtype) return TTP_OK;
    return ttpi::fail(TTP_ERR_INVALID, std::string(what) + " have different types");
}

}  // namespace
}  // namespace ttp

using namespace ttp;

extern "C" {

int ttp_checkpoint8_pack(ttp_ctx* ctx, const ttp_matrix* x, const ttp_checkpoint8* kept) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = ttpi::check_matrix(x, "the activation"))) return rc;
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(x, x->rows, x->cols, "the activation", false))) return rc;
        if ((rc = check_kept(b, kept, x->rows, x->cols, true))) return rc;
        return x->dtype == TTP_DTYPE_BF16
                   ? pack_rows<uint16_t, kPack>(op.stream, *x, nullptr, *kept)
                   : pack_rows<float, kPack>(op.stream, *x, nullptr, *kept);
    });
}

int ttp_checkpoint8_restore(ttp_ctx* ctx, const ttp_checkpoint8* kept, const ttp_matrix* x) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = ttpi::check_matrix(x, "the activation"))) return rc;
        ttpi::Buffers b(ctx);
        if ((rc = check_kept(b, kept, x->rows, x->cols, false))) return rc;
        if ((rc = b.matrix(x, x->rows, x->cols, "the activation", true))) return rc;
        return x->dtype == TTP_DTYPE_BF16
                   ? unpack_rows<uint16_t, kRestore>(op.stream, *kept, nullptr, *x)
                   : unpack_rows<float, kRestore>(op.stream, *kept, nullptr, *x);
    });
}

int ttp_gelu_checkpoint8(ttp_ctx* ctx, const ttp_matrix* x, int approximate, const ttp_matrix* y,
                         const ttp_checkpoint8* kept) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = check_approximate(approximate))) return rc;
        if ((rc = ttpi::check_matrix(x, "the input"))) return rc;
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(x, x->rows, x->cols, "the input", false))) return rc;
        if ((rc = b.matrix(y, x->rows, x->cols, "the output", true, x))) return rc;
        if ((rc = check_same_type(x, y, "the input and the output"))) return rc;
        if ((rc = check_kept(b, kept, x->rows, x->cols, true))) return rc;
        const bool bf16 = x->dtype == TTP_DTYPE_BF16;
        if (approximate == TTP_GELU_TANH)
            return bf16 ? pack_rows<uint16_t, kGeluTanh>(op.stream, *x, y, *kept)
                        : pack_rows<float, kGeluTanh>(op.stream, *x, y, *kept);
        return bf16 ? pack_rows<uint16_t, kGeluErf>(op.stream, *x, y, *kept)
                    : pack_rows<float, kGeluErf>(op.stream, *x, y, *kept);
    });
}

int ttp_gelu_backward8(ttp_ctx* ctx, const ttp_checkpoint8* kept, int approximate,
                       const ttp_matrix* dy, const ttp_matrix* dx) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = check_approximate(approximate))) return rc;
        if ((rc = ttpi::check_matrix(dy, "the output's gradient"))) return rc;
        ttpi::Buffers b(ctx);
        if ((rc = check_kept(b, kept, dy->rows, dy->cols, false))) return rc;
        if ((rc = b.matrix(dy, dy->rows, dy->cols, "the output's gradient", false))) return rc;
        if ((rc = b.matrix(dx, dy->rows, dy->cols, "the input's gradient", true, dy))) return rc;
        if ((rc = check_same_type(dy, dx, "the gradients"))) return rc;
        const bool bf16 = dy->dtype == TTP_DTYPE_BF16;
        if (approximate == TTP_GELU_TANH)
            return bf16 ? unpack_rows<uint16_t, kSlopeTanh>(op.stream, *kept, dy, *dx)
                        : unpack_rows<float, kSlopeTanh>(op.stream, *kept, dy, *dx);
        return bf16 ? unpack_rows<uint16_t, kSlopeErf>(op.stream, *kept, dy, *dx)
                    : unpack_rows<float, kSlopeErf>(op.stream, *kept, dy, *dx);
    });
}

}  // extern "C"
