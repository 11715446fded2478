// dropout.hip — dropout from a counter-based generator, with a residual.
//
// Bound by memory, with the generator's operations close behind: a lane has one group of 8 columns,
// whose mask is one Philox call, so nothing of it is stored or read.  16384 x 1600 bf16 with a
// residual: 27 us, 5.9 TB/s; a copy of as many bytes that does not pass the caches reaches 6.7.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "columns8.hpp"
#include "context.hpp"
#include "dropout.hpp"
#include "matrix.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

constexpr int kDropoutBlock = 256;

struct DropoutArgs {
    Dropout d;
    uint64_t first_group;  // of the launch's first row
    uint32_t rows, cols, groups;
    Divider by_groups;
};

// Lane i: 8 columns.  y may be x or the residual: a lane reads its elements before it writes them.
template <class T, bool kResidual>
__global__ __launch_bounds__(kDropoutBlock) void dropout_kernel(const T* x, uint64_t x_stride,
                                                                const T* res, uint64_t res_stride,
                                                                T* y, uint64_t y_stride,
                                                                DropoutArgs a) {
    const uint32_t i = blockIdx.x * kDropoutBlock + threadIdx.x;
    if (i >= a.rows * a.groups) return;
    const uint32_t row = divide(i, a.by_groups), col = (i - row * a.groups) * 8;
    float v[8], r[8];
    load_cols(x + row * x_stride, col, a.cols, v);
    if constexpr (kResidual) load_cols(res + row * res_stride, col, a.cols, r);
    const u32x4 w = philox(seed_of(a.d), a.d.stream, a.first_group + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const bool keep = keeps(w, j, a.d.threshold);
        const float kept = v[j] * a.d.factor;
        if constexpr (kResidual)
            v[j] = keep ? r[j] + kept : r[j];
        else
            v[j] = keep ? kept : 0.0f;
    }
    store_cols(y + row * y_stride, col, a.cols, v);
}

// A launch covers fewer than 2^30 groups (Divider's range, and 2^32 work-items).
template <class T>
int dropout_rows(hipStream_t stream, const Dropout& d, const ttp_matrix& x, const ttp_matrix* res,
                 const ttp_matrix& y) {
    const uint32_t groups = (uint32_t)((x.cols + 7) / 8);
    const uint64_t most = std::max<uint64_t>((1u << 30) / groups, 1);
    for (uint64_t r = 0; r < x.rows; r += most) {
        const uint32_t rows = (uint32_t)std::min<uint64_t>(most, x.rows - r);
        const DropoutArgs a{d, r * groups, rows, (uint32_t)x.cols, groups, divider(groups)};
        const dim3 grid((rows * groups + kDropoutBlock - 1) / kDropoutBlock), block(kDropoutBlock);
        const T* px = (const T*)x.data + r * x.stride;
        T* py = (T*)y.data + r * y.stride;
        (void)hipGetLastError();
        if (res)
            hipLaunchKernelGGL((dropout_kernel<T, true>), grid, block, 0, stream, px, x.stride,
                               (const T*)res->data + r * res->stride, res->stride, py, y.stride, a);
        else
            hipLaunchKernelGGL((dropout_kernel<T, false>), grid, block, 0, stream, px, x.stride,
                               (const T*)nullptr, (uint64_t)0, py, y.stride, a);
        TTPI_HIP(hipGetLastError());
    }
    return TTP_OK;
}

}  // namespace
}  // namespace ttp

using namespace ttp;
using ttpi::fail;

extern "C" int ttp_dropout_forward(ttp_ctx* ctx, const ttp_dropout* dropout, const ttp_matrix* x,
                                   const ttp_matrix* residual, const ttp_matrix* y) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = check_dropout(dropout))) return rc;
        if ((rc = ttpi::check_matrix(x, "the input"))) return rc;
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(x, x->rows, x->cols, "the input", false))) return rc;
        if (residual && (rc = b.matrix(residual, x->rows, x->cols, "the residual", false)))
            return rc;
        if (dropout->device_seed && (rc = b.array(dropout->device_seed, 1, 8, "the seed", false)))
            return rc;
        const ttp_matrix* in_place = residual && y && y->data == residual->data ? residual : x;
        if ((rc = b.matrix(y, x->rows, x->cols, "the output", true, in_place))) return rc;
        if (x->dtype != y->dtype || (residual && residual->dtype != y->dtype))
            return fail(TTP_ERR_INVALID, "the input, the residual and the output have different types");
        const Dropout d = dropout_of(*dropout);
        return x->dtype == TTP_DTYPE_BF16 ? dropout_rows<uint16_t>(op.stream, d, *x, residual, *y)
                                          : dropout_rows<float>(op.stream, d, *x, residual, *y);
    });
}
