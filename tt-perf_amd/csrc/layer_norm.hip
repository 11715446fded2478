// layer_norm.hip — layer norm and its gradients.
//
//   m = mean x,  r = 1 / sqrt(mean (x - m)^2 + eps),  y = (x - m) r w + b
//   h = (x - m) r,  g = dy w,  dx = add + r (g - mean g - h mean(g h)),  dw = sum dy h,  db = sum dy
//
// Bound by memory.  A row of up to 1536 columns is a wave's, one of up to 8192 a block's of four or
// eight waves: it is read once, into registers, and its sums are taken there.  Longer rows are read
// again for each sum.  The backward keeps the weight's and the bias's sums of its rows in registers
// too: a block has a range of rows, writes one partial sum per column, and join_columns_kernel adds
// those up in order.
//
// Rows far from 0: a sum in fp32, rounded to the mean m', is off by some units of the mean, which in
// the variance and beside small deviations is much (1e4 with a deviation of 0.1: y 1e-2 off).  So the
// variance is that of the differences d = x - m', exact to their own unit, and what they still have
// in common, c = mean d, is taken off: m = m' + c, variance = mean d^2 - c^2, y from d - c (4e-7 off).
//
// bf16, us: 8192 x 1280 forward 10.8 and backward, with a gradient to add, 18.7 (4.5 TB/s) + 3.9;
// 16384 x 1600 27 and 40 (5.3 TB/s) + 4.8; 8192 x 1280 fp32 18 and 31 (5.4 TB/s) + 4.  At 1280 columns
// every row of 8192 is under way at once, from its loads to its stores; waves that take several rows
// with the next one's loads ahead (11.0), more of them to a CU (registers spill: 25) and four waves to
// a row (14.8 and 20.2) gave nothing.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "columns8.hpp"
#include "context.hpp"
#include "matrix.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

constexpr uint32_t kWaveCols = 512;  // columns of a wave's step: 8 a lane

// a vector of the store's parameters, or a constant
struct Vector {
    const void* data;  // null: every element is `otherwise`
    bool bf16;
    float otherwise;
};
__device__ __forceinline__ void load_vector(const Vector& p, uint32_t c, uint32_t cols,
                                            float (&v)[8]) {
    if (!p.data) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = p.otherwise;
    } else if (p.bf16) {
        load_cols((const uint16_t*)p.data, c, cols, v);
    } else {
        load_cols((const float*)p.data, c, cols, v);
    }
}

// the wave's sum in every lane, by a butterfly without LDS permutes (see wave_sum)
__device__ __forceinline__ double wave_total(double x) { return wave_sum(x); }
// (the steps within 32 lanes)
__device__ __forceinline__ float half_total(float x) {
    {
        const uint32_t u = __float_as_uint(x);
        const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
    const auto add = [&](uint32_t u) { x += __uint_as_float(u); };
    add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x128, 0xF, 0xF, true));
    add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x124, 0xF, 0xF, true));
    add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0x4E, 0xF, 0xF, true));
    add(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), 0xB1, 0xF, 0xF, true));
    return x;
}
// a's sum in the lower 32 lanes, b's in the upper: two sums for the steps of one
__device__ __forceinline__ float wave_totals(float a, float b) {
    const auto s =
        __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return half_total(__uint_as_float(s[0]) + __uint_as_float(s[1]));
}
__device__ __forceinline__ float wave_total(float x) { return wave_totals(x, x); }

// The sums of N numbers (fp32: one or two) over the kWaves waves of a row, in every lane.
template <int kWaves, int N, class F>
__device__ __forceinline__ void row_sums(F (&x)[N], F* lds) {
    constexpr bool kPair = N == 2 && sizeof(F) == 4;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    if constexpr (kPair) {
        x[0] = wave_totals(x[0], x[1]);
        if constexpr (kWaves == 1) {
            const int u = (int)__float_as_uint(x[0]);
            x[0] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(u, 0));
            x[1] = __uint_as_float((uint32_t)__builtin_amdgcn_readlane(u, 32));
        }
    } else {
#pragma unroll
        for (int n = 0; n < N; ++n) x[n] = wave_total(x[n]);
    }
    if constexpr (kWaves > 1) {
        __syncthreads();  // the last sums have been read
        if constexpr (kPair) {
            if (lane % 32 == 0) lds[wave * 2 + lane / 32] = x[0];
        } else if (lane == 0) {
#pragma unroll
            for (int n = 0; n < N; ++n) lds[wave * N + n] = x[n];
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < N; ++n) {
            F s = lds[n];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) s += lds[w * N + n];
            x[n] = s;
        }
    }
}

struct NormArgs {
    uint64_t rows;
    uint32_t cols;
    double eps;
    Vector weight, bias;
    const void *x, *in;  // in: dy of the backward
    const void* add;
    void* out;           // y or dx
    uint64_t x_stride, in_stride, add_stride, out_stride;
    float *mean, *rstd;
    float* parts;        // backward: per block the columns' sums of dy h, then those of dy
};

// ---- rows in registers ------------------------------------------------------------------------
// A lane's 8 columns of a step, from `first` on, of which the row's last lane may have fewer: it
// takes the row's last 8 and counts those from `at + j >= first` on, a lane behind the row's end
// none.  So every lane loads, without a branch, and the loads of a row are all under way before the
// first is used.  (Rows of fewer than 8 columns, kShort, are read one by one.)
struct Place8 {
    uint32_t first, at;
    __device__ __forceinline__ bool has(int j) const { return at + j >= first; }
};
__device__ __forceinline__ Place8 place8(uint32_t first, uint32_t cols) {
    return {first, min(first, max(cols, 8u) - 8)};
}
template <class T>
struct Raw8 {
    u32x4 w[sizeof(T) / 2];
    __device__ __forceinline__ void load(const T* p) {
#pragma unroll
        for (uint32_t k = 0; k < sizeof(T) / 2; ++k) w[k] = load16(p + k * kPer<T>);
    }
    __device__ __forceinline__ void load_some(const T* p, uint32_t n) {  // the first n, then 0
        float v[8];
        load_cols(p, 0, n, v);
#pragma unroll
        for (uint32_t k = 0; k < sizeof(T) / 2; ++k) {
            float q[kPer<T>];
#pragma unroll
            for (int j = 0; j < kPer<T>; ++j) q[j] = v[k * kPer<T> + j];
            w[k] = pack(q, p);
        }
    }
    __device__ __forceinline__ void values(float (&v)[8]) const {
#pragma unroll
        for (uint32_t k = 0; k < sizeof(T) / 2; ++k) {
            float q[kPer<T>];
            unpack(w[k], q, (const T*)nullptr);
#pragma unroll
            for (int j = 0; j < kPer<T>; ++j) v[k * kPer<T> + j] = q[j];
        }
    }
};
template <bool kShort, class T>
__device__ __forceinline__ void load_place(Raw8<T>& r, const T* row, Place8 p, uint32_t cols) {
    if constexpr (kShort)
        r.load_some(row, p.first ? 0u : cols);
    else
        r.load(row + p.at);
}
template <bool kShort, class T>
__device__ __forceinline__ void store_place(T* row, Place8 p, uint32_t cols, const float (&v)[8]) {
    if (!kShort && p.first + 8 <= cols) {
        store_cols(row, p.first, cols, v);
    } else if (p.first < cols) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (p.has(j) && p.at + j < cols) narrow(v[j], row + p.at + j);
    }
}
// The same of a vector of parameters (null: none).
template <bool kShort, class W>
__device__ __forceinline__ void load_param(Raw8<W>& r, const Vector& p, Place8 at, uint32_t cols) {
    if (p.data) load_place<kShort>(r, (const W*)p.data, at, cols);
}
template <class W>
__device__ __forceinline__ void param_values(const Raw8<W>& r, const Vector& p, float (&v)[8]) {
    if (p.data) {
        r.values(v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p.otherwise;
    }
}

// kWaves waves have a row of up to kC steps of 512 kWaves columns.
template <class T, class Y, class W, int kWaves, int kC, bool kShort>
__global__ __launch_bounds__(kWaves == 1 ? 256 : 64 * kWaves) void norm_kernel(NormArgs a) {
    __shared__ float lds[2 * kWaves];
    const uint32_t lane = kWaves == 1 ? threadIdx.x & 63 : threadIdx.x, cols = a.cols;
    const uint64_t row =
        kWaves == 1 ? (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (uint64_t)blockIdx.x;
    if (row >= a.rows) return;  // (a wave, or the block, together)
    const auto place = [&](int k) { return place8((k * 64 * kWaves + lane) * 8, cols); };
    const T* x = (const T*)a.x + row * a.x_stride;
    Raw8<T> raw[kC];
    Raw8<W> weight[kC], bias[kC];
#pragma unroll
    for (int k = 0; k < kC; ++k) load_place<kShort>(raw[k], x, place(k), cols);
#pragma unroll
    for (int k = 0; k < kC; ++k) load_param<kShort>(weight[k], a.weight, place(k), cols);
#pragma unroll
    for (int k = 0; k < kC; ++k) load_param<kShort>(bias[k], a.bias, place(k), cols);
    const float share = 1.0f / (float)cols;
    float v[kC][8];
    float s[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < kC; ++k) {
        raw[k].values(v[k]);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] += place(k).has(j) ? v[k][j] : 0.0f;
    }
    row_sums<kWaves>(s, lds);
    const float m = s[0] / (float)cols;
    float d[2] = {0.0f, 0.0f};  // the sums of the differences and of their squares
#pragma unroll
    for (int k = 0; k < kC; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const bool in = place(k).has(j) && (!kShort || j < (int)cols);
            v[k][j] = in ? v[k][j] - m : 0.0f;
            d[0] += v[k][j];
            d[1] = __builtin_fmaf(v[k][j], v[k][j], d[1]);
        }
    row_sums<kWaves>(d, lds);
    const float c = d[0] * share, var = __builtin_fmaf(-c, c, d[1] * share);
    const float r = 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + (float)a.eps);  // (NaN stays NaN)
    const float cr = c * r;
    if (lane == 0) {
        a.mean[row] = m + c;
        a.rstd[row] = r;
    }
    Y* y = (Y*)a.out + row * a.out_stride;
#pragma unroll
    for (int k = 0; k < kC; ++k) {
        float w[8], b[8];
        param_values(weight[k], a.weight, w);
        param_values(bias[k], a.bias, b);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            w[j] = __builtin_fmaf(__builtin_fmaf(v[k][j], r, -cr), w[j], b[j]);
        store_place<kShort>(y, place(k), cols, w);
    }
}

// Rows of this block: a wave each (kWaves 1), or all its waves' together; the next row's loads are
// under way while a row is worked on.  A row's x and dy stay in their own type and are widened again
// for dx, which leaves registers for that.
constexpr int kBackwardWaves = 8;
template <class T, class G, class W, int kWaves, int kC, bool kShort>
__global__ __launch_bounds__(64 * (kWaves == 1 ? kBackwardWaves : kWaves))
void norm_backward_kernel(NormArgs a, uint64_t per) {
    constexpr uint32_t kRows = kWaves == 1 ? kBackwardWaves : 1;  // at a time
    constexpr uint32_t kHalf = kRows / 2, kSums = kC * kWaveCols;
    __shared__ float lds[kWaves == 1 ? kHalf * 2 * kSums : 2 * kWaves];
    const uint32_t lane = kWaves == 1 ? threadIdx.x & 63 : threadIdx.x, cols = a.cols;
    const uint32_t wave = kWaves == 1 ? threadIdx.x >> 6 : 0;
    const uint64_t first = blockIdx.x * per, end = min(first + per, a.rows);
    const float n = (float)cols;
    const auto place = [&](int k) { return place8((k * 64 * kWaves + lane) * 8, cols); };
    struct Row {
        Raw8<T> x[kC];
        Raw8<G> dy[kC];
        float m, r;
    } next;
    const auto load_row = [&](uint64_t row) {
        next.m = a.mean[row];
        next.r = a.rstd[row];
#pragma unroll
        for (int k = 0; k < kC; ++k) {
            load_place<kShort>(next.x[k], (const T*)a.x + row * a.x_stride, place(k), cols);
            load_place<kShort>(next.dy[k], (const G*)a.in + row * a.in_stride, place(k), cols);
        }
    };
    if (first + wave < end) load_row(first + wave);
    Raw8<W> weight[kC];
    float sum_w[kC][8], sum_b[kC][8];
#pragma unroll
    for (int k = 0; k < kC; ++k) {
        load_param<kShort>(weight[k], a.weight, place(k), cols);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum_w[k][j] = sum_b[k][j] = 0.0f;
    }
    for (uint64_t row = first + wave; row < end; row += kRows) {
        const Row now = next;
        Raw8<T> add[kC];
        if (a.add)
#pragma unroll
            for (int k = 0; k < kC; ++k)
                load_place<kShort>(add[k], (const T*)a.add + row * a.add_stride, place(k), cols);
        if (row + kRows < end) load_row(row + kRows);
        // h and dy of step k, 0 where they are another lane's
        const auto widen_step = [&](int k, float(&h)[8], float(&g)[8]) {
            now.x[k].values(h);
            now.dy[k].values(g);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const bool in = place(k).has(j) && (!kShort || j < (int)cols);
                h[j] = in ? (h[j] - now.m) * now.r : 0.0f;
                g[j] = in ? g[j] : 0.0f;
            }
        };
        float s[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < kC; ++k) {
            float h[8], g[8], w[8];
            widen_step(k, h, g);
            param_values(weight[k], a.weight, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                sum_w[k][j] += g[j] * h[j];
                sum_b[k][j] += g[j];
                g[j] *= w[j];
                s[0] += g[j];
                s[1] += g[j] * h[j];
            }
        }
        row_sums<kWaves>(s, lds);
        const float mean_g = s[0] / n, mean_gh = s[1] / n;
        T* dx = (T*)a.out + row * a.out_stride;
#pragma unroll
        for (int k = 0; k < kC; ++k) {
            float h[8], g[8], w[8], o[8] = {};
            widen_step(k, h, g);
            param_values(weight[k], a.weight, w);
            if (a.add) add[k].values(o);
#pragma unroll
            for (int j = 0; j < 8; ++j)
                o[j] += now.r * (g[j] * w[j] - mean_g - h[j] * mean_gh);
            store_place<kShort>(dx, place(k), cols, o);
        }
    }
    // (a lane's sums are of its columns from Place8::at on; those of another lane are 0)
    float* part = a.parts + (uint64_t)blockIdx.x * 2 * cols;
    if constexpr (kWaves == 1) {  // one half of the waves' sums, the other half's added, then in order
#pragma unroll
        for (uint32_t half = 0; half < 2; ++half) {
            if (wave / kHalf == half)
#pragma unroll
                for (int k = 0; k < kC; ++k)
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        float* p = lds + (wave % kHalf) * 2 * kSums + (k * 8 + j) * 64 + lane;
                        p[0] = half ? p[0] + sum_w[k][j] : sum_w[k][j];
                        p[kSums] = half ? p[kSums] + sum_b[k][j] : sum_b[k][j];
                    }
            __syncthreads();
        }
        for (uint32_t c = threadIdx.x; c < cols; c += 64 * kRows) {
            // column c is its lane's j-th, counted from where that lane's 8 begin
            const uint32_t k = c / kWaveCols, l = c % kWaveCols / 8;
            const uint32_t j = c - place8(c / 8 * 8, cols).at;
            const float* p = lds + (k * 8 + j) * 64 + l;
            float w = p[0], b = p[kSums];
#pragma unroll
            for (uint32_t t = 1; t < kHalf; ++t) {
                w += p[t * 2 * kSums];
                b += p[t * 2 * kSums + kSums];
            }
            part[c] = w;
            part[cols + c] = b;
        }
    } else {
#pragma unroll
        for (int k = 0; k < kC; ++k)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const Place8 p = place(k);
                const uint32_t c = p.at + j;
                if (p.first < cols && p.has(j) && c < cols) {
                    part[c] = sum_w[k][j];
                    part[cols + c] = sum_b[k][j];
                }
            }
    }
}

// ---- rows that registers do not hold -----------------------------------------------------------
// A block per row, which reads it once for each sum and once more; the sums in 64 bits, the mean as
// fp32 and what its rounding left.
template <class T, class Y>
__global__ __launch_bounds__(256) void norm_long_kernel(NormArgs a) {
    __shared__ double lds[8];
    const uint64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    double s[1] = {0.0};
    for (uint64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
        float v[8];
        load_cols(x, (uint32_t)c, a.cols, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) s[0] += v[j];
    }
    row_sums<4>(s, lds);
    const float m = (float)(s[0] / a.cols), left = (float)(s[0] / a.cols - m);
    s[0] = 0.0;
    for (uint64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
        float v[8];
        load_cols(x, (uint32_t)c, a.cols, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = c + j < a.cols ? v[j] - m : 0.0f;
            s[0] += (double)d * d;
        }
    }
    row_sums<4>(s, lds);
    const double var = s[0] / a.cols - (double)left * left;
    const float r = (float)(1.0 / sqrt((var < 0.0 ? 0.0 : var) + a.eps)), left_r = left * r;
    if (threadIdx.x == 0) {
        a.mean[row] = m;
        a.rstd[row] = r;
    }
    Y* y = (Y*)a.out + row * a.out_stride;
    for (uint64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
        float v[8], w[8], b[8];
        load_cols(x, (uint32_t)c, a.cols, v);
        load_vector(a.weight, (uint32_t)c, a.cols, w);
        load_vector(a.bias, (uint32_t)c, a.cols, b);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            v[j] = __builtin_fmaf(__builtin_fmaf(v[j] - m, r, -left_r), w[j], b[j]);
        store_cols(y, (uint32_t)c, a.cols, v);
    }
}

// dx alone, behind the columns' sums: it may be written over what they read.
template <class T, class G>
__global__ __launch_bounds__(256) void norm_backward_long_kernel(NormArgs a) {
    __shared__ double lds[8];
    const uint64_t row = blockIdx.x;
    const T* x = (const T*)a.x + row * a.x_stride;
    const G* dy = (const G*)a.in + row * a.in_stride;
    const float m = a.mean[row], r = a.rstd[row];
    double s[2] = {0.0, 0.0};
    for (uint64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
        float h[8], g[8], w[8];
        load_cols(x, (uint32_t)c, a.cols, h);
        load_cols(dy, (uint32_t)c, a.cols, g);
        load_vector(a.weight, (uint32_t)c, a.cols, w);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float gw = c + j < a.cols ? g[j] * w[j] : 0.0f;
            s[0] += gw;
            s[1] += (double)gw * (c + j < a.cols ? (h[j] - m) * r : 0.0f);
        }
    }
    row_sums<4>(s, lds);
    const float mean_g = (float)(s[0] / a.cols), mean_gh = (float)(s[1] / a.cols);
    T* dx = (T*)a.out + row * a.out_stride;
    for (uint64_t c = threadIdx.x * 8; c < a.cols; c += 2048) {
        float h[8], g[8], w[8], o[8] = {};
        load_cols(x, (uint32_t)c, a.cols, h);
        load_cols(dy, (uint32_t)c, a.cols, g);
        load_vector(a.weight, (uint32_t)c, a.cols, w);
        if (a.add) load_cols((const T*)a.add + row * a.add_stride, (uint32_t)c, a.cols, o);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            o[j] += r * (g[j] * w[j] - mean_g - (h[j] - m) * r * mean_gh);
        store_cols(dx, (uint32_t)c, a.cols, o);
    }
}

// The columns' sums over a range of rows: 8 columns a lane.
template <class T, class G>
__global__ __launch_bounds__(256) void norm_columns_kernel(NormArgs a, uint64_t per) {
    const uint32_t tiles = (a.cols + 2047) / 2048, part = blockIdx.x / tiles;
    const uint64_t at = (uint64_t)(blockIdx.x % tiles) * 2048 + threadIdx.x * 8;
    if (at >= a.cols) return;
    const uint32_t c = (uint32_t)at;
    const uint64_t end = min((part + 1) * per, a.rows);
    float sum_w[8] = {}, sum_b[8] = {};
    for (uint64_t row = part * per; row < end; ++row) {
        float h[8], g[8];
        load_cols((const T*)a.x + row * a.x_stride, c, a.cols, h);
        load_cols((const G*)a.in + row * a.in_stride, c, a.cols, g);
        const float m = a.mean[row], r = a.rstd[row];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            sum_w[j] += g[j] * ((h[j] - m) * r);
            sum_b[j] += g[j];
        }
    }
    float* p = a.parts + (uint64_t)part * 2 * a.cols + c;
#pragma unroll
    for (int j = 0; j < 8; ++j)
        if (c + j < a.cols) {
            p[j] = sum_w[j];
            p[a.cols + j] = sum_b[j];
        }
}

// ---- the parts' sums into the gradients -------------------------------------------------------
struct JoinArgs {
    const float* parts;
    uint32_t n, cols;      // parts; columns
    void *dw, *db;         // null: no such tensor
    bool bf16, dw_first, db_first;
};
__device__ __forceinline__ void put(void* p, bool bf16, bool first, uint32_t c, float v) {
    if (bf16) {
        uint16_t* q = (uint16_t*)p + c;
        narrow(first ? v : widen(*q) + v, q);
    } else {
        float* q = (float*)p + c;
        *q = first ? v : *q + v;
    }
}
// 64 columns of a block (the bias's behind the weight's), whose 16 waves have the parts in turn.
__global__ __launch_bounds__(1024) void join_columns_kernel(JoinArgs a) {
    __shared__ float lds[16][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t c = (uint64_t)blockIdx.x * 64 + lane, all = 2ull * a.cols;
    const uint32_t per = (a.n + 15) / 16, end = min((wave + 1) * per, a.n);
    const float* p = a.parts + min(c, all - 1);
    float v = 0.0f;
    uint32_t k = wave * per;
    for (; k + 8 <= end; k += 8) {
        float w[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j] = p[(k + j) * all];
#pragma unroll
        for (int j = 0; j < 8; ++j) v += w[j];
    }
    for (; k < end; ++k) v += p[k * all];
    lds[wave][lane] = v;
    __syncthreads();
    if (wave || c >= all) return;
#pragma unroll
    for (int w = 1; w < 16; ++w) v += lds[w][lane];
    if (c < a.cols) {
        if (a.dw) put(a.dw, a.bf16, a.dw_first, (uint32_t)c, v);
    } else if (a.db) {
        put(a.db, a.bf16, a.db_first, (uint32_t)(c - a.cols), v);
    }
}

// ---- launches ---------------------------------------------------------------------------------
constexpr uint32_t kLongCols = 8192;  // rows longer than that are not kept in registers
constexpr uint64_t kMostCols = 1u << 24;

// f(waves of a row, steps, whether it is short): the shape that holds a row of `cols` <= kLongCols
template <class F>
void with_shape(uint32_t cols, F&& f) {
    using std::integral_constant;
    if (cols < 8)
        f(integral_constant<int, 1>(), integral_constant<int, 1>(), std::true_type());
    else if (cols <= kWaveCols)
        f(integral_constant<int, 1>(), integral_constant<int, 1>(), std::false_type());
    else if (cols <= 2 * kWaveCols)
        f(integral_constant<int, 1>(), integral_constant<int, 2>(), std::false_type());
    else if (cols <= 3 * kWaveCols)
        f(integral_constant<int, 1>(), integral_constant<int, 3>(), std::false_type());
    else if (cols <= 4 * kWaveCols)
        f(integral_constant<int, 4>(), integral_constant<int, 1>(), std::false_type());
    else if (cols <= 8 * kWaveCols)
        f(integral_constant<int, 8>(), integral_constant<int, 1>(), std::false_type());
    else
        f(integral_constant<int, 8>(), integral_constant<int, 2>(), std::false_type());
}

// A launch has fewer than 2^32 work-items: f(first row, rows) over ranges of rows.
template <class F>
int for_row_ranges(uint64_t rows, F&& f) {
    constexpr uint64_t kMost = (1u << 23) - 8;  // of up to 512 lanes each
    for (uint64_t r = 0; r < rows; r += kMost) {
        (void)hipGetLastError();
        f(r, std::min(kMost, rows - r));
        TTPI_HIP(hipGetLastError());
    }
    return TTP_OK;
}
// The arguments of the rows from r on.
template <class T, class In, class Out>
NormArgs from_row(NormArgs a, uint64_t r, uint64_t rows) {
    a.rows = rows;
    a.x = (const T*)a.x + r * a.x_stride;
    if (a.in) a.in = (const In*)a.in + r * a.in_stride;
    if (a.add) a.add = (const T*)a.add + r * a.add_stride;
    a.out = (Out*)a.out + r * a.out_stride;
    a.mean += r;
    a.rstd += r;
    return a;
}

template <class T, class Y, class W>
int norm_rows(const ttpi::Op& op, const NormArgs& all) {
    return for_row_ranges(all.rows, [&](uint64_t r, uint64_t rows) {
        const NormArgs a = from_row<T, T, Y>(all, r, rows);
        if (a.cols > kLongCols) {
            hipLaunchKernelGGL((norm_long_kernel<T, Y>), dim3((uint32_t)rows), dim3(256), 0,
                               op.stream, a);
            return;
        }
        with_shape(a.cols, [&](auto waves, auto steps, auto is_short) {
            const uint64_t blocks = waves == 1 ? (rows + 3) / 4 : rows;
            hipLaunchKernelGGL((norm_kernel<T, Y, W, waves(), steps(), is_short()>),
                               dim3((uint32_t)blocks), dim3(waves == 1 ? 256 : 64 * waves), 0,
                               op.stream, a);
        });
    });
}

// The parts that the columns' sums are taken in, and the rows of each.
struct Parts {
    uint32_t n;
    uint64_t per;
};
Parts parts_of(const ttpi::Op& op, uint64_t rows, uint32_t cols) {
    uint64_t n, step = 1;
    if (cols > kLongCols) {
        const uint64_t tiles = ((uint64_t)cols + 2047) / 2048;
        n = std::max<uint64_t>(4 * (uint64_t)op.num_cus / tiles, 1);
    } else if (cols > 3 * kWaveCols) {
        // blocks that a CU's registers hold; 4096 x 5120 bf16 with one to a CU 39 us, two 46, four 58;
        // 8192 x 2560 with two 35, three 38; 16384 x 1600 with two 43, four 40
        n = (cols > 8 * kWaveCols ? 1 : cols > 4 * kWaveCols ? 2 : 4) * (uint64_t)op.num_cus;
    } else {
        n = (uint64_t)op.num_cus;
        step = kBackwardWaves;  // a row for each of the block's waves
    }
    const uint64_t per = std::max<uint64_t>((rows + n - 1) / n, 1);
    const uint64_t whole = (per + step - 1) / step * step;
    return {(uint32_t)((rows + whole - 1) / whole), whole};
}

template <class T, class G, class W>
int norm_backward_rows(const ttpi::Op& op, const NormArgs& a, const Parts& p) {
    (void)hipGetLastError();
    if (a.cols > kLongCols) {
        const uint32_t tiles = (a.cols + 2047) / 2048;
        hipLaunchKernelGGL((norm_columns_kernel<T, G>), dim3(p.n * tiles), dim3(256), 0, op.stream,
                           a, p.per);
        TTPI_HIP(hipGetLastError());
        const int rc = for_row_ranges(a.rows, [&](uint64_t r, uint64_t rows) {
            hipLaunchKernelGGL((norm_backward_long_kernel<T, G>), dim3((uint32_t)rows), dim3(256),
                               0, op.stream, (from_row<T, G, T>(a, r, rows)));
        });
        if (rc) return rc;
    } else {
        with_shape(a.cols, [&](auto waves, auto steps, auto is_short) {
            hipLaunchKernelGGL((norm_backward_kernel<T, G, W, waves(), steps(), is_short()>),
                               dim3(p.n), dim3(64 * (waves == 1 ? kBackwardWaves : waves())), 0,
                               op.stream, a, p.per);
        });
    }
    TTPI_HIP(hipGetLastError());
    return TTP_OK;
}

// f(a value of x's type, of y's or dy's, of the parameters')
template <class F>
int with_types(int x, int y, bool params_bf16, F&& f) {
    const uint16_t h = 0;
    const float s = 0.0f;
    const auto with_params = [&](auto t, auto g) {
        return params_bf16 ? f(t, g, h) : f(t, g, s);
    };
    if (x == TTP_DTYPE_BF16)
        return y == TTP_DTYPE_BF16 ? with_params(h, h) : with_params(h, s);
    return y == TTP_DTYPE_BF16 ? with_params(s, h) : with_params(s, s);
}

int check_cols(uint64_t cols) {
    if (cols <= kMostCols) return TTP_OK;
    return ttpi::fail(TTP_ERR_RANGE, "layer norm takes rows of at most 2^24 columns");
}

// A weight or bias of `cols` elements (or none), to be read.
int vector_param(ttp_ctx* ctx, ttpi::Buffers& b, uint32_t index, uint64_t cols, float otherwise,
                 const char* what, Vector* out) {
    *out = {nullptr, false, otherwise};
    if (index == TTP_NO_TENSOR) return TTP_OK;
    ttpi::Param p{};
    int rc = ttpi::param(ctx, index, &p);
    if (rc) return rc;
    if (p.numel != cols)
        return ttpi::fail(TTP_ERR_RANGE, "tensor " + std::to_string(index) + " has " +
                                             std::to_string(p.numel) + " elements, not " +
                                             std::to_string(cols));
    *out = {p.data, p.bf16, otherwise};
    return b.own(p.data, cols, p.bf16 ? 2 : 4, what, false);
}

}  // namespace
}  // namespace ttp

using namespace ttp;
using ttpi::fail;

extern "C" {

int ttp_layer_norm(ttp_ctx* ctx, uint32_t weight, uint32_t bias, const ttp_matrix* x, double eps,
                   const ttp_matrix* y, float* mean, float* rstd) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if (!(eps >= 0.0 && eps <= 1e30)) return fail(TTP_ERR_INVALID, "eps must be 0 or more");
        if ((rc = ttpi::check_matrix(x, "the input"))) return rc;
        const uint64_t rows = x->rows, cols = x->cols;
        if ((rc = check_cols(cols))) return rc;
        NormArgs a{};
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(x, rows, cols, "the input", false))) return rc;
        if ((rc = vector_param(ctx, b, weight, cols, 1.0f, "the weight", &a.weight))) return rc;
        if ((rc = vector_param(ctx, b, bias, cols, 0.0f, "the bias", &a.bias))) return rc;
        if ((rc = b.matrix(y, rows, cols, "the output", true, x))) return rc;
        if ((rc = b.array(mean, rows, 4, "the means", true))) return rc;
        if ((rc = b.array(rstd, rows, 4, "the reciprocal deviations", true))) return rc;
        if (!rows) return TTP_OK;
        a.rows = rows;
        a.cols = (uint32_t)cols;
        a.eps = eps;
        a.x = x->data;
        a.x_stride = x->stride;
        a.out = y->data;
        a.out_stride = y->stride;
        a.mean = mean;
        a.rstd = rstd;
        return with_types(x->dtype, y->dtype, a.weight.bf16 || a.bias.bf16,
                          [&](auto t, auto g, auto w) {
                              return norm_rows<decltype(t), decltype(g), decltype(w)>(op, a);
                          });
    });
}

int ttp_layer_norm_backward(ttp_ctx* ctx, uint32_t weight, uint32_t bias, const ttp_matrix* x,
                            const ttp_matrix* dy, const float* mean, const float* rstd,
                            const ttp_matrix* add, const ttp_matrix* dx) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = ttpi::check_matrix(x, "the input"))) return rc;
        const uint64_t rows = x->rows, cols = x->cols;
        if ((rc = check_cols(cols))) return rc;
        const bool has_weight = weight != TTP_NO_TENSOR, has_bias = bias != TTP_NO_TENSOR;
        if (has_weight && weight == bias)
            return fail(TTP_ERR_INVALID, "the weight and the bias are the same tensor");
        ttpi::GradTarget w{}, s{};
        if (has_weight && (rc = ttpi::grad_target(ctx, weight, &w))) return rc;
        if (has_bias && (rc = ttpi::grad_target(ctx, bias, &s))) return rc;
        NormArgs a{};
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(x, rows, cols, "the input", false))) return rc;
        if ((rc = b.matrix(dy, rows, cols, "the output's gradient", false))) return rc;
        if (add && (rc = b.matrix(add, rows, cols, "the gradient to add", false))) return rc;
        if ((rc = b.array(mean, rows, 4, "the means", false))) return rc;
        if ((rc = b.array(rstd, rows, 4, "the reciprocal deviations", false))) return rc;
        Vector ignored;
        if ((rc = vector_param(ctx, b, weight, cols, 1.0f, "the weight", &a.weight))) return rc;
        if ((rc = vector_param(ctx, b, bias, cols, 0.0f, "the bias", &ignored))) return rc;
        const uint64_t size = w.bf16 || s.bf16 ? 2 : 4;
        if (has_weight && (rc = b.own(w.data, cols, size, "the weight's gradient", true)))
            return rc;
        if (has_bias && (rc = b.own(s.data, cols, size, "the bias's gradient", true))) return rc;
        const ttp_matrix* place = !dx                            ? x
                                  : add && dx->data == add->data ? add
                                  : dy->data == dx->data         ? dy
                                                                 : x;
        if ((rc = b.matrix(dx, rows, cols, "the input's gradient", true, place))) return rc;
        if (dx->dtype != x->dtype || (add && add->dtype != x->dtype))
            return fail(TTP_ERR_INVALID,
                        "the input, its gradient and the gradient to add have different types");
        a.rows = rows;
        a.cols = (uint32_t)cols;
        a.x = x->data;
        a.x_stride = x->stride;
        a.in = dy->data;
        a.in_stride = dy->stride;
        a.add = add ? add->data : nullptr;
        a.add_stride = add ? add->stride : 0;
        a.out = dx->data;
        a.out_stride = dx->stride;
        a.mean = const_cast<float*>(mean);
        a.rstd = const_cast<float*>(rstd);
        const Parts p = parts_of(op, rows, a.cols);
        void* ws = nullptr;
        if (p.n && (rc = ttpi::workspace(ctx, (uint64_t)p.n * 2 * cols * 4, &ws))) return rc;
        a.parts = (float*)ws;
        if (p.n) {
            rc = with_types(x->dtype, dy->dtype, a.weight.bf16, [&](auto t, auto g, auto w) {
                return norm_backward_rows<decltype(t), decltype(g), decltype(w)>(op, a, p);
            });
            if (rc) return rc;
        }
        if (has_weight || has_bias) {
            const JoinArgs j{a.parts, p.n, a.cols, w.data, s.data, size == 2, w.first, s.first};
            const uint32_t blocks = (uint32_t)((2 * cols + 63) / 64);
            (void)hipGetLastError();
            hipLaunchKernelGGL(join_columns_kernel, dim3(blocks), dim3(1024), 0, op.stream, j);
            TTPI_HIP(hipGetLastError());
        }
        if (has_weight) ttpi::grad_written(ctx, weight);
        if (has_bias) ttpi::grad_written(ctx, bias);
        return TTP_OK;
    });
}

}  // extern "C"
