// losses.hip — token log-probabilities, the preference loss and the clipped policy loss, with the
// logits' gradient.
//
// With z a row of logits, y its token, m = max z and s = sum exp(z - m):
//   logp = (z_y - m) - log s,   p_v = exp(z_v - m) / s,   dlogp/dz_v = [v = y] - p_v
// so a loss that is a function of the rows' logp gives dz_v = c ([v = y] - p_v) with one number c
// per row.  Everything is bound by the logits: they are read once (twice where c depends on other
// rows) and the gradient is written once; the arithmetic is about ten VALU operations and two
// exponentials per logit.
//
//   row_scores_kernel   (m, s) of each row in one pass with a running maximum, then logp and the
//                       row's part of the loss.  Few rows are split over the vocabulary and
//                       joined by the launch's last block.
//   pair_losses_kernel  sums over sequences, the pairs' losses, the rows' c (preference)
//   row_sums_kernel     sums of the rows' losses and the number of rows that count (policy)
//   row_grads_kernel    the gradient from (m, s, c)
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "context.hpp"
#include "device.hpp"
#include "matrix.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

// ---- (maximum, sum of exponentials) ---------------------------------------------------------
struct Stat {
    float m, s;  // s = sum exp(z - m); nothing yet: (-inf, 0)
};
// What the exponents are taken from: an all -inf part has the sum 0, not exp(-inf + inf).
__device__ __forceinline__ float stat_base(float m) { return m == -INFINITY ? 0.0f : m; }

__device__ __forceinline__ Stat join(Stat a, Stat b) {
    const float m = fmaxf(a.m, b.m), base = stat_base(m);
    return {m, a.s * exp2_fast((a.m - base) * kLog2e) + b.s * exp2_fast((b.m - base) * kLog2e)};
}
template <int N>
__device__ __forceinline__ Stat join(Stat a, const float (&v)[N]) {
    float m = a.m;
#pragma unroll
    for (int k = 0; k < N; ++k) m = fmaxf(m, v[k]);  // (skips NaN, which the sum then holds)
    const float base = stat_base(m);
    float s = a.s * exp2_fast((a.m - base) * kLog2e);
#pragma unroll
    for (int k = 0; k < N; ++k) s += exp2_fast((v[k] - base) * kLog2e);
    return {m, s};
}
__device__ __forceinline__ Stat shfl_xor(Stat a, int off) {
    return {__shfl_xor(a.m, off), __shfl_xor(a.s, off)};
}
// The block's, in every lane of it.
template <int kThreads>
__device__ __forceinline__ Stat block_join(Stat a, Stat* lds) {
#pragma unroll
    for (int off = 32; off; off >>= 1) a = join(a, shfl_xor(a, off));
    if constexpr (kThreads > 64) {
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
        __syncthreads();
        a = lds[0];
#pragma unroll
        for (int w = 1; w < kThreads / 64; ++w) a = join(a, lds[w]);
        __syncthreads();
    }
    return a;
}

// ---- a row's part of the loss ---------------------------------------------------------------
enum Loss { kScore, kPreference, kPolicy };

struct RowArgs {
    const void* z;
    uint64_t rows, stride;
    uint32_t cols;
    const int64_t* targets;
    float* logps;
    // preference: the row's part of its sequence's sum, its statistics and its c (set to 0 here,
    // by pair_losses_kernel where a sequence covers the row)
    const float* ref;
    double* part;
    Stat* stats;
    float* coef;
    // policy: part is the row's loss, part_kl its k
    const float *old, *adv;
    double* part_kl;
    float clip_lo, clip_hi, kl_coef;
};

template <class T>
__device__ __forceinline__ float row_logp(const RowArgs& a, uint64_t row, int64_t y, Stat st) {
    if (y < 0) return 0.0f;
    if (y >= (int64_t)a.cols) return NAN;
    const float zy = widen(((const T*)a.z)[row * a.stride + (uint64_t)y]);
    return (zy - st.m) - logf(st.s);
}

struct PolicyRow {
    float loss, kl, coef;
};
// One row's loss, k and c = dloss/dlogp (each before the division by D), once per row, in fp32:
// their sums are in fp64.
__device__ __forceinline__ PolicyRow policy_row(const RowArgs& a, uint64_t row, float logp) {
    const float r = expf(logp - a.old[row]), adv = a.adv[row];
    const float held = r < a.clip_lo ? a.clip_lo : r > a.clip_hi ? a.clip_hi : r;
    const float plain = r * adv, clipped = held * adv;
    PolicyRow o;
    // the smaller one; a NaN of either is the loss's, and the gradient's
    const bool free = plain <= clipped || plain != plain;
    o.loss = -(free ? plain : clipped);
    o.coef = free ? -plain : clipped != clipped ? clipped : 0.0f;
    o.kl = 0.0f;
    if (a.ref) {
        const float g = a.ref[row] - logp, e = expm1f(g);
        o.kl = e - g;
        if (a.kl_coef != 0.0f) {
            o.loss += a.kl_coef * o.kl;
            o.coef -= a.kl_coef * e;
        }
    }
    return o;
}

// One lane, once the row's statistics are whole.
template <class T, Loss kLoss>
__device__ __forceinline__ void finish_row(const RowArgs& a, uint64_t row, Stat st) {
    const int64_t y = a.targets[row];
    const float logp = row_logp<T>(a, row, y, st);
    a.logps[row] = logp;
    if constexpr (kLoss == kPreference) {
        a.part[row] = y < 0 ? 0.0 : (double)logp - (a.ref ? (double)a.ref[row] : 0.0);
        a.stats[row] = st;
        a.coef[row] = 0.0f;
    } else if constexpr (kLoss == kPolicy) {
        PolicyRow p = {0.0f, 0.0f, 0.0f};
        if (y >= 0) p = policy_row(a, row, logp);
        a.part[row] = (double)p.loss;
        a.part_kl[row] = (double)p.kl;
        a.stats[row] = st;
        a.coef[row] = p.coef;
    }
}

// ---- row_scores_kernel ------------------------------------------------------------------------
constexpr int kRowBlock = 256;
constexpr int kAhead = 4;  // 16-byte loads in flight per lane

// The statistics of z[lo, hi) (each lane its share); hi - lo a whole number of 16-byte chunks but
// for the row's last part.
template <class T, int kThreads>
__device__ __forceinline__ Stat part_stats(const T* z, uint32_t lo, uint32_t hi) {
    constexpr int P = kPer<T>;
    const uint32_t chunks = (hi - lo) / P;
    Stat st = {-INFINITY, 0.0f};
    uint32_t c = threadIdx.x;
    for (; c + (kAhead - 1) * kThreads < chunks; c += kAhead * kThreads) {
        u32x4 w[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) w[k] = load16(z + lo + (uint64_t)(c + k * kThreads) * P);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            float v[P];
            unpack(w[k], v, z);
            st = join(st, v);
        }
    }
    for (; c < chunks; c += kThreads) {
        float v[P];
        unpack(load16(z + lo + (uint64_t)c * P), v, z);
        st = join(st, v);
    }
    const uint32_t at = lo + chunks * P + threadIdx.x;
    if (at < hi) {
        const float v[1] = {widen(z[at])};
        st = join(st, v);
    }
    return st;
}

// Block b: part b % splits of row b / splits (b + k gridDim.x: of a further row).  splits > 1:
// every block has one item, and the launch's last block joins the parts of all rows.
template <class T, Loss kLoss>
__global__ __launch_bounds__(kRowBlock) void row_scores_kernel(RowArgs a, uint32_t splits,
                                                               uint32_t per, double* parts,
                                                               uint32_t* tickets) {
    __shared__ Stat lds[kRowBlock / 64];
    __shared__ uint32_t last;
    const uint64_t items = a.rows * splits;
    for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const uint64_t row = i / splits;
        const uint32_t part = (uint32_t)(i - row * splits);
        Stat st = {-INFINITY, 0.0f};
        if (a.targets[row] >= 0) {  // a masked row's logits are not read
            const uint32_t lo = part * per;
            const uint32_t hi = part + 1 == splits ? a.cols : lo + per;
            st = part_stats<T, kRowBlock>((const T*)a.z + row * a.stride, lo, hi);
            st = block_join<kRowBlock>(st, lds);
        }
        if (threadIdx.x == 0) {
            if (splits == 1)
                finish_row<T, kLoss>(a, row, st);
            else
                st_device(parts + i, __builtin_bit_cast(double, st));
        }
    }
    if (splits == 1 || !is_last_block(tickets, &last)) return;
    // `lanes` lanes per row (a power of two, at most a wave), each one part
    uint32_t lanes = 1;
    while (lanes < splits) lanes *= 2;
    const uint32_t p = threadIdx.x % lanes, step = kRowBlock / lanes;
    for (uint64_t base = 0; base < a.rows; base += step) {
        const uint64_t row = base + threadIdx.x / lanes;
        Stat st = {-INFINITY, 0.0f};
        if (row < a.rows && p < splits)
            st = __builtin_bit_cast(Stat, ld_device(parts + row * splits + p));
        for (uint32_t off = lanes / 2; off; off >>= 1) st = join(st, shfl_xor(st, (int)off));
        if (row < a.rows && p == 0) finish_row<T, kLoss>(a, row, st);
    }
}

// ---- pair_losses_kernel -----------------------------------------------------------------------
struct PairArgs {
    const int64_t* starts;
    uint64_t rows, pairs;
    const double* part;
    double* pair_loss;
    float beta, smoothing;
    const float* loss_scale;
    float *coef, *margins, *loss;
};
__device__ __forceinline__ uint64_t bounded(int64_t x, uint64_t lo, uint64_t hi) {
    return x < (int64_t)lo ? lo : (uint64_t)x > hi ? hi : (uint64_t)x;
}
// log(1 + exp(x))
__device__ __forceinline__ double softplus(double x) {
    return fmax(x, 0.0) + log1p(exp(-fabs(x)));
}

// Block p: pair p.  Sums in fp64 (a margin is the small difference of sums over hundreds of
// tokens), each lane's share in row order, then the block's lanes in a fixed order.
__global__ __launch_bounds__(kBlock) void pair_losses_kernel(PairArgs a, uint32_t* tickets) {
    __shared__ double lds[kBlock / 64];
    __shared__ uint32_t last;
    __shared__ float c;
    const uint64_t p = blockIdx.x;
    uint64_t lo[2], hi[2];
    double d[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const uint64_t s = p + k * a.pairs;
        lo[k] = bounded(a.starts[s], 0, a.rows);
        hi[k] = bounded(a.starts[s + 1], lo[k], a.rows);
        double x = 0.0;
        for (uint64_t t = lo[k] + threadIdx.x; t < hi[k]; t += kBlock) x += a.part[t];
        d[k] = block_sum(x, lds);
    }
    if (threadIdx.x == 0) {
        const double eps = (double)a.smoothing, h = (double)a.beta * (d[0] - d[1]);
        a.margins[p] = (float)h;
        st_device(a.pair_loss + p, (1.0 - eps) * softplus(-h) + eps * softplus(h));
        // (each sigmoid by itself: their difference would lose the small one)
        const double dh = eps / (1.0 + exp(-h)) - (1.0 - eps) / (1.0 + exp(h));
        const double scale = a.loss_scale ? (double)*a.loss_scale : 1.0;
        c = (float)(dh * (double)a.beta / (double)a.pairs * scale);
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k)
        for (uint64_t t = lo[k] + threadIdx.x; t < hi[k]; t += kBlock) a.coef[t] = k ? -c : c;
    if (!is_last_block(tickets, &last)) return;
    double x = 0.0;
    for (uint64_t k = threadIdx.x; k < a.pairs; k += kBlock) x += ld_device(a.pair_loss + k);
    x = block_sum(x, lds);
    if (threadIdx.x == 0) *a.loss = (float)(x / (double)a.pairs);
}

// ---- row_sums_kernel ----------------------------------------------------------------------------
constexpr uint32_t kSumBlocks = 64;
struct SumArgs {
    const int64_t* targets;
    uint64_t rows, per;  // rows per block
    const double *part, *part_kl;
    double* sums;      // 3 per block
    double denominator;  // 0: the unmasked rows
    const float* loss_scale;
    float *loss, *kl;
    float* norm;  // what the rows' c is multiplied with: the loss scale / D
};
__global__ __launch_bounds__(kBlock) void row_sums_kernel(SumArgs a, uint32_t* tickets) {
    __shared__ double lds[kBlock / 64];
    __shared__ uint32_t last;
    const uint64_t lo = blockIdx.x * a.per, hi = min(lo + a.per, a.rows);
    double x[3] = {0.0, 0.0, 0.0};
    for (uint64_t t = lo + threadIdx.x; t < hi; t += kBlock) {
        x[0] += a.targets[t] >= 0 ? 1.0 : 0.0;
        x[1] += a.part[t];
        x[2] += a.part_kl[t];
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        x[k] = block_sum(x[k], lds);
        if (threadIdx.x == 0) st_device(a.sums + 3 * blockIdx.x + k, x[k]);
    }
    if (!is_last_block(tickets, &last)) return;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        double v = threadIdx.x < gridDim.x ? ld_device(a.sums + 3 * threadIdx.x + k) : 0.0;
        x[k] = block_sum(v, lds);
    }
    if (threadIdx.x == 0) {
        const double d = a.denominator > 0.0 ? a.denominator : fmax(x[0], 1.0);
        *a.loss = (float)(x[1] / d);
        *a.kl = (float)(x[2] / d);
        *a.norm = (float)((a.loss_scale ? (double)*a.loss_scale : 1.0) / d);
    }
}

// ---- row_grads_kernel ---------------------------------------------------------------------------
struct GradArgs {
    const void* z;
    void* g;  // may be z
    uint64_t rows, z_stride, g_stride;
    uint32_t cols;
    const int64_t* targets;
    const Stat* stats;
    const float* coef;
    const float* norm;  // null: 1
};
// Block b: part b % splits of row b / splits.  Each element is read before it is written by the
// same lane, so the gradient may take the logits' place.
template <class T>
__global__ __launch_bounds__(kRowBlock) void row_grads_kernel(GradArgs a, uint32_t splits,
                                                              uint32_t per) {
    constexpr int P = kPer<T>;
    const uint64_t items = a.rows * splits;
    for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const uint64_t row = i / splits;
        const uint32_t part = (uint32_t)(i - row * splits);
        const uint32_t lo = part * per, hi = part + 1 == splits ? a.cols : lo + per;
        const uint32_t chunks = (hi - lo) / P;
        const T* z = (const T*)a.z + row * a.z_stride + lo;
        T* g = (T*)a.g + row * a.g_stride + lo;
        const int64_t y = a.targets[row];
        const float c = a.coef[row] * (a.norm ? *a.norm : 1.0f);
        const Stat st = a.stats[row];
        const uint32_t tail = chunks * P + threadIdx.x;
        if (y < 0 || c == 0.0f) {
            // a row that does not count, or not at all (c = 0, of a masked row, of one in no
            // sequence, of a clipped ratio): zeros, also where its logits are not finite
            for (uint32_t k = threadIdx.x; k < chunks; k += kRowBlock)
                store16(g + (uint64_t)k * P, u32x4{0, 0, 0, 0});
            if (tail < hi - lo) narrow(0.0f, g + tail);
            continue;
        }
        // past the vocabulary (its logp and c are NaN): no element
        const uint32_t at = y < (int64_t)a.cols ? (uint32_t)y - lo : ~0u;
        const float f = -c / st.s;
        for (uint32_t k = threadIdx.x; k < chunks; k += kRowBlock) {
            float v[P];
            unpack(load16(z + (uint64_t)k * P), v, z);
#pragma unroll
            for (int j = 0; j < P; ++j) {
                v[j] = f * exp2_fast((v[j] - st.m) * kLog2e);
                if (k * P + j == at) v[j] += c;
            }
            store16(g + (uint64_t)k * P, pack(v, z));
        }
        if (tail < hi - lo) {
            float v = f * exp2_fast((widen(z[tail]) - st.m) * kLog2e);
            if (tail == at) v += c;
            narrow(v, g + tail);
        }
    }
}

// ---- launches -----------------------------------------------------------------------------------
uint32_t grid_of(uint64_t items) { return (uint32_t)std::min<uint64_t>(items, 1u << 22); }

// Rows are split over the vocabulary until the launch has about four blocks for each CU; a part
// is a whole number of 16-byte chunks, 8 KiB at least, a row in 64 parts at most.
struct Split {
    uint32_t splits, per;
};
Split split_rows(uint64_t rows, uint32_t cols, uint32_t size, int cus) {
    const uint64_t row_bytes = (uint64_t)cols * size;
    uint64_t n = rows ? std::max<uint64_t>((uint64_t)cus * 4 / rows, 1) : 1;
    n = std::max<uint64_t>(std::min({n, (uint64_t)64, row_bytes / 8192}), 1);
    const uint32_t unit = 16 / size;
    const uint32_t per = (uint32_t)(((cols + n - 1) / n + unit - 1) / unit * unit);
    const uint32_t splits = std::max<uint32_t>((cols + per - 1) / per, 1);
    return {splits, per};
}

template <Loss kLoss>
int launch_scores(const ttpi::Op& op, const RowArgs& a, int dtype, Split sp, double* parts) {
    if (!a.rows) return TTP_OK;
    const dim3 grid(grid_of(a.rows * sp.splits)), block(kRowBlock);
    (void)hipGetLastError();
    if (dtype == TTP_DTYPE_BF16)
        hipLaunchKernelGGL((row_scores_kernel<uint16_t, kLoss>), grid, block, 0, op.stream, a,
                           sp.splits, sp.per, parts, op.tickets);
    else
        hipLaunchKernelGGL((row_scores_kernel<float, kLoss>), grid, block, 0, op.stream, a,
                           sp.splits, sp.per, parts, op.tickets);
    TTPI_HIP(hipGetLastError());
    return TTP_OK;
}

int launch_grads(const ttpi::Op& op, const GradArgs& a, int dtype) {
    if (!a.rows) return TTP_OK;
    const Split sp = split_rows(a.rows, a.cols, (uint32_t)ttpi::elem_size(dtype), op.num_cus);
    const dim3 grid(grid_of(a.rows * sp.splits)), block(kRowBlock);
    (void)hipGetLastError();
    if (dtype == TTP_DTYPE_BF16)
        hipLaunchKernelGGL(row_grads_kernel<uint16_t>, grid, block, 0, op.stream, a, sp.splits,
                           sp.per);
    else
        hipLaunchKernelGGL(row_grads_kernel<float>, grid, block, 0, op.stream, a, sp.splits,
                           sp.per);
    TTPI_HIP(hipGetLastError());
    return TTP_OK;
}

// The parts of a context's scratch memory, each 256-byte aligned.
struct Scratch {
    uint64_t bytes = 0;
    uint64_t add(uint64_t n) {
        const uint64_t at = bytes;
        bytes += (n + 255) / 256 * 256;
        return at;
    }
};

}  // namespace
}  // namespace ttp

using namespace ttp;
using ttpi::fail;

extern "C" {

int ttp_token_logprobs(ttp_ctx* ctx, const ttp_matrix* logits, const int64_t* targets,
                       float* logps) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = ttpi::check_matrix(logits, "the logits"))) return rc;
        const uint64_t rows = logits->rows;
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(logits, rows, logits->cols, "the logits", false))) return rc;
        if ((rc = b.array(targets, rows, 8, "the targets", false))) return rc;
        if ((rc = b.array(logps, rows, 4, "the log-probabilities", true))) return rc;
        const Split sp = split_rows(rows, (uint32_t)logits->cols,
                                    (uint32_t)ttpi::elem_size(logits->dtype), op.num_cus);
        void* parts = nullptr;
        if (sp.splits > 1 && (rc = ttpi::workspace(ctx, rows * sp.splits * 8, &parts))) return rc;
        RowArgs a{};
        a.z = logits->data;
        a.rows = rows;
        a.stride = logits->stride;
        a.cols = (uint32_t)logits->cols;
        a.targets = targets;
        a.logps = logps;
        return launch_scores<kScore>(op, a, logits->dtype, sp, (double*)parts);
    });
}

int ttp_preference_loss(ttp_ctx* ctx, const ttp_preference_args* p) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if (!p) return fail(TTP_ERR_INVALID, "null arguments");
        if ((rc = ttpi::check_matrix(p->logits, "the logits"))) return rc;
        if (!p->pairs || p->pairs > (1u << 20))
            return fail(TTP_ERR_RANGE, "pairs must be 1 to 2^20");
        if (!(p->beta > 0.0) || !std::isfinite(p->beta))
            return fail(TTP_ERR_INVALID, "beta must be positive");
        if (!(p->label_smoothing >= 0.0 && p->label_smoothing <= 0.5))
            return fail(TTP_ERR_INVALID, "label_smoothing must be in [0, 0.5]");
        const uint64_t rows = p->logits->rows, cols = p->logits->cols;
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(p->logits, rows, cols, "the logits", false))) return rc;
        if ((rc = b.array(p->targets, rows, 8, "the targets", false))) return rc;
        if ((rc = b.array(p->starts, 2 * p->pairs + 1, 8, "the sequences' starts", false)))
            return rc;
        if (p->ref_logps &&
            (rc = b.array(p->ref_logps, rows, 4, "the reference's log-probabilities", false)))
            return rc;
        if (p->grad) {
            if ((rc = b.matrix(p->grad, rows, cols, "the gradient", true, p->logits))) return rc;
            if (p->grad->dtype != p->logits->dtype)
                return fail(TTP_ERR_INVALID, "the gradient has another type than the logits");
        }
        if ((rc = b.array(p->logps, rows, 4, "the log-probabilities", true))) return rc;
        if ((rc = b.array(p->margins, p->pairs, 4, "the margins", true))) return rc;
        if ((rc = b.array(p->loss, 1, 4, "the loss", true))) return rc;

        const Split sp = split_rows(rows, (uint32_t)cols,
                                    (uint32_t)ttpi::elem_size(p->logits->dtype), op.num_cus);
        Scratch s;
        const uint64_t part = s.add(rows * 8), stats = s.add(rows * 8), coef = s.add(rows * 4),
                       pair_loss = s.add(p->pairs * 8),
                       parts = s.add(sp.splits > 1 ? rows * sp.splits * 8 : 0);
        void* ws;
        if ((rc = ttpi::workspace(ctx, s.bytes, &ws))) return rc;
        char* w = (char*)ws;

        RowArgs a{};
        a.z = p->logits->data;
        a.rows = rows;
        a.stride = p->logits->stride;
        a.cols = (uint32_t)cols;
        a.targets = p->targets;
        a.logps = p->logps;
        a.ref = p->ref_logps;
        a.part = (double*)(w + part);
        a.stats = (Stat*)(w + stats);
        a.coef = (float*)(w + coef);
        if ((rc = launch_scores<kPreference>(op, a, p->logits->dtype, sp, (double*)(w + parts))))
            return rc;

        PairArgs pa{};
        pa.starts = p->starts;
        pa.rows = rows;
        pa.pairs = p->pairs;
        pa.part = a.part;
        pa.pair_loss = (double*)(w + pair_loss);
        pa.beta = (float)p->beta;
        pa.smoothing = (float)p->label_smoothing;
        pa.loss_scale = op.loss_scale;
        pa.coef = a.coef;
        pa.margins = p->margins;
        pa.loss = p->loss;
        (void)hipGetLastError();
        hipLaunchKernelGGL(pair_losses_kernel, dim3((uint32_t)p->pairs), dim3(kBlock), 0,
                           op.stream, pa, op.tickets);
        TTPI_HIP(hipGetLastError());
        if (!p->grad) return TTP_OK;
        GradArgs g{a.z,    p->grad->data, rows,    a.stride, p->grad->stride,
                   a.cols, p->targets,    a.stats, a.coef,   nullptr};
        return launch_grads(op, g, p->logits->dtype);
    });
}

int ttp_policy_loss(ttp_ctx* ctx, const ttp_policy_args* p) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if (!p) return fail(TTP_ERR_INVALID, "null arguments");
        if ((rc = ttpi::check_matrix(p->logits, "the logits"))) return rc;
        if (!(p->clip_low >= 0.0 && p->clip_low <= 1.0))
            return fail(TTP_ERR_INVALID, "clip_low must be in [0, 1]");
        if (!(p->clip_high >= 0.0) || !std::isfinite(p->clip_high))
            return fail(TTP_ERR_INVALID, "clip_high must not be negative");
        if (!(p->kl_coef >= 0.0) || !std::isfinite(p->kl_coef))
            return fail(TTP_ERR_INVALID, "kl_coef must not be negative");
        if (p->kl_coef > 0.0 && !p->ref_logps && p->logits->rows)  // (empty arrays are null)
            return fail(TTP_ERR_INVALID, "kl_coef needs the reference's log-probabilities");
        if (!(p->denominator >= 0.0) || !std::isfinite(p->denominator))
            return fail(TTP_ERR_INVALID, "denominator must be positive, or 0 for the rows' count");
        const uint64_t rows = p->logits->rows, cols = p->logits->cols;
        ttpi::Buffers b(ctx);
        if ((rc = b.matrix(p->logits, rows, cols, "the logits", false))) return rc;
        if ((rc = b.array(p->targets, rows, 8, "the targets", false))) return rc;
        if ((rc = b.array(p->old_logps, rows, 4, "the old log-probabilities", false))) return rc;
        if ((rc = b.array(p->advantages, rows, 4, "the advantages", false))) return rc;
        if (p->ref_logps &&
            (rc = b.array(p->ref_logps, rows, 4, "the reference's log-probabilities", false)))
            return rc;
        if (p->grad) {
            if ((rc = b.matrix(p->grad, rows, cols, "the gradient", true, p->logits))) return rc;
            if (p->grad->dtype != p->logits->dtype)
                return fail(TTP_ERR_INVALID, "the gradient has another type than the logits");
        }
        if ((rc = b.array(p->logps, rows, 4, "the log-probabilities", true))) return rc;
        if ((rc = b.array(p->loss, 1, 4, "the loss", true))) return rc;
        if ((rc = b.array(p->kl, 1, 4, "the mean k", true))) return rc;

        const Split sp = split_rows(rows, (uint32_t)cols,
                                    (uint32_t)ttpi::elem_size(p->logits->dtype), op.num_cus);
        Scratch s;
        const uint64_t part = s.add(rows * 8), part_kl = s.add(rows * 8), stats = s.add(rows * 8),
                       coef = s.add(rows * 4), sums = s.add(kSumBlocks * 3 * 8),
                       norm = s.add(4), parts = s.add(sp.splits > 1 ? rows * sp.splits * 8 : 0);
        void* ws;
        if ((rc = ttpi::workspace(ctx, s.bytes, &ws))) return rc;
        char* w = (char*)ws;

        RowArgs a{};
        a.z = p->logits->data;
        a.rows = rows;
        a.stride = p->logits->stride;
        a.cols = (uint32_t)cols;
        a.targets = p->targets;
        a.logps = p->logps;
        a.ref = p->ref_logps;
        a.part = (double*)(w + part);
        a.stats = (Stat*)(w + stats);
        a.coef = (float*)(w + coef);
        a.old = p->old_logps;
        a.adv = p->advantages;
        a.part_kl = (double*)(w + part_kl);
        a.clip_lo = (float)(1.0 - p->clip_low);
        a.clip_hi = (float)(1.0 + p->clip_high);
        a.kl_coef = (float)p->kl_coef;
        if ((rc = launch_scores<kPolicy>(op, a, p->logits->dtype, sp, (double*)(w + parts))))
            return rc;

        SumArgs sa{};
        sa.targets = p->targets;
        sa.rows = rows;
        const uint32_t blocks =
            (uint32_t)std::max<uint64_t>(std::min<uint64_t>((rows + kBlock - 1) / kBlock,
                                                            kSumBlocks), 1);
        sa.per = (rows + blocks - 1) / blocks;
        sa.part = a.part;
        sa.part_kl = a.part_kl;
        sa.sums = (double*)(w + sums);
        sa.denominator = p->denominator;
        sa.loss_scale = op.loss_scale;
        sa.loss = p->loss;
        sa.kl = p->kl;
        sa.norm = (float*)(w + norm);
        (void)hipGetLastError();
        hipLaunchKernelGGL(row_sums_kernel, dim3(blocks), dim3(kBlock), 0, op.stream, sa,
                           op.tickets);
        TTPI_HIP(hipGetLastError());
        if (!p->grad) return TTP_OK;
        GradArgs g{a.z,    p->grad->data, rows,    a.stride, p->grad->stride,
                   a.cols, p->targets,    a.stats, a.coef,   sa.norm};
        return launch_grads(op, g, p->logits->dtype);
    });
}

}  // extern "C"
