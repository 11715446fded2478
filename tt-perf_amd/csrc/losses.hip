// losses.hip — token log-probabilities, the preference loss and the clipped policy loss, with the
// logits' gradient.
//
// With z a row of logits, y its token, m = max z and s = sum exp(z - m):
//   logp = (z_y - m) - log s,   p_v = exp(z_v - m) / s,   dlogp/dz_v = [v = y] - p_v
// so a loss that is a function of the rows' logp gives dz_v = c ([v = y] - p_v) with one number c
// per row.  The floor is the logits read once and the gradient written once; the arithmetic is
// about ten VALU operations and one exponential per logit for the statistics, and as many again
// for the gradient.
//
//   row_scores_kernel   (m, s) of parts of rows, a wave each; rows of one part are finished at once
//   finish_rows_kernel  joins the parts of the others: logp, and the row's part of the loss
//   pair_losses_kernel  sums over sequences, the pairs' losses, the rows' c (preference)
//   row_grads_kernel    the gradient from (m, s, c): the logits are read a second time
//   policy_rows_kernel  the policy loss and its gradient in one pass: c depends on its own row, so
//                       the row stays in registers between its statistics and its gradient
//   row_sums_kernel     the number of rows that count, and sums of the rows' losses (policy)
//
// A preference row's c depends on all rows of its pair, gigabytes of them, so its logits cannot
// stay; a policy row longer than a block's registers takes the same two passes.  Statistics are in
// fp32, sums over rows in fp64.  Every sum's order depends on the shapes alone.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "context.hpp"
#include "device.hpp"
#include "matrix.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

// ---- (maximum, sum of exponentials) ---------------------------------------------------------
struct Stat {
    float m, s;  // s = sum exp(z - m); nothing: (-inf, 0)
};
// What the exponents are taken from: an all -inf part has the sum 0, not exp(-inf + inf).
__device__ __forceinline__ float stat_base(float m) { return m == -INFINITY ? 0.0f : m; }
// exp(z - base).  The difference first: one fused operation on z log2 e would leave the rounding
// of base log2 e in every row, and overflow at the type's lowest value.
__device__ __forceinline__ float power(float z, float base) {
    return exp2_fast((z - base) * kLog2e);
}

// The wave's sum or maximum in every lane, by a butterfly without LDS permutes (see wave_sum).
template <int kCtrl>
__device__ __forceinline__ float dpp(float x) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), kCtrl,
                                                                 0xF, 0xF, true));
}
template <class F>
__device__ __forceinline__ float wave_all(float x, F&& f) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    x = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false,
                                                    false);
    x = f(__uint_as_float(b[0]), __uint_as_float(b[1]));
    x = f(x, dpp<0x128>(x));  // row_ror:8
    x = f(x, dpp<0x124>(x));  // row_ror:4
    x = f(x, dpp<0x4E>(x));   // quad_perm:[2,3,0,1]
    return f(x, dpp<0xB1>(x));  // quad_perm:[1,0,3,2]
}
__device__ __forceinline__ float wave_max(float x) {
    return wave_all(x, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float wave_add(float x) {
    return wave_all(x, [](float a, float b) { return a + b; });
}

constexpr uint32_t kNone16 = 0xFF80FF80u, kNone32 = 0xFF800000u;  // -inf
template <class T>
__device__ __forceinline__ u32x4 no_logits() {
    const uint32_t n = sizeof(T) == 2 ? kNone16 : kNone32;
    return u32x4{n, n, n, n};
}

// A wave's statistics of its lanes' kLoads chunks and one more logit each (-inf where a lane has
// none): the wave's maximum first, so that no sum has to be rescaled.  kLean: the chunks are
// unpacked again for the sum (kept from the maximum, their values take twice the registers).
template <class T, int kLoads, bool kLean>
__device__ __forceinline__ Stat wave_stat(u32x4* w, float extra) {
    constexpr int P = kPer<T>;
    float m = extra;
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
        float v[P];
        unpack(w[k], v, (const T*)nullptr);
#pragma unroll
        for (int j = 0; j < P; ++j) m = fmaxf(m, v[j]);  // (skips NaN, which the sum then holds)
    }
    m = wave_max(m);
    if constexpr (kLean) {
#pragma unroll
        for (int k = 0; k < kLoads; ++k) asm volatile("" : "+v"(w[k]));
    }
    const float base = stat_base(m);
    float s = power(extra, base);
#pragma unroll
    for (int k = 0; k < kLoads; ++k) {
        float v[P];
        unpack(w[k], v, (const T*)nullptr);
#pragma unroll
        for (int j = 0; j < P; ++j) s += power(v[j], base);
    }
    return {m, wave_add(s)};
}

// A row's parts 0 .. splits - 1 together, f(k) giving part k: `lanes` lanes (a power of two, at
// most a wave) take every lanes-th, each in order.  The result is in all of them.
template <class F>
__device__ __forceinline__ Stat join_parts(uint32_t splits, uint32_t lanes, F&& f) {
    const uint32_t p = threadIdx.x % lanes;
    float m = -INFINITY, s = 0.0f;
    for (uint32_t k = p; k < splits; k += lanes) m = fmaxf(m, f(k).m);
    for (uint32_t off = lanes / 2; off; off >>= 1) m = fmaxf(m, __shfl_xor(m, (int)off));
    const float base = stat_base(m);
    for (uint32_t k = p; k < splits; k += lanes) {
        const Stat x = f(k);
        s += x.s * power(x.m, base);
    }
    for (uint32_t off = lanes / 2; off; off >>= 1) s += __shfl_xor(s, (int)off);
    return {m, s};
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
    // by pair_losses_kernel or few_pairs where a sequence covers the row)
    const float* ref;
    double* part;
    Stat* stats;
    float* coef;
    // policy: part is the row's loss, part_kl its k
    const float *old, *adv;
    double* part_kl;
    float clip_lo, clip_hi, kl_coef;
};

// The token's logit; past the vocabulary NaN.  (A masked row's is not asked for.)
template <class T>
__device__ __forceinline__ float token_logit(const RowArgs& a, uint64_t row, int64_t y) {
    return y < (int64_t)a.cols ? widen(((const T*)a.z)[row * a.stride + (uint64_t)y]) : NAN;
}
__device__ __forceinline__ float row_logp(float zy, Stat st) {
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
    const float logp = y < 0 ? 0.0f : row_logp(token_logit<T>(a, row, y), st);
    a.logps[row] = logp;
    if constexpr (kLoss == kPreference) {
        st_device(a.part + row, y < 0 ? 0.0 : (double)logp - (a.ref ? (double)a.ref[row] : 0.0));
        a.stats[row] = st;
        // (at memory before another block of this launch writes the sequence's c)
        __hip_atomic_store(a.coef + row, 0.0f, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    } else if constexpr (kLoss == kPolicy) {
        PolicyRow p = {0.0f, 0.0f, 0.0f};
        if (y >= 0) p = policy_row(a, row, logp);
        a.part[row] = (double)p.loss;
        a.part_kl[row] = (double)p.kl;
        a.stats[row] = st;
        a.coef[row] = p.coef;
    }
}

// ---- a sequence's part of the loss ------------------------------------------------------------
__device__ __forceinline__ uint64_t bounded(int64_t x, uint64_t lo, uint64_t hi) {
    return x < (int64_t)lo ? lo : (uint64_t)x > hi ? hi : (uint64_t)x;
}
// log(1 + exp(x))
__device__ __forceinline__ double softplus(double x) {
    return fmax(x, 0.0) + log1p(exp(-fabs(x)));
}

struct PairArgs {
    const int64_t* starts;
    uint64_t rows, pairs;
    const double* part;
    double* pair_loss;
    double beta, smoothing;
    const float* loss_scale;
    float *coef, *margins, *loss;
};
// One pair's loss from its margin h, and its c = scale dloss/dmargin beta / pairs.  Without
// smoothing the second term is left out: at a margin of +inf it would be 0 x inf.
__device__ __forceinline__ double pair_loss(const PairArgs& a, double h) {
    const double eps = a.smoothing;
    return (1.0 - eps) * softplus(-h) + (eps > 0.0 ? eps * softplus(h) : 0.0);
}
__device__ __forceinline__ float pair_coef(const PairArgs& a, double h) {
    // (each sigmoid by itself: their difference would lose the small one)
    const double eps = a.smoothing, dh = eps / (1.0 + exp(-h)) - (1.0 - eps) / (1.0 + exp(h));
    const double scale = a.loss_scale ? (double)*a.loss_scale : 1.0;
    return (float)(dh * a.beta / (double)a.pairs * scale);
}

// The pairs of few rows, by the block that sees them all finished: 16 lanes to a sequence.  Up to
// kFewPairs and kFewRows: a launch less is 3 us of the host (250 to 4000 rows, 4 or 16 pairs: 26 to
// 23.5 us a call, the GPU's time the same; 64 pairs take it 6 us more).
constexpr uint32_t kFewPairs = 16, kFewRows = 4096;
static_assert(kBlock == 256);
__device__ __forceinline__ void few_pairs(const PairArgs& a) {
    constexpr uint32_t kLanes = 16, kLoads = 16;
    __shared__ double d[2 * kFewPairs], lds[kBlock / 64];
    __shared__ float c[kFewPairs];
    const uint32_t t = threadIdx.x, lane = t % kLanes, sequences = 2 * (uint32_t)a.pairs;
    for (uint32_t s = t / kLanes; s < sequences; s += kBlock / kLanes) {
        const uint32_t lo = (uint32_t)bounded(a.starts[s], 0, a.rows);
        const uint32_t hi = (uint32_t)bounded(a.starts[s + 1], lo, a.rows);
        double x = 0.0;
        // (the loads of 256 rows together: each comes from memory)
        for (uint32_t r = lo + lane; r < hi; r += kLanes * kLoads) {
            double v[kLoads];
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k)
                v[k] = ld_device(a.part + min(r + k * kLanes, hi - 1));
#pragma unroll
            for (uint32_t k = 0; k < kLoads; ++k) x += r + k * kLanes < hi ? v[k] : 0.0;
        }
        for (uint32_t off = kLanes / 2; off; off >>= 1) x += __shfl_xor(x, (int)off);
        if (lane == 0) d[s] = x;
    }
    __syncthreads();
    double x = 0.0;
    if (t < a.pairs) {
        const double h = a.beta * (d[t] - d[t + a.pairs]);
        a.margins[t] = (float)h;
        x = pair_loss(a, h);
        c[t] = pair_coef(a, h);
    }
    x = block_sum(x, lds);
    if (t == 0) *a.loss = (float)(x / (double)a.pairs);
    for (uint32_t s = t / kLanes; s < sequences; s += kBlock / kLanes) {
        const uint32_t lo = (uint32_t)bounded(a.starts[s], 0, a.rows);
        const uint32_t hi = (uint32_t)bounded(a.starts[s + 1], lo, a.rows);
        const float v = s < a.pairs ? c[s] : -c[s - a.pairs];
        for (uint32_t r = lo + lane; r < hi; r += kLanes) a.coef[r] = v;
    }
}

// ---- row_scores_kernel ------------------------------------------------------------------------
// A row is cut into 16-byte chunks from its first element on, its last elements (fewer than a
// chunk) by themselves, and the chunks into parts of 256, one wave's four loads per lane.  Which
// lane takes what, and in which order sums are joined, depends on the number of columns alone: a
// row's bits do not depend on where it lies.
constexpr int kRowBlock = 256;
constexpr int kLoads = 4;
constexpr uint32_t kPart = kLoads * 64;

// Where a wave is: a part of a row, and whether the row counts (a masked row is not read).
struct Place {
    uint64_t row;
    uint32_t part;
    bool live;
};
// A part on its way through a wave.  Its loads are issued without a branch, so that what is waited
// for can be counted and the next part's stay in flight: lanes that have no chunk load the row's
// last one, and a row without one, or that does not count, loads from `other`.
template <class T>
struct Part {
    u32x4 w[kLoads];
    T last;

    // (kOnce: no gradient kernel reads them again soon)
    template <bool kOnce>
    __device__ __forceinline__ void load(const RowArgs& a, const Place& at, const void* other) {
        constexpr int P = kPer<T>;
        const uint32_t chunks = a.cols / P, lane = threadIdx.x & 63;
        const T* z = at.live ? (const T*)a.z + at.row * a.stride : (const T*)other;
        last = z[at.live ? min(chunks * P + lane, a.cols - 1) : 0u];
        const T* first = chunks ? z : (const T*)other;
        const uint32_t top = at.live && chunks ? chunks - 1 : 0;
#pragma unroll
        for (int k = 0; k < kLoads; ++k) {
            const uint32_t c = min(at.part * kPart + k * 64 + lane, top);
            const T* p = first + (uint64_t)c * P;
            w[k] = kOnce ? load16_once(p) : load16(p);
        }
    }
    __device__ __forceinline__ Stat stat(const RowArgs& a, const Place& at, uint32_t splits) {
        constexpr int P = kPer<T>;
        const uint32_t chunks = a.cols / P, lane = threadIdx.x & 63;
        float extra = -INFINITY;
        if (at.part + 1 == splits) {
            if (chunks * P + lane < a.cols) extra = widen(last);
#pragma unroll
            for (int k = 0; k < kLoads; ++k)
                if (at.part * kPart + k * 64 + lane >= chunks) w[k] = no_logits<T>();
        }
        return wave_stat<T, kLoads, false>(w, extra);
    }
};

// Wave i: part i % splits of row i / splits, and on by the launch's waves.  With `last_joins`
// (every wave then has one part) the launch's last block joins the rows' parts, else
// finish_rows_kernel does; rows of one part are finished at once.
// Bound by the exponentials and the reading, about evenly.  Parts rather than rows per block:
// the waves in flight then sweep a narrow window of memory.  Measured: 8192 rows of 50257 bf16, one
// in ten masked, 131 us, 5.65 TB/s of the logits it reads (on the 16-byte grid 5.9, fp32 6.1); one
// such row in 7 blocks 6 us, of which three quarters are the launch, the first loads and the join.
template <class T, Loss kLoss>
__global__ __launch_bounds__(kRowBlock) void row_scores_kernel(RowArgs a, uint32_t splits,
                                                               uint32_t lanes, double* parts,
                                                               uint32_t last_joins,
                                                               PairArgs pairs, uint32_t* tickets) {
    constexpr uint32_t kWaves = kRowBlock / 64;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    // a step of all the launch's waves, as rows and parts: no division per part
    const uint32_t step = gridDim.x * kWaves;
    const uint32_t step_rows = step / splits, step_parts = step - step_rows * splits;
    // (by the scalar unit: nothing writes to the targets meanwhile, and vector loads in flight are
    // not waited for)
    const auto* targets = (const __attribute__((address_space(4))) int64_t*)(uintptr_t)a.targets;
    const auto look = [&](Place& p) { p.live = p.row < a.rows && targets[p.row] >= 0; };
    const auto behind = [&](const Place& p) {
        Place n{p.row + step_rows, p.part + step_parts, false};
        if (n.part >= splits) {
            n.part -= splits;
            n.row += 1;
        }
        look(n);
        return n;
    };
    const auto finish = [&](Part<T>& p, const Place& at) {
        Stat st = {-INFINITY, 0.0f};
        if (at.live) st = p.stat(a, at, splits);
        if ((threadIdx.x & 63) == 0) {
            if (splits == 1)
                finish_row<T, kLoss>(a, at.row, st);
            else
                st_device(parts + at.row * splits + at.part, __builtin_bit_cast(double, st));
        }
    };
    // the next part's logits are on their way while one is summed
    constexpr bool kOnce = kLoss == kScore;
    const uint32_t first = blockIdx.x * kWaves + wave;
    Part<T> one, two;
    Place at{first / splits, 0, false}, next;
    at.part = first - (uint32_t)at.row * splits;
    look(at);
    if (at.row < a.rows) {
        one.template load<kOnce>(a, at, tickets);
        for (;;) {
            next = behind(at);
            two.template load<kOnce>(a, next, tickets);
            finish(one, at);
            if (next.row >= a.rows) break;
            at = behind(next);
            one.template load<kOnce>(a, at, tickets);
            finish(two, next);
            if (at.row >= a.rows) break;
        }
    }
    const bool here = kLoss == kPreference && pairs.starts && (splits == 1 || last_joins);
    if (!last_joins && !here) return;
    __shared__ uint32_t last;
    // every wave's parts are at memory before the block takes its ticket
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (!is_last_block(tickets, &last)) return;
    const uint32_t rows = kRowBlock / lanes;
    if (last_joins)
        for (uint64_t base = 0; base < a.rows; base += rows) {
            const uint64_t row = min(base + threadIdx.x / lanes, a.rows - 1);
            const Stat st = join_parts(splits, lanes, [&](uint32_t k) {
                return __builtin_bit_cast(Stat, ld_device(parts + row * splits + k));
            });
            if (base + threadIdx.x / lanes < a.rows && threadIdx.x % lanes == 0)
                finish_row<T, kLoss>(a, row, st);
        }
    if constexpr (kLoss == kPreference)
        if (here) {
            asm volatile("" ::: "memory");
            __builtin_amdgcn_s_waitcnt(0);
            __syncthreads();
            few_pairs(pairs);
        }
}

// The parts of long rows, `lanes` lanes to a row.  Bound by its launch: 9733 rows of 25 parts 5 us.
template <class T, Loss kLoss>
__global__ __launch_bounds__(kRowBlock) void finish_rows_kernel(RowArgs a, uint32_t splits,
                                                                uint32_t lanes,
                                                                const double* parts, PairArgs pairs,
                                                                uint32_t* tickets) {
    const uint32_t rows = kRowBlock / lanes;
    for (uint64_t base = (uint64_t)blockIdx.x * rows; base < a.rows;
         base += (uint64_t)gridDim.x * rows) {
        const uint64_t row = min(base + threadIdx.x / lanes, a.rows - 1);
        const Stat st = join_parts(splits, lanes, [&](uint32_t k) {
            return __builtin_bit_cast(Stat, parts[row * splits + k]);
        });
        if (base + threadIdx.x / lanes < a.rows && threadIdx.x % lanes == 0)
            finish_row<T, kLoss>(a, row, st);
    }
    if constexpr (kLoss == kPreference) {
        if (!pairs.starts) return;
        __shared__ uint32_t last;
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
        if (is_last_block(tickets, &last)) few_pairs(pairs);
    }
}

// ---- pair_losses_kernel -----------------------------------------------------------------------
// Block p: pair p.  Sums in fp64 (a margin is the small difference of sums over hundreds of
// tokens), each lane's share in row order, then the block's lanes in a fixed order.  Bound by its
// launch and three waits in a row (a sequence, the block's sums, the last block): 5 to 7 us.
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
        const double h = a.beta * (d[0] - d[1]);
        a.margins[p] = (float)h;
        st_device(a.pair_loss + p, pair_loss(a, h));
        c = pair_coef(a, h);
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
// Bound by its launch and the last block's wait: 5 us for 16384 rows.
constexpr uint32_t kSumBlocks = 64;
struct SumArgs {
    const int64_t* targets;
    uint64_t rows, per;  // rows per block
    const double *part, *part_kl;  // null: the norm alone
    double* sums;      // 3 per block
    double denominator;  // 0: the unmasked rows
    const float* loss_scale;
    float *loss, *kl;
    float* norm;  // what the rows' c is multiplied with: the loss scale / D
};
__device__ __forceinline__ double denominator_of(const SumArgs& a, double unmasked) {
    return a.denominator > 0.0 ? a.denominator : fmax(unmasked, 1.0);
}
__device__ __forceinline__ float norm_of(const SumArgs& a, double d) {
    return (float)((a.loss_scale ? (double)*a.loss_scale : 1.0) / d);
}
__global__ __launch_bounds__(kBlock) void row_sums_kernel(SumArgs a, uint32_t* tickets) {
    __shared__ double lds[kBlock / 64];
    __shared__ uint32_t last;
    const uint64_t lo = blockIdx.x * a.per, hi = min(lo + a.per, a.rows);
    double x[3] = {0.0, 0.0, 0.0};
    for (uint64_t t = lo + threadIdx.x; t < hi; t += kBlock) {
        x[0] += a.targets[t] >= 0 ? 1.0 : 0.0;
        if (a.part) {
            x[1] += a.part[t];
            x[2] += a.part_kl[t];
        }
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
        const double d = denominator_of(a, x[0]);
        if (a.part) {
            *a.loss = (float)(x[1] / d);
            *a.kl = (float)(x[2] / d);
        }
        *a.norm = norm_of(a, d);
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
constexpr int kGradBlock = 256;
constexpr uint32_t kGradPart = 512;  // chunks of a part: two for each lane
// The row's values: f exp(z - m), f = -c / s.
template <class T>
__device__ __forceinline__ u32x4 grad16(u32x4 w, const T* type, float f, float m) {
    float v[kPer<T>];
    unpack(w, v, type);
#pragma unroll
    for (int k = 0; k < kPer<T>; ++k) v[k] = f * power(v[k], m);
    return pack(v, type);
}

// Block b: part b % splits of row b / splits (kLanes 64: four rows per block, of at most 128
// chunks).  Each element is read before it is written by the same lane, so the gradient may take
// the logits' place.  Bound by HBM: 9733 rows of 50257 bf16, three in ten masked, 300 us, 5.5 TB/s
// read and written.
template <class T, int kLanes>
__global__ __launch_bounds__(kGradBlock) void row_grads_kernel(GradArgs a, uint32_t splits) {
    constexpr int P = kPer<T>, kRows = kGradBlock / kLanes, kLoads = 2;
    const uint32_t t = threadIdx.x % kLanes, chunks = a.cols / P;
    const uint64_t items = (a.rows + kRows - 1) / kRows * splits;
    for (uint64_t i = blockIdx.x; i < items; i += gridDim.x) {
        const uint64_t group = i / splits;
        const uint32_t part = (uint32_t)(i - group * splits);
        const uint64_t row = group * kRows + __builtin_amdgcn_readfirstlane(threadIdx.x / kLanes);
        if (kRows > 1 && row >= a.rows) continue;
        const T* z = (const T*)a.z + row * a.z_stride;
        T* g = (T*)a.g + row * a.g_stride;
        const int64_t y = a.targets[row];
        const float c = a.coef[row] * (a.norm ? *a.norm : 1.0f);
        const Stat st = a.stats[row];
        const uint32_t first = part * kGradPart + t;
        const uint32_t e = part + 1 == splits ? chunks * P + t : a.cols;
        if (y < 0 || c == 0.0f) {
            // a row that does not count, or not at all (c = 0, of a masked row, of one in no
            // sequence, of a clipped ratio): zeros, also where its logits are not finite
#pragma unroll
            for (int k = 0; k < kLoads; ++k)
                if (first + k * kLanes < chunks)
                    store16_once(g + (uint64_t)(first + k * kLanes) * P, u32x4{0, 0, 0, 0});
            if (e < a.cols) narrow(0.0f, g + e);
            continue;
        }
        const float f = -c / st.s;
        u32x4 w[kLoads];
        float zy = 0.0f;
        // the token's chunk (this lane's, or none of its): c more, in fp32
        const uint64_t cy = (uint64_t)y / P;
        const bool own = y < (int64_t)a.cols && cy < chunks &&
                         (cy == first || cy == first + (uint64_t)kLanes);
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (first + k * kLanes < chunks)
                w[k] = load16_once(z + (uint64_t)(first + k * kLanes) * P);
        if (own) zy = widen(z[y]);
#pragma unroll
        for (int k = 0; k < kLoads; ++k)
            if (first + k * kLanes < chunks)
                store16_once(g + (uint64_t)(first + k * kLanes) * P, grad16(w[k], z, f, st.m));
        if (own) narrow(f * power(zy, st.m) + c, g + y);
        if (e < a.cols) {
            const float v = f * power(widen(z[e]), st.m);
            narrow((int64_t)e == y ? v + c : v, g + e);
        }
    }
}

// ---- policy_rows_kernel -------------------------------------------------------------------------
// The policy loss and its gradient in one pass: a row's logits stay in kThreads lanes' registers
// (kChunks 16-byte chunks each) from the statistics to the gradient, which needs nothing of other
// rows but their number (in *o.norm, the loss scale / D).  One row per kThreads lanes; without a
// gradient (o.g null) the losses alone.  The statistics are taken and joined part by part as
// row_scores_kernel and its joins do, so that a token's log-probability has the same bits here as
// there: the first step on a rollout finds ratios of exactly 1.
// Bound by HBM, and by how few rows a CU holds: one row's loads have to cover another's
// exponentials and stores.  16384 rows of 50257 bf16 every 50304 565 us, 5.8 TB/s; every 50257, so
// off the 16-byte grid, 720 us (the loads' share of the difference 60 us, the stores' 20) where two
// passes take 854 (816 over batches of rows that the 256 MB cache holds); 1021 rows of 50257 fp32
// 78 us, 5.2 TB/s.

// Up to this many rows the launch does everything (`tickets` given): each block counts the rows by
// itself, and the last one adds up the losses.  (One launch for three: 1021 rows of 50257 fp32 85.8
// to 78.3 us, a call over few rows 26 to 20 us of the host, 2000 rows of 50257 bf16 94.8 to 93.6.
// Above, every block's count of all rows and one block's sum take longer than launches of their
// own: 4000 rows 204 us against 187.)
constexpr uint32_t kAlone = 2048;
template <class T, int kThreads, int kChunks>
__global__ __launch_bounds__(kThreads < 256 ? 256 : kThreads) void policy_rows_kernel(
    RowArgs a, GradArgs o, SumArgs sums, uint32_t* tickets) {
    constexpr int P = kPer<T>;
    constexpr bool kWaves = kThreads == 64;  // a row is a wave, and one part
    constexpr int kRows = kWaves ? 4 : 1;
    constexpr uint32_t kGroups = kThreads / 64;
    constexpr int kParts = (kChunks + kLoads - 1) / kLoads;  // of a wave
    static_assert(kChunks % kLoads == 0 || kParts == 1);
    __shared__ Stat lds[kWaves ? 1 : kGroups * kParts];
    __shared__ uint32_t counted[kGroups];
    const bool alone = tickets != nullptr;
    const uint32_t t = threadIdx.x % kThreads, lane = t & 63, chunks = a.cols / P;
    // (the same in a wave: its addresses are one scalar and 32 bits per lane)
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint64_t row = (uint64_t)blockIdx.x * kRows + (kWaves ? wave : 0);
    // The rows that count, of those that this wave looks at.  (Out here: behind the masked row's
    // return, the 1024-lane shapes took 680 us for 565, alone or not.)
    uint32_t n = 0;
    if (alone && o.g && !(sums.denominator > 0.0)) {
#pragma unroll
        for (uint32_t i = 0; i < kAlone; i += kThreads) {
            const bool one = i + t < a.rows && a.targets[i + t] >= 0;
            n += __popcll(__ballot(one));
        }
        if (!kWaves && lane == 0) counted[wave] = n;
    }
    const auto do_row = [&]() {
        const T* z = (const T*)a.z + row * a.stride;
        T* g = (T*)o.g + row * o.g_stride;
        const int64_t y = a.targets[row];
        const uint32_t splits = kWaves ? 1 : (chunks + kPart - 1) / kPart;
        // chunk k of this lane; and for the lanes of the last part's wave the row's last elements
        const auto chunk = [&](int k) {
            return kWaves ? lane + k * 64
                          : (wave + k / kLoads * kGroups) * kPart + k % kLoads * 64 + lane;
        };
        const uint32_t e = kWaves || (splits - 1) % kGroups == wave ? chunks * P + lane : a.cols;
        // f(k, its bytes from the row's start) for this lane's chunks in the row
        const auto each = [&](auto&& f) {
#pragma unroll
            for (int k = 0; k < kChunks; ++k)
                if (chunk(k) < chunks) f(k, chunk(k) * 16);
        };
        const auto zeros = [&]() {
            each([&](int, uint32_t b) { store16_once((T*)((char*)g + b), u32x4{0, 0, 0, 0}); });
            if (e < a.cols) narrow(0.0f, g + e);
        };
        if (y < 0) {
            if (t == 0) {
                a.logps[row] = 0.0f;
                st_device(a.part + row, 0.0);
                st_device(a.part_kl + row, 0.0);
            }
            if (o.g) zeros();
            return;
        }
        // (read now: behind the statistics every row would wait for it)
        float norm = !alone && o.g ? *o.norm : 0.0f;
        // (first, and without a branch to wait in: their values are there once the chunks are)
        const T last_z = z[min(e, a.cols - 1)];
        const T token_z = z[min((uint64_t)y, (uint64_t)a.cols - 1)];
        u32x4 w[kChunks];
#pragma unroll
        for (int k = 0; k < kChunks; ++k) w[k] = no_logits<T>();
        each([&](int k, uint32_t b) { w[k] = load16_once((const T*)((const char*)z + b)); });
        const float ze = e < a.cols ? widen(last_z) : -INFINITY;
        float zy = y < (int64_t)a.cols ? widen(token_z) : NAN;
        asm volatile("" : "+v"(zy));  // read before any lane writes a gradient in its place
        Stat st;
        if constexpr (kWaves) {
            st = wave_stat<T, kChunks, true>(w, ze);
        } else {
#pragma unroll
            for (int j = 0; j < kParts; ++j) {
                const uint32_t part = wave + j * kGroups;
                if (part < splits) {
                    st = wave_stat<T, kLoads, true>(w + kLoads * j,
                                                    part + 1 == splits ? ze : -INFINITY);
                    if (lane == 0) lds[part] = st;
                }
            }
            __syncthreads();
            uint32_t lanes = 1;
            while (lanes < splits && lanes < 64) lanes *= 2;
            st = join_parts(splits, lanes, [&](uint32_t k) { return lds[k]; });
        }
        // every lane for itself: a second wait for one lane's result costs more
        const float logp = row_logp(zy, st);
        const PolicyRow p = policy_row(a, row, logp);
        if (t == 0) {
            a.logps[row] = logp;
            st_device(a.part + row, (double)p.loss);
            st_device(a.part_kl + row, (double)p.kl);
        }
        if (!o.g) return;
        if (alone) {
            if (!kWaves) {
                n = 0;
#pragma unroll
                for (uint32_t i = 0; i < kGroups; ++i) n += counted[i];
            }
            norm = norm_of(sums, denominator_of(sums, (double)n));
        }
        const float c = p.coef * norm;
        if (c == 0.0f) {
            zeros();
            return;
        }
        const float f = -c / st.s;
        // the packed registers are unpacked once more: kept from before, the values would take two
        // to four times the registers
#pragma unroll
        for (int k = 0; k < kChunks; ++k) asm volatile("" : "+v"(w[k]));
        // a row off the 16-byte grid: its stores share cache lines, which L2 puts together
        if ((uintptr_t)g % 16 == 0)
            each([&](int k, uint32_t b) {
                store16_once((T*)((char*)g + b), grad16(w[k], z, f, st.m));
            });
        else
            each([&](int k, uint32_t b) {
                store16((T*)((char*)g + b), grad16(w[k], z, f, st.m));
            });
        if (e < a.cols) {
            const float v = f * power(ze, st.m);
            narrow((int64_t)e == y ? v + c : v, g + e);
        }
        // the token's own: c more, in fp32, by the lane that has written its chunk
        const uint64_t cy = (uint64_t)y / P;
        if (cy < chunks) {
            const uint32_t x = (uint32_t)cy;
            const uint32_t owner = kWaves ? x % 64 : x / kPart % kGroups * 64 + x % 64;
            if (owner == t) narrow(f * power(zy, st.m) + c, g + y);
        }
    };
    if (row < a.rows) do_row();  // (whole waves are past the end, and only where a row is a wave)
    if (!alone) return;
    // the sums, by the launch's last block
    __shared__ uint32_t last;
    if constexpr (kWaves) {  // each wave has stored a row's part
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0);
        __syncthreads();
    }
    if (!is_last_block(tickets, &last)) return;
    constexpr uint32_t kBlockWaves = kWaves ? 4 : kGroups;
    __shared__ double parts[3][kBlockWaves];
    double x[3] = {0.0, 0.0, 0.0};
    for (uint64_t i = threadIdx.x; i < a.rows; i += kBlockWaves * 64) {
        x[0] += a.targets[i] >= 0 ? 1.0 : 0.0;
        x[1] += ld_device(a.part + i);
        x[2] += ld_device(a.part_kl + i);
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        x[k] = wave_sum(x[k]);
        if (lane == 0) parts[k][threadIdx.x / 64] = x[k];
    }
    __syncthreads();
    if (threadIdx.x) return;
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        x[k] = 0.0;
        for (uint32_t i = 0; i < kBlockWaves; ++i) x[k] += parts[k][i];
    }
    const double d = denominator_of(sums, x[0]);
    *sums.loss = (float)(x[1] / d);
    *sums.kl = (float)(x[2] / d);
}

// ---- launches -----------------------------------------------------------------------------------
uint32_t grid_of(uint64_t items) { return (uint32_t)std::min<uint64_t>(items, 1u << 22); }

uint32_t row_chunks(uint32_t cols, int dtype) {
    return cols / (16 / (uint32_t)ttpi::elem_size(dtype));
}

// Up to 1024 parts in all are joined by the launch's last block (a row of 50257 bf16: one launch
// instead of two), more by a launch of their own.
struct Split {
    uint32_t splits, lanes;
    bool last_joins;
    uint64_t parts;  // scratch entries
};
Split split_rows(uint64_t rows, uint32_t cols, int dtype) {
    const uint32_t chunks = row_chunks(cols, dtype);
    if (chunks <= kPart) return {1, 1, false, 0};
    const uint32_t splits = (chunks + kPart - 1) / kPart;
    uint32_t lanes = 1;
    while (lanes < splits && lanes < 64) lanes *= 2;
    return {splits, lanes, rows * splits <= 1024, rows * splits};
}

template <Loss kLoss, class T>
int launch_scores_of(const ttpi::Op& op, const RowArgs& a, Split sp, double* parts,
                     const PairArgs& pairs) {
    if (!a.rows) return TTP_OK;
    // (four rounds of blocks that fit the GPU at once: each wave starts its next part while it
    // sums one, and the rounds even out what masked rows leave)
    const dim3 block(kRowBlock), grid((uint32_t)std::min<uint64_t>((a.rows * sp.splits + 3) / 4,
                                                                   (uint64_t)op.num_cus * 32));
    (void)hipGetLastError();
    hipLaunchKernelGGL((row_scores_kernel<T, kLoss>), grid, block, 0, op.stream, a, sp.splits,
                       sp.lanes, parts, sp.last_joins ? 1u : 0u, pairs, op.tickets);
    TTPI_HIP(hipGetLastError());
    if (sp.splits == 1 || sp.last_joins) return TTP_OK;
    const uint64_t per_block = kRowBlock / sp.lanes;
    hipLaunchKernelGGL((finish_rows_kernel<T, kLoss>),
                       dim3(grid_of((a.rows + per_block - 1) / per_block)), block, 0, op.stream, a,
                       sp.splits, sp.lanes, (const double*)parts, pairs, op.tickets);
    TTPI_HIP(hipGetLastError());
    return TTP_OK;
}
// `pairs` (preference): finished in the same launches, where its starts are given.
template <Loss kLoss>
int launch_scores(const ttpi::Op& op, const RowArgs& a, int dtype, Split sp, double* parts,
                  const PairArgs& pairs = {}) {
    return dtype == TTP_DTYPE_BF16 ? launch_scores_of<kLoss, uint16_t>(op, a, sp, parts, pairs)
                                   : launch_scores_of<kLoss, float>(op, a, sp, parts, pairs);
}

template <class T>
int launch_grads_of(const ttpi::Op& op, const GradArgs& a) {
    if (!a.rows) return TTP_OK;
    const uint32_t chunks = a.cols / kPer<T>;
    (void)hipGetLastError();
    if (chunks <= 128) {
        hipLaunchKernelGGL((row_grads_kernel<T, 64>), dim3(grid_of((a.rows + 3) / 4)),
                           dim3(kGradBlock), 0, op.stream, a, 1u);
    } else {
        const uint32_t splits = (chunks + kGradPart - 1) / kGradPart;
        hipLaunchKernelGGL((row_grads_kernel<T, kGradBlock>), dim3(grid_of(a.rows * splits)),
                           dim3(kGradBlock), 0, op.stream, a, splits);
    }
    TTPI_HIP(hipGetLastError());
    return TTP_OK;
}
int launch_grads(const ttpi::Op& op, const GradArgs& a, int dtype) {
    return dtype == TTP_DTYPE_BF16 ? launch_grads_of<uint16_t>(op, a)
                                   : launch_grads_of<float>(op, a);
}

// The one-pass policy kernel's shape for rows of `chunks` chunks: f<lanes, chunks per lane>, or
// false where no shape holds them.  1024 lanes, two rows or one on a CU (16384 rows of 50257 bf16
// every 50304, so on the 16-byte grid: 565 us, 618 with 256 lanes; 1021 rows of 50257 fp32 78 us, 3
// us more with 512), but where rows lie anywhere and three of them fit a CU's registers, 256 lanes
// (the same rows every 50257: 725 us, 769 with 1024 lanes).
template <class F>
bool policy_shape(uint32_t chunks, bool on_grid, F&& f) {
#define TTP_SHAPE(T, C)                                                 \
    if (chunks <= T * C) {                                              \
        f(std::integral_constant<int, T>{}, std::integral_constant<int, C>{}); \
        return true;                                                    \
    }
    TTP_SHAPE(64, 1)
    TTP_SHAPE(64, 4)
    TTP_SHAPE(256, 4)
    TTP_SHAPE(256, 8)
    TTP_SHAPE(256, 16)
    if (!on_grid) {
        TTP_SHAPE(256, 28)
    }
    TTP_SHAPE(1024, 8)
    TTP_SHAPE(1024, 12)
    TTP_SHAPE(1024, 16)
    TTP_SHAPE(1024, 20)
#undef TTP_SHAPE
    return false;
}
template <class T>
int launch_policy(const ttpi::Op& op, const RowArgs& a, const GradArgs& g, const SumArgs& sums) {
    (void)hipGetLastError();
    const bool on_grid = ((uintptr_t)a.z | a.stride * sizeof(T)) % 16 == 0;
    policy_shape(a.cols / kPer<T>, on_grid, [&](auto lanes, auto chunks) {
        constexpr int kLanes = lanes, kChunks = chunks, kRows = kLanes < 256 ? 256 / kLanes : 1;
        hipLaunchKernelGGL((policy_rows_kernel<T, kLanes, kChunks>),
                           dim3((uint32_t)((a.rows + kRows - 1) / kRows)),
                           dim3(kLanes < 256 ? 256 : kLanes), 0, op.stream, a, g, sums,
                           a.rows <= kAlone ? op.tickets : nullptr);
    });
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
        const Split sp = split_rows(rows, (uint32_t)logits->cols, logits->dtype);
        void* parts = nullptr;
        if (sp.parts && (rc = ttpi::workspace(ctx, sp.parts * 8, &parts))) return rc;
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

        const Split sp = split_rows(rows, (uint32_t)cols, p->logits->dtype);
        Scratch s;
        const uint64_t part = s.add(rows * 8), stats = s.add(rows * 8), coef = s.add(rows * 4),
                       pair_loss = s.add(p->pairs * 8),
                       parts = s.add(sp.parts * 8);
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
        PairArgs pa{};
        pa.starts = p->starts;
        pa.rows = rows;
        pa.pairs = p->pairs;
        pa.part = a.part;
        pa.pair_loss = (double*)(w + pair_loss);
        pa.beta = p->beta;
        pa.smoothing = p->label_smoothing;
        pa.loss_scale = op.loss_scale;
        pa.coef = a.coef;
        pa.margins = p->margins;
        pa.loss = p->loss;
        const bool few = rows && rows <= kFewRows && p->pairs <= kFewPairs;
        if ((rc = launch_scores<kPreference>(op, a, p->logits->dtype, sp, (double*)(w + parts),
                                             few ? pa : PairArgs{})))
            return rc;
        if (!few) {
            (void)hipGetLastError();
            hipLaunchKernelGGL(pair_losses_kernel, dim3((uint32_t)p->pairs), dim3(kBlock), 0,
                               op.stream, pa, op.tickets);
            TTPI_HIP(hipGetLastError());
        }
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

        const Split sp = split_rows(rows, (uint32_t)cols, p->logits->dtype);
        Scratch s;
        const uint64_t part = s.add(rows * 8), part_kl = s.add(rows * 8), stats = s.add(rows * 8),
                       coef = s.add(rows * 4), sums = s.add(kSumBlocks * 3 * 8),
                       norm = s.add(4), parts = s.add(sp.parts * 8);
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
        SumArgs sa{};
        sa.targets = p->targets;
        sa.rows = rows;
        const uint32_t blocks =
            (uint32_t)std::max<uint64_t>(std::min<uint64_t>((rows + kBlock - 1) / kBlock,
                                                            kSumBlocks), 1);
        sa.per = (rows + blocks - 1) / blocks;
        sa.sums = (double*)(w + sums);
        sa.denominator = p->denominator;
        sa.loss_scale = op.loss_scale;
        sa.loss = p->loss;
        sa.kl = p->kl;
        sa.norm = (float*)(w + norm);
        const auto launch_sums = [&]() -> int {
            (void)hipGetLastError();
            hipLaunchKernelGGL(row_sums_kernel, dim3(blocks), dim3(kBlock), 0, op.stream, sa,
                               op.tickets);
            TTPI_HIP(hipGetLastError());
            return TTP_OK;
        };
        GradArgs g{a.z,    p->grad ? p->grad->data : nullptr, rows, a.stride,
                   p->grad ? p->grad->stride : 0, a.cols, p->targets, a.stats, a.coef, sa.norm};
        // One pass where a row fits the registers of a block and the rows one launch: the number
        // of rows that count first, the losses' sums behind it.
        const bool one_pass =
            rows && rows <= (1u << 21) &&
            policy_shape(row_chunks((uint32_t)cols, p->logits->dtype), true, [](auto, auto) {});
        if (one_pass) {
            const bool alone = rows <= kAlone;
            if (!alone && p->grad && (rc = launch_sums())) return rc;
            rc = p->logits->dtype == TTP_DTYPE_BF16 ? launch_policy<uint16_t>(op, a, g, sa)
                                                    : launch_policy<float>(op, a, g, sa);
            if (rc || alone) return rc;
            sa.part = a.part;
            sa.part_kl = a.part_kl;
            return launch_sums();
        }
        if ((rc = launch_scores<kPolicy>(op, a, p->logits->dtype, sp, (double*)(w + parts))))
            return rc;
        sa.part = a.part;
        sa.part_kl = a.part_kl;
        if ((rc = launch_sums())) return rc;
        return p->grad ? launch_grads(op, g, p->logits->dtype) : TTP_OK;
    });
}

}  // extern "C"
