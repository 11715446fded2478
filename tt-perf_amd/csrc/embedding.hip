// embedding.hip — embedding lookup, and its gradient by sorted tokens.
//
// The lookup is bound by memory: a lane has 8 columns of a row.
//
// The gradient's row v is the sum of the rows of dy whose token is v, in their order.  Two or three
// launches: sort_tokens_kernel puts the tokens in order (equal ones by their rows), sum_rows_kernel
// walks the sorted list in chunks of equal length, so that frequent tokens cost no more than rare
// ones, and writes every run of one token that lies within a chunk; what a chunk has of a run that
// crosses its ends goes to scratch memory, and join_runs_kernel adds these up in order.  No sum
// depends on when a block runs.
//
// The sort: a block has every kParts-th token of the table.  It counts the tokens of all rows that
// are another block's before its own, which is where its own begin, so the blocks need nothing of
// each other; it reads the list of tokens (128 KB of a batch of 16384) from the L2 for that.  Its
// own it lists in order, then places them by their token through a counter for each in the LDS:
// 64 at a time by one wave, whose ballots tell each entry how many equal ones stand before it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "columns8.hpp"
#include "context.hpp"
#include "matrix.hpp"
#include "vector16.hpp"

namespace ttp {
namespace {

// ---- lookup -----------------------------------------------------------------------------------
constexpr int kLookupBlock = 256;
struct LookupArgs {
    const void *table, *positions_table;  // positions_table null: none
    uint64_t vocab, positions_vocab;
    const int64_t *tokens, *positions;
    float scale;
    uint32_t rows, cols, groups;
    Divider by_groups;
};

// 8 columns of the table's row `t`: zeros for a negative one, NaN for one past the table
template <class W>
__device__ __forceinline__ void table_cols(const void* table, uint64_t vocab, int64_t t, uint32_t c,
                                           uint32_t cols, float (&v)[8]) {
    const float other = t < 0 ? 0.0f : __uint_as_float(0x7FC00000u);
    if (t >= 0 && (uint64_t)t < vocab) {
        load_cols((const W*)table + (uint64_t)t * cols, c, cols, v);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = other;
    }
}

template <class W, class Y>
__global__ __launch_bounds__(kLookupBlock) void lookup_kernel(Y* y, uint64_t y_stride,
                                                              LookupArgs a) {
    const uint32_t i = blockIdx.x * kLookupBlock + threadIdx.x;
    if (i >= a.rows * a.groups) return;
    const uint32_t row = divide(i, a.by_groups), c = (i - row * a.groups) * 8;
    float v[8], p[8] = {};
    table_cols<W>(a.table, a.vocab, a.tokens[row], c, a.cols, v);
    if (a.positions_table)
        table_cols<W>(a.positions_table, a.positions_vocab, a.positions[row], c, a.cols, p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = a.scale * v[j] + p[j];
    store_cols(y + row * y_stride, c, a.cols, v);
}

template <class W, class Y>
int lookup_rows(hipStream_t stream, LookupArgs a, const ttp_matrix& y) {
    a.cols = (uint32_t)y.cols;
    a.groups = (a.cols + 7) / 8;
    a.by_groups = divider(a.groups);
    const uint64_t most = std::max<uint64_t>((1u << 30) / a.groups, 1);
    const int64_t *tokens = a.tokens, *positions = a.positions;
    for (uint64_t r = 0; r < y.rows; r += most) {
        a.rows = (uint32_t)std::min<uint64_t>(most, y.rows - r);
        a.tokens = tokens + r;
        a.positions = positions ? positions + r : nullptr;
        (void)hipGetLastError();
        hipLaunchKernelGGL((lookup_kernel<W, Y>),
                           dim3((a.rows * a.groups + kLookupBlock - 1) / kLookupBlock),
                           dim3(kLookupBlock), 0, stream, (Y*)y.data + r * y.stride, y.stride, a);
        TTPI_HIP(hipGetLastError());
    }
    return TTP_OK;
}

// ---- the gradient -----------------------------------------------------------------------------
constexpr int kSortBlock = 1024;
constexpr uint32_t kMostKeys = 8192;  // tokens of a block: a counter each in the LDS
constexpr uint32_t kChunk = 32;       // sorted rows that a wave adds up
constexpr uint32_t kSlab = 256;       // columns of a wave, 4 a lane

struct Entry {
    uint32_t token, row;
};

struct GradArgs {
    const int64_t* tokens;
    const void* dy;
    uint64_t dy_stride;
    uint32_t rows, cols, vocab;
    uint32_t parts, keys;  // blocks of the sort; tokens of each
    uint32_t slabs;
    float scale;
    void* grad;
    bool first;         // assign, zeros where no token is
    Entry* listed;      // a block's tokens in the order of the rows
    Entry* sorted;
    uint32_t* count;    // of sorted entries
    float* partial;     // per chunk its first and its last run's sums, where they cross its ends
};

// The sum over the block's lanes before this one, and over all of them.
struct Before {
    uint32_t before, all;
};
__device__ __forceinline__ Before block_before(uint32_t x, uint32_t* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t s = x;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t up = (uint32_t)__shfl_up((int)s, d);
        s += lane >= d ? up : 0u;
    }
    __syncthreads();  // the last totals have been read
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    uint32_t base = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSortBlock / 64; ++w) {
        const uint32_t t = lds[w];
        base += w < wave ? t : 0u;
        all += t;
    }
    return {base + s - x, all};
}

template <class G>
__global__ __launch_bounds__(kSortBlock) void sort_tokens_kernel(GradArgs a) {
    __shared__ uint32_t lds[kSortBlock / 64];
    __shared__ uint32_t counts[kMostKeys];
    const uint32_t t = threadIdx.x, part = blockIdx.x;
    for (uint32_t k = t; k < a.keys; k += kSortBlock) counts[k] = 0;
    __syncthreads();

    // how many tokens are an earlier block's, and how often each of this block's occurs
    uint32_t less = 0;
    for (uint64_t r = t; r < a.rows; r += kSortBlock) {
        const int64_t v = a.tokens[r];
        if (v < 0 || v >= (int64_t)a.vocab) continue;
        const uint32_t p = (uint32_t)v % a.parts;
        less += p < part;
        if (p == part) atomicAdd(&counts[(uint32_t)v / a.parts], 1u);
    }
    const uint32_t base = block_before(less, lds).all;

    // this block's, in the order of the rows
    uint32_t n = 0;
    for (uint64_t r0 = 0; r0 < a.rows; r0 += kSortBlock) {
        const int64_t v = r0 + t < a.rows ? a.tokens[r0 + t] : -1;
        const bool mine =
            v >= 0 && v < (int64_t)a.vocab && (uint32_t)v % a.parts == part;
        const Before b = block_before(mine, lds);
        if (mine) a.listed[base + n + b.before] = {(uint32_t)v, (uint32_t)(r0 + t)};
        n += b.all;
    }
    if (part == a.parts - 1 && t == 0) *a.count = base + n;

    // rows that no token names
    if (a.first) {
        G* grad = (G*)a.grad;
        for (uint32_t k = t >> 6; k < a.keys; k += kSortBlock / 64) {
            const uint64_t v = (uint64_t)k * a.parts + part;
            if (v >= a.vocab || counts[k]) continue;
            G* row = grad + v * a.cols;
            const float zeros[8] = {};
            for (uint64_t c = (t & 63) * 8; c < a.cols; c += 512)
                store_cols(row, (uint32_t)c, a.cols, zeros);
        }
    }
    __syncthreads();

    // where each token's begin: kMostKeys / kSortBlock counters a lane
    constexpr uint32_t kOf = kMostKeys / kSortBlock;
    uint32_t c[kOf], sum = 0;
#pragma unroll
    for (uint32_t k = 0; k < kOf; ++k) {
        c[k] = t * kOf + k < a.keys ? counts[t * kOf + k] : 0u;
        sum += c[k];
    }
    uint32_t at = block_before(sum, lds).before;
#pragma unroll
    for (uint32_t k = 0; k < kOf; ++k) {
        if (t * kOf + k < a.keys) counts[t * kOf + k] = at;
        at += c[k];
    }
    __syncthreads();  // (the list, too: written and read by this block alone)
    if (t >= 64) return;
    for (uint32_t i = 0; i < n; i += 64) {
        const bool in = i + t < n;
        const Entry e = in ? a.listed[base + i + t] : Entry{0, 0};
        const uint32_t key = e.token / a.parts;
        uint64_t same = __ballot(in);
        for (uint32_t bit = 0; (a.keys - 1) >> bit; ++bit) {
            const uint64_t ones = __ballot((key >> bit) & 1);
            same &= (key >> bit) & 1 ? ones : ~ones;
        }
        const uint32_t before = __popcll(same & ((1ull << t) - 1));
        if (in) {
            const uint32_t to = counts[key] + before;
            a.sorted[base + to] = e;
        }
        __builtin_amdgcn_wave_barrier();
        if (in && (same >> t) == 1) counts[key] += before + 1;  // the last of its token
        __builtin_amdgcn_wave_barrier();
    }
}

// 4 columns of a row, those past the row's end as 0
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
__device__ __forceinline__ f32x4 load4(const uint16_t* row, uint32_t c, uint32_t cols) {
    if (c + 4 <= cols) {
        const u32x2 w = *reinterpret_cast<const u32x2_any*>(row + c);
        return f32x4{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
    }
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (c + k < cols) v[k] = widen(row[c + k]);
    return v;
}
__device__ __forceinline__ f32x4 load4(const float* row, uint32_t c, uint32_t cols) {
    f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c + 4 <= cols) {
        const u32x4 w = load16(row + c);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = __uint_as_float(w[k]);
        return v;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (c + k < cols) v[k] = row[c + k];
    return v;
}
__device__ __forceinline__ void store4(uint16_t* row, uint32_t c, uint32_t cols, f32x4 v) {
    if (c + 4 <= cols) {
        const u32x2 w = {bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3])};
        *reinterpret_cast<u32x2_any*>(row + c) = w;
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (c + k < cols) narrow(v[k], row + c + k);
}
__device__ __forceinline__ void store4(float* row, uint32_t c, uint32_t cols, f32x4 v) {
    if (c + 4 <= cols) {
        const float w[4] = {v[0], v[1], v[2], v[3]};
        store16(row + c, pack(w, row));
        return;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (c + k < cols) row[c + k] = v[k];
}

// A token's sum into its row of the gradient.
template <class O>
__device__ __forceinline__ void put_row(const GradArgs& a, uint32_t token, uint32_t c, f32x4 v) {
    O* row = (O*)a.grad + (uint64_t)token * a.cols;
    v *= a.scale;
    if (!a.first) v = load4(row, c, a.cols) + v;
    store4(row, c, a.cols, v);
}

// A wave: a chunk of sorted rows, a slab of their columns.
template <class G, class O>
__global__ __launch_bounds__(256) void sum_rows_kernel(GradArgs a, uint32_t waves) {
    const uint32_t w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= waves) return;
    const uint32_t lane = threadIdx.x & 63, chunk = w / a.slabs, slab = w % a.slabs;
    const uint32_t count = __builtin_amdgcn_readfirstlane(*a.count), first = chunk * kChunk;
    if (first >= count) return;
    const uint32_t n = min(kChunk, count - first), c = slab * kSlab + lane * 4;
    // this chunk's entries in the lanes, the one before and the one behind
    const Entry e = a.sorted[first + min(lane, n - 1)];
    const bool enters = first && a.sorted[first - 1].token == a.sorted[first].token;
    const bool leaves =
        first + n < count && a.sorted[first + n].token == a.sorted[first + n - 1].token;
    const G* dy = (const G*)a.dy;
    const bool in = c < a.cols;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    uint32_t run = 0;  // how many runs are behind us
    constexpr uint32_t kAhead = 8;
    for (uint32_t i = 0; i < n; i += kAhead) {
        f32x4 v[kAhead];
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)e.row, min(i + k, n - 1));
            v[k] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (in && i + k < n) v[k] = load4(dy + r * a.dy_stride, c, a.cols);
        }
#pragma unroll
        for (uint32_t k = 0; k < kAhead; ++k) {
            if (i + k >= n) break;
            const uint32_t token =
                (uint32_t)__builtin_amdgcn_readlane((int)e.token, min(i + k, n - 1));
            const uint32_t next =
                (uint32_t)__builtin_amdgcn_readlane((int)e.token, min(i + k + 1, n - 1));
            sum += v[k];
            const bool last = i + k + 1 == n;
            if (!last && next == token) continue;
            const bool in_before = run == 0 && enters, goes_on = last && leaves;
            if (in) {
                if (!in_before && !goes_on)
                    put_row<O>(a, token, c, sum);
                else  // (a run through the whole chunk counts as its first, if it came in)
                    *reinterpret_cast<f32x4*>(
                        a.partial + (((uint64_t)chunk * 2 + (in_before ? 0 : 1)) * a.slabs + slab) *
                                        kSlab + lane * 4) = sum;
            }
            sum = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            ++run;
        }
    }
}

// The runs that leave the chunk in which they begin: a wave of that chunk adds up what the chunks
// have, in order.
template <class O>
__global__ __launch_bounds__(256) void join_runs_kernel(GradArgs a, uint32_t waves) {
    const uint32_t w = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (w >= waves) return;
    const uint32_t lane = threadIdx.x & 63, chunk = w / a.slabs, slab = w % a.slabs;
    const uint32_t count = __builtin_amdgcn_readfirstlane(*a.count), end = (chunk + 1) * kChunk;
    if (end >= count) return;
    const uint32_t token = a.sorted[end - 1].token, c = slab * kSlab + lane * 4;
    if (a.sorted[end].token != token) return;
    if (chunk && a.sorted[end - kChunk].token == token &&
        a.sorted[end - kChunk - 1].token == token)
        return;  // it began before
    const auto at = [&](uint32_t k, uint32_t which) {
        return reinterpret_cast<const f32x4*>(
            a.partial + (((uint64_t)k * 2 + which) * a.slabs + slab) * kSlab + lane * 4);
    };
    f32x4 sum = *at(chunk, 1);
    for (uint32_t k = chunk + 1; k * kChunk < count && a.sorted[k * kChunk].token == token; ++k)
        sum += *at(k, 0);
    if (c < a.cols) put_row<O>(a, token, c, sum);
}

template <class G, class O>
int add_rows(const ttpi::Op& op, const GradArgs& a) {
    (void)hipGetLastError();
    hipLaunchKernelGGL(sort_tokens_kernel<O>, dim3(a.parts), dim3(kSortBlock), 0, op.stream, a);
    TTPI_HIP(hipGetLastError());
    const uint32_t chunks = (uint32_t)(((uint64_t)a.rows + kChunk - 1) / kChunk);
    const uint32_t waves = chunks * a.slabs;  // (fewer than 2^26)
    const dim3 grid((waves + 3) / 4);
    if (!waves) return TTP_OK;
    hipLaunchKernelGGL((sum_rows_kernel<G, O>), grid, dim3(256), 0, op.stream, a, waves);
    TTPI_HIP(hipGetLastError());
    if (chunks > 1) {
        hipLaunchKernelGGL(join_runs_kernel<O>, grid, dim3(256), 0, op.stream, a, waves);
        TTPI_HIP(hipGetLastError());
    }
    return TTP_OK;
}

// A table of rows of `cols`, to be read.
int table_param(ttp_ctx* ctx, ttpi::Buffers& b, uint32_t index, uint64_t cols, const char* what,
                ttpi::Param* p) {
    int rc = ttpi::param(ctx, index, p);
    if (rc) return rc;
    if (!p->numel || p->numel % cols)
        return ttpi::fail(TTP_ERR_RANGE, "tensor " + std::to_string(index) + " has " +
                                             std::to_string(p->numel) + " elements, not rows of " +
                                             std::to_string(cols));
    return b.array(p->data, p->numel, p->bf16 ? 2 : 4, what, false);
}

int check_scale(double scale) {
    if (std::isfinite((float)scale)) return TTP_OK;
    return ttpi::fail(TTP_ERR_INVALID, "scale must be a finite number (in fp32)");
}

}  // namespace
}  // namespace ttp

using namespace ttp;
using ttpi::fail;

extern "C" {

int ttp_embedding(ttp_ctx* ctx, uint32_t table, const int64_t* tokens, double scale,
                  uint32_t position_table, const int64_t* positions, const ttp_matrix* y) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = check_scale(scale))) return rc;
        if ((rc = ttpi::check_matrix(y, "the output"))) return rc;
        const bool has_positions = position_table != TTP_NO_TENSOR;
        if (has_positions != (positions != nullptr) && (has_positions ? y->rows != 0 : true))
            return fail(TTP_ERR_INVALID, "a table of positions and the positions go together");
        ttpi::Buffers b(ctx);
        ttpi::Param t{}, p{};
        if ((rc = table_param(ctx, b, table, y->cols, "the table", &t))) return rc;
        if (has_positions &&
            (rc = table_param(ctx, b, position_table, y->cols, "the table of positions", &p)))
            return rc;
        if ((rc = b.array(tokens, y->rows, 8, "the tokens", false))) return rc;
        if (has_positions && (rc = b.array(positions, y->rows, 8, "the positions", false)))
            return rc;
        if ((rc = b.matrix(y, y->rows, y->cols, "the output", true))) return rc;
        LookupArgs a{};
        a.table = t.data;
        a.positions_table = p.data;
        a.vocab = t.numel / y->cols;
        a.positions_vocab = p.numel / y->cols;
        a.tokens = tokens;
        a.positions = has_positions ? positions : nullptr;
        a.scale = (float)scale;
        const bool bf16 = y->dtype == TTP_DTYPE_BF16;
        if (t.bf16)
            return bf16 ? lookup_rows<uint16_t, uint16_t>(op.stream, a, *y)
                        : lookup_rows<uint16_t, float>(op.stream, a, *y);
        return bf16 ? lookup_rows<float, uint16_t>(op.stream, a, *y)
                    : lookup_rows<float, float>(op.stream, a, *y);
    });
}

int ttp_accumulate_embedding_grad(ttp_ctx* ctx, uint32_t table, const int64_t* tokens, double scale,
                                  const ttp_matrix* dy) {
    return ttpi::guarded([&]() -> int {
        ttpi::Op op;
        int rc = ttpi::begin(ctx, &op);
        if (rc) return rc;
        if ((rc = check_scale(scale))) return rc;
        if ((rc = ttpi::check_matrix(dy, "the output's gradient"))) return rc;
        ttpi::GradTarget g{};
        if ((rc = ttpi::grad_target(ctx, table, &g))) return rc;
        const uint64_t rows = dy->rows, cols = dy->cols;
        if (!g.numel || g.numel % cols)
            return fail(TTP_ERR_RANGE, "tensor " + std::to_string(table) + " has " +
                                           std::to_string(g.numel) + " elements, not rows of " +
                                           std::to_string(cols));
        const uint64_t vocab = g.numel / cols;
        if (vocab >= (1ull << 31))
            return fail(TTP_ERR_RANGE, "the table has 2^31 rows or more");
        ttpi::Buffers b(ctx);
        if ((rc = b.array(tokens, rows, 8, "the tokens", false))) return rc;
        if ((rc = b.matrix(dy, rows, cols, "the output's gradient", false))) return rc;
        if ((rc = b.array(g.data, g.numel, g.bf16 ? 2 : 4, "the table's gradient", true)))
            return rc;
        GradArgs a{};
        a.tokens = tokens;
        a.dy = dy->data;
        a.dy_stride = dy->stride;
        a.rows = (uint32_t)rows;
        a.cols = (uint32_t)cols;
        a.vocab = (uint32_t)vocab;
        const uint64_t fewest = (vocab + kMostKeys - 1) / kMostKeys;
        a.parts = (uint32_t)std::max<uint64_t>(fewest, std::min<uint64_t>(op.num_cus, vocab));
        a.keys = (uint32_t)((vocab + a.parts - 1) / a.parts);
        a.slabs = (a.cols + kSlab - 1) / kSlab;
        a.scale = (float)scale;
        a.grad = g.data;
        a.first = g.first;
        const uint64_t chunks = (rows + kChunk - 1) / kChunk;
        if (chunks * a.slabs >= (1ull << 26))
            return fail(TTP_ERR_RANGE, "the output's gradient is too large for one launch");
        // partial sums, listed and sorted entries, their count
        const uint64_t partial = chunks * 2 * a.slabs * kSlab * 4;
        void* ws;
        if ((rc = ttpi::workspace(ctx, partial + 2 * rows * sizeof(Entry) + 16, &ws))) return rc;
        a.partial = (float*)ws;
        a.listed = (Entry*)((char*)ws + partial);
        a.sorted = a.listed + rows;
        a.count = (uint32_t*)(a.sorted + rows);
        const bool bf16 = dy->dtype == TTP_DTYPE_BF16;
        if (g.bf16)
            rc = bf16 ? add_rows<uint16_t, uint16_t>(op, a) : add_rows<float, uint16_t>(op, a);
        else
            rc = bf16 ? add_rows<uint16_t, float>(op, a) : add_rows<float, float>(op, a);
        if (rc) return rc;
        ttpi::grad_written(ctx, table);
        return TTP_OK;
    });
}

}  // extern "C"
