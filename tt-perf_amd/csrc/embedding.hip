// embedding.hip — embedding lookup, and its gradient by sorted tokens.
//
// The lookup is bound by memory and by how little of it a lane has under way: its token, then 8 columns
// of that token's row, then the result (16384 x 768 bf16 with a table of positions: 10.6 us for the 36 MB
// of a batch with 5,900 different tokens, 3.4 TB/s).
//
// The gradient's row v is the sum of the rows of dy whose token is v.  Up to 512 rows few_rows_kernel
// looks for them itself, in eight sums that take them in turn.  For more there are three launches:
// sort_tokens_kernel puts the tokens in order (equal ones by their rows), sum_rows_kernel walks the
// sorted list in chunks of equal length, so that frequent tokens cost no more than rare ones, and
// writes every run of one token that lies within a chunk; what a chunk has of a run that crosses its
// ends goes to scratch memory, and join_runs_kernel adds these up, four sums in turn, while its other
// blocks write zeros where no token is.  The order of a sum follows from the list of tokens (which other
// tokens there are says where a run is cut), never from when a block runs.
// Measured, 16384 x 768 bf16 into 50257 rows: sort 12 us, sums 15 (5 of them to find their rows),
// joins beside 77 MB of zeros 14 (40 in all, as called); added to a gradient that is there 12, 13 and
// 6.  4099 x 384 fp32 into 65 rows: 7, 4 and 6 us.
//
// The sort: block p has the tokens p, p + parts, p + 2 parts ..., at most kMostKeys of the table's.
// It counts the tokens of all rows that are another block's before its own, which is where its own
// begin, so the blocks need nothing of each other; for that it reads the list of tokens (128 KB of
// a batch of 16384) from the L2.  Its own it lists in the order of the rows; each wave counts an
// equal share of the list by token, the counts' sums say where each wave's entries of each token
// go, and within 64 entries ballots tell how many equal ones stand before.  A block of one token has
// its entries in order as soon as they are listed (65 tokens, 4099 rows: 7.0 us instead of 8.8).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "columns8.hpp"
#include "context.hpp"
#include "embedding_cut.hpp"
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
constexpr int kSortBlock = 1024, kSortWaves = kSortBlock / 64;
constexpr uint32_t kMostKeys = 1024;  // tokens of a block: a counter for each and each wave
constexpr uint32_t kRounds = 16;      // tokens that a lane holds at a time
constexpr uint32_t kSortTile = kSortBlock * kRounds;
constexpr uint32_t kListed = 2048;    // entries that the LDS lists, more go to scratch memory
constexpr uint32_t kChunk = 16;       // sorted rows that a wave adds up
constexpr uint32_t kSlab = 256;       // columns of a wave, 4 a lane

struct Entry {
    uint32_t token, row;
};

struct GradArgs {
    const int64_t* tokens;
    const void* dy;
    uint64_t dy_stride;
    uint32_t rows, cols, vocab;
    uint32_t parts_log2, keys;  // blocks of the sort; tokens of each (few tokens: of a wave)
    uint32_t row0;              // few tokens: the launch's first row of the table
    uint32_t slabs;
    float scale;
    void* grad;
    bool first;       // assign, zeros where no token is
    uint32_t fills;   // waves that write those zeros
    Entry* listed;    // a block's tokens in the order of the rows, where the LDS does not hold them
    Entry* sorted;
    uint64_t* named;  // for each block of the sort, a bit for each of its tokens
    uint32_t* count;  // of sorted entries
    float* partial;   // per chunk its first and its last run's sums, where they cross its ends
};

// The sum over the waves before this one of a number that is the same in each of a wave's lanes, and
// over all waves.
struct Before {
    uint32_t before, all;
};
__device__ __forceinline__ Before waves_before(uint32_t x, uint32_t* lds) {
    const int wave = threadIdx.x >> 6;
    __syncthreads();  // the last totals have been read
    if ((threadIdx.x & 63) == 0) lds[wave] = x;
    __syncthreads();
    Before b{0, 0};
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
        const uint32_t t = lds[w];
        b.before += w < wave ? t : 0u;
        b.all += t;
    }
    return b;
}

__global__ __launch_bounds__(kSortBlock) void sort_tokens_kernel(GradArgs a) {
    __shared__ uint32_t totals[kSortWaves];
    __shared__ uint32_t counts[kSortWaves][kMostKeys];
    __shared__ Entry list[kListed];
    const uint32_t t = threadIdx.x, lane = t & 63, part = blockIdx.x;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t in_part = (1u << a.parts_log2) - 1;
    const uint64_t below = (1ull << lane) - 1;
    for (uint32_t w = 0; w < kSortWaves; ++w)
        for (uint32_t k = t; k < a.keys; k += kSortBlock) counts[w][k] = 0;

    // A tile of tokens: each wave has 64 neighbours a round.  -1: none of the table's.
    uint32_t v[kRounds];
    const auto load_tile = [&](uint32_t r0) {
        int64_t x[kRounds];
#pragma unroll
        for (uint32_t k = 0; k < kRounds; ++k) {
            const uint64_t r = (uint64_t)r0 + wave * (kRounds * 64) + k * 64 + lane;
            x[k] = r < a.rows ? a.tokens[r] : -1;
        }
#pragma unroll
        for (uint32_t k = 0; k < kRounds; ++k)
            v[k] = x[k] >= 0 && x[k] < (int64_t)a.vocab ? (uint32_t)x[k] : ~0u;
    };
    const auto mine = [&](uint32_t k) { return v[k] != ~0u && (v[k] & in_part) == part; };

    // how many tokens are an earlier block's
    uint32_t less = 0;
    for (uint64_t r0 = 0; r0 < a.rows; r0 += kSortTile) {
        load_tile((uint32_t)r0);
#pragma unroll
        for (uint32_t k = 0; k < kRounds; ++k)
            less += __popcll(__ballot(v[k] != ~0u && (v[k] & in_part) < part));
    }
    const uint32_t base = waves_before(less, totals).all;

    // this block's, in the order of the rows; those beyond the LDS's list at their place in memory
    uint32_t n = 0;
    for (uint64_t r0 = 0; r0 < a.rows; r0 += kSortTile) {
        if (a.rows > kSortTile) load_tile((uint32_t)r0);
        uint32_t here = 0;
#pragma unroll
        for (uint32_t k = 0; k < kRounds; ++k) here += __popcll(__ballot(mine(k)));
        const Before b = waves_before(here, totals);
        uint32_t at = n + b.before;
#pragma unroll
        for (uint32_t k = 0; k < kRounds; ++k) {
            const uint64_t m = __ballot(mine(k));
            if (mine(k)) {
                const uint32_t to = at + __popcll(m & below);
                const Entry e{v[k], (uint32_t)r0 + wave * (kRounds * 64) + k * 64 + lane};
                if (a.keys == 1)
                    a.sorted[base + to] = e;
                else if (to < kListed)
                    list[to] = e;
                else
                    a.listed[base + to] = e;
            }
            at += __popcll(m);
        }
        n += b.all;
    }
    if (part == in_part && t == 0) *a.count = base + n;
    if (a.keys == 1) {  // (the order of the rows is all)
        if (t == 0) a.named[part] = n != 0;
        return;
    }
    __syncthreads();  // (the list in memory, too: this block alone writes and reads its part)
    const auto entry = [&](uint32_t i) { return i < kListed ? list[i] : a.listed[base + i]; };

    // each wave's share by token
    const uint32_t share = (n + kSortBlock - 1) / kSortBlock * 64;
    const uint32_t begin = min(wave * share, n), end = min(begin + share, n);
    for (uint32_t i = begin + lane; i < end; i += 64)
        atomicAdd(&counts[wave][entry(i).token >> a.parts_log2], 1u);
    __syncthreads();
    // where they go: behind the lesser tokens, and behind the earlier waves' equal ones
    uint32_t sum = 0;
    if (t < a.keys)
        for (uint32_t w = 0; w < kSortWaves; ++w) {
            const uint32_t c = counts[w][t];
            counts[w][t] = sum;
            sum += c;
        }
    const uint64_t named = __ballot(sum != 0);
    if (lane == 0 && wave * 64 < a.keys) a.named[part * ((a.keys + 63) / 64) + wave] = named;
    uint32_t upto = sum;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t up = (uint32_t)__shfl_up((int)upto, d);
        upto += (int)lane >= d ? up : 0u;
    }
    const uint32_t start =
        waves_before((uint32_t)__builtin_amdgcn_readlane((int)upto, 63), totals).before + upto - sum;
    if (t < a.keys)
        for (uint32_t w = 0; w < kSortWaves; ++w) counts[w][t] += start;
    __syncthreads();
    for (uint32_t i = begin; i < end; i += 64) {
        const bool in = i + lane < end;
        const Entry e = in ? entry(i + lane) : Entry{0, 0};
        const uint32_t key = e.token >> a.parts_log2;
        uint64_t same = __ballot(in);
        for (uint32_t bit = 0; (a.keys - 1) >> bit; ++bit) {
            const uint64_t ones = __ballot((key >> bit) & 1);
            same &= (key >> bit) & 1 ? ones : ~ones;
        }
        const uint32_t before = __popcll(same & below);
        if (in) a.sorted[base + counts[wave][key] + before] = e;
        __builtin_amdgcn_wave_barrier();
        if (in && (same >> lane) == 1) counts[wave][key] += before + 1;  // the last of its token
        __builtin_amdgcn_wave_barrier();
    }
}

// 4 columns of a row as they lie in memory: a lane's in a slab.  The lane that has fewer than 4 left
// takes the row's last 4 (and writes its own of them); rows of fewer than 4 are read one by one.
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(2)));
struct Columns {
    uint32_t at;    // the first of the 4
    uint32_t skip;  // how many of them another lane writes (4: all)
};
__device__ __forceinline__ Columns columns_of(uint32_t c, uint32_t cols) {
    if (cols < 4) return {0, c ? 4u : 0u};
    return c + 4 <= cols ? Columns{c, 0} : Columns{cols - 4, min(c - (cols - 4), 4u)};
}
template <class T>
struct Raw4;
template <>
struct Raw4<uint16_t> {
    u32x2 w;
    __device__ __forceinline__ void load(const uint16_t* p) {
        w = *reinterpret_cast<const u32x2_any*>(p);
    }
    __device__ __forceinline__ void load_some(const uint16_t* p, uint32_t n) {  // 1 to 3
        w = u32x2{p[0], n > 2 ? p[2] : 0u};
        w.x |= n > 1 ? (uint32_t)p[1] << 16 : 0u;
    }
    __device__ __forceinline__ void here() { asm volatile("" : "+v"(w)); }
    __device__ __forceinline__ f32x4 values() const {
        return f32x4{bf16_lo(w.x), bf16_hi(w.x), bf16_lo(w.y), bf16_hi(w.y)};
    }
};
template <>
struct Raw4<float> {
    u32x4 w;
    __device__ __forceinline__ void load(const float* p) { w = load16(p); }
    __device__ __forceinline__ void load_some(const float* p, uint32_t n) {
        w = u32x4{__float_as_uint(p[0]), n > 1 ? __float_as_uint(p[1]) : 0u,
                  n > 2 ? __float_as_uint(p[2]) : 0u, 0u};
    }
    __device__ __forceinline__ void here() { asm volatile("" : "+v"(w)); }
    __device__ __forceinline__ f32x4 values() const { return __builtin_bit_cast(f32x4, w); }
};
__device__ __forceinline__ void store4(uint16_t* p, f32x4 v) {
    *reinterpret_cast<u32x2_any*>(p) = u32x2{bf16_pack(v[0], v[1]), bf16_pack(v[2], v[3])};
}
__device__ __forceinline__ void store4(float* p, f32x4 v) {
    const float w[4] = {v[0], v[1], v[2], v[3]};
    store16(p, pack(w, p));
}

template <class O>
__device__ __forceinline__ void old_row(Raw4<O>& old, const O* p, uint32_t cols) {
    if (cols >= 4)
        old.load(p);
    else
        old.load_some(p, cols);
}
// A token's sum into its row of the gradient, at this lane's columns.
template <class O>
__device__ __forceinline__ void put_row(O* p, uint32_t cols, float scale, bool first, Columns c,
                                        f32x4 v, const Raw4<O>& old) {
    v *= scale;
    if (!first) v = old.values() + v;
    if (cols >= 4 && !c.skip) {
        store4(p, v);
    } else {
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (k >= c.skip && c.at + k < cols) narrow(v[k], p + k);
    }
}

// Zeros in those of 16 rows that no token names, runs of them in one.
constexpr uint32_t kFillRows = 16;
template <class O>
__device__ __forceinline__ void fill_zeros(const GradArgs& a, uint32_t row0) {
    const uint32_t lane = threadIdx.x & 63, row = row0 + lane;
    bool none = false;
    if (lane < kFillRows && row < a.vocab) {
        const uint32_t part = row & ((1u << a.parts_log2) - 1), key = row >> a.parts_log2;
        none = !(a.named[part * ((a.keys + 63) / 64) + key / 64] >> (key % 64) & 1);
    }
    uint32_t left = (uint32_t)__ballot(none);
    while (left) {
        const uint32_t first = (uint32_t)__builtin_ctz(left);
        const uint32_t n = (uint32_t)__builtin_ctz(~(left >> first));  // (16 bits: there is a 0)
        left &= ~(((1u << n) - 1) << first);
        O* p = (O*)a.grad + (uint64_t)(row0 + first) * a.cols;
        const uint64_t all = (uint64_t)n * a.cols;
        const float zeros[8] = {};
        for (uint64_t at = lane * 8; at < all; at += 512)
            store_cols(p + at, 0, (uint32_t)min(all - at, 8ul), zeros);
    }
}

// A wave: a chunk of sorted rows, a slab of their columns.  All rows' loads are asked for at once; each
// row's sum from its run's beginning on stays in registers, and a loop over the runs' ends takes it
// from there, four at a time (written out for each row it was slower; through the LDS too few waves
// fit a CU).  kNarrow: rows of fewer than 4 columns.
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int kSumWaves = 4;
template <class G, class O, bool kNarrow>
__global__ __launch_bounds__(64 * kSumWaves) void sum_rows_kernel(GradArgs a, uint32_t waves) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t w = blockIdx.x * kSumWaves + wave;
    if (w >= waves) return;
    const uint32_t lane = threadIdx.x & 63, chunk = w / a.slabs, slab = w % a.slabs;
    const uint32_t first = chunk * kChunk;
    const Columns c = columns_of(slab * kSlab + lane * 4, a.cols);
    // this chunk's entries in the lanes from 1 on, behind the one before and before the one behind
    const uint32_t at = first + min(lane, kChunk + 1);
    const Entry e = a.sorted[min(at ? at - 1 : 0u, a.rows - 1)];
    const uint32_t count = __builtin_amdgcn_readfirstlane(*a.count);
    if (first >= count) return;
    const uint32_t n = min(kChunk, count - first);
    Raw4<G> v[kChunk];
#pragma unroll
    for (uint32_t k = 0; k < kChunk; ++k) {
        const uint32_t r = (uint32_t)__builtin_amdgcn_readlane((int)e.row, min(k, n - 1) + 1);
        const G* p = (const G*)a.dy + r * a.dy_stride + c.at;
        if constexpr (kNarrow)
            v[k].load_some(p, a.cols);
        else
            v[k].load(p);
    }
    // (or the compiler moves each load to its use, behind the use before it)
#pragma unroll
    for (uint32_t k = 0; k < kChunk; ++k) v[k].here();
    // bit i: entry i continues the run of the one before (of the chunk's: 1 to n; n + 1 is behind)
    const uint32_t left = (uint32_t)__shfl_up((int)e.token, 1);
    const uint64_t same = __ballot(lane && e.token == left);
    const bool enters = first && (same >> 1 & 1);
    const bool leaves = first + n < count && (same >> (n + 1) & 1);
    static_assert(kChunk == 16);
    f32x16 sums[4];  // of this lane's 4 columns
#pragma unroll
    for (uint32_t k = 0; k < kChunk; ++k) {
        const f32x4 x = v[k].values();
        const bool on = k && (same >> (k + 1) & 1);
#pragma unroll
        for (int j = 0; j < 4; ++j) sums[j][k] = on ? sums[j][k ? k - 1 : 0] + x[j] : x[j];
    }
    const auto run = [&](uint32_t k) {  // (k is the same in every lane)
        return f32x4{sums[0][k], sums[1][k], sums[2][k], sums[3][k]};
    };
    if (c.skip == 4) return;
    uint64_t ends = (~same >> 2 | 1ull << (n - 1)) & ((1ull << n) - 1);  // of the chunk's entries
    float* const partial = a.partial + ((uint64_t)chunk * 2 * a.slabs + slab) * kSlab + lane * 4;
    const uint32_t second = a.slabs * kSlab, cols = a.cols;
    const float scale = a.scale;
    const bool first_one = a.first;
    // what crosses the chunk's ends (a run through the whole chunk counts as its first)
    if (enters) {
        *reinterpret_cast<f32x4*>(partial) = run((uint32_t)__builtin_ctzll(ends));
        ends &= ends - 1;
    }
    if (ends && leaves) {
        *reinterpret_cast<f32x4*>(partial + second) = run(n - 1);
        ends &= ~(1ull << (n - 1));
    }
    O* const grad = (O*)a.grad + c.at;
#pragma unroll 1
    while (ends) {
        constexpr int kAtOnce = 4;
        uint32_t k[kAtOnce];
        O* p[kAtOnce];
        Raw4<O> old[kAtOnce];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {  // (the last one again where there are fewer)
            k[j] = ends ? (uint32_t)__builtin_ctzll(ends) : k[j ? j - 1 : 0];
            ends &= ends - 1;
            p[j] = grad + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)e.token, k[j] + 1) *
                              cols;
            if (!first_one) old_row(old[j], p[j], cols);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j)
            if (!j || k[j] != k[j - 1]) put_row(p[j], cols, scale, first_one, c, run(k[j]), old[j]);
    }
}

// The first blocks have the runs that leave the chunk in which they begin: a wave of that chunk adds up
// what the chunks have, in order, four sums in turn.  The others write the zeros.
template <class O>
__global__ __launch_bounds__(256) void join_runs_kernel(GradArgs a, uint32_t waves) {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t joins = (waves + 3) / 4;
    if (blockIdx.x >= joins) {
        for (uint64_t row = ((blockIdx.x - joins) * 4 + wave) * kFillRows; row < a.vocab;
             row += (uint64_t)a.fills * kFillRows)
            fill_zeros<O>(a, (uint32_t)row);
        return;
    }
    const uint32_t w = blockIdx.x * 4 + wave;
    if (w >= waves) return;
    const uint32_t lane = threadIdx.x & 63, chunk = w / a.slabs, slab = w % a.slabs;
    const uint32_t end = (chunk + 1) * kChunk;
    const Columns c = columns_of(slab * kSlab + lane * 4, a.cols);
    // in the lanes: before this chunk, its first and last, the one behind
    const uint32_t which = lane == 0   ? end - kChunk - (chunk ? 1 : 0)
                           : lane == 1 ? end - kChunk
                                       : end - (lane == 2 ? 1 : 0);
    const uint32_t mine = a.sorted[min(which, a.rows - 1)].token;
    const uint32_t count = __builtin_amdgcn_readfirstlane(*a.count);
    if (end >= count) return;
    const uint32_t token = (uint32_t)__builtin_amdgcn_readlane((int)mine, 2);
    if ((uint32_t)__builtin_amdgcn_readlane((int)mine, 3) != token) return;
    if (chunk && (uint32_t)__builtin_amdgcn_readlane((int)mine, 1) == token &&
        (uint32_t)__builtin_amdgcn_readlane((int)mine, 0) == token)
        return;  // it began before
    const auto at = [&](uint32_t k, uint32_t which) {
        return *reinterpret_cast<const f32x4*>(
            a.partial + (((uint64_t)k * 2 + which) * a.slabs + slab) * kSlab + lane * 4);
    };
    f32x4 s0 = at(chunk, 1), s1 = {0.0f, 0.0f, 0.0f, 0.0f}, s2 = s1, s3 = s1;
    for (uint32_t k0 = chunk + 1;; k0 += 64) {
        const uint64_t i = (uint64_t)(k0 + lane) * kChunk;  // where 64 chunks begin
        const bool goes_on = i < count && a.sorted[min(i, (uint64_t)a.rows - 1)].token == token;
        const uint32_t n = __ffsll(~__ballot(goes_on)) ? __ffsll(~__ballot(goes_on)) - 1 : 64;
        uint32_t k = 0;
#pragma unroll 4
        for (; k + 8 <= n; k += 8) {
            const uint32_t i = k0 + k;
            const f32x4 v0 = at(i, 0), v1 = at(i + 1, 0), v2 = at(i + 2, 0), v3 = at(i + 3, 0);
            const f32x4 v4 = at(i + 4, 0), v5 = at(i + 5, 0), v6 = at(i + 6, 0), v7 = at(i + 7, 0);
            s0 += v0, s1 += v1, s2 += v2, s3 += v3;
            s0 += v4, s1 += v5, s2 += v6, s3 += v7;
        }
        for (; k < n; ++k) s0 += at(k0 + k, 0);
        if (n < 64) break;
    }
    if (c.skip == 4) return;
    O* p = (O*)a.grad + (uint64_t)token * a.cols + c.at;
    Raw4<O> old;
    if (!a.first) old_row(old, p, a.cols);
    put_row(p, a.cols, a.scale, a.first, c, (s0 + s1) + (s2 + s3), old);
}

// Few tokens, in one launch (embedding_cut.hpp): a wave has `keys` rows of the gradient and a slab of
// their columns, and looks through all tokens for those rows.  Where there are none, the waves of these
// rows share their zeros; else each row's list goes through the LDS, and its rows of dy are added up 16
// at a time, in eight sums.  Up to 512 tokens, us (sorted / so): 500 x 768 into 50257 rows bf16 31.5 /
// 19.5 and fp32 40.1 / 33.0 (the zeros alone 13.0 and 29.1), 300 x 1600 into 5000 rows 23.8 / 11.7, 200 x
// 384 into 65 rows 18.2 / 11.7; slower only where most of them are one token, whose list is one wave's a
// slab (512 x 384 in full: 18 / 25).
constexpr uint32_t kFewTokens = 512, kFewWords = kFewTokens / 64;
template <class G, class O, bool kNarrow>
__global__ __launch_bounds__(64 * kSumWaves) void few_rows_kernel(GradArgs a, uint32_t waves) {
    __shared__ uint32_t lists[kSumWaves][kFewTokens];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t w = blockIdx.x * kSumWaves + wave;
    if (w >= waves) return;
    const uint32_t lane = threadIdx.x & 63, slab = w % a.slabs;
    const uint32_t row0 = a.row0 + w / a.slabs * a.keys, n = min(a.keys, a.vocab - row0);
    const Columns c = columns_of(slab * kSlab + lane * 4, a.cols);
    uint32_t* const list = lists[wave];
    int64_t token[kFewWords];
#pragma unroll
    for (uint32_t k = 0; k < kFewWords; ++k)
        token[k] = k * 64 + lane < a.rows ? a.tokens[k * 64 + lane] : -1;
    uint32_t key[kFewWords];  // of this wave's rows; n: none of them
#pragma unroll
    for (uint32_t k = 0; k < kFewWords; ++k)
        key[k] = token[k] >= (int64_t)row0 && token[k] < (int64_t)(row0 + n)
                     ? (uint32_t)token[k] - row0
                     : n;
    bool any = false;
#pragma unroll
    for (uint32_t k = 0; k < kFewWords; ++k) any |= key[k] != n;
    O* p = (O*)a.grad + (uint64_t)row0 * a.cols;
    if (!__ballot(any)) {  // (so in the other slabs of these rows: each has a share of them all)
        if (!a.first) return;
        const uint64_t all = (uint64_t)n * a.cols;
        const float zeros[8] = {};
        for (uint64_t at = ((uint64_t)slab * 64 + lane) * 8; at < all; at += (uint64_t)a.slabs * 512)
            store_cols(p + at, 0, (uint32_t)min(all - at, 8ul), zeros);
        return;
    }
    const G* const dy = (const G*)a.dy + c.at;
    p += c.at;
    for (uint32_t i = 0; i < n; ++i, p += a.cols) {
        uint32_t count = 0;
#pragma unroll
        for (uint32_t k = 0; k < kFewWords; ++k) {
            const uint64_t m = __ballot(key[k] == i);
            if (key[k] == i) list[count + __popcll(m & ((1ull << lane) - 1))] = k * 64 + lane;
            count += __popcll(m);
        }
        if (!count && !a.first) continue;
        __builtin_amdgcn_wave_barrier();
        Raw4<O> old;
        if (!a.first) old_row(old, p, a.cols);
        f32x4 sums[8] = {};
        for (uint32_t k0 = 0; k0 < count; k0 += 16) {
            const uint32_t mine = list[min(k0 + (lane & 15), count - 1)];
            Raw4<G> v[16];
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k) {
                const G* q = dy + (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)mine, k) *
                                      a.dy_stride;
                if constexpr (kNarrow)
                    v[k].load_some(q, a.cols);
                else
                    v[k].load(q);
            }
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k) v[k].here();
            if (k0 + 16 <= count) {
#pragma unroll
                for (uint32_t k = 0; k < 16; ++k) sums[k % 8] += v[k].values();
            } else {
#pragma unroll
                for (uint32_t k = 0; k < 16; ++k)
                    if (k0 + k < count) sums[k % 8] += v[k].values();
            }
        }
        __builtin_amdgcn_wave_barrier();
        if (c.skip < 4)
            put_row(p, a.cols, a.scale, a.first, c,
                    ((sums[0] + sums[1]) + (sums[2] + sums[3])) +
                        ((sums[4] + sums[5]) + (sums[6] + sums[7])),
                    old);
    }
}

template <class G, class O>
int add_few_rows(const ttpi::Op& op, GradArgs a) {
    const FewRowsCut cut = cut_few_rows(a.vocab, a.slabs, (uint64_t)op.num_cus);
    a.keys = cut.keys;
    for (uint64_t r = 0; r < a.vocab; r += cut.rows) {
        const uint64_t rows = std::min<uint64_t>(cut.rows, a.vocab - r);
        a.row0 = (uint32_t)r;
        const uint32_t waves = (uint32_t)((rows + a.keys - 1) / a.keys) * a.slabs;
        const dim3 grid((waves + kSumWaves - 1) / kSumWaves), block(64 * kSumWaves);
        (void)hipGetLastError();
        if (a.cols < 4)
            hipLaunchKernelGGL((few_rows_kernel<G, O, true>), grid, block, 0, op.stream, a, waves);
        else
            hipLaunchKernelGGL((few_rows_kernel<G, O, false>), grid, block, 0, op.stream, a, waves);
        TTPI_HIP(hipGetLastError());
    }
    return TTP_OK;
}

template <class G, class O>
int add_rows(const ttpi::Op& op, const GradArgs& a) {
    (void)hipGetLastError();
    hipLaunchKernelGGL(sort_tokens_kernel, dim3(1u << a.parts_log2), dim3(kSortBlock), 0, op.stream, a);
    TTPI_HIP(hipGetLastError());
    const uint32_t chunks = (uint32_t)(((uint64_t)a.rows + kChunk - 1) / kChunk);
    const uint32_t waves = chunks * a.slabs;  // (fewer than 2^25)
    const dim3 sums((waves + kSumWaves - 1) / kSumWaves);
    if (waves && a.cols < 4)
        hipLaunchKernelGGL((sum_rows_kernel<G, O, true>), sums, dim3(64 * kSumWaves), 0, op.stream, a,
                           waves);
    else if (waves)
        hipLaunchKernelGGL((sum_rows_kernel<G, O, false>), sums, dim3(64 * kSumWaves), 0, op.stream, a,
                           waves);
    TTPI_HIP(hipGetLastError());
    const uint32_t joins = chunks > 1 ? waves : 0;
    if (a.fills || joins) {
        hipLaunchKernelGGL(join_runs_kernel<O>, dim3(a.fills / 4 + (joins + 3) / 4), dim3(256), 0,
                           op.stream, a, joins);
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
    return b.own(p->data, p->numel, p->bf16 ? 2 : 4, what, false);
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
        if (vocab >= (1ull << 30))
            return fail(TTP_ERR_RANGE, "the table has 2^30 rows or more");
        ttpi::Buffers b(ctx);
        if ((rc = b.array(tokens, rows, 8, "the tokens", false))) return rc;
        if ((rc = b.matrix(dy, rows, cols, "the output's gradient", false))) return rc;
        if ((rc = b.own(g.data, g.numel, g.bf16 ? 2 : 4, "the table's gradient", true)))
            return rc;
        GradArgs a{};
        a.tokens = tokens;
        a.dy = dy->data;
        a.dy_stride = dy->stride;
        a.rows = (uint32_t)rows;
        a.cols = (uint32_t)cols;
        a.vocab = (uint32_t)vocab;
        // blocks: as many as there are CUs (or tokens), more where their counters would not do
        const uint64_t blocks = std::min<uint64_t>((uint64_t)op.num_cus, vocab);
        while ((1ull << a.parts_log2) < blocks ||
               (vocab + (1ull << a.parts_log2) - 1) >> a.parts_log2 > kMostKeys)
            ++a.parts_log2;
        a.keys = (uint32_t)((vocab + (1ull << a.parts_log2) - 1) >> a.parts_log2);
        a.slabs = (a.cols + kSlab - 1) / kSlab;
        a.scale = (float)scale;
        a.grad = g.data;
        a.first = g.first;
        const bool bf16 = dy->dtype == TTP_DTYPE_BF16;
        if (rows <= kFewTokens) {
            if (g.bf16)
                rc = bf16 ? add_few_rows<uint16_t, uint16_t>(op, a)
                          : add_few_rows<float, uint16_t>(op, a);
            else
                rc = bf16 ? add_few_rows<uint16_t, float>(op, a) : add_few_rows<float, float>(op, a);
            if (rc) return rc;
            ttpi::grad_written(ctx, table);
            return TTP_OK;
        }
        const uint64_t chunks = (rows + kChunk - 1) / kChunk;
        if (chunks * a.slabs >= (1ull << 25))
            return fail(TTP_ERR_RANGE, "the output's gradient is too large for one launch");
        // partial sums, listed and sorted entries, which tokens there are, the entries' count
        const uint64_t partial = chunks * 2 * a.slabs * kSlab * 4;
        const uint64_t named = ((uint64_t)(a.keys + 63) / 64) << a.parts_log2;
        void* ws;
        if ((rc = ttpi::workspace(ctx, partial + 2 * rows * sizeof(Entry) + named * 8 + 16, &ws)))
            return rc;
        a.partial = (float*)ws;
        a.listed = (Entry*)((char*)ws + partial);
        a.sorted = a.listed + rows;
        a.named = (uint64_t*)(a.sorted + rows);
        a.count = (uint32_t*)(a.named + named);
        const uint64_t fills = (vocab + 4 * kFillRows - 1) / (4 * kFillRows) * 4;
        if (a.first) a.fills = (uint32_t)std::min<uint64_t>(fills, 1u << 20);
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
