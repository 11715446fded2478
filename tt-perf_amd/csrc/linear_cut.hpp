// linear_cut.hpp — how a linear product is cut into tiles and parts (host code, of numbers alone).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace ttp {

// The shapes of linear_direct_kernel and the two of any alignment.
enum class LinearShape { kThin, kSmall, kWide, kLarge, kThinAny, kAny };

namespace {

// What a tile costs, fitted to measurements (100 products, each in 1 to 24 parts): ns per step of
// a block that has the GPU to itself, and of each where as many are on it as fit; ns before its first
// step and behind its last one.
struct LinearCost {
    LinearShape shape;
    uint32_t rows, outs, step, per_cu;
    double alone, shared, ends;
};

struct LinearCut {
    LinearShape shape;
    uint32_t tile_rows, tile_outs;
    uint32_t parts, per;  // parts of the summed index, and its elements in each
    double ns;            // what it should take
};

constexpr uint32_t kThinRows = 32;  // a token or a few: a matrix is read for them

// The number of parts that should take the least time.  A part has three steps or more; parts cost
// their fp32 sums' way to the caches and back, at about 12 TB/s, and a launch: 2.5 us of the GPU and 3
// of the host, which bounds short calls.  (What this chooses takes 3% more than the best of those
// measured; bf16 on the grid, 0.1%.)
inline LinearCut cut_parts(uint64_t rows, uint64_t cols, uint64_t outs, const LinearCost& c,
                           uint64_t cus) {
    LinearCut best{c.shape, c.rows, c.outs, 0, 0, 0.0};
    const uint64_t tiles = ((rows + c.rows - 1) / c.rows) * ((outs + c.outs - 1) / c.outs);
    const uint64_t steps = (cols + c.step - 1) / c.step, slots = c.per_cu * cus;
    const uint64_t most =
        tiles >= slots ? 1 : std::max<uint64_t>(std::min<uint64_t>(steps / 3, 32), 1);
    for (uint64_t n = 1; n <= most; ++n) {
        const uint64_t per = (steps + n - 1) / n, parts = (steps + per - 1) / per;
        const uint64_t blocks = tiles * parts, left = blocks % slots;
        double ns = (double)(blocks / slots) * (c.shared * (double)per + c.ends);
        if (left)
            ns += (c.alone + (c.shared - c.alone) * (double)left / (double)slots) * (double)per + c.ends;
        if (parts > 1) ns += 4500.0 + 8.0 * (double)parts * (double)rows * (double)outs / 12e3;
        if (n == 1 || ns < best.ns) {
            best.ns = ns;
            best.parts = (uint32_t)parts;
            best.per = (uint32_t)(per * c.step);
        }
    }
    return best;
}

// The fastest shape of those that the operands allow.
// Measured, bf16, us as called (W as it is / transposed): 8192 x 1280 x 5120 large 134 / 126, wide 117 /
// 127, small 124 / 124, any alignment 167; 8192 x 5120 x 1280 large 100 / 89, wide 122 / 141, small 131 /
// 125, any 181; 4096 x 1600 x 6400 large 108, wide 95, small 103; 2048 x 6400 x 1600 large 85 in one part
// and 54 in three, small 72; 1024 x 768 x 2304 small 14, large 23; 128 x 6401 x 1601 any 114 in one part,
// 22 in twelve.
inline LinearCut choose_linear_cut(uint64_t rows, uint64_t cols, uint64_t outs, bool direct,
                                   bool bf16, bool transposed, uint64_t cus) {
    using S = LinearShape;
    if (!direct) {
        // (1 x 768 x 50257 transposed fp32: thin 35 us, the other 64; 64 rows 56 and 67, 96 rows 73 and
        // 67; bf16 769 columns, 32 rows: 20 and 25, 33 rows 30 and 25)
        if (rows <= (bf16 ? kThinRows : 2 * kThinRows)) {
            const LinearCost thin =
                bf16 ? LinearCost{S::kThinAny, 32, 128, 32, 4, 290.0, 1410.0, 2400.0}
                     : LinearCost{S::kThinAny, 32, 128, 32, 4, 800.0, 2410.0, 2600.0};
            return cut_parts(rows, cols, outs, thin, cus);
        }
        const LinearCost any = bf16 ? LinearCost{S::kAny, 128, 128, 32, 2, 370.0, 780.0, 6700.0}
                                    : LinearCost{S::kAny, 128, 128, 32, 2, 1430.0, 2690.0, 6800.0};
        return cut_parts(rows, cols, outs, any, cus);
    }
    if (rows <= kThinRows)
        return cut_parts(rows, cols, outs, {S::kThin, 32, 64, 64, 3, 116.0, 530.0, 2100.0}, cus);
    LinearCut best =
        cut_parts(rows, cols, outs, {S::kSmall, 128, 128, 64, 2, 375.0, 920.0, 5900.0}, cus);
    for (const LinearCost& c :
         {LinearCost{S::kWide, 128, 256, 32, 2, transposed ? 283.0 : 248.0, transposed ? 944.0 : 828.0,
                     10800.0},
          LinearCost{S::kLarge, 256, 160, 64, 1, 495.0, 911.0, 13100.0}}) {
        const LinearCut cut = cut_parts(rows, cols, outs, c, cus);
        if (cut.ns < best.ns) best = cut;
    }
    return best;
}

}  // namespace
}  // namespace ttp
