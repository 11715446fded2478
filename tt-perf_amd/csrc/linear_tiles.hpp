// linear_tiles.hpp — how a linear gradient's work is cut into tiles and parts (host code, of
// numbers alone).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace ttp {
namespace {

constexpr uint32_t kWideTile = 256, kNarrowTile = 128;  // columns and outputs of a tile
constexpr uint32_t kStepRows = 32;                      // rows of a step

// What a tile costs, measured: ns per row of a block that has its CU to itself, and of two that
// share one; and ns before its first and behind its last step.  The wide tile moves half the bytes
// per operation, the narrow one wastes less of a small gradient and needs fewer parts.
// (8192 x 1280 x 5120 bf16: 137 us with wide tiles, 175 with narrow ones; 16384 x 1600 x 1600: 118
// and 133; 4096 x 384 x 1536: 34 and 26.)
struct Cost {
    double one, two, ends;
};
constexpr Cost kWideCost{30.0, 60.0, 8000.0}, kNarrowCost{15.0, 22.0, 4000.0},
    kPlanesCost{30.0, 56.0, 4000.0};

struct Cut {
    bool wide;
    uint32_t tiles_a, tiles_b, parts;
    uint64_t per;  // rows of a part (a whole number of steps)
    double ns;     // what it should take
};

// Cuts the work into tiles and the rows into parts of 128 or more: the number of parts that should
// take the least time.  Parts cost their fp32 tiles' way to memory and back, about 5 TB/s, a
// launch, and the join's loads one after the other.
inline Cut cut_rows(uint64_t rows, uint32_t cols, uint32_t outs, uint32_t tile, uint64_t cus,
                    const Cost& c) {
    Cut best{tile == kWideTile, (cols + tile - 1) / tile, (outs + tile - 1) / tile, 0, 0, 0.0};
    const uint64_t tiles = (uint64_t)best.tiles_a * best.tiles_b;
    const uint64_t most = std::max<uint64_t>(std::min<uint64_t>(rows / 128, 64), 1);
    for (uint64_t n = 1; n <= most; ++n) {
        const uint64_t per = ((rows + n - 1) / n + kStepRows - 1) / kStepRows * kStepRows;
        const uint64_t parts = per ? std::max<uint64_t>((rows + per - 1) / per, 1) : 1;
        const uint64_t blocks = tiles * parts, left = blocks % (2 * cus);
        double ns = (double)(blocks / (2 * cus)) * (c.two * (double)per + c.ends);
        if (left) ns += (left > cus ? c.two : c.one) * (double)per + c.ends;
        if (parts > 1)
            ns += 3000.0 + 150.0 * (double)parts + 8.0 * (double)parts * cols * outs / 5e3;
        if (n == 1 || ns < best.ns) {
            best.ns = ns;
            best.per = per;
            best.parts = (uint32_t)parts;
        }
    }
    return best;
}

// The faster of the tiles there are: both for a bf16 dy, the narrow one for an fp32 one, whose
// three products each are a cost of its own.
inline Cut choose_cut(uint64_t rows, uint32_t cols, uint32_t outs, bool bf16, uint64_t cus) {
    const Cut narrow =
        cut_rows(rows, cols, outs, kNarrowTile, cus, bf16 ? kNarrowCost : kPlanesCost);
    if (!bf16) return narrow;
    const Cut wide = cut_rows(rows, cols, outs, kWideTile, cus, kWideCost);
    return wide.ns < narrow.ns ? wide : narrow;
}

}  // namespace
}  // namespace ttp
