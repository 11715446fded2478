// embedding_cut.hpp — how an embedding gradient of few tokens is cut into waves and launches (host
// code, of numbers alone).
#pragma once

#include <stdint.h>

#include <algorithm>

namespace ttp {
namespace {

struct FewRowsCut {
    uint32_t keys;  // rows of the table that a wave has
    uint64_t rows;  // of a launch: whole waves, fewer than 2^32 work-items
};

// Rows of a wave: as many as leave the CUs 16 waves each, up to 8 (with 16, 256 neighbouring tokens of
// 50257 took 28 us instead of 17).  A launch has up to 2^25 waves: only tables of 2^28 rows or more, or
// of as many slabs, take a second one.
inline FewRowsCut cut_few_rows(uint64_t vocab, uint64_t slabs, uint64_t cus) {
    constexpr uint64_t kMostWaves = 1u << 25;
    const uint64_t keys =
        std::max<uint64_t>(std::min<uint64_t>(vocab * slabs / (16 * cus), 8), 1);
    return {(uint32_t)keys, std::max<uint64_t>(kMostWaves / slabs, 1) * keys};
}

}  // namespace
}  // namespace ttp
