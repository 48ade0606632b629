// Which tiles a workgroup that stays takes, in plain C++ (constexpr: host and device alike), so that the ends can be tried on the
// host: the counts come from offsets on the device, and the loop over a span has to end whatever those are.
#pragma once
#include <stdint.h>

namespace bh {

struct TileSpan {
    uint32_t at, end, step;  // tiles at, at + step, ... below end
};

// Of row_tiles x columns tiles, the first `most` (below 2^31) at most: workgroups go to the 8 XCDs in turn, XCD i gets the i-th
// eighth of the tiles, its workgroups tile by tile in turn. `workgroups` is a multiple of 8. at + step does not wrap.
constexpr TileSpan tile_span(uint32_t row_tiles, uint32_t columns, uint32_t most, uint32_t workgroup, uint32_t workgroups) {
    const uint64_t all = (uint64_t)row_tiles * columns, tiles = all < most ? all : most;
    const uint64_t share = (tiles + 7) / 8, from = (workgroup & 7) * share;
    return {(uint32_t)(from + (workgroup >> 3)), (uint32_t)(from + share < tiles ? from + share : tiles), workgroups >> 3};
}

}  // namespace bh
