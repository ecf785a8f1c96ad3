// How the logits of mi_beam_select (beam.hip) are cut up, and what fits where between its launches.  Plain C++.
#pragma once
#include <cstddef>
#include <cstdint>

namespace mi {

// A wavefront takes a tile of 4096 logits of a row, 64 to a lane, and leaves the sum of their exponentials and the greatest of each lane's.
constexpr int kTile = 4096, kBins = 64;
constexpr int kMostBeams = 64, kMostOut = 64;

constexpr int tiles_of_row(int vocab) { return (vocab + kTile - 1) / kTile; }
// Lane `lane`'s `e`-th logit of tile `tile` (e = 0 .. 63): pieces of 8 neighbours, the lanes' side by side.
constexpr int token_of(int tile, int lane, int e) { return tile * kTile + e / 8 * (8 * kBins) + lane * 8 + e % 8; }

// Of a tile between the launches: the sum and what it is relative to, and the bins' maxima.
constexpr size_t kTileBytes = 2 * sizeof(float) + kBins * sizeof(uint16_t);

// Groups whose tiles fit `bytes`; 0: not even one does.
constexpr int64_t groups_that_fit(size_t bytes, int beams, int vocab) {
    return static_cast<int64_t>(bytes / (kTileBytes * static_cast<size_t>(beams) * static_cast<size_t>(tiles_of_row(vocab))));
}

// fp16 bits as numbers that ascend with the value: both zeros alike, -infinity below kLeast, all finite ones from there on.
constexpr uint32_t kLeast = 0x0400;
constexpr uint32_t ascending(uint32_t h) { return h == 0x8000u ? 0x8000u : h & 0x8000u ? 0xffffu & ~h : h | 0x8000u; }
constexpr uint32_t half_bits(uint32_t a) { return a & 0x8000u ? a & 0x7fffu : 0xffffu & ~a; }

}  // namespace mi
