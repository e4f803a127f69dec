// How a call of attention over whole prompts is run (prompt.hip), from what the host knows of it.
#pragma once
#include "kv4_attend.hpp"

namespace hck {

constexpr int kRowsOfWave = 32, kPromptWaves = 4, kTileRows = kRowsOfWave * kPromptWaves;
constexpr int kPieces(int dim) { return 1 + dim / 8; }  // of a lane in a slot

// The parts that a tile of so many units comes in where a call has room for `parts` of `part` units each, and where one ends.  A
// tile may have more units than that: without `causal` its rows see all of a sequence, however little of it `most` allows for.
// The last part takes what is left then.
constexpr int parts_of(int units, int part, int parts) { return std::min((units - 1) / part + 1, parts); }
constexpr int part_end(int units, int part, int parts, int p) { return p == parts - 1 ? units : std::min(units, (p + 1) * part); }

// How a call is run, from what the host knows of it.
struct WholeWay {
  int64_t items;
  int tiles, part, parts;
  WholeWay(int64_t tokens, int64_t seqs, int heads, int group, int most, bool causal) {
    tiles = (int)(((int64_t)most * group + kTileRows - 1) / kTileRows);
    // every sequence has a tile that may not be full, beside the full ones
    items = std::min((int64_t)tiles * seqs, tokens * group / kTileRows + seqs);
    // Few tiles of long sequences are cut into parts, as many as run at once and no more: of the tiles of one sequence with
    // `causal` that is longest / 2 / part + 1 / 2 for each; of several, whose lengths the host does not know, half as many parts
    // are reckoned with.  A part costs its sums' way through memory and the join some 5 us, which
    // is what 8 units take (one sequence, 128 dims, whole and in parts: 4000 tokens, 6 heads over 2, 85 and 53 us; 6000, 8 over
    // 4, 144 and 105; 2000, 32 over 8, in more parts than run at once, 53 and 72).
    const int64_t longest = ((int64_t)most + kUnit - 1) / kUnit, each = items * heads;
    int64_t units = longest;
    if (causal && 2 * kSlots > each) units = (longest / (seqs > 1 ? 2 : 1) * each + 2 * kSlots - each - 1) / (2 * kSlots - each);
    if (!causal && kSlots > each) units = (longest + kSlots / each - 1) / (kSlots / each);
    part = (int)std::min(longest, std::max<int64_t>(kLeast, units));
    parts = longest > part + kJoin ? parts_of((int)longest, part, INT32_MAX) : 1;
  }
  size_t bytes(int heads, int dim) const {
    return parts > 1 ? (size_t)items * parts * heads * (kPromptWaves * 64 * kPieces(dim)) * sizeof(f32x4) : 0;
  }
  static constexpr int kSlots = 2 * kComputeUnits, kLeast = 8, kJoin = 8;
};

}  // namespace hck
