// Offsets (key position - query position) and the bias table that the kernels of battn_fwd.hip and battn_bwd.hip keep of
// them in LDS: its extent, and which 32 x 32 blocks read it.
#pragma once

namespace gt {

// The table holds the offsets -dsat - EXT .. dsat + EXT, under a causal mask .. EXT.
constexpr int EXT = 64;
constexpr int ext_entries(int dsat, bool causal) { return dsat + 2 * EXT + 1 + (causal ? 0 : dsat); }

// A block with the offsets dmin .. dmax (32 keys, 32 consecutive queries) takes one constant where all of them share it:
// beyond the last border, or, under a causal mask, ahead of every query (none of its keys is seen). Any other block has
// an offset inside (-dsat, dsat), causal: inside (-dsat, 0], and so all of its 63 offsets in the table.
constexpr bool one_bias(int dmin, int dmax, int dsat, bool causal) {
  return dmax <= -dsat || dmin >= (causal ? 1 : dsat);
}

}  // namespace gt
