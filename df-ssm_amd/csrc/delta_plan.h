// Arithmetic of the chunked delta rule's launches, for the host and the device alike (constexpr functions serve both),
// with nothing of HIP in it.
#pragma once
#include <stdint.h>

namespace dfssm {

// A launch goes over the chunks in slots [slot0, slot1) of the call's chunk numbering, whose records are held at once.
// Of a sequence with chunks in slots [first, first + nch): the first chunk and the number that the launch has. None for
// one that lies before or behind it, whatever its length.
struct PassChunks {
  int64_t begin;
  int64_t count;
};
constexpr PassChunks pass_chunks(int64_t first, int64_t nch, int64_t slot0, int64_t slot1) {
  int64_t begin = slot0 - first, end = slot1 - first;
  begin = begin < 0 ? 0 : begin;
  end = end > nch ? nch : end;
  return PassChunks{begin, end > begin ? end - begin : 0};
}

// Tiles of 16 value columns to a workgroup of the chain, of `heads` sequences times value heads and `tiles` tiles a head.
// Few: one, so that all CUs have one or two and a chunk passes quickly. Many: four, which make P once for 64 columns.
// With 1, 2, 4: 64 heads of 4 tiles, 16411 tokens 593, 695 and 890 us; 12 x 2 heads of 8 tiles 227, 264 and 327; 12 x 64
// heads of 4, ragged, 367, 234 and 211; 64 x 80 heads of 4 tiles 1884, 1235 and 1005.
constexpr int chain_tiles(int64_t heads, int64_t tiles) {
  return heads * ((tiles + 1) / 2) <= 256 ? 1 : (heads * ((tiles + 3) / 4) <= 256 ? 2 : 4);
}

}  // namespace dfssm
