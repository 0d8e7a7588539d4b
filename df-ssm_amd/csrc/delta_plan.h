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

}  // namespace dfssm
