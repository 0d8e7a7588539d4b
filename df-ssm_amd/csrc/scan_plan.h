// Arithmetic of the chunked selective scan's launches, for the host and the device alike (constexpr functions serve both),
// with nothing of HIP in it.
#pragma once
#include <stdint.h>

#include "places.h"

namespace dfssm {

constexpr int kScanChunk = 64;  // tokens of a chunk
constexpr int kScanCols = 32;   // columns p of a wave
constexpr int kScanWaves = 4;   // waves of a workgroup, which share B and C

// Workgroups of a sequence (or a segment of one): each has up to four blocks of 32 columns of one group's heads.
constexpr int64_t scan_wgs(int H, int G, int P) {
  const int64_t blocks = (int64_t)(H / G) * ((P + kScanCols - 1) / kScanCols);
  return G * ((blocks + kScanWaves - 1) / kScanWaves);
}

// Tokens of a segment. A sequence longer than that is cut into segments that run beside each other, from states
// that a pass over all but the last of them makes first: about 768 workgroups, where two are resident on each of 256 CUs. Fewer
// leave CUs idle where sequences are unequal, more have longer chains and more states to move. (With 512, 768, 1024 and 1536, in
// replayed graphs: 16411 tokens x 64 heads 232, 242, 259 and 277 us; twelve ragged sequences 199, 175, 171 and 176; 64 x 512
// tokens x 80 heads, cut by none, 447, 448, 445 and 446.)
constexpr int64_t scan_segment(int64_t n_tokens, int n_seq, int64_t wgs) {
  const int64_t chunks = n_tokens / kScanChunk + n_seq;
  int64_t m = (chunks * wgs + 768 - 1) / 768;
  m = m < 4 ? 4 : m;
  return m * kScanChunk;
}

// Segments of a sequence of `len` tokens; one of an empty sequence, whose state is passed on. (Tokens and segments fit 31 bits.)
constexpr int scan_segments(int64_t len, int seg) { return len > seg ? (int)(((uint32_t)len + seg - 1) / (uint32_t)seg) : 1; }

// Whether a place has a segment of the sequence that was found for it, whose first place is `first`: places behind the
// sequence's last segment have none, nor have those before the first of all sequences, which begins behind row 0 then.
constexpr bool scan_holds(int64_t place, int64_t first, int64_t len, int seg) {
  return place >= first && place - first < scan_segments(len, seg);
}

// Places of the launch's numbering: segments of `seg` tokens, sequence b from place_of(t0, b, seg) on.
constexpr int64_t scan_places(int64_t n_tokens, int n_seq, int64_t seg) { return n_tokens / seg + n_seq; }

}  // namespace dfssm
