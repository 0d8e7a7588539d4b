// The numbering of tiles over packed sequences, for the host and the device alike (constexpr functions serve both), with nothing
// of HIP in it.
#pragma once
#include <stdint.h>

namespace dfssm {

// The place of the first tile of c tokens of sequence b, which begins at token t0.
constexpr int64_t place_of(int64_t t0, int b, int64_t c) { return t0 / c + b; }

// The last of n sequences that starts at or before a place, by as many looks at 64 of them at once as it takes; sequence 0 where
// none does. started(lo, step, end) counts those of sequences lo, lo + step, .. lo + 63 step below `end` that do.
template <class Started>
constexpr int last_started(int n, Started started) {
  int lo = 0;
  while (n > 1) {
    const int step = (n + 63) / 64, end = lo + n, k = started(lo, step, end);  // (the starts rise, so it is the first k)
    lo += (k > 0 ? k - 1 : 0) * step;
    n = step < end - lo ? step : end - lo;
  }
  return lo;
}

}  // namespace dfssm
