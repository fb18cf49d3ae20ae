// What rows of windowed attention see, alone and together (plain C++: the tests build it for
// the host).
#pragma once

namespace stride_tc {

// A row sees [0, sink_end) and [lo, pos]; pos = -1: nothing.
struct Sight {
  int pos, lo, sink_end;
  constexpr bool sees(int t) const { return t <= pos && (t >= lo || t < sink_end); }
};

constexpr Sight sight_at(int pos, int window, int sinks, int limit) {
  const int p = pos < limit - 1 ? pos : limit - 1;
  if (window <= 0) return {p, 0, 0};
  const int from = p - window + 1;
  return {p, from > 0 ? from : 0, sinks < p + 1 ? sinks : p + 1};
}

// Do row b and row a before it belong to one run of a tile, whose rows' keys and values are
// fetched together from the first to the last position that a window holds? Where they are of
// one sequence and no position between their windows is seen by neither: pages there may be
// gone. Positions are below the limit, -1 without one; such a row's neighbours see from 0 on
// where it is in their run, so that theirs have no hole either.
constexpr bool one_run(int slot_a, int pos_a, int slot_b, int pos_b, int window) {
  return slot_a == slot_b && (window <= 0 || (pos_a > pos_b ? pos_a - pos_b : pos_b - pos_a) <= window);
}

}  // namespace stride_tc
