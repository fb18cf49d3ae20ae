"""What a run of neighbouring rows sees together (CPU: the rule of
stride_amd/csrc/serve_sight.hpp built for the host). The tiles of windowed attention fetch
[0, the furthest row's sinks) and [the nearest row's window, the furthest row]; every position
there must be seen by some row of the run, since the pages of others may be gone."""
import os
import subprocess

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "stride_amd", "csrc")

PROBE = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "serve_sight.hpp"
using namespace stride_tc;
bool by_slot(int a, int, int b, int, int) { return a == b; }
template <class F>
long unseen(F together) {
  long bad = 0;
  srand(1);
  const int limit = 200;
  for (int round = 0; round < 20000; ++round) {
    const int rows = 1 + rand() % 9, windows[] = {0, 1, 2, 7, 30, 199, 2147483647}, window = windows[rand() % 7], sinks = rand() % 3 * (rand() % 220);
    std::vector<int> slot(rows), pos(rows);
    for (int j = 0; j < rows; ++j) {
      const int how = rand() % 6;
      slot[j] = j && how ? slot[j - 1] : rand() % 3 - 1;
      pos[j] = how == 1 ? -1 : how < 4 && j ? pos[j - 1] + rand() % 3 - (how == 3) : rand() % (limit + 20) - 5;
      if (pos[j] > limit - 1) pos[j] = limit - 1;
      if (pos[j] < -1 || slot[j] < 0) pos[j] = -1;
    }
    for (int r0 = 0, r1; r0 < rows; r0 = r1) {
      for (r1 = r0 + 1; r1 < rows && together(slot[r1 - 1], pos[r1 - 1], slot[r1], pos[r1], window); ++r1) {}
      int low = limit, high = -1;
      for (int j = r0; j < r1; ++j)
        if (pos[j] >= 0) low = pos[j] < low ? pos[j] : low, high = pos[j] > high ? pos[j] : high;
      if (high < 0) continue;
      const Sight near = sight_at(low, window, sinks, limit), far = sight_at(high, window, sinks, limit);
      for (int t = 0; t <= high; ++t) {
        bool some = false;
        for (int j = r0; j < r1; ++j) some = some || sight_at(pos[j], window, sinks, limit).sees(t);
        bad += some != (t < far.sink_end || t >= near.lo);
      }
    }
  }
  return bad;
}
int definition() {  // t <= p and (window <= 0, or p - t < window, or t < sinks)
  int bad = 0;
  for (int window : {-2147483647 - 1, 0, 1, 5, 60, 2147483647})
    for (int sinks : {0, 1, 9, 70, 2147483647})
      for (int p = -1; p < 70; ++p)
        for (int t = 0; t < 70; ++t) {
          const int at = p < 64 ? p : 63;
          bad += sight_at(p, window, sinks, 64).sees(t) != (t <= at && (window <= 0 || at - t < window || t < sinks));
        }
  return bad;
}
int main() { printf("%d %d %ld %ld\n", definition(), one_run(1, 2147483390, 1, -1, 5), unseen(one_run), unseen(by_slot)); }
"""


def test_a_run_sees_all_that_is_fetched_for_it(tmp_path):
    src, exe = tmp_path / "probe.cpp", tmp_path / "probe"
    src.write_text(PROBE)
    subprocess.run(["g++", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    wrong, joined, bad, by_slot = map(int, subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split())
    assert wrong == 0 and joined == 0
    assert by_slot > 0  # rows of one slot with a gap between their windows would fetch what none sees
    assert bad == 0


def test_the_kernels_use_the_rule():
    text = open(os.path.join(CSRC, "serve_attn.hip")).read()
    tile = text[text.index("void k_tile("):text.index("auto next_run")]
    assert "one_run(slots[t - 1], poss[t - 1], slots[t], poss[t], p.window)" in tile and "slots[t] != slots[t - 1]" not in tile
    rows = text[text.index("bool unit_done("):text.index("void k_rows(")]
    assert "one_run(p.row_slot[i - 1]" in rows and "p.row_slot[i] != p.row_slot[i - 1]" not in rows
