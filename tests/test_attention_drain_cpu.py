"""How long the attention kernels' loading threads stay after a wait has run
out, and what they wait for: csrc/ring_drain.h, compiled for the host and run
against a ring whose barriers and clock are made up."""
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "drama3_offloading_b200" / "csrc"

MAIN = r"""
#include "ring_drain.h"
#include <cstdio>
#include <vector>

// A ring of n slots after m loads.  A barrier's wait for a parity returns at
// once if the phase of that parity is over: phases over so far are counted.
struct Ring {
  std::vector<int> over;
  bool filled(int i, uint32_t parity) const { return ((over[i] - 1) & 1) == (int)parity; }
};

int main() {
  const uint64_t budget = 2000000000ull, step = 20000;
  for (int n : {3, 5, 6, 10})
    for (int m = 0; m < 4 * n; ++m)
      for (int missing = -1; missing < n; ++missing) {
        // every load has landed, but for the last one of slot `missing`
        Ring r;
        for (int i = 0; i < n; ++i) {
          const int loads = m / n + (i < m % n ? 1 : 0);
          r.over.push_back(loads - (i == missing && loads > 0 ? 1 : 0));
        }
        const bool whole = missing < 0 || (m / n + (missing < m % n ? 1 : 0)) == 0;
        uint64_t t = 77;
        int asked_behind = 0;
        const bool all = d3::drain_ring(
            n, m % n, (uint32_t)(m / n) & 1, budget,
            [&](int i, uint32_t par) {
              t += r.filled(i, par) ? 0 : step;
              if (missing >= 0 && i > missing) ++asked_behind;
              return r.filled(i, par);
            },
            [&] { return t; });
        if (all != whole) return printf("n %d m %d missing %d: all %d\n", n, m, missing, all), 1;
        if (whole && t != 77) return printf("n %d m %d: waited for nothing\n", n, m), 1;
        if (!whole && (t - 77 > budget + (n + 1) * step || t - 77 < budget)) return printf("n %d m %d: %f s\n", n, m, (t - 77) * 1e-9), 1;
        if (missing >= 0 && missing < n - 1 && !asked_behind) return printf("slots behind the missing one left out\n"), 1;
      }
  // no slot ever fills: one budget, not one a slot
  uint64_t t = 0;
  if (d3::drain_ring(10, 4, 1, budget, [&](int, uint32_t) { t += step; return false; }, [&] { return t; })) return 2;
  if (t > budget + 20 * step) return printf("%f s for ten slots\n", t * 1e-9), 1;
  return 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_a_drain_takes_one_budget_and_waits_for_what_was_asked_for(tmp_path):
    (tmp_path / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-Wall", "-Werror", "-I", str(CSRC), "-o", str(tmp_path / "drain"),
                    str(tmp_path / "main.cpp")], check=True)
    run = subprocess.run([str(tmp_path / "drain")], capture_output=True, text=True)
    assert run.returncode == 0, run.stdout


def test_no_loading_thread_waits_a_budget_a_slot():
    """Both kernels drain by it: no loop of whole waits over the slots."""
    for name in ("attn_rows.cuh", "attn_chunk.cuh"):
        src = (CSRC / name).read_text()
        assert "drain_ring(" in src
        for loop in src.split("for (int i = 0; i < ")[1:]:
            body = loop.splitlines()[0]
            assert "mbar_wait(" not in body, body
