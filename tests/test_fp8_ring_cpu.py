"""The bookkeeping of the fp8 product's ring of asynchronous copies (csrc/fp8_ring.cuh), compiled for the host against
a model of the barriers.  No GPU."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "advanced_optimizers_b200", "csrc")

# Two CTAs fill the slots of a ring in order; a slot's barrier completes a phase when both CTAs' parts of a fill have
# landed, and a fill begins once the one before it was used up.  Both stop anywhere.  What is still on its way then has
# to be waited for: a wait for a parity returns at once when the current phase has the other one.
MODEL = r"""
#include <cstdio>
#include <cstdlib>
#include "fp8_ring.cuh"
using namespace advopt::fp8;
int main() {
  const int SLOTS = 3;
  srand(1);
  long outstanding = 0;
  for (int trial = 0; trial < 200000; ++trial) {
    Fills f[2];
    int count[2][SLOTS] = {}, landed[2][SLOTS] = {}, phase[SLOTS] = {}, at[2] = {}, used[2] = {};
    auto settle = [&]() {
      for (int s = 0; s < SLOTS; ++s)
        while (count[0][s] > phase[s] && count[1][s] > phase[s] && landed[0][s] > phase[s] && landed[1][s] > phase[s]) ++phase[s];
    };
    const int steps = rand() % 60;
    for (int i = 0; i < steps; ++i) {
      const int r = rand() & 1, s = at[r] % SLOTS;
      if (rand() % 3 == 0) {                       // something lands
        const int t = rand() % SLOTS;
        if (landed[r][t] < count[r][t]) ++landed[r][t];
        settle();
      } else if (phase[s] >= count[r][s]) {        // the fill before has landed and been used up
        if (f[r].any(s) && f[r].latest(s) != ((count[r][s] - 1) & 1)) return printf("release parity\n"), 1;
        f[r].next(s);
        ++count[r][s];
        ++at[r];
      }
    }
    bool blocked[SLOTS] = {};
    for (int r = 0; r < 2; ++r)
      await_fills(f[r], SLOTS, [&](int s, uint32_t parity) { blocked[s] |= (uint32_t)(phase[s] & 1) == parity; });
    for (int r = 0; r < 2; ++r)
      for (int s = 0; s < SLOTS; ++s)
        if (landed[r][s] < count[r][s]) {
          ++outstanding;
          if (!blocked[s]) return printf("slot %d of CTA %d was not waited for\n", s, r), 1;
        }
    for (int s = 0; s < SLOTS; ++s)
      if (blocked[s] && phase[s] >= count[0][s] && phase[s] >= count[1][s]) return printf("a wait that nothing ends\n"), 1;
  }
  printf("ok %ld\n", outstanding);
  return outstanding < 100000;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a host C++ compiler")
def test_every_load_on_its_way_is_waited_for(tmp_path):
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-O1", "-I" + CSRC, "-o", str(exe), str(src)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.startswith("ok"), r.stdout
