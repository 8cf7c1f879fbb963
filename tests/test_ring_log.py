"""The log of copies in flight (csrc/ring.cuh), compiled for the host and driven like the paged decode's
producer: lanes issue side by side, consumers release slots in any order, and somewhere a wait gives
up.  Whatever happened before, the waits that the log asks for must cover every copy still in
flight, and each must be one that the slot's barrier ends."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "butterfly_b200", "csrc")

_PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <random>
#include "ring.cuh"

struct Bar {                 // a barrier whose phases end when the copy of that phase has landed
  int issued = 0, landed = 0;
  bool done(unsigned parity) const { return (landed & 1) != (int)parity; }  // the phase of that parity is over
};

template <int WARPS, int SLOTS>
long run(std::mt19937& g, bool give_up) {
  using R = bna::Ring<WARPS, SLOTS>;
  const int kLanes = 8;
  Bar full[SLOTS];
  int consumed[SLOTS] = {}, log[SLOTS] = {}, used[WARPS] = {};
  auto coin = [&](int n) { return (int)(g() % n); };
  bool ok = true;
  const int fail_at = give_up ? coin(120) : 1 << 30;
  int granules = 0;
  for (int seg = 0; seg < 1 + coin(6) && ok; ++seg) {
    const int n = 1 + coin(70);
    for (int w = 0; w < n && ok; w += kLanes) {
      const int lanes = n - w < kLanes ? n - w : kLanes;
      bool all = true;
      for (int l = 0; l < lanes; ++l, ++granules) {
        const int warp = (w + l) % WARPS, use = used[warp] + (w + l) / WARPS, s = R::slot(use, warp);
        // this lane's wait for a free slot: runs out at random once the trouble has begun
        if (granules >= fail_at && coin(2)) { all = false; continue; }
        while (consumed[s] < full[s].issued) {  // the copy before lands, and is consumed
          if (full[s].landed < full[s].issued) ++full[s].landed;
          ++consumed[s];
        }
        if ((int)R::parity(use) != (full[s].issued & 1)) return -1;  // the phase this use stands for
        R::log(log, use, warp);
        ++full[s].issued;
        if (coin(3) == 0) ++full[s].landed;  // (some land at once)
      }
      ok = all;
    }
    if (!ok) break;
    for (int c = 0; c < WARPS; ++c) used[c] += (n - c + WARPS - 1) / WARPS;
  }
  // the drain: a wait ends once the slot's copies have landed; anything left in flight is a fault
  long faults = 0;
  for (int lane = 0; lane < 32; ++lane)
    R::settle(log, lane, 32, [&](int s, unsigned parity) {
      full[s].landed = full[s].issued;         // time passes
      if (!full[s].done(parity)) ++faults;     // a wait that never ends
    });
  for (int s = 0; s < SLOTS; ++s) faults += full[s].landed != full[s].issued;
  return faults;
}

int main() {
  std::mt19937 g(7);
  long faults = 0;
  for (int i = 0; i < 20000; ++i) {
    for (long f : {run<8, 16>(g, i & 1), run<4, 16>(g, i & 1), run<4, 8>(g, i & 1)}) {
      if (f < 0) { std::puts("parity"); return 2; }
      faults += f;
    }
  }
  std::printf("%ld\n", faults);
  return faults != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="no host compiler")
def test_every_copy_in_flight_is_waited_for(tmp_path):
    src, exe = tmp_path / "ring.cpp", tmp_path / "ring"
    src.write_text(_PROGRAM)
    subprocess.run(["g++", "-O1", "-std=c++17", f"-I{CSRC}", str(src), "-o", str(exe)], check=True, capture_output=True, timeout=300)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout
