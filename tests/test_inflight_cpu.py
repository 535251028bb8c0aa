"""CPU: the bookkeeping by which a warp knows the copies that it has to wait for before its block leaves
(csrc/sage_inflight.cuh), run on the host against a model of the chunk kernel's ring: slots, barriers with phases, copies
that land late, a producer that gives up anywhere."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tribench_b200", "csrc")

MODEL = r"""
#include "sage_inflight.cuh"
#include <cstdio>
#include <cstdlib>
#include <vector>

struct Barrier { int done = 0; bool passes(unsigned parity) const { return (unsigned)(done & 1) != parity; } };  // phases completed
struct Copy { Barrier* bar; bool landed = false; };

static unsigned long long state;
static unsigned rnd(unsigned n) { state = state * 6364136223846793005ull + 1442695040888963407ull; return (unsigned)(state >> 33) % n; }

int main(int argc, char** argv) {
  long unlanded = 0, waits = 0;
  for (int run = 0; run < 20000; ++run) {
    state = 977 * run + 1;
    const int NS = rnd(2) ? 2 : 4, tiles = 1 + rnd(12), stop = rnd(2 * tiles + 1);  // operands issued before giving up
    const bool always_raw = rnd(3) == 0;                                             // an INT8 cache
    std::vector<Barrier> kfull(NS), vfull(NS), vraw(NS);
    std::vector<Copy> k(tiles), v(tiles);
    std::vector<bool> raw(tiles), used(tiles, false);
    sage::ValueCopies values;
    int issued = 0, tiles_k = 0, tiles_v = 0;
    auto land = [](Copy& x) { if (x.bar && !x.landed) { x.landed = true; ++x.bar->done; } };
    auto consume = [&](int j) {  // a tile is used once both operands are there; a raw V is finished first
      land(k[j]); land(v[j]);
      if (raw[j]) ++vfull[j % NS].done;
      used[j] = true;
    };
    for (int it = 0; it < tiles && issued < stop; ++it) {
      const int s = it % NS;
      raw[it] = always_raw || rnd(2);
      if (it >= NS && !used[it - NS]) consume(it - NS);  // the slot's wait
      k[it].bar = &kfull[s];
      tiles_k = it + 1;
      ++issued;
      if (rnd(2)) land(k[it]);
      if (issued >= stop) break;
      v[it].bar = raw[it] ? &vraw[s] : &vfull[s];
      tiles_v = it + 1;
      if (!always_raw) values.note(s, it / NS, raw[it]);
      ++issued;
      if (rnd(2)) land(v[it]);
      // consumers may be ahead of the slot's reuse
      for (int j = it > NS ? it - NS : 0; j <= it; ++j)
        if (!used[j] && (j == 0 || used[j - 1]) && rnd(3) == 0) consume(j);
    }
    // gave up (or finished) here: every copy that has not landed must be waited for
    struct Wait { Barrier* bar; unsigned parity; };
    const sage::CopyLedger ck = sage::ring_copies(tiles_k, NS), cv = always_raw ? sage::ring_copies(tiles_v, NS) : values.raw;
    std::vector<Wait> w;
    for (int s = 0; s < NS; ++s) {
      if (ck.pending(s)) w.push_back({&kfull[s], ck.phase(s)});
      if (values.full.pending(s)) w.push_back({&vfull[s], values.full.phase(s)});
      if (cv.pending(s)) w.push_back({&vraw[s], cv.phase(s)});
    }
    for (auto* ops : {&k, &v})
      for (Copy& x : *ops)
        if (x.bar && !x.landed) {
          ++unlanded;
          bool waited = false;
          for (Wait& y : w) waited |= y.bar == x.bar && !y.bar->passes(y.parity);
          if (!waited) { std::printf("run %d: a copy in flight that no wait covers\n", run); return 1; }
        }
    for (auto* ops : {&k, &v})
      for (Copy& x : *ops) land(x);
    for (Wait& y : w) {  // and no wait is for a phase that never comes
      ++waits;
      if (!y.bar->passes(y.parity)) { std::printf("run %d: a wait that does not end\n", run); return 1; }
    }
  }
  std::printf("%ld copies in flight, %ld waits\n", unlanded, waits);
  return unlanded > 1000 ? 0 : 2;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_copy_in_flight_is_waited_for(tmp_path):
    src, exe = tmp_path / "model.cpp", tmp_path / "model"
    src.write_text(MODEL)
    subprocess.run(["g++", "-std=c++17", "-O1", "-x", "c++", "-I", CSRC, str(src), "-o", str(exe)], check=True)
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout
