"""What a kernel waits for before it ends, after one of its waits has run out (csrc/waits.h, compiled here for the
CPU): every copy and chain of instructions that is under way, at the phase that its end completes."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "raven_b200", "csrc")

# The thread of a team that starts its copies and instructions, on barriers that count phases as the hardware's do: a
# wait for a parity is over when the phase in progress has the other one. `late`: the copy (of copies in order) or the
# chain that has not ended when the thread's first wait for it gives up; whatever is started behind it has not ended either.
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <vector>
#include "waits.h"
using namespace raven_score4;

struct Barrier { uint32_t completed = 0; bool over(uint32_t parity) const { return (completed & 1u) != parity; } };

int run(uint32_t depth, uint32_t blocks, uint32_t groups, int late_copy, int late_chain) {
  std::vector<Barrier> full(depth);
  Barrier done;
  Ring stages;
  Chain chain;
  std::vector<int> under_way(depth, 0);  // copies into a stage that have not ended
  int chains = 0, copies = 0, started = 0;
  bool ok = true, stuck = false;
  auto end_copy = [&](uint32_t s) { --under_way[s], ++full[s].completed; };
  auto copy_next = [&]() {
    if ((uint32_t)copies == blocks) return;
    if (copies++ == late_copy) stuck = true;
    const uint32_t s = stages.slot;
    ++under_way[s];
    if (under_way[s] > 1) { printf("a copy over another\n"); exit(1); }
    stages.begun(depth);
    if (!stuck) end_copy(s);
  };
  for (uint32_t i = 0; i < depth; ++i) copy_next();
  for (uint32_t b = 0; b < blocks; ++b) {
    if (ok && !full[stages.now].over(stages.parity())) ok = false;
    if (ok && under_way[stages.now]) { printf("a stage taken early\n"); exit(1); }
    if (ok) stages.taken(depth);
    for (uint32_t g = 0; g < groups; ++g) {
      if (ok) {
        if (g == 0) copy_next();
        if (started++ == late_chain) stuck = true;
        ++chains;
        if (!stuck) { --chains; ++done.completed; }
      }
      if (ok && !done.over(chain.phase)) ok = false;
      if (ok) chain.over();
    }
  }
  if ((late_copy >= 0 || late_chain >= 0) == ok) { printf("nothing ran out\n"); return 1; }
  // the end: what is late ends now, each only when it is waited for; a wait must not be over before
  int bad = 0;
  stages.rest(depth, [&](uint32_t s, uint32_t parity) {
    if (under_way[s] && full[s].over(parity)) bad = 1;
    if (under_way[s]) end_copy(s);
    if (!full[s].over(parity)) bad = 2;
  });
  chain.rest([&](uint32_t parity) {
    if (!chains) return;  // runs out
    if (done.over(parity)) bad = 3;
    while (chains) --chains, ++done.completed;
    if (!done.over(parity)) bad = 4;
  });
  for (uint32_t s = 0; s < depth; ++s)
    if (under_way[s]) bad = 5;
  if (chains) bad = 6;
  if (bad) printf("depth %u blocks %u groups %u copy %d chain %d: %d\n", depth, blocks, groups, late_copy, late_chain, bad);
  return bad;
}

int main() {
  int bad = 0;
  for (uint32_t depth = 2; depth <= 4; ++depth)
    for (uint32_t blocks = 1; blocks <= 11; ++blocks)
      for (uint32_t groups = 1; groups <= 4; ++groups) {
        bad |= run(depth, blocks, groups, -1, -1);
        for (uint32_t k = 0; k < blocks; ++k) bad |= run(depth, blocks, groups, (int)k, -1);
        for (uint32_t k = 0; k < blocks * groups; ++k) bad |= run(depth, blocks, groups, -1, (int)k);
      }
  puts(bad ? "bad" : "good");
  return bad != 0;
}
"""


def test_what_is_under_way_is_waited_for(tmp_path):
    gxx = shutil.which("g++")
    if not gxx:
        pytest.skip("no g++")
    src, exe = tmp_path / "waits.cpp", tmp_path / "waits"
    src.write_text(PROGRAM)
    subprocess.run([gxx, "-std=c++17", "-Wall", "-Werror", "-I", CSRC, "-o", str(exe), str(src)], check=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True)
    assert res.returncode == 0, res.stdout[:2000]


def test_the_wide_kernel_keeps_its_waits_so():
    """The kernel's own source: phases are kept by the two structures alone, and an end after a wait that ran out asks them."""
    with open(os.path.join(CSRC, "score4_wide.cuh")) as f:
        text = f.read()
    for line in ("if (ok) chain.over();", "stages.taken(p.depth);", "stages.rest(p.depth,", "chain.rest("):
        assert text.count(line) == 1, line
    assert "phase ^=" not in text and "phases ^=" not in text
