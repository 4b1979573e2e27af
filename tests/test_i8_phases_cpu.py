"""The phases that the pair kernel's leader waits for before it leaves (csrc/i8/i8_phases.h).

A CTA must not exit while an arrival from its peer is on its way to a barrier in its
shared memory. The header the kernel takes its parities from is compiled here
against a model of an mbarrier: for every number of tiles, the last waits hold until
the very last arrival has landed, and then return."""
import os
import re
import subprocess

from conftest import ROOT

HARNESS = r"""
#include <cstdio>
#include <cstdlib>

#include "i8_phases.h"

using namespace aegis::i8;

struct Barrier {  // an mbarrier's phase and the arrivals it still expects
  int count, left;
  long phase = 0;
  explicit Barrier(int n) : count(n), left(n) {}
  void arrive() {
    if (--left == 0) {
      left = count;
      ++phase;
    }
  }
  bool done(uint32_t parity) const { return uint32_t(phase & 1) != parity; }
};
#define CHECK(x) \
  do { \
    if (!(x)) { std::printf("line %d, n %d: %s\n", __LINE__, n, #x); std::exit(1); } \
  } while (0)

int main() {
  // Accumulators: n tiles; 16 epilogue warps read each. `late` arrivals of the last tiles come after the MMA lane's loop.
  for (int n = 1; n <= 40; ++n)
    for (int late = 1; late <= 32 && late <= 16 * n; ++late) {
      Barrier full[2] = {Barrier(1), Barrier(1)}, empty[2] = {Barrier(16), Barrier(16)};
      AccumulatorTurn mma, epi;
      int read_tiles = 0, read_warps = 0;
      auto land = [&] {
        if (read_warps == 0) CHECK(full[epi.acc].done(epi.full()));
        empty[epi.acc].arrive();
        if (++read_warps == 16) {
          read_warps = 0;
          ++read_tiles;
          epi.next();
        }
      };
      for (int i = 0; i < n; ++i) {
        // The lane waits for the accumulator: arrivals land until it is free.
        while (!empty[mma.acc].done(mma.read(mma.acc))) land();
        full[mma.acc].arrive();
        mma.next();
      }
      const int all = 16 * n;
      while (read_tiles * 16 + read_warps < all - late) land();
      for (; read_tiles * 16 + read_warps < all;) {
        CHECK(!(empty[0].done(mma.read(0)) && empty[1].done(mma.read(1))));  // the leader may not leave yet
        land();
      }
      CHECK(empty[0].done(mma.read(0)) && empty[1].done(mma.read(1)));
    }
  // Slots: n published, each given back by every one of 18 readers; the owner runs at most `depth` ahead.
  const int depth = 4, readers = 18;
  for (int n = 1; n <= 40; ++n)
    for (int late = 1; late <= depth * readers && late <= n * readers; ++late) {
      Barrier empty[depth] = {Barrier(readers), Barrier(readers), Barrier(readers), Barrier(readers)};
      int landed = 0;
      auto land = [&] { empty[landed++ / readers % depth].arrive(); };
      for (int seq = 0; seq < n; ++seq)
        while (!empty[seq % depth].done((uint32_t(seq / depth) & 1u) ^ 1u)) land();
      auto over = [&] {
        bool all = true;
        for (int i = 0; i < depth; ++i) all = all && empty[i].done(slot_read(n, i, depth));
        return all;
      };
      while (landed < n * readers - late) land();
      while (landed < n * readers) {
        CHECK(!over());
        land();
      }
      CHECK(over());
    }
  std::puts("ok");
}
"""


def test_last_waits_hold_until_every_arrival_has_landed(tmp_path):
    src, exe = tmp_path / "t.cpp", tmp_path / "t"
    src.write_text(HARNESS)
    subprocess.run(["g++", "-std=c++20", "-Wall", "-Wextra", "-Werror", "-I" + os.path.join(ROOT, "aegis-core_b200", "csrc", "i8"),
                    str(src), "-o", str(exe)], check=True)
    assert subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout == "ok\n"


def test_the_pair_kernel_waits_before_it_leaves():
    """Its remote arrivals are a slot's and an accumulator's: the leader waits for both before the cluster's last barrier."""
    text = open(os.path.join(ROOT, "aegis-core_b200", "csrc", "i8", "i8_pair.cuh")).read()
    kernel = text[text.index("i8_pair_kernel("):]
    last = kernel.index("cluster_step()")
    for wait in (r"mbar_wait_teardown\(sched\.empty_bar\(i\), slot_read\(owner\.seq, i, umma::kSchedDepth\)",
                 r"mbar_wait_teardown\(tempty_bar\(acc\), turn\.read\(acc\)"):
        assert len(re.findall(wait, kernel[:last])) == 1
    assert kernel.rindex("ptx::cluster_sync()") < last and "if (*abort_flag) ptx::cluster_sync();" in kernel
