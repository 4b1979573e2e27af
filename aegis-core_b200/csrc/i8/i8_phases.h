#pragma once
// Which phase of an mbarrier a wait names, for the two rings whose barriers in the
// leader of a CTA pair its peer arrives on: the TMEM accumulators and the schedule's
// slots. Plain arithmetic, for the host too.
//
// A barrier's phases count from 0; a wait with parity p returns once the phase in
// progress has a parity other than p. The n-th use (from 0) of a ring's place
// waits for the place to be free with parity (n & 1) ^ 1: at once for the first
// use, then for the phase that the readers of use n - 1 complete. The same wait
// after the last use returns when those readers' arrivals have landed, remote ones
// too: that is how the leader knows that nothing is on its way to its barriers.
#include <cstdint>

#ifdef __CUDACC__
#define AEGIS_I8_HD __host__ __device__ __forceinline__
#else
#define AEGIS_I8_HD inline
#endif

namespace aegis::i8 {

// Two accumulators in turn.
struct AccumulatorTurn {
  int acc = 0;         // the next one to use
  uint32_t phase = 0;  // the parity of its uses so far

  AEGIS_I8_HD void next() {
    acc ^= 1;
    if (acc == 0) phase ^= 1u;
  }
  // Parity that waits for the present use to be full.
  AEGIS_I8_HD uint32_t full() const { return phase; }
  // Parity that waits until every use of accumulator `a` so far has been read.
  AEGIS_I8_HD uint32_t read(int a) const { return a < acc ? phase : phase ^ 1u; }
};

// Parity that waits until slot i of a ring of `depth`, of which `seq` uses have been
// made in turn, has been read every time.
AEGIS_I8_HD uint32_t slot_read(int seq, int i, int depth) {
  const int next = seq + ((i - seq) % depth + depth) % depth;  // the next use of slot i
  return (uint32_t(next / depth) & 1u) ^ 1u;
}

}  // namespace aegis::i8
