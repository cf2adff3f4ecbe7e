// The drain of the linear layer's copies (prime-tts_b200/csrc/drain.h) against a model of the ring: for every
// number of stages and every pair of points at which the producers can stop, each copy that was issued
// has landed when the drain is through, and no wait is passed by an older phase of the same parity.
#include <cstdio>
#include <vector>

#include "drain.h"

struct Barrier {       // two arrivals to a phase, and the bytes of both halves
  int phase = 0, arrived = 0, flying = 0;
  void settle() {
    if (arrived == 2 && flying == 0) ++phase, arrived = 0;
  }
};

int main() {
  long bad = 0, runs = 0;
  for (int stages = 2; stages <= 10; ++stages)
    for (int used = 0; used <= 3 * stages; ++used)         // fills that the consumer has used
      for (int a = used; a <= used + stages; ++a)           // a producer is at most `stages` ahead of it
        for (int b = used; b <= used + stages; ++b) {
          ++runs;
          std::vector<Barrier> bar(stages);
          const int most = a > b ? a : b;
          for (int i = 0; i < most; ++i) {
            Barrier &x = bar[i % stages];
            x.arrived = (i < a) + (i < b);
            x.flying = i < used ? 0 : x.arrived;            // (used: both halves landed)
            x.settle();
          }
          const ptb::Drain d = ptb::drain_of(a, b, stages);
          for (int i = d.begin; i < d.end; ++i) {
            Barrier &x = bar[i % stages];
            if (i >= d.matched) ++x.arrived;
            x.settle();
            // a wait for parity p passes when the current phase's parity differs from p
            const bool passes_early = (x.phase & 1) != static_cast<int>(ptb::fill_parity(i, stages));
            if (passes_early && x.flying > 0) ++bad;
            x.flying = 0;                                   // ... else it waits until they land
            x.settle();
            if ((x.phase & 1) == static_cast<int>(ptb::fill_parity(i, stages))) ++bad;   // it would wait for good
          }
          for (const Barrier &x : bar) bad += x.flying > 0;
        }
  std::printf("%ld %ld\n", runs, bad);
  return 0;
}
