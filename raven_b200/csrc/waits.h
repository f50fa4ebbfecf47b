// Which phase of which barrier a thread waits for that keeps copies and instructions
// under way. A phase counts as over only when a wait for it has ended well: after one
// that ran out, `rest` names what the thread has to wait for before its shared memory is
// given up. No CUDA in here: tests compile it.
#pragma once

#include <cstdint>

#ifdef __CUDACC__
#define RAVEN_BOTH __host__ __device__
#else
#define RAVEN_BOTH
#endif

namespace raven_score4 {

// A ring of stages, each with a barrier, copied into and taken in turn.
struct Ring {
  uint32_t now = 0, slot = 0;  // the stage that is taken next, that is copied into next
  uint32_t phases = 0;         // parity of each stage's phase that is not over
  uint32_t pending = 0;        // stages with a copy under way

  RAVEN_BOTH static uint32_t next(uint32_t stage, uint32_t depth) { return stage + 1 == depth ? 0 : stage + 1; }
  RAVEN_BOTH uint32_t parity() const { return phases >> now & 1u; }
  RAVEN_BOTH void begun(uint32_t depth) {  // a copy into stage `slot`
    pending |= 1u << slot;
    slot = next(slot, depth);
  }
  RAVEN_BOTH void taken(uint32_t depth) {  // the wait for stage `now` has ended well
    phases ^= 1u << now;
    pending &= ~(1u << now);
    now = next(now, depth);
  }
  template <typename F>
  RAVEN_BOTH void rest(uint32_t depth, F&& wait) const {  // wait(stage, parity)
    for (uint32_t i = 0; i < depth; ++i)
      if (pending >> i & 1u) wait(i, phases >> i & 1u);
  }
};

// Chains of instructions, one at a time, that arrive at one barrier. Whether one is under way takes a register more,
// which kernels of 96 columns do not have (88 bytes spilled, 96 x 250007 x 128 38 -> 43 us): after a wait that ran out
// the phase in progress is waited for in any case, for as long as a wait may take where there is none.
struct Chain {
  uint32_t phase = 0;

  RAVEN_BOTH void over() { phase ^= 1u; }  // the wait for it has ended well
  template <typename F>
  RAVEN_BOTH void rest(F&& wait) const {  // wait(parity)
    wait(phase);
  }
};

}  // namespace raven_score4
