// The consuming side of a ring of S stages that a warp fills and empties in
// order: which stage comes next, and what is still in flight after a wait that
// ran out.  Plain C++, so that a test can compile it by itself.
#pragma once

#include <stdint.h>

#include "host_device.cuh"

namespace b2k {

struct RingUse {
  uint32_t used = 0, phase = 0;  // fills taken; phase of the next one's barrier
  int stage = 0;                 // the next one's
  bool dead = false;             // a wait ran out

  B2K_HOST_DEVICE void step(int S) {
    ++used;
    if (++stage == S) {
      stage = 0;
      phase ^= 1;
    }
  }
  // The stage of the next fill, once wait(stage, phase) has it; -1 from the
  // first wait that runs out on, whose fill stays among those not taken.
  template <typename Wait> B2K_HOST_DEVICE int take(int S, Wait wait) {
    if (dead || !wait(stage, phase)) {
      dead = true;
      return -1;
    }
    const int s = stage;
    step(S);
    return s;
  }
  // Waits (each wait bounded) for every fill that was issued and not taken.
  template <typename Wait> B2K_HOST_DEVICE void drain(uint32_t issued, int S, Wait wait) {
    for (; used != issued; step(S)) wait(stage, phase);
  }
};

}  // namespace b2k
