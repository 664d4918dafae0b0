// The order of waits and copies in a warp's ring of S stages, one copy and one
// mbarrier phase to a use of a stage: S - 1 copies are asked for ahead, then one for
// each unit that has been waited for.  Plain arithmetic, on the host too.
#pragma once

#ifdef __CUDACC__
#define BS_HD __host__ __device__ __forceinline__
#else
#define BS_HD inline
#endif

namespace bs {

template <int S>
struct Ring {
  int stage = 0, phase = 0;  // of the next unit
  int flying = S - 1;        // copies asked for and not waited for, when the next unit is

  // Waits for the next unit's copy.  When the wait runs out, those in flight are waited
  // for once more, each with its own limit, so that none lands after its memory has gone
  // to another use; the caller asks for no more then.  wait(stage, parity, again) says
  // whether the phase has ended, at once where another wait ran out before.
  template <class Wait>
  BS_HD bool take(Wait&& wait) {
    if (wait(stage, phase, false)) return true;
    for (int j = 0; j < flying; ++j) wait((stage + j) % S, phase ^ (stage + j >= S), true);
    flying = 0;
    return false;
  }
  // Where the next copy goes, with `on`; without, there is one less in flight.
  BS_HD int place(bool on) {
    if (!on) --flying;
    return (stage + S - 1) % S;
  }
  BS_HD void next() {
    if (++stage == S) stage = 0, phase ^= 1;
  }
};

}  // namespace bs
