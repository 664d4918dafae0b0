// Runs the ring of csrc/bs_ring.cuh as a warp of the streaming kernels does, against a
// model of its barriers, for every number of units, every order in which copies land
// late, and every wait that may run out.  Prints "BAD 0" when no copy was asked for into
// a stage whose last one had not been waited for, every unit that was worked on had its
// own copy, and nothing was left in flight at the end.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "bs_ring.cuh"

struct Stage {
  int parity = 0;       // of the phase under way
  bool armed = false;   // a copy was asked for in it
  int unit = -1;        // which
  bool late = false;    // its first wait runs out
};

template <int S>
static long run(int units, unsigned late, long* worked) {
  Stage st[S];
  long bad = 0;
  bs::Ring<S> ring;
  int asked = 0;
  bool ran_out = false;
  bool more = units > 0;
  auto load = [&](int at) {
    if (!more) return;
    if (st[at].armed) ++bad;                 // the copy before is still under way
    st[at].armed = true, st[at].unit = asked, st[at].late = late >> asked & 1;
    if (++asked == units) more = false;
  };
  auto land = [&](int at) { st[at].armed = false, st[at].parity ^= 1; };
  for (int s = 0; s < S - 1; ++s) {
    ring.place(more);
    load(s);
  }
  for (int u = 0; u < units; ++u) {
    bool mine = false;
    more = ring.take([&](int s, int parity, bool again) {
      Stage& x = st[s];
      if (x.parity != parity) return true;   // that phase has ended
      if (!x.armed) {                        // nothing will ever end it: no wait, once one ran out
        bad += again || !ran_out;
        return false;
      }
      if (x.late && !again) return ran_out = true, false;
      if (!again) mine = x.unit == u;
      land(s);
      return true;
    }) && more;
    if (mine) ++*worked;
    load(ring.place(more));
    ring.next();
  }
  for (int s = 0; s < S; ++s) bad += st[s].armed;
  if (!late && *worked != units) ++bad;
  return bad;
}

template <int S>
static long all() {
  long bad = 0;
  for (int units = 0; units <= 12; ++units)
    for (unsigned late = 0; late < 1u << units; ++late) {
      long worked = 0;
      bad += run<S>(units, late, &worked);
    }
  return bad;
}

int main() {
  const long bad = all<2>() + all<3>() + all<4>();
  std::printf("BAD %ld\n", bad);
  return bad != 0;
}
