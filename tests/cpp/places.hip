// Whose place a tile's place is, on the CPU: the kernels' search, 64 requests to a round, over requests whose rows start
// anywhere: always a request there is, and the first one, in front of its tiles, for places before its own.
#include <cstdio>
#include <random>
#include <vector>

#include "paging.h"

using namespace efh;

static long place_of(int start, int r, int f, int d) { return static_cast<long>(start) * f / d + r; }

int main() {
  if (last_lane(0) != 0 || last_lane(1) != 0 || last_lane(3) != 1 || last_lane(~0ull) != 63) return std::printf("last_lane\n"), 1;
  std::mt19937 rng(5);
  long checked = 0, bad = 0;
  for (int round = 0; round < 300; ++round) {
    const int n = 1 + rng() % (round % 3 ? 70 : 5000), f = 1 + rng() % 8, d = round % 2 ? 128 : 32;
    std::vector<int> start(n + 1, static_cast<int>(rng() % 2 ? rng() % 2000 : 0));
    for (int r = 0; r < n; ++r) start[r + 1] = start[r] + (rng() % 3 ? rng() % 9 : rng() % 300);
    const long places = (static_cast<long>(start[n]) * f + d - 1) / d + n;
    for (int i = 0; i < 200; ++i, ++checked) {
      const long place = i < 8 ? i : static_cast<long>(rng() % places);
      int lo = 0, len = n, req = -1, first = 0;
      for (;;) {
        const int step = (len + 63) / 64;
        uint64_t below = 0;
        int starts[64];
        for (int lane = 0; lane < 64; ++lane) {
          starts[lane] = start[std::min(lo + lane * step, n)];
          if (lane * step < len && place_of(starts[lane], lo + lane * step, f, d) <= place) below |= 1ull << lane;
        }
        const int at = last_lane(below);
        if (step == 1) {
          req = lo + at;
          first = starts[at];
          break;
        }
        lo += at * step;
        len = std::min(step, len - at * step);
      }
      if (req < 0 || req >= n || first != start[req]) {
        ++bad;
        continue;
      }
      const long tile = place - place_of(first, req, f, d);
      const bool none = place < place_of(start[0], 0, f, d);
      if (none ? req != 0 || tile >= 0 : tile < 0 || (req + 1 < n && place >= place_of(start[req + 1], req + 1, f, d))) ++bad;
    }
  }
  std::printf("%ld checked, %ld wrong\n", checked, bad);
  return bad ? 1 : 0;
}
