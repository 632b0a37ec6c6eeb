// The passes of a prompt's tile (passes_of of paged_split.hpp) against the runs themselves in 64
// bits: every unit with a token of a run exactly once, in order, and no other between; the tests of a
// unit against a run; all of it up to the last token that a sequence may hold.
#include <algorithm>
#include <cstdint>
#include <cstdio>
#include <random>
#include <vector>

#include "../../adaptq_amd/csrc/paged_split.hpp"

int main() {
  std::mt19937 rng(1);
  const auto below = [&](int n) { return (int)(rng() % n); };
  long cases = 0;
  for (int round = 0; round < 300000; ++round) {
    const int keys = below(2) ? 64 : 32;
    const int top = below(2) ? aq::kMaxTokens : 1 + below(2000);
    // a run near the end of the tokens, and one before it, maybe empty, maybe over it
    const int e = top - below(std::min(top, 150) + 1), w = e - below(std::min(e, 300) + 1);
    const int lo = below(4) ? below(std::min(w, 200) + 1) : std::max(0, w - below(200));
    const int pe = below(3) ? (int)std::min((int64_t)top, (int64_t)lo + below(300)) : lo;
    const aq::Passes p = aq::passes_of(lo, pe, w, e, keys);
    std::vector<int64_t> want;
    const auto run = [&](int64_t a, int64_t b) {
      for (int64_t u = a / keys; a < b && u * keys < b; ++u) want.push_back(u);
    };
    run(lo, pe);
    run(w, e);
    std::sort(want.begin(), want.end());
    want.erase(std::unique(want.begin(), want.end()), want.end());
    std::vector<int64_t> got;
    for (int i = 0; i < p.count; ++i) got.push_back(aq::unit_of(p, i));
    if (got != want) {
      std::printf("[%d, %d) [%d, %d) keys %d: %zu units for %zu\n", lo, pe, w, e, keys, got.size(),
                  want.size());
      return 1;
    }
    for (const int64_t u : got) {
      if (u * keys >= top) return std::printf("a unit behind the tokens\n"), 1;
      const int t0 = (int)u * keys;
      const int64_t end = u * keys + keys;
      for (const auto &r : {std::pair<int, int>{lo, pe}, {w, e}, {0, top}, {0x7FFFFFFF, 0},
                            {0, 0x7FFFFFFF}}) {
        const auto [a, b] = r;
        const bool meets = t0 < b && end > a;
        if (aq::unit_within(t0, keys, a, b) != (t0 >= a && end <= b) ||
            aq::unit_meets(t0, keys, a, b) != meets)
          return std::printf("unit %d of %d against [%d, %d)\n", t0, keys, a, b), 1;
      }
      if (aq::unit_end(t0, keys, top) != std::min(end, (int64_t)top))
        return std::printf("the end of unit %d\n", t0), 1;
      ++cases;
    }
  }
  std::printf("ok %ld\n", cases);
  return 0;
}
