// The tokens that a query sees (seen_span of paged_split.hpp) against the rule itself, token by
// token: visited by exactly one unit of the launch if it is seen, and no unit twice.
#include <cstdio>
#include <cstdlib>
#include <algorithm>
#include <random>
#include <vector>

#include "../../adaptq_amd/csrc/paged_split.hpp"

int main() {
  std::mt19937 rng(1);
  const auto below = [&](int n) { return (int)(rng() % n); };
  long cases = 0;
  for (int round = 0; round < 400000; ++round) {
    const int unit = below(2) ? 32 : 16, least = below(3) ? 1 : 16;
    const int cap = 16 * below(30), extra = below(2);
    const int most = below(2) ? 40 : 600;
    const int length = below(most) - 3;
    const int window = below(3) ? 1 + below(most) : 0;
    const int first = below(3) ? below(most) - 5 : 0, prefix = below(3) ? below(most) - 5 : 0;
    const aq::SeenSpan s = aq::seen_span(length, extra, window, cap, unit, least, first, prefix);
    const int held = length < 0 ? 0 : length + extra, n = held < cap ? held : cap;
    std::vector<int> visits(n + 64, 0);
    if (s.n != n || s.units < 1 || (s.short_ && s.units != least)) return std::printf("n\n"), 1;
    // as the kernel goes over a segment whole: units from first_unit on, none behind units_end
    const int end = std::min(s.first_unit + s.units, (n + unit - 1) / unit - s.gap);
    for (int u = s.first_unit; u < end; ++u) {
      const int t0 = aq::real_unit(s, u) * unit;
      if (t0 < 0 || t0 >= n) return std::printf("unit behind the tokens\n"), 1;
      for (int t = t0; t < t0 + unit; ++t) ++visits[t];
    }
    for (int t = 0; t < n; ++t) {
      const int p = held - 1;
      const bool seen = t >= first && (t < prefix || (window == 0 || t > p - window));
      const bool is = t >= s.lo && t < s.n && (t < s.hole0 || t >= s.hole1);
      if (is != seen || (seen && visits[t] != 1) || visits[t] > 1) {
        std::printf("length %d extra %d cap %d window %d first %d prefix %d unit %d: token %d is "
                    "seen %d, should be %d, visited %d times\n",
                    length, extra, cap, window, first, prefix, unit, t, is, seen, visits[t]);
        return 1;
      }
      ++cases;
    }
    // without the new arguments it is the span that the unmasked kernel has
    const aq::TokenSpan a = aq::token_span(length, extra, window, cap, unit, least);
    const aq::SeenSpan b = aq::seen_span(length, extra, window, cap, unit, least, 0, 0);
    if (a.n != b.n || (n > 0 && a.lo < n && (a.lo != b.lo || a.first_unit != b.first_unit ||
                                            a.units != b.units || a.short_ != b.short_)))
      return std::printf("not the unmasked span\n"), 1;
  }
  std::printf("ok %ld\n", cases);
  return 0;
}
