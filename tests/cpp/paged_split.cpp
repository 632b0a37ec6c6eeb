// The cut of the paged attention's work, on the CPU: every unit of every segment is
// in exactly one piece, a cut segment's pieces are those its blocks count and use
// different slots, and token spans are what window, capacity and lengths leave.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "../../adaptq_amd/csrc/paged_split.hpp"

using namespace aq;

static void fail(const char *what) {
  std::fprintf(stderr, "%s\n", what);
  std::exit(1);
}

static void check_span(int length, int extra, int window, int64_t cap, int unit) {
  const TokenSpan s = token_span(length, extra, window, cap, unit, 1);
  const TokenSpan t = token_span(length, extra, window, cap, unit, 8);
  if (t.lo != s.lo || t.n != s.n || t.first_unit != s.first_unit ||
      t.units != (s.units < 8 ? 8 : s.units) || t.short_ != (s.units <= 8))
    fail("least");
  const int64_t held = length < 0 ? 0 : (int64_t)length + extra;
  int64_t n = held < cap ? held : cap;
  if (n > 0x7FFFFFE0) n = 0x7FFFFFE0;
  int64_t lo = window > 0 && held > window ? held - window : 0;
  if (lo > n) lo = n;
  if (s.n != n || s.lo != lo || s.units < 1) fail("span");
  if (lo < n) {
    if ((int64_t)s.first_unit * unit > lo) fail("span starts late");
    if ((int64_t)(s.first_unit + 1) * unit <= lo) fail("span starts early");
    if ((int64_t)(s.first_unit + s.units) * unit < n) fail("span ends early");
    if ((int64_t)(s.first_unit + s.units - 1) * unit >= n) fail("span ends late");
  }
}

static void check_cut(const std::vector<int> &units, int segs, int blocks, int waves, int short_units) {
  int64_t total = 0;
  std::vector<int64_t> base;
  for (int u : units) {
    base.push_back(total);
    total += (int64_t)u * segs;
  }
  const int64_t share = share_of(total, blocks, waves);
  if (share % waves || share * blocks < total) fail("share");
  std::map<std::pair<int, int>, std::vector<char>> seen;     // (sequence, segment) -> units
  std::map<std::pair<int, int>, int> pieces, expected;
  std::map<std::pair<int, int>, int64_t> firsts;
  std::set<std::pair<int64_t, int>> slots;
  std::set<int64_t> counters;
  for (int64_t b = 0; b < blocks; ++b) {
    const int64_t start = b * share, end = start + share < total ? start + share : total;
    if (start >= end) continue;
    int64_t at = start;
    size_t q = 0;
    while (q + 1 < base.size() && base[q + 1] <= at) ++q;
    Start s = start_at(at, base[q], units[q]);
    while (at < end) {
      if (s.seg < 0 || s.seg >= segs || s.u0 < 0 || s.u0 >= units[q]) fail("start");
      const bool small = units[q] <= short_units;
      const Piece p = piece_at((int)b, start, end, at, s.u0, units[q], small, share);
      if (p.u1 <= s.u0 || p.u1 > units[q]) fail("piece");
      if (p.empty != (small && s.u0 > 0)) fail("empty");
      if (small && !(p.whole && p.pieces == 1 && p.u1 == units[q])) fail("short");
      if (p.empty) {
        at += p.u1 - s.u0;
        s.u0 = 0;
        if (++s.seg == segs) {
          s.seg = 0;
          ++q;
        }
        continue;
      }
      const auto key = std::make_pair((int)q, s.seg);
      auto &v = seen[key];
      v.resize(units[q]);
      for (int u = s.u0; u < p.u1; ++u)
        if (v[u]++) fail("unit twice");
      if (p.whole != (p.pieces == 1)) fail("whole");
      if (!p.whole) {
        if (!slots.insert({b, p.slot}).second) fail("slot twice");
        ++pieces[key];
        expected[key] = p.pieces;
        if (pieces[key] == 1) {
          firsts[key] = p.first;
          if (p.first != b || p.slot != 1 || !counters.insert(b).second) fail("first");
        } else {
          if (firsts[key] != p.first || p.slot != 0) fail("later piece");
          if (b != p.first + pieces[key] - 1) fail("pieces are consecutive blocks");
        }
      }
      at += p.u1 - s.u0;
      s.u0 = 0;
      if (++s.seg == segs) {
        s.seg = 0;
        ++q;
      }
    }
  }
  for (size_t q = 0; q < units.size(); ++q)
    for (int s = 0; s < segs; ++s) {
      const auto key = std::make_pair((int)q, s);
      if ((int)seen[key].size() != units[q]) fail("segment missing");
      for (char c : seen[key])
        if (c != 1) fail("unit missing");
      if (pieces[key] != expected[key]) fail("piece count");
    }
}

static void check_large() {
  // beyond 32 bits of units: a block inside the last of many long segments
  const int units = (1 << 27) - 1, segs = 700, blocks = 512;
  const int64_t total = (int64_t)units * segs, share = share_of(total, blocks, 4);
  for (int64_t b : {0, 1, 255, 510, 511}) {
    const int64_t start = b * share, end = start + share < total ? start + share : total;
    const Start s = start_at(start, 0, units);
    if ((int64_t)s.seg * units + s.u0 != start || s.u0 >= units) fail("large start");
    const Piece p = piece_at((int)b, start, end, start, s.u0, units, false, share);
    const int64_t begin = (int64_t)s.seg * units;
    if (p.first != begin / share || p.first + p.pieces - 1 != (begin + units - 1) / share)
      fail("large piece");
  }
}

static void check_pages() {
  for (int blocks = 1; blocks <= 4096; ++blocks) {
    const PageOf p = page_of_blocks(16 * blocks);
    if (p.blocks != blocks) fail("page blocks");
    for (int64_t b : {0ll, 1ll, (1ll << 27) - 1, (1ll << 27) - 2, (1ll << 26) + 7})
      for (int64_t x : {b, b / blocks * blocks, b / blocks * blocks - 1, b / blocks * blocks + 1})
        if (x >= 0 && x < 1ll << 27 && page_column(p, (int)x) != x / blocks) fail("page column");
    for (int x = 0; x < 3 * blocks; ++x)
      if (page_column(p, x) != x / blocks) fail("page column");
  }
}

int main() {
  check_pages();
  check_large();
  const int edge[] = {-2147483647 - 1, -1, 0, 1, 15, 16, 17, 31, 32, 33, 1000, 2147483615, 2147483647};
  for (int n : edge)
    for (int extra : {0, 1})
      for (int window : {0, 1, 16, 31, 32, 33, 500, 2147483647})
        for (int64_t cap : {(int64_t)0, (int64_t)16, (int64_t)48, (int64_t)1008, (int64_t)1 << 40})
          for (int unit : {16, 32}) check_span(n, extra, window, cap, unit);
  std::mt19937 g(1);
  for (int i = 0; i < 3000; ++i) {
    std::vector<int> units(1 + g() % 20);
    const int top = 1 << (g() % 9);
    for (int &u : units) u = 1 + g() % top;
    check_cut(units, 1 + g() % 9, 1 + g() % 300, 1 << (g() % 4),
              g() % 3 ? 0 : g() % 40);
  }
  std::puts("ok");
}
