// The cut of the paged attention's work where the lengths changed under a call, so that its
// blocks do not agree on the total: whatever lengths a block reads, and however often they
// change between its reads, the pieces that it counts are those of blocks of its launch.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "../../adaptq_amd/csrc/paged_split.hpp"

using namespace aq;

static void fail(const char *what) {
  std::fprintf(stderr, "%s\n", what);
  std::exit(1);
}

int main() {
  std::mt19937 g(5);
  long cut = 0, further = 0;
  for (int i = 0; i < 200000; ++i) {
    const int waves = 4, blocks = 1 + g() % 512, segs = 1 + g() % 8, n_seqs = 1 + g() % 5;
    const int least = 1 + g() % 16, unit = 16 << g() % 2;
    const auto length = [&]() { return (int)(g() >> (g() % 31)) & 0x7FFFFFFF; };
    const auto span = [&]() {
      return token_span(length(), g() % 2, g() % 3 ? 0 : g() % 4096, (int64_t)1 << (4 + g() % 28),
                        unit, least);
    };
    // what one block reads: a total, then the sequences before its start, then each one's length
    int64_t total = 0;
    for (int b = 0; b < n_seqs; ++b) total += (int64_t)span().units * segs;
    const int64_t share = share_of(total, blocks, waves);
    const int block = g() % blocks;
    const int64_t start = block * share;
    int64_t end = start + share;
    if (end > total) end = total;
    if (start >= end) continue;
    int64_t base = 0;
    int seq = 0;
    TokenSpan s = span();
    while (seq < n_seqs && base + (int64_t)s.units * segs <= start) {
      base += (int64_t)s.units * segs;
      s = span();
      ++seq;
    }
    if (seq == n_seqs) continue;  // the kernel returns
    Start st = start_at(start, base, s.units);
    int64_t at = start;
    while (at < end && seq < n_seqs) {
      if (st.seg < 0 || st.seg >= segs || st.u0 < 0 || st.u0 >= s.units) fail("start");
      const Piece p = piece_at(block, start, end, at, st.u0, s.units, s.short_, share, blocks);
      if (p.u1 <= st.u0 || p.u1 > s.units) fail("piece");
      if (!p.empty && !p.whole) {
        ++cut;
        if (p.first < 0 || p.first > block || p.pieces < 1 || p.first + p.pieces > blocks)
          fail("pieces of blocks that there are not");
        const Piece q = piece_at(block, start, end, at, st.u0, s.units, s.short_, share);
        if (q.first + q.pieces > blocks) ++further;
      }
      at += p.u1 - st.u0;
      st.u0 = 0;
      if (++st.seg == segs) {
        st.seg = 0;
        ++seq;
        s = span();
      }
    }
  }
  if (cut < 10000 || further < 1000) fail("too few");
  std::puts("ok");
}
