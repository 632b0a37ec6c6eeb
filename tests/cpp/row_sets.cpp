// Overlap of strided rows against the bytes themselves, on small sets: what is called
// apart shares no byte, and the layouts that calls use are recognised.
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>

#include "../../adaptq_amd/csrc/row_sets.hpp"

using namespace aq;

static void fail(const char *what) {
  std::fprintf(stderr, "%s\n", what);
  std::exit(1);
}

struct Set {
  size_t at;
  int n[3];
  size_t nb[3];
};

// Its bytes; *twice: whether two rows share one.
static std::set<size_t> bytes(const Set &s, size_t row, int dims, bool *twice) {
  std::set<size_t> b;
  *twice = false;
  for (int i = 0; i < s.n[0]; ++i)
    for (int j = 0; j < s.n[1]; ++j)
      for (int k = 0; k < (dims > 2 ? s.n[2] : 1); ++k)
        for (size_t x = 0; x < row; ++x)
          if (!b.insert(s.at + i * s.nb[0] + j * s.nb[1] + (dims > 2 ? k * s.nb[2] : 0) + x).second)
            *twice = true;
  return b;
}

int main() {
  std::mt19937 g(3);
  int apart = 0, rows_ok = 0;
  for (int i = 0; i < 200000; ++i) {
    const int dims = 2 + g() % 2;
    const size_t row = 1 + g() % 4;
    Set s[2];
    for (Set &x : s) {
      x.at = 1000 + g() % 60;
      for (int d = 0; d < 3; ++d) {
        x.n[d] = 1 + g() % 3;
        x.nb[d] = g() % 24;
      }
    }
    if (g() % 2)  // columns of one tensor
      for (int d = 1; d < 3; ++d) {
        s[1].n[d] = s[0].n[d];
        s[1].nb[d] = s[0].nb[d];
      }
    bool twice[2];
    const std::set<size_t> a = bytes(s[0], row, dims, &twice[0]), b = bytes(s[1], row, dims, &twice[1]);
    const void *p = reinterpret_cast<const void *>(s[0].at), *q = reinterpret_cast<const void *>(s[1].at);
    const Span sp = span_of(p, row, s[0].n, s[0].nb, dims);
    if (sp.lo != *a.begin() || sp.hi != *a.rbegin() + 1) fail("span");
    for (int k = 0; k < 2; ++k)
      if (rows_apart(row, s[k].n, s[k].nb, dims)) {
        ++rows_ok;
        if (twice[k]) fail("rows called apart share a byte");
      }
    if (sets_apart(p, row, s[0].n, s[0].nb, q, s[1].n, s[1].nb, dims)) {
      ++apart;
      for (size_t x : a)
        if (b.count(x)) fail("sets called apart share a byte");
    }
  }
  if (apart < 1000 || rows_ok < 1000) fail("too few");
  // queries, keys and values side by side in one tensor of 7 heads of 8 bytes: all apart
  const int nq[3] = {4, 5, 2}, nk[3] = {2, 5, 2};
  const size_t nb[3] = {8, 56, 280};
  const char *t = reinterpret_cast<const char *>(4096);
  if (!sets_apart(t, 8, nq, nb, t + 32, nk, nb, 3) || !sets_apart(t + 32, 8, nk, nb, t, nq, nb, 3))
    fail("columns of one tensor");
  if (sets_apart(t, 8, nq, nb, t + 24, nk, nb, 3)) fail("columns that overlap");
  // contiguous, heads first, and one row for all
  const size_t heads_first[3] = {40, 8, 160}, none[3] = {0, 0, 0};
  if (!rows_apart(8, nq, nb, 3) || !rows_apart(8, nq, heads_first, 3) || rows_apart(8, nq, none, 3))
    fail("layouts");
  std::puts("ok");
}
