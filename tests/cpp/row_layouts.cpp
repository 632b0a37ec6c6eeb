// Sets of rows that are parts of one tensor, its axes in any order: they are called apart
// exactly where they share no byte, however their rows alternate.
#include <algorithm>
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
};

static std::set<size_t> bytes(const Set &s, const size_t *nb, size_t row, int dims) {
  std::set<size_t> b;
  for (int i = 0; i < s.n[0]; ++i)
    for (int j = 0; j < s.n[1]; ++j)
      for (int k = 0; k < (dims > 2 ? s.n[2] : 1); ++k)
        for (size_t x = 0; x < row; ++x)
          b.insert(s.at + i * nb[0] + j * nb[1] + (dims > 2 ? k * nb[2] : 0) + x);
  return b;
}

int main() {
  std::mt19937 g(7);
  int apart = 0, inside = 0, shared = 0;
  for (int i = 0; i < 60000; ++i) {
    // a dense tensor of heads, tokens, batches and parts (queries, keys, values), any order
    const size_t row = 1 + g() % 4;
    const int dims = 2 + g() % 2;
    int size[4], order[4] = {0, 1, 2, 3};
    for (int d = 0; d < 4; ++d) size[d] = 1 + g() % 4;
    if (dims == 2) size[2] = 1;
    std::shuffle(order, order + 4, g);
    size_t stride[4], whole = row + g() % 3;
    for (int d : order) {
      stride[d] = whole;
      whole *= size[d];
      whole += g() % 2 ? 0 : g() % 5;
    }
    // two parts of it: ranges of heads, tokens and batches, every one or every other
    int step[3];
    size_t nb[3];
    for (int d = 0; d < 3; ++d) {
      step[d] = 1 + g() % 2;
      nb[d] = stride[d] * step[d];
    }
    Set s[2];
    for (Set &x : s) {
      x.at = 1000 + stride[3] * (g() % size[3]);
      for (int d = 0; d < 3; ++d) {
        const int first = g() % size[d];
        x.n[d] = 1 + g() % ((size[d] - 1 - first) / step[d] + 1);
        x.at += first * stride[d];
      }
    }
    const std::set<size_t> a = bytes(s[0], nb, row, dims), b = bytes(s[1], nb, row, dims);
    bool disjoint = true;
    for (size_t x : a) disjoint = disjoint && !b.count(x);
    const void *p = reinterpret_cast<const void *>(s[0].at), *q = reinterpret_cast<const void *>(s[1].at);
    for (const bool turned : {false, true}) {
      const bool got = turned ? sets_apart(q, row, s[1].n, nb, p, s[0].n, nb, dims)
                              : sets_apart(p, row, s[0].n, nb, q, s[1].n, nb, dims);
      if (got && !disjoint) fail("sets called apart share a byte");
      if (!got && disjoint) fail("parts of one tensor that share no byte are not called apart");
    }
    if (!rows_apart(row, s[0].n, nb, dims)) fail("rows of a part called overlapping");
    (disjoint ? apart : shared)++;
    if (disjoint && *a.begin() < *b.rbegin() && *b.begin() < *a.rbegin()) ++inside;
  }
  if (inside < 2000 || shared < 2000) fail("too few");
  // by name: per-head queries, keys and values; heads-first halves of a batch; one token
  const char *t = reinterpret_cast<const char *>(4096);
  const int n[3] = {4, 5, 2}, one[3] = {4, 1, 1};
  const size_t per_head[3] = {24, 96, 480}, heads_first[3] = {40, 8, 320};
  if (!sets_apart(t, 8, n, per_head, t + 8, n, per_head, 3) ||
      !sets_apart(t, 8, one, per_head, t + 16, one, per_head, 3) ||
      !sets_apart(t, 8, n, heads_first, t + 160, n, heads_first, 3) ||
      sets_apart(t, 8, n, per_head, t + 7, n, per_head, 3) ||
      sets_apart(t, 8, n, heads_first, t + 152, n, heads_first, 3))
    fail("layouts");
  std::puts("ok");
}
