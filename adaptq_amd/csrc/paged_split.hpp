// paged_split.hpp -- how the paged attention's work is cut into blocks (host and
// device; tests/cpp/paged_split.cpp runs it on the CPU).
//
// A unit is a few tokens of one sequence that a wave takes in one pass.  A segment
// is the attention of one (sequence, key head, tile of up to 16 query heads): the
// sequence's units.  All segments' units in a row, sequence by sequence, are cut
// into equal shares, one a block, whatever the sequences' lengths; the lengths are
// read on the device, so the cut follows them in a captured graph too.  A block
// finishes the segments that lie inside its share and leaves a partial result for
// the ones that its share cuts: one that began before it (slot 0) and one that goes
// on behind it (slot 1).  A cut segment is joined by the block that finishes last.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define AQ_SPLIT_HD __host__ __device__ __forceinline__
#else
#define AQ_SPLIT_HD inline
#endif

namespace aq {

// The tokens that a sequence's attention is over: [lo, n), and their units.
struct TokenSpan {
  int lo, n;
  int first_unit, units;  // at least one unit, so that an empty sequence has a segment
};

// length: tokens held (negative: none), extra: more by now; cap: tokens that the table
// has columns for.
AQ_SPLIT_HD TokenSpan token_span(int length, int extra, int window, int64_t cap, int unit) {
  int64_t held = length < 0 ? 0 : (int64_t)length + extra;
  TokenSpan s;
  const int64_t lo = window > 0 && held > window ? held - window : 0;
  if (held > cap) held = cap;
  // (whole units of int tokens: the last one of 2^31 - 1 would end beyond)
  if (held > 0x7FFFFFE0) held = 0x7FFFFFE0;
  s.n = (int)held;
  s.lo = (int)(lo < held ? lo : held);
  s.first_unit = s.lo / unit;
  s.units = s.n > 0 ? (s.n - 1) / unit + 1 - s.first_unit : 1;
  if (s.units < 1) s.units = 1;
  return s;
}

// Units of a block: an equal share of the total, in whole passes of the block's waves.
AQ_SPLIT_HD int64_t share_of(int64_t total, int blocks, int waves) {
  int64_t s = (total + blocks - 1) / blocks;
  s = (s + waves - 1) / waves * waves;
  return s > waves ? s : waves;
}

// A block's next piece of work: units [u0, u1) of segment `seg` of a sequence whose
// segments begin at unit `base` and have `units` units each.
struct Piece {
  int seg, u0, u1;
  bool whole;       // the whole segment
  int slot;         // where its partial result goes (not whole)
  int64_t first;    // the first block with a piece of the segment, and how many have one
  int pieces;
};

AQ_SPLIT_HD Piece piece_at(int64_t at, int64_t end, int64_t base, int units, int64_t share) {
  Piece p;
  const int64_t off = at - base;
  p.seg = (int)(off / units);
  p.u0 = (int)(off - (int64_t)p.seg * units);
  p.u1 = end - at < units - p.u0 ? p.u0 + (int)(end - at) : units;
  p.whole = p.u0 == 0 && p.u1 == units;
  p.slot = p.u0 == 0 ? 1 : 0;
  const int64_t begin = base + (int64_t)p.seg * units;
  p.first = begin / share;
  p.pieces = (int)((begin + units - 1) / share - p.first) + 1;
  return p;
}

}  // namespace aq
