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
// Short segments are never cut: the block that one begins in has all of it.
#pragma once

#include <stdint.h>

#ifdef __HIPCC__
#define AQ_SPLIT_HD __host__ __device__ __forceinline__
#else
#define AQ_SPLIT_HD inline
#endif

namespace aq {

// Tokens of a sequence: whole units of them end within an int.
constexpr int kMaxTokens = 0x7FFFFFE0;

// Pages of blocks of 16 tokens: block b lies in page b / blocks = b * mul >> shift.  mul is
// 2^shift / blocks rounded up, by less than one, so b * mul is over 2^shift * (b / blocks) by
// less than b < 2^27: that is less than 2^shift / blocks, the distance to the next page, as
// shift = 27 + log2(blocks) rounded up.
struct PageOf {
  uint64_t mul;
  int shift, blocks;
};

inline PageOf page_of_blocks(int page_size) {
  PageOf p;
  p.blocks = page_size / 16;
  int bits = 0;
  while ((1 << bits) < p.blocks) ++bits;
  p.shift = 27 + bits;
  p.mul = (((uint64_t)1 << p.shift) + p.blocks - 1) / p.blocks;
  return p;
}

AQ_SPLIT_HD int page_column(const PageOf &p, int block) {
  return (int)((uint64_t)(uint32_t)block * p.mul >> p.shift);
}

// The tokens that a sequence's attention is over: [lo, n), and their units.
struct TokenSpan {
  int lo, n;
  int first_unit, units;  // units: at least `least`, those behind the last token empty
  bool short_;            // no more than `least` of them: not cut
};

// length: tokens held (negative: none), extra: more by now; cap: tokens that the table
// has columns for.  least: what a segment costs at the least, in units, so that a share
// does not fill with many short ones; 1 or more, for an empty sequence has segments too.
AQ_SPLIT_HD TokenSpan token_span(int length, int extra, int window, int64_t cap, int unit,
                                 int least) {
  int64_t held = length < 0 ? 0 : (int64_t)length + extra;
  TokenSpan s;
  const int64_t lo = window > 0 && held > window ? held - window : 0;
  if (held > cap) held = cap;
  if (held > kMaxTokens) held = kMaxTokens;
  s.n = (int)held;
  s.lo = (int)(lo < held ? lo : held);
  s.first_unit = s.lo / unit;
  s.units = s.n > 0 ? (s.n - 1) / unit + 1 - s.first_unit : 1;
  s.short_ = s.units <= least;
  if (s.short_) s.units = least;
  return s;
}

// The same where tokens before `first` are hidden and those before `prefix` stay seen behind a
// window: [lo, n) without [hole0, hole1).  Units inside the hole are not counted: from gap_at on,
// unit u of the launch is unit u + gap of the sequence.
struct SeenSpan : TokenSpan {
  int hole0, hole1;
  int gap_at, gap;
};

AQ_SPLIT_HD SeenSpan seen_span(int length, int extra, int window, int64_t cap, int unit, int least,
                               int first, int prefix) {
  SeenSpan s;
  const TokenSpan all = token_span(length, extra, 0, cap, unit, 1);
  const int n = all.n;
  const int64_t held = length < 0 ? 0 : (int64_t)length + extra;
  const int64_t back = window > 0 && held > window ? held - window : 0;
  const int w = (int)(back < n ? back : n);
  const int f = first < 0 ? 0 : first < n ? first : n, p = prefix < 0 ? 0 : prefix < n ? prefix : n;
  s.n = n;
  s.hole0 = s.hole1 = n;
  if (w <= p) {
    s.lo = f;
  } else if (f >= p) {
    s.lo = f > w ? f : w;
  } else {
    s.lo = f;
    s.hole0 = p;
    s.hole1 = w;
  }
  s.first_unit = s.lo / unit;
  s.units = s.lo < n ? (n - 1) / unit + 1 - s.first_unit : 1;
  s.gap_at = 0x7FFFFFFF;
  s.gap = 0;
  if (s.hole0 < s.hole1) {
    // the units that hold tokens before the hole end here; those behind it may begin in the same
    const int end = (s.hole0 - 1) / unit + 1, next = s.hole1 / unit;
    if (next > end) {
      s.gap_at = end;
      s.gap = next - end;
      // (a window that ends behind the table leaves nothing behind the hole)
      s.units -= s.hole1 < n ? s.gap : (n - 1) / unit + 1 - end;
    }
  }
  s.short_ = s.units <= least;
  if (s.short_) s.units = least;
  return s;
}

AQ_SPLIT_HD int real_unit(const SeenSpan &s, int unit) {
  return unit >= s.gap_at ? unit + s.gap : unit;
}

// The passes of a prompt's tile: the units of `keys` tokens that hold tokens of the runs [lo, pe)
// and [w, e), either of which may be empty.  Pass i is unit first + i, or, behind what lies
// between the runs, first + i + gap.  Tokens end at kMaxTokens, a unit of 64 may end beyond an
// int: its first token and the runs' ends are what is compared.
struct Passes {
  int first, count;
  int gap_at, gap;
};

AQ_SPLIT_HD Passes passes_of(int lo, int pe, int w, int e, int keys) {
  Passes p = {0, 0, 0x7FFFFFFF, 0};
  int end = 0;
  if (w < e) {
    p.first = w / keys;
    end = (e - 1) / keys + 1;
  }
  if (lo < pe) {
    const int p0 = lo / keys, p1 = (pe - 1) / keys + 1;
    if (p.first >= end) {
      p.first = p0;
      end = p1;
    } else {
      if (p.first > p1) {
        p.gap_at = p1;
        p.gap = p.first - p1;
      }
      end = (end > p1 ? end : p1) - p.gap;
      p.first = p0 < p.first ? p0 : p.first;
    }
  }
  p.count = end - p.first;
  return p;
}

AQ_SPLIT_HD int unit_of(const Passes &p, int pass) {
  const int u = p.first + pass;
  return u >= p.gap_at ? u + p.gap : u;
}

// Whether the unit's tokens from t0 on all lie in [a, b); whether some do (a and b not negative);
// and where they end among n > t0 tokens.
AQ_SPLIT_HD bool unit_within(int t0, int keys, int a, int b) { return t0 >= a && t0 <= b - keys; }
AQ_SPLIT_HD bool unit_meets(int t0, int keys, int a, int b) { return t0 < b && t0 > a - keys; }
AQ_SPLIT_HD int unit_end(int t0, int keys, int n) { return n - t0 < keys ? n : t0 + keys; }

// Units of a block: an equal share of the total, in whole passes of the block's waves.
AQ_SPLIT_HD int64_t share_of(int64_t total, int blocks, int waves) {
  const int64_t s = ((total + blocks - 1) / blocks + waves - 1) / waves * waves;
  return s > waves ? s : waves;
}

// A block's piece of a segment of `units` units: [u0, u1), empty if it is another block's.
// The block has units [start, end) of the whole, of which `at` is the segment's u0.
struct Piece {
  int u1;             // where the block goes on
  bool empty;
  bool whole;         // the whole segment
  int slot;           // where its partial result goes (not whole)
  int first, pieces;  // the first block with a piece of the segment, and how many have one
};

// blocks: of the launch; pieces are counted up to there, should the lengths have changed since
// the total was added up.
AQ_SPLIT_HD Piece piece_at(int block, int64_t start, int64_t end, int64_t at, int u0, int units,
                           bool short_, int64_t share, int blocks = 1 << 30) {
  Piece p;
  if (short_) {
    p.u1 = units;
    p.empty = u0 > 0;
    p.whole = true;
    p.slot = 0;
    p.first = block;
    p.pieces = 1;
    return p;
  }
  p.empty = false;
  p.u1 = end - at < units - u0 ? u0 + (int)(end - at) : units;
  p.whole = u0 == 0 && p.u1 == units;
  p.slot = u0 == 0 ? 1 : 0;
  // of the segment's units, those before this block and up to the last (both below 2^28, so
  // a larger share divides them as 2^31 does)
  const uint32_t s = share < 0x80000000 ? (uint32_t)share : 0x80000000u;
  const int64_t before = start - (at - u0);
  p.first = before > 0 ? block - (int)(((uint32_t)before + s - 1) / s) : block;
  const int last = block + (int)((uint32_t)(units - 1 - before) / s);
  p.pieces = (last < blocks ? last : blocks - 1) - p.first + 1;
  return p;
}

// Where a block begins: segment and unit within it, of a sequence whose segments begin at
// unit `base` of the whole.
struct Start {
  int seg, u0;
};

AQ_SPLIT_HD Start start_at(int64_t at, int64_t base, int units) {
  const int64_t off = at - base;
  const int seg = off >> 32 ? (int)(off / units) : (int)((uint32_t)off / (uint32_t)units);
  return {seg, (int)(off - (int64_t)seg * units)};
}

}  // namespace aq
