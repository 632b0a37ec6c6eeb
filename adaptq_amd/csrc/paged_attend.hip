// paged_attend.hip -- attention of one new token per sequence over its pages.
//
// For the g query heads of a key head and the tokens t of [lo, n):
//   s_t = scale <q, k_t>,  o = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),
// with m the running maximum, in one pass over the rows.  Bound: the rows' bytes
// (2 * dim values a token and key head, used once by g heads), so everything else
// stays out of the way of the loads:
//
// * A wave takes a unit of 32 tokens (16 in fp32) for up to 16 query heads.  Both
//   products run on the matrix cores as 16 x 16 tiles straight from the registers
//   that the rows were loaded into, with no LDS and no exchange of lanes:
//   - S = K q^T: the operand K wants lane (row r, group g) to hold 8 channels of
//     token r, which is one 16-byte load; which 8 is free as long as q agrees.
//   - O^T = V^T P^T: P^T comes out of the first product in the layout that the
//     second wants (lane = query head, its registers = tokens) if token t of the
//     operand is the token whose score sits there; so group g loads the rows of
//     tokens 4g..4g+3 of each 16, 8 channels a lane, whole rows a load, and
//     transposes the 8 x 8 values of its tokens and channels in its own registers.
//   Both tiles have the query head in the lane, so the running maximum, the sum and
//   the rescaling are lane-local but for one maximum over the four groups.
// * The rows of the next unit are loaded before this one's are used, and the page
//   numbers of the one behind it before that.
// * Work is cut evenly over the resident blocks whatever the lengths (paged_split.hpp).
//
// Precision: scores, statistics and sums in fp32.  Queries and weights enter the
// half-precision products as the sum of three bf16 numbers, which holds fp32's 24 bits,
// or of two fp16 numbers, which leaves 2^-20 of them (scaled by a power of two a row so
// that none is too large or too small for it): 2^-9 of the output's own rounding.  (Two
// bf16 numbers, 2^-16, left one output of some hundreds a rounding away from fp32's.)
// fp32 rows use the fp32 matrix instructions.
#include <float.h>

#include <algorithm>

#include "paged.hpp"
#include "paged_split.hpp"
#include "rotary.hpp"

namespace aq {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kTile = 16;  // query heads of a segment
constexpr int kMaxBlocks = 1024;
// What a segment counts at the least, and what is never cut: its start and end cost a block
// about as much as the rows of 16 units (5 us).
constexpr int kMinUnits = 16;
constexpr int kBatch = 8;             // pieces of a join whose loads are in flight at once
constexpr int kGroup = 16;            // pieces of a group of a join
constexpr int kJoinAtOnce = 1 << 14;  // floats that are joined without groups
constexpr int kBeyond = 1 << 30;  // an offset behind every buffer

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(4))) int cint;  // uniform loads

struct Args {
  PagedShape p;
  PagedSeqs q;
  PagedAttend a;
  PagedAppend n;       // a step's rows (n.k null: attention alone)
  float scale2;        // of the scores, to base 2
  int group, q_tiles;  // query heads of a key head, and their tiles of 16
  int segs;            // segments of a sequence
  int64_t cap;         // tokens that the table has columns for
  PageOf page_of;
  int row_bytes;
  bool out_vec;
  int cus;
  float *partial;
  int *counters;        // [kMaxBlocks]: parts there of the segment cut first by a block
  int *group_counters;  // [2 * kMaxBlocks]: pieces there of the group that a slot begins
};

// What differs between the types of the rows.
template <typename T, int DP>
struct Kind {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kUnit = kHalf ? 32 : 16;
  static constexpr int kSubs = kUnit / 16;
  static constexpr int kVec = 16 / (int)sizeof(T);  // values of a K load
  static constexpr int kChunks = DP / (4 * kVec);   // K loads of a row
  // channels of a V load: a row over 16 lanes, at most 16 bytes each
  static constexpr int kVVec = DP / 16 < kVec ? DP / 16 : kVec;
  static constexpr int kVChunks = DP / (16 * kVVec);
  static constexpr int kVRows = kUnit / 4;  // rows of V that a lane loads
  // numbers of the type that queries and weights are cut into
  static constexpr int kTerms = !kHalf ? 1 : __is_same(T, _Float16) ? 2 : 3;
};

template <int BYTES>
struct VecOf {
  typedef u32x4 type;
};
template <>
struct VecOf<8> {
  typedef u32x2 type;
};

// A unit's rows as they were loaded.
template <typename T, int DP>
struct Rows {
  typedef Kind<T, DP> K;
  typedef typename VecOf<K::kVVec * sizeof(T)>::type V;
  u32x4 k[K::kSubs][K::kChunks];
  V v[K::kVRows][K::kVChunks];
};

// Where a unit's blocks of 16 tokens lie: the page (-1: nowhere) and the first slot.
template <int SUBS>
struct Where {
  int page[SUBS], slot[SUBS];
};

__device__ __forceinline__ float cross_max(float x) {  // over lanes l, l ^ 16, l ^ 32, l ^ 48
  const uint32_t a = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const float y = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const uint32_t b = __float_as_uint(y);
  const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ float cross_sum(float x) {
  const uint32_t a = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const float y = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  const uint32_t b = __float_as_uint(y);
  const auto s = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c, Bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Two values as sums of numbers of the type: the first the largest one that is below (in
// magnitude), the next the same of the rest or, as the last, the rest rounded.  Each has the
// value's sign and is not 0 for a value that is not (in fp16 from 2^-12 on, of what comes scaled
// to 2^14 and more; in bf16 from 2^-100 on): a product with an infinity stays that infinity.
__device__ __forceinline__ uint32_t below(float x) { return __float_as_uint(x) - (x != 0.0f); }

__device__ __forceinline__ void split2(float x, float y, uint32_t (&t)[2], _Float16) {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  t[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(__uint_as_float(below(x)),
                                                                 __uint_as_float(below(y))));
  const v2 h = __builtin_bit_cast(v2, t[0]);
  t[1] = __builtin_bit_cast(uint32_t,
                            __builtin_amdgcn_cvt_pkrtz(x - (float)h[0], y - (float)h[1]));
}
__device__ __forceinline__ void split2(float x, float y, uint32_t (&t)[3], Bf16) {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t a = below(x), b = below(y);
    t[i] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    x -= __uint_as_float(a & 0xFFFF0000u);
    y -= __uint_as_float(b & 0xFFFF0000u);
  }
  t[2] = __builtin_bit_cast(uint32_t, v2{(__bf16)x, (__bf16)y});
}

template <typename T, int TERMS>
__device__ __forceinline__ void split8(const float *x, u32x4 (&to)[TERMS]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t t[TERMS];
    split2(x[2 * i], x[2 * i + 1], t, T());
#pragma unroll
    for (int j = 0; j < TERMS; ++j) to[j][i] = t[j];
  }
}

// Partial results pass between blocks that may sit on different dies, whose L2 caches do not
// see each other's lines: they are stored past them and read past them (the device's scope,
// as its relaxed atomics are).  A fence of that scope instead writes back and drops a whole
// L2: it cost tens of microseconds a call.
__device__ __forceinline__ void put_shared(float *p, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t *>(p),
                     (uint64_t)__float_as_uint(y) << 32 | __float_as_uint(x), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 get_shared2(const float *p) {
  const uint64_t w = __hip_atomic_load(reinterpret_cast<const uint64_t *>(p), __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((uint32_t)w), __uint_as_float((uint32_t)(w >> 32)));
}
__device__ __forceinline__ f32x4 get_shared4(const float *p) {
  const float2 a = get_shared2(p), b = get_shared2(p + 2);
  return {a.x, a.y, b.x, b.y};
}
// Every store of this wave has reached the memory that all dies see.
__device__ __forceinline__ void stores_done() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// A partial result: the rows' sums [16][DP], then (m, l) of each row.
constexpr int part_floats(int dp) { return kTile * (dp + 2); }

// Where piece k of a cut segment lies: the first one began it (slot 1 of its block), the
// others go on with it (slot 0 of the blocks behind).
__device__ __forceinline__ int piece_slot(int first, int k) {
  return k == 0 ? 2 * first + 1 : 2 * (first + k);
}

// Pieces k0, k0 + step, ... (n of them) of a segment together, in their order, by the block
// that finished last.  Threads beyond one per 4 channels of a row share the pieces; a thread
// has the loads of kBatch pieces in flight at once.  put(row, channel, sums, max, sum).
template <int DP, typename Put>
__device__ __forceinline__ void join(const Args &g, int first, int piece0, int step, int n,
                                     int rows, int tid, float *lds, Put put) {
  constexpr int kPart = part_floats(DP);
  const int items = rows * (DP / 4), parts = max(1, kThreads / items);
  for (int i0 = 0; i0 < items; i0 += kThreads) {
    const int part = parts > 1 ? tid / items : 0;
    const int item = parts > 1 ? tid - part * items : i0 + tid;
    const bool mine = part < parts && item < items;
    const int row = item / (DP / 4), d = item % (DP / 4) * 4;
    float m = -INFINITY, l = 0.0f;
    f32x4 y = {0, 0, 0, 0};
    if (mine)
      for (int k0 = part; k0 < n; k0 += parts * kBatch) {
        float2 ml[kBatch];
        f32x4 x[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          const int k = min(k0 + j * parts, n - 1);  // (the last again: no weight)
          const float *from = g.partial + (int64_t)piece_slot(first, piece0 + k * step) * kPart;
          ml[j] = get_shared2(from + kTile * DP + 2 * row);
          x[j] = get_shared4(from + row * DP + d);
        }
        float top = m;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (k0 + j * parts >= n) ml[j].x = -INFINITY;
          top = fmaxf(top, ml[j].x);
        }
        if (top == -INFINITY) continue;
        const float keep = __builtin_amdgcn_exp2f(m - top);
        l *= keep;
        y *= keep;
        m = top;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (ml[j].x == -INFINITY) continue;
          const float e = __builtin_amdgcn_exp2f(ml[j].x - top);
          l = fmaf(e, ml[j].y, l);
          y += e * x[j];
        }
      }
    if (parts > 1) {
      float *at = lds + 8 * tid;
      if (mine) {
        *reinterpret_cast<f32x4 *>(at) = y;
        at[4] = m;
        at[5] = l;
      }
      __syncthreads();
      if (mine && part == 0) {
        float top = m;
        for (int k = 1; k < parts; ++k) top = fmaxf(top, at[8 * k * items + 4]);
        if (top != -INFINITY) {
          const float keep = __builtin_amdgcn_exp2f(m - top);
          l *= keep;
          y *= keep;
          for (int k = 1; k < parts; ++k) {
            const float *from = at + 8 * k * items;
            if (from[4] == -INFINITY) continue;
            const float e = __builtin_amdgcn_exp2f(from[4] - top);
            l = fmaf(e, from[5], l);
            y += e * *reinterpret_cast<const f32x4 *>(from);
          }
          m = top;
        }
      }
    }
    if (mine && part == 0) put(row, d, y, m, l);
  }
}

// A wave's running state over its units.
template <int DP>
struct State {
  float m, l;        // of query head lane & 15; l of this lane's tokens only
  f32x4 acc[DP / 16];
};

// DP: dim padded to 64, 128 or 256; EXACT: dim is DP; ONCE: one tile of query heads reads a row.
template <typename T, int DP, bool EXACT, bool ONCE>
struct Attend {
  typedef Kind<T, DP> K;
  typedef aq::Rows<T, DP> Rows;
  typedef aq::Where<K::kSubs> Where;
  static constexpr int kPolicy = ONCE ? 2 : 0;  // nt: the row leaves the caches first
  static constexpr int kQ = K::kHalf ? K::kChunks : DP / 4;  // operand registers of q
  // fp16 weights are taken times 2^15 (so is their sum): small ones stay normal numbers
  static constexpr float kLift = __is_same(T, _Float16) ? 15.0f : 0.0f;

  // this wave's view of a segment
  const Args &g;
  const int lane, row16, group4;
  int k_off[EXACT ? 1 : K::kChunks], v_off[EXACT ? 1 : 4 * K::kVChunks];  // bytes in 16 rows
  TokenSpan span;
  const int *table;
  int head, u_end;
  u32x4 qh[K::kHalf ? kQ : 1];  // the first numbers of the queries; the others are in LDS:
  const u32x4 *q_low;           // [kTerms - 1][kChunks][64 lanes]
  float qf[K::kHalf ? 1 : kQ];
  int q_shift = 0;  // fp16: the operands are the query times 2^-q_shift

  __device__ Attend(const Args &args, int lane_, const u32x4 *low)
      : g(args), lane(lane_), row16(lane_ & 15), group4(lane_ >> 4), q_low(low + lane_) {
    const int row = g.row_bytes, size = (int)sizeof(T);
    if (EXACT) {  // the rest of the offsets are constants
      k_off[0] = row16 * DP * size + K::kVec * group4 * size;
      v_off[0] = 4 * group4 * DP * size + K::kVVec * row16 * size;
    } else {  // channels past dim lie beyond every buffer: they load as 0
#pragma unroll
      for (int c = 0; c < K::kChunks; ++c)
        k_off[c] = k_channel(c) < g.p.dim ? row16 * row + k_channel(c) * size : kBeyond;
#pragma unroll
      for (int c = 0; c < K::kVChunks; ++c)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = K::kVVec * (row16 + 16 * c);
          v_off[4 * c + j] = d < g.p.dim ? (4 * group4 + j) * row + d * size : kBeyond;
        }
    }
  }

  __device__ int k_channel(int chunk) const {  // first of the 8 (4) channels of a K load
    return K::kVec * (group4 + 4 * chunk);
  }

  __device__ Where locate(int unit) const {
    Where w;
#pragma unroll
    for (int s = 0; s < K::kSubs; ++s) {
      const int b = unit * K::kSubs + s;  // block of 16 tokens
      w.page[s] = -1;
      w.slot[s] = 0;
      if (unit < u_end && b * 16 < span.n) {
        const int col = page_column(g.page_of, b);
        const int page = ((cint *)(uint64_t)table)[col];
        w.page[s] = page < g.p.n_pages ? page : -1;
        w.slot[s] = (b - col * g.page_of.blocks) * 16;
      }
    }
    return w;
  }

  // Rows of 16 tokens as a buffer that ends behind the last token (and is empty where
  // there is no page): whatever lies behind it loads as 0, without a branch.
  __device__ __amdgpu_buffer_rsrc_t rows16(const void *pool, const Where &w, int s, int t0) const {
    const int64_t page = max(w.page[s], 0);
    const char *at = static_cast<const char *>(pool) +
                     ((page * g.p.n_heads + head) * g.p.page_size + w.slot[s]) * g.row_bytes;
    const int rows = w.page[s] < 0 ? 0 : max(0, min(16, span.n - (t0 + 16 * s)));
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char *>(at), 0, __builtin_amdgcn_readfirstlane(rows * g.row_bytes), 0x00020000);
  }

  // A step's token: its rows, the key rotated, into its slot, by the wave that will load it.
  __device__ void append(int seq, int at) const {
    const int col = page_column(g.page_of, at >> 4);
    const int page = ((cint *)(uint64_t)table)[col];
    if (page < 0 || page >= g.p.n_pages) return;
    const int slot = at - col * g.p.page_size;
    const int64_t row = ((int64_t)page * g.p.n_heads + head) * g.p.page_size + slot;
    T *k = reinterpret_cast<T *>(static_cast<char *>(g.p.k_pages) + row * g.row_bytes);
    T *v = reinterpret_cast<T *>(static_cast<char *>(g.p.v_pages) + row * g.row_bytes);
    const T *kin = reinterpret_cast<const T *>(static_cast<const char *>(g.n.k) +
                                               seq * (int64_t)g.n.k_nb[1] + head * (int64_t)g.n.k_nb[0]);
    const T *vin = reinterpret_cast<const T *>(static_cast<const char *>(g.n.v) +
                                               seq * (int64_t)g.n.v_nb[1] + head * (int64_t)g.n.v_nb[0]);
    const RotaryTable &rt = g.p.rotary;
    for (int i = lane; i < g.p.dim / 2; i += 64) {
      const bool turns = i < rt.pairs;
      const int2 c = turns ? chunk_at<1>(i, rt.pairs, rt.interleaved) : make_int2(2 * i, 2 * i + 1);
      RowVec<T, 1> x{{kin[c.x]}}, y{{kin[c.y]}};
      if (turns) {
        const float2 cs = rotary_cos_sin(rt.steps[i], at, rt.amplitude);
        rotate_pairs<T, 1>(x, y, &cs, rt.interleaved, false);
      }
      k[c.x] = x.x[0];
      k[c.y] = y.x[0];
      v[2 * i] = vin[2 * i];
      v[2 * i + 1] = vin[2 * i + 1];
    }
  }

  __device__ void load(Rows &r, const Where &w, int unit) const {
    const int t0 = unit * K::kUnit;
    // (opaque here, so that what is added stays part of the loads instead of taking a
    // register each outside the loop)
    int k0 = k_off[0], v0 = v_off[0];
    asm volatile("" : "+v"(k0), "+v"(v0));
#pragma unroll
    for (int s = 0; s < K::kSubs; ++s) {
      const auto k = rows16(g.p.k_pages, w, s, t0);
#pragma unroll
      for (int c = 0; c < K::kChunks; ++c)
        r.k[s][c] = __builtin_amdgcn_raw_buffer_load_b128(
            k, EXACT ? k0 + c * 64 : k_off[EXACT ? 0 : c], 0, kPolicy);
    }
#pragma unroll
    for (int s = 0; s < K::kSubs; ++s) {
      const auto v = rows16(g.p.v_pages, w, s, t0);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < K::kVChunks; ++c) {
          constexpr int size = (int)sizeof(T);
          const int off = EXACT ? v0 + (j * DP + 16 * c * K::kVVec) * size
                                : v_off[EXACT ? 0 : 4 * c + j];
          if constexpr (K::kVVec * sizeof(T) == 8)
            r.v[4 * s + j][c] = __builtin_amdgcn_raw_buffer_load_b64(v, off, 0, kPolicy);
          else
            r.v[4 * s + j][c] = __builtin_amdgcn_raw_buffer_load_b128(v, off, 0, kPolicy);
        }
    }
  }

  __device__ void use(State<DP> &st, Rows &r, const Where &w, int unit) const {
    const int t0 = unit * K::kUnit;
    bool full = t0 >= span.lo && t0 + K::kUnit <= span.n, any = false;
#pragma unroll
    for (int s = 0; s < K::kSubs; ++s) {
      full = full && w.page[s] >= 0;
      any = any || (w.page[s] >= 0 && t0 + 16 * s + 16 > span.lo);
    }
    if (!any) return;  // (uniform)

    f32x4 s[K::kSubs];
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i) s[i] = f32x4{0, 0, 0, 0};
    if constexpr (K::kHalf) {
#pragma unroll
      for (int c = 0; c < K::kChunks; ++c)
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i) s[i] = mfma(r.k[i][c], qh[c], s[i], T());
#pragma unroll
      for (int t = 0; t < (K::kTerms - 1) * K::kChunks; ++t) {
        const u32x4 q = q_low[64 * t];
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i) s[i] = mfma(r.k[i][t % K::kChunks], q, s[i], T());
      }
    } else {
      f32x4 s2 = s[0];
#pragma unroll
      for (int c = 0; c < K::kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(r.k[0][c][i]), qf[4 * c + i],
                                                      s[0], 0, 0, 0);
          s2 = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(r.k[0][c][i + 1]),
                                                    qf[4 * c + i + 1], s2, 0, 0, 0);
        }
      s[0] += s2;
    }
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i)
      if constexpr (__is_same(T, _Float16)) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          s[i][j] = __builtin_amdgcn_ldexpf(s[i][j], q_shift) * g.scale2;
      } else {
        s[i] *= g.scale2;
      }
    if (!full) {
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = t0 + 16 * i + 4 * group4 + j;
          if (!(w.page[i] >= 0 && t >= span.lo && t < span.n)) s[i][j] = -INFINITY;
          // rows behind the last token were loaded as 0; those before the window are there
          if (t < span.lo)
#pragma unroll
            for (int c = 0; c < K::kVChunks; ++c) r.v[4 * i + j][c] = typename Rows::V(0u);
        }
    }
    // at least one token is here, so the maximum is finite from now on
    float top = fmaxf(st.m, -FLT_MAX);
    {
      float x = -INFINITY;
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i)
        x = fmaxf(x, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
      top = fmaxf(top, cross_max(x));
    }
    if (__any(top > st.m)) {
      const float keep = __builtin_amdgcn_exp2f(st.m - top);
      st.l *= keep;
#pragma unroll
      for (int i = 0; i < DP / 16; ++i) st.acc[i] *= keep;
      st.m = top;
    }
    float p[K::kUnit / 4];
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        p[4 * i + j] = __builtin_amdgcn_exp2f(s[i][j] - (top - kLift));
        st.l += p[4 * i + j];
      }
    if constexpr (K::kHalf) {
      u32x4 pt[K::kTerms];
      split8<T>(p, pt);
#pragma unroll
      for (int c = 0; c < K::kVChunks; ++c)
#pragma unroll
        for (int w2 = 0; w2 < K::kVVec / 2; ++w2) {
          u32x4 a, b;  // the 8 tokens of channels 2 w2 and 2 w2 + 1
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            a[x] = __builtin_amdgcn_perm(r.v[2 * x + 1][c][w2], r.v[2 * x][c][w2], 0x05040100u);
            b[x] = __builtin_amdgcn_perm(r.v[2 * x + 1][c][w2], r.v[2 * x][c][w2], 0x07060302u);
          }
          f32x4 &y = st.acc[c * K::kVVec + 2 * w2], &z = st.acc[c * K::kVVec + 2 * w2 + 1];
#pragma unroll
          for (int t = 0; t < K::kTerms; ++t) {
            y = mfma(a, pt[t], y, T());
            z = mfma(b, pt[t], z, T());
          }
        }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int c = 0; c < K::kVChunks; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            st.acc[4 * c + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                __uint_as_float(r.v[j][c][i]), p[j], st.acc[4 * c + i], 0, 0, 0);
    }
  }
};

// The lengths of up to 64 sequences, one a lane, and where their units end among the units
// of all of them.
struct Ends {
  int length;
  int64_t end, units;
};

__device__ __forceinline__ Ends ends_of(const Args &g, int lane, int unit, int b0) {
  const int b = b0 + lane;
  Ends e;
  e.length = g.q.lengths[min(b, g.q.n_seqs - 1)];
  e.units = 0;
  if (b < g.q.n_seqs)
    e.units = (int64_t)token_span(e.length, g.a.extra, g.a.window, g.cap, unit, kMinUnits).units *
              g.segs;
  e.end = e.units;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    if (k >= g.q.n_seqs) break;  // (uniform)
    const int64_t y = __shfl_up(e.end, k, 64);
    if (lane >= k) e.end += y;
  }
  return e;
}

__device__ __forceinline__ int64_t uniform(int64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane((uint32_t)x, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((uint32_t)(x >> 32), lane);
  return (int64_t)((uint64_t)hi << 32 | lo);
}

template <typename T, int DP, bool EXACT, bool ONCE, bool STEP>
__global__ __launch_bounds__(kThreads, DP == 256 ? 1 : 2) void attend_kernel(
    const Args g) {
  typedef Kind<T, DP> K;
  typedef Attend<T, DP, EXACT, ONCE> A;
  constexpr int S = DP + 4;
  __shared__ __align__(16) float s_acc[kWaves][kTile][S];  // first: the queries, in [0]
  __shared__ __align__(16) u32x4 s_q[K::kHalf ? (K::kTerms - 1) * K::kChunks * 64 : 1];
  __shared__ float s_m[kWaves][kTile], s_l[kWaves][kTile];
  __shared__ int s_last;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int dim = g.p.dim;

  // the block's share of the units, and the sequence that it begins in
  Ends e = ends_of(g, lane, K::kUnit, 0);
  const int n_seqs = g.q.n_seqs;
  int64_t total = uniform(e.end, min(n_seqs, 64) - 1);
  for (int b0 = 64; b0 < n_seqs; b0 += 64)
    total += uniform(ends_of(g, lane, K::kUnit, b0).end, min(n_seqs - b0, 64) - 1);
  const int64_t share = share_of(total, (int)gridDim.x, kWaves);
  const int64_t start = blockIdx.x * share, end = min(start + share, total);
  if (start >= end) return;
  int64_t base = 0;
  uint64_t past = __ballot(e.end > start);
  int seq = 0;
  while (!past && seq + 64 < n_seqs) {
    base += uniform(e.end, 63);
    seq += 64;
    e = ends_of(g, lane, K::kUnit, seq);
    past = __ballot(base + e.end > start && seq + lane < n_seqs);
  }
  if (!past) return;  // (only if the lengths changed under the call)
  const int first = __ffsll((unsigned long long)past) - 1;
  seq += first;
  int length = __builtin_amdgcn_readlane(e.length, first);
  base += uniform(e.end, first) - uniform(e.units, first);
  int64_t at = start;

  // this thread's pair of channels of the queries: a pair of the rotation, or two side by side
  const RotaryTable &rt = g.p.rotary;
  const int pair = tid % (DP / 2);
  const bool turns = pair < rt.pairs;
  const int c0 = !turns || rt.interleaved ? 2 * pair : pair;
  const int c1 = !turns || rt.interleaved ? 2 * pair + 1 : pair + rt.pairs;
  const uint64_t step = turns ? rt.steps[pair] : 0;

  A w(g, lane, s_q);
  int seg = -1, u0 = 0;
  const auto next = [&](const Piece &pc) {
    at += pc.u1 - u0;
    u0 = 0;
    if (++seg == g.segs) {
      seg = 0;
      if (++seq < n_seqs) length = ((cint *)(uint64_t)g.q.lengths)[seq];
      else at = end;
    }
  };
  while (at < end) {
    w.span = token_span(length, g.a.extra, g.a.window, g.cap, K::kUnit, kMinUnits);
    if (seg < 0) {
      const Start s = start_at(at, base, w.span.units);
      seg = __builtin_amdgcn_readfirstlane(s.seg);
      u0 = __builtin_amdgcn_readfirstlane(s.u0);
    }
    const Piece pc =
        piece_at(blockIdx.x, start, end, at, u0, w.span.units, w.span.short_, share, gridDim.x);
    if (pc.empty) {
      next(pc);
      continue;
    }
    const int head = __builtin_amdgcn_readfirstlane(seg / g.q_tiles);
    const int q0 = (seg - head * g.q_tiles) * kTile;
    const int rows = min(kTile, g.group - q0);
    const int64_t qh0 = (int64_t)head * g.group + q0;
    w.head = head;
    w.table = g.q.table + (int64_t)seq * g.q.stride;
    // (a short segment counts for more units than it has)
    w.u_end = min(w.span.first_unit + pc.u1, (w.span.n + K::kUnit - 1) / K::kUnit);
    int u = w.span.first_unit + u0 + wave;

    if (STEP && length >= 0 && length < g.cap) {
      // the token goes into its page by the wave whose units hold it
      const int last = length / K::kUnit, off = last - (w.span.first_unit + u0);
      if (last < w.u_end && off >= 0 && off % kWaves == wave) {
        w.append(seq, length);
        stores_done();
      }
    }
    typename A::Rows r0, r1;
    typename A::Where w0 = w.locate(u), w1 = w.locate(u + kWaves);
    w.load(r0, w0, u);

    // the queries, rotated, into LDS and from there into operands
    const char *q_at = static_cast<const char *>(g.a.q) + (int64_t)seq * g.a.q_nb[1] +
                       qh0 * (int64_t)g.a.q_nb[0];
    {
      float2 cs = make_float2(1.0f, 0.0f);
      if (turns) cs = rotary_cos_sin(step, length < 0 ? 0 : length + (g.a.extra - 1), rt.amplitude);
      for (int row = tid / (DP / 2); row < rows; row += 2 * kThreads / DP) {
        const T *q = reinterpret_cast<const T *>(q_at + row * (int64_t)g.a.q_nb[0]);
        const float x = c0 < dim ? row_get(q[c0]) : 0.0f, y = c1 < dim ? row_get(q[c1]) : 0.0f;
        s_acc[0][row][c0] = turns ? fmaf(x, cs.x, -(y * cs.y)) : x;
        s_acc[0][row][c1] = turns ? fmaf(y, cs.x, x * cs.y) : y;
      }
    }
    __syncthreads();
    // (rows that are no query's hold anything: their columns of the products go nowhere)
    if constexpr (K::kHalf) {
      // A rotated fp16 query may lie anywhere in fp32's range (the amplitude): the row's largest
      // value is taken to 2^14 to 2^15, where two fp16 numbers hold 2^-20 of it and of every
      // value down to 2^-16 of it, and 2^-38 of the largest below that; exact, as the shift is a
      // power of two.  (An infinity or NaN makes the row's scores that, whatever the rest.)
      if constexpr (__is_same(T, _Float16)) {
        float top = 0.0f;
#pragma unroll
        for (int c = 0; c < K::kChunks; ++c)
#pragma unroll
          for (int i = 0; i < 8; ++i)
            top = fmaxf(top, fabsf(s_acc[0][w.row16][w.k_channel(c) + i]));
        w.q_shift = __builtin_amdgcn_frexp_expf(cross_max(top)) - 15;
      }
#pragma unroll
      for (int c = 0; c < K::kChunks; ++c) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          x[i] = s_acc[0][w.row16][w.k_channel(c) + i];
          if constexpr (__is_same(T, _Float16)) x[i] = __builtin_amdgcn_ldexpf(x[i], -w.q_shift);
        }
        u32x4 q[K::kTerms];
        split8<T>(x, q);
        w.qh[c] = q[0];
        if (c % kWaves == wave)
#pragma unroll
          for (int t = 1; t < K::kTerms; ++t) s_q[((t - 1) * K::kChunks + c) * 64 + lane] = q[t];
      }
    } else {
#pragma unroll
      for (int c = 0; c < K::kChunks; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) w.qf[4 * c + i] = s_acc[0][w.row16][w.k_channel(c) + i];
    }
    __syncthreads();  // s_q is whole; before s_acc is written again

    State<DP> st;
    st.m = -INFINITY;
    st.l = 0.0f;
#pragma unroll
    for (int i = 0; i < DP / 16; ++i) st.acc[i] = f32x4{0, 0, 0, 0};
    while (u < w.u_end) {
      w.load(r1, w1, u + kWaves);
      typename A::Where next = w.locate(u + 2 * kWaves);
      w.use(st, r0, w0, u);
      u += kWaves;
      if (u >= w.u_end) break;
      w0 = next;
      w.load(r0, w0, u + kWaves);
      next = w.locate(u + 2 * kWaves);
      w.use(st, r1, w1, u);
      u += kWaves;
      w1 = next;
    }

    // the waves' parts together
    st.l = cross_sum(st.l);
    if (w.row16 < rows) {
#pragma unroll
      for (int c = 0; c < K::kVChunks; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = K::kVVec * (16 * c + 4 * w.group4 + r);
#pragma unroll
          for (int i = 0; i < K::kVVec; ++i)
            s_acc[wave][w.row16][d + i] = st.acc[c * K::kVVec + i][r];
        }
      if (w.group4 == 0) {
        s_m[wave][w.row16] = st.m;
        s_l[wave][w.row16] = st.l;
      }
    }
    __syncthreads();
    char *o_at = static_cast<char *>(g.a.out) + (int64_t)seq * g.a.out_nb[1];
    const auto put = [&](int row, int d, f32x4 y, float m, float l) {
      T *o = reinterpret_cast<T *>(o_at + (qh0 + row) * (int64_t)g.a.out_nb[0]) + d;
      if (d >= dim) return;
      y = m == -INFINITY ? f32x4{0, 0, 0, 0} : y / l;  // no tokens: zeros
      RowVec<T, 4> v;
#pragma unroll
      for (int i = 0; i < 4; ++i) row_put(v.x[i], y[i]);
      if (g.out_vec) {
        *reinterpret_cast<RowVec<T, 4> *>(o) = v;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = v.x[i];
      }
    };
    constexpr int kPart = part_floats(DP);
    int slot = 2 * blockIdx.x + pc.slot;  // where this block's part of a cut segment goes
    const auto put_part = [&](int row, int d, f32x4 y) {
      float *part = g.partial + (int64_t)slot * kPart + row * DP + d;
      put_shared(part, y[0], y[1]);
      put_shared(part + 2, y[2], y[3]);
    };
    const auto put_stats = [&](int row, float m, float l) {
      put_shared(g.partial + (int64_t)slot * kPart + kTile * DP + 2 * row, m, l);
    };
    for (int i = tid; i < rows * (DP / 4); i += kThreads) {
      const int row = i / (DP / 4), d = i % (DP / 4) * 4;
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int k = 0; k < kWaves; ++k) m = fmaxf(m, s_m[k][row]);
      f32x4 y = {0, 0, 0, 0};
      if (m != -INFINITY) {
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
          const float e = __builtin_amdgcn_exp2f(s_m[k][row] - m);
          l = fmaf(e, s_l[k][row], l);
          y += e * *reinterpret_cast<const f32x4 *>(&s_acc[k][row][d]);
        }
      }
      if (pc.whole) {
        put(row, d, y, m, l);
      } else {
        put_part(row, d, y);
        if (d == 0) put_stats(row, m, l);
      }
    }
    if (!pc.whole) {
      // Joined by the block that finishes last: all pieces at once, or, where they are more
      // than 64 KB, by groups whose last blocks leave the group's part each, and those then
      // (a CU reads some 20 GB/s past the caches.  65,536 tokens, one key head of 128, 16
      // query heads: 256 pieces at once 83 us, in groups 28; 84 pieces of one row 20 and 22).
      const int k = blockIdx.x - pc.first;
      const bool grouped = pc.pieces > kGroup && pc.pieces * rows * DP > kJoinAtOnce;
      int piece0 = grouped ? k / kGroup * kGroup : 0, step = 1;
      int n = grouped ? min(kGroup, pc.pieces - piece0) : pc.pieces;
      int *counter = grouped ? g.group_counters + piece_slot(pc.first, piece0)
                             : g.counters + pc.first;
      for (bool last = !grouped;; last = true) {
        stores_done();
        __syncthreads();
        if (tid == 0)
          s_last = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED,
                                          __HIP_MEMORY_SCOPE_AGENT) == n - 1;
        __syncthreads();
        if (!s_last) break;
        if (tid == 0)  // for the next call
          __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        slot = piece_slot(pc.first, piece0);
        join<DP>(g, pc.first, piece0, step, n, rows, tid, &s_acc[0][0][0],
                 [&](int row, int d, f32x4 y, float m, float l) {
                   if (last) {
                     put(row, d, y, m, l);
                   } else {
                     put_part(row, d, y);  // read by this item's threads alone
                     if (d == 0) {
                       s_m[0][row] = m;
                       s_l[0][row] = l;
                     }
                   }
                 });
        if (last) break;
        __syncthreads();  // every thread has read the first piece's (max, sum)
        if (tid < rows) put_stats(tid, s_m[0][tid], s_l[0][tid]);
        piece0 = 0;
        step = kGroup;
        n = (pc.pieces + kGroup - 1) / kGroup;
        counter = g.counters + pc.first;
      }
    }
    __syncthreads();
    next(pc);
  }
}

// Blocks that the card holds at once: two a CU, one at d256.
int most_blocks(int cus, int dp) { return std::min(kMaxBlocks, dp == 256 ? cus : 2 * cus); }

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

template <typename T, int DP, bool ONCE>
auto *kernel_of(const Args &g) {
  return g.p.dim == DP ? (g.n.k ? attend_kernel<T, DP, true, ONCE, true>
                                : attend_kernel<T, DP, true, ONCE, false>)
                       : (g.n.k ? attend_kernel<T, DP, false, ONCE, true>
                                : attend_kernel<T, DP, false, ONCE, false>);
}

template <typename T, int DP>
hipError_t launch(const Args &g, hipStream_t s) {
  // as many blocks as the card holds at once, or as there may be work for
  constexpr int unit = Kind<T, DP>::kUnit;
  int64_t longest = (g.cap + unit - 1) / unit;
  if (g.a.window > 0) longest = std::min(longest, (int64_t)g.a.window / unit + 2);
  const int64_t segments = g.q.n_seqs * (int64_t)g.segs;
  const int64_t most = segments * std::max(longest, (int64_t)kMinUnits);
  // Two blocks a CU overlap one's ends of segments with the other's rows (64 sequences x 8
  // heads of 8,192 tokens 315 us, with one 320; 88 segments of up to 20 units 18.6 and 18.9;
  // 1,666 of a few tokens 40 and 51), and with little work a wave of theirs has one unit
  // where it would have two (28 segments of 63 units 15.8 and 17.1).  Few long segments are
  // cut into twice as many pieces by them, and joining those costs more (one sequence of
  // 32,768 tokens, 8 heads: 32.6 us, with one block a CU 29.7; 36 segments of 128 units 27.9
  // and 25.8; one segment of 2,048 units, 8 query heads 23.4 and 19.7).  How long they may be is
  // the table's width, for the lengths are on the device: 32, 48 and 56 segments of up to
  // 1,280, 640 and 4,000 tokens take as long with a table of 8,192 or 131,072 tokens as with
  // one of their own (13.3, 13.2 and 23.9 us, within 0.1).
  const bool few_long = segments < g.cus / 16 ||
                        (segments < g.cus / 4 && most > 2 * kWaves * (int64_t)g.cus);
  const int resident = std::min(most_blocks(g.cus, DP), few_long ? g.cus : 2 * g.cus);
  const int blocks = (int)std::min((most + kWaves - 1) / kWaves, (int64_t)resident);
  // Rows that one tile of query heads reads are marked to leave the caches first (64
  // sequences x 8 heads of 8,192 tokens: 315 us, unmarked 358).  Rows that further tiles
  // read stay (one sequence of 131,072 tokens, 32 query heads on one: 32.0 us, marked 34.7;
  // 32 sequences of 8,192, 256 on 8: 311 and 308).
  if (g.q_tiles == 1)
    kernel_of<T, DP, true>(g)<<<blocks, kThreads, 0, s>>>(g);
  else
    kernel_of<T, DP, false>(g)<<<blocks, kThreads, 0, s>>>(g);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_type(const Args &g, hipStream_t s) {
  switch (padded_dim(g.p.dim)) {
    case 64: return launch<T, 64>(g, s);
    case 128: return launch<T, 128>(g, s);
    default: return launch<T, 256>(g, s);
  }
}

}  // namespace

size_t paged_workspace_bytes(const PagedShape &p) {
  return 4 * sizeof(int) * kMaxBlocks +
         2 * sizeof(float) * part_floats(padded_dim(p.dim)) * most_blocks(p.cus, padded_dim(p.dim));
}

hipError_t launch_paged_attend(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                               const PagedAppend *step, void *workspace, hipStream_t s) {
  Args g{};
  if (step) g.n = *step;
  g.p = p;
  g.q = q;
  g.a = a;
  const float log2e = 1.44269504088896340736f;
  g.scale2 = a.scale * log2e;
  g.group = a.q_heads / p.n_heads;
  g.q_tiles = (g.group + kTile - 1) / kTile;
  g.segs = p.n_heads * g.q_tiles;
  g.cap = std::min((int64_t)q.width * p.page_size, (int64_t)kMaxTokens);
  g.page_of = page_of_blocks(p.page_size);
  g.row_bytes = p.dim * (p.io == IoType::F32 ? 4 : 2);
  size_t x = reinterpret_cast<uintptr_t>(a.out) | a.out_nb[0] | a.out_nb[1];
  g.out_vec = x % (p.io == IoType::F32 ? 16 : 8) == 0;
  g.cus = p.cus;
  g.counters = static_cast<int *>(workspace);
  g.group_counters = g.counters + kMaxBlocks;
  g.partial = reinterpret_cast<float *>(g.counters + 4 * kMaxBlocks);
  switch (p.io) {
    case IoType::F32: return launch_type<float>(g, s);
    case IoType::F16: return launch_type<_Float16>(g, s);
    default: return launch_type<Bf16>(g, s);
  }
}

}  // namespace aq
