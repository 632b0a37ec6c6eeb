// paged_prompt.hip -- attention of several new tokens per sequence over its pages.
//
// For query p of a head and the tokens t that it sees (PagedScores):
//   s_t = scale <q, k_t>, capped and biased;  o = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m)
// in one pass over the rows with the running maximum m.  Bound: the matrix cores, 4 * dim
// operations a pair of query and token, with the exponentials beside them.
//
// * A row of a tile is a (token, query head) of one key head: its g query heads side by
//   side, so a tile of 128 rows reads the keys and values once for all of them and short
//   prompts fill it.  A wave has 32 rows, a block of four waves shares 64 tokens of keys
//   and values (32 in fp32) in LDS.
// * S^T = K Q^T and O^T = V^T P^T, as 32 x 32 tiles: both have the query in the lane, so
//   maximum, sum and rescaling stay in the lane but for one exchange between its halves,
//   and P^T goes from the first product's registers into the second's as it is, if the
//   values' tokens are taken in the order that the registers hold them: group i of four
//   tokens in half (i & 1) of the wave.
// * Rows of half types go from memory into LDS without passing registers, the next pass's while
//   this one's are used (one barrier a pass), and values are transposed as they are read.  fp32
//   rows are held in registers on the way.
// * Tiles of few queries over many tokens are cut over the tokens, and joined by a second
//   launch.
//
// Rows of half types: products of their values are exact and summed in fp32; rotated queries
// are rounded to the type, as Rotary's are; weights enter as two numbers of it, 2^-16 of a
// weight in bf16 and 2^-20 in fp16 (one number would be off by up to 2^-8 or 2^-11 each: as
// much as the outputs' own rounding, which then came to 1.4 to 1.7 times that of fp32
// weights).  fp32 rows use the fp32 matrix instructions.
#include <float.h>

#include <algorithm>

#include "paged.hpp"
#include "paged_split.hpp"
#include "rotary.hpp"
#include "scores.hpp"

namespace aq {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kRows = 32 * kWaves;  // of a tile
constexpr int kBeyond = 1 << 30;
constexpr int kBatch = 8;  // pieces of a join whose loads are in flight at once
// A maximum is followed only when it grows by more than this (in powers of two): weights
// are then up to 2^8 of what they would be, and most passes leave the sums as they are.  A sum
// of values of 2^119 and more may pass fp32's end by that; such a tile is gone over again with
// the maximum followed always.  (Sums of weights up to 1 still end where fp32 does.)
constexpr float kLazy = 8.0f;
// A piece's weight in a join at the least, fp32's smallest number: infinities of a piece of no
// weight stay what they are, and finite values stay below 2^-21.
constexpr float kLeast = 0x1p-149f;

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(4))) int cint;  // uniform loads

struct Args {
  PagedShape p;
  PagedSeqs q;
  PagedPrompt a;
  float scale2;        // of the scores, to base 2, positive
  float cap_in, cap2;  // 1 / cap of a score, cap to base 2
  bool cap_rough;      // (scores.hpp)
  bool flip;           // a negative scale: the queries change sign
  int group;           // query heads of a key head
  int64_t cap;         // tokens that the table has columns for
  PageOf page_of;
  int row_bytes;
  bool q_vec, out_vec;
  int64_t first_block, tiles;  // tiles: a bound, for every key head
  int splits;
  float *partial;  // [tiles][heads][splits][kRows][DP + 2]
};

// DP: dim padded to 64, 128 or 256, as rows lie in LDS; DC: to a multiple of 32, as the products
// take them.
template <typename T, int DP>
struct Kind {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kKeys = kHalf ? 64 : 32;     // tokens of a pass
  static constexpr int kSubs = kKeys / 32;
  static constexpr int kVec = 16 / (int)sizeof(T);  // values of 16 bytes
  static constexpr int kBlocks = kKeys / 16;        // blocks of 16 tokens, which lie together
  // a wave loads its share of the tokens, which lies in one block of 16; 16 bytes a lane
  static constexpr int kRowLoads = DP / kVec;
  static constexpr int kPasses = kKeys * kRowLoads / kThreads;
  static constexpr int kWaveRows = kKeys / kWaves;
  static constexpr int kRowsAPass = 64 / kRowLoads;
  // bytes of a row in LDS: half types whole rows, turned by the row, fp32 with room behind
  static constexpr int kKStride = DP * sizeof(T) + (kHalf ? 0 : 16);
  static constexpr int kVStride = DP * sizeof(T) + (kHalf ? 0 : 32);
  static constexpr int kBuffer = kKeys * (kKStride + kVStride);
  // which 16 bytes of a row lie in place 0 (half types): rows that are read together, 16 of keys
  // at one place and 4 of values at two pairs of places, lie in different banks
  static constexpr int key_turn(int row) { return DP == 64 ? row >> 1 & 7 : row & 15; }
  static constexpr int value_turn(int row) { return DP == 64 ? 4 * (row >> 1 & 1) : 4 * (row & 3); }
  // waves of a SIMD: at 64 channels there is room for three, which hide each other's exponentials
  // (2 prompts of 4,096, bf16, 16 query heads on 4, capped: 377 us, with two 391; as they are or
  // biased the same within 1; packed documents, fp16, 42.6, with four, which spill, 54)
  static constexpr int kResident = DP == 256 ? 1 : DP == 128 ? 2 : 3;
  // fp16 weights are taken times 2^7 (so is their sum): small ones stay normal numbers, and with
  // kLazy the largest stay below 2^15
  static constexpr float kLift = __is_same(T, _Float16) ? 7.0f : 0.0f;
};

__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c, _Float16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a),
                                                __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c, Bf16) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a),
                                                 __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

__device__ __forceinline__ uint32_t pack2(float x, float y, _Float16) {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, v2{(_Float16)x, (_Float16)y});
}
__device__ __forceinline__ uint32_t pack2(float x, float y, Bf16) {
  typedef __bf16 v2 __attribute__((ext_vector_type(2)));
  return __builtin_bit_cast(uint32_t, v2{(__bf16)x, (__bf16)y});
}

// Two weights as sums of two numbers of the type: what it holds of them, and the rest.
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo, Bf16 t) {
  const uint32_t a = __float_as_uint(x), b = __float_as_uint(y);
  hi = __builtin_amdgcn_perm(b, a, 0x07060302u);
  lo = pack2(x - __uint_as_float(a & 0xFFFF0000u), y - __uint_as_float(b & 0xFFFF0000u), t);
}
__device__ __forceinline__ void split2(float x, float y, uint32_t &hi, uint32_t &lo, _Float16 t) {
  typedef _Float16 v2 __attribute__((ext_vector_type(2)));
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
  const v2 h = __builtin_bit_cast(v2, hi);
  lo = pack2(x - (float)h[0], y - (float)h[1], t);
}

// Values that are infinite or NaN: whether there are, and zeros in their place.
template <typename T>
__device__ __forceinline__ bool wild(uint32_t x) {
  constexpr uint32_t top = __is_same(T, float) ? 0x7F800000u : __is_same(T, Bf16) ? 0x7F80u : 0x7C00u;
  if (sizeof(T) == 4) return (x & top) == top;
  return (x & top) == top || (x & top << 16) == top << 16;
}
template <typename T>
__device__ __forceinline__ uint32_t tamed(uint32_t x) {
  if (sizeof(T) == 4) return wild<T>(x) ? 0 : x;
  const uint32_t lo = x & 0xFFFFu, hi = x & 0xFFFF0000u;
  return (wild<T>(lo) ? 0 : lo) | (wild<T>(hi) ? 0 : hi);
}

template <typename T>
__device__ __forceinline__ bool wild4(u32x4 x) {
  return wild<T>(x[0]) || wild<T>(x[1]) || wild<T>(x[2]) || wild<T>(x[3]);
}
template <typename T>
__device__ __forceinline__ u32x4 tamed4(u32x4 x) {
  return u32x4{tamed<T>(x[0]), tamed<T>(x[1]), tamed<T>(x[2]), tamed<T>(x[3])};
}

// 16 bytes a lane of a buffer at each of the offsets, straight into LDS, in the lanes' order from
// `to` on; what lies beyond the buffer arrives as 0.  The caller waits (vmcnt) before it reads
// them.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"  // m0 is the compiler's, and named for that
template <int N>
__device__ __forceinline__ void load_lds(__amdgpu_buffer_rsrc_t from, const int (&off)[N],
                                         uint32_t to) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(to + 1024 * i), "v"(off[i]), "s"(from)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

// Of each 16 lanes the 4 x 16 values that they point at, a row of 16 four lanes: a column each.
__device__ __forceinline__ u32x2 read_tr(const char *lds) {
  typedef short v4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (__attribute__((address_space(3))) v4 *)(uintptr_t)(uint32_t)(uintptr_t)(
                     __attribute__((address_space(3))) const char *)lds));
}

__device__ __forceinline__ float half_max(float x) {  // over lanes l and l ^ 32
  const uint32_t a = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const uint32_t a = __float_as_uint(x);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
  for (int k = 32; k; k >>= 1) x = min(x, __shfl_xor(x, k, 64));
  return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) { return -wave_min(-x); }

// A tile: rows r0 to r0 + rows - 1 of a sequence's queries, of which there are `count`
// tokens from token q0 of the call on.
struct Tile {
  int seq, q0, count, r0, rows;  // rows 0: no tile
};

__device__ __forceinline__ Tile find_tile(const Args &g, int64_t index, int lane) {
  Tile t{0, 0, 0, 0, 0};
  int64_t base = 0;
  for (int b0 = 0; b0 < g.q.n_seqs; b0 += 64) {
    const int b = b0 + lane;
    int o0 = 0, o1 = 0;
    if (b < g.q.n_seqs) {
      o0 = min(max(g.a.offsets[b], 0), g.a.n_tokens);
      o1 = min(max(g.a.offsets[b + 1], o0), g.a.n_tokens);
    }
    const int64_t n = ((int64_t)(o1 - o0) * g.group + kRows - 1) / kRows;
    int64_t end = n;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const int64_t y = __shfl_up(end, k, 64);
      if (lane >= k) end += y;
    }
    const uint64_t past = __ballot(base + end > index);
    if (past) {
      const int l = __ffsll((unsigned long long)past) - 1;
      // within a sequence the last tiles, which see the most tokens, begin first
      const int64_t in = __shfl(base + end, l, 64) - 1 - index;
      t.seq = b0 + l;
      t.q0 = __builtin_amdgcn_readlane(o0, l);
      t.count = __builtin_amdgcn_readlane(o1, l) - t.q0;
      t.r0 = __builtin_amdgcn_readfirstlane((int)in) * kRows;
      t.rows = (int)min((int64_t)kRows, (int64_t)t.count * g.group - t.r0);
      return t;
    }
    base += __shfl(end, 63, 64);
  }
  return t;
}

// The tokens a row sees: [a, pe) and [w, e).
struct Sight {
  int a, pe, w, e;
};

template <typename T, int DP, int DC, bool SHAPED>
__global__ __launch_bounds__(kThreads, (Kind<T, DP>::kResident)) void prompt_kernel(const Args g) {
  typedef Kind<T, DP> K;
  extern __shared__ __align__(16) char lds[];
  __shared__ int s_red[kWaves][8];
  __shared__ __align__(4) uint8_t s_page[2][4];  // whether a block of 16 tokens has a page
  __shared__ int s_wild[2];  // the first and the last pass with an infinity or NaN among its values
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int dim = g.p.dim, heads = g.p.n_heads;
  // heads fastest: a head's tiles run on one die where there are eight heads, and share its
  // rows in that die's cache
  const int64_t block = g.first_block + blockIdx.x;
  const int head = (int)(block % heads);
  const int64_t rest = block / heads;
  const int64_t index = rest % g.tiles;
  const int split = (int)(rest / g.tiles);
  const Tile tile = find_tile(g, index, lane);
  if (tile.rows <= 0) return;

  // this lane's row
  const int row = wave * 32 + col;
  const bool live = row < tile.rows;
  const int r = tile.r0 + (live ? row : 0);
  const int token = r / g.group, q_head = head * g.group + (r - token * g.group);
  const int flat = tile.q0 + token;
  const int length = ((cint *)(uint64_t)g.q.lengths)[tile.seq];
  const int at = (int)max((int64_t)length - tile.count + token, (int64_t)INT_MIN + 1);
  const int n = (int)min((int64_t)max(length, 0), min(g.cap, (int64_t)kMaxTokens));
  Sight see;
  {
    const PagedScores &m = g.a.scores;
    const int pre = m.prefix ? min(max(m.prefix[flat], 0), n) : 0;
    see.a = m.first ? min(max(m.first[flat], 0), n) : 0;
    see.e = max(min(max(at, -1) + 1, n), pre);
    see.pe = max(pre, see.a);
    const int64_t w = m.window > 0 ? (int64_t)at - m.window + 1 : 0;
    see.w = (int)min(max(w, (int64_t)see.a), (int64_t)see.e);
    if (see.w <= see.pe) see.w = see.a, see.pe = see.a;  // one run
    if (!live) see = Sight{INT_MAX, 0, INT_MAX, 0};
  }
  // what the rows of this wave and of the block see between them: the runs [lo, pe) and
  // [w, e), and what all of them see: [w_all, e_all)
  const bool pre = see.pe > see.a;
  const int wave_lo = wave_min(pre ? see.a : see.w), wave_e = wave_max(see.e);
  const int wave_w_all = wave_max(live ? see.w : 0), wave_e_all = wave_min(live ? see.e : INT_MAX);
  const bool wave_pre = __any(pre);
  const int red[6] = {wave_min(pre ? see.a : INT_MAX), wave_max(pre ? see.pe : 0),
                      wave_min(see.w), wave_e, wave_w_all, wave_e_all};
  if (lane < 6) {
    int x = red[0];
#pragma unroll
    for (int i = 1; i < 6; ++i) x = lane == i ? red[i] : x;
    s_red[wave][lane] = x;
  }
  if (tid == 0) s_wild[0] = INT_MAX, s_wild[1] = -1;
  __syncthreads();
  int lo = INT_MAX, pe = 0, w = INT_MAX, e = 0, w_all = 0, e_all = INT_MAX;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    lo = min(lo, s_red[k][0]);
    pe = max(pe, s_red[k][1]);
    w = min(w, s_red[k][2]);
    e = max(e, s_red[k][3]);
    w_all = max(w_all, s_red[k][4]);
    e_all = min(e_all, s_red[k][5]);
  }
  lo = __builtin_amdgcn_readfirstlane(lo), pe = __builtin_amdgcn_readfirstlane(pe);
  w = __builtin_amdgcn_readfirstlane(w), e = __builtin_amdgcn_readfirstlane(e);
  w_all = __builtin_amdgcn_readfirstlane(w_all), e_all = __builtin_amdgcn_readfirstlane(e_all);

  const Passes passes = passes_of(lo, pe, w, e, K::kKeys);
  const int units = passes.count;
  const int i0 = (int)((int64_t)units * split / g.splits),
            i1 = (int)((int64_t)units * (split + 1) / g.splits);

  // where this thread's parts of the rows lie.  Half types: LDS is filled in the order of the
  // lanes, so the lane's own part of a row is turned.
  const int *table = g.q.table + (int64_t)tile.seq * g.q.stride;
  const int wave_row = wave * K::kWaveRows;  // first of the wave's tokens of a pass
  const int l_row = lane / K::kRowLoads, l_chunk = lane % K::kRowLoads;
  int k_off[K::kPasses], v_off[K::kPasses];
#pragma unroll
  for (int p = 0; p < K::kPasses; ++p) {
    const int row = p * K::kRowsAPass + l_row, in = (wave_row & 15) + row;
    const int kc = K::kVec * (K::kHalf ? l_chunk ^ K::key_turn(in) : l_chunk);
    const int vc = K::kVec * (K::kHalf ? l_chunk ^ K::value_turn(in) : l_chunk);
    k_off[p] = kc < dim ? in * g.row_bytes + kc * (int)sizeof(T) : kBeyond;
    v_off[p] = vc < dim ? in * g.row_bytes + vc * (int)sizeof(T) : kBeyond;
  }
  const uint32_t lds_at = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)lds);
  u32x4 k_in[K::kHalf ? 1 : K::kPasses], v_in[K::kHalf ? 1 : K::kPasses];

  const auto real = [&](int i) { return unit_of(passes, i); };
  // Where the wave's tokens of 64 passes lie, a pass a lane: the offset of their block's rows in
  // the pools, and how many bytes of it are there (0: no page, or no tokens).
  uint64_t at64 = 0;
  int bytes64 = 0;
  const auto locate = [&](int i) {
    const int b = (real(i + lane) * K::kKeys + wave_row) >> 4;
    bytes64 = 0;
    at64 = 0;
    if (i + lane < i1 && b * 16 < n) {
      const int c = page_column(g.page_of, b);
      const int page = table[c];
      if (page >= 0 && page < g.p.n_pages) {
        at64 = (((uint64_t)page * heads + head) * g.p.page_size + (b - c * g.page_of.blocks) * 16) *
               (uint64_t)g.row_bytes;
        bytes64 = min(16, n - 16 * b) * g.row_bytes;
      }
    }
  };
  // A block's rows as a buffer that ends behind the last token.  Half types: straight into LDS,
  // where the buffer of pass i is free.
  const auto load = [&](int i) {
    const int j = (i - i0) & 63;
    if (j == 0 && i != i0) locate(i);
    const uint64_t at = (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(at64 >> 32), j) << 32 |
                        (uint32_t)__builtin_amdgcn_readlane((int)at64, j);
    const int bytes = __builtin_amdgcn_readlane(bytes64, j);
    const auto ks = __builtin_amdgcn_make_buffer_rsrc(static_cast<char *>(g.p.k_pages) + at, 0,
                                                      bytes, 0x00020000);
    const auto vs = __builtin_amdgcn_make_buffer_rsrc(static_cast<char *>(g.p.v_pages) + at, 0,
                                                      bytes, 0x00020000);
    const int buffer = (i - i0) & 1;
    if constexpr (K::kHalf) {
      const uint32_t to = lds_at + buffer * K::kBuffer + wave_row * K::kKStride;
      load_lds(ks, k_off, to);
      load_lds(vs, v_off, to + K::kKeys * K::kKStride);
    } else {
#pragma unroll
      for (int p = 0; p < K::kPasses; ++p) {
        k_in[p] = __builtin_amdgcn_raw_buffer_load_b128(ks, k_off[p], 0, 0);
        v_in[p] = __builtin_amdgcn_raw_buffer_load_b128(vs, v_off[p], 0, 0);
      }
    }
    if (lane == 0 && wave_row % 16 == 0) s_page[buffer][wave_row / 16] = bytes > 0;
  };
  const auto all_seen = [&](int t0) { return unit_within(t0, K::kKeys, w_all, e_all); };
  // The loads of pass i are in LDS (of this wave).  An infinity or NaN among the values of a token
  // that some query does not see must not meet its weight of 0: zeros take its place, and at the
  // end it is added for the queries that do see it.  A weight's second number may be 0 too, or a
  // weight below the smallest number: where that shows, the passes that all queries see are gone
  // over in the same way (tame_all).
  bool tame_all = false;
  float lazy = kLazy;
  const auto found = [&](int i) {
    if (lane == 0) {
      atomicMin(&s_wild[0], i);
      atomicMax(&s_wild[1], i);
    }
  };
  const auto arrive = [&](int i) {
    char *to = lds + ((i - i0) & 1) * K::kBuffer;
    char *v_to = to + K::kKeys * K::kKStride;
    const bool whole = !tame_all && all_seen(real(i) * K::kKeys);
    if constexpr (K::kHalf) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      if (whole) return;
#pragma unroll
      for (int p = 0; p < K::kPasses; ++p) {
        u32x4 *at = reinterpret_cast<u32x4 *>(v_to + wave_row * K::kVStride + p * 1024 + lane * 16);
        const u32x4 y = *at;
        if (!__any(wild4<T>(y))) continue;
        found(i);
        *at = tamed4<T>(y);
      }
    } else {
#pragma unroll
      for (int p = 0; p < K::kPasses; ++p) {
        const int row = wave_row + p * K::kRowsAPass + l_row;
        u32x4 y = v_in[p];
        if (!whole && __any(wild4<T>(y))) {
          found(i);
          y = tamed4<T>(y);
        }
        *reinterpret_cast<u32x4 *>(to + row * K::kKStride + l_chunk * 16) = k_in[p];
        *reinterpret_cast<u32x4 *>(v_to + row * K::kVStride + l_chunk * 16) = y;
      }
    }
  };

  // under way while the queries come; but LDS holds the cosines first
  const bool early = !K::kHalf || g.p.rotary.pairs == 0;
  locate(i0);
  if (early && i0 < i1) load(i0);

  // the queries, rotated: cosines and sines of the tile's tokens through LDS
  const RotaryTable &rt = g.p.rotary;
  const char *q_at = static_cast<const char *>(g.a.q) + flat * (int64_t)g.a.q_nb[1] +
                     q_head * (int64_t)g.a.q_nb[0];
  const T *q_row = reinterpret_cast<const T *>(q_at);
  float2 *s_cs = reinterpret_cast<float2 *>(lds);
  const int token0 = tile.r0 / g.group;
  if (rt.pairs) {
    const int tokens = (tile.r0 + tile.rows - 1) / g.group - token0 + 1;
    for (int i = tid; i < tokens * rt.pairs; i += kThreads) {
      const int t = i / rt.pairs;
      s_cs[i] = rotary_cos_sin(rt.steps[i - t * rt.pairs],
                               (int)((int64_t)length - tile.count + token0 + t), rt.amplitude);
    }
    __syncthreads();
  }
  u32x4 qh[K::kHalf ? DC / 16 : 1];
  float qf[K::kHalf ? 1 : DC / 2];
  {
    const float2 *cs = s_cs + (token - token0) * rt.pairs;
    constexpr int N = K::kVec, kStep = 2 * N;
    typedef RowVec<T, N> Vec;
    const auto vec = [&](int d0) {  // channels d0 to d0 + N - 1
      Vec x;
      if (g.q_vec && d0 + N <= dim) return load_rows<false, T, N>(q_row + d0);
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (d0 + i < dim) x.x[i] = q_row[d0 + i];
        else row_put(x.x[i], 0.0f);
      return x;
    };
    Vec x[DC / kStep];
#pragma unroll
    for (int c = 0; c < DC / kStep; ++c) x[c] = vec(kStep * c + N * half);
    if (rt.pairs && !rt.interleaved && rt.pairs % N == 0) {
      // the pairs' other members are vectors too
      Vec y[DC / kStep];
#pragma unroll
      for (int c = 0; c < DC / kStep; ++c) {
        const int d0 = kStep * c + N * half;
        y[c] = vec(d0 < rt.pairs ? d0 + rt.pairs : d0 < 2 * rt.pairs ? d0 - rt.pairs : d0);
      }
#pragma unroll
      for (int c = 0; c < DC / kStep; ++c) {
        const int d0 = kStep * c + N * half;
        if (d0 >= 2 * rt.pairs) continue;
        const bool one = d0 < rt.pairs;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float u = row_get(x[c].x[i]), v = row_get(y[c].x[i]);
          const float2 a = cs[one ? d0 + i : d0 + i - rt.pairs];
          row_put(x[c].x[i], one ? fmaf(u, a.x, -(v * a.y)) : fmaf(u, a.x, v * a.y));
        }
      }
    } else if (rt.pairs) {
#pragma unroll
      for (int c = 0; c < DC / kStep; ++c) {
        const Vec own = x[c];
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int d = kStep * c + N * half + i;
          if (d >= 2 * rt.pairs) continue;
          const bool one = rt.interleaved ? !(i & 1) : d < rt.pairs;
          const int pair = rt.interleaved ? d >> 1 : one ? d : d - rt.pairs;
          const float u = row_get(own.x[i]);
          const float v = row_get(rt.interleaved ? own.x[i ^ 1]
                                                 : q_row[one ? d + rt.pairs : d - rt.pairs]);
          const float2 a = cs[pair];
          row_put(x[c].x[i], one ? fmaf(u, a.x, -(v * a.y)) : fmaf(u, a.x, v * a.y));
        }
      }
    }
#pragma unroll
    for (int c = 0; c < DC / kStep; ++c) {
      if constexpr (K::kHalf) {
        qh[c] = __builtin_bit_cast(u32x4, x[c]);
        if (g.flip) qh[c] ^= 0x80008000u;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          qf[N * c + i] = g.flip ? -row_get(x[c].x[i]) : row_get(x[c].x[i]);
      }
    }
  }
  float slope2 = 0.0f;
  if (SHAPED && g.a.scores.slopes) slope2 = g.a.scores.slopes[q_head] * kLog2e;
  if (rt.pairs) __syncthreads();  // the cosines are read: LDS is the rows' now

  f32x16 acc[DC / 32];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < DC / 32; ++i) acc[i] = f32x16{0};

  // where this lane reads: keys 16 bytes of its row, values 4 tokens of 16 channels a group of 16
  // lanes, 8 bytes each, which the load transposes
  const uint32_t k_at = col * K::kKStride + ((half ^ K::key_turn(col)) << 4);
  const int in16 = lane & 15;
  const uint32_t v_at0 = K::kKeys * K::kKStride + (4 * half + (in16 >> 2)) * K::kVStride +
                         (((2 * ((lane >> 4) & 1) + ((lane >> 1) & 1)) ^ K::value_turn(in16 >> 2))
                          << 4) +
                         8 * (lane & 1);

  typedef f32x16 Scores[K::kSubs];
  const auto products = [&](Scores &s, int buffer) {
    const char *buf = lds + buffer * K::kBuffer;
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i) s[i] = f32x16{0};
    if constexpr (K::kHalf) {
#pragma unroll
      for (int c = 0; c < DC / 16; ++c)
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i) {
          const u32x4 k = *reinterpret_cast<const u32x4 *>(buf + (k_at ^ (c << 5)) +
                                                           32 * i * K::kKStride);
          s[i] = mfma(k, qh[c], s[i], T());
        }
    } else {
#pragma unroll
      for (int c = 0; c < DC / 8; ++c) {
        const f32x4 k =
            *reinterpret_cast<const f32x4 *>(buf + col * K::kKStride + 32 * c + 16 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[i], qf[4 * c + i], s[0], 0, 0, 0);
      }
    }
  };
  // What follows the products of a pass.
  const auto weigh = [&](Scores &s, int buffer, int t0) {
    const char *buf = lds + buffer * K::kBuffer;
    const char *v_at = buf + K::kKeys * K::kKStride;
    const uint32_t there_are = *reinterpret_cast<const uint32_t *>(s_page[buffer]);
    const uint32_t pages = __builtin_amdgcn_readfirstlane(there_are);
    constexpr uint32_t kAll = K::kBlocks == 4 ? 0x01010101u : 0x0101u;
    const bool full = unit_within(t0, K::kKeys, wave_w_all, wave_e_all) && (pages & kAll) == kAll;
    const int t1 = t0 + 4 * half;
    float scale2 = g.scale2;
    if constexpr (SHAPED) {
      const PagedScores &sc = g.a.scores;
      const float cap_in = g.cap_in, cap2 = g.cap2;
      if (K::kHalf && g.cap_rough) {
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[i][j] = capped<false>(s[i][j], cap_in, cap2);
      } else if (sc.softcap > 0.0f) {
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[i][j] = capped<true>(s[i][j], cap_in, cap2);
      } else {
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i) s[i] *= scale2;
      }
      if (sc.slopes) {
        const float d0 = (float)(at - t1);
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j)
            s[i][j] = fmaf(-slope2, fabsf(d0 - (float)(32 * i + 8 * (j / 4) + j % 4)), s[i][j]);
      }
      scale2 = 1.0f;
    }
    float top = -INFINITY;
    if (!full) {
      // t is in [w, e) if t - w is below e - w as a number without sign; likewise [a, pe)
      bool any = false;
      const uint32_t in_w = t1 - see.w, in_a = t1 - see.a;
      const uint32_t size_w = max(see.e - see.w, 0), size_a = max(see.pe - see.a, 0);
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int d = 32 * i + 8 * (j / 4) + j % 4;
          bool there = in_w + d < size_w;
          if (wave_pre) there = there || in_a + d < size_a;
          there = there && (pages >> 8 * (2 * i + j / 8) & 1);
          any = any || there;
          s[i][j] = there ? s[i][j] : -INFINITY;
        }
      if (any) top = -FLT_MAX;
    } else {
      top = -FLT_MAX;  // there are tokens, so the maximum is finite, whatever they score
    }
    {
      float y = -INFINITY;
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) y = fmaxf(y, s[i][j]);
      top = half_max(fmaxf(top, y * scale2));
    }
    if (__any(top > m + lazy)) {  // (m is minus infinity at first)
      const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      l *= keep;
#pragma unroll
      for (int i = 0; i < DC / 32; ++i) acc[i] *= keep;
      m = to;
    }
    const float from = fmaxf(m, -FLT_MAX) - K::kLift;
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        s[i][j] = __builtin_amdgcn_exp2f(SHAPED ? s[i][j] - from : fmaf(s[i][j], scale2, -from));
        l += s[i][j];
      }
    if constexpr (K::kHalf) {
#pragma unroll
      for (int k = 0; k < K::kKeys / 16; ++k) {
        u32x4 p, rest;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint32_t hi, lo;
          split2(s[k / 2][8 * (k % 2) + 2 * j], s[k / 2][8 * (k % 2) + 2 * j + 1], hi, lo, T());
          p[j] = hi;
          rest[j] = lo;
        }
#pragma unroll
        for (int i = 0; i < DC / 32; ++i) {
          const char *from = buf + (v_at0 ^ (i << 6)) + 16 * k * K::kVStride;
          const u32x2 v0 = read_tr(from), v1 = read_tr(from + 8 * K::kVStride);
          const u32x4 v = {v0[0], v0[1], v1[0], v1[1]};
          acc[i] = mfma(v, p, acc[i], T());
          acc[i] = mfma(v, rest, acc[i], T());
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < DC / 32; ++i) {
          const float v = *reinterpret_cast<const float *>(
              v_at + (8 * (j / 4) + 4 * half + j % 4) * K::kVStride + (32 * i + col) * 4);
          acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[0][j], acc[i], 0, 0, 0);
        }
    }
  };

  if (!early && i0 < i1) load(i0);
#pragma clang loop unroll(disable)
  for (;;) {
    for (int i = i0; i < i1; ++i) {
      arrive(i);
      __syncthreads();  // pass i is there, and the buffer of pass i - 1 free
      if (i + 1 < i1) load(i + 1);
      const int t0 = real(i) * K::kKeys;
      if (unit_meets(t0, K::kKeys, wave_lo, wave_e)) {
        Scores s;
        products(s, (i - i0) & 1);
        weigh(s, (i - i0) & 1, t0);
      }
    }
    // a sum that is not finite, of weights that are numbers: once more without the values that
    // make it so, and if it is too large by itself, with smaller weights
    float zero = 0.0f;
#pragma unroll
    for (int i = 0; i < DC / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; ++j) zero = fmaf(acc[i][j], 0.0f, zero);
    const bool weighed = half_sum(l) <= FLT_MAX;  // (not NaN)
    const bool odd = live && weighed && zero != 0.0f;
    if (!__syncthreads_or(odd) || lazy == 0.0f) break;
    if (tame_all) lazy = 0.0f;
    tame_all = true;
    m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < DC / 32; ++i) acc[i] = f32x16{0};
    locate(i0);
    if (i0 < i1) load(i0);
  }

  if (s_wild[1] >= 0) {
    // the tokens of the passes that not every query sees whole, one by one
    for (int i = s_wild[0]; i <= s_wild[1]; ++i) {
      const int t0 = real(i) * K::kKeys;
      if (!tame_all && all_seen(t0)) continue;
      for (int t = t0, end = unit_end(t0, K::kKeys, n); t < end; ++t) {
        const int c = page_column(g.page_of, t >> 4);
        const int page = ((cint *)(uint64_t)table)[c];
        if (page < 0 || page >= g.p.n_pages) continue;
        const T *v = reinterpret_cast<const T *>(
            static_cast<const char *>(g.p.v_pages) +
            (((int64_t)page * heads + head) * g.p.page_size + (t - c * g.p.page_size)) *
                g.row_bytes);
        const bool there = (t >= see.w && t < see.e) || (t >= see.a && t < see.pe);
        bool some = false;
        for (int d = lane; d < dim; d += 64) some = some || !(fabsf(row_get(v[d])) <= FLT_MAX);
        if (!__any(some)) continue;
#pragma unroll
        for (int k = 0; k < DC / 32; ++k)
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const int d = 32 * k + 8 * (j / 4) + 4 * half + j % 4;
            const float x = d < dim ? row_get(v[d]) : 0.0f;
            if (there && !(fabsf(x) <= FLT_MAX)) acc[k][j] += x;
          }
      }
    }
  }
  l = half_sum(l);
  if (!live) return;
  if (g.splits > 1) {
    float *part = g.partial + (((index * heads + head) * g.splits + split) * kRows + row) * (DP + 2);
#pragma unroll
    for (int i = 0; i < DC / 32; ++i)
#pragma unroll
      for (int j = 0; j < 16; j += 2)
        *reinterpret_cast<float2 *>(part + 32 * i + 8 * (j / 4) + 4 * half + j % 4) =
            make_float2(acc[i][j], acc[i][j + 1]);
    if (half == 0) *reinterpret_cast<float2 *>(part + DP) = make_float2(m, l);
    return;
  }
  T *o = reinterpret_cast<T *>(static_cast<char *>(g.a.out) + flat * (int64_t)g.a.out_nb[1] +
                               q_head * (int64_t)g.a.out_nb[0]);
#pragma unroll
  for (int i = 0; i < DC / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const int d = 32 * i + 2 * j + 4 * half;
      if (d >= dim) continue;
      RowVec<T, 4> y;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        row_put(y.x[k], m == -INFINITY ? 0.0f : acc[i][j + k] / l);  // nothing seen: zeros
      if (g.out_vec) {
        *reinterpret_cast<RowVec<T, 4> *>(o + d) = y;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) o[d + k] = y.x[k];
      }
    }
}

// The parts of cut tiles together, in their order.
template <typename T, int DP>
__global__ __launch_bounds__(kThreads) void join_kernel(const Args g) {
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t block = g.first_block + blockIdx.x;
  constexpr int kItems = kRows * DP / 4, kBlocksATile = kItems / (4 * kThreads);
  const int64_t at = block / kBlocksATile;
  const int head = (int)(at % g.p.n_heads);
  const Tile tile = find_tile(g, at / g.p.n_heads, lane);
  if (tile.rows <= 0) return;
  const int item0 = (int)(block % kBlocksATile) * 4 * kThreads;
  for (int item = item0 + tid; item < item0 + 4 * kThreads; item += kThreads) {
    const int row = item / (DP / 4), d = item % (DP / 4) * 4;
    if (row >= tile.rows || d >= g.p.dim) continue;
    const float *part = g.partial + (at * g.splits * kRows + row) * (DP + 2);
    float m = -INFINITY, l = 0.0f;
    f32x4 y = {0, 0, 0, 0};
    constexpr int64_t kPart = (int64_t)kRows * (DP + 2);
    for (int k0 = 0; k0 < g.splits; k0 += kBatch) {
      float2 ml[kBatch], a[kBatch], b[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {  // (the last again: no weight)
        const float *from = part + min(k0 + k, g.splits - 1) * kPart;
        ml[k] = *reinterpret_cast<const float2 *>(from + DP);
        a[k] = *reinterpret_cast<const float2 *>(from + d);
        b[k] = *reinterpret_cast<const float2 *>(from + d + 2);
      }
      float to = m;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (k0 + k >= g.splits) ml[k].x = -INFINITY;
        to = fmaxf(to, ml[k].x);
      }
      if (to == -INFINITY) continue;
      const float keep = fmaxf(__builtin_amdgcn_exp2f(m - to), kLeast);
      l *= keep;
      y *= keep;
      m = to;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        if (ml[k].x == -INFINITY) continue;
        const float e = fmaxf(__builtin_amdgcn_exp2f(ml[k].x - to), kLeast);
        l = fmaf(e, ml[k].y, l);
        y += e * f32x4{a[k].x, a[k].y, b[k].x, b[k].y};
      }
    }
    const int r = tile.r0 + row, token = r / g.group;
    T *o = reinterpret_cast<T *>(static_cast<char *>(g.a.out) +
                                 (tile.q0 + token) * (int64_t)g.a.out_nb[1] +
                                 (head * g.group + (r - token * g.group)) * (int64_t)g.a.out_nb[0]);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      row_put(o[d + k], m == -INFINITY ? 0.0f : y[k] / l);
  }
}

int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

struct Cut {
  int64_t tiles;
  int splits;
};

// Tiles (a bound: the offsets are on the device), and into how many pieces each is cut: until
// there are two blocks a CU, of fp32, where a pass takes the matrix cores sixteen times as long
// and a piece more is cheap beside it, four (3 prompts of 1,277 tokens, 4 heads of 96, window 500:
// 140 -> 132 us); pieces of at least four passes.
Cut cut_of(const PagedShape &p, int q_heads, int n_tokens, int n_seqs, int64_t cap) {
  const int64_t rows = (int64_t)n_tokens * (q_heads / p.n_heads);
  const bool half = p.io != IoType::F32;
  Cut c;
  c.tiles = std::min(rows / kRows + n_seqs, rows);
  const int64_t blocks = c.tiles * p.n_heads, want = (half ? 2 : 4) * (int64_t)p.cus;
  const int64_t most = std::max<int64_t>(1, cap / (half ? 256 : 128));
  c.splits = (int)std::min(most, std::max<int64_t>(1, (want + (half ? 0 : blocks / 2)) / blocks));
  return c;
}

template <typename Launch>
hipError_t over_blocks(Args &g, int64_t blocks, Launch launch) {
  constexpr int64_t kMost = (((int64_t)1 << 32) - 1) / kThreads;
  for (int64_t b = 0; b < blocks; b += kMost) {
    g.first_block = b;
    launch((int)std::min(kMost, blocks - b));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int DP, int DC>
hipError_t launch(Args &g, hipStream_t s) {
  typedef Kind<T, DP> K;
  const bool shaped = g.a.scores.softcap > 0 || g.a.scores.slopes;
  const auto kernel = shaped ? prompt_kernel<T, DP, DC, true> : prompt_kernel<T, DP, DC, false>;
  // the rows twice, or the cosines of a tile's tokens before them
  const int tokens = std::min(kRows, kRows / g.group + 2);
  const int bytes = std::max(2 * K::kBuffer, tokens * g.p.rotary.pairs * (int)sizeof(float2));
  hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return e;
  e = over_blocks(g, g.tiles * g.p.n_heads * g.splits,
                  [&](int blocks) { kernel<<<blocks, kThreads, bytes, s>>>(g); });
  if (e != hipSuccess || g.splits == 1) return e;
  return over_blocks(g, g.tiles * g.p.n_heads * (kRows * DP / 4 / (4 * kThreads)),
                     [&](int blocks) { join_kernel<T, DP><<<blocks, kThreads, 0, s>>>(g); });
}

template <typename T>
hipError_t launch_type(Args &g, hipStream_t s) {
  const int dim = g.p.dim;
  if (dim <= 64) return launch<T, 64, 64>(g, s);
  if (dim <= 96) return launch<T, 128, 96>(g, s);
  if (dim <= 128) return launch<T, 128, 128>(g, s);
  if (dim <= 192) return launch<T, 256, 192>(g, s);
  return launch<T, 256, 256>(g, s);
}

int64_t cap_of(const PagedShape &p, int width) {
  return std::min((int64_t)width * p.page_size, (int64_t)kMaxTokens);
}

}  // namespace

size_t paged_prompt_workspace(const PagedShape &p, int q_heads, int n_tokens, int n_seqs,
                              int table_width) {
  if (n_tokens == 0 || n_seqs == 0) return 0;
  const Cut c = cut_of(p, q_heads, n_tokens, n_seqs, cap_of(p, table_width));
  if (c.splits == 1) return 0;
  return sizeof(float) * c.tiles * p.n_heads * c.splits * kRows * (padded_dim(p.dim) + 2);
}

hipError_t launch_paged_prompt(const PagedShape &p, const PagedSeqs &q, const PagedPrompt &a,
                               void *workspace, hipStream_t s) {
  Args g{};
  g.p = p;
  g.q = q;
  g.a = a;
  g.flip = a.scale < 0;
  const float scale = g.flip ? -a.scale : a.scale;
  g.scale2 = scale * kLog2e;
  if (a.scores.softcap > 0) {
    g.cap_in = scale / a.scores.softcap;
    g.cap2 = a.scores.softcap * kLog2e;
    g.cap_rough = a.scores.softcap <= kRoughCap;
  }
  g.group = a.q_heads / p.n_heads;
  g.cap = cap_of(p, q.width);
  g.page_of = page_of_blocks(p.page_size);
  const int size = p.io == IoType::F32 ? 4 : 2;
  g.row_bytes = p.dim * size;
  g.q_vec = (reinterpret_cast<uintptr_t>(a.q) | a.q_nb[0] | a.q_nb[1]) % 16 == 0;
  g.out_vec = (reinterpret_cast<uintptr_t>(a.out) | a.out_nb[0] | a.out_nb[1]) % (4 * size) == 0;
  const Cut c = cut_of(p, a.q_heads, a.n_tokens, q.n_seqs, g.cap);
  g.tiles = c.tiles;
  g.splits = c.splits;
  g.partial = static_cast<float *>(workspace);
  switch (p.io) {
    case IoType::F32: return launch_type<float>(g, s);
    case IoType::F16: return launch_type<_Float16>(g, s);
    default: return launch_type<Bf16>(g, s);
  }
}

}  // namespace aq
