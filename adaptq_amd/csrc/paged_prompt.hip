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
// * Values are transposed on their way into LDS: a lane loads 4 tokens of up to 8 channels
//   and writes each channel's 4 tokens together.  Addresses are turned by the channel so
//   that neither side meets in a bank.
// * The next tokens' rows are loaded into registers while these are used, and go into the
//   other half of LDS after: one barrier a pass.
// * Tiles of few queries over many tokens are cut over the tokens, and joined by a second
//   launch.
//
// Rows of half types: products of their values are exact and summed in fp32; rotated queries
// are rounded to the type, as Rotary's are; weights are rounded to it, by up to 2^-9 (bf16)
// and 2^-12 (fp16) of each on the average, independently, where the output itself rounds by
// as much once: their mean over the tokens adds less than that (1.4 times the error of one
// rounding in all; a second number for the weights' rest would cost half as much again on
// the matrix cores).  Their sum takes them unrounded.  fp32 rows use the fp32 matrix
// instructions.
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
constexpr int kRows = 128;  // of a tile
constexpr int kBeyond = 1 << 30;
// A maximum is followed only when it grows by more than this (in powers of two): weights
// are then up to 2^8 of what they would be, which no sum or type minds, and most passes
// leave the sums as they are.
constexpr float kLazy = 8.0f;

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

template <typename T, int DP>
struct Kind {
  static constexpr bool kHalf = sizeof(T) == 2;
  static constexpr int kKeys = kHalf ? 64 : 32;     // tokens of a pass
  static constexpr int kSubs = kKeys / 32;
  static constexpr int kVec = 16 / (int)sizeof(T);  // values of 16 bytes
  static constexpr int kBlocks = kKeys / 16;        // blocks of 16 tokens, which lie together
  // K: 16 bytes a lane and pass of the threads
  static constexpr int kRowLoads = DP / kVec;
  static constexpr int kKPasses = kKeys * kRowLoads / kThreads;
  static constexpr int kKStride = DP * sizeof(T) + 16;
  // V, half types: 4 tokens of kVVec channels a lane
  static constexpr int kVVec = DP / 16 < 8 ? DP / 16 : 8;
  static constexpr int kVPasses = kHalf ? DP / (16 * kVVec) : kKPasses;
  static constexpr int kVBytes = kHalf ? DP * kKeys * 2 : kKeys * (DP + 8) * 4;
  static constexpr int kBuffer = kKeys * kKStride + kVBytes;
  static constexpr int kQ = kHalf ? DP / 16 : DP / 2;  // operand registers of the queries
  static constexpr int kResident = DP == 256 ? 1 : 2;
};

template <int BYTES>
struct VecOf {
  typedef u32x4 type;
};
template <>
struct VecOf<8> {
  typedef u32x2 type;
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

template <typename T, int DP, bool EXACT, bool SHAPED>
__global__ __launch_bounds__(kThreads, (Kind<T, DP>::kResident)) void prompt_kernel(const Args g) {
  typedef Kind<T, DP> K;
  extern __shared__ __align__(16) char lds[];
  __shared__ int s_red[kWaves][8];
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
  const int red[6] = {wave_min(pre ? see.a : INT_MAX), wave_max(pre ? see.pe : 0),
                      wave_min(see.w), wave_e, wave_max(live ? see.w : 0),
                      wave_min(live ? see.e : INT_MAX)};
  if (lane < 6) {
    int x = red[0];
#pragma unroll
    for (int i = 1; i < 6; ++i) x = lane == i ? red[i] : x;
    s_red[wave][lane] = x;
  }
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

  // the passes: units of kKeys tokens, in one run or two
  int u_first = w / K::kKeys, u_end = (e + K::kKeys - 1) / K::kKeys, gap_at = INT_MAX, gap = 0;
  if (w >= e) u_first = u_end = 0;
  if (lo < pe) {
    const int p0 = lo / K::kKeys, p1 = (pe + K::kKeys - 1) / K::kKeys;
    if (u_first >= u_end) {
      u_first = p0;
      u_end = p1;
    } else {
      if (u_first > p1) {
        gap_at = p1;
        gap = u_first - p1;
      }
      u_end = max(u_end, p1) - gap;
      u_first = min(p0, u_first);
    }
  }
  const int units = u_end - u_first;
  const int i0 = (int)((int64_t)units * split / g.splits),
            i1 = (int)((int64_t)units * (split + 1) / g.splits);

  // where this thread's parts of the rows lie
  const int *table = g.q.table + (int64_t)tile.seq * g.q.stride;
  const int k_row = tid / K::kRowLoads, k_chunk = tid % K::kRowLoads;
  constexpr int kKRowsAPass = kThreads / K::kRowLoads;
  const int v_chunk = tid & 15, v_quad = tid >> 4;
  typedef typename VecOf<K::kVVec * sizeof(T)>::type VLoad;
  u32x4 k_in[K::kKPasses], v_in4[K::kHalf ? 1 : K::kVPasses];
  VLoad v_in[K::kHalf ? K::kVPasses : 1][4];

  struct Where {
    int page[K::kBlocks], slot[K::kBlocks];
  };
  const auto real = [&](int i) {  // unit of pass i
    const int u = u_first + i;
    return u >= gap_at ? u + gap : u;
  };
  const auto locate = [&](int i) {
    Where x;
    const int u = real(i);
#pragma unroll
    for (int k = 0; k < K::kBlocks; ++k) {
      const int b = u * K::kBlocks + k;
      x.page[k] = -1;
      x.slot[k] = 0;
      if (i < i1 && b * 16 < n) {
        const int c = page_column(g.page_of, b);
        const int page = ((cint *)(uint64_t)table)[c];
        x.page[k] = page < g.p.n_pages ? page : -1;
        x.slot[k] = (b - c * g.page_of.blocks) * 16;
      }
    }
    return x;
  };
  // 16 tokens' rows as a buffer that ends behind the last one and is empty without a page
  const auto rows16 = [&](const void *pool, const Where &x, int k, int t0) {
    const int64_t page = max(x.page[k], 0);
    const char *from = static_cast<const char *>(pool) +
                       ((page * heads + head) * g.p.page_size + x.slot[k]) * g.row_bytes;
    const int rows = x.page[k] < 0 ? 0 : max(0, min(16, n - (t0 + 16 * k)));
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(from), 0,
                                             __builtin_amdgcn_readfirstlane(rows * g.row_bytes),
                                             0x00020000);
  };
  const auto pick = [&](const Where &x, int k) {  // block k, the same for the whole wave
    Where y;
    y.page[0] = x.page[0];
    y.slot[0] = x.slot[0];
#pragma unroll
    for (int j = 1; j < K::kBlocks; ++j) {
      y.page[0] = k == j ? x.page[j] : y.page[0];
      y.slot[0] = k == j ? x.slot[j] : y.slot[0];
    }
    return y;
  };
  const auto load = [&](const Where &x, int i) {
    const int t0 = real(i) * K::kKeys;
#pragma unroll
    for (int p = 0; p < K::kKPasses; ++p) {
      const int blk = __builtin_amdgcn_readfirstlane((p * kKRowsAPass + k_row) >> 4);
      const auto from = rows16(g.p.k_pages, pick(x, blk), 0, t0 + 16 * blk);
      const int in = (p * kKRowsAPass + k_row) & 15, c = k_chunk * K::kVec;
      k_in[p] = __builtin_amdgcn_raw_buffer_load_b128(
          from, EXACT || c < dim ? in * g.row_bytes + c * (int)sizeof(T) : kBeyond, 0, 0);
      if constexpr (!K::kHalf) {
        const auto vfrom = rows16(g.p.v_pages, pick(x, blk), 0, t0 + 16 * blk);
        v_in4[p] = __builtin_amdgcn_raw_buffer_load_b128(
            vfrom, EXACT || c < dim ? in * g.row_bytes + c * (int)sizeof(T) : kBeyond, 0, 0);
      }
    }
    if constexpr (K::kHalf) {
      // the wave's 16 tokens are one block
      const auto from = rows16(g.p.v_pages, pick(x, wave), 0, t0 + 16 * wave);
#pragma unroll
      for (int p = 0; p < K::kVPasses; ++p) {
        const int c = (v_chunk + 16 * p) * K::kVVec;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int off = EXACT || c < dim
                              ? ((v_quad & 3) * 4 + j) * g.row_bytes + c * (int)sizeof(T)
                              : kBeyond;
          if constexpr (K::kVVec == 4)
            v_in[p][j] = __builtin_amdgcn_raw_buffer_load_b64(from, off, 0, 0);
          else
            v_in[p][j] = __builtin_amdgcn_raw_buffer_load_b128(from, off, 0, 0);
        }
      }
    }
  };
  const auto store = [&](char *to) {
    char *v_to = to + K::kKeys * K::kKStride;
#pragma unroll
    for (int p = 0; p < K::kKPasses; ++p) {
      *reinterpret_cast<u32x4 *>(to + (p * kKRowsAPass + k_row) * K::kKStride + k_chunk * 16) =
          k_in[p];
      if constexpr (!K::kHalf)
        *reinterpret_cast<u32x4 *>(v_to + ((p * kKRowsAPass + k_row) * (DP + 8) + k_chunk * 4) * 4) =
            v_in4[p];
    }
    if constexpr (K::kHalf) {
      const int unit = v_quad / 4 * 2 + (v_quad & 1), part = (v_quad >> 1) & 1;
#pragma unroll
      for (int p = 0; p < K::kVPasses; ++p)
#pragma unroll
        for (int i = 0; i < K::kVVec; ++i) {
          const uint32_t sel = i & 1 ? 0x07060302u : 0x05040100u;
          u32x2 x;
          x[0] = __builtin_amdgcn_perm(v_in[p][1][i / 2], v_in[p][0][i / 2], sel);
          x[1] = __builtin_amdgcn_perm(v_in[p][3][i / 2], v_in[p][2][i / 2], sel);
          const int ch = (v_chunk + 16 * p) * K::kVVec + i;
          *reinterpret_cast<u32x2 *>(v_to + ch * 128 + ((unit ^ ((ch ^ (ch >> 3)) & 7)) << 4) +
                                     part * 8) = x;
        }
    }
  };

  Where here = locate(i0), next = locate(i0 + 1);
  if (i0 < i1) load(here, i0);

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
      s_cs[i] = rotary_cos_sin(rt.steps[i - t * rt.pairs], length - tile.count + token0 + t,
                               rt.amplitude);
    }
    __syncthreads();
  }
  u32x4 qh[K::kHalf ? K::kQ : 1];
  float qf[K::kHalf ? 1 : K::kQ];
  {
    const float2 *cs = s_cs + (token - token0) * rt.pairs;
    constexpr int N = K::kVec, kStep = 2 * N;
#pragma unroll
    for (int c = 0; c < DP / kStep; ++c) {
      const int d0 = kStep * c + N * half;
      RowVec<T, N> x;
      if (g.q_vec && d0 + N <= dim) {
        x = load_rows<false, T, N>(q_row + d0);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (d0 + i < dim) x.x[i] = q_row[d0 + i];
          else row_put(x.x[i], 0.0f);
      }
      if (d0 < 2 * rt.pairs) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int d = d0 + i;
          if (d >= 2 * rt.pairs) break;
          const bool one = rt.interleaved ? !(d & 1) : d < rt.pairs;
          const int pair = rt.interleaved ? d >> 1 : one ? d : d - rt.pairs;
          const int other = rt.interleaved ? d ^ 1 : one ? d + rt.pairs : d - rt.pairs;
          const float u = row_get(x.x[i]), v = row_get(q_row[other]);
          const float2 a = cs[pair];
          row_put(x.x[i], one ? fmaf(u, a.x, -(v * a.y)) : fmaf(u, a.x, v * a.y));
        }
      }
      if constexpr (K::kHalf) {
        qh[c] = __builtin_bit_cast(u32x4, x);
        if (g.flip) qh[c] ^= 0x80008000u;
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) qf[N * c + i] = g.flip ? -row_get(x.x[i]) : row_get(x.x[i]);
      }
    }
  }
  float slope2 = 0.0f;
  if (SHAPED && g.a.scores.slopes) slope2 = g.a.scores.slopes[q_head] * kLog2e;
  if (rt.pairs) __syncthreads();  // the cosines are read: LDS is the rows' now

  f32x16 acc[DP / 32];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = f32x16{0};

  const auto use = [&](const char *buf, const Where &x, int t0) {
    const char *v_at = buf + K::kKeys * K::kKStride;
    f32x16 s[K::kSubs];
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i) s[i] = f32x16{0};
    if constexpr (K::kHalf) {
#pragma unroll
      for (int c = 0; c < DP / 16; ++c)
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i) {
          const u32x4 k = *reinterpret_cast<const u32x4 *>(buf + (32 * i + col) * K::kKStride +
                                                           32 * c + 16 * half);
          s[i] = mfma(k, qh[c], s[i], T());
        }
    } else {
#pragma unroll
      for (int c = 0; c < DP / 8; ++c) {
        const f32x4 k =
            *reinterpret_cast<const f32x4 *>(buf + col * K::kKStride + 32 * c + 16 * half);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          s[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(k[i], qf[4 * c + i], s[0], 0, 0, 0);
      }
    }
    bool full = t0 >= w_all && t0 + K::kKeys <= e_all;
#pragma unroll
    for (int k = 0; k < K::kBlocks; ++k) full = full && x.page[k] >= 0;
    const int t1 = t0 + 4 * half;
    float scale2 = g.scale2;
    if constexpr (SHAPED) {
      const PagedScores &sc = g.a.scores;
      const float cap_in = g.cap_in, cap2 = g.cap2;
      if (sc.softcap > 0.0f) {
#pragma unroll
        for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
          for (int j = 0; j < 16; ++j) s[i][j] = cap2 * tanh_of<!K::kHalf>(s[i][j] * cap_in);
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
      bool any = false;
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const int t = t1 + 32 * i + 8 * (j / 4) + j % 4;
          const bool there = x.page[2 * i + j / 8] >= 0 &&
                             ((t >= see.w && t < see.e) || (t >= see.a && t < see.pe));
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
    if (__any(top > m + kLazy)) {  // (m is minus infinity at first)
      const float to = fmaxf(m, top), keep = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - to);
      l *= keep;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] *= keep;
      m = to;
    }
    const float from = fmaxf(m, -FLT_MAX);
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
        u32x4 p;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          p[j] = pack2(s[k / 2][8 * (k % 2) + 2 * j], s[k / 2][8 * (k % 2) + 2 * j + 1], T());
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const int ch = 32 * i + col;
          const u32x4 v = *reinterpret_cast<const u32x4 *>(
              v_at + ch * 128 + (((2 * k + half) ^ ((ch ^ (ch >> 3)) & 7)) << 4));
          acc[i] = mfma(v, p, acc[i], T());
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j)
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const float v = *reinterpret_cast<const float *>(
              v_at + ((8 * (j / 4) + 4 * half + j % 4) * (DP + 8) + 32 * i + col) * 4);
          acc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(v, s[0][j], acc[i], 0, 0, 0);
        }
    }
  };

  if (i0 < i1) store(lds);
  __syncthreads();
  for (int i = i0; i < i1; ++i) {
    const Where after = locate(i + 2);
    if (i + 1 < i1) load(next, i + 1);
    const int t0 = real(i) * K::kKeys;
    if (t0 < wave_e && t0 + K::kKeys > wave_lo) use(lds + ((i - i0) & 1) * K::kBuffer, here, t0);
    if (i + 1 < i1) store(lds + ((i - i0 + 1) & 1) * K::kBuffer);
    __syncthreads();
    here = next;
    next = after;
  }

  l = half_sum(l);
  if (!live) return;
  if (g.splits > 1) {
    float *part = g.partial + (((index * heads + head) * g.splits + split) * kRows + row) * (DP + 2);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i)
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
  for (int i = 0; i < DP / 32; ++i)
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      const int d = 32 * i + 2 * j + 4 * half;
      if (!EXACT && d >= dim) continue;
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
    for (int k = 0; k < g.splits; ++k, part += (int64_t)kRows * (DP + 2)) {
      const float2 ml = *reinterpret_cast<const float2 *>(part + DP);
      if (ml.x == -INFINITY) continue;
      const float2 a = *reinterpret_cast<const float2 *>(part + d);
      const float2 b = *reinterpret_cast<const float2 *>(part + d + 2);
      const float to = fmaxf(m, ml.x);
      const float keep = __builtin_amdgcn_exp2f(m - to), e = __builtin_amdgcn_exp2f(ml.x - to);
      l = fmaf(l, keep, e * ml.y);
      y = y * keep + e * f32x4{a.x, a.y, b.x, b.y};
      m = to;
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

// Tiles (a bound: the offsets are on the device), and into how many pieces each is cut.
Cut cut_of(const PagedShape &p, int q_heads, int n_tokens, int n_seqs, int64_t cap) {
  const int group = q_heads / p.n_heads;
  Cut c;
  c.tiles = std::min((int64_t)n_tokens * group / kRows + n_seqs, (int64_t)n_tokens * group);
  const int64_t blocks = c.tiles * p.n_heads, want = 2 * p.cus;
  const int64_t most = std::max<int64_t>(1, cap / 256);
  c.splits = (int)std::min(most, std::max<int64_t>(1, want / blocks));
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

template <typename T, int DP>
hipError_t launch(Args &g, hipStream_t s) {
  typedef Kind<T, DP> K;
  const bool shaped = g.a.scores.softcap > 0 || g.a.scores.slopes, exact = g.p.dim == DP;
  const auto kernel = exact ? (shaped ? prompt_kernel<T, DP, true, true>
                                      : prompt_kernel<T, DP, true, false>)
                            : (shaped ? prompt_kernel<T, DP, false, true>
                                      : prompt_kernel<T, DP, false, false>);
  // the rows twice, or the cosines of a tile's tokens before them
  const int group = g.group, tokens = std::min(kRows, kRows / group + 2);
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
  switch (padded_dim(g.p.dim)) {
    case 64: return launch<T, 64>(g, s);
    case 128: return launch<T, 128>(g, s);
    default: return launch<T, 256>(g, s);
  }
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
