// paged4_attend.hpp -- attention of one new token per sequence over pages of 4-bit values: what
// the kernel of paged_attend.hpp takes in place of exact rows.
//
// The codes become bf16 in the lanes that loaded them (one conversion a pair of values, with its
// scale; exact, so nothing is lost), and from there on the products are those of bf16 rows:
// queries and weights as three numbers, whatever type the queries come in.  A lane's load of a
// key is 16 bytes, 32 channels under one scale; its load of values 16 bytes too, 4 tokens of 8
// channels (paged4.hpp lays them out for that).  Bound: the bytes, 17/32 a value; with a quarter
// of the exact cache's to load, the conversions and the products of three numbers come near
// them.
#pragma once

#include "paged4.hpp"
#include "paged_attend.hpp"

namespace aq {

namespace {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// 8 channels of codes as 4 pairs of bf16.
__device__ __forceinline__ u32x4 bf16_of(uint32_t codes, float scale) {
  u32x4 y;
  y[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0));
  y[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1));
  y[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2));
  y[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3));
  return y;
}

template <int DP>
struct Kind4 {
  static constexpr bool kHalf = true;
  static constexpr int kUnit = 32;
  static constexpr int kSubs = kUnit / 16;
  static constexpr int kChunks = DP / 32;         // operands of a key's row
  static constexpr int kKVec = DP / 4 < 32 ? DP / 4 : 32;  // channels of a K load
  static constexpr int kKLoads = DP / (4 * kKVec);
  static constexpr int kVVec = DP <= 64 ? 4 : 8;  // channels of a V load, of 4 tokens
  static constexpr int kVChunks = DP / (16 * kVVec);
  static constexpr int kTerms = 3;
};

template <int DP>
struct Rows4 {
  typedef Kind4<DP> K;
  typedef typename VecOf<K::kKVec / 2>::type KLoad;
  typedef typename VecOf<2 * K::kVVec>::type VLoad;
  KLoad k[K::kSubs][K::kKLoads];
  VLoad v[K::kSubs][K::kVChunks];
  uint32_t ks[K::kSubs][K::kKLoads], vs[K::kSubs][K::kVChunks];  // scales: one, of 4 tokens
};

// PACKED: up to 4 query heads.  Of a product's 16 columns the three numbers of a query take a
// column each, (query head, number) in lane head + 4 * number, so that one product does what
// three do otherwise; a score is the sum over its three columns, and so is an output at the end
// (64 sequences x 8 heads of 8,192 tokens, 4 query heads each: 102 us, unpacked 132).
template <int DP_, bool ONCE, bool STEP, bool SHAPED_, bool PACKED>
struct Attend4 {
  typedef Bf16 Product;
  static constexpr int DP = DP_;
  static constexpr bool kStep = STEP, SHAPED = SHAPED_;
  static constexpr int kSpan = SHAPED ? kShaped : kPlain;
  typedef Kind4<DP> K;
  typedef Rows4<DP> Rows;
  typedef aq::Where<K::kSubs> Where;
  static constexpr int kPolicy = ONCE ? 2 : 0;
  static constexpr float kLift = 0.0f;
  static constexpr bool kPacked = PACKED;
  __device__ int query_row() const { return PACKED ? row16 & 3 : row16; }

  const Args &g;
  const int lane, row16, group4;
  int k_off[K::kKLoads], ks_off[K::kKLoads], v_off[K::kVChunks], vs_off[K::kVChunks];
  typename SpanOf<kSpan>::type span;
  const int *table;
  int head, u_end;
  float slope2 = 0.0f;
  float *score_row = nullptr;
  int64_t query_at = 0;
  u32x4 qh[K::kChunks];
  const u32x4 *q_low;
  float qf[1];
  int q_shift = 0;

  __device__ Attend4(const Args &args, int lane_, const u32x4 *low)
      : g(args), lane(lane_), row16(lane_ & 15), group4(lane_ >> 4), q_low(low + lane_) {
    const int dim = g.p.dim, blocks = dim / kBlock4;
#pragma unroll
    for (int i = 0; i < K::kKLoads; ++i) {  // channels past dim lie beyond every buffer
      const int d = k_channel(i * (K::kKVec / 8));
      k_off[i] = d < dim ? row16 * (dim / 2) + d / 2 : kBeyond;
      ks_off[i] = d < dim ? 8 * dim + row16 * blocks + d / kBlock4 : kBeyond;
    }
#pragma unroll
    for (int c = 0; c < K::kVChunks; ++c) {
      const int d = K::kVVec * (row16 + 16 * c);
      v_off[c] = d < dim ? (group4 * (dim / K::kVVec) + row16 + 16 * c) * 2 * K::kVVec : kBeyond;
      vs_off[c] = d < dim ? 8 * dim + (group4 * blocks + d / kBlock4) * 4 : kBeyond;
    }
  }

  __device__ float query(const char *row, int d) const { return io_load(row, d, g.p.io); }
  __device__ float turned(float x) const { return x; }
  __device__ void output(char *row, int d, f32x4 y) const {
#pragma unroll
    for (int i = 0; i < 4; ++i) io_store(row, d + i, g.p.io, y[i]);
  }

  __device__ int k_channel(int chunk) const {  // first of the 8 channels of an operand
    constexpr int per = K::kKVec / 8;
    return chunk / per * 4 * K::kKVec + K::kKVec * group4 + 8 * (chunk % per);
  }

  __device__ Where locate(int unit) const {
    Where w;
#pragma unroll
    for (int s = 0; s < K::kSubs; ++s) {
      const int b = span.real(unit) * K::kSubs + s;
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

  // A block of 16 tokens as a buffer, empty where there is no page.
  __device__ __amdgpu_buffer_rsrc_t block16(const void *pool, const Where &w, int s) const {
    const char *at = static_cast<const char *>(pool) + block4_at(g.p, max(w.page[s], 0), head, w.slot[s]);
    return __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char *>(at), 0,
        __builtin_amdgcn_readfirstlane(w.page[s] < 0 ? 0 : block4_bytes(g.p.dim)), 0x00020000);
  }

  __device__ void append(int seq, int at) const {
    const int col = page_column(g.page_of, at >> 4);
    const int page = ((cint *)(uint64_t)table)[col];
    if (page < 0 || page >= g.p.n_pages) return;
    const int slot = at - col * g.p.page_size, chunk = lane & 31;
    const bool value = lane >= 32;
    if (chunk >= g.p.dim / 8) return;  // (whole groups of four lanes)
    const char *row = value ? static_cast<const char *>(g.n.v) + seq * (int64_t)g.n.v_nb[1] +
                                  head * (int64_t)g.n.v_nb[0]
                            : static_cast<const char *>(g.n.k) + seq * (int64_t)g.n.k_nb[1] +
                                  head * (int64_t)g.n.k_nb[0];
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = io_load(row, 8 * chunk + i, g.p.io);
    const RotaryTable &rt = g.p.rotary;
    if (!value && rt.pairs)
      rotate8(x, row, chunk, g.p.io, rt,
              [&](int pair) { return rotary_cos_sin(rt.steps[pair], at, rt.amplitude); });
    int byte;
    const uint32_t codes = encode4(x, &byte);
    store4(static_cast<char *>(value ? g.p.v_pages : g.p.k_pages) + block4_at(g.p, page, head, slot),
           slot & 15, chunk, codes, byte, value, g.p.dim);
  }

  __device__ void load(Rows &r, const Where &w, int) const {
#pragma unroll
    for (int s = 0; s < K::kSubs; ++s) {
      const auto k = block16(g.p.k_pages, w, s);
#pragma unroll
      for (int i = 0; i < K::kKLoads; ++i) {
        if constexpr (K::kKVec == 16)
          r.k[s][i] = __builtin_amdgcn_raw_buffer_load_b64(k, k_off[i], 0, kPolicy);
        else
          r.k[s][i] = __builtin_amdgcn_raw_buffer_load_b128(k, k_off[i], 0, kPolicy);
        r.ks[s][i] = __builtin_amdgcn_raw_buffer_load_b8(k, ks_off[i], 0, kPolicy);
      }
      const auto v = block16(g.p.v_pages, w, s);
#pragma unroll
      for (int c = 0; c < K::kVChunks; ++c) {
        if constexpr (K::kVVec == 4)
          r.v[s][c] = __builtin_amdgcn_raw_buffer_load_b64(v, v_off[c], 0, kPolicy);
        else
          r.v[s][c] = __builtin_amdgcn_raw_buffer_load_b128(v, v_off[c], 0, kPolicy);
        r.vs[s][c] = __builtin_amdgcn_raw_buffer_load_b32(v, vs_off[c], 0, kPolicy);
      }
    }
  }

  __device__ void use(State<DP> &st, Rows &r, const Where &w, int unit) const {
    const int t0 = span.real(unit) * K::kUnit;
    bool full = span.all_seen(t0, t0 + K::kUnit), any = false;
#pragma unroll
    for (int s = 0; s < K::kSubs; ++s) {
      full = full && w.page[s] >= 0;
      any = any || (w.page[s] >= 0 && span.any_seen(t0 + 16 * s, t0 + 16 * s + 16));
    }
    if (!any) return;  // (uniform)

    f32x4 s[K::kSubs];
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i) s[i] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int c = 0; c < K::kChunks; ++c) {
      constexpr int per = K::kKVec / 8;
      u32x4 q1, q2;
      if constexpr (!PACKED) {
        q1 = q_low[64 * c];
        q2 = q_low[64 * (K::kChunks + c)];
      }
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i) {
        const u32x4 k = bf16_of(r.k[i][c / per][c % per], scale4(r.ks[i][c / per]));
        s[i] = mfma(k, qh[c], s[i], Bf16());
        if constexpr (!PACKED) {
          s[i] = mfma(k, q1, s[i], Bf16());
          s[i] = mfma(k, q2, s[i], Bf16());
        }
      }
    }
    if constexpr (PACKED)
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][j] = packed_sum(s[i][j]);
    const float scale2 = SHAPED && g.sc.softcap > 0.0f ? g.cap_in : g.scale2;
#pragma unroll
    for (int i = 0; i < K::kSubs; ++i) s[i] *= scale2;
    if constexpr (SHAPED) shape_scores(g, s, slope2, (float)(query_at - (t0 + 4 * group4)));
    if (!full) {
#pragma unroll
      for (int i = 0; i < K::kSubs; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int t = t0 + 16 * i + 4 * group4 + j;
          if (w.page[i] >= 0 && span.sees(t)) continue;
          s[i][j] = -INFINITY;
          // what is there is no value of this query's: zeros in its place
#pragma unroll
          for (int c = 0; c < K::kVChunks; ++c) {
            if constexpr (K::kVVec == 8)
              r.v[i][c][j] = 0;
            else
              r.v[i][c][j / 2] &= j % 2 ? 0x0000FFFFu : 0xFFFF0000u;
            r.vs[i][c] = (r.vs[i][c] & ~(255u << (8 * j))) | 127u << (8 * j);
          }
        }
    }
    if constexpr (SHAPED) keep_scores<K::kSubs>(score_row, s, w.page, t0 + 4 * group4);
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
#pragma unroll
    for (int u = 0; u < K::kSubs / 2; ++u) {  // 32 tokens a product
      float p[8];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[4 * i + j] = __builtin_amdgcn_exp2f(s[2 * u + i][j] - top);
          st.l += p[4 * i + j];
        }
      u32x4 pt[3];
      if constexpr (PACKED) {
        const int term = row16 >> 2;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float rest = p[i] - __uint_as_float(__float_as_uint(p[i]) & 0xFFFF0000u);
          const float last = rest - __uint_as_float(__float_as_uint(rest) & 0xFFFF0000u);
          p[i] = term == 0 ? p[i] : term == 1 ? rest : term == 2 ? last : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pt[0][i] = __builtin_amdgcn_perm(__float_as_uint(p[2 * i + 1]), __float_as_uint(p[2 * i]),
                                           0x07060302u);
      } else {
        split8<Bf16>(p, pt);
      }
#pragma unroll
      for (int c = 0; c < K::kVChunks; ++c) {
        u32x4 x[8];  // of each token, its channels
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const auto &v = r.v[2 * u + i][c];
            const uint32_t four = r.vs[2 * u + i][c];
            // (byte j to the exponent's place)
            const float scale = __uint_as_float(j == 3 ? four >> 1 : four << (23 - 8 * j));
            if constexpr (K::kVVec == 8) {
              x[4 * i + j] = bf16_of(v[j], scale);
            } else {  // two tokens a word
              const u32x4 y = bf16_of(v[j / 2], scale);
              x[4 * i + j][0] = y[j % 2 * 2];
              x[4 * i + j][1] = y[j % 2 * 2 + 1];
            }
          }
#pragma unroll
        for (int w2 = 0; w2 < K::kVVec / 2; ++w2) {
          u32x4 a, b;  // the 8 tokens of channels 2 w2 and 2 w2 + 1
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            a[k] = __builtin_amdgcn_perm(x[2 * k + 1][w2], x[2 * k][w2], 0x05040100u);
            b[k] = __builtin_amdgcn_perm(x[2 * k + 1][w2], x[2 * k][w2], 0x07060302u);
          }
          f32x4 &y = st.acc[c * K::kVVec + 2 * w2], &z = st.acc[c * K::kVVec + 2 * w2 + 1];
#pragma unroll
          for (int t = 0; t < (PACKED ? 1 : 3); ++t) {
            y = mfma(a, pt[t], y, Bf16());
            z = mfma(b, pt[t], z, Bf16());
          }
        }
      }
    }
  }
};

template <int DP, bool STEP, bool SHAPED>
hipError_t launch4_rows(const Args &g, hipStream_t s) {
  if (g.group <= 4) {  // (one tile of query heads: rows are read once)
    const auto kernel = attend_kernel<Attend4<DP, true, STEP, SHAPED, true>>;
    return launch_attend<DP, Kind4<DP>::kUnit>(g, kernel, kernel, s);
  }
  return launch_attend<DP, Kind4<DP>::kUnit>(
      g, attend_kernel<Attend4<DP, true, STEP, SHAPED, false>>,
      attend_kernel<Attend4<DP, false, STEP, SHAPED, false>>, s);
}

template <int DP, bool SHAPED>
hipError_t launch4(const Args &g, hipStream_t s) {
  return g.n.k ? launch4_rows<DP, true, SHAPED>(g, s) : launch4_rows<DP, false, SHAPED>(g, s);
}

template <bool SHAPED>
hipError_t launch4_dim(const Args &g, hipStream_t s) {
  switch (padded_dim(g.p.dim)) {
    case 64: return launch4<64, SHAPED>(g, s);
    case 128: return launch4<128, SHAPED>(g, s);
    default: return launch4<256, SHAPED>(g, s);
  }
}

}  // namespace

}  // namespace aq
