// paged_evict.hip -- eviction by accumulated weight: which tokens of a (sequence, key head)
// stay, and their rows to the front of its pages or into other pages.
//
// Two launches.  select_kernel finds, per (sequence, key head), the smallest weight that stays
// by its bits from the highest on (a count of each digit's values, three times), and
// writes the indexes that stay in their order.  move_kernel copies rows by that list.  Bound:
// the rows that stay, read and written once, and the weights.
#include <algorithm>

#include "paged.hpp"
#include "paged_split.hpp"

namespace aq {

namespace {

constexpr int kSelect = 1024;
constexpr int kSelectWaves = kSelect / 64;
constexpr int kBatch = 16;  // weights that a thread has under way
constexpr uint32_t kZero = 0x80000000u;  // the key of a weight of 0
constexpr int kHeld = 1 << 15;  // keys in LDS: 128 KB
// Digits of 11, 11 and 10 bits: the first holds sign, exponent and two bits more, so that even
// weights of like size spread over many counters (a counter takes one lane at a time).
constexpr int kBins = 1 << 11;
constexpr int kMove = 256;
constexpr int kInFlight = 8;  // rows of 16 bytes that a thread has under way

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct Args {
  PagedShape p;
  PagedSeqs q;
  PagedEvict e;
  int64_t cap;
  int row_bytes;
  int slices;     // in place: parts of a row that a block takes, keys and values apart
  int chunks;     // into other pages: blocks of a (sequence, key head)
  int held;       // keys that LDS holds
  int64_t first_block;
};

// Weights in the order of their bits: larger weights have larger keys, both zeros the same one.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// 32 neighbouring digits, which one lane adds up, 64 counters apart.
__device__ __forceinline__ int counter_of(int digit) { return (digit & 31) << 6 | digit >> 5; }

__device__ __forceinline__ int tokens_of(const Args &g, int seq) {
  const int64_t n = max(g.q.lengths[seq], 0);
  return (int)min(n, g.cap);
}

__global__ __launch_bounds__(kSelect) void select_kernel(const Args g) {
  extern __shared__ __align__(16) uint32_t s_key[];
  __shared__ int s_count[kBins];  // of digit d at counter_of(d)
  __shared__ int s_gt[kSelectWaves], s_eq[kSelectWaves];
  __shared__ uint32_t s_digit;
  __shared__ int s_above;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t block = g.first_block + blockIdx.x;
  const int head = (int)(block % g.p.n_heads), seq = (int)(block / g.p.n_heads);
  const int n = tokens_of(g, seq), keep = g.e.keep;
  int *kept = g.e.kept + block * keep;
  if (n <= keep) {
    for (int j = tid; j < keep; j += kSelect) kept[j] = j < n ? j : -1;
    return;
  }
  const float *w = g.e.weights + seq * g.e.nb[1] + head * g.e.nb[0];
  const int old = n - g.e.recent;  // tokens before the newest, which stay
  int room = keep - g.e.recent;    // of those, so many stay
  // the keys of the first kHeld tokens stay in LDS, the others' are read again
  const int held = min(old, g.held);
  for (int t0 = 0; room > 0 && t0 < held; t0 += kBatch * kSelect) {
    float x[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) x[j] = w[min(t0 + j * kSelect + tid, held - 1)];
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (t0 + j * kSelect + tid < held) s_key[t0 + j * kSelect + tid] = key_of(x[j]);
  }
  // the key of the last one that stays, digit by digit; `room` becomes how many of that key
  uint32_t prefix = 0;
  for (int top = 32; room > 0 && top > 0;) {
    const int shift = max(top - 11, 0), bins = 1 << (top - shift);
    const uint32_t beyond = top == 32 ? 0 : 1u << top;
    for (int i = tid; i < kBins; i += kSelect) s_count[i] = 0;
    __syncthreads();
    const auto count = [&](uint32_t key, bool there) {
      there = there && ((key ^ prefix) < beyond || beyond == 0);
      // tokens without any weight are many, and counted together
      const bool zero = there && key == kZero;
      const uint64_t zeros = __ballot(zero);
      if (zeros && lane == 0)
        atomicAdd(&s_count[counter_of(kZero >> shift & (bins - 1))], __popcll(zeros));
      if (there && !zero) atomicAdd(&s_count[counter_of(key >> shift & (bins - 1))], 1);
    };
    for (int t0 = 0; t0 < held; t0 += 4 * kSelect) {
      const int t = t0 + 4 * tid;  // (LDS has room for whole fours)
      const u32x4 key = *reinterpret_cast<const u32x4 *>(s_key + min(t, g.held - 4));
#pragma unroll
      for (int j = 0; j < 4; ++j) count(key[j], t + j < held);
    }
    for (int t0 = held; t0 < old; t0 += kBatch * kSelect) {
      float x[kBatch];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) x[j] = w[min(t0 + j * kSelect + tid, old - 1)];
#pragma unroll
      for (int j = 0; j < kBatch; ++j) count(key_of(x[j]), t0 + j * kSelect + tid < old);
    }
    __syncthreads();
    if (wave == 0) {  // the digit at which `room` values from the top are reached
      constexpr int kEach = kBins / 64;
      const int first = kBins - 1 - kEach * lane;  // from the largest digit on
      int c[kEach], sum = 0;
#pragma unroll
      for (int i = 0; i < kEach; ++i) c[i] = s_count[counter_of(first - i)];
#pragma unroll
      for (int i = 0; i < kEach; ++i) sum += c[i];
      int end = sum;
#pragma unroll
      for (int k = 1; k < 64; k <<= 1) {
        const int y = __shfl_up(end, k, 64);
        if (lane >= k) end += y;
      }
      int above = end - sum;
      if (above < room && end >= room) {
        int digit = 0, before = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
          if (above < room) {  // (the last time that this holds, above + c[i] is enough)
            digit = first - i;
            before = above;
          }
          above += c[i];
        }
        s_digit = digit;
        s_above = before;
      }
    }
    __syncthreads();
    prefix |= s_digit << shift;
    room -= s_above;
    top = shift;
    __syncthreads();
  }
  // each wave's run of the older tokens: how many stay, and of those with the last key the first
  // `room`; then the indexes in order
  const int per = ((old + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
  const int t0 = min(wave * per, old), t1 = min(t0 + per, old);
  const bool none = keep == g.e.recent;
  int gt = 0, eq = 0;
  // of 4 x 64 tokens from u0 on the lane's, 64 apart
  const auto keys_at = [&](int u0, uint32_t (&key)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = min(u0 + 64 * j + lane, t1 - 1);
      key[j] = u0 + 256 <= held ? s_key[t] : t < held ? s_key[t] : key_of(w[t]);
    }
  };
  for (int u0 = t0; !none && u0 < t1; u0 += 256) {
    uint32_t key[4];
    keys_at(u0, key);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = u0 + 64 * j + lane < t1;
      gt += __popcll(__ballot(in && key[j] > prefix));
      eq += __popcll(__ballot(in && key[j] == prefix));
    }
  }
  if (lane == 0) {
    s_gt[wave] = gt;
    s_eq[wave] = eq;
  }
  __syncthreads();
  int at = 0, ties = 0;
  for (int k = 0; k < wave; ++k) {
    at += s_gt[k] + min(s_eq[k], max(room - ties, 0));
    ties += s_eq[k];
  }
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int u0 = t0; !none && u0 < t1; u0 += 256) {
    uint32_t key[4];
    keys_at(u0, key);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = u0 + 64 * j + lane;
      const bool tie = t < t1 && key[j] == prefix;
      const uint64_t tied = __ballot(tie);
      const bool stays =
          (t < t1 && key[j] > prefix) || (tie && ties + __popcll(tied & below) < room);
      const uint64_t all = __ballot(stays);
      if (stays) kept[at + __popcll(all & below)] = t;
      at += __popcll(all);
      ties += __popcll(tied);
    }
  }
  for (int j = tid; j < g.e.recent; j += kSelect) kept[keep - g.e.recent + j] = old + j;
}

// Where token t of a sequence lies: row in the pages, or -1.
__device__ __forceinline__ int64_t row_of(const Args &g, const int *table, int width, int head,
                                          int t) {
  const int col = t / g.p.page_size;
  if (col >= width) return -1;
  const int page = table[col];
  if (page < 0 || page >= g.p.n_pages) return -1;
  return ((int64_t)page * g.p.n_heads + head) * g.p.page_size + (t - col * g.p.page_size);
}

// A sequence's weights after its rows: those that stay to the front, zeros behind.  In place and
// in order, as in move_kernel.
__device__ __forceinline__ void move_weights(const Args &g, float *w, const int *kept, int n,
                                             int tid) {
  const int keep = g.e.keep;
  for (int j0 = 0; j0 < keep; j0 += kInFlight * kMove) {
    float x[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int j = j0 + i * kMove + tid;
      if (j < keep) x[i] = w[kept[j]];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int j = j0 + i * kMove + tid;
      if (j < keep) w[j] = x[i];
    }
  }
  __syncthreads();  // (the last ones read lie behind)
  for (int j = keep + tid; j < n; j += kMove) w[j] = 0.0f;
}

// In place: token kept[j] >= j goes to j, with j ascending, so a chunk's rows may be written once
// all of that chunk are read: rows of later chunks lie behind everything written so far.  A block
// takes a part of 128 bytes (or what there is) of the keys' or values' rows of one (sequence, key
// head), a whole line, and parts do not meet.
__global__ __launch_bounds__(kMove) void move_kernel(const Args g) {
  const int tid = threadIdx.x;
  const int64_t block = g.first_block + blockIdx.x;
  const int roles = 2 * g.slices + 1;
  const int role = (int)(block % roles);
  const int64_t of = block / roles;
  const int head = (int)(of % g.p.n_heads), seq = (int)(of / g.p.n_heads);
  const int n = tokens_of(g, seq), keep = g.e.keep;
  if (n <= keep) return;
  const int *kept = g.e.kept + of * keep;
  if (role == 2 * g.slices) {
    move_weights(g, g.e.weights + seq * g.e.nb[1] + head * g.e.nb[0], kept, n, tid);
    return;
  }
  const int slice = role >> 1;
  char *pool = static_cast<char *>(role & 1 ? g.p.v_pages : g.p.k_pages) + 128 * slice;
  const int parts = min(128, g.row_bytes - 128 * slice) / 16;  // of 16 bytes
  const int per = kMove / parts;                               // rows of a pass of the threads
  const int part = tid % parts, row0 = tid / parts;
  const int *table = g.q.table + (int64_t)seq * g.q.stride;
  const int chunk = per * kInFlight;
  for (int j0 = 0; j0 < keep; j0 += chunk) {
    const int last = min(j0 + chunk, keep) - 1;
    if (kept[last] == last) continue;  // all of them stay where they are
    u32x4 x[kInFlight];
    int64_t to[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int j = j0 + i * per + row0;
      to[i] = -1;
      if (row0 < per && j <= last) {
        const int64_t from = row_of(g, table, g.q.width, head, kept[j]);
        if (from >= 0) {
          to[i] = row_of(g, table, g.q.width, head, j);
          x[i] = *reinterpret_cast<const u32x4 *>(pool + from * g.row_bytes + 16 * part);
        }
      }
    }
    // every thread's rows have come before any is written
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kInFlight; ++i)
      if (to[i] >= 0) *reinterpret_cast<u32x4 *>(pool + to[i] * g.row_bytes + 16 * part) = x[i];
  }
}

// Into other pages: a block takes a run of tokens of one (sequence, key head), keys and values.
constexpr int kRun = 64;

__global__ __launch_bounds__(kMove) void copy_kernel(const Args g) {
  __shared__ int64_t s_from[kRun], s_to[kRun];
  const int tid = threadIdx.x;
  const int64_t block = g.first_block + blockIdx.x;
  const int chunk = (int)(block % g.chunks);
  const int64_t of = block / g.chunks;
  const int head = (int)(of % g.p.n_heads), seq = (int)(of / g.p.n_heads);
  const int n = tokens_of(g, seq), keep = g.e.keep;
  const int *kept = g.e.kept + of * keep;
  if (chunk == g.chunks - 1) {
    if (n > keep) move_weights(g, g.e.weights + seq * g.e.nb[1] + head * g.e.nb[0], kept, n, tid);
    return;
  }
  const int j0 = chunk * kRun, rows = min(kRun, min(n, keep) - j0);
  if (rows <= 0) return;
  if (tid < rows) {
    const int *table = g.q.table + (int64_t)seq * g.q.stride;
    const int *into = g.e.into + (int64_t)seq * g.e.into_stride;
    const int64_t from = row_of(g, table, g.q.width, head, kept[j0 + tid]);
    s_from[tid] = from;
    s_to[tid] = from < 0 ? -1 : row_of(g, into, g.e.into_width, head, j0 + tid);
  }
  __syncthreads();
  const int parts = g.row_bytes / 16, items = 2 * rows * parts;
  for (int i0 = 0; i0 < items; i0 += kInFlight * kMove) {
    u32x4 x[kInFlight];
    char *to[kInFlight];
#pragma unroll
    for (int k = 0; k < kInFlight; ++k) {
      int i = i0 + k * kMove + tid;
      to[k] = nullptr;
      if (i >= items) continue;
      const bool value = i >= rows * parts;
      i -= value ? rows * parts : 0;
      const int row = i / parts, part = i - row * parts;
      if (s_to[row] < 0) continue;
      char *pool = static_cast<char *>(value ? g.p.v_pages : g.p.k_pages) + 16 * part;
      to[k] = pool + s_to[row] * g.row_bytes;
      x[k] = __builtin_nontemporal_load(
          reinterpret_cast<const u32x4 *>(pool + s_from[row] * g.row_bytes));
    }
#pragma unroll
    for (int k = 0; k < kInFlight; ++k)
      if (to[k]) *reinterpret_cast<u32x4 *>(to[k]) = x[k];
  }
}

template <typename Launch>
hipError_t over_blocks(Args &g, int64_t blocks, int threads, Launch launch) {
  const int64_t most = (((int64_t)1 << 32) - 1) / threads;
  for (int64_t b = 0; b < blocks; b += most) {
    g.first_block = b;
    launch((int)std::min(most, blocks - b));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace

hipError_t launch_paged_evict(const PagedShape &p, const PagedSeqs &q, const PagedEvict &e,
                              hipStream_t s) {
  Args g{};
  g.p = p;
  g.q = q;
  g.e = e;
  g.cap = std::min((int64_t)q.width * p.page_size, (int64_t)kMaxTokens);
  g.row_bytes = p.dim * (p.io == IoType::F32 ? 4 : 2);
  const int64_t rows = (int64_t)q.n_seqs * p.n_heads;
  g.held = (int)std::max<int64_t>(4, std::min<int64_t>(g.cap, kHeld));  // (a multiple of 4)
  hipError_t r = hipFuncSetAttribute(reinterpret_cast<const void *>(select_kernel),
                                     hipFuncAttributeMaxDynamicSharedMemorySize, 4 * kHeld);
  if (r != hipSuccess) return r;
  r = over_blocks(g, rows, kSelect, [&](int blocks) {
    select_kernel<<<blocks, kSelect, 4 * g.held, s>>>(g);
  });
  if (r != hipSuccess) return r;
  if (e.into) {
    g.chunks = (e.keep + kRun - 1) / kRun + 1;
    return over_blocks(g, rows * g.chunks, kMove,
                       [&](int blocks) { copy_kernel<<<blocks, kMove, 0, s>>>(g); });
  }
  g.slices = (g.row_bytes + 127) / 128;
  return over_blocks(g, rows * (2 * g.slices + 1), kMove,
                     [&](int blocks) { move_kernel<<<blocks, kMove, 0, s>>>(g); });
}

}  // namespace aq
