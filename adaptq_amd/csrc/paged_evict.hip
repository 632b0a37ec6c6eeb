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
constexpr uint32_t kZero = 0x80000000u;  // the key of a weight of 0
// Weights that a thread holds: those of so many tokens are read once, longer sequences' in
// stretches of as many, for each of the three digits and for the list (32,768 tokens, 8 heads,
// both launches: 56 us; from LDS, and one counter a digit, 65).
constexpr int kHeld = 32;
constexpr int kStretch = kHeld * kSelect;
// Digits of 11, 11 and 10 bits: the first holds sign, exponent and two bits more, so that even
// weights of like size spread over many counters.  A counter takes one lane at a time, so there
// are some of each digit, side by side.
constexpr int kBins = 1 << 11;
constexpr int kCopies = 4;
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
  int64_t first_block;
};

// Weights in the order of their bits: larger weights have larger keys, both zeros the same one.
__device__ __forceinline__ uint32_t key_of(float w) {
  const uint32_t u = __float_as_uint(w + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ int tokens_of(const Args &g, int seq) {
  const int64_t n = max(g.q.lengths[seq], 0);
  return (int)min(n, g.cap);
}

__global__ __launch_bounds__(kSelect) void select_kernel(const Args g) {
  __shared__ __align__(16) int s_count[kBins * kCopies];
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
    for (int64_t j = tid; j < keep; j += kSelect) kept[j] = j < n ? (int)j : -1;
    return;
  }
  const float *w = g.e.weights + seq * g.e.nb[1] + head * g.e.nb[0];
  const int old = n - g.e.recent;  // tokens before the newest, which stay
  int room = keep - g.e.recent;    // of those, so many stay
  // The keys of a stretch: each wave a run of its tokens, 64 neighbours a step.
  uint32_t key[kHeld];
  int t0 = 0, count = 0, steps = 0;  // the run, the same `steps` for all waves
  const auto hold = [&](int64_t from) {
    const int m = (int)min((int64_t)kStretch, old - from);
    const int per = ((m + kSelectWaves - 1) / kSelectWaves + 63) / 64 * 64;
    steps = per / 64;
    t0 = (int)min(from + wave * per, (int64_t)old - 1);
    count = min(max(m - wave * per, 0), per);
#pragma unroll
    for (int j0 = 0; j0 < kHeld; j0 += 8) {
      if (j0 >= steps) break;
#pragma unroll
      for (int j = j0; j < j0 + 8; ++j)
        key[j] = __float_as_uint(w[min((int64_t)t0 + 64 * j + lane, (int64_t)old - 1)]);
    }
#pragma unroll
    for (int j0 = 0; j0 < kHeld; j0 += 8) {
      if (j0 >= steps) break;
#pragma unroll
      for (int j = j0; j < j0 + 8; ++j) key[j] = key_of(__uint_as_float(key[j]));
    }
  };
  const auto each_key = [&](auto use) {  // use(key, step, whether the lane has one)
#pragma unroll
    for (int j0 = 0; j0 < kHeld; j0 += 4) {
      if (j0 >= steps) break;
#pragma unroll
      for (int j = j0; j < j0 + 4; ++j) use(key[j], j, 64 * j + lane < count);
    }
  };
  const bool once = old <= kStretch;
  if (room > 0 && once) hold(0);
  // the key of the last one that stays, digit by digit; `room` becomes how many of that key
  const bool none = room <= 0;
  uint32_t prefix = 0;
  for (int top = 32; !none && top > 0;) {
    const int shift = max(top - 11, 0), bins = 1 << (top - shift);
    const uint32_t beyond = top == 32 ? 0 : 1u << top;
    for (int i = 4 * tid; i < kBins * kCopies; i += 4 * kSelect)
      *reinterpret_cast<u32x4 *>(s_count + i) = u32x4{0, 0, 0, 0};
    __syncthreads();
    for (int64_t from = 0; from < old; from += kStretch) {
      if (!once) hold(from);
      each_key([&](uint32_t k, int, bool there) {
        there = there && ((k ^ prefix) < beyond || beyond == 0);
        if (!__any(there)) return;
        // tokens without any weight are many, and counted together
        const bool zero = there && k == kZero;
        const uint64_t zeros = __ballot(zero);
        if (zeros && lane == 0)
          atomicAdd(&s_count[(kZero >> shift & (bins - 1)) * kCopies], __popcll(zeros));
        if (there && !zero)
          atomicAdd(&s_count[(k >> shift & (bins - 1)) * kCopies + lane % kCopies], 1);
      });
    }
    __syncthreads();
    // the digit at which `room` values from the top are reached: two digits a thread, the
    // largest first
    static_assert(kBins == 2 * kSelect, "two digits a thread");
    const int digit = kBins - 1 - 2 * tid;
    int c[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int k = 0; k < kCopies; ++k) c[i] += s_count[(digit - i) * kCopies + k];
    const int sum = c[0] + c[1];
    int end = sum;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const int y = __shfl_up(end, k, 64);
      if (lane >= k) end += y;
    }
    if (lane == 63) s_gt[wave] = end;
    __syncthreads();
    int above = end - sum;
    for (int k = 0; k < wave; ++k) above += s_gt[k];
    if (above < room && above + sum >= room) {
      const bool second = above + c[0] < room;
      s_digit = digit - second;
      s_above = above + (second ? c[0] : 0);
    }
    __syncthreads();
    prefix |= s_digit << shift;
    room -= s_above;
    top = shift;
  }
  // each wave's run of the older tokens: how many stay, and of those with the last key the first
  // `room`; then the indexes in order
  int at = 0, ties = 0;
  const uint64_t below = ((uint64_t)1 << lane) - 1;
  for (int64_t from = 0; !none && from < old; from += kStretch) {
    if (!once) hold(from);
    int gt = 0, eq = 0;
    each_key([&](uint32_t k, int, bool there) {
      gt += __popcll(__ballot(there && k > prefix));
      eq += __popcll(__ballot(there && k == prefix));
    });
    __syncthreads();
    if (lane == 0) {
      s_gt[wave] = gt;
      s_eq[wave] = eq;
    }
    __syncthreads();
    int to = 0, tied_before = 0;  // of this wave
    for (int k = 0; k < kSelectWaves; ++k) {
      if (k == wave) {
        to = at;
        tied_before = ties;
      }
      at += s_gt[k] + min(s_eq[k], max(room - ties, 0));
      ties += s_eq[k];
    }
    each_key([&](uint32_t k, int j, bool there) {
      const bool tie = there && k == prefix;
      const uint64_t tied = __ballot(tie);
      const bool stays =
          (there && k > prefix) || (tie && tied_before + __popcll(tied & below) < room);
      const uint64_t all = __ballot(stays);
      if (stays) kept[to + __popcll(all & below)] = t0 + 64 * j + lane;
      to += __popcll(all);
      tied_before += __popcll(tied);
    });
  }
  for (int64_t j = tid; j < g.e.recent; j += kSelect)
    kept[keep - g.e.recent + j] = old + (int)j;
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
  for (int64_t j0 = 0; j0 < keep; j0 += kInFlight * kMove) {
    float x[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int64_t j = j0 + i * kMove + tid;
      if (j < keep) x[i] = w[kept[j]];
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int64_t j = j0 + i * kMove + tid;
      if (j < keep) w[j] = x[i];
    }
  }
  __syncthreads();  // (the last ones read lie behind)
  for (int64_t j = (int64_t)keep + tid; j < n; j += kMove) w[j] = 0.0f;
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
  for (int64_t j0 = 0; j0 < keep; j0 += chunk) {
    const int last = (int)min(j0 + chunk, (int64_t)keep) - 1;
    if (kept[last] == last) continue;  // all of them stay where they are
    u32x4 x[kInFlight];
    int64_t to[kInFlight];
#pragma unroll
    for (int i = 0; i < kInFlight; ++i) {
      const int64_t j = j0 + i * per + row0;
      to[i] = -1;
      if (row0 < per && j <= last) {
        const int64_t from = row_of(g, table, g.q.width, head, kept[j]);
        if (from >= 0) {
          to[i] = row_of(g, table, g.q.width, head, (int)j);
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
  const hipError_t r = over_blocks(
      g, rows, kSelect, [&](int blocks) { select_kernel<<<blocks, kSelect, 0, s>>>(g); });
  if (r != hipSuccess) return r;
  if (e.into) {
    // (of the tokens that a sequence can hold: keep may be up to the last int)
    g.chunks = (int)((std::min((int64_t)e.keep, g.cap) + kRun - 1) / kRun) + 1;
    return over_blocks(g, rows * g.chunks, kMove,
                       [&](int blocks) { copy_kernel<<<blocks, kMove, 0, s>>>(g); });
  }
  g.slices = (g.row_bytes + 127) / 128;
  return over_blocks(g, rows * (2 * g.slices + 1), kMove,
                     [&](int blocks) { move_kernel<<<blocks, kMove, 0, s>>>(g); });
}

}  // namespace aq
