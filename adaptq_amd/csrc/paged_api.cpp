// paged_api.cpp -- the C ABI of the rotary positions and of the paged cache
// (include/adaptq.h, part 3): argument checks, handles, launches.
//
// Nothing here synchronises or allocates after a handle's creation: a call is one
// launch on the caller's stream, or a few in a row (prompts whose tiles are cut, the
// weights of tokens, eviction, more blocks than a launch takes), and may be captured
// into a graph.
#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <new>
#include <vector>

#include "../../include/adaptq.h"
#include "host.hpp"
#include "paged.hpp"
#include "row_sets.hpp"

namespace {

using aq::DeviceGuard;
using aq::hip_fail;
using aq::require_handle;
using aq::require_pointer;
using aq::rows_apart;
using aq::set_errorf;
using aq::sets_apart;
using aq::Span;
using aq::span_of;

constexpr int kMaxRotaryDim = 1024;
constexpr int kMaxPagedDim = 256;
constexpr int kMaxHeads = 1 << 15;  // of one set of rows
constexpr int kPageUnit = 16;
constexpr int kMaxPageSize = 1 << 16;

struct Rotary {
  int device = 0;
  std::vector<uint64_t> steps;  // per pair, in 2^-64 turns a position
  uint64_t *d_steps = nullptr;
  bool interleaved = false;
  float amplitude = 1.0f;
  aq::RotaryTable table() const { return {d_steps, (int)steps.size(), interleaved, amplitude}; }
};

struct Paged {
  int device = 0;
  aq::PagedShape shape{};
  uint64_t *d_steps = nullptr;
  void *ws = nullptr;
  bool four = false;  // pages of 4-bit values
  size_t pool = 0;    // bytes of each
};

bool exact_pages(const Paged *p, const char *fn) {
  if (!p->four) return true;
  set_errorf(fn, "the cache holds 4-bit values");
  return false;
}
bool four_bits(const Paged *p, const char *fn) {
  if (p->four) return true;
  set_errorf(fn, "the cache holds exact rows");
  return false;
}

size_t size_of(int io_type) { return io_type == ADAPTQ_IO_F32 ? 4 : 2; }

bool io_ok(int io_type, const char *fn) {
  if (io_type >= ADAPTQ_IO_F32 && io_type <= ADAPTQ_IO_BF16) return true;
  set_errorf(fn, "io_type must be ADAPTQ_IO_F32, _F16 or _BF16");
  return false;
}

bool strides_ok(size_t size, const int *n, const size_t *nb, int dims, const char *fn) {
  for (int i = 0; i < dims; ++i) {
    if (nb[i] % size) {
      set_errorf(fn, "strides must be multiples of the element size");
      return false;
    }
    if (n[i] > 1 && nb[i] > ((size_t)1 << 60) / (size_t)n[i]) {
      set_errorf(fn, "strides out of range");
      return false;
    }
  }
  return true;
}

bool aligned_to(const void *p, size_t size, const char *fn) {
  if (reinterpret_cast<uintptr_t>(p) % size == 0) return true;
  set_errorf(fn, "pointers must be aligned to the element size");
  return false;
}

// The rotation of each pair per position, in turns.
bool rotary_steps(int dim, double base, int scaling, double factor, int context, double slow,
                  double fast, std::vector<uint64_t> *steps) {
  const long double two_pi = 6.283185307179586476925286766559005768L;
  const int pairs = dim / 2;
  long double b = base;
  if (scaling == ADAPTQ_ROTARY_NTK) b *= powl(factor, (long double)dim / (dim - 2));
  // the ramp of ADAPTQ_ROTARY_YARN: the pairs (as numbers) that turn fast and slow
  // times over the context
  long double ramp_lo = 0, ramp_hi = 0;
  if (scaling == ADAPTQ_ROTARY_YARN) {
    ramp_lo = floorl(dim * logl(context / (fast * two_pi)) / (2 * logl(base)));
    ramp_hi = ceill(dim * logl(context / (slow * two_pi)) / (2 * logl(base)));
    if (ramp_lo < 0) ramp_lo = 0;
    if (ramp_hi > dim - 1) ramp_hi = dim - 1;
    if (ramp_hi <= ramp_lo) ramp_hi = ramp_lo + 0.001L;
  }
  for (int i = 0; i < pairs; ++i) {
    long double f = powl(b, -2.0L * i / dim);
    long double keep = 1;  // the share of f that is not slowed down
    if (scaling == ADAPTQ_ROTARY_LINEAR) keep = 0;
    if (scaling == ADAPTQ_ROTARY_BANDS) keep = (context * f / two_pi - slow) / (fast - slow);
    if (scaling == ADAPTQ_ROTARY_YARN) keep = 1 - (i - ramp_lo) / (ramp_hi - ramp_lo);
    keep = keep < 0 ? 0 : keep > 1 ? 1 : keep;
    f = keep * f + (1 - keep) * f / factor;
    const long double turns = f / two_pi;
    if (!(turns >= 0 && turns < 1)) return false;
    (*steps)[i] = (uint64_t)(turns * 18446744073709551616.0L + 0.5L);
  }
  return true;
}

// Device copy of the steps, on the current device.
hipError_t upload_steps(const std::vector<uint64_t> &steps, uint64_t **out) {
  const size_t bytes = sizeof(uint64_t) * steps.size();
  hipError_t e = hipMalloc(out, bytes);
  if (e != hipSuccess) {
    *out = nullptr;
    return e;
  }
  e = hipMemcpy(*out, steps.data(), bytes, hipMemcpyHostToDevice);
  if (e != hipSuccess) {
    (void)hipFree(*out);
    *out = nullptr;
  }
  return e;
}

// Table, lengths and count of a call's sequences.
bool seqs_ok(const int *table, int width, int stride, const int *lengths, int n_seqs,
             const char *fn) {
  if (n_seqs < 0 || width < 0) {
    set_errorf(fn, "negative n_seqs or table_width");
    return false;
  }
  if (n_seqs == 0) return true;
  if ((width > 0 && !require_pointer(table, fn, "d_table")) ||
      !require_pointer(lengths, fn, "d_lengths"))
    return false;
  if (stride < width) {
    set_errorf(fn, "table_stride is smaller than table_width");
    return false;
  }
  return aligned_to(table, 4, fn) && aligned_to(lengths, 4, fn);
}

bool over_pages(const Paged *p, const Span &x) {
  for (const void *q : {p->shape.k_pages, p->shape.v_pages}) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(q);
    if (x.lo < lo + p->pool && lo < x.hi) return true;
  }
  return false;
}

// Rows of a call against the cache: strides, alignment, and the pages' own memory.
bool rows_ok(const Paged *p, const void *rows, const char *name, int heads, int n, size_t nb1,
             size_t nb2, bool written, const char *fn) {
  const aq::PagedShape &s = p->shape;
  const size_t size = size_of((int)s.io), row = size * s.dim;
  const int counts[2] = {heads, n};
  const size_t nb[2] = {nb1, nb2};
  if (!require_pointer(rows, fn, name) || !aligned_to(rows, size, fn) ||
      !strides_ok(size, counts, nb, 2, fn))
    return false;
  if (written && !rows_apart(row, counts, nb, 2)) {
    set_errorf(fn, "output rows overlap");
    return false;
  }
  if (over_pages(p, span_of(rows, row, counts, nb, 2))) {
    set_errorf(fn, "rows overlap the pages");
    return false;
  }
  return true;
}

bool append_ok(const Paged *p, const void *k, const void *v, int n_tokens, const size_t *nb,
               const char *fn) {
  return rows_ok(p, k, "d_k", p->shape.n_heads, n_tokens, nb[0], nb[1], false, fn) &&
         rows_ok(p, v, "d_v", p->shape.n_heads, n_tokens, nb[2], nb[3], false, fn);
}

bool attend_ok(const Paged *p, const void *q, const void *out, int q_heads, int n_seqs,
               const size_t *nb, float scale, int window, const char *fn) {
  if (q_heads <= 0 || q_heads > kMaxHeads || q_heads % p->shape.n_heads) {
    set_errorf(fn, "n_q_heads must be a multiple of the cache's n_heads, up to 32768");
    return false;
  }
  if (!std::isfinite(scale * 1.5f)) {  // the kernel takes it times log2(e)
    set_errorf(fn, "scale must be finite, up to 2.2e38");
    return false;
  }
  if (window < 0) {
    set_errorf(fn, "negative window");
    return false;
  }
  if ((long long)n_seqs * q_heads > INT_MAX) {
    set_errorf(fn, "too many sequences");
    return false;
  }
  if (n_seqs == 0) return true;
  return rows_ok(p, q, "d_q", q_heads, n_seqs, nb[0], nb[1], false, fn) &&
         rows_ok(p, out, "d_out", q_heads, n_seqs, nb[2], nb[3], true, fn);
}

bool scores_ok(const adaptq_scores_t *s, float scale, aq::PagedScores *to, const char *fn) {
  *to = aq::PagedScores{};
  if (!s) return true;
  if (!(s->softcap >= 0.0f && std::isfinite(s->softcap * 1.5f))) {  // (times log2(e) in the kernel)
    set_errorf(fn, "softcap must not be negative, up to 2.2e38");
    return false;
  }
  if (s->softcap > 0.0f && (s->softcap < 0x1p-100f || !std::isfinite(scale / s->softcap))) {
    set_errorf(fn, "softcap must be 0 or at least 2^-100, and scale / softcap finite");
    return false;
  }
  if (s->window < 0) {
    set_errorf(fn, "negative window");
    return false;
  }
  if (!aligned_to(s->d_slopes, 4, fn) || !aligned_to(s->d_prefix, 4, fn) ||
      !aligned_to(s->d_first, 4, fn))
    return false;
  *to = {s->softcap, s->window, s->d_slopes, s->d_prefix, s->d_first};
  return true;
}

bool workspace_ok(const void *ws, size_t bytes, size_t needed, const char *fn) {
  if (needed == 0) return true;
  if (bytes < needed) {
    set_errorf(fn, "the workspace is too small");
    return false;
  }
  return require_pointer(ws, fn, "d_workspace") && aligned_to(ws, 16, fn);
}

float scale_of(const Paged *p, float scale) {
  return scale != 0.0f ? scale : (float)(1.0 / std::sqrt((double)p->shape.dim));
}

bool out_apart(const Paged *p, const void *out, int out_heads, size_t o1, size_t o2,
               const void *in, int in_heads, size_t i1, size_t i2, int n, const char *fn) {
  const size_t row = size_of((int)p->shape.io) * p->shape.dim;
  const int no[2] = {out_heads, n}, ni[2] = {in_heads, n};
  const size_t so[2] = {o1, o2}, si[2] = {i1, i2};
  if (sets_apart(out, row, no, so, in, ni, si, 2)) return true;
  set_errorf(fn, "d_out overlaps an input");
  return false;
}

aq::PagedAttend attend_args(const Paged *p, const void *q, void *out, int q_heads, size_t q1,
                            size_t q2, size_t o1, size_t o2, float scale, int window, int extra) {
  aq::PagedAttend a{};
  a.q = q;
  a.out = out;
  a.q_nb[0] = q1;
  a.q_nb[1] = q2;
  a.out_nb[0] = o1;
  a.out_nb[1] = o2;
  a.q_heads = q_heads;
  a.scale = scale_of(p, scale);
  a.window = window;
  a.extra = extra;
  return a;
}

void destroy_paged(Paged *p) {
  DeviceGuard g(p->device);
  if (p->d_steps) (void)hipFree(p->d_steps);  // waits for the device
  if (p->ws) (void)hipFree(p->ws);
  delete p;
}

Paged *create_paged(void *d_k_pages, void *d_v_pages, int n_pages, int page_size, int n_heads,
                    int dim, int io_type, adaptq_rotary_t rotary, bool four, const char *fn) {
  if (!require_pointer(d_k_pages, fn, "d_k_pages") || !require_pointer(d_v_pages, fn, "d_v_pages") ||
      !io_ok(io_type, fn))
    return nullptr;
  if (n_pages <= 0 || n_heads <= 0 || n_heads > kMaxHeads) {
    set_errorf(fn, "n_pages must be positive, n_heads from 1 to 32768");
    return nullptr;
  }
  if (page_size <= 0 || page_size % kPageUnit || page_size > kMaxPageSize) {
    set_errorf(fn, "page_size must be a multiple of 16 up to 65536");
    return nullptr;
  }
  if (dim <= 0 || dim % (four ? 32 : 8) || dim > kMaxPagedDim) {
    set_errorf(fn, four ? "dim must be a multiple of 32 up to 256"
                        : "dim must be a multiple of 8 up to 256");
    return nullptr;
  }
  if (!aligned_to(d_k_pages, 16, fn) || !aligned_to(d_v_pages, 16, fn)) {
    set_errorf(fn, "pages must be aligned to 16 bytes");
    return nullptr;
  }
  const size_t token = four ? (size_t)17 * dim / 32 : size_of(io_type) * dim;
  const size_t page = token * page_size * (size_t)n_heads;
  if ((size_t)n_pages > ((size_t)1 << 60) / page) {
    set_errorf(fn, "the pages are too large");
    return nullptr;
  }
  const uintptr_t k = reinterpret_cast<uintptr_t>(d_k_pages),
                  v = reinterpret_cast<uintptr_t>(d_v_pages);
  if (k < v + page * n_pages && v < k + page * n_pages) {
    set_errorf(fn, "d_k_pages and d_v_pages overlap");
    return nullptr;
  }
  const Rotary *r = static_cast<Rotary *>(rotary);
  if (r && 2 * (int)r->steps.size() > dim) {
    set_errorf(fn, "the rotary's rotary_dim is larger than dim");
    return nullptr;
  }
  int device = 0, cus = 0;
  if (hip_fail(hipGetDevice(&device), fn) ||
      hip_fail(hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, device), fn))
    return nullptr;
  Paged *p = new (std::nothrow) Paged();
  if (!p) {
    set_errorf(fn, "host allocation failed");
    return nullptr;
  }
  p->device = device;
  p->four = four;
  p->pool = page * n_pages;
  p->shape = {d_k_pages, d_v_pages, n_pages, page_size, n_heads, dim,
              static_cast<aq::IoType>(io_type), {}, cus};
  hipError_t e = hipSuccess;
  if (r) {
    p->shape.rotary = r->table();
    e = upload_steps(r->steps, &p->d_steps);  // its own: the rotary may be destroyed
    p->shape.rotary.steps = p->d_steps;
  }
  const size_t ws = aq::paged_workspace_bytes(p->shape);
  if (e == hipSuccess && ws) {
    e = hipMalloc(&p->ws, ws);
    if (e != hipSuccess) p->ws = nullptr;
    if (e == hipSuccess) e = hipMemset(p->ws, 0, ws);
    if (e == hipSuccess) e = hipDeviceSynchronize();  // before any stream may use it
  }
  if (hip_fail(e, fn)) {
    destroy_paged(p);
    return nullptr;
  }
  aq::clear_error();
  return p;
}

int paged_append(Paged *p, const void *d_k, const void *d_v, int n_tokens, const size_t *nb,
                 const aq::PagedSeqs &q, const int *d_offsets, void *stream, const char *fn) {
  if (n_tokens < 0) {
    set_errorf(fn, "negative n_tokens");
    return -1;
  }
  if (!seqs_ok(q.table, q.width, q.stride, q.lengths, q.n_seqs, fn)) return -1;
  if (!d_offsets && n_tokens != q.n_seqs) {
    set_errorf(fn, "without d_offsets, n_tokens must be n_seqs (one token a sequence)");
    return -1;
  }
  if (n_tokens == 0 || q.n_seqs == 0) {
    aq::clear_error();
    return 0;
  }
  if (!append_ok(p, d_k, d_v, n_tokens, nb, fn)) return -1;
  if (d_offsets && !aligned_to(d_offsets, 4, fn)) return -1;
  const aq::PagedAppend a{d_k, d_v, {nb[0], nb[1]}, {nb[2], nb[3]}, n_tokens, d_offsets};
  DeviceGuard g(p->device);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (hip_fail(p->four ? aq::launch_paged4_append(p->shape, q, a, s)
                       : aq::launch_paged_append(p->shape, q, a, s),
               fn))
    return -1;
  aq::clear_error();
  return 0;
}

// Queries of a call of one token a sequence, and for a step (k) its rows.
struct Token {
  const void *k, *v;
  size_t kv_nb[4];
  const void *q;
  void *out;
  int q_heads;
  size_t q_nb[4];  // of q, of out
  float scale;
  int window;
};

int paged_token(Paged *p, const Token &t, const aq::PagedSeqs &q, const aq::PagedScores *scores,
                const aq::PagedWeights *weights, void *stream, const char *fn) {
  if (!seqs_ok(q.table, q.width, q.stride, q.lengths, q.n_seqs, fn) ||
      !attend_ok(p, t.q, t.out, t.q_heads, q.n_seqs, t.q_nb, t.scale, t.window, fn))
    return -1;
  if (q.n_seqs == 0) {
    aq::clear_error();
    return 0;
  }
  const int H = p->shape.n_heads;
  const size_t *nb = t.q_nb, *knb = t.kv_nb;
  if (t.k && !append_ok(p, t.k, t.v, q.n_seqs, knb, fn)) return -1;
  if (!out_apart(p, t.out, t.q_heads, nb[2], nb[3], t.q, t.q_heads, nb[0], nb[1], q.n_seqs, fn))
    return -1;
  if (t.k && (!out_apart(p, t.out, t.q_heads, nb[2], nb[3], t.k, H, knb[0], knb[1], q.n_seqs, fn) ||
              !out_apart(p, t.out, t.q_heads, nb[2], nb[3], t.v, H, knb[2], knb[3], q.n_seqs, fn)))
    return -1;
  const aq::PagedAppend ap{t.k, t.v, {knb[0], knb[1]}, {knb[2], knb[3]}, q.n_seqs, nullptr};
  const aq::PagedAppend *step = t.k ? &ap : nullptr;
  const aq::PagedAttend a = attend_args(p, t.q, t.out, t.q_heads, nb[0], nb[1], nb[2], nb[3],
                                        t.scale, t.window, t.k ? 1 : 0);
  DeviceGuard g(p->device);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  hipError_t e;
  if (p->four)
    e = aq::launch_paged4_attend(p->shape, q, a, step, scores ? *scores : aq::PagedScores{}, p->ws, s);
  else if (scores)
    e = aq::launch_paged_shaped(p->shape, q, a, step, *scores,
                                weights ? *weights : aq::PagedWeights{}, p->ws, s);
  else
    e = aq::launch_paged_attend(p->shape, q, a, step, p->ws, s);
  if (hip_fail(e, fn)) return -1;
  aq::clear_error();
  return 0;
}

// Whether a prompt goes through the single-token kernel: its queries make one tile of 16 rows a
// key head and sequence on the average, and it takes the masks.  One such tile costs what one
// query does (32 sequences of up to 4,000 tokens, 8 heads, 4 queries of 4 heads each 71.5 us,
// through a prompt's tiles 111; 8 of 8,192, fp32, 8 queries of 2, a window of 1,000 34.5 and 51;
// one of 16,000, 4 queries of 4, 43.2 and 44.8), two read all rows twice (8 of up to 1,500, 6
// queries of 4, 35.4 and 33.9; four tiles, 16 of up to 4,000, 87 and 63).  The average decides, for
// the offsets are on the device; a chunk among single tokens is no slower by it (4 query heads of
// 8, 63 single tokens and a chunk of 190 over 4,096 tokens each: 280 us, through a prompt's tiles
// 317; the chunk over 16,384, the others over 1,024: 468 and 570).
constexpr int kFewRows = 16;
bool few_queries(const Paged *p, const aq::PagedPrompt &a, int n_seqs) {
  const long long rows = (long long)a.n_tokens * (a.q_heads / p->shape.n_heads);
  return rows <= kFewRows * (long long)n_seqs && !a.scores.first &&
         !(a.scores.prefix && a.scores.window > 0);
}

// Weights [n_seqs][n_heads][tokens] of a call, and the memory their scores take meanwhile.
bool weights_ok(const Paged *p, float *w, size_t nb1, size_t nb2, const aq::PagedSeqs &q,
                aq::PagedWeights *to, const char *fn) {
  *to = aq::PagedWeights{};
  if (!w) return true;
  const size_t nb[2] = {nb1, nb2};
  const int n[2] = {p->shape.n_heads, q.n_seqs};
  if (!aligned_to(w, 4, fn) || !strides_ok(4, n, nb, 2, fn)) return false;
  const size_t row = (size_t)q.width * p->shape.page_size * 4;
  if (!rows_apart(row, n, nb, 2)) {
    set_errorf(fn, "d_weights has rows of fewer than table_width * page_size values");
    return false;
  }
  if (q.n_seqs > 0 && over_pages(p, span_of(w, row, n, nb, 2))) {
    set_errorf(fn, "d_weights overlaps the pages");
    return false;
  }
  to->weights = w;
  to->nb[0] = (int64_t)(nb1 / 4);
  to->nb[1] = (int64_t)(nb2 / 4);
  return true;
}

int paged_scored(Paged *p, const Token &t, const aq::PagedSeqs &q, const adaptq_scores_t *scores,
                 float *d_weights, size_t w_nb1, size_t w_nb2, void *ws, size_t ws_bytes,
                 void *stream, const char *fn) {
  aq::PagedScores sc;
  aq::PagedWeights w;
  if (q.n_seqs < 0 || q.width < 0) return paged_token(p, t, q, nullptr, nullptr, stream, fn);
  if (!scores_ok(scores, scale_of(p, t.scale), &sc, fn) ||
      !weights_ok(p, d_weights, w_nb1, w_nb2, q, &w, fn))
    return -1;
  if (w.weights) {
    if (t.q_heads <= 0 || t.q_heads % p->shape.n_heads || (long long)q.n_seqs * t.q_heads > INT_MAX)
      return paged_token(p, t, q, nullptr, nullptr, stream, fn);  // (refuses)
    if (!workspace_ok(ws, ws_bytes,
                      aq::paged_weights_workspace(p->shape, t.q_heads, q.n_seqs, q.width), fn))
      return -1;
    w.workspace = ws;
    // the sums against the rows of the call, each from its first byte to its last
    const size_t row = size_of((int)p->shape.io) * p->shape.dim, w_nb[2] = {w_nb1, w_nb2};
    const int nw[2] = {p->shape.n_heads, q.n_seqs}, nq[2] = {t.q_heads, q.n_seqs};
    const Span x = span_of(w.weights, (size_t)q.width * p->shape.page_size * 4, nw, w_nb, 2);
    const auto meets = [&](const void *rows, const int *n, const size_t *nb) {
      if (!rows || q.n_seqs == 0) return false;
      const Span y = span_of(rows, row, n, nb, 2);
      return x.lo < y.hi && y.lo < x.hi;
    };
    if (meets(t.q, nq, t.q_nb) || meets(t.out, nq, t.q_nb + 2) || meets(t.k, nw, t.kv_nb) ||
        meets(t.v, nw, t.kv_nb + 2)) {
      set_errorf(fn, "d_weights overlaps rows of the call");
      return -1;
    }
  }
  Token to = t;
  to.window = sc.window;
  return paged_token(p, to, q, &sc, &w, stream, fn);
}

}  // namespace

extern "C" {

adaptq_rotary_t adaptq_rotary_create(int rotary_dim, int interleaved, double base, int scaling,
                                     double factor, int context, double slow, double fast,
                                     double amplitude) {
  const char *fn = "adaptq_rotary_create";
  if (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > kMaxRotaryDim) {
    set_errorf(fn, "rotary_dim must be even, from 2 to 1024");
    return nullptr;
  }
  if (scaling < ADAPTQ_ROTARY_PLAIN || scaling > ADAPTQ_ROTARY_BANDS) {
    set_errorf(fn, "unknown scaling");
    return nullptr;
  }
  const bool ramp = scaling == ADAPTQ_ROTARY_YARN || scaling == ADAPTQ_ROTARY_BANDS;
  if (!(std::isfinite(base) && base > 1.0) || !(std::isfinite(factor) && factor >= 1.0) ||
      !(std::isfinite((float)amplitude) && amplitude >= 0.0)) {
    set_errorf(fn, "base must be above 1, factor at least 1, amplitude not negative (nor beyond fp32)");
    return nullptr;
  }
  if (scaling == ADAPTQ_ROTARY_NTK && rotary_dim == 2) {
    set_errorf(fn, "ADAPTQ_ROTARY_NTK needs more than one pair");
    return nullptr;
  }
  if (slow == 0.0) slow = 1.0;
  if (fast == 0.0) fast = scaling == ADAPTQ_ROTARY_YARN ? 32.0 : 4.0;
  if (ramp && !(context > 0 && std::isfinite(slow) && std::isfinite(fast) && slow > 0.0 &&
                fast > slow)) {
    set_errorf(fn, "this scaling needs context > 0 and fast > slow > 0");
    return nullptr;
  }
  Rotary *r = new (std::nothrow) Rotary();
  if (!r) {
    set_errorf(fn, "host allocation failed");
    return nullptr;
  }
  try {
    r->steps.resize((size_t)rotary_dim / 2);
  } catch (const std::bad_alloc &) {
    delete r;
    set_errorf(fn, "host allocation failed");
    return nullptr;
  }
  r->interleaved = interleaved != 0;
  if (amplitude == 0.0)
    amplitude = scaling == ADAPTQ_ROTARY_YARN ? 0.1 * std::log(factor) + 1.0 : 1.0;
  r->amplitude = (float)amplitude;
  if (!rotary_steps(rotary_dim, base, scaling, factor, context, slow, fast, &r->steps)) {
    delete r;
    set_errorf(fn, "parameters out of range");
    return nullptr;
  }
  if (hip_fail(hipGetDevice(&r->device), fn) || hip_fail(upload_steps(r->steps, &r->d_steps), fn)) {
    delete r;
    return nullptr;
  }
  aq::clear_error();
  return r;
}

void adaptq_rotary_destroy(adaptq_rotary_t h) {
  if (!h) return;
  Rotary *r = static_cast<Rotary *>(h);
  DeviceGuard g(r->device);
  (void)hipFree(r->d_steps);  // waits for the device: no kernel still reads them
  delete r;
}

int adaptq_rotary_device(adaptq_rotary_t h, const adaptq_rows_t *rows, int n_rows, int dim,
                         int io_type, const int *d_positions, size_t pos_stride, int n_batch,
                         int n_tokens, int backward, void *stream) {
  const char *fn = "adaptq_rotary_device";
  if (!require_handle(h, fn) || !require_pointer(rows, fn, "rows") || !io_ok(io_type, fn)) return -1;
  const Rotary *r = static_cast<Rotary *>(h);
  if (n_rows < 1 || n_rows > 2) {
    set_errorf(fn, "n_rows must be 1 or 2");
    return -1;
  }
  if (dim < 2 * (int)r->steps.size() || dim > kMaxRotaryDim) {
    set_errorf(fn, "dim must be from rotary_dim to 1024");
    return -1;
  }
  if (n_batch < 0 || n_tokens < 0 || (long long)n_batch * n_tokens > INT_MAX) {
    set_errorf(fn, "n_batch or n_tokens out of range");
    return -1;
  }
  if (n_batch == 0 || n_tokens == 0) {
    aq::clear_error();
    return 0;
  }
  if (!require_pointer(d_positions, fn, "d_positions") || !aligned_to(d_positions, 4, fn)) return -1;
  if (pos_stride != 0 && pos_stride < (size_t)n_tokens) {
    set_errorf(fn, "pos_stride must be 0 or at least n_tokens");
    return -1;
  }
  const size_t size = size_of(io_type), row = size * dim;
  aq::RotaryCall c{};
  int counts[2][3];
  for (int i = 0; i < n_rows; ++i) {
    const adaptq_rows_t &x = rows[i];
    aq::RotaryRows &y = c.rows[i];
    if (!require_pointer(x.in, fn, "rows.in") || !require_pointer(x.out, fn, "rows.out")) return -1;
    if (x.n_heads <= 0 || x.n_heads > kMaxHeads) {
      set_errorf(fn, "n_heads must be from 1 to 32768");
      return -1;
    }
    counts[i][0] = x.n_heads;
    counts[i][1] = n_tokens;
    counts[i][2] = n_batch;
    y = {x.in, x.out, x.n_heads, {x.in_nb1, x.in_nb2, x.in_nb3}, {x.out_nb1, x.out_nb2, x.out_nb3}};
    // a stride that no index takes says nothing about where rows lie
    for (int k = 0; k < 3; ++k)
      if (counts[i][k] == 1) y.in_nb[k] = y.out_nb[k] = 0;
    if (!aligned_to(x.in, size, fn) || !aligned_to(x.out, size, fn) ||
        !strides_ok(size, counts[i], y.in_nb, 3, fn) || !strides_ok(size, counts[i], y.out_nb, 3, fn))
      return -1;
    if (!rows_apart(row, counts[i], y.out_nb, 3)) {
      set_errorf(fn, "output rows overlap");
      return -1;
    }
  }
  for (int i = 0; i < n_rows; ++i)
    for (int j = 0; j < n_rows; ++j) {
      // an output may be its own input in place, and shares nothing with any other rows
      const aq::RotaryRows &o = c.rows[i], &x = c.rows[j];
      const bool in_place = i == j && o.in == o.out && o.in_nb[0] == o.out_nb[0] &&
                            o.in_nb[1] == o.out_nb[1] && o.in_nb[2] == o.out_nb[2];
      if (!in_place && !sets_apart(o.out, row, counts[i], o.out_nb, x.in, counts[j], x.in_nb, 3)) {
        set_errorf(fn, "an output overlaps an input (and is not it)");
        return -1;
      }
      if (i < j &&
          !sets_apart(o.out, row, counts[i], o.out_nb, x.out, counts[j], x.out_nb, 3)) {
        set_errorf(fn, "the outputs overlap");
        return -1;
      }
    }
  c.n_rows = n_rows;
  c.positions = d_positions;
  c.pos_stride = pos_stride;
  c.n_batch = n_batch;
  c.n_tokens = n_tokens;
  c.dim = dim;
  c.io = static_cast<aq::IoType>(io_type);
  c.backward = backward != 0;
  DeviceGuard g(r->device);
  if (hip_fail(aq::launch_rotary(r->table(), c, static_cast<hipStream_t>(stream)), fn)) return -1;
  aq::clear_error();
  return 0;
}

adaptq_paged_t adaptq_paged_create(void *d_k_pages, void *d_v_pages, int n_pages, int page_size,
                                   int n_heads, int dim, int io_type, adaptq_rotary_t rotary) {
  return create_paged(d_k_pages, d_v_pages, n_pages, page_size, n_heads, dim, io_type, rotary,
                      false, "adaptq_paged_create");
}

void adaptq_paged_destroy(adaptq_paged_t h) {
  if (!h) return;
  destroy_paged(static_cast<Paged *>(h));
}

int adaptq_paged_append_device(adaptq_paged_t h, const void *d_k, const void *d_v, int n_tokens,
                               size_t k_nb1, size_t k_nb2, size_t v_nb1, size_t v_nb2,
                               const int *d_table, int table_width, int table_stride,
                               const int *d_lengths, int n_seqs, const int *d_offsets,
                               void *stream) {
  const char *fn = "adaptq_paged_append_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!exact_pages(p, fn)) return -1;
  const size_t nb[4] = {k_nb1, k_nb2, v_nb1, v_nb2};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_append(p, d_k, d_v, n_tokens, nb, q, d_offsets, stream, fn);
}

int adaptq_paged_attend_device(adaptq_paged_t h, const void *d_q, void *d_out, int n_q_heads,
                               size_t q_nb1, size_t q_nb2, size_t out_nb1, size_t out_nb2,
                               const int *d_table, int table_width, int table_stride,
                               const int *d_lengths, int n_seqs, float scale, int window,
                               void *stream) {
  const char *fn = "adaptq_paged_attend_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!exact_pages(p, fn)) return -1;
  const Token t{nullptr, nullptr, {}, d_q, d_out, n_q_heads, {q_nb1, q_nb2, out_nb1, out_nb2},
                scale, window};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_token(p, t, q, nullptr, nullptr, stream, fn);
}

int adaptq_paged_step_device(adaptq_paged_t h, const void *d_k, const void *d_v, size_t k_nb1,
                             size_t k_nb2, size_t v_nb1, size_t v_nb2, const void *d_q,
                             void *d_out, int n_q_heads, size_t q_nb1, size_t q_nb2,
                             size_t out_nb1, size_t out_nb2, const int *d_table, int table_width,
                             int table_stride, const int *d_lengths, int n_seqs, float scale,
                             int window, void *stream) {
  const char *fn = "adaptq_paged_step_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!exact_pages(p, fn) || (n_seqs > 0 && !require_pointer(d_k, fn, "d_k"))) return -1;
  const Token t{d_k, d_v, {k_nb1, k_nb2, v_nb1, v_nb2}, d_q, d_out, n_q_heads,
                {q_nb1, q_nb2, out_nb1, out_nb2}, scale, window};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_token(p, t, q, nullptr, nullptr, stream, fn);
}

size_t adaptq_paged_weights_workspace(adaptq_paged_t h, int n_q_heads, int n_seqs,
                                      int table_width) {
  if (!h || n_q_heads <= 0 || n_seqs <= 0 || table_width < 0) return 0;
  const Paged *p = static_cast<Paged *>(h);
  return aq::paged_weights_workspace(p->shape, n_q_heads, n_seqs, table_width);
}

int adaptq_paged_attend_scores_device(adaptq_paged_t h, const void *d_q, void *d_out,
                                      int n_q_heads, size_t q_nb1, size_t q_nb2, size_t out_nb1,
                                      size_t out_nb2, const int *d_table, int table_width,
                                      int table_stride, const int *d_lengths, int n_seqs,
                                      float scale, const adaptq_scores_t *scores,
                                      float *d_weights, size_t w_nb1, size_t w_nb2,
                                      void *d_workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "adaptq_paged_attend_scores_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!exact_pages(p, fn)) return -1;
  const Token t{nullptr, nullptr, {}, d_q, d_out, n_q_heads, {q_nb1, q_nb2, out_nb1, out_nb2},
                scale, 0};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_scored(p, t, q, scores, d_weights, w_nb1, w_nb2, d_workspace, workspace_bytes,
                      stream, fn);
}

int adaptq_paged_step_scores_device(adaptq_paged_t h, const void *d_k, const void *d_v,
                                    size_t k_nb1, size_t k_nb2, size_t v_nb1, size_t v_nb2,
                                    const void *d_q, void *d_out, int n_q_heads, size_t q_nb1,
                                    size_t q_nb2, size_t out_nb1, size_t out_nb2,
                                    const int *d_table, int table_width, int table_stride,
                                    const int *d_lengths, int n_seqs, float scale,
                                    const adaptq_scores_t *scores, float *d_weights, size_t w_nb1,
                                    size_t w_nb2, void *d_workspace, size_t workspace_bytes,
                                    void *stream) {
  const char *fn = "adaptq_paged_step_scores_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!exact_pages(p, fn) || (n_seqs > 0 && !require_pointer(d_k, fn, "d_k"))) return -1;
  const Token t{d_k, d_v, {k_nb1, k_nb2, v_nb1, v_nb2}, d_q, d_out, n_q_heads,
                {q_nb1, q_nb2, out_nb1, out_nb2}, scale, 0};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_scored(p, t, q, scores, d_weights, w_nb1, w_nb2, d_workspace, workspace_bytes,
                      stream, fn);
}

int adaptq_paged_evict_device(adaptq_paged_t h, float *d_weights, size_t w_nb1, size_t w_nb2,
                              const int *d_table, int table_width, int table_stride,
                              const int *d_lengths, int n_seqs, int keep, int recent,
                              const int *d_into, int into_width, int into_stride, int *d_kept,
                              void *stream) {
  const char *fn = "adaptq_paged_evict_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!exact_pages(p, fn)) return -1;
  if (p->shape.rotary.pairs) {
    set_errorf(fn, "a cache with a rotary takes positions from its lengths, which eviction changes");
    return -1;
  }
  if (keep <= 0 || recent < 0 || recent > keep) {
    set_errorf(fn, "keep must be positive, recent from 0 to keep");
    return -1;
  }
  if (!seqs_ok(d_table, table_width, table_stride, d_lengths, n_seqs, fn)) return -1;
  if (d_into && (into_width < 0 || into_stride < into_width)) {
    set_errorf(fn, "into_stride is smaller than into_width, or one is negative");
    return -1;
  }
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  aq::PagedWeights w;
  if (n_seqs == 0) {
    aq::clear_error();
    return 0;
  }
  if (!require_pointer(d_weights, fn, "d_weights") || !require_pointer(d_kept, fn, "d_kept") ||
      !aligned_to(d_kept, 4, fn) || !aligned_to(d_into, 4, fn) ||
      !weights_ok(p, d_weights, w_nb1, w_nb2, q, &w, fn))
    return -1;
  if ((size_t)n_seqs * p->shape.n_heads > ((size_t)1 << 58) / (size_t)keep) {
    set_errorf(fn, "d_kept is too large");
    return -1;
  }
  const aq::PagedEvict e{w.weights, {w.nb[0], w.nb[1]}, keep, recent,
                         d_into, into_width, into_stride, d_kept};
  DeviceGuard g(p->device);
  if (hip_fail(aq::launch_paged_evict(p->shape, q, e, static_cast<hipStream_t>(stream)), fn))
    return -1;
  aq::clear_error();
  return 0;
}

adaptq_paged4_t adaptq_paged4_create(void *d_k_pages, void *d_v_pages, int n_pages, int page_size,
                                     int n_heads, int dim, int io_type, adaptq_rotary_t rotary) {
  return create_paged(d_k_pages, d_v_pages, n_pages, page_size, n_heads, dim, io_type, rotary,
                      true, "adaptq_paged4_create");
}

void adaptq_paged4_destroy(adaptq_paged4_t h) {
  if (h) destroy_paged(static_cast<Paged *>(h));
}

int adaptq_paged4_append_device(adaptq_paged4_t h, const void *d_k, const void *d_v, int n_tokens,
                                size_t k_nb1, size_t k_nb2, size_t v_nb1, size_t v_nb2,
                                const int *d_table, int table_width, int table_stride,
                                const int *d_lengths, int n_seqs, const int *d_offsets,
                                void *stream) {
  const char *fn = "adaptq_paged4_append_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!four_bits(p, fn)) return -1;
  const size_t nb[4] = {k_nb1, k_nb2, v_nb1, v_nb2};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_append(p, d_k, d_v, n_tokens, nb, q, d_offsets, stream, fn);
}

int adaptq_paged4_read_device(adaptq_paged4_t h, float *d_k, float *d_v, int n_tokens,
                              const int *d_table, int table_width, int table_stride,
                              const int *d_lengths, int n_seqs, const int *d_offsets,
                              void *stream) {
  const char *fn = "adaptq_paged4_read_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!four_bits(p, fn)) return -1;
  if (n_tokens < 0) {
    set_errorf(fn, "negative n_tokens");
    return -1;
  }
  if (!seqs_ok(d_table, table_width, table_stride, d_lengths, n_seqs, fn)) return -1;
  if (!d_offsets && n_tokens != n_seqs) {
    set_errorf(fn, "without d_offsets, n_tokens must be n_seqs (one token a sequence)");
    return -1;
  }
  if (n_tokens == 0 || n_seqs == 0) {
    aq::clear_error();
    return 0;
  }
  if (!require_pointer(d_k, fn, "d_k") || !require_pointer(d_v, fn, "d_v") ||
      !aligned_to(d_k, 16, fn) || !aligned_to(d_v, 16, fn) || !aligned_to(d_offsets, 4, fn))
    return -1;
  const size_t bytes = (size_t)n_tokens * p->shape.n_heads * p->shape.dim * 4;
  const uintptr_t k = reinterpret_cast<uintptr_t>(d_k), v = reinterpret_cast<uintptr_t>(d_v);
  if (k < v + bytes && v < k + bytes) {
    set_errorf(fn, "d_k and d_v overlap");
    return -1;
  }
  for (const uintptr_t x : {k, v})
    for (const void *pool : {p->shape.k_pages, p->shape.v_pages}) {
      const uintptr_t lo = reinterpret_cast<uintptr_t>(pool);
      if (x < lo + p->pool && lo < x + bytes) {
        set_errorf(fn, "rows overlap the pages");
        return -1;
      }
    }
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  DeviceGuard g(p->device);
  if (hip_fail(aq::launch_paged4_read(p->shape, q, n_tokens, d_offsets, d_k, d_v,
                                      static_cast<hipStream_t>(stream)),
               fn))
    return -1;
  aq::clear_error();
  return 0;
}

int adaptq_paged4_attend_device(adaptq_paged4_t h, const void *d_q, void *d_out, int n_q_heads,
                                size_t q_nb1, size_t q_nb2, size_t out_nb1, size_t out_nb2,
                                const int *d_table, int table_width, int table_stride,
                                const int *d_lengths, int n_seqs, float scale,
                                const adaptq_scores_t *scores, void *stream) {
  const char *fn = "adaptq_paged4_attend_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!four_bits(p, fn)) return -1;
  const Token t{nullptr, nullptr, {}, d_q, d_out, n_q_heads, {q_nb1, q_nb2, out_nb1, out_nb2},
                scale, 0};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_scored(p, t, q, scores, nullptr, 0, 0, nullptr, 0, stream, fn);
}

int adaptq_paged4_step_device(adaptq_paged4_t h, const void *d_k, const void *d_v, size_t k_nb1,
                              size_t k_nb2, size_t v_nb1, size_t v_nb2, const void *d_q,
                              void *d_out, int n_q_heads, size_t q_nb1, size_t q_nb2,
                              size_t out_nb1, size_t out_nb2, const int *d_table, int table_width,
                              int table_stride, const int *d_lengths, int n_seqs, float scale,
                              const adaptq_scores_t *scores, void *stream) {
  const char *fn = "adaptq_paged4_step_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!four_bits(p, fn) || (n_seqs > 0 && !require_pointer(d_k, fn, "d_k"))) return -1;
  const Token t{d_k, d_v, {k_nb1, k_nb2, v_nb1, v_nb2}, d_q, d_out, n_q_heads,
                {q_nb1, q_nb2, out_nb1, out_nb2}, scale, 0};
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  return paged_scored(p, t, q, scores, nullptr, 0, 0, nullptr, 0, stream, fn);
}

size_t adaptq_paged_prompt_workspace(adaptq_paged_t h, int n_q_heads, int n_tokens, int n_seqs,
                                     int table_width) {
  if (!h || n_q_heads <= 0 || n_tokens <= 0 || n_seqs <= 0 || table_width < 0) return 0;
  const Paged *p = static_cast<Paged *>(h);
  if (n_q_heads % p->shape.n_heads) return 0;
  return aq::paged_prompt_workspace(p->shape, n_q_heads, n_tokens, n_seqs, table_width);
}

size_t adaptq_paged_prompt_scores_workspace(adaptq_paged_t h, int n_q_heads, int n_tokens,
                                            int n_seqs, int table_width,
                                            const adaptq_scores_t *scores) {
  if (!h || n_q_heads <= 0 || n_tokens <= 0 || n_seqs <= 0 || table_width < 0) return 0;
  const Paged *p = static_cast<Paged *>(h);
  if (n_q_heads % p->shape.n_heads) return 0;
  aq::PagedPrompt a{};
  a.q_heads = n_q_heads;
  a.n_tokens = n_tokens;
  if (scores) a.scores = {0.0f, scores->window, nullptr, scores->d_prefix, scores->d_first};
  if (few_queries(p, a, n_seqs)) return 0;
  return aq::paged_prompt_workspace(p->shape, n_q_heads, n_tokens, n_seqs, table_width);
}

int adaptq_paged_prompt_device(adaptq_paged_t h, const void *d_q, void *d_out, int n_q_heads,
                               int n_tokens, size_t q_nb1, size_t q_nb2, size_t out_nb1,
                               size_t out_nb2, const int *d_table, int table_width,
                               int table_stride, const int *d_lengths, int n_seqs,
                               const int *d_offsets, float scale, const adaptq_scores_t *scores,
                               void *d_workspace, size_t workspace_bytes, void *stream) {
  const char *fn = "adaptq_paged_prompt_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  if (!exact_pages(p, fn)) return -1;
  if (n_tokens < 0) {
    set_errorf(fn, "negative n_tokens");
    return -1;
  }
  const size_t nb[4] = {q_nb1, q_nb2, out_nb1, out_nb2};
  aq::PagedPrompt a{};
  if (!seqs_ok(d_table, table_width, table_stride, d_lengths, n_seqs, fn) ||
      !attend_ok(p, d_q, d_out, n_q_heads, n_tokens, nb, scale, 0, fn) ||
      !scores_ok(scores, scale_of(p, scale), &a.scores, fn))
    return -1;
  if (n_tokens == 0 || n_seqs == 0) {
    aq::clear_error();
    return 0;
  }
  if (!require_pointer(d_offsets, fn, "d_offsets") || !aligned_to(d_offsets, 4, fn) ||
      !out_apart(p, d_out, n_q_heads, out_nb1, out_nb2, d_q, n_q_heads, q_nb1, q_nb2, n_tokens,
                 fn))
    return -1;
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  a.q = d_q;
  a.out = d_out;
  a.q_nb[0] = q_nb1;
  a.q_nb[1] = q_nb2;
  a.out_nb[0] = out_nb1;
  a.out_nb[1] = out_nb2;
  a.q_heads = n_q_heads;
  a.n_tokens = n_tokens;
  a.offsets = d_offsets;
  a.scale = scale_of(p, scale);
  const bool few = few_queries(p, a, n_seqs);
  if (!few && !workspace_ok(d_workspace, workspace_bytes,
                            aq::paged_prompt_workspace(p->shape, n_q_heads, n_tokens, n_seqs,
                                                       table_width),
                            fn))
    return -1;
  DeviceGuard g(p->device);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (hip_fail(few ? aq::launch_paged_few(p->shape, q, a, p->ws, s)
                   : aq::launch_paged_prompt(p->shape, q, a, d_workspace, s),
               fn))
    return -1;
  aq::clear_error();
  return 0;
}

}  // extern "C"
