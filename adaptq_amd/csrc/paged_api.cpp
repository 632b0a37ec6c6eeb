// paged_api.cpp -- the C ABI of the rotary positions and of the paged cache
// (include/adaptq.h, part 3): argument checks, handles, launches.
//
// Nothing here synchronises or allocates after a handle's creation: every call is
// one launch on the caller's stream and may be captured into a graph.
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
};

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
  const Span x = span_of(rows, row, counts, nb, 2);
  const size_t pool = row * s.page_size * s.n_heads * (size_t)s.n_pages;
  for (const void *q : {s.k_pages, s.v_pages}) {
    const uintptr_t lo = reinterpret_cast<uintptr_t>(q);
    if (x.lo < lo + pool && lo < x.hi) {
      set_errorf(fn, "rows overlap the pages");
      return false;
    }
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
  a.scale = scale != 0.0f ? scale : (float)(1.0 / std::sqrt((double)p->shape.dim));
  a.window = window;
  a.extra = extra;
  return a;
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
  const char *fn = "adaptq_paged_create";
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
  if (dim <= 0 || dim % 8 || dim > kMaxPagedDim) {
    set_errorf(fn, "dim must be a multiple of 8 up to 256");
    return nullptr;
  }
  if (!aligned_to(d_k_pages, 16, fn) || !aligned_to(d_v_pages, 16, fn)) {
    set_errorf(fn, "pages must be aligned to 16 bytes");
    return nullptr;
  }
  const size_t page = size_of(io_type) * dim * page_size * (size_t)n_heads;
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
    adaptq_paged_destroy(p);
    return nullptr;
  }
  aq::clear_error();
  return p;
}

void adaptq_paged_destroy(adaptq_paged_t h) {
  if (!h) return;
  Paged *p = static_cast<Paged *>(h);
  DeviceGuard g(p->device);
  if (p->d_steps) (void)hipFree(p->d_steps);  // waits for the device
  if (p->ws) (void)hipFree(p->ws);
  delete p;
}

int adaptq_paged_append_device(adaptq_paged_t h, const void *d_k, const void *d_v, int n_tokens,
                               size_t k_nb1, size_t k_nb2, size_t v_nb1, size_t v_nb2,
                               const int *d_table, int table_width, int table_stride,
                               const int *d_lengths, int n_seqs, const int *d_offsets,
                               void *stream) {
  const char *fn = "adaptq_paged_append_device";
  if (!require_handle(h, fn)) return -1;
  const Paged *p = static_cast<Paged *>(h);
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
  const size_t nb[4] = {k_nb1, k_nb2, v_nb1, v_nb2};
  if (!append_ok(p, d_k, d_v, n_tokens, nb, fn)) return -1;
  if (d_offsets && !aligned_to(d_offsets, 4, fn)) return -1;
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  const aq::PagedAppend a{d_k, d_v, {k_nb1, k_nb2}, {v_nb1, v_nb2}, n_tokens, d_offsets};
  DeviceGuard g(p->device);
  if (hip_fail(aq::launch_paged_append(p->shape, q, a, static_cast<hipStream_t>(stream)), fn))
    return -1;
  aq::clear_error();
  return 0;
}

int adaptq_paged_attend_device(adaptq_paged_t h, const void *d_q, void *d_out, int n_q_heads,
                               size_t q_nb1, size_t q_nb2, size_t out_nb1, size_t out_nb2,
                               const int *d_table, int table_width, int table_stride,
                               const int *d_lengths, int n_seqs, float scale, int window,
                               void *stream) {
  const char *fn = "adaptq_paged_attend_device";
  if (!require_handle(h, fn)) return -1;
  Paged *p = static_cast<Paged *>(h);
  const size_t nb[4] = {q_nb1, q_nb2, out_nb1, out_nb2};
  if (!seqs_ok(d_table, table_width, table_stride, d_lengths, n_seqs, fn) ||
      !attend_ok(p, d_q, d_out, n_q_heads, n_seqs, nb, scale, window, fn))
    return -1;
  if (n_seqs == 0) {
    aq::clear_error();
    return 0;
  }
  if (!out_apart(p, d_out, n_q_heads, out_nb1, out_nb2, d_q, n_q_heads, q_nb1, q_nb2, n_seqs, fn))
    return -1;
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  const aq::PagedAttend a =
      attend_args(p, d_q, d_out, n_q_heads, q_nb1, q_nb2, out_nb1, out_nb2, scale, window, 0);
  DeviceGuard g(p->device);
  if (hip_fail(aq::launch_paged_attend(p->shape, q, a, nullptr, p->ws, static_cast<hipStream_t>(stream)),
               fn))
    return -1;
  aq::clear_error();
  return 0;
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
  const size_t knb[4] = {k_nb1, k_nb2, v_nb1, v_nb2}, qnb[4] = {q_nb1, q_nb2, out_nb1, out_nb2};
  if (!seqs_ok(d_table, table_width, table_stride, d_lengths, n_seqs, fn) ||
      !attend_ok(p, d_q, d_out, n_q_heads, n_seqs, qnb, scale, window, fn))
    return -1;
  if (n_seqs == 0) {
    aq::clear_error();
    return 0;
  }
  const int H = p->shape.n_heads;
  if (!append_ok(p, d_k, d_v, n_seqs, knb, fn) ||
      !out_apart(p, d_out, n_q_heads, out_nb1, out_nb2, d_q, n_q_heads, q_nb1, q_nb2, n_seqs, fn) ||
      !out_apart(p, d_out, n_q_heads, out_nb1, out_nb2, d_k, H, k_nb1, k_nb2, n_seqs, fn) ||
      !out_apart(p, d_out, n_q_heads, out_nb1, out_nb2, d_v, H, v_nb1, v_nb2, n_seqs, fn))
    return -1;
  const aq::PagedSeqs q{d_table, table_width, table_stride, d_lengths, n_seqs};
  const aq::PagedAppend ap{d_k, d_v, {k_nb1, k_nb2}, {v_nb1, v_nb2}, n_seqs, nullptr};
  const aq::PagedAttend a =
      attend_args(p, d_q, d_out, n_q_heads, q_nb1, q_nb2, out_nb1, out_nb2, scale, window, 1);
  DeviceGuard g(p->device);
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (hip_fail(aq::launch_paged_attend(p->shape, q, a, &ap, p->ws, s), fn)) return -1;
  aq::clear_error();
  return 0;
}

}  // extern "C"
