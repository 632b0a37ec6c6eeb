// adapter_python.cpp -- pybind11 module `adaptq_py` over the C ABI.
//
// Same Python surface as the reference's adapters/adapter_python.cpp:30-93:
// class MHAContext(n_heads, head_dim, k_bits, v_bits, capacity, seed=0,
// v_mass=0.95, hybrid_thresh=512) with append / compute / compute_batch /
// reset / kv_bytes and the n_heads / head_dim properties, so the reference's
// adaptq.Engine runs on it unchanged.  Creation failure raises RuntimeError
// with adaptq_last_error() (the reference would carry a NULL handle on).
#include <pybind11/numpy.h>
#include <pybind11/pybind11.h>
#include <cstdint>

#include <stdexcept>
#include <string>

#include "adaptq_mha_backend.h"

namespace py = pybind11;

namespace {

using farray = py::array_t<float, py::array::c_style | py::array::forcecast>;

class PyMHAContext {
 public:
  PyMHAContext(int n_heads, int head_dim, int k_bits, int v_bits, int capacity,
               uint64_t seed, float v_mass, int hybrid_thresh)
      : backend_(n_heads, head_dim, k_bits, v_bits, capacity, seed, v_mass, hybrid_thresh),
        head_dim_(head_dim),
        n_heads_(n_heads) {
    if (!backend_.ok()) throw std::runtime_error(std::string(adaptq_last_error()));
  }

  void append(int head, farray key, farray val, int pos) {
    if (key.ndim() != 1 || val.ndim() != 1 || key.shape(0) != head_dim_ ||
        val.shape(0) != head_dim_)
      throw std::invalid_argument("key/val dim mismatch");
    backend_.append_kv(head, key.data(), val.data(), pos);
  }

  farray compute(int head, farray query) {
    if (query.ndim() != 1 || query.shape(0) != head_dim_)
      throw std::invalid_argument("query dim mismatch");
    farray out(head_dim_);
    backend_.compute(head, query.data(), out.mutable_data());
    return out;
  }

  farray compute_batch(int head, farray queries) {
    if (queries.ndim() != 2 || queries.shape(1) != head_dim_)
      throw std::invalid_argument("queries dim mismatch");
    const int nq = (int)queries.shape(0);
    farray out({nq, head_dim_});
    backend_.compute_batch(head, queries.data(), nq, out.mutable_data());
    return out;
  }

  // Whole-MHA forms (adaptq_mha_append_all / _compute_all): one call for all
  // heads instead of the reference Engine's per-head loop.
  void append_all(farray keys, farray vals, int pos) {
    if (keys.ndim() != 2 || vals.ndim() != 2 || keys.shape(0) != n_heads_ ||
        vals.shape(0) != n_heads_ || keys.shape(1) != head_dim_ || vals.shape(1) != head_dim_)
      throw std::invalid_argument("keys/vals must be (n_heads, head_dim)");
    if (adaptq_mha_append_all(backend_.handle(), keys.data(), vals.data(), pos) != 0)
      throw std::runtime_error(adaptq_last_error());
  }

  farray compute_all(farray queries) {
    if (queries.ndim() != 2 || queries.shape(0) != n_heads_ || queries.shape(1) != head_dim_)
      throw std::invalid_argument("queries must be (n_heads, head_dim)");
    farray out({n_heads_, head_dim_});
    if (adaptq_mha_compute_all(backend_.handle(), queries.data(), out.mutable_data()) < 0)
      throw std::runtime_error(adaptq_last_error());
    return out;
  }

  // Device pointers (torch-ROCm tensors' data_ptr()), asynchronous on stream.
  void append_all_device(uintptr_t d_keys, uintptr_t d_vals, int n_tokens, int pos,
                         uintptr_t stream) {
    if (adaptq_mha_append_all_device(backend_.handle(), reinterpret_cast<const float *>(d_keys),
                                     reinterpret_cast<const float *>(d_vals), n_tokens, pos,
                                     reinterpret_cast<void *>(stream)) != 0)
      throw std::runtime_error(adaptq_last_error());
  }

  int compute_all_device(uintptr_t d_queries, uintptr_t d_outs, uintptr_t stream) {
    const int n = adaptq_mha_compute_all_device(
        backend_.handle(), reinterpret_cast<const float *>(d_queries),
        reinterpret_cast<float *>(d_outs), reinterpret_cast<void *>(stream));
    if (n < 0) throw std::runtime_error(adaptq_last_error());
    return n;
  }

  // Append one token and decode one query for every head (rows of io_type).
  int step_device(uintptr_t d_keys, uintptr_t d_vals, uintptr_t d_queries, uintptr_t d_outs,
                  int io_type, int pos, uintptr_t stream) {
    const int n = adaptq_mha_step_device(
        backend_.handle(), reinterpret_cast<const void *>(d_keys),
        reinterpret_cast<const void *>(d_vals), reinterpret_cast<const void *>(d_queries),
        reinterpret_cast<void *>(d_outs), io_type, pos, reinterpret_cast<void *>(stream));
    if (n < 0) throw std::runtime_error(adaptq_last_error());
    return n;
  }

  void reset() { backend_.reset(); }
  size_t kv_bytes() const { return backend_.kv_bytes(); }
  int n_heads() const { return n_heads_; }
  int head_dim() const { return head_dim_; }

 private:
  AdaptQMHABackend backend_;
  int head_dim_, n_heads_;
};

// Handles of the rotary positions and the paged cache; addresses are device
// pointers (torch-ROCm tensors' data_ptr()), strides bytes.
using addr = uintptr_t;

void *ptr(addr a) { return reinterpret_cast<void *>(a); }
const float *floats(addr a) { return reinterpret_cast<const float *>(a); }
const int *ints(addr a) { return reinterpret_cast<const int *>(a); }
void check(int rc) {
  if (rc != 0) throw std::runtime_error(adaptq_last_error());
}

class PyRotary {
 public:
  PyRotary(int dim, bool interleaved, double base, int scaling, double factor, int context,
           double slow, double fast, double amplitude)
      : h_(adaptq_rotary_create(dim, interleaved, base, scaling, factor, context, slow, fast,
                                amplitude)) {
    if (!h_) throw std::runtime_error(adaptq_last_error());
  }
  ~PyRotary() { adaptq_rotary_destroy(h_); }
  PyRotary(const PyRotary &) = delete;
  PyRotary &operator=(const PyRotary &) = delete;
  adaptq_rotary_t handle() const { return h_; }

  void rotate(addr positions, size_t pos_stride, int n_batch, int n_tokens, int dim, int io,
              bool backward, addr stream, addr q, addr q_out, int q_heads, size_t q1, size_t q2,
              size_t q3, size_t qo1, size_t qo2, size_t qo3, addr k, addr k_out, int k_heads,
              size_t k1, size_t k2, size_t k3, size_t ko1, size_t ko2, size_t ko3) {
    const adaptq_rows_t rows[2] = {{ptr(q), ptr(q_out), q_heads, q1, q2, q3, qo1, qo2, qo3},
                                   {ptr(k), ptr(k_out), k_heads, k1, k2, k3, ko1, ko2, ko3}};
    check(adaptq_rotary_device(h_, rows, k ? 2 : 1, dim, io, ints(positions), pos_stride, n_batch,
                               n_tokens, backward, ptr(stream)));
  }

 private:
  adaptq_rotary_t h_;
};

class PyPagedCache {
 public:
  PyPagedCache(addr k_pages, addr v_pages, int n_pages, int page_size, int n_heads, int dim,
               int io, const PyRotary *rotary)
      : h_(adaptq_paged_create(ptr(k_pages), ptr(v_pages), n_pages, page_size, n_heads, dim, io,
                               rotary ? rotary->handle() : nullptr)) {
    if (!h_) throw std::runtime_error(adaptq_last_error());
  }
  ~PyPagedCache() { adaptq_paged_destroy(h_); }
  PyPagedCache(const PyPagedCache &) = delete;
  PyPagedCache &operator=(const PyPagedCache &) = delete;

  void append(addr k, addr v, int n_tokens, size_t k1, size_t k2, size_t v1, size_t v2, addr table,
              int width, int stride, addr lengths, int n_seqs, addr offsets, addr stream) {
    check(adaptq_paged_append_device(h_, ptr(k), ptr(v), n_tokens, k1, k2, v1, v2, ints(table),
                                     width, stride, ints(lengths), n_seqs, ints(offsets),
                                     ptr(stream)));
  }
  void attend(addr q, addr out, int q_heads, size_t q1, size_t q2, size_t o1, size_t o2,
              addr table, int width, int stride, addr lengths, int n_seqs, float scale, int window,
              addr stream) {
    check(adaptq_paged_attend_device(h_, ptr(q), ptr(out), q_heads, q1, q2, o1, o2, ints(table),
                                     width, stride, ints(lengths), n_seqs, scale, window,
                                     ptr(stream)));
  }
  size_t prompt_workspace(int q_heads, int n_tokens, int n_seqs, int width, int window, addr prefix,
                          addr first) {
    const adaptq_scores_t s = {0, window, nullptr, ints(prefix), ints(first)};
    return adaptq_paged_prompt_scores_workspace(h_, q_heads, n_tokens, n_seqs, width, &s);
  }
  void prompt(addr q, addr out, int q_heads, size_t q1, size_t q2, size_t o1, size_t o2,
              int n_tokens, addr table, int width, int stride, addr lengths, int n_seqs,
              addr offsets, float scale, int window, float softcap, addr slopes, addr prefix,
              addr first, addr workspace, size_t bytes, addr stream) {
    const adaptq_scores_t s = {softcap, window, floats(slopes), ints(prefix), ints(first)};
    check(adaptq_paged_prompt_device(h_, ptr(q), ptr(out), q_heads, n_tokens, q1, q2, o1, o2,
                                     ints(table), width, stride, ints(lengths), n_seqs,
                                     ints(offsets), scale, &s, ptr(workspace), bytes, ptr(stream)));
  }
  void step(addr k, addr v, size_t k1, size_t k2, size_t v1, size_t v2, addr q, addr out,
            int q_heads, size_t q1, size_t q2, size_t o1, size_t o2, addr table, int width,
            int stride, addr lengths, int n_seqs, float scale, int window, addr stream) {
    check(adaptq_paged_step_device(h_, ptr(k), ptr(v), k1, k2, v1, v2, ptr(q), ptr(out), q_heads,
                                   q1, q2, o1, o2, ints(table), width, stride, ints(lengths),
                                   n_seqs, scale, window, ptr(stream)));
  }

  size_t weights_workspace(int q_heads, int n_seqs, int width) {
    return adaptq_paged_weights_workspace(h_, q_heads, n_seqs, width);
  }
  // attend and step (k not 0) with scores of their own
  void scored(addr k, addr v, size_t k1, size_t k2, size_t v1, size_t v2, addr q, addr out,
              int q_heads, size_t q1, size_t q2, size_t o1, size_t o2, addr table, int width,
              int stride, addr lengths, int n_seqs, float scale, int window, float softcap,
              addr slopes, addr prefix, addr first, addr weights, size_t w1, size_t w2,
              addr workspace, size_t bytes, addr stream) {
    const adaptq_scores_t s = {softcap, window, floats(slopes), ints(prefix), ints(first)};
    float *w = reinterpret_cast<float *>(weights);
    if (k)
      check(adaptq_paged_step_scores_device(h_, ptr(k), ptr(v), k1, k2, v1, v2, ptr(q), ptr(out),
                                            q_heads, q1, q2, o1, o2, ints(table), width, stride,
                                            ints(lengths), n_seqs, scale, &s, w, w1, w2,
                                            ptr(workspace), bytes, ptr(stream)));
    else
      check(adaptq_paged_attend_scores_device(h_, ptr(q), ptr(out), q_heads, q1, q2, o1, o2,
                                              ints(table), width, stride, ints(lengths), n_seqs,
                                              scale, &s, w, w1, w2, ptr(workspace), bytes,
                                              ptr(stream)));
  }
  void evict(addr weights, size_t w1, size_t w2, addr table, int width, int stride, addr lengths,
             int n_seqs, int keep, int recent, addr into, int into_width, int into_stride,
             addr kept, addr stream) {
    check(adaptq_paged_evict_device(h_, reinterpret_cast<float *>(weights), w1, w2, ints(table),
                                    width, stride, ints(lengths), n_seqs, keep, recent, ints(into),
                                    into_width, into_stride, reinterpret_cast<int *>(kept),
                                    ptr(stream)));
  }

 private:
  adaptq_paged_t h_;
};

class PyPagedCache4 {
 public:
  PyPagedCache4(addr k_pages, addr v_pages, int n_pages, int page_size, int n_heads, int dim,
                int io, const PyRotary *rotary)
      : h_(adaptq_paged4_create(ptr(k_pages), ptr(v_pages), n_pages, page_size, n_heads, dim, io,
                                rotary ? rotary->handle() : nullptr)) {
    if (!h_) throw std::runtime_error(adaptq_last_error());
  }
  ~PyPagedCache4() { adaptq_paged4_destroy(h_); }
  PyPagedCache4(const PyPagedCache4 &) = delete;
  PyPagedCache4 &operator=(const PyPagedCache4 &) = delete;

  void append(addr k, addr v, int n_tokens, size_t k1, size_t k2, size_t v1, size_t v2, addr table,
              int width, int stride, addr lengths, int n_seqs, addr offsets, addr stream) {
    check(adaptq_paged4_append_device(h_, ptr(k), ptr(v), n_tokens, k1, k2, v1, v2, ints(table),
                                      width, stride, ints(lengths), n_seqs, ints(offsets),
                                      ptr(stream)));
  }
  void read(addr k, addr v, int n_tokens, addr table, int width, int stride, addr lengths,
            int n_seqs, addr offsets, addr stream) {
    check(adaptq_paged4_read_device(h_, reinterpret_cast<float *>(k), reinterpret_cast<float *>(v),
                                    n_tokens, ints(table), width, stride, ints(lengths), n_seqs,
                                    ints(offsets), ptr(stream)));
  }
  // attend and step (k not 0)
  void scored(addr k, addr v, size_t k1, size_t k2, size_t v1, size_t v2, addr q, addr out,
              int q_heads, size_t q1, size_t q2, size_t o1, size_t o2, addr table, int width,
              int stride, addr lengths, int n_seqs, float scale, int window, float softcap,
              addr slopes, addr prefix, addr first, addr stream) {
    const adaptq_scores_t s = {softcap, window, floats(slopes), ints(prefix), ints(first)};
    if (k)
      check(adaptq_paged4_step_device(h_, ptr(k), ptr(v), k1, k2, v1, v2, ptr(q), ptr(out),
                                      q_heads, q1, q2, o1, o2, ints(table), width, stride,
                                      ints(lengths), n_seqs, scale, &s, ptr(stream)));
    else
      check(adaptq_paged4_attend_device(h_, ptr(q), ptr(out), q_heads, q1, q2, o1, o2, ints(table),
                                        width, stride, ints(lengths), n_seqs, scale, &s,
                                        ptr(stream)));
  }

 private:
  adaptq_paged4_t h_;
};

}  // namespace

PYBIND11_MODULE(adaptq_py, m) {
  m.doc() = "AdapTQ quantised KV-cache attention on gfx950 (HIP)";
  py::class_<PyMHAContext>(m, "MHAContext")
      .def(py::init<int, int, int, int, int, uint64_t, float, int>(), py::arg("n_heads"),
           py::arg("head_dim"), py::arg("k_bits"), py::arg("v_bits"), py::arg("capacity"),
           py::arg("seed") = 0, py::arg("v_mass") = 0.95f, py::arg("hybrid_thresh") = 512)
      .def("append", &PyMHAContext::append, py::arg("head"), py::arg("key"), py::arg("val"),
           py::arg("pos"))
      .def("compute", &PyMHAContext::compute, py::arg("head"), py::arg("query"))
      .def("compute_batch", &PyMHAContext::compute_batch, py::arg("head"), py::arg("queries"))
      .def("append_all", &PyMHAContext::append_all, py::arg("keys"), py::arg("vals"),
           py::arg("pos") = 0)
      .def("compute_all", &PyMHAContext::compute_all, py::arg("queries"))
      .def("append_all_device", &PyMHAContext::append_all_device, py::arg("d_keys"),
           py::arg("d_vals"), py::arg("n_tokens"), py::arg("pos"), py::arg("stream"))
      .def("compute_all_device", &PyMHAContext::compute_all_device, py::arg("d_queries"),
           py::arg("d_outs"), py::arg("stream"))
      .def("step_device", &PyMHAContext::step_device, py::arg("d_keys"), py::arg("d_vals"),
           py::arg("d_queries"), py::arg("d_outs"), py::arg("io_type"), py::arg("pos"),
           py::arg("stream"))
      .def("reset", &PyMHAContext::reset)
      .def("kv_bytes", &PyMHAContext::kv_bytes)
      .def_property_readonly("n_heads", &PyMHAContext::n_heads)
      .def_property_readonly("head_dim", &PyMHAContext::head_dim);

  // what adaptq_amd.rotary and adaptq_amd.paged call, in the order of their arguments
  py::class_<PyRotary>(m, "Rotary")
      .def(py::init<int, bool, double, int, double, int, double, double, double>())
      .def("rotate", &PyRotary::rotate)
      .def("rotate", [](PyRotary &r, addr positions, size_t pos_stride, int n_batch, int n_tokens,
                        int dim, int io, bool backward, addr stream, addr q, addr q_out,
                        int q_heads, size_t q1, size_t q2, size_t q3, size_t qo1, size_t qo2,
                        size_t qo3) {
        r.rotate(positions, pos_stride, n_batch, n_tokens, dim, io, backward, stream, q, q_out,
                 q_heads, q1, q2, q3, qo1, qo2, qo3, 0, 0, 0, 0, 0, 0, 0, 0, 0);
      });
  py::class_<PyPagedCache>(m, "PagedCache")
      .def(py::init<addr, addr, int, int, int, int, int, const PyRotary *>())
      .def("append", &PyPagedCache::append)
      .def("attend", &PyPagedCache::attend)
      .def("prompt_workspace", &PyPagedCache::prompt_workspace)
      .def("prompt", &PyPagedCache::prompt)
      .def("step", &PyPagedCache::step)
      .def("weights_workspace", &PyPagedCache::weights_workspace)
      .def("scored", &PyPagedCache::scored)
      .def("evict", &PyPagedCache::evict);
  py::class_<PyPagedCache4>(m, "PagedCache4")
      .def(py::init<addr, addr, int, int, int, int, int, const PyRotary *>())
      .def("append", &PyPagedCache4::append)
      .def("read", &PyPagedCache4::read)
      .def("scored", &PyPagedCache4::scored);
}
