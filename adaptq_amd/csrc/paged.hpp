// paged.hpp -- host-side launchers of the rotary and paged-cache kernels
// (rotary.hip, paged.hip).  All are asynchronous on the given stream and return
// the HIP launch status.
#pragma once

#include <algorithm>

#include "launch.hpp"

namespace aq {

// A kernel over `tokens` tokens, tokens_per_block of them a block of 256 threads:
// launch(first token, blocks), in one launch but for the most tokens, as a launch has at most
// 2^32 - 1 threads.
template <typename Launch>
hipError_t launch_over_tokens(int tokens, int tokens_per_block, Launch launch) {
  constexpr int64_t kMost = (((int64_t)1 << 32) - 1) / 256;
  const int64_t blocks = ((int64_t)tokens + tokens_per_block - 1) / tokens_per_block;
  for (int64_t b = 0; b < blocks; b += kMost) {
    launch((int)(b * tokens_per_block), (int)std::min(kMost, blocks - b));
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// A rotation, its per-pair steps (see rotary.hpp) in device memory.
struct RotaryTable {
  const uint64_t *steps;  // [pairs]; pairs 0: no rotation
  int pairs;
  bool interleaved;
  float amplitude;
};

struct RotaryRows {
  const void *in;
  void *out;
  int n_heads;
  size_t in_nb[3], out_nb[3];  // byte strides between heads, tokens, batches
};

struct RotaryCall {
  RotaryRows rows[2];
  int n_rows;
  const int *positions;
  size_t pos_stride;
  int n_batch, n_tokens, dim;
  IoType io;
  bool backward;
};

hipError_t launch_rotary(const RotaryTable &t, const RotaryCall &c, hipStream_t s);

// The pages of a cache: [n_pages][n_heads][page_size][dim] of io, keys and values.
struct PagedShape {
  void *k_pages, *v_pages;
  int n_pages, page_size, n_heads, dim;
  IoType io;
  RotaryTable rotary;
  int cus;  // compute units of the device
};

// Which pages a sequence's tokens lie in, and how many it holds.
struct PagedSeqs {
  const int *table;  // [n_seqs] rows of `width` page numbers, `stride` apart
  int width, stride;
  const int *lengths;
  int n_seqs;
};

struct PagedAppend {
  const void *k, *v;
  size_t k_nb[2], v_nb[2];  // byte strides between heads, tokens
  int n_tokens;
  const int *offsets;  // [n_seqs + 1], or null: one token a sequence
};

hipError_t launch_paged_append(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a,
                               hipStream_t s);

struct PagedAttend {
  const void *q;
  void *out;
  size_t q_nb[2], out_nb[2];
  int q_heads;
  float scale;
  int window;  // 0: all tokens
  int extra;   // tokens beyond `lengths` that a sequence holds by now
};

// What happens to scores on their way into the softmax, and which tokens a query at position p
// of n tokens sees: first <= t < n and (t < prefix or p - window < t <= p).
struct PagedScores {
  float softcap;        // 0: none
  int window;           // 0: all tokens
  const float *slopes;  // [q_heads], of the distance; null: none
  const int *prefix;    // of each query; null: 0
  const int *first;     // of each query; null: 0
};

// Several queries a sequence: its last offsets[b + 1] - offsets[b] tokens.
struct PagedPrompt {
  const void *q;
  void *out;
  size_t q_nb[2], out_nb[2];
  int q_heads, n_tokens;
  const int *offsets;
  float scale;
  PagedScores scores;
};

// Bytes of workspace that a prompt's attention of this shape takes, from its caller.
size_t paged_prompt_workspace(const PagedShape &p, int q_heads, int n_tokens, int n_seqs,
                              int table_width);
hipError_t launch_paged_prompt(const PagedShape &p, const PagedSeqs &q, const PagedPrompt &a,
                               void *workspace, hipStream_t s);
// The same for a few queries a sequence, without first tokens, and with a window or prefixes but
// not both; workspace is the handle's.
hipError_t launch_paged_few(const PagedShape &p, const PagedSeqs &q, const PagedPrompt &a,
                            void *workspace, hipStream_t s);

// Bytes of workspace an attention of this shape may need, zeroed once when it is made.
size_t paged_workspace_bytes(const PagedShape &p);
// step: one token a sequence, written into its page by the same launch (a.extra 1), or null.
hipError_t launch_paged_attend(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                               const PagedAppend *step, void *workspace, hipStream_t s);


// Where the weights of tokens are added up, fp32 [n_seqs][n_heads][tokens], strides in values;
// null: not asked for.  workspace: paged_weights_workspace bytes.
struct PagedWeights {
  float *weights;
  int64_t nb[2];  // between heads, sequences
  void *workspace;
};

size_t paged_weights_workspace(const PagedShape &p, int q_heads, int n_seqs, int width);
// As launch_paged_attend, with scores of its own; workspace is the handle's.
hipError_t launch_paged_shaped(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                               const PagedAppend *step, const PagedScores &sc,
                               const PagedWeights &w, void *workspace, hipStream_t s);

// Eviction: per sequence and key head the `keep` tokens that stay, of those the `recent` last
// ones, to the front of its pages or into others.
struct PagedEvict {
  float *weights;  // [n_seqs][n_heads][tokens], strides in values
  int64_t nb[2];
  int keep, recent;
  const int *into;  // [n_seqs] rows of into_width pages, into_stride apart; null: in place
  int into_width, into_stride;
  int *kept;  // [n_seqs][n_heads][keep]
};

hipError_t launch_paged_evict(const PagedShape &p, const PagedSeqs &q, const PagedEvict &e,
                              hipStream_t s);

// Pages of 4-bit values (paged4.hpp): PagedShape's pools hold them, its io is the rows' type.
hipError_t launch_paged4_append(const PagedShape &p, const PagedSeqs &q, const PagedAppend &a,
                                hipStream_t s);
// k, v: [n_tokens][n_heads][dim] fp32, of the tokens that an append of these arguments writes.
hipError_t launch_paged4_read(const PagedShape &p, const PagedSeqs &q, int n_tokens,
                              const int *offsets, float *k, float *v, hipStream_t s);
hipError_t launch_paged4_attend(const PagedShape &p, const PagedSeqs &q, const PagedAttend &a,
                                const PagedAppend *step, const PagedScores &sc, void *workspace,
                                hipStream_t s);

}  // namespace aq
