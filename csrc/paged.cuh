// A paged cache of keys and values, and the batch of sequences whose new tokens a call brings.
//
// keys, values   [pages, kv_heads, page rows, 128]; a page holds a power of two of tokens
// tables         int32 [sequences, width]: the page of each stretch of a sequence
// starts         int32 [sequences + 1]: sequence b brings the rows [starts[b], starts[b + 1]) of the call
// lengths        int32 [sequences]: tokens of sequence b in the cache, those rows included, so row i of its n
//                lies at position length - n + i
//
// All of it is read on the GPU, so a captured graph serves whatever the batch holds when it is replayed. What
// the host cannot see is checked here: a sequence whose numbers do not fit (negative or falling starts, more new
// tokens than length, a length beyond its table) takes no part, a page outside the pool is not touched, and both
// record kOutOfBounds in the status word.
#pragma once

#include "common.cuh"

namespace tdsv {

constexpr int kHeadDim = 128;

struct PagedBatch {
  const int* tables;
  const int* starts;
  const int* lengths;
  int64_t table_stride;
  int seqs, width, rows, pages, page_shift, kv_heads;
};

struct PagedSequence {
  int start = 0, n = 0, length = 0;  // n = 0: takes no part
};

__device__ __forceinline__ PagedSequence paged_sequence(const PagedBatch& p, int b, int* status) {
  PagedSequence s;
  const int first = p.starts[b], end = p.starts[b + 1], length = p.lengths[b];
  const bool fits = first >= 0 && end >= first && end <= p.rows && length >= end - first &&
                    static_cast<int64_t>(length) <= static_cast<int64_t>(p.width) << p.page_shift;
  if (!fits) {
    report_status(status, kOutOfBounds);
    return s;
  }
  s.start = first;
  s.n = end - first;
  s.length = length;
  return s;
}

// The sequence of row t, or `seqs` for a row behind the last one. Taken by a whole warp: a lane compares one start,
// so 32 sequences cost one load.
__device__ __forceinline__ int paged_find(const PagedBatch& p, int t) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int i = 0; i < p.seqs; i += 32) {
    const bool past = i + lane < p.seqs && p.starts[i + lane + 1] <= t;
    const unsigned votes = __ballot_sync(0xffffffffu, past);
    before += __popc(votes);
    if (votes != 0xffffffffu) break;
  }
  return before;
}

// Host: checks the cache and the batch and fills the kernels' view of them.
PagedBatch paged_batch(const at::Tensor& keys, const at::Tensor& values, const at::Tensor& tables,
                       const at::Tensor& starts, const at::Tensor& lengths, int64_t rows, const char* what);
// Strides of a pool's pages, heads and rows, in elements.
struct PoolStrides {
  int64_t page, head, row;
};
PoolStrides pool_strides(const at::Tensor& pool);

}  // namespace tdsv
