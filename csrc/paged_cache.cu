// The new tokens of a step on their way into a paged cache: from the packed projection [T, (Hq + 2 Hkv) 128], the
// norms of queries and keys over each head, their rotation by the token's position, keys and values written to
// their pages, queries returned.
//
//     y = x / sqrt(mean(x^2) + eps) * w          (each head of 128)
//     out_i = y_i cos a_i - y_(i+64) sin a_i,  out_(i+64) = y_(i+64) cos a_i + y_i sin a_i,  a_i = position * f_i
//
// All in fp32, rounded once when stored. The angle is reduced in 64 bits before its sine is taken: fp32 leaves
// 0.002 of position 40000 times a frequency of 1, half a step of bf16.
#include "paged.cuh"

namespace tdsv {

namespace {

constexpr int kThreads = 256;
constexpr int kGroups = kThreads / 16;  // 16 lanes take one head
constexpr int kHalf = kHeadDim / 2;

template <typename T>
struct alignas(8) Four {
  T v[4];
};

// Lane l of 16 has dims [4 l, 4 l + 4) and their partners 64 further: a rotation needs no other lane.
template <typename T, int TOKENS>
__global__ void __launch_bounds__(kThreads) paged_append_kernel(
    const T* __restrict__ qkv, int64_t qkv_stride, const T* __restrict__ wq, const T* __restrict__ wk,
    const int64_t* __restrict__ positions, const float* __restrict__ freqs, T* __restrict__ q_out, T* __restrict__ keys,
    T* __restrict__ values, PoolStrides ks, PoolStrides vs, PagedBatch batch, int hq, float eps, int* __restrict__ status) {
  __shared__ float cosines[TOKENS][kHalf], sines[TOKENS][kHalf];
  __shared__ int page_of[TOKENS], row_of[TOKENS];  // page -1: the token is not stored
  const int tid = threadIdx.x, lane = tid & 15, group = tid >> 4;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * TOKENS;
  const int here = static_cast<int>(min(static_cast<int64_t>(TOKENS), batch.rows - first));
  const int hkv = batch.kv_heads, heads = hq + 2 * hkv;

  for (int i = tid; i < here * kHalf; i += kThreads) {
    // turns of the circle, whole ones dropped
    double turn = static_cast<double>(positions[first + i / kHalf]) * static_cast<double>(freqs[i % kHalf]) *
                  0.15915494309189533577;
    turn -= rint(turn);
    sincospif(2.f * static_cast<float>(turn), &sines[i / kHalf][i % kHalf], &cosines[i / kHalf][i % kHalf]);
  }
  for (int t = tid >> 5; t < here; t += kThreads / 32) {
    const int row = static_cast<int>(first) + t;
    const int b = paged_find(batch, row);
    int page = -1, at = 0;
    if (b < batch.seqs) {
      const PagedSequence s = paged_sequence(batch, b, status);
      if (row >= s.start && row < s.start + s.n) {
        at = s.length - s.n + row - s.start;
        page = batch.tables[b * batch.table_stride + (at >> batch.page_shift)];
        at &= (1 << batch.page_shift) - 1;
        if (page < 0 || page >= batch.pages) {
          report_status(status, kOutOfBounds);
          page = -1;
        }
      }
    }
    if ((tid & 31) == 0) page_of[t] = page, row_of[t] = at;
  }
  float w[2][8];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const T* from = i == 0 ? wq : wk;
    const Four<T> lo = *reinterpret_cast<const Four<T>*>(from + 4 * lane);
    const Four<T> hi = *reinterpret_cast<const Four<T>*>(from + kHalf + 4 * lane);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[i][j] = to_float<T>(lo.v[j]), w[i][4 + j] = to_float<T>(hi.v[j]);
  }
  __syncthreads();

  const int items = here * heads;
  for (int base = 0; base < items; base += kGroups) {  // (the same number of turns for all: they shuffle)
    const int item = base + group;
    const bool some = item < items;
    const int t = some ? item / heads : 0, h = some ? item - t * heads : 0;
    const T* from = qkv + (first + t) * qkv_stride + static_cast<int64_t>(h) * kHeadDim + 4 * lane;
    Four<T> lo = *reinterpret_cast<const Four<T>*>(from), hi = *reinterpret_cast<const Four<T>*>(from + kHalf);
    const bool plain = h >= hq + hkv, is_q = h < hq;
    float x[8], sum = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = to_float<T>(lo.v[j]), x[4 + j] = to_float<T>(hi.v[j]);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum += x[j] * x[j];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!some) continue;
    T* to;
    if (is_q) {
      to = q_out + ((first + t) * hq + h) * kHeadDim;
    } else {
      const int page = page_of[t];
      if (page < 0) continue;
      const PoolStrides& s = plain ? vs : ks;
      to = (plain ? values : keys) + page * s.page + (plain ? h - hq - hkv : h - hq) * s.head + row_of[t] * s.row;
    }
    if (!plain) {
      const float r = 1.f / sqrtf(sum * (1.f / kHeadDim) + eps);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float c = cosines[t][4 * lane + j], s = sines[t][4 * lane + j];
        const float a = x[j] * r * (is_q ? w[0][j] : w[1][j]), b = x[4 + j] * r * (is_q ? w[0][4 + j] : w[1][4 + j]);
        lo.v[j] = from_float<T>(a * c - b * s);
        hi.v[j] = from_float<T>(b * c + a * s);
      }
    }
    *reinterpret_cast<Four<T>*>(to + 4 * lane) = lo;
    *reinterpret_cast<Four<T>*>(to + kHalf + 4 * lane) = hi;
  }
}

}  // namespace

PoolStrides pool_strides(const at::Tensor& pool) {
  // (a dimension of one has any stride; it is never stepped)
  auto stride = [&](int d) { return pool.size(d) == 1 ? int64_t(kHeadDim) : pool.stride(d); };
  return {stride(0), stride(1), stride(2)};
}

PagedBatch paged_batch(const at::Tensor& keys, const at::Tensor& values, const at::Tensor& tables,
                       const at::Tensor& starts, const at::Tensor& lengths, int64_t rows, const char* what) {
  for (const at::Tensor& t : {keys, values}) {
    TDSV_CHECK(t.is_cuda() && t.has_storage() && t.data_ptr() != nullptr, what, ": the cache must have device storage");
    TDSV_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf, what, ": the cache must be bf16 or fp16");
    TDSV_CHECK(t.dim() == 4 && t.size(3) == kHeadDim && t.stride(3) == 1, what,
               ": a cache is [pages, heads, page, ", kHeadDim, "] with dense rows");
    TDSV_CHECK(t.sizes() == keys.sizes() && t.scalar_type() == keys.scalar_type() && t.device() == keys.device(), what,
               ": keys and values must be alike");
    TDSV_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, what, ": the cache must start on 16 bytes");
    for (int d = 0; d < 3; ++d)
      TDSV_CHECK(t.size(d) == 1 || (t.stride(d) % 8 == 0 && t.stride(d) > 0), what,
                 ": pages, heads and rows of the cache must lie multiples of 16 bytes apart");
  }
  const int64_t page = keys.size(2);
  TDSV_CHECK(page >= 16 && (page & (page - 1)) == 0 && page <= (1 << 20), what,
             ": a page holds a power of two of tokens, 16 or more");
  TDSV_CHECK(keys.size(0) >= 1 && keys.size(0) < (int64_t(1) << 31) && keys.size(1) >= 1 && keys.size(1) <= 65535, what,
             ": cache sizes");
  for (const at::Tensor& t : {tables, starts, lengths})
    TDSV_CHECK(t.is_cuda() && t.device() == keys.device() && t.scalar_type() == at::kInt, what,
               ": tables, starts and lengths must be int32 on the cache's device");
  check_cuda_tensor(starts, "starts");
  check_cuda_tensor(lengths, "lengths");
  const int64_t seqs = lengths.numel();
  TDSV_CHECK(tables.dim() == 2 && tables.size(0) == seqs && starts.numel() == seqs + 1 &&
                 (tables.size(1) <= 1 || tables.stride(1) == 1),
             what, ": tables [sequences, pages], starts [sequences + 1], lengths [sequences]");
  TDSV_CHECK(rows < (int64_t(1) << 31) && seqs < (int64_t(1) << 24) && tables.size(1) < (int64_t(1) << 31), what,
             ": batch too large");
  PagedBatch p{};
  p.tables = tables.data_ptr<int>();
  p.starts = starts.data_ptr<int>();
  p.lengths = lengths.data_ptr<int>();
  p.table_stride = tables.stride(0);
  p.seqs = static_cast<int>(seqs);
  p.width = static_cast<int>(tables.size(1));
  p.rows = static_cast<int>(rows);
  p.pages = static_cast<int>(keys.size(0));
  p.kv_heads = static_cast<int>(keys.size(1));
  while ((int64_t(1) << p.page_shift) < page) ++p.page_shift;
  return p;
}

// q [T, hq, 128]; the keys and values of the batch's tokens are written to the cache.
at::Tensor paged_append(const at::Tensor& qkv, const at::Tensor& wq, const at::Tensor& wk, const at::Tensor& positions,
                        const at::Tensor& freqs, int64_t hq, double eps, at::Tensor& keys, at::Tensor& values,
                        const at::Tensor& tables, const at::Tensor& starts, const at::Tensor& lengths) {
  constexpr const char* what = "paged_append";
  TDSV_CHECK(qkv.is_cuda() && qkv.has_storage() && qkv.dim() == 2, what, ": qkv must be [rows, (hq + 2 hkv) 128] on a GPU");
  c10::cuda::CUDAGuard guard(qkv.device());
  TDSV_CHECK(keys.device() == qkv.device(), what, ": the cache must be on qkv's device");
  const int64_t rows = qkv.size(0);
  const PagedBatch batch = paged_batch(keys, values, tables, starts, lengths, rows, what);
  TDSV_CHECK(hq >= 1 && qkv.size(1) == (hq + 2 * batch.kv_heads) * kHeadDim && qkv.scalar_type() == keys.scalar_type(), what,
             ": qkv must hold hq + 2 hkv heads in the cache's type");
  TDSV_CHECK(qkv.stride(1) == 1 && (rows <= 1 || qkv.stride(0) % 4 == 0) &&
                 reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 8 == 0,
             what, ": qkv's rows must be dense and 8-byte aligned");
  for (const at::Tensor& w : {wq, wk}) {
    check_cuda_tensor(w, "norm weight");
    TDSV_CHECK(w.device() == qkv.device() && w.scalar_type() == qkv.scalar_type() && w.numel() == kHeadDim &&
                   reinterpret_cast<uintptr_t>(w.data_ptr()) % 8 == 0,
               what, ": norm weights must be 128 values of qkv's type");
  }
  check_cuda_tensor(positions, "positions");
  check_cuda_tensor(freqs, "freqs");
  TDSV_CHECK(positions.device() == qkv.device() && positions.scalar_type() == at::kLong && positions.numel() == rows, what,
             ": int64 positions, one per row");
  TDSV_CHECK(freqs.device() == qkv.device() && freqs.scalar_type() == at::kFloat && freqs.numel() == kHalf, what,
             ": 64 fp32 frequencies");
  auto q = at::empty({rows, hq, kHeadDim}, qkv.options());
  if (rows == 0) return q;
  auto launch = [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto go = [&](auto kern, int tokens) {
      kern<<<static_cast<unsigned>((rows + tokens - 1) / tokens), kThreads, 0, stream()>>>(
          static_cast<const T*>(qkv.data_ptr()), qkv.stride(0), static_cast<const T*>(wq.data_ptr()),
          static_cast<const T*>(wk.data_ptr()), positions.data_ptr<int64_t>(), freqs.data_ptr<float>(),
          static_cast<T*>(q.data_ptr()), static_cast<T*>(keys.data_ptr()), static_cast<T*>(values.data_ptr()),
          pool_strides(keys), pool_strides(values), batch, static_cast<int>(hq), static_cast<float>(eps), status_word_ptr());
    };
    if (rows >= 8 * num_sms()) go(paged_append_kernel<T, 4>, 4);
    else go(paged_append_kernel<T, 1>, 1);
  };
  if (qkv.scalar_type() == at::kHalf) launch(static_cast<__half*>(nullptr));
  else launch(static_cast<__nv_bfloat16*>(nullptr));
  TDSV_LAUNCH_CHECK();
  return q;
}

}  // namespace tdsv
