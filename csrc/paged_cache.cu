// The new tokens of a step on their way into a paged cache: from the packed projection [T, (Hq + 2 Hkv) 128], the
// norms of queries and keys over each head, their rotation by the token's position, keys and values written to
// their pages, queries returned.
//
//     y = x / sqrt(mean(x^2) + eps) * w          (each head of 128)
//     out_i = y_i cos a_i - y_(i+64) sin a_i,  out_(i+64) = y_(i+64) cos a_i + y_i sin a_i,  a_i = position * f_i
//
// All in fp32, rounded once when stored. The angle is reduced in 64 bits before its sine is taken: fp32 leaves
// 0.002 of position 40000 times a frequency of 1, half a step of bf16. Each value is read and written once, so memory bounds
// it; with eight lanes a head, 16-byte accesses and packed fp32 arithmetic 10614 tokens of 40 heads (217 MB) take 47 us,
// 4.6 TB/s (68 us with 8-byte accesses that did not run ahead, 61 us with scalar arithmetic).
#include "logit_rows.cuh"
#include "paged.cuh"

namespace tdsv {

namespace {

constexpr int kThreads = 256;
constexpr int kLanes = 8;                   // of a head
constexpr int kGroups = kThreads / kLanes;  // heads at work
constexpr int kHalf = kHeadDim / 2;

// Lane l of 8 has dims [8 l, 8 l + 8) and their partners 64 further: a rotation needs no other lane. The values of a
// block's next heads are on their way while the angles are taken and the heads before them are worked on.
template <typename T, int TOKENS>
__global__ void __launch_bounds__(kThreads, 4) paged_append_kernel(
    const T* __restrict__ qkv, int64_t qkv_stride, const T* __restrict__ wq, const T* __restrict__ wk,
    const int64_t* __restrict__ positions, const float* __restrict__ freqs, T* __restrict__ q_out, T* __restrict__ keys,
    T* __restrict__ values, PoolStrides ks, PoolStrides vs, PagedBatch batch, int hq, float eps, int* __restrict__ status) {
  __shared__ alignas(16) float cosines[TOKENS][kHalf], sines[TOKENS][kHalf];
  __shared__ alignas(16) float weights[2][kHeadDim];
  __shared__ int page_of[TOKENS], row_of[TOKENS];  // page -1: the token is not stored
  const int tid = threadIdx.x, lane = tid % kLanes, group = tid / kLanes;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * TOKENS;
  const int here = static_cast<int>(min(static_cast<int64_t>(TOKENS), batch.rows - first));
  const int hkv = batch.kv_heads, heads = hq + 2 * hkv, items = here * heads;
  const T* mine = qkv + first * qkv_stride + 8 * lane;

  int t = group / heads, h = group - t * heads;  // token and head of item `group`
  uint4 lo = make_uint4(0, 0, 0, 0), hi = lo;
  const auto fetch = [&] {
    const T* from = mine + t * qkv_stride + static_cast<int64_t>(h) * kHeadDim;
    lo = load_stream(from);
    hi = load_stream(from + kHalf);
  };
  if (group < items) fetch();

  for (int i = tid; i < here * kHalf; i += kThreads) {
    // turns of the circle, whole ones dropped
    double turn = static_cast<double>(positions[first + i / kHalf]) * static_cast<double>(freqs[i % kHalf]) *
                  0.15915494309189533577;
    turn -= rint(turn);
    sincospif(2.f * static_cast<float>(turn), &sines[i / kHalf][i % kHalf], &cosines[i / kHalf][i % kHalf]);
  }
  weights[tid / kHeadDim][tid % kHeadDim] = to_float<T>((tid < kHeadDim ? wq : wk)[tid % kHeadDim]);
  for (int x = tid >> 5; x < here; x += kThreads / 32) {
    const int row = static_cast<int>(first) + x;
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
    if ((tid & 31) == 0) page_of[x] = page, row_of[x] = at;
  }
  __syncthreads();

  for (int base = 0; base < items; base += kGroups) {  // (the same number of turns for all: they shuffle)
    const bool some = base + group < items;
    const int token = t, head = h;
    uint4 a = lo, b = hi;
    h += kGroups;
    while (h >= heads) h -= heads, ++t;
    if (base + kGroups + group < items) fetch();
    F2 x[4], y[4], squares = pair(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      x[j].f = unpack_pair<T>(a, j);
      y[j].f = unpack_pair<T>(b, j);
      squares = fma2(x[j], x[j], fma2(y[j], y[j], squares));
    }
    float sum = some ? squares.f.x + squares.f.y : 0.f;
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!some) continue;
    const bool plain = head >= hq + hkv, is_q = head < hq;
    T* to;
    if (is_q) {
      to = q_out + ((first + token) * hq + head) * kHeadDim;
    } else {
      const int page = page_of[token];
      if (page < 0) continue;
      const PoolStrides& s = plain ? vs : ks;
      to = (plain ? values : keys) + page * s.page + (plain ? head - hq - hkv : head - hq) * s.head + row_of[token] * s.row;
    }
    if (!plain) {
      const float r = 1.f / sqrtf(sum * (1.f / kHeadDim) + eps);
      const F2 rr = pair(r, r);
      const float* w = weights[is_q ? 0 : 1] + 8 * lane;
      uint32_t out[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const auto two = [&](const float* at) { return pair(at[2 * j], at[2 * j + 1]); };
        const F2 c = two(&cosines[token][8 * lane]), s = two(&sines[token][8 * lane]);
        const F2 u = mul2(mul2(x[j], two(w)), rr), v = mul2(mul2(y[j], two(w + kHalf)), rr);
        const F2 first = fma2(u, c, mul2(pair(-v.f.x, -v.f.y), s)), second = fma2(v, c, mul2(u, s));
        out[j] = pack_pair<T>(first.f.x, first.f.y);
        out[4 + j] = pack_pair<T>(second.f.x, second.f.y);
      }
      a = make_uint4(out[0], out[1], out[2], out[3]);
      b = make_uint4(out[4], out[5], out[6], out[7]);
    }
    *reinterpret_cast<uint4*>(to + 8 * lane) = a;
    *reinterpret_cast<uint4*>(to + kHalf + 8 * lane) = b;
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
  TDSV_CHECK(qkv.stride(1) == 1 && (rows <= 1 || qkv.stride(0) % 8 == 0) &&
                 reinterpret_cast<uintptr_t>(qkv.data_ptr()) % 16 == 0,
             what, ": qkv's rows must be dense and 16-byte aligned");
  for (const at::Tensor& w : {wq, wk}) {
    check_cuda_tensor(w, "norm weight");
    TDSV_CHECK(w.device() == qkv.device() && w.scalar_type() == qkv.scalar_type() && w.numel() == kHeadDim,
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
    // Four tokens a block share its angles' and weights' latency once every SM has some: 1184 rows take 12.3 us in blocks of
    // four and 14.3 in blocks of one, 10000 rows 47 and 68; 300 rows take 10.2 and 8.2.
    if (rows >= 4 * num_sms()) go(paged_append_kernel<T, 4>, 4);
    else go(paged_append_kernel<T, 1>, 1);
  };
  if (qkv.scalar_type() == at::kHalf) launch(static_cast<__half*>(nullptr));
  else launch(static_cast<__nv_bfloat16*>(nullptr));
  TDSV_LAUNCH_CHECK();
  return q;
}

}  // namespace tdsv
