// Statistics of rows of logits at a temperature T (y = x / T, p = softmax(y)):
//
//   log_probs  ln p of one given token per row
//   entropy    H = -sum p ln p
//   top        the k largest logits, ties to the lowest index, with their ln p
//
// and the gradient of all three. With upstream g (log-probability), h (entropy), u_j (alternatives):
//   dx_i = [ g (d_it - p_i) + sum_j u_j (d_ij - p_i) - h p_i (ln p_i + H) ] / T
//
// A row whose target is the ignore index is not read: zeros, ids -1, zero gradient. Masked logits
// (-inf) have p = 0 and are never alternatives (id -1, ln p = -inf). A row that is masked throughout
// has ln p = -inf, H = 0 and no gradient. NaN or +inf in a row that is read gives NaN.
#include "logit_rows.cuh"

namespace tdsv {

namespace {

constexpr int kStatThreads = 256;
constexpr int kMaxTop = 128;

// Saved for the backward: m, log2 S, H and a spare per row; S = 0 is stored as log2 S = +inf.
__device__ __forceinline__ float4 saved_stats(const RowStats& st, float entropy) {
  return make_float4(st.s == 0.f ? 0.f : st.m, st.s == 0.f ? INFINITY : log2f(st.s), entropy, 0.f);
}

// The larger logit first, then the lower index.
__device__ __forceinline__ bool before(float a, int ia, float b, int ib) { return a > b || (a == b && ia < ib); }

template <typename T>
__global__ void __launch_bounds__(kStatThreads)
    stats_fwd_kernel(const T* __restrict__ logits, RowLayout layout, int v, const int64_t* __restrict__ targets,
                     int64_t ignore_index, float c2, int top, float* __restrict__ log_probs,
                     float* __restrict__ entropy, int64_t* __restrict__ top_ids, float* __restrict__ top_lp,
                     float4* __restrict__ saved, int* status) {
  __shared__ RowStats scratch[33];
  __shared__ float best_v[32];
  __shared__ int best_i[32];
  const int64_t r = blockIdx.x;
  const T* row = logits + layout.offset(r);
  const int64_t target = targets != nullptr ? targets[r] : 0;
  if (targets != nullptr && target == ignore_index) {
    if (threadIdx.x == 0) {
      log_probs[r] = 0.f;
      entropy[r] = 0.f;
      if (saved != nullptr) saved[r] = make_float4(0.f, INFINITY, 0.f, 0.f);
    }
    for (int j = threadIdx.x; j < top; j += blockDim.x) {
      top_ids[r * top + j] = -1;
      top_lp[r * top + j] = -INFINITY;
    }
    return;
  }
  RowStats st;
  for (int i = threadIdx.x; i < v; i += blockDim.x) st.add(to_float<T>(row[i]), c2);
  st = block_merge(st, c2, scratch);
  const float log2s = log2f(st.s);
  if (threadIdx.x == 0) {
    const float ent = st.s == 0.f ? 0.f : kLn2 * (log2s - st.w / st.s);
    entropy[r] = ent;
    if (targets != nullptr) {
      float lp = NAN;
      if (target >= 0 && target < v) {
        lp = st.s == 0.f ? -INFINITY : kLn2 * ((to_float<T>(row[target]) - st.m) * c2 - log2s);
      } else {
        report_status(status, kOutOfBounds);
      }
      log_probs[r] = lp;
    }
    if (saved != nullptr) saved[r] = saved_stats(st, ent);
  }
  float last = INFINITY;
  int last_i = -1;
  for (int j = 0; j < top; ++j) {
    float b = -INFINITY;
    int bi = 0x7fffffff;
    for (int i = threadIdx.x; i < v; i += blockDim.x) {
      const float x = to_float<T>(row[i]);
      if (before(last, last_i, x, i) && before(x, i, b, bi)) b = x, bi = i;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ob = __shfl_xor_sync(0xffffffffu, b, o);
      const int oi = __shfl_xor_sync(0xffffffffu, bi, o);
      if (before(ob, oi, b, bi)) b = ob, bi = oi;
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) best_v[threadIdx.x >> 5] = b, best_i[threadIdx.x >> 5] = bi;
    __syncthreads();
    b = best_v[0], bi = best_i[0];
    for (int w = 1; w < kStatThreads / 32; ++w)
      if (before(best_v[w], best_i[w], b, bi)) b = best_v[w], bi = best_i[w];
    if (threadIdx.x == 0) {
      const bool none = b == -INFINITY;
      top_ids[r * top + j] = none ? -1 : bi;
      top_lp[r * top + j] = none ? -INFINITY : kLn2 * ((b - st.m) * c2 - log2s);
    }
    last = b, last_i = bi;
  }
}

template <typename T>
__global__ void __launch_bounds__(kStatThreads)
    stats_bwd_kernel(const T* __restrict__ logits, RowLayout layout, int v, const int64_t* __restrict__ targets,
                     float c2, float inv_t, int top, const int64_t* __restrict__ top_ids,
                     const float4* __restrict__ saved, const float* __restrict__ g_lp, const float* __restrict__ g_ent,
                     const float* __restrict__ g_top, T* __restrict__ dlogits) {
  __shared__ int64_t at[kMaxTop + 1];
  __shared__ float grad[kMaxTop + 1];
  __shared__ float scratch[32];
  const int64_t r = blockIdx.x;
  const T* row = logits + layout.offset(r);
  T* out = dlogits + r * v;
  const float4 s = saved[r];
  if (s.y == INFINITY) {  // ignored, or nothing unmasked
    for (int i = threadIdx.x; i < v; i += blockDim.x) out[i] = from_float<T>(0.f);
    return;
  }
  // places that are not only -p_i (...): the target and the alternatives
  const int places = g_top != nullptr ? top + 1 : 1;
  float mine = 0.f;
  for (int j = threadIdx.x; j < places; j += blockDim.x) {
    const int64_t id = j < places - 1 ? top_ids[r * top + j] : (targets != nullptr ? targets[r] : -1);
    const bool there = id >= 0 && id < v;
    float u = 0.f;
    if (there) u = j < places - 1 ? g_top[r * top + j] : (g_lp != nullptr ? g_lp[r] : 0.f);
    at[j] = there ? id : -1;
    grad[j] = u;
    mine += u;
  }
  const float g = block_sum(mine, scratch);
  const float h = g_ent != nullptr ? g_ent[r] : 0.f;
  // T dx_i = p_i (a + b log2 p_i) + (d_i terms)
  const float a = -(g + h * s.z), b = -h * kLn2;
  for (int i = threadIdx.x; i < v; i += blockDim.x) {
    const float y = fmaxf((to_float<T>(row[i]) - s.x) * c2 - s.y, kMinExponent);
    out[i] = from_float<T>(inv_t * (exp2_fast(y) * (a + b * y)));
  }
  __syncthreads();
  for (int j = threadIdx.x; j < places; j += blockDim.x) {
    if (at[j] < 0) continue;
    float u = 0.f;  // equal places write the same sum
    for (int k = 0; k < places; ++k) u += at[k] == at[j] ? grad[k] : 0.f;
    const float y = fmaxf((to_float<T>(row[at[j]]) - s.x) * c2 - s.y, kMinExponent);
    out[at[j]] = from_float<T>(inv_t * (u + exp2_fast(y) * (a + b * y)));  // (u and a cancel where p = 1)
  }
}

}  // namespace

// (log_probs, entropy, top_ids, top_log_probs, saved): flat over the rows of logits [..., V].
std::vector<at::Tensor> token_stats_fwd(const at::Tensor& logits_in, const c10::optional<at::Tensor>& targets,
                                        double temperature, int64_t top, int64_t ignore_index, bool save) {
  check_logits(logits_in, "token_statistics");
  const int64_t vocab = logits_in.size(-1), rows = logits_in.numel() / vocab;
  TDSV_CHECK(top >= 0 && top <= kMaxTop && top <= vocab, "token_statistics: top must be in [0, min(", kMaxTop,
             ", vocabulary)]");
  TDSV_CHECK(rows < (int64_t(1) << 31), "token_statistics: too many rows");
  c10::cuda::CUDAGuard guard(logits_in.device());
  RowLayout layout;
  at::Tensor logits = logits_in;
  if (!row_layout(logits, layout)) {
    logits = logits.contiguous();
    TDSV_CHECK(row_layout(logits, layout), "token_statistics: logits layout");
  }
  const bool has_target = targets.has_value() && targets->defined();
  if (has_target) {
    check_cuda_tensor(*targets, "targets");
    TDSV_CHECK(targets->scalar_type() == at::kLong && targets->numel() == rows, "token_statistics: int64 targets, one per row");
  }
  const auto f32 = logits.options().dtype(at::kFloat);
  auto log_probs = at::empty({has_target ? rows : 0}, f32);
  auto entropy = at::empty({rows}, f32);
  auto top_ids = at::empty({top > 0 ? rows : 0, top}, logits.options().dtype(at::kLong));
  auto top_lp = at::empty({top > 0 ? rows : 0, top}, f32);
  auto saved = at::empty({save ? rows : 0, 4}, f32);
  if (rows == 0) return {log_probs, entropy, top_ids, top_lp, saved};
  const float c2 = static_cast<float>(1.4426950408889634 / temperature);
  with_logit_type(logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    stats_fwd_kernel<T><<<static_cast<unsigned>(rows), kStatThreads, 0, stream()>>>(
        static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab),
        has_target ? targets->data_ptr<int64_t>() : nullptr, ignore_index, c2, static_cast<int>(top),
        has_target ? log_probs.data_ptr<float>() : nullptr, entropy.data_ptr<float>(),
        top ? top_ids.data_ptr<int64_t>() : nullptr, top ? top_lp.data_ptr<float>() : nullptr,
        save ? reinterpret_cast<float4*>(saved.data_ptr<float>()) : nullptr, status_word_ptr());
  });
  TDSV_LAUNCH_CHECK();
  return {log_probs, entropy, top_ids, top_lp, saved};
}

// Contiguous gradient of the logits, in their shape and type.
at::Tensor token_stats_bwd(const at::Tensor& logits_in, const c10::optional<at::Tensor>& targets,
                           const at::Tensor& top_ids, const at::Tensor& saved, double temperature,
                           const c10::optional<at::Tensor>& g_log_probs, const c10::optional<at::Tensor>& g_entropy,
                           const c10::optional<at::Tensor>& g_top) {
  check_logits(logits_in, "token_statistics");
  const int64_t vocab = logits_in.size(-1), rows = logits_in.numel() / vocab;
  c10::cuda::CUDAGuard guard(logits_in.device());
  RowLayout layout;
  at::Tensor logits = logits_in;
  if (!row_layout(logits, layout)) {
    logits = logits.contiguous();
    TDSV_CHECK(row_layout(logits, layout), "token_statistics: logits layout");
  }
  auto dlogits = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  if (rows == 0) return dlogits;
  check_cuda_tensor(saved, "saved");
  check_cuda_tensor(top_ids, "top_ids");
  TDSV_CHECK(saved.scalar_type() == at::kFloat && saved.numel() == 4 * rows, "token_statistics: saved row statistics");
  auto pointer = [&](const c10::optional<at::Tensor>& t, int64_t count) -> const float* {
    if (!t.has_value() || !t->defined()) return nullptr;
    check_cuda_tensor(*t, "gradient");
    TDSV_CHECK(t->scalar_type() == at::kFloat && t->numel() == count, "token_statistics: fp32 gradients, one per output");
    return t->data_ptr<float>();
  };
  const bool has_target = targets.has_value() && targets->defined();
  if (has_target) {
    check_cuda_tensor(*targets, "targets");
    TDSV_CHECK(targets->scalar_type() == at::kLong && targets->numel() == rows, "token_statistics: int64 targets, one per row");
  }
  const int top = static_cast<int>(top_ids.size(1));
  TDSV_CHECK(top <= kMaxTop, "token_statistics: too many alternatives");
  const float *g_lp = pointer(g_log_probs, rows), *g_ent = pointer(g_entropy, rows), *g_alt = pointer(g_top, rows * top);
  const float c2 = static_cast<float>(1.4426950408889634 / temperature), inv_t = static_cast<float>(1.0 / temperature);
  with_logit_type(logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    stats_bwd_kernel<T><<<static_cast<unsigned>(rows), kStatThreads, 0, stream()>>>(
        static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab),
        has_target ? targets->data_ptr<int64_t>() : nullptr, c2, inv_t, top,
        top ? top_ids.data_ptr<int64_t>() : nullptr, reinterpret_cast<const float4*>(saved.data_ptr<float>()), g_lp,
        g_ent, top ? g_alt : nullptr, static_cast<T*>(dlogits.data_ptr()));
  });
  TDSV_LAUNCH_CHECK();
  return dlogits;
}

}  // namespace tdsv
