// Distillation from a teacher's top alternatives: for each row the K recorded token ids and their
// log-probabilities t_k, against the student's y = x / T, p = softmax(y):
//
//   q_k = exp(t_k) / sum exp(t)                                  renormalised, or
//   q_k = exp(t_k),  q_rest = max(0, 1 - sum q_k)                with the tail as one more outcome
//   row = sum q_k (ln q_k - ln p_k) + q_rest (ln q_rest - ln p_rest),   p_rest = sum of p outside the K
//   total = sum_r w_r row_r
//
// The gradient is written in the same launch, since the weights are known: with Q = sum q_k + q_rest
//   dx_i = w / T (Q p_i - q_i)                  for an alternative
//   dx_i = w / T p_i (Q - q_rest / p_rest)      for every other token
//
// p_rest never comes from 1 - sum p_k. A bitmap of the alternatives in shared memory lets the pass over
// the row sum the other tokens on their own (m_r, S_r); the alternatives' sum (m_a, S_a) joins
// afterwards. So a student that puts nearly everything on the alternatives still has an exact p_rest, and
// the gradient outside is one exponential times a constant of the row. In that constant Q p_rest - q_rest
// is formed as sum q p_rest - q_rest p_a, whose terms do not cancel where either has little mass:
//   dx_i = 2^((x_i - m_r) c2) A,   A = w / T (sum q p_rest - q_rest p_a) / S_r.
//
// A row without alternatives (every id negative; without the tail also: no finite t_k) is not read: loss
// 0, zero gradient. Where no token is left outside the alternatives, the tail has no outcome and is
// dropped. Repeated ids count as one token whose q is the sum.
#include "logit_rows.cuh"

namespace tdsv {

namespace {

constexpr int kDistillThreads = 256;
constexpr int kMaxAlternatives = 128;

template <typename T, typename I, bool GRAD>
__global__ void __launch_bounds__(kDistillThreads)
    distill_kernel(const T* __restrict__ logits, RowLayout layout, int v, const I* __restrict__ ids,
                   const float* __restrict__ teacher, int k, const float* __restrict__ weights, float c2, float inv_t,
                   bool tail, float* __restrict__ rows_out, float* __restrict__ weighted, T* __restrict__ dlogits,
                   int* status) {
  extern __shared__ uint32_t bitmap[];
  __shared__ RowStats scratch[33];
  __shared__ float fscratch[32];
  __shared__ int at[kMaxAlternatives];
  __shared__ float q_s[kMaxAlternatives];
  const int64_t r = blockIdx.x;
  const T* row = logits + layout.offset(r);
  T* out = GRAD ? dlogits + r * v : nullptr;
  for (int i = threadIdx.x; i < (v + 31) / 32; i += blockDim.x) bitmap[i] = 0;
  __syncthreads();
  // one thread per alternative
  const int j = threadIdx.x;
  int id = -1;
  float t = -INFINITY;
  bool bad = false;
  if (j < k) {
    const int64_t raw = static_cast<int64_t>(ids[r * k + j]);
    bad = raw >= v;
    if (raw >= 0 && raw < v) id = static_cast<int>(raw), t = teacher[r * k + j];
    at[j] = id;
  }
  if (bad) report_status(status, kOutOfBounds);
  bool first = false;
  if (id >= 0) first = !(atomicOr(&bitmap[id >> 5], 1u << (id & 31)) >> (id & 31) & 1u);
  const int found = __syncthreads_count(id >= 0);
  if (__syncthreads_or(id >= 0 && !first)) {  // repeated ids: the first of each counts, whatever the order above
    first = id >= 0;
    for (int i = 0; i < j && first; ++i) first = at[i] != id;
  }
  const bool any_bad = __syncthreads_or(bad);
  const float tmax = block_max(t, fscratch);
  const bool any_nan = __syncthreads_or(t != t);
  const float w = weights != nullptr ? weights[r] : 1.f;
  if (!any_bad && !any_nan && (found == 0 || (!tail && tmax == -INFINITY))) {
    if (threadIdx.x == 0) rows_out[r] = 0.f, weighted[r] = 0.f;
    if (GRAD)
      for (int i = threadIdx.x; i < v; i += blockDim.x) out[i] = from_float<T>(0.f);
    return;
  }
  // the teacher's distribution
  const float shift = tail ? 0.f : tmax;
  float q = t == -INFINITY ? 0.f : expf(t - shift);
  const float qsum = block_sum(q, fscratch);
  float log_q = t - shift;
  float q_rest = 0.f;
  if (tail) {
    q_rest = fmaxf(0.f, 1.f - qsum);
  } else {
    q /= qsum;
    log_q -= logf(qsum);
  }
  if (j < k) q_s[j] = q;
  // the student outside the alternatives, and at them
  RowStats rest;
  for (int i = threadIdx.x; i < v; i += blockDim.x) {
    if (bitmap[i >> 5] >> (i & 31) & 1u) continue;
    rest.add(to_float<T>(row[i]), c2);
  }
  rest = block_merge(rest, c2, scratch);
  const float x = id >= 0 ? to_float<T>(row[id]) : -INFINITY;
  RowStats one;
  if (first) one.add(x, c2);
  const RowStats chosen = block_merge(one, c2, scratch);
  RowStats all = chosen;
  all.merge(rest, c2);
  const float log2s = log2f(all.s);
  if (tail && rest.s == 0.f) q_rest = 0.f;
  float part = 0.f;
  if (j < k && id >= 0 && q != 0.f) part = q * (log_q - kLn2 * ((x - all.m) * c2 - log2s));
  float loss = block_sum(part, fscratch);
  if (q_rest > 0.f) loss += q_rest * (logf(q_rest) - kLn2 * ((rest.m - all.m) * c2 + log2f(rest.s) - log2s));
  const bool empty = all.s == 0.f;  // every logit is masked: no distribution, no gradient
  if (empty) loss = INFINITY;
  if (any_bad) loss = NAN;
  if (threadIdx.x == 0) rows_out[r] = loss, weighted[r] = w * loss;
  if (!GRAD) return;
  const float whole = tail ? qsum + q_rest : 1.f;
  const float scale = w * inv_t;
  float outside = 0.f;
  if (rest.s != 0.f) {
    const float p_rest = exp2_fast((rest.m - all.m) * c2) * rest.s / all.s;
    const float p_chosen = chosen.s == 0.f ? 0.f : exp2_fast((chosen.m - all.m) * c2) * chosen.s / all.s;
    outside = scale * ((tail ? qsum : 1.f) * p_rest - q_rest * p_chosen) / rest.s;
  }
  const float base = rest.s == 0.f ? 0.f : rest.m;  // (every other logit is -inf there)
  if (any_bad) outside = NAN;
  for (int i = threadIdx.x; i < v; i += blockDim.x) {
    const float y = (to_float<T>(row[i]) - base) * c2;
    out[i] = from_float<T>(outside * exp2_fast(y));
  }
  __syncthreads();
  if (j < k && id >= 0) {
    float mass = 0.f;
    for (int i = 0; i < k; ++i) mass += at[i] == id ? q_s[i] : 0.f;
    const float d = empty ? 0.f : scale * (whole * exp2_fast((x - all.m) * c2 - log2s) - mass);
    out[id] = from_float<T>(any_bad ? NAN : d);
  }
}

// x *= *factor, unless it is one: the gradient was written for an upstream gradient of one.
template <typename T>
__global__ void scale_kernel(T* __restrict__ x, int64_t n, const float* __restrict__ factor) {
  const float f = *factor;
  if (f == 1.f) return;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x)
    x[i] = from_float<T>(to_float<T>(x[i]) * f);
}

}  // namespace

// (total [], rows [R], dlogits like logits, or empty where no gradient is asked for).
std::vector<at::Tensor> distill_fwd(const at::Tensor& logits_in, const at::Tensor& ids, const at::Tensor& teacher,
                                    const c10::optional<at::Tensor>& weights, double temperature, bool tail, bool grad) {
  check_logits(logits_in, "distillation_loss");
  const int64_t vocab = logits_in.size(-1), rows = logits_in.numel() / vocab;
  check_cuda_tensor(ids, "teacher_ids");
  check_cuda_tensor(teacher, "teacher_log_probs");
  TDSV_CHECK(ids.dim() == 2 && ids.size(0) == rows && ids.size(1) >= 1 && ids.size(1) <= kMaxAlternatives,
             "distillation_loss: teacher_ids must be [rows, 1 .. ", kMaxAlternatives, "]");
  TDSV_CHECK(ids.scalar_type() == at::kLong || ids.scalar_type() == at::kInt, "distillation_loss: int32 or int64 teacher_ids");
  TDSV_CHECK(teacher.sizes() == ids.sizes() && teacher.scalar_type() == at::kFloat,
             "distillation_loss: fp32 teacher_log_probs of the ids' shape");
  TDSV_CHECK(rows < (int64_t(1) << 31), "distillation_loss: too many rows");
  c10::cuda::CUDAGuard guard(logits_in.device());
  const bool weighted_rows = weights.has_value() && weights->defined();
  if (weighted_rows) {
    check_cuda_tensor(*weights, "weights");
    TDSV_CHECK(weights->scalar_type() == at::kFloat && weights->numel() == rows, "distillation_loss: fp32 weights, one per row");
  }
  RowLayout layout;
  at::Tensor logits = logits_in;
  if (!row_layout(logits, layout)) {
    logits = logits.contiguous();
    TDSV_CHECK(row_layout(logits, layout), "distillation_loss: logits layout");
  }
  const auto f32 = logits.options().dtype(at::kFloat);
  auto row_loss = at::empty({rows}, f32);
  auto weighted = at::empty({rows}, f32);
  auto dlogits = grad ? at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous))
                      : at::empty({0}, logits.options());
  if (rows == 0) return {weighted.sum(), row_loss, dlogits};
  const int k = static_cast<int>(ids.size(1));
  const int bitmap_bytes = static_cast<int>((vocab + 31) / 32 * 4);
  TDSV_CHECK(bitmap_bytes <= 200 * 1024, "distillation_loss: vocabulary too large");
  const float c2 = static_cast<float>(1.4426950408889634 / temperature), inv_t = static_cast<float>(1.0 / temperature);
  auto run = [&](auto* tag, auto* itag, auto has_grad) {
    using T = std::remove_pointer_t<decltype(tag)>;
    using I = std::remove_pointer_t<decltype(itag)>;
    auto kern = distill_kernel<T, I, decltype(has_grad)::value>;
    TDSV_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024));
    kern<<<static_cast<unsigned>(rows), kDistillThreads, bitmap_bytes, stream()>>>(
        static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab), ids.data_ptr<I>(),
        teacher.data_ptr<float>(), k, weighted_rows ? weights->data_ptr<float>() : nullptr, c2, inv_t, tail,
        row_loss.data_ptr<float>(), weighted.data_ptr<float>(), grad ? static_cast<T*>(dlogits.data_ptr()) : nullptr,
        status_word_ptr());
  };
  with_logit_type(logits.scalar_type(), [&](auto* tag) {
    auto with_ids = [&](auto* itag) {
      if (grad) run(tag, itag, std::true_type{});
      else run(tag, itag, std::false_type{});
    };
    if (ids.scalar_type() == at::kLong) with_ids(static_cast<int64_t*>(nullptr));
    else with_ids(static_cast<int32_t*>(nullptr));
  });
  TDSV_LAUNCH_CHECK();
  return {weighted.sum(), row_loss, dlogits};
}

// dlogits *= factor (a device scalar), in place; nothing is touched where it is one.
void distill_scale(at::Tensor& dlogits, const at::Tensor& factor) {
  check_cuda_tensor(dlogits, "dlogits");
  check_cuda_tensor(factor, "gradient");
  TDSV_CHECK(factor.scalar_type() == at::kFloat && factor.numel() == 1, "distillation_loss: fp32 scalar gradient");
  const int64_t n = dlogits.numel();
  if (n == 0) return;
  c10::cuda::CUDAGuard guard(dlogits.device());
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>((n + 2047) / 2048, 8 * num_sms()));
  with_logit_type(dlogits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    scale_kernel<T><<<grid, 256, 0, stream()>>>(static_cast<T*>(dlogits.data_ptr()), n, factor.data_ptr<float>());
  });
  TDSV_LAUNCH_CHECK();
}

}  // namespace tdsv
