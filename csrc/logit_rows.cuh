// Rows of logits: addressing, running softmax statistics and their merge, shared by the kernels that
// score tokens (token_stats.cu) and distil from a teacher's alternatives (distill.cu).
//
// With y = x / T every kernel works in base 2: c2 = log2(e) / T, and a row is summarised by
//     m  a reference near the row's maximum (any value of the row that no exponent overflows against)
//     S  = sum 2^((x - m) c2)
//     W  = sum 2^((x - m) c2) (x - m) c2
// so that  ln sum e^y = m / T + ln S  and the entropy is  ln S - ln 2 * W / S. x - m is formed first
// and exactly scaled after, so logits of any common offset lose nothing; W is a sum relative to m, so
// the entropy has no cancellation of large terms. All three are fp32.
#pragma once

#include "common.cuh"

namespace tdsv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// 2^y is zero in fp32 below y = -150; W multiplies by the clamped exponent so that a masked logit
// (-inf) adds 0 * -kMinExponent and not 0 * -inf.
constexpr float kMinExponent = -1.0e4f;

// One row of a logits tensor whose leading dimensions collapse to two strides (in elements): a slice
// such as logits[:, :-1] or a padded vocabulary cut to size is read in place.
struct RowLayout {
  int64_t inner;     // rows of the inner leading dimension
  int64_t outer_stride;
  int64_t inner_stride;
  __device__ __forceinline__ int64_t offset(int64_t r) const {
    return (r / inner) * outer_stride + (r % inner) * inner_stride;
  }
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct RowStats {
  float m = -INFINITY, s = 0.f, w = 0.f;

  // Move the reference to `to` (>= m for finite values); a sum of nothing has no reference yet.
  __device__ __forceinline__ void rebase(float to, float c2) {
    if (s == 0.f) {
      m = to;
      return;
    }
    const float d = (m - to) * c2;
    const float f = exp2_fast(d);
    w = (w + s * fmaxf(d, kMinExponent)) * f;
    s *= f;
    m = to;
  }
  __device__ __forceinline__ void add(float x, float c2) {
    if (x > m) rebase(x, c2);
    if (x == -INFINITY) return;
    const float y = (x - m) * c2;
    const float e = exp2_fast(y);
    s += e;
    w += e * fmaxf(y, kMinExponent);
  }
  __device__ __forceinline__ void merge(const RowStats& o, float c2) {
    if (o.s == 0.f) return;  // (a NaN sum is not equal to zero and is merged)
    RowStats a = o;
    if (s == 0.f) {
      *this = a;
      return;
    }
    const float to = fmaxf(m, a.m);
    rebase(to, c2);
    a.rebase(to, c2);
    s += a.s;
    w += a.w;
  }
};

__device__ __forceinline__ RowStats warp_merge(RowStats v, float c2) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RowStats u;
    u.m = __shfl_xor_sync(0xffffffffu, v.m, o);
    u.s = __shfl_xor_sync(0xffffffffu, v.s, o);
    u.w = __shfl_xor_sync(0xffffffffu, v.w, o);
    v.merge(u, c2);
  }
  return v;
}

// Block-wide merge in a fixed order; every thread gets the result. `scratch` holds 33 entries.
__device__ __forceinline__ RowStats block_merge(RowStats v, float c2, RowStats* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = (blockDim.x + 31) >> 5;
  v = warp_merge(v, c2);
  __syncthreads();
  if (lane == 0) scratch[warp] = v;
  __syncthreads();
  if (warp == 0) {
    RowStats t;
    if (lane < warps) t = scratch[lane];
    t = warp_merge(t, c2);
    if (lane == 0) scratch[32] = t;
  }
  __syncthreads();
  return scratch[32];
}

// Host: the two-stride view of a logits tensor's leading dimensions, or false where a copy is needed.
inline bool row_layout(const at::Tensor& t, RowLayout& out) {
  const int64_t d = t.dim();
  if (d < 1 || (t.size(d - 1) > 1 && t.stride(d - 1) != 1)) return false;
  std::vector<std::pair<int64_t, int64_t>> dims;  // (size, stride), outermost first, ones dropped
  for (int64_t i = 0; i + 1 < d; ++i) {
    if (t.size(i) == 1) continue;
    if (!dims.empty() && dims.back().second == t.stride(i) * t.size(i)) dims.back() = {dims.back().first * t.size(i), t.stride(i)};
    else dims.push_back({t.size(i), t.stride(i)});
  }
  if (dims.size() > 2) return false;
  out.inner = dims.empty() ? 1 : dims.back().first;
  out.inner_stride = dims.empty() ? 0 : dims.back().second;
  out.outer_stride = dims.size() == 2 ? dims[0].second : 0;
  return true;
}

inline void check_logits(const at::Tensor& t, const char* what) {
  TDSV_CHECK(t.is_cuda() && t.has_storage(), what, ": logits must be a CUDA tensor with device storage");
  TDSV_CHECK(t.dim() >= 1 && t.size(t.dim() - 1) >= 1, what, ": logits must be [..., vocabulary]");
  TDSV_CHECK(t.size(t.dim() - 1) < (int64_t(1) << 30), what, ": vocabulary too large");
  TDSV_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kHalf || t.scalar_type() == at::kFloat, what,
             ": logits must be bf16, fp16 or fp32");
}

// Calls f with a null pointer of the logits' device type as the tag.
template <typename F>
void with_logit_type(at::ScalarType type, F&& f) {
  if (type == at::kBFloat16) f(static_cast<__nv_bfloat16*>(nullptr));
  else if (type == at::kHalf) f(static_cast<__half*>(nullptr));
  else f(static_cast<float*>(nullptr));
}

}  // namespace tdsv
