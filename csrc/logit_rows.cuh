// Rows of logits: addressing, running softmax statistics and their merge, shared by the kernels that
// score tokens (token_stats.cu) and distil from a teacher's alternatives (distill.cu).
//
// With y = x / T every kernel works in base 2: c2 = log2(e) / T, and a row is summarised by
//     m  the maximum of what was summed, or a value little below or above it
//     S  = sum 2^((x - m) c2)
//     W  = sum 2^((x - m) c2) (x - m) c2
// so that  ln sum e^y = m / T + ln S  and the entropy is  ln S - ln 2 * W / S. x - m is formed first
// and exactly scaled after, so logits of any common offset lose nothing (a log-probability is (x - m) / T - ln S: in
// base 2 a token masked by its type's lowest value would leave fp32's range); W is a sum relative to m, so
// the entropy has no cancellation of large terms. All three are fp32.
#pragma once

#include "common.cuh"

#include <type_traits>

namespace tdsv {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
// 2^y is zero in fp32 below y = -150; W multiplies by the clamped exponent so that a masked logit
// (-inf) adds 0 * -kMinExponent and not 0 * -inf.
constexpr float kMinExponent = -1.0e4f;

// One row of a logits tensor whose leading dimensions collapse to two strides (in elements): a slice
// such as logits[:, :-1] or a padded vocabulary cut to size is read in place.
struct RowLayout {
  uint32_t inner;  // rows of the inner leading dimension (a 64-bit division would cost a block some 200 cycles)
  int64_t outer_stride;
  int64_t inner_stride;
  __device__ __forceinline__ int64_t offset(uint32_t r) const {
    const uint32_t o = r / inner;
    return o * outer_stride + (r - o * inner) * inner_stride;
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

// What a backward needs of a row: m, 1 / S and W / S; 1 / S = 0 where the row has no gradient.
__device__ __forceinline__ float4 saved_stats(const RowStats& st) {
  if (st.s == 0.f) return make_float4(0.f, 0.f, 0.f, 0.f);
  return make_float4(st.m, 1.f / st.s, st.w / st.s, 0.f);
}

// Joins 32 statistics: the maximum first, so that each moves its reference once (a tree of pairwise merges is a
// chain of 1700 cycles).
__device__ __forceinline__ RowStats warp_join(const RowStats& v, float c2) {
  const bool some = v.s != 0.f;  // (NaN is something)
  RowStats r;
  r.m = warp_max(some ? v.m : -INFINITY);
  const float d = (v.m - r.m) * c2, f = exp2_fast(d);
  r.s = warp_sum(some ? v.s * f : 0.f);
  r.w = warp_sum(some ? (v.w + v.s * fmaxf(d, kMinExponent)) * f : 0.f);
  return r;
}

// The same for THREADS threads; every thread gets the result.
template <int THREADS>
struct JoinScratch {
  float m[THREADS / 32], s[THREADS / 32], w[THREADS / 32];
};
template <int THREADS>
__device__ __forceinline__ RowStats block_join(const RowStats& v, float c2, JoinScratch<THREADS>& sc) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const bool some = v.s != 0.f;  // (NaN is something)
  float m = warp_max(some ? v.m : -INFINITY);
  if (lane == 0) sc.m[warp] = m;
  __syncthreads();
  m = sc.m[0];
#pragma unroll
  for (int i = 1; i < THREADS / 32; ++i) m = fmaxf(m, sc.m[i]);
  const float d = (v.m - m) * c2, f = exp2_fast(d);
  const float s = warp_sum(some ? v.s * f : 0.f);
  const float w = warp_sum(some ? (v.w + v.s * fmaxf(d, kMinExponent)) * f : 0.f);
  if (lane == 0) sc.s[warp] = s, sc.w[warp] = w;
  __syncthreads();
  RowStats r;
  r.m = m;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) r.s += sc.s[i], r.w += sc.w[i];
  return r;
}

// ---- vectors of logits: 16 bytes, 8 or 4 values -----------------------------------------------------
__device__ __forceinline__ uint4 load_stream(const void* p) {  // read once: keep it out of L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}

template <typename T>
struct LogitVec {
  static constexpr int kSize = 16 / sizeof(T);
  static constexpr int kPairs = kSize / 2;
};

// The pair `i` of a vector as two floats.
template <typename T>
__device__ __forceinline__ float2 unpack_pair(const uint4& v, int i);
template <>
__device__ __forceinline__ float2 unpack_pair<__nv_bfloat16>(const uint4& v, int i) {
  const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack_pair<__half>(const uint4& v, int i) {
  const uint32_t w = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack_pair<float>(const uint4& v, int i) {
  return i == 0 ? make_float2(__uint_as_float(v.x), __uint_as_float(v.y))
                : make_float2(__uint_as_float(v.z), __uint_as_float(v.w));
}

// The largest of `n` vectors (NaN is passed over), compared in the logits' own type.
template <typename T, int n>
__device__ __forceinline__ float vec_max(const uint4 (&v)[n]) {
  if constexpr (sizeof(T) == 2) {
    using T2 = std::conditional_t<std::is_same_v<T, __half>, __half2, __nv_bfloat162>;
    auto as2 = [](uint32_t w) { return *reinterpret_cast<const T2*>(&w); };
    T2 m = __hmax2(__hmax2(as2(v[0].x), as2(v[0].y)), __hmax2(as2(v[0].z), as2(v[0].w)));
#pragma unroll
    for (int i = 1; i < n; ++i)
      m = __hmax2(m, __hmax2(__hmax2(as2(v[i].x), as2(v[i].y)), __hmax2(as2(v[i].z), as2(v[i].w))));
    uint4 w{};
    w.x = *reinterpret_cast<const uint32_t*>(&m);
    const float2 f = unpack_pair<T>(w, 0);
    return fmaxf(f.x, f.y);
  } else {
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < n; ++i)
      m = fmaxf(m, fmaxf(fmaxf(__uint_as_float(v[i].x), __uint_as_float(v[i].y)),
                         fmaxf(__uint_as_float(v[i].z), __uint_as_float(v[i].w))));
    return m;
  }
}

// Packed fp32 pairs (add, mul and fma of two at once).
union F2 {
  float2 f;
  uint64_t u;
};
__device__ __forceinline__ F2 pair(float a, float b) {
  F2 r;
  r.f = make_float2(a, b);
  return r;
}
__device__ __forceinline__ F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.u) : "l"(a.u), "l"(b.u));
  return r;
}
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.u) : "l"(a.u), "l"(b.u), "l"(c.u));
  return r;
}

// A thread's running statistics over vectors, whose maximum is taken first. The reference m starts at the
// maximum of the warp's first vectors and moves only when a value passes it by more than 2^kHeadroom, so the
// common step has no running maximum to carry and, for a value, half a subtraction, half a product, one
// exponential, half a sum and half a multiply-add. W then has positive terms of at most kHeadroom, beside
// which it can only be small where the largest weight is 2^kHeadroom times all others': its relative error
// stays within 2^kHeadroom roundings, 1e-6. (Moving m with every maximum costs some lane of a warp its
// moves in nine of ten steps, 20 instructions each.) Pairs are summed apart, which also halves the rounding of
// a long sum.
constexpr float kHeadroom = 4.f;

template <bool ENTROPY>
struct VecStats {
  float m = 0.f, limit = -INFINITY;  // nothing seen: any value sets the reference
  F2 s = pair(0.f, 0.f), w = pair(0.f, 0.f);

  __device__ __forceinline__ void raise(float to, float c2) {
    const float d = limit == -INFINITY ? 0.f : (m - to) * c2;
    const float f = exp2_fast(d), dc = fmaxf(d, kMinExponent);
    if (ENTROPY) {
      w.f.x = (w.f.x + s.f.x * dc) * f;
      w.f.y = (w.f.y + s.f.y * dc) * f;
    }
    s.f.x *= f;
    s.f.y *= f;
    m = to;
    limit = to + kHeadroom / c2;
  }
  // Before the first values: a reference that is one of the warp's values (none where all are masked).
  __device__ __forceinline__ void start(float warps_max, float c2) {
    if (warps_max > limit) raise(warps_max, c2);
  }
  template <typename T>
  __device__ __forceinline__ void add_vec(const uint4& v, float c2) {
    const F2 neg = pair(-m, -m), c = pair(c2, c2);
#pragma unroll
    for (int i = 0; i < LogitVec<T>::kPairs; ++i) {
      F2 x;
      x.f = unpack_pair<T>(v, i);
      const F2 y = mul2(add2(x, neg), c);
      const F2 e = pair(exp2_fast(y.f.x), exp2_fast(y.f.y));
      s = add2(s, e);
      if (ENTROPY) w = fma2(e, pair(fmaxf(y.f.x, kMinExponent), fmaxf(y.f.y, kMinExponent)), w);
    }
  }
  __device__ __forceinline__ void add_one(float x, float c2) {
    if (x > limit) raise(x, c2);
    const float y = (x - m) * c2, e = exp2_fast(y);
    s.f.x += e;
    if (ENTROPY) w.f.x += e * fmaxf(y, kMinExponent);
  }
  __device__ __forceinline__ RowStats total() const {
    RowStats r;
    r.m = m;
    r.s = s.f.x + s.f.y;
    r.w = w.f.x + w.f.y;
    return r;
  }
};

// A row cut at 16-byte boundaries: `head` single values, `vecs` vectors, `tail` single values.
struct RowCut {
  int head, vecs, tail;
};
template <typename T>
__device__ __forceinline__ RowCut cut_row(const T* row, int v) {
  RowCut c;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
  c.head = min(v, off == 0 ? 0 : LogitVec<T>::kSize - off);
  c.vecs = (v - c.head) / LogitVec<T>::kSize;
  c.tail = v - c.head - c.vecs * LogitVec<T>::kSize;
  return c;
}

// ---- the gradient's pass: out_i = 2^y_i (a + b y_i), y_i = (x_i - m) c2 ---------------------------------
template <typename T>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// (the one rounding of the gradient to the logits' type; PLAIN: b is zero)
template <typename T, bool PLAIN>
__device__ __forceinline__ uint4 gradient_vec(const uint4& v, float m, float c2, float a, float b) {
  const F2 neg = pair(-m, -m), c = pair(c2, c2), aa = pair(a, a), bb = pair(b, b);
  F2 d[LogitVec<T>::kPairs];
#pragma unroll
  for (int i = 0; i < LogitVec<T>::kPairs; ++i) {
    F2 x;
    x.f = unpack_pair<T>(v, i);
    F2 y = mul2(add2(x, neg), c);
    if (PLAIN) {
      d[i] = mul2(pair(exp2_fast(y.f.x), exp2_fast(y.f.y)), aa);
    } else {
      y = pair(fmaxf(y.f.x, kMinExponent), fmaxf(y.f.y, kMinExponent));
      d[i] = mul2(pair(exp2_fast(y.f.x), exp2_fast(y.f.y)), fma2(bb, y, aa));
    }
  }
  uint4 o;
  if constexpr (sizeof(T) == 2) {
    o.x = pack_pair<T>(d[0].f.x, d[0].f.y);
    o.y = pack_pair<T>(d[1].f.x, d[1].f.y);
    o.z = pack_pair<T>(d[2].f.x, d[2].f.y);
    o.w = pack_pair<T>(d[3].f.x, d[3].f.y);
  } else {
    o.x = __float_as_uint(d[0].f.x);
    o.y = __float_as_uint(d[0].f.y);
    o.z = __float_as_uint(d[1].f.x);
    o.w = __float_as_uint(d[1].f.y);
  }
  return o;
}
__device__ __forceinline__ float gradient_one(float x, float m, float c2, float a, float b) {
  const float y = fmaxf((x - m) * c2, kMinExponent);
  return exp2_fast(y) * (a + b * y);
}

// 16 bytes that start `bytes` (a multiple of 2 below 16, the same for the whole block) into lo, hi.
__device__ __forceinline__ uint4 shift_vec(const uint4& lo, const uint4& hi, int bytes) {
  uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
  if (bytes & 8) {
#pragma unroll
    for (int j = 0; j < 6; ++j) w[j] = w[j + 2];
  }
  if (bytes & 4) {
#pragma unroll
    for (int j = 0; j < 5; ++j) w[j] = w[j + 1];
  }
  if (bytes & 2) {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = __funnelshift_r(w[j], w[j + 1], 16);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// out[0, n) = gradient of row[0, n), by the threads of one block in vectors that are aligned at `out`. The
// logits may lie at another offset in their 16 bytes: two of their vectors are then joined by a shift, so
// that both sides move 16 bytes a thread whatever the vocabulary and the pitch are. `row` is in global or
// shared memory, kAhead vectors a thread are loaded at once; nothing outside [0, n) is read.
template <typename T, int THREADS, bool PLAIN, int kAhead>
__device__ __forceinline__ void write_gradient(const T* row, T* out, int n, float m, float c2, float a, float b) {
  constexpr int kSize = LogitVec<T>::kSize;
  const RowCut cut = cut_row(out, n);
  const int tid = threadIdx.x;
  if (tid < cut.head) out[tid] = from_float<T>(gradient_one(to_float<T>(row[tid]), m, c2, a, b));
  if (tid >= 32 && tid < 32 + cut.tail) {
    const int i = n - cut.tail + tid - 32;
    out[i] = from_float<T>(gradient_one(to_float<T>(row[i]), m, c2, a, b));
  }
  const T* from = row + cut.head;
  uint4* to = reinterpret_cast<uint4*>(out + cut.head);
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
  if (off == 0) {
    const uint4* x = reinterpret_cast<const uint4*>(from);
    for (int i = tid; i < cut.vecs; i += THREADS * kAhead) {
      uint4 v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u * THREADS < cut.vecs) v[u] = x[i + u * THREADS];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (i + u * THREADS < cut.vecs) to[i + u * THREADS] = gradient_vec<T, PLAIN>(v[u], m, c2, a, b);
    }
    return;
  }
  // the vectors whose two halves lie inside the row; at most the first and the last do not
  const uint4* x = reinterpret_cast<const uint4*>(from - off);
  const int first = off > cut.head ? 1 : 0;
  const int last = min(cut.vecs, (n - cut.head + off) / kSize - 1);  // vector i needs (i + 2) kSize <= n - head + off
  for (int i = first + tid; i < last; i += THREADS * kAhead) {
    uint4 lo[kAhead], hi[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i + u * THREADS < last) lo[u] = x[i + u * THREADS], hi[u] = x[i + u * THREADS + 1];
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (i + u * THREADS < last)
        to[i + u * THREADS] = gradient_vec<T, PLAIN>(shift_vec(lo[u], hi[u], off * static_cast<int>(sizeof(T))), m, c2, a, b);
  }
  // (two vectors at most, one value a thread)
  if (tid < 2 * kSize && cut.vecs > 0) {
    const int i = tid < kSize ? 0 : cut.vecs - 1;
    const bool todo = tid < kSize ? first == 1 : last < cut.vecs && (cut.vecs > 1 || first == 0);
    const int e = cut.head + i * kSize + tid % kSize;
    if (todo) out[e] = from_float<T>(gradient_one(to_float<T>(row[e]), m, c2, a, b));
  }
}

template <typename T, int THREADS>
__device__ __forceinline__ void write_zeros(T* out, int n) {
  const RowCut cut = cut_row(out, n);
  if (threadIdx.x < cut.head) out[threadIdx.x] = from_float<T>(0.f);
  if (threadIdx.x < cut.tail) out[n - cut.tail + threadIdx.x] = from_float<T>(0.f);
  uint4* to = reinterpret_cast<uint4*>(out + cut.head);
  for (int i = threadIdx.x; i < cut.vecs; i += THREADS) to[i] = make_uint4(0, 0, 0, 0);
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
  const int64_t inner = dims.empty() ? 1 : dims.back().first;
  if (inner > 0x7fffffff) return false;
  out.inner = static_cast<uint32_t>(std::max<int64_t>(inner, 1));
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
