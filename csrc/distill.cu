// Distillation from a teacher's top alternatives: for each row the K recorded token ids and their
// log-probabilities t_k, against the student's y = x / T, p = softmax(y):
//
//   q_k = exp(t_k) / sum exp(t)                                  renormalised, or
//   q_k = exp(t_k),  q_rest = max(0, 1 - sum q_k)                with the tail as one more outcome
//   row = sum q_k (ln q_k - ln p_k) + q_rest (ln q_rest - ln p_rest),   p_rest = sum of p outside the K
//   total = sum_r w_r row_r
//
// The gradient is written in the same launch, since the weights are known, for an upstream gradient of one (see
// distill_again_kernel for any other): with Q = sum q_k + q_rest
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
// A row of weight zero has its loss reported, but no share of the total and a gradient of zeros, even where its loss
// is infinite or its logits are NaN. A row without alternatives (every id negative; without the tail also: no finite t_k) is not read: loss
// 0, zero gradient. Where no token is left outside the alternatives, the tail has no outcome and is
// dropped. Repeated ids count as one token whose q is the sum.
#include "logit_rows.cuh"

#include <cooperative_groups.h>
#include <mutex>

namespace tdsv {

namespace {

constexpr int kDistillThreads = 256;
constexpr int kMaxAlternatives = 128;
constexpr int kPerLane = kMaxAlternatives / 32;
constexpr int kAhead = 4;        // vectors a thread has in flight
constexpr int kMaxCluster = 16;  // above 8 the kernel is allowed it explicitly

// What one warp works out for a row and the block then uses.
struct RowPlan {
  int read;                             // whether the row is read at all
  int bad;                              // an id beyond the vocabulary
  int copied;                           // whether the bulk copy was started
  float q_sum, q_rest;                  // the alternatives' mass and the rest
  double q_gap, log_chosen;             // sum q (ln q - ln 2 y) and ln of chosen_s: see the loss below
  float chosen_m, chosen_s;             // the student's sum over the alternatives
  int masked;                           // a weight of zero: no share of the total and no gradient, whatever the row holds
  float base;                           // reference of the pass that writes the gradient
  float outside;                        // A above
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

// 148 SMs hold 740 blocks: rows that start just after those of now. (At 128 rows whatever their blocks, 1500 x 129280 fp32,
// sixteen blocks a row, takes 375 us in place of 367 and 8192 x 10000 fp32, one block a row, 124 in place of 127.)
constexpr int kBlocksAhead = 1024;
__device__ __forceinline__ void prefetch_l2(const void* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

// Warp 0 says that its part of the block's state is ready (and goes on); the other warps wait for it.
__device__ __forceinline__ void named_barrier_arrive() {
  asm volatile("bar.arrive 1, %0;" ::"n"(kDistillThreads) : "memory");
}
__device__ __forceinline__ void named_barrier_wait() {
  asm volatile("bar.sync 1, %0;" ::"n"(kDistillThreads) : "memory");
}

// A cluster of blocks takes a row, each block a stretch of it. With the gradient, the stretch is copied to
// shared memory by one bulk copy that starts as soon as the row is known to have alternatives; it is summed
// there, and the gradient is formed there after the cluster has joined its sums. So a row costs one read and
// one write, whatever its length (up to the shared memory of 16 blocks). Five blocks on an SM are in
// different phases, which keeps copies, sums and stores going at once: the phases of one block alone are a chain
// of latencies. Without the gradient a stretch passes through registers.
//
// 4096 rows of 151936 bf16 with 64 alternatives take 585 us, 4.3 TB/s of the two passes over memory (floor 380): bound
// by a block's chain of phases and, at half of their rate, by the two exponentials of every value. The loss alone of
// 2000 rows takes 129 us: 2.7 rounds of 740 blocks, each of which waits for its alternatives before it sums.
//
// One warp deals with the alternatives, up to four a lane, without block barriers.
template <typename T, typename I, bool GRAD>
__global__ void __launch_bounds__(kDistillThreads, 5)
    distill_kernel(const T* __restrict__ logits, RowLayout layout, int v, const I* __restrict__ ids,
                   const float* __restrict__ teacher, int k, const float* __restrict__ weights, float c2, float inv_t,
                   bool tail, float* __restrict__ rows_out, float* __restrict__ weighted, T* __restrict__ dlogits,
                   float2* __restrict__ saved, float* __restrict__ saved_chosen, int* status) {
  namespace cg = cooperative_groups;
  constexpr int kSize = LogitVec<T>::kSize;
  extern __shared__ uint4 smem[];  // GRAD: the stretch (one vector ahead of it, one after); then its bitmap
  __shared__ JoinScratch<kDistillThreads> scratch;
  __shared__ RowStats parts[kMaxCluster];
  __shared__ int repeats[kMaxCluster];  // whether a block met an id twice
  __shared__ int at[kMaxAlternatives];
  __shared__ float q_s[kMaxAlternatives];
  __shared__ float e_s[kMaxAlternatives];  // 2^y of an alternative; then its gradient
  __shared__ RowPlan plan;
  __shared__ uint64_t arrived;  // mbarrier of the bulk copy
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  if (blocks > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  const int tid = threadIdx.x, lane = tid & 31;
  const int64_t r = blockIdx.x / static_cast<unsigned>(blocks);
  const T* row = logits + layout.offset(static_cast<uint32_t>(r));

  // this block's stretch: vectors [v0, v1) of the row, and the single values at the row's ends
  const RowCut cut = cut_row(row, v);
  const int per = (cut.vecs + blocks - 1) / blocks;
  const int v0 = min(cut.vecs, part * per), v1 = min(cut.vecs, v0 + per);
  const int e_vec = cut.head + v0 * kSize;  // the first vector's first element
  const int first = part == 0 ? 0 : e_vec, last = part == blocks - 1 ? v : cut.head + v1 * kSize;
  const uint4* base = reinterpret_cast<const uint4*>(row + cut.head) + v0;
  const int vecs = v1 - v0;
  uint4* kept = smem + 1;                                        // GRAD
  T* kept_values = reinterpret_cast<T*>(kept) - (e_vec - first);  // element `first`
  uint32_t* bitmap = reinterpret_cast<uint32_t*>(smem + (GRAD ? per + 2 : 0));  // element e is bit e - e_vec + 32
  uint4 next[kAhead];
  auto load = [&](int from) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = from + u * kDistillThreads + tid;
      if (i < vecs) next[u] = load_stream(base + i);
    }
  };
  if (!GRAD) load(0);
  float single = -INFINITY;
  int single_at = -1;
  if (tid < e_vec - first) single_at = first + tid;
  const int after = last - e_vec - vecs * kSize;
  if (tid >= 32 && tid < 32 + after) single_at = last - after + tid - 32;

  // ---- the alternatives (warp 0), while the other warps clear the bitmap
  int id[kPerLane];
  float t[kPerLane], w = 1.f;
  bool bad = false;
  int found = 0;
  if (tid < 32) {
    if (weights != nullptr) w = weights[r];
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
      const int a = j * 32 + lane;
      id[j] = -1, t[j] = -INFINITY;
      if (a < k) {
        const int64_t raw = static_cast<int64_t>(ids[r * k + a]);
        t[j] = teacher[r * k + a];
        bad |= raw >= v;
        if (raw >= 0 && raw < v) id[j] = static_cast<int>(raw);
      }
      at[a] = id[j];
      found += id[j] >= 0;
    }
    if (GRAD) {
      const bool copy = vecs > 0 && __any_sync(0xffffffffu, found > 0 || bad);
      if (lane == 0) {
        mbar_init(&arrived, 1);
        fence_barrier_init();
        fence_proxy_async_smem();
      }
      if (lane == 0 && copy) {
        mbar_arrive_expect_tx(&arrived, static_cast<uint32_t>(vecs) * 16);
        bulk_load(kept, base, static_cast<uint32_t>(vecs) * 16, &arrived);
      }
      if (lane == 0) plan.copied = copy;
    }
  } else {
    const int words = (vecs * kSize + kSize + 31) / 32 + 1;
    for (int i = tid - 32; i < words; i += kDistillThreads - 32) bitmap[i] = 0;
    // The alternatives of a row that will start about when this one ends: from memory they would hold up the
    // row's copy behind all the others' (start to known alternatives: 8100 of a block's 25300 cycles).
    const int64_t later = r + kBlocksAhead / blocks;
    if (part == 0 && tid >= kDistillThreads - 32 && later * blocks < gridDim.x) {
      if (lane * 16 < k) prefetch_l2(ids + later * k + lane * 16);  // 64 or 128 bytes of ids a lane
      if (lane * 32 < k) prefetch_l2(teacher + later * k + lane * 32);
    }
  }
  if (single_at >= 0) single = to_float<T>(row[single_at]);
  if (GRAD && single_at >= 0) kept_values[single_at - first] = row[single_at];
  __syncthreads();

  if (tid < 32) {
    float x[kPerLane], shift = -INFINITY;
    bool nan = false, repeated = false;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
      if (id[j] < 0) t[j] = -INFINITY;
      if (id[j] >= 0) {
        nan |= t[j] != t[j];
        shift = fmaxf(shift, t[j]);
        if (id[j] >= first && id[j] < last) {
          const int bit = id[j] - e_vec + 32;
          repeated |= (atomicOr(&bitmap[bit >> 5], 1u << (bit & 31)) >> (bit & 31) & 1u) != 0;
        }
      }
    }
    bad = __any_sync(0xffffffffu, bad);
    nan = __any_sync(0xffffffffu, nan);
    found = __reduce_add_sync(0xffffffffu, found);
    repeated = __any_sync(0xffffffffu, repeated);
    shift = warp_max(shift);
    if (lane == 0) {
      plan.read = bad || nan || (found > 0 && (tail || shift != -INFINITY));
      plan.bad = bad;
      repeats[part] = repeated;
      if (bad && part == 0) report_status(status, kOutOfBounds);
    }
    __syncwarp();
    named_barrier_arrive();
    // what of the loss and the gradient does not need the other tokens, while the other warps go on
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) x[j] = id[j] >= 0 ? to_float<T>(row[id[j]]) : -INFINITY;
    if (tail) shift = 0.f;
    float q[kPerLane], q_sum = 0.f;
    double q_gap = 0.0;  // (terms of ten and more that leave a divergence of a tenth: 64 bits, off the others' path)
    RowStats chosen;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
      q[j] = t[j] == -INFINITY ? 0.f : expf(t[j] - shift);
      q_sum += q[j];
      if (id[j] >= 0) chosen.m = fmaxf(chosen.m, x[j]);
    }
    q_sum = warp_sum(q_sum);
    chosen.m = warp_max(chosen.m);
    if (chosen.m == -INFINITY) chosen.m = 0.f;
    const float log_sum = tail ? 0.f : logf(q_sum);
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
      if (!tail) q[j] /= q_sum;
      const float y = (x[j] - chosen.m) * c2, e = exp2_fast(y);
      if (id[j] >= 0) chosen.s += e;
      if (q[j] != 0.f)
        q_gap += static_cast<double>(q[j]) * (static_cast<double>(t[j]) - shift - log_sum -
                                              0.6931471805599453 * (static_cast<double>(x[j]) - chosen.m) * c2);
      q_s[j * 32 + lane] = q[j];
      e_s[j * 32 + lane] = e;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) q_gap += __shfl_xor_sync(0xffffffffu, q_gap, o);
    chosen.s = warp_sum(chosen.s);
    if (lane == 0) {
      plan.q_sum = tail ? q_sum : 1.f;
      plan.q_rest = tail ? fmaxf(0.f, 1.f - q_sum) : 0.f;
      plan.q_gap = q_gap;
      plan.log_chosen = log(static_cast<double>(chosen.s));
      plan.chosen_m = chosen.m;
      plan.chosen_s = chosen.s;
    }
    __syncwarp();
  } else {
    named_barrier_wait();
  }
  if (!plan.read) {  // the same for the whole cluster
    if (tid == 0 && part == 0) rows_out[r] = 0.f, weighted[r] = 0.f;
    if (GRAD) {
      if (tid == 0 && part == 0) saved[r] = make_float2(INFINITY, 0.f);
      if (plan.copied) mbar_wait(&arrived, 0, status, kTimeoutFull);
      write_zeros<T, kDistillThreads>(dlogits + r * v + first, last - first);
    }
    if (blocks > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    return;
  }

  // ---- the student outside the alternatives: one pass
  VecStats<false> st;
  const uint8_t* bytes = reinterpret_cast<const uint8_t*>(bitmap);
  auto without_chosen = [&](uint4& x, int i) {
    const uint32_t chosen = sizeof(T) == 2 ? bytes[i + 4] : bytes[(i >> 1) + 4] >> (4 * (i & 1)) & 15u;
    if (chosen == 0) return;
    uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < kSize; ++e) {
      if (!(chosen >> e & 1u)) continue;
      if constexpr (sizeof(T) == 4) {
        w[e] = 0xff800000u;
      } else {
        const uint32_t masked = std::is_same_v<T, __half> ? 0xfc00u : 0xff80u;
        w[e >> 1] = e & 1 ? (w[e >> 1] & 0xffffu) | masked << 16 : (w[e >> 1] & 0xffff0000u) | masked;
      }
    }
    x = make_uint4(w[0], w[1], w[2], w[3]);
  };
  if (GRAD && plan.copied) mbar_wait(&arrived, 0, status, kTimeoutFull);
  if constexpr (GRAD) {
    // (the reference is a value of the rest: an alternative far above all of it would round it away)
    // Warp 0, which has the alternatives to see to, takes no part.
    uint4 one[1];
    float mx = -INFINITY;
    const int i0 = tid >= 32 ? tid - 32 : vecs;
    if (i0 < vecs) {
      one[0] = kept[i0];
      without_chosen(one[0], i0);
      mx = vec_max<T, 1>(one);
    }
    st.start(warp_max(mx), c2);
#pragma unroll 2
    for (int i = i0; i < vecs; i += kDistillThreads - 32) {
      one[0] = kept[i];
      without_chosen(one[0], i);
      mx = vec_max<T, 1>(one);
      if (mx > st.limit) st.raise(mx, c2);
      st.add_vec<T>(one[0], c2);
    }
  } else {
    for (int from = 0; from < vecs; from += kDistillThreads * kAhead) {
      uint4 now[kAhead];
      const int mine = (vecs - from - tid + kDistillThreads - 1) / kDistillThreads;
#pragma unroll
      for (int u = 0; u < kAhead; ++u) now[u] = next[u];
      if (from + kDistillThreads * kAhead < vecs) load(from + kDistillThreads * kAhead);
      float mx = -INFINITY;
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u < mine) {
          without_chosen(now[u], from + u * kDistillThreads + tid);
          const uint4 one[1] = {now[u]};
          mx = fmaxf(mx, vec_max<T, 1>(one));
        }
      if (from == 0) st.start(warp_max(mx), c2);
      if (mx > st.limit) st.raise(mx, c2);
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (u < mine) st.add_vec<T>(now[u], c2);
    }
  }
  if (single_at >= 0) {
    const int bit = single_at - e_vec + 32;
    if (!(bitmap[bit >> 5] >> (bit & 31) & 1u)) st.add_one(single, c2);
  }
  RowStats rest = block_join<kDistillThreads>(st.total(), c2, scratch);
  if (blocks > 1) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
    if (tid < blocks) {
      *cluster.map_shared_rank(&parts[part], tid) = rest;
      if (tid != part) *cluster.map_shared_rank(&repeats[part], tid) = repeats[part];
    }
    cluster.sync();
  }

  // ---- the row's loss and constants (warp 0 of every block, the same everywhere)
  if (tid < 32) {
    if (blocks > 1) rest = warp_join(lane < blocks ? parts[lane] : RowStats(), c2);
    RowStats chosen;
    chosen.m = plan.chosen_m, chosen.s = plan.chosen_s;
    const bool repeated = __any_sync(0xffffffffu, lane < blocks && repeats[lane] != 0);
    double merged = 0.0;
    if (repeated) {  // one token: the first place of an id counts, with the mass of all of its places
      chosen.s = 0.f;
      for (int a = lane; a < k; a += 32) {
        bool counts = at[a] >= 0;
        float mass = 0.f;
        for (int i = 0; i < k; ++i) {
          if (at[i] != at[a]) continue;
          counts &= i >= a;
          mass += q_s[i];
        }
        if (counts) chosen.s += e_s[a];
        // q_gap has a term q_k ln q_k for each place; the token's is q ln q, its places' q_k ln q in sum
        if (q_s[a] > 0.f) merged += q_s[a] * log(static_cast<double>(mass) / q_s[a]);
      }
      chosen.s = warp_sum(chosen.s);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) merged += __shfl_xor_sync(0xffffffffu, merged, o);
    }
    RowStats all = chosen;
    all.merge(rest, c2);
    // The student's mass at and outside the alternatives. With ln p_k = ln 2 y_k - ln S_a + ln p_a the loss is
    //   sum q (ln q - ln 2 y + ln S_a) - q_sum ln p_a + q_rest (ln q_rest - ln p_rest)
    // whose first part is known before the row is, in 64 bits, and whose logarithms are of masses: small numbers, so
    // a small divergence keeps its digits. (Below 1e-30 a mass's logarithm comes from its parts.)
    const float q_sum = plan.q_sum, q_rest = rest.s == 0.f ? 0.f : plan.q_rest;
    const float to_p = chosen.s == 0.f ? 0.f : exp2_fast((chosen.m - all.m) * c2) / all.s, p_chosen = chosen.s * to_p;
    const float p_rest = rest.s == 0.f ? 0.f : exp2_fast((rest.m - all.m) * c2) * rest.s / all.s;
    // (in 64 bits where it comes from the parts: (x - m) / T of a token masked by the lowest value leaves fp32's range at
    // T < 1, while the teacher's mass times it may not)
    auto log_mass = [&](float p, const RowStats& of) {
      return p > 1e-30f ? static_cast<double>(logf(p))
                        : static_cast<double>(of.m - all.m) * inv_t + kLn2 * (log2f(of.s) - log2f(all.s));
    };
    float loss = 0.f;
    if (q_sum > 0.f) {  // (a masked token with mass: q_gap is +inf)
      const double log_chosen = repeated ? log(static_cast<double>(chosen.s)) : plan.log_chosen;
      loss = chosen.s == 0.f ? INFINITY
                             : static_cast<float>(plan.q_gap + merged + q_sum * (log_chosen - log_mass(p_chosen, chosen)));
    }
    if (q_rest > 0.f) loss += static_cast<float>(q_rest * (logf(q_rest) - log_mass(p_rest, rest)));
    const bool empty = all.s == 0.f;  // every logit is masked: no distribution, no gradient
    if (empty) loss = INFINITY;
    if (plan.bad) loss = NAN;
    const float scale = w * inv_t, whole = q_sum + q_rest;
    const float outside = rest.s == 0.f ? 0.f : scale * (q_sum * p_rest - q_rest * p_chosen) / rest.s;
    if (GRAD) {
      for (int a = lane; a < k; a += 32) {
        float mass = q_s[a];
        if (repeated) {  // ... with the mass of all of its places
          mass = 0.f;
          for (int i = 0; i < k; ++i) mass += at[i] == at[a] ? q_s[i] : 0.f;
        }
        const float d = plan.bad ? NAN : empty ? 0.f : scale * (whole * (e_s[a] * to_p) - mass);
        e_s[a] = d;
        if (part == 0) saved_chosen[r * k + a] = d;
      }
    }
    if (lane == 0) {
      if (part == 0) rows_out[r] = loss, weighted[r] = w == 0.f ? 0.f : w * loss;  // (a loss may be infinite or NaN)
      plan.masked = w == 0.f;
      plan.base = rest.s == 0.f ? 0.f : rest.m;  // (every other logit is -inf there)
      plan.outside = plan.bad ? NAN : outside;
      if (GRAD && part == 0) saved[r] = make_float2(w == 0.f ? INFINITY : plan.base, plan.outside);
    }
  }
  if constexpr (GRAD) {
    __syncthreads();
    T* out = dlogits + r * v;
    if (plan.masked) return write_zeros<T, kDistillThreads>(out + first, last - first);
    write_gradient<T, kDistillThreads, true, 1>(kept_values, out + first, last - first, plan.base, c2, plan.outside, 0.f);
    __syncthreads();
    if (tid < k && at[tid] >= first && at[tid] < last) out[at[tid]] = from_float<T>(e_s[tid]);
  }
}

// total = sum of x, in an order that depends on n alone.
__global__ void __launch_bounds__(1024) sum_kernel(const float* __restrict__ x, int64_t n, float* __restrict__ total) {
  __shared__ float scratch[32];
  float s = 0.f;
  for (int64_t i = threadIdx.x; i < n; i += blockDim.x) s += x[i];
  s = block_sum(s, scratch);
  if (threadIdx.x == 0) *total = s;
}

// The gradient once more, for an upstream gradient other than one: from the logits, the reference and the constant A of
// each row and the unrounded gradients of its alternatives, so that it is rounded once and an fp16 loss scale meets the
// values before they are lost (w = 1 / 4096 puts every p below 1e-4 under fp16's smallest step). One read and one write of
// the logits, as scaling the rounded gradient would be. A reference of infinity marks a row whose zeros (or NaN) stay.
constexpr int kAgainBytes = 32768;
template <typename T, typename I>
__global__ void __launch_bounds__(kDistillThreads)
    distill_again_kernel(const T* __restrict__ logits, RowLayout layout, int v, int64_t items, int parts,
                         const I* __restrict__ ids, int k, const float2* __restrict__ saved,
                         const float* __restrict__ saved_chosen, const float* __restrict__ factor, float c2,
                         T* __restrict__ dlogits) {
  constexpr int kStretch = kAgainBytes / static_cast<int>(sizeof(T));
  const float f = *factor;
  if (f == 1.f) return;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / parts;
    const int first = static_cast<int>(item - r * parts) * kStretch, n = min(kStretch, v - first);
    const float2 s = saved[r];
    if (s.x == INFINITY) continue;
    T* out = dlogits + r * v;
    write_gradient<T, kDistillThreads, true, 4>(logits + layout.offset(static_cast<uint32_t>(r)) + first, out + first, n,
                                                s.x, c2, f * s.y, 0.f);
    __syncthreads();
    for (int j = threadIdx.x; j < k; j += kDistillThreads) {
      const int64_t id = static_cast<int64_t>(ids[r * k + j]);
      if (id >= first && id < first + n) out[id] = from_float<T>(f * saved_chosen[r * k + j]);
    }
  }
}

constexpr int kMostShared = 200 * 1024;

// A row is split so that a block's stretch takes at most about 40 KB (with the gradient: five blocks' worth of
// shared memory on an SM) or, where rows are few, until every SM holds four blocks; a stretch stays several
// vectors a thread. (Without the gradient a finer split costs more, by each block's own start, than the fuller
// last round of blocks gives: 152 us against 129 for 2000 rows of 151936.)
int blocks_per_row(int64_t rows, int64_t vocab, int64_t item, bool grad) {
  const int64_t round = 4 * num_sms(), bytes = vocab * item;
  int blocks = 1;
  while (grad && blocks < kMaxCluster && bytes > 40960 * blocks) blocks *= 2;
  while (blocks < 8 && rows * blocks * 2 <= round && bytes / (blocks * 2) >= kDistillThreads * 16) blocks *= 2;
  return blocks;
}

}  // namespace

// (total [], the rows' divergences, the gradient like logits, what distill_again needs); the last two are undefined
// where no gradient is asked for.
std::vector<at::Tensor> distill_fwd(const at::Tensor& logits_in, const at::Tensor& ids, const at::Tensor& teacher,
                                    const c10::optional<at::Tensor>& weights, double temperature, bool tail, bool grad) {
  check_logits(logits_in, "distillation_loss");
  const int64_t vocab = logits_in.size(-1), rows = logits_in.numel() / vocab;
  check_cuda_tensor(ids, "teacher_ids");
  check_cuda_tensor(teacher, "teacher_log_probs");
  TDSV_CHECK(ids.dim() == logits_in.dim() && ids.size(-1) >= 1 && ids.size(-1) <= kMaxAlternatives &&
                 ids.numel() == rows * ids.size(-1),
             "distillation_loss: teacher_ids must be [..., 1 .. ", kMaxAlternatives, "]");
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
  auto row_loss = at::empty(logits.sizes().slice(0, logits.dim() - 1), f32);
  auto weighted = at::empty({rows}, f32);  // each row's share of the total
  auto total = at::empty({}, f32);         // (no view: autograd refuses to update a Function's view in place)
  auto dlogits = grad ? at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous))
                      : at::Tensor();
  const int k = static_cast<int>(ids.size(-1));
  auto saved = grad ? at::empty({rows * (k + 2)}, f32) : at::Tensor();  // per row: reference and A; then its alternatives
  if (rows == 0) return {total.zero_(), row_loss, dlogits, saved};
  const int item = static_cast<int>(logits.element_size());
  const int blocks = blocks_per_row(rows, vocab, item, grad);
  // the largest stretch of a block: its vectors, one ahead and one after, and a bit for each value
  const int64_t vecs = (vocab * item / 16 + blocks - 1) / blocks, values = vecs * 16 / item;
  const int64_t smem = (grad ? (vecs + 2) * 16 : 0) + ((values + 16 / item + 31) / 32 + 1) * 4;
  TDSV_CHECK(smem <= kMostShared, "distillation_loss: vocabulary too large");
  TDSV_CHECK(rows * blocks < (int64_t(1) << 31), "distillation_loss: too many rows");
  const float c2 = static_cast<float>(1.4426950408889634 / temperature), inv_t = static_cast<float>(1.0 / temperature);
  auto run = [&](auto* tag, auto* itag, auto has_grad) {
    using T = std::remove_pointer_t<decltype(tag)>;
    using I = std::remove_pointer_t<decltype(itag)>;
    auto kern = distill_kernel<T, I, decltype(has_grad)::value>;
    static std::once_flag once;
    std::call_once(once, [&] {
      TDSV_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostShared));
      TDSV_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    });
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(rows * blocks));
    config.blockDim = dim3(kDistillThreads);
    config.dynamicSmemBytes = static_cast<size_t>(smem);
    config.stream = stream();
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(blocks);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    TDSV_CUDA_CHECK(cudaLaunchKernelEx(
        &config, kern, static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab),
        static_cast<const I*>(ids.data_ptr<I>()), static_cast<const float*>(teacher.data_ptr<float>()), k,
        static_cast<const float*>(weighted_rows ? weights->data_ptr<float>() : nullptr), c2, inv_t, tail,
        row_loss.data_ptr<float>(), weighted.data_ptr<float>(), grad ? static_cast<T*>(dlogits.data_ptr()) : nullptr,
        grad ? reinterpret_cast<float2*>(saved.data_ptr<float>()) : nullptr,
        grad ? saved.data_ptr<float>() + 2 * rows : nullptr, status_word_ptr()));
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
  sum_kernel<<<1, static_cast<unsigned>(std::min<int64_t>(1024, (rows + 31) / 32 * 32)), 0, stream()>>>(
      weighted.data_ptr<float>(), rows, total.data_ptr<float>());
  TDSV_LAUNCH_CHECK();
  return {total, row_loss, dlogits, saved};
}

// dlogits for an upstream gradient of `factor` (a device scalar), in place; nothing is touched where it is one.
void distill_again(at::Tensor& dlogits, const at::Tensor& logits_in, const at::Tensor& ids, const at::Tensor& saved,
                   const at::Tensor& factor, double temperature) {
  check_logits(logits_in, "distillation_loss");
  const int64_t vocab = logits_in.size(-1), rows = logits_in.numel() / vocab;
  check_cuda_tensor(dlogits, "dlogits");
  check_cuda_tensor(ids, "teacher_ids");
  check_cuda_tensor(saved, "saved");
  check_cuda_tensor(factor, "gradient");
  TDSV_CHECK(dlogits.sizes() == logits_in.sizes() && dlogits.scalar_type() == logits_in.scalar_type(),
             "distillation_loss: gradient like the logits");
  TDSV_CHECK(factor.scalar_type() == at::kFloat && factor.numel() == 1, "distillation_loss: fp32 scalar gradient");
  if (rows == 0) return;
  const int k = static_cast<int>(ids.size(-1));
  TDSV_CHECK(ids.numel() == rows * k && saved.scalar_type() == at::kFloat && saved.numel() == rows * (k + 2),
             "distillation_loss: saved rows");
  c10::cuda::CUDAGuard guard(logits_in.device());
  RowLayout layout;
  at::Tensor logits = logits_in;
  if (!row_layout(logits, layout)) {
    logits = logits.contiguous();
    TDSV_CHECK(row_layout(logits, layout), "distillation_loss: logits layout");
  }
  const float c2 = static_cast<float>(1.4426950408889634 / temperature);
  const int64_t stretch = kAgainBytes / logits.element_size(), parts = (vocab + stretch - 1) / stretch;
  // (eight blocks an SM, so that a factor of one costs a launch and not a pass over the rows)
  const unsigned grid = static_cast<unsigned>(std::min<int64_t>(rows * parts, 8 * num_sms()));
  with_logit_type(logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto run = [&](auto* itag) {
      using I = std::remove_pointer_t<decltype(itag)>;
      distill_again_kernel<T, I><<<grid, kDistillThreads, 0, stream()>>>(
          static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab), rows * parts, static_cast<int>(parts),
          ids.data_ptr<I>(), k, reinterpret_cast<const float2*>(saved.data_ptr<float>()),
          saved.data_ptr<float>() + 2 * rows, factor.data_ptr<float>(), c2, static_cast<T*>(dlogits.data_ptr()));
    };
    if (ids.scalar_type() == at::kLong) run(static_cast<int64_t*>(nullptr));
    else run(static_cast<int32_t*>(nullptr));
  });
  TDSV_LAUNCH_CHECK();
}

}  // namespace tdsv
