// Statistics of rows of logits at a temperature T (y = x / T, p = softmax(y)):
//
//   log_probs  ln p of one given token per row
//   entropy    H = -sum p ln p
//   top        the k largest logits, ties to the lowest index, with their ln p
//
// and the gradient of all three. With upstream g (log-probability), h (entropy), u_j (alternatives):
//   dx_i = [ g (d_it - p_i) + sum_j u_j (d_ij - p_i) - h p_i (ln p_i + H) ] / T
//
// where ln p_i + H = ln 2 (y_i - W / S) in the terms of logit_rows.cuh: the logarithm of S drops out, so the
// entropy's gradient stays exact where one token has nearly all of the mass.
//
// A row whose target is the ignore index is not read: zeros, ids -1, zero gradient. Masked logits
// (-inf) have p = 0 and are never alternatives (id -1, ln p = -inf). A row that is masked throughout
// has ln p = -inf, H = 0 and no gradient. NaN or +inf in a row that is read gives NaN.
#include "logit_rows.cuh"

#include <cfloat>

#include <cooperative_groups.h>

namespace tdsv {

namespace {

constexpr int kStatThreads = 256;
constexpr int kMaxTop = 128;
constexpr int kUnroll = 4;          // vectors a thread has in flight
constexpr int kBatch = kStatThreads * kUnroll;
constexpr int kCandidates = 2176;   // candidates for the alternatives that a block can hold: kKept vectors' values too
constexpr int kMaxCluster = 8;

// Floats as whole numbers of the same order (both zeros are one value), and back.
__device__ __forceinline__ uint32_t order_key(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
constexpr uint32_t kMaskedKey = 0x007fffffu;  // of -inf: every finite value's key is larger
constexpr uint32_t kInfKey = 0xff800000u;     // of +inf: NaN's keys are larger
// A candidate: the larger value first, then the lower index.
__device__ __forceinline__ uint64_t candidate(uint32_t key, int i) {
  return static_cast<uint64_t>(key) << 32 | (0xffffffffu - static_cast<uint32_t>(i));
}
__device__ __forceinline__ uint32_t candidate_key(uint64_t c) { return static_cast<uint32_t>(c >> 32); }

// Values of a 16-bit type differ in the key's upper bits alone: thresholds move in those.
template <typename T>
constexpr int kKeyShift = std::is_same_v<T, __nv_bfloat16> ? 16 : std::is_same_v<T, __half> ? 13 : 0;

// The largest threshold found in [lo, hi) that at least `want` reach, given that this holds at lo and not at
// hi: halving steps, until at most `want + slack` reach it or nothing lies between. `count(t)` gives every
// caller the number that reach t; `kept` is that number at the result, if it was counted.
template <typename F>
__device__ __forceinline__ uint32_t raise_threshold(uint32_t lo, uint32_t hi, int want, int slack, int& kept, F&& count) {
  while (hi - lo > 1) {
    const uint32_t mid = lo + (hi - lo) / 2;
    const int all = count(mid);
    if (all >= want) {
      lo = mid;
      kept = all;
      if (all <= want + slack) break;
    } else {
      hi = mid;
    }
  }
  return lo;
}
// The same in quarters: count3(a, b, c) gives three numbers, 10 bits each, so a step takes two halvings.
template <typename F>
__device__ __forceinline__ uint32_t raise_threshold_by4(uint32_t lo, uint32_t hi, int want, int slack, int& kept,
                                                        F&& count3) {
  while (hi - lo > 1) {
    const uint32_t d = hi - lo, a = lo + max(d / 4, 1u), b = max(lo + d / 2, a), c = max(lo + d / 4 * 3, b);
    const uint32_t all = count3(a, b, c);
    const int na = all & 1023u, nb = all >> 10 & 1023u, nc = all >> 20;
    if (nc >= want) lo = c, kept = nc;
    else if (nb >= want) lo = b, hi = c, kept = nb;
    else if (na >= want) lo = a, hi = b, kept = na;
    else hi = a;
    if (kept >= want && kept <= want + slack) break;
  }
  return lo;
}

constexpr int kKept = 2 * kMaxTop;
static_assert(kCandidates >= 8 * kKept + 2 * 7, "the values of the kept vectors fit");
struct TopScratch {
  uint64_t kept[kKept];          // the selected candidates, before they are ranked
  uint32_t maxima[kStatThreads]; // of each thread's first batch
  int counts[16];
  int n, kept_n, gathered;
  float first, threshold;
};

// One warp's threshold over n keys, `stride` words apart, from `lo` up (or from below, should fewer than `want`
// reach it); `kept` keys reach the result. A selection is a chain of short steps: one warp takes it through
// without a block barrier, its keys in registers (32 kRegs of them; more are read again each step). The keys
// may still be arriving: a threshold that enough of them reach only gets easier to reach.
template <typename T, int kRegs>
__device__ __forceinline__ uint32_t warp_threshold(const volatile uint32_t* keys, int stride, int n, uint32_t lo,
                                                   int want, int slack, int& kept) {
  constexpr int kShift = kKeyShift<T>;
  const int lane = threadIdx.x & 31;
  lo >>= kShift;
  uint32_t k[kRegs], hi = 0, least = 0xffffffffu;
#pragma unroll
  for (int j = 0; j < kRegs; ++j) {
    // (places beyond n hold 0, which reaches no threshold above 0)
    k[j] = j * 32 + lane < n ? keys[(j * 32 + lane) * stride] >> kShift : 0;
    hi = max(hi, k[j]);
    if (j * 32 + lane < n) least = min(least, k[j]);
  }
  for (int i = kRegs * 32 + lane; i < n; i += 32) {
    hi = max(hi, keys[i * stride] >> kShift);
    least = 0;
  }
  hi = __reduce_max_sync(0xffffffffu, hi) + 1;
  lo = max(lo, __reduce_min_sync(0xffffffffu, least));  // all n reach the least
  auto count = [&](uint32_t t) {
    int c = 0;
#pragma unroll
    for (int j = 0; j < kRegs; ++j) c += k[j] >= t;
    for (int i = kRegs * 32 + lane; i < n; i += 32) c += keys[i * stride] >> kShift >= t;
    return static_cast<int>(__reduce_add_sync(0xffffffffu, c));
  };
  kept = count(lo);
  if (kept < want) {
    lo = 0;
    kept = n;
  }
  if (kept <= want + slack) return lo << kShift;
  if (n > kRegs * 32) return raise_threshold(lo, max(hi, lo + 1), want, slack, kept, count) << kShift;
  return raise_threshold_by4(lo, max(hi, lo + 1), want, slack, kept, [&](uint32_t ta, uint32_t tb, uint32_t tc) {
    uint32_t ca = 0, cb = 0, cc = 0;
#pragma unroll
    for (int j = 0; j < kRegs; ++j) ca += k[j] >= ta, cb += k[j] >= tb, cc += k[j] >= tc;
    return __reduce_add_sync(0xffffffffu, ca | cb << 10 | cc << 20);
  }) << kShift;
}

// The value from which a threshold's unit starts; the lowest finite one where that is masked (-inf) or NaN, so
// that what reaches a threshold is never either.
template <typename T>
__device__ __forceinline__ float threshold_value(uint32_t t) {
  return t >> kKeyShift<T> <= kMaskedKey >> kKeyShift<T> || t > kInfKey ? -FLT_MAX : key_value(t);
}

// One warp: the candidates among the n in `buf` whose key reaches the want-th largest (all where there are
// fewer; 0 fills places without one) go to sc.kept, in any order, and their number is returned. Where more are
// equal at the end than fit, those above and the `want` lowest indices of the equal ones go.
template <typename T>
__device__ __forceinline__ int select_top(const uint64_t* buf, int n, uint32_t lo, int want, TopScratch& sc) {
  constexpr int kShift = kKeyShift<T>;
  const int lane = threadIdx.x & 31;
  uint64_t least = 1;  // the first candidate that is kept
  if (n > want) {
    int kept = 0;
    const uint32_t cut = max(warp_threshold<T, 16>(reinterpret_cast<const uint32_t*>(buf) + 1, 2, n, lo, want, 0, kept), 1u);
    least = static_cast<uint64_t>(cut) << 32;
    if (kept > kKept && cut >> kShift != 0) {
      auto tied = [&](uint64_t c) { return candidate_key(c) >> kShift == cut >> kShift; };
      int above = 0;
      uint32_t key = 0;  // (one unit of keys holds one value)
      for (int i = lane; i < n; i += 32) {
        above += candidate_key(buf[i]) >> kShift > cut >> kShift;
        if (tied(buf[i])) key = candidate_key(buf[i]);
      }
      above = __reduce_add_sync(0xffffffffu, above);
      const uint32_t t = raise_threshold(0, 0xffffffffu, want, kKept - want - above, kept, [&](uint32_t at) {
        int c = 0;
        for (int i = lane; i < n; i += 32) c += tied(buf[i]) && static_cast<uint32_t>(buf[i]) >= at;
        return static_cast<int>(__reduce_add_sync(0xffffffffu, c));
      });
      least = static_cast<uint64_t>(__reduce_max_sync(0xffffffffu, key)) << 32 | t;
    }
  }
  int m = 0;
#pragma unroll 4
  for (int i0 = 0; i0 < n; i0 += 32) {
    const uint64_t c = i0 + lane < n ? buf[i0 + lane] : 0;
    const bool keep = c >= least;
    const uint32_t mask = __ballot_sync(0xffffffffu, keep);
    const int at = m + __popc(mask & ((1u << lane) - 1u));
    if (keep && at < kKept) sc.kept[at] = c;
    m += __popc(mask);
  }
  __syncwarp();
  return min(m, kKept);
}

// The block: ranks the m kept candidates by counting, four threads to each; emit(rank, candidate) once each.
template <typename F>
__device__ __forceinline__ void rank_kept(const TopScratch& sc, int m, F&& emit) {
  const int quarter = threadIdx.x & 3;
  for (int i0 = 0; i0 < m; i0 += kStatThreads / 4) {
    const int i = i0 + static_cast<int>(threadIdx.x >> 2);
    const uint64_t c = i < m ? sc.kept[i] : 0;
    int rank = 0;
#pragma unroll 4
    for (int j = quarter; j < m; j += 4) rank += sc.kept[j] > c;
    rank += __shfl_xor_sync(0xffffffffu, rank, 1);
    rank += __shfl_xor_sync(0xffffffffu, rank, 2);
    if (quarter == 0 && i < m) emit(rank, c);
  }
}

// The exact way for a block's part of a row whose candidates do not fit (rows in rising order, thousands of
// equal values): halve the value, then the index among equals, re-reading the part each time, until what is
// left fits. The whole block takes part. Returns the number of candidates put into `buf`.
template <typename T>
__device__ __noinline__ int collect_again(const T* row, int first, int last, int want, uint64_t* buf, TopScratch& sc) {
  constexpr int kShift = kKeyShift<T>;
  auto block_count = [&](auto&& hit) {
    int c = 0;
    for (int i = first + threadIdx.x; i < last; i += kStatThreads) c += hit(order_key(to_float<T>(row[i])), i);
    c = __reduce_add_sync(0xffffffffu, c);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sc.counts[threadIdx.x >> 5] = c;
    __syncthreads();
    c = 0;
    for (int w = 0; w < kStatThreads / 32; ++w) c += sc.counts[w];
    return c;
  };
  int kept = 0;
  // (+inf is the largest key that counts; NaN lies above it)
  uint32_t cut = raise_threshold(kMaskedKey >> kShift, (kInfKey >> kShift) + 1, want, kCandidates - want, kept,
                                 [&](uint32_t t) { return block_count([&](uint32_t k, int) { return k >> kShift >= t; }); });
  int until = last;  // of the values at `cut`, those before this index
  if (cut == kMaskedKey >> kShift) {
    cut = (kMaskedKey >> kShift) + 1;  // fewer than `want` are unmasked
  } else if (kept > kCandidates) {
    const int above = block_count([&](uint32_t k, int) { return k >> kShift > cut; });
    // (an index counts down, so that "at least" is again a threshold from below)
    until = last - static_cast<int>(raise_threshold(0, static_cast<uint32_t>(last - first), want - above, 0, kept, [&](uint32_t t) {
              return block_count([&](uint32_t k, int i) {
                return k >> kShift == cut && static_cast<uint32_t>(last - 1 - i) >= t;
              });
            }));
  }
  __syncthreads();
  if (threadIdx.x == 0) sc.n = 0;
  __syncthreads();
  for (int i = first + threadIdx.x; i < last; i += kStatThreads) {
    const uint32_t key = order_key(to_float<T>(row[i]));
    if (key > kInfKey || key >> kShift < cut || (key >> kShift == cut && i >= until)) continue;
    const int at = atomicAdd(&sc.n, 1);
    if (at < kCandidates) buf[at] = candidate(key, i);
  }
  __syncthreads();
  return min(sc.n, kCandidates);
}

// A block (or a cluster of blocks, each on a stretch of the row) reads a row once in 16-byte vectors.
//
// Alternatives are found by whole vectors first: a vector is a candidate when its maximum reaches a threshold
// that the maxima of at least `top` vectors reach. The first threshold comes from the threads' maxima of the
// first batch; later vectors have to pass it (equal values there lose by their index), and it is raised after 2,
// 4, 8, ... batches, so that a row gives some top * log2 of its batches candidates. The common step costs one
// comparison for a thread's batch, a candidate some 20 instructions (by single values it was 67, and 4096 rows
// with 64 alternatives took 546 us). At the end the `top` first vectors hold all of the `top` first values: they
// are read once more, value by value.
//
// Bound by memory without alternatives: 3001 rows of 151936 bf16 take 144 us, 6.3 TB/s. With 64 alternatives 4096 rows
// take 340 us (3.7 TB/s): the selections of a row are serial phases that the four blocks of an SM cover in part.
// Four blocks of 256 threads hold 64 KB of loads in flight an SM, which the registers allow and the latency needs.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kStatThreads, 4)
    stats_fwd_kernel(const T* __restrict__ logits, RowLayout layout, int v, const int64_t* __restrict__ targets,
                     int64_t ignore_index, float c2, float inv_t, int top, float* __restrict__ log_probs,
                     float* __restrict__ entropy, int64_t* __restrict__ top_ids, float* __restrict__ top_lp,
                     float4* __restrict__ saved, int* status) {
  namespace cg = cooperative_groups;
  constexpr int kSize = LogitVec<T>::kSize;
  extern __shared__ __align__(16) uint64_t top_smem[];  // [kCandidates], then [blocks of the cluster][kKept]
  __shared__ JoinScratch<kStatThreads> scratch;
  __shared__ RowStats parts[kMaxCluster];
  __shared__ TopScratch sc;
  const cg::cluster_group cluster = cg::this_cluster();
  const int blocks = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
  const int tid = threadIdx.x;
  const int64_t r = blockIdx.x / static_cast<unsigned>(blocks);
  const T* row = logits + layout.offset(static_cast<uint32_t>(r));
  const RowCut cut = cut_row(row, v);
  const int per = (cut.vecs + blocks - 1) / blocks;
  const int v0 = min(cut.vecs, part * per), v1 = min(cut.vecs, v0 + per);
  const uint4* base = reinterpret_cast<const uint4*>(row + cut.head);
  uint4 next[kUnroll];  // on its way while the batch before is summed
  auto load = [&](int from) {
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = from + u * kStatThreads + tid;
      if (i < v1) next[u] = load_stream(base + i);
    }
  };
  load(v0);  // (before the target is known: it arrives at the same time)
  const int64_t target = targets != nullptr ? targets[r] : 0;
  if (targets != nullptr && target == ignore_index) {  // (the whole cluster leaves)
    if (part != 0) return;
    if (tid == 0) {
      log_probs[r] = 0.f;
      entropy[r] = 0.f;
      if (saved != nullptr) saved[r] = saved_stats(RowStats());
    }
    for (int j = tid; j < top; j += kStatThreads) {
      top_ids[r * top + j] = -1;
      top_lp[r * top + j] = -INFINITY;
    }
    return;
  }
  // every block of the cluster runs before another writes to its shared memory (waited for below)
  if (blocks > 1) {
    if (TOP && tid == 0) sc.gathered = 0;
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  }
  // the values before the first vector and after the last: one per thread, of two warps
  float single = -INFINITY;
  int single_at = 0;
  if (part == 0 && tid < cut.head) single_at = tid, single = to_float<T>(row[tid]);
  if (part == blocks - 1 && tid >= 32 && tid < 32 + cut.tail)
    single_at = v - cut.tail + tid - 32, single = to_float<T>(row[single_at]);
  VecStats<true> st;

  if constexpr (TOP) {
    // (a place that is taken but not yet written reads as no candidate)
    for (int i = tid; i < kCandidates / 2; i += kStatThreads) reinterpret_cast<uint4*>(top_smem)[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) sc.n = 0, sc.threshold = -FLT_MAX;
    __syncthreads();
  }
  int batch = 0;
  // a batch of which every thread has all vectors, or the last one
  auto step = [&](auto whole, int from) {
    uint4 now[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) now[u] = next[u];
    float tops[kUnroll], mx = -INFINITY;
    const int mine = decltype(whole)::value ? kUnroll : (v1 - from - tid + kStatThreads - 1) / kStatThreads;
    if constexpr (TOP || !decltype(whole)::value) {
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const uint4 one[1] = {now[u]};
        tops[u] = u < mine ? vec_max<T, 1>(one) : -INFINITY;
        mx = fmaxf(mx, tops[u]);
      }
    } else {
      mx = vec_max<T, kUnroll>(now);
    }
    if (from + kBatch < v1) load(from + kBatch);
    if (batch == 0) st.start(warp_max(mx), c2);
    if (mx > st.limit) st.raise(mx, c2);
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
      if (u < mine) st.add_vec<T>(now[u], c2);
    if constexpr (TOP) {
      float threshold;
      if (batch == 0) {
        sc.maxima[tid] = order_key(mx);
        __syncthreads();
        if (tid < 32) {
          int kept;
          const uint32_t t = warp_threshold<T, kStatThreads / 32>(sc.maxima, 1, kStatThreads, 0, top, top / 4, kept);
          if (tid == 0) {
            sc.first = threshold_value<T>(t);
            sc.threshold = threshold_value<T>(max(t, kMaskedKey) + (1u << kKeyShift<T>));
          }
        }
        __syncthreads();
        threshold = sc.first;
      } else {
        threshold = *const_cast<volatile float*>(&sc.threshold);
      }
      if (mx >= threshold) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
          if (tops[u] >= threshold) {
            const int at = atomicAdd(&sc.n, 1);
            if (at < kCandidates) top_smem[at] = candidate(order_key(tops[u]), from + u * kStatThreads + tid);
          }
      }
      // after 2, 4, 8, ... batches a warp, another each time, raises the threshold; the others go on meanwhile
      if (batch > 0 && ((batch + 1) & batch) == 0 && from + 2 * kBatch < v1 && tid >> 5 == (__ffs(batch + 1) & 7)) {
        // (other warps add candidates and may raise the threshold meanwhile: one lane reads both for the warp, whose
        // branches and reductions have to be the same for every lane)
        __syncwarp();
        int n = 0;
        if ((tid & 31) == 0) {
          n = min(*const_cast<volatile int*>(&sc.n), kCandidates);
          threshold = *const_cast<volatile float*>(&sc.threshold);
        }
        n = __shfl_sync(0xffffffffu, n, 0);
        threshold = __shfl_sync(0xffffffffu, threshold, 0);
        if (n > top) {
          const uint32_t* keys = reinterpret_cast<const uint32_t*>(top_smem) + 1;
          int kept;
          const uint32_t t = warp_threshold<T, 8>(keys, 2, n, order_key(threshold), top, top / 4, kept);
          if ((tid & 31) == 0 && t > order_key(threshold)) *const_cast<volatile float*>(&sc.threshold) = threshold_value<T>(t);
        }
      }
    }
    ++batch;
  };
  int from = v0;
  for (; from + kBatch <= v1; from += kBatch) step(std::true_type{}, from);
  if (from < v1) step(std::false_type{}, from);
  if (single != -INFINITY) st.add_one(single, c2);
  RowStats all = block_join<kStatThreads>(st.total(), c2, scratch);
  if (blocks > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // the row's candidates: this block's, or what every block of the cluster sends to the first one
  int row_n = 0;
  if constexpr (TOP) {
    __syncthreads();
    const int n = sc.n;
    const uint32_t lo = order_key(sc.threshold);
    __syncthreads();
    if (n > kCandidates) {
      const int first = part == 0 ? 0 : cut.head + v0 * kSize;
      const int last = part == blocks - 1 ? v : cut.head + v1 * kSize;
      row_n = collect_again(row, first, last, top, top_smem, sc);
    } else {
      if (tid < 32) {
        const int m = select_top<T>(top_smem, n, lo, top, sc);
        // the least maximum of `top` vectors, from which a value can be among the first
        uint32_t least = 0xffffffffu;
        for (int j = tid; j < m; j += 32) least = min(least, candidate_key(sc.kept[j]));
        least = __reduce_min_sync(0xffffffffu, least);
        if (tid == 0) sc.kept_n = m, sc.n = 0, sc.first = m < top ? -FLT_MAX : key_value(least);
      }
      __syncthreads();
      const int m = sc.kept_n;
      const float least = sc.first;
      auto push = [&](float x, int i) {
        if (!(x >= least)) return;
        top_smem[atomicAdd(&sc.n, 1)] = candidate(order_key(x), i);  // (kKept vectors fit, and the single values)
      };
      for (int j = tid; j < m * kSize; j += kStatThreads) {
        const int i = cut.head + static_cast<int>(0xffffffffu - static_cast<uint32_t>(sc.kept[j / kSize])) * kSize + j % kSize;
        push(to_float<T>(row[i]), i);
      }
      push(single, single_at);
      __syncthreads();
      row_n = sc.n;
    }
    if (blocks > 1) {
      // this block's first `top`, in any order, behind the other blocks' in the leader's shared memory
      if (tid < 32) {
        const int m = select_top<T>(top_smem, row_n, 0, top, sc);
        int first = 0;
        if (tid == 0) first = atomicAdd(cluster.map_shared_rank(&sc.gathered, 0), m);
        first = __shfl_sync(0xffffffffu, first, 0);
        uint64_t* lead = cluster.map_shared_rank(top_smem, 0) + kCandidates + first;
        for (int j = tid; j < m; j += 32) lead[j] = sc.kept[j];
      }
    }
  }
  if (blocks > 1) {
    if (tid == 0) *cluster.map_shared_rank(&parts[part], 0) = all;
    cluster.sync();
    if (part != 0) return;
    all = warp_join((tid & 31) < blocks ? parts[tid & 31] : RowStats(), c2);
    if (TOP) row_n = sc.gathered;
  }
  if constexpr (TOP) {
    if (tid < 32) {
      const int m = select_top<T>(top_smem + (blocks > 1 ? kCandidates : 0), row_n, 0, top, sc);
      if (tid == 0) sc.kept_n = m;
    }
    __syncthreads();
    const int m = sc.kept_n;
    const float log_s = kLn2 * log2f(all.s);
    for (int j = min(m, top) + tid; j < top; j += kStatThreads) {
      top_ids[r * top + j] = -1;
      top_lp[r * top + j] = -INFINITY;
    }
    rank_kept(sc, m, [&](int rank, uint64_t c) {
      if (rank >= top) return;
      top_ids[r * top + rank] = 0xffffffffu - static_cast<uint32_t>(c);
      top_lp[r * top + rank] = (key_value(candidate_key(c)) - all.m) * inv_t - log_s;
    });
  }
  if (tid == 0) {
    const float log2s = log2f(all.s);
    const float ent = all.s == 0.f ? 0.f : kLn2 * (log2s - all.w / all.s);
    entropy[r] = ent;
    if (targets != nullptr) {
      float lp = NAN;
      if (target >= 0 && target < v) {
        lp = all.s == 0.f ? -INFINITY : (to_float<T>(row[target]) - all.m) * inv_t - kLn2 * log2s;
      } else {
        report_status(status, kOutOfBounds);
      }
      log_probs[r] = lp;
    }
    if (saved != nullptr) saved[r] = saved_stats(all);
  }
}

// A block writes the gradient of one stretch of a row: long enough to hide its start, short enough that the last round
// of blocks is short. Bound by memory: one read and one write; 2047 x 151669 in rows that are aligned differently on
// both sides take 311 us with their forward, 1.6 GB at 5.2 TB/s.
constexpr int kStretchBytes = 32768;

template <typename T>
__global__ void __launch_bounds__(kStatThreads)
    stats_bwd_kernel(const T* __restrict__ logits, RowLayout layout, int v, int parts,
                     const int64_t* __restrict__ targets, float c2, float inv_t, int top,
                     const int64_t* __restrict__ top_ids, const float4* __restrict__ saved,
                     const float* __restrict__ g_lp, const float* __restrict__ g_ent, const float* __restrict__ g_top,
                     T* __restrict__ dlogits) {
  __shared__ int at[kMaxTop + 1];
  __shared__ float grad[kMaxTop + 1];
  __shared__ float scratch[32];
  constexpr int kStretch = kStretchBytes / static_cast<int>(sizeof(T));
  const int64_t r = blockIdx.x / static_cast<unsigned>(parts);
  const int first = static_cast<int>(blockIdx.x - static_cast<unsigned>(r) * static_cast<unsigned>(parts)) * kStretch, n = min(kStretch, v - first);
  const T* row = logits + layout.offset(static_cast<uint32_t>(r));
  T* out = dlogits + r * v;
  const float4 s = saved[r];
  if (s.y == 0.f) {  // ignored, or nothing unmasked
    write_zeros<T, kStatThreads>(out + first, n);
    return;
  }
  // places that are not only -p_i (...): the target and the alternatives
  const int64_t target = targets != nullptr ? targets[r] : -1;
  const bool has_target = g_lp != nullptr && target >= 0 && target < v;
  float g = has_target ? g_lp[r] : 0.f;
  if (g_top != nullptr) {
    float mine = 0.f;
    for (int j = threadIdx.x; j <= top; j += kStatThreads) {
      const int64_t id = j < top ? top_ids[r * top + j] : (has_target ? target : -1);
      const bool there = id >= 0 && id < v;
      const float u = !there ? 0.f : j < top ? g_top[r * top + j] : g;
      at[j] = there ? static_cast<int>(id) : -1;
      grad[j] = u;
      mine += u;
    }
    g = block_sum(mine, scratch);
  }
  const float h = g_ent != nullptr ? g_ent[r] * kLn2 : 0.f;
  // T dx_i = 2^y_i (a + b y_i) / S + (d_i terms),  y_i = (x_i - m) c2
  const float a = -(g - h * s.z), b = -h;
  const float scale = inv_t * s.y;
  write_gradient<T, kStatThreads, false, 4>(row + first, out + first, n, s.x, c2, scale * a, scale * b);
  __syncthreads();
  // (u and a cancel where p = 1: they are added before anything is scaled)
  auto special = [&](int i, float u) {
    const float y = fmaxf((to_float<T>(row[i]) - s.x) * c2, kMinExponent);
    out[i] = from_float<T>(inv_t * (u + s.y * exp2_fast(y) * (a + b * y)));
  };
  if (g_top == nullptr) {
    if (threadIdx.x == 0 && has_target && target >= first && target < first + n) special(static_cast<int>(target), g);
    return;
  }
  for (int j = threadIdx.x; j <= top; j += kStatThreads) {
    if (at[j] < first || at[j] >= first + n) continue;
    float u = 0.f;  // equal places write the same sum
    for (int k = 0; k <= top; ++k) u += at[k] == at[j] ? grad[k] : 0.f;
    special(at[j], u);
  }
}

// A row is split over a cluster while there are too few rows for every SM to hold four blocks and each part is
// still several batches of loads. (Beyond that a split only costs: 3001 rows of 151936 take 144 us whole, 6.3 TB/s,
// and 156 in halves; 64 rows take 14.2 us whole, 10.9 in halves and 10.5 in quarters or eighths.)
int blocks_per_row(int64_t rows, int64_t vocab, int64_t item) {
  int blocks = 1;
  while (blocks < kMaxCluster && rows * blocks * 2 <= 4 * num_sms() && vocab * item / (blocks * 2) >= kStatThreads * 16)
    blocks *= 2;
  return blocks;
}

}  // namespace

// (log_probs, entropy, top_ids, top_log_probs, saved) over the rows of logits [..., V]; what is not asked for is
// undefined (None).
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
  const auto shape = logits.sizes().slice(0, logits.dim() - 1);
  at::Tensor log_probs, top_ids, top_lp, saved;
  if (has_target) log_probs = at::empty(shape, f32);
  auto entropy = at::empty(shape, f32);
  if (top > 0) {
    auto wide = shape.vec();
    wide.push_back(top);
    top_ids = at::empty(wide, f32.dtype(at::kLong));
    top_lp = at::empty(wide, f32);
  }
  if (save) saved = at::empty({rows, 4}, f32);
  if (rows == 0) return {log_probs, entropy, top_ids, top_lp, saved};
  const float c2 = static_cast<float>(1.4426950408889634 / temperature), inv_t = static_cast<float>(1.0 / temperature);
  const int blocks = blocks_per_row(rows, vocab, logits.element_size());
  with_logit_type(logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto launch = [&](auto kern, size_t smem) {
      cudaLaunchConfig_t config{};
      config.gridDim = dim3(static_cast<unsigned>(rows * blocks));
      config.blockDim = dim3(kStatThreads);
      config.dynamicSmemBytes = smem;
      config.stream = stream();
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = static_cast<unsigned>(blocks);
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      config.attrs = &attr;
      config.numAttrs = 1;
      TDSV_CUDA_CHECK(cudaLaunchKernelEx(
          &config, kern, static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab),
          static_cast<const int64_t*>(has_target ? targets->data_ptr<int64_t>() : nullptr), ignore_index, c2,
          inv_t, static_cast<int>(top), has_target ? log_probs.data_ptr<float>() : nullptr, entropy.data_ptr<float>(),
          top ? top_ids.data_ptr<int64_t>() : nullptr, top ? top_lp.data_ptr<float>() : nullptr,
          save ? reinterpret_cast<float4*>(saved.data_ptr<float>()) : nullptr, status_word_ptr()));
    };
    if (top > 0) launch(stats_fwd_kernel<T, true>, (kCandidates + (blocks > 1 ? blocks * kKept : 0)) * sizeof(uint64_t));
    else launch(stats_fwd_kernel<T, false>, 0);
  });
  TDSV_LAUNCH_CHECK();
  return {log_probs, entropy, top_ids, top_lp, saved};
}

// Contiguous gradient of the logits, in their shape and type.
at::Tensor token_stats_bwd(const at::Tensor& logits_in, const c10::optional<at::Tensor>& targets,
                           const c10::optional<at::Tensor>& top_ids, const at::Tensor& saved, double temperature,
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
  const bool has_top = top_ids.has_value() && top_ids->defined();
  if (has_top) {
    check_cuda_tensor(*top_ids, "top_ids");
    TDSV_CHECK(top_ids->scalar_type() == at::kLong && top_ids->dim() >= 1 && top_ids->size(-1) <= kMaxTop &&
                   top_ids->numel() == rows * top_ids->size(-1),
               "token_statistics: top_ids");
  }
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
  const int top = has_top ? static_cast<int>(top_ids->size(-1)) : 0;
  const float *g_lp = pointer(g_log_probs, rows), *g_ent = pointer(g_entropy, rows), *g_alt = pointer(g_top, rows * top);
  const float c2 = static_cast<float>(1.4426950408889634 / temperature), inv_t = static_cast<float>(1.0 / temperature);
  const int64_t stretch = kStretchBytes / logits.element_size(), parts = (vocab + stretch - 1) / stretch;
  TDSV_CHECK(rows * parts < (int64_t(1) << 31), "token_statistics: too many rows");
  with_logit_type(logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    stats_bwd_kernel<T><<<static_cast<unsigned>(rows * parts), kStatThreads, 0, stream()>>>(
        static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab), static_cast<int>(parts),
        has_target ? targets->data_ptr<int64_t>() : nullptr, c2, inv_t, top,
        top ? top_ids->data_ptr<int64_t>() : nullptr, reinterpret_cast<const float4*>(saved.data_ptr<float>()), g_lp,
        g_ent, top ? g_alt : nullptr, static_cast<T*>(dlogits.data_ptr()));
  });
  TDSV_LAUNCH_CHECK();
  return dlogits;
}

}  // namespace tdsv
