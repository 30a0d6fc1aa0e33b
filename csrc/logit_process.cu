// What a sampler does to the logits before it draws a token: penalties for tokens that were said, biases, and the
// mask of a grammar. For token v of a row, with c the number of times that the row's history holds v as output
// and `said` whether it holds v at all:
//
//     x <- x / r if x > 0 else x r     where said                      (repetition r)
//     x <- x - f c - p                 where c > 0                     (frequency f, presence p)
//     x <- x + sum of v's biases
//     x <- -inf                        where the grammar's bit is clear
//
// in fp32, rounded once to the logits' type.
//
// A row is cut into slices of the vocabulary, a block each. A block counts the history's tokens of its slice in
// shared memory (whole numbers: the order of the atomics changes nothing), and whoever counts a token first puts it on a
// list. Then it copies the slice under the mask in 16-byte vectors, which never pass through fp32; a vector that the mask
// hides altogether is not read. Last the tokens on the list, few and evenly spread over the threads, are written anew.
// (Applied to the vectors on their way, the penalties cost 224 us in place of 112 at 512 x 151669: frequent tokens are
// neighbours, and the few warps that hold them work off eight tokens a thread, one after another.)
// What bounds it is the chain of a block's phases, each a latency long, so six blocks share an SM with two vectors a thread
// in flight: 512 x 151669 bf16 with histories, biases and masks in 84 us (98 us with four blocks and four vectors), 3.8 TB/s;
// 64 x 129280 fp32 with histories of up to 8192 tokens in 31 us.
#include "logit_rows.cuh"

namespace tdsv {

namespace {

constexpr int kThreads = 256;
constexpr int kAhead = 2;          // vectors or touched tokens a thread has in flight
constexpr int kIds = 4;            // ids of the history
constexpr int kListed = 256;       // biases of a slice that shared memory holds

// A token's count and two flags. 16 bits hold the counts of histories below 2^14 tokens, in half the shared memory, so
// that four blocks of the largest slice fit an SM; longer ones take 32.
template <typename C>
struct Count {
  static constexpr uint32_t kPrompt = sizeof(C) == 2 ? 0x8000u : 0x80000000u, kBiased = kPrompt >> 1, kTimes = kBiased - 1;
  static constexpr int kMost = static_cast<int>(sizeof(C) == 2 ? kTimes : kTimes >> 1);
  // Whether it is the first that is heard of the token.
  static __device__ __forceinline__ bool add(uint32_t* words, int token, uint32_t what, bool flag) {
    constexpr int kEach = 4 / sizeof(C);
    const int shift = token % kEach * 16;
    uint32_t* word = words + token / kEach;
    const uint32_t was = flag ? atomicOr(word, what << shift) : atomicAdd(word, what << shift);
    return (was >> shift & (kPrompt | (kPrompt - 1u))) == 0;
  }
};

template <typename T>
__device__ __forceinline__ uint32_t minus_inf_pair() {  // two of a 16-bit type, or one of fp32
  if constexpr (std::is_same_v<T, __nv_bfloat16>) return 0xff80ff80u;
  else if constexpr (std::is_same_v<T, __half>) return 0xfc00fc00u;
  else return 0xff800000u;
}
template <typename T>
__device__ __forceinline__ uint32_t mask_word(uint32_t w, uint32_t bits) {
  if constexpr (sizeof(T) == 4) {
    return bits & 1u ? w : minus_inf_pair<T>();
  } else {
    const uint32_t keep = (bits & 1u ? 0x0000ffffu : 0u) | (bits & 2u ? 0xffff0000u : 0u);
    return (w & keep) | (minus_inf_pair<T>() & ~keep);
  }
}
template <typename T>
__device__ __forceinline__ uint4 mask_vec(uint4 v, uint32_t bits) {
  constexpr int kStep = 4 / sizeof(T);
  v.x = mask_word<T>(v.x, bits);
  v.y = mask_word<T>(v.y, bits >> kStep);
  v.z = mask_word<T>(v.z, bits >> 2 * kStep);
  v.w = mask_word<T>(v.w, bits >> 3 * kStep);
  return v;
}

// The mask's bits from token `at` of the slice on, `count` (at most 8) of them; all set without a mask.
__device__ __forceinline__ uint32_t mask_bits(const uint32_t* words, int at, int count) {
  if (words == nullptr) return 0xffffffffu;
  const int shift = at & 31;
  uint32_t bits = words[at >> 5] >> shift;
  if (shift + count > 32) bits |= words[(at >> 5) + 1] << (32 - shift);
  return bits;
}

// out[0, n) = row[0, n) where the mask allows it. Vectors are aligned at `out`; where the logits lie at another
// offset in their 16 bytes, two of theirs are joined.
template <typename T>
__device__ __forceinline__ void copy_masked(const T* row, T* out, int n, const uint32_t* words) {
  constexpr int kSize = LogitVec<T>::kSize;
  constexpr uint32_t kAll = (1u << kSize) - 1;
  const RowCut cut = cut_row(out, n);
  const int tid = threadIdx.x;
  const auto one = [&](int i) { out[i] = mask_bits(words, i, 1) & 1u ? row[i] : from_float<T>(-INFINITY); };
  if (tid < cut.head) one(tid);
  if (tid >= 32 && tid < 32 + cut.tail) one(n - cut.tail + tid - 32);
  const T* from = row + cut.head;
  uint4* to = reinterpret_cast<uint4*>(out + cut.head);
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(from) & 15) / sizeof(T));
  // the vectors whose parts all lie inside the row: with an offset, at most the first and the last do not
  const uint4* x = reinterpret_cast<const uint4*>(from - off);
  const int first = off > cut.head ? 1 : 0;
  const int last = off == 0 ? cut.vecs : min(cut.vecs, (n - cut.head + off) / kSize - 1);
  for (int i = first + tid; i < last; i += kThreads * kAhead) {
    uint4 lo[kAhead], hi[kAhead];
    uint32_t bits[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int at = i + u * kThreads;
      bits[u] = at < last ? mask_bits(words, cut.head + at * kSize, kSize) & kAll : 0u;
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (bits[u] == 0) continue;
      lo[u] = load_stream(x + i + u * kThreads);
      if (off != 0) hi[u] = load_stream(x + i + u * kThreads + 1);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (i + u * kThreads >= last) continue;
      uint4 v = lo[u];
      if (off != 0) v = shift_vec(lo[u], hi[u], off * static_cast<int>(sizeof(T)));
      to[i + u * kThreads] = mask_vec<T>(v, bits[u]);
    }
  }
  if (off != 0 && tid < 2 * kSize && cut.vecs > 0) {  // (two vectors at most, one value a thread)
    const int i = tid < kSize ? 0 : cut.vecs - 1;
    const bool todo = tid < kSize ? first == 1 : last < cut.vecs && (cut.vecs > 1 || first == 0);
    if (todo) one(cut.head + i * kSize + tid % kSize);
  }
}

struct Penalties {
  const void* history;         // ids so far [rows, history], int64 or int32; null: none
  const int* lengths;          // of each row's history; null: all of it
  const int* prompt_lengths;   // of its part that is not output; null: 0
  const float *repetition, *presence, *frequency;  // one per row; null: the number
  float repetition_, presence_, frequency_;
  const int64_t* bias_ids;     // [rows, biases]; null: none
  const float* bias;
  const uint32_t* allowed;     // [rows, words]; null: all
  int64_t history_stride, bias_stride, allowed_stride;
  int history_size, biases;
  bool wide;  // ids of 64 bits
};

// What a row's touched tokens become.
struct Change {
  float repetition, presence, frequency;
  const int* ids;         // biases of the slice, in their order (token within the slice)
  const float* values;
  int biases;
  // of the whole row, where shared memory does not hold the slice's
  const int64_t* row_ids;
  int begin;

  template <typename C>
  __device__ __forceinline__ float operator()(float x, uint32_t count, int v) const {
    const uint32_t times = count & Count<C>::kTimes;
    if (times != 0 || (count & Count<C>::kPrompt)) x = x > 0.f ? x / repetition : x * repetition;
    if (times != 0) x = x - frequency * static_cast<float>(times) - presence;
    if (count & Count<C>::kBiased) {
      float sum = 0.f;
      if (row_ids == nullptr) {
        for (int k = 0; k < biases; ++k) sum += ids[k] == v ? values[k] : 0.f;
      } else {
        for (int k = 0; k < biases; ++k) sum += row_ids[k] == begin + v ? values[k] : 0.f;
      }
      x += sum;
    }
    return x;
  }
};

// The slice's logits towards L2, which a block asks for before it counts: by one warp, unless a sample of the mask's words
// says that most of them stay unread.
template <typename T>
__device__ __forceinline__ void prefetch_slice(const T* row, int n, const uint32_t* words) {
  const int lane = threadIdx.x & 31;
  const bool open = words == nullptr || words[(n / 32) * lane / 32] != 0;
  if (__popc(__ballot_sync(0xffffffffu, open)) < 8 || lane != 0) return;
  const uintptr_t start = (reinterpret_cast<uintptr_t>(row) + 15) & ~uintptr_t(15);
  const uintptr_t end = reinterpret_cast<uintptr_t>(row + n) & ~uintptr_t(15);
  if (start < end)
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(start), "r"(static_cast<uint32_t>(end - start)) : "memory");
}

// C: the counts' type; void where no token is touched. Dynamic shared memory: counts [slice], list [room].
template <typename T, typename C>
__global__ void __launch_bounds__(kThreads, 6)
    process_kernel(const T* __restrict__ logits, RowLayout layout, int vocab, int slice, int parts,
                   const __grid_constant__ Penalties p, T* __restrict__ out, int* __restrict__ status) {
  constexpr bool kTouched = !std::is_void_v<C>;
  using Word = std::conditional_t<kTouched, C, uint16_t>;
  extern __shared__ uint4 smem[];
  const uint32_t r = blockIdx.x / parts;
  const int begin = static_cast<int>(blockIdx.x - r * parts) * slice, n = min(slice, vocab - begin);
  const int tid = threadIdx.x;
  const T* row = logits + layout.offset(r) + begin;
  T* to = out + static_cast<int64_t>(r) * vocab + begin;
  const uint32_t* words = p.allowed == nullptr ? nullptr : p.allowed + r * p.allowed_stride + begin / 32;
  if constexpr (!kTouched) {
    copy_masked(row, to, n, words);
  } else {
    __shared__ int listed_ids[kListed];
    __shared__ float listed_values[kListed];
    __shared__ int listed, touched;
    if (tid < 32) prefetch_slice(row, n, words);
    uint32_t* counts = reinterpret_cast<uint32_t*>(smem);
    uint16_t* list = reinterpret_cast<uint16_t*>(reinterpret_cast<Word*>(smem) + slice);
    for (int i = tid; i < static_cast<int>(slice * sizeof(Word) / 16); i += kThreads) smem[i] = make_uint4(0, 0, 0, 0);
    if (tid == 0) listed = 0, touched = 0;
    __syncthreads();
    const auto count = [&](int64_t id, uint32_t what, bool flag) {
      const int v = static_cast<int>(id - begin);
      if (Count<Word>::add(counts, v, what, flag)) list[atomicAdd(&touched, 1)] = static_cast<uint16_t>(v);
    };
    if (p.history != nullptr) {
      int length = p.history_size;
      if (p.lengths != nullptr) {
        const int given = p.lengths[r];
        if (given > length || given < 0) report_status(status, kOutOfBounds);
        length = max(0, min(given, length));
      }
      const int prompt = p.prompt_lengths == nullptr ? 0 : p.prompt_lengths[r];
      const int64_t* wide = static_cast<const int64_t*>(p.history) + r * p.history_stride;
      const int* narrow = static_cast<const int*>(p.history) + r * p.history_stride;
      for (int i = tid; i < length; i += kThreads * kIds) {
        int64_t id[kIds];
#pragma unroll
        for (int u = 0; u < kIds; ++u) {
          const int at = i + u * kThreads;
          id[u] = at >= length ? -1 : p.wide ? wide[at] : narrow[at];
        }
#pragma unroll
        for (int u = 0; u < kIds; ++u) {
          if (id[u] >= vocab) report_status(status, kOutOfBounds);
          if (id[u] < begin || id[u] >= begin + n) continue;
          const bool said = i + u * kThreads < prompt;
          count(id[u], said ? Count<Word>::kPrompt : 1u, said);
        }
      }
    }
    if (p.biases > 0 && tid >= kThreads - 32) {  // one warp lists those of the slice in their order
      const int64_t* ids = p.bias_ids + r * p.bias_stride;
      const float* values = p.bias + r * p.bias_stride;
      const int lane = tid & 31;
      int at = 0;
      for (int k = 0; k < p.biases; k += 32) {
        const int64_t id = k + lane < p.biases ? ids[k + lane] : -1;
        if (id >= vocab) report_status(status, kOutOfBounds);
        const bool mine = id >= begin && id < begin + n;
        const uint32_t votes = __ballot_sync(0xffffffffu, mine);
        const int place = at + __popc(votes & ((1u << lane) - 1u));
        if (mine) {
          count(id, Count<Word>::kBiased, true);
          if (place < kListed) listed_ids[place] = static_cast<int>(id - begin), listed_values[place] = values[k + lane];
        }
        at += __popc(votes);
      }
      if (lane == 0) listed = at;
    }
    copy_masked(row, to, n, words);
    Change change{};
    change.repetition = p.repetition == nullptr ? p.repetition_ : p.repetition[r];
    change.presence = p.presence == nullptr ? p.presence_ : p.presence[r];
    change.frequency = p.frequency == nullptr ? p.frequency_ : p.frequency[r];
    __syncthreads();  // the list and the counts, and the copies that it replaces
    change.ids = listed_ids;
    change.values = listed_values;
    change.biases = listed;
    if (listed > kListed) {
      change.row_ids = p.bias_ids + r * p.bias_stride;
      change.values = p.bias + r * p.bias_stride;
      change.biases = p.biases;
      change.begin = begin;
    }
    const Word* count_of = reinterpret_cast<const Word*>(smem);
    for (int i = tid; i < touched; i += kThreads * kAhead) {
      int v[kAhead];
      float x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int at = i + u * kThreads;
        v[u] = at < touched ? list[at] : -1;
        if (v[u] >= 0 && !(mask_bits(words, v[u], 1) & 1u)) v[u] = -1;
        if (v[u] >= 0) x[u] = to_float<T>(row[v[u]]);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (v[u] >= 0) to[v[u]] = from_float<T>(change.template operator()<Word>(x[u], count_of[v[u]], v[u]));
    }
  }
}

// Tokens of a slice (a multiple of 32): the fewer slices, the less often a history is read; more of them while there are
// too few blocks for the SMs.
int slice_size(int64_t rows, int64_t vocab) {
  int64_t slice = 16384;
  while (slice > 1024 && rows * ((vocab + slice - 1) / slice) < 4 * num_sms()) slice /= 2;
  return static_cast<int>(slice);
}

}  // namespace

// Contiguous, in the logits' shape and type.
at::Tensor process_logits(const at::Tensor& logits_in, const c10::optional<at::Tensor>& history,
                          const c10::optional<at::Tensor>& lengths, const c10::optional<at::Tensor>& prompt_lengths,
                          const c10::optional<at::Tensor>& repetition, const c10::optional<at::Tensor>& presence,
                          const c10::optional<at::Tensor>& frequency, double repetition_, double presence_,
                          double frequency_, const c10::optional<at::Tensor>& bias_ids,
                          const c10::optional<at::Tensor>& bias, const c10::optional<at::Tensor>& allowed) {
  constexpr const char* what = "process_logits";
  check_logits(logits_in, what);
  const int64_t vocab = logits_in.size(-1), rows = logits_in.numel() / vocab;
  c10::cuda::CUDAGuard guard(logits_in.device());
  RowLayout layout;
  at::Tensor logits = logits_in;
  if (!row_layout(logits, layout)) {
    logits = logits.contiguous();
    TDSV_CHECK(row_layout(logits, layout), what, ": logits layout");
  }
  auto out = at::empty(logits.sizes(), logits.options().memory_format(at::MemoryFormat::Contiguous));
  if (rows == 0) return out;
  auto given = [&](const c10::optional<at::Tensor>& t, at::ScalarType type, const char* name) {
    if (!t.has_value() || !t->defined()) return false;
    TDSV_CHECK(t->is_cuda() && t->has_storage() && t->device() == logits.device() && t->scalar_type() == type, what, ": ",
               name, " has the wrong type or device");
    return true;
  };
  auto per_row = [&](const c10::optional<at::Tensor>& t, at::ScalarType type, const char* name) -> const void* {
    if (!given(t, type, name)) return nullptr;
    check_cuda_tensor(*t, name);
    TDSV_CHECK(t->numel() == rows, what, ": ", name, " must hold one value per row");
    return t->data_ptr();
  };
  // [rows, size], rows any stride apart (0: the same for all)
  auto table = [&](const at::Tensor& t, const char* name) {
    TDSV_CHECK(t.dim() == 2 && t.size(0) == rows && (t.size(1) <= 1 || t.stride(1) == 1), what, ": ", name,
               " must be [rows, size] with dense rows");
    TDSV_CHECK(t.size(1) < (int64_t(1) << 29), what, ": ", name, " is too wide");
    return rows == 1 ? int64_t(0) : t.stride(0);
  };
  Penalties p{};
  if (history.has_value() && history->defined() && history->size(-1) > 0) {
    p.wide = history->scalar_type() == at::kLong;
    given(history, p.wide ? at::kLong : at::kInt, "history");
    p.history_stride = table(*history, "history");
    p.history_size = static_cast<int>(history->size(1));
    p.history = history->data_ptr();
    p.lengths = static_cast<const int*>(per_row(lengths, at::kInt, "lengths"));
    p.prompt_lengths = static_cast<const int*>(per_row(prompt_lengths, at::kInt, "prompt_lengths"));
  }
  p.repetition_ = static_cast<float>(repetition_);
  p.presence_ = static_cast<float>(presence_);
  p.frequency_ = static_cast<float>(frequency_);
  p.repetition = static_cast<const float*>(per_row(repetition, at::kFloat, "repetition"));
  p.presence = static_cast<const float*>(per_row(presence, at::kFloat, "presence"));
  p.frequency = static_cast<const float*>(per_row(frequency, at::kFloat, "frequency"));
  if (given(bias_ids, at::kLong, "bias_ids") && bias_ids->size(-1) > 0) {
    TDSV_CHECK(given(bias, at::kFloat, "bias") && bias->sizes() == bias_ids->sizes(), what, ": bias and bias_ids must be alike");
    p.bias_stride = table(*bias_ids, "bias_ids");
    TDSV_CHECK(table(*bias, "bias") == p.bias_stride, what, ": bias and bias_ids must lie alike");
    p.biases = static_cast<int>(bias_ids->size(1));
    p.bias_ids = bias_ids->data_ptr<int64_t>();
    p.bias = bias->data_ptr<float>();
  }
  if (given(allowed, at::kInt, "allowed")) {
    p.allowed_stride = table(*allowed, "allowed");
    TDSV_CHECK(allowed->size(1) >= (vocab + 31) / 32, what, ": allowed must hold a bit per token");
    p.allowed = reinterpret_cast<const uint32_t*>(allowed->data_ptr<int>());
  }
  const int slice = slice_size(rows, vocab);
  const int64_t parts = (vocab + slice - 1) / slice;
  TDSV_CHECK(rows * parts < (int64_t(1) << 31), what, ": too many rows");
  with_logit_type(logits.scalar_type(), [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    // a block's list holds each of its tokens once
    const int64_t room = std::min<int64_t>(slice, static_cast<int64_t>(p.history_size) + p.biases);
    auto launch = [&](auto kern, int64_t count_bytes) {
      const size_t smem = static_cast<size_t>(slice * count_bytes + (count_bytes != 0 ? 2 * room : 0));
      if (smem > 32 * 1024) TDSV_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
      kern<<<static_cast<unsigned>(rows * parts), kThreads, smem, stream()>>>(
          static_cast<const T*>(logits.data_ptr()), layout, static_cast<int>(vocab), slice, static_cast<int>(parts), p,
          static_cast<T*>(out.data_ptr()), status_word_ptr());
    };
    if (p.history == nullptr && p.bias_ids == nullptr) launch(process_kernel<T, void>, 0);
    else if (p.history_size <= Count<uint16_t>::kMost) launch(process_kernel<T, uint16_t>, 2);
    else launch(process_kernel<T, uint32_t>, 4);
  });
  TDSV_LAUNCH_CHECK();
  return out;
}

}  // namespace tdsv
