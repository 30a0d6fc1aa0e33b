// Token statistics straight from hidden states and the LM head's weight: the logits
//   X[M, N] = hidden[M, K] weight[N, K]^T        (bf16 operands, fp32 accumulators)
// exist only in tensor memory. One persistent tcgen05 kernel, two epilogues:
//
//   statistics  each 128 x BN tile of X is reduced, row by row, to (m, S, W) of logit_rows.cuh; the column
//               of the row's target is kept. A second kernel joins the tiles of a row in a fixed order.
//   gradient    the tile is recomputed and leaves as  dX = 2^y (a + b y) + d_it g / T  in bf16, with y
//               from the fp32 accumulators and a, b from the saved row statistics (logits rounded to bf16 first
//               would put an error of 2^-9 |x| into ln p). dX feeds the plain GEMMs of dhidden and dweight.
//
// Roles inside a CTA (192 threads, one CTA per SM): warp 0 feeds a ring of 128B-swizzled stages by TMA,
// one thread of warp 1 issues the MMAs into a double-buffered accumulator, warps 2-5 are the epilogue. A
// thread of the epilogue owns one row (its TMEM lane), so the reduction needs no shuffles. Every wait is
// bounded (common.cuh); a timeout records a status code and the CTA drains and exits.
#include "logit_rows.cuh"

#include <mutex>

namespace tdsv {

namespace {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int BK = 64;
constexpr int kThreads = 192;
constexpr int kStages = 4;
constexpr int kStageA = BM * BK * 2;
constexpr int kStageB = BN * BK * 2;
constexpr int kStageC = 32 * 128;
constexpr int kSmemBytes = kStages * (kStageA + kStageB) + 4 * kStageC + 1024 /*align*/ + 256 /*barriers*/;

struct HeadParams {
  int M, N, K;
  float c2, inv_t;
  const int64_t* targets;  // [M]
  // statistics
  float *part_m, *part_s, *part_w;  // [column tiles, M]
  float* target_logit;              // [M]
  // gradient
  const float4* saved;  // [M]: m, 1 / S, W / S
  const float *g, *h;   // [M] or null
  int64_t ignore_index;
  int* status;
};

// Tiles run down the rows first, so a column block of the weight is read from HBM once.
struct HeadTile {
  int m0, n0, nb;
};
__device__ __forceinline__ bool head_tile(const HeadParams& p, int tile, HeadTile& t) {
  const int m_blocks = (p.M + BM - 1) / BM, n_blocks = (p.N + BN - 1) / BN;
  if (tile >= m_blocks * n_blocks) return false;
  t.nb = tile / m_blocks;
  t.m0 = (tile % m_blocks) * BM;
  t.n0 = t.nb * BN;
  return true;
}

template <bool GRAD>
__global__ void __launch_bounds__(kThreads, 1)
    lm_head_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                   const __grid_constant__ CUtensorMap tma_c, const HeadParams p) {
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kStages * kStageA;
  uint8_t* smem_c = smem_b + kStages * kStageB;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_c + 4 * kStageC);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;  // [2]
  uint64_t* tempty = tfull + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  int* aborted = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 4);
    }
    *aborted = 0;
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(tmem_slot, 2 * BN);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  const int kb_count = (p.K + BK - 1) / BK;

  if (warp == 0) {
    if (lane == 0) {
      tma_prefetch_desc(&tma_a);
      tma_prefetch_desc(&tma_b);
      uint32_t it = 0;
      HeadTile t;
      for (int tile = blockIdx.x; head_tile(p, tile, t); tile += gridDim.x) {
        for (int kb = 0; kb < kb_count; ++kb, ++it) {
          const int s = it % kStages;
          const uint32_t ph = (it / kStages) & 1;
          if (!mbar_wait(&empty[s], ph ^ 1, p.status, kTimeoutEmpty)) { *aborted = 1; break; }
          if (*(volatile int*)aborted) break;
          mbar_arrive_expect_tx(&full[s], kStageA + kStageB);
          tma_load_2d(smem_a + s * kStageA, &tma_a, &full[s], kb * BK, t.m0);
          tma_load_2d(smem_b + s * kStageB, &tma_b, &full[s], kb * BK, t.n0);
        }
        if (*(volatile int*)aborted) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = make_idesc_bf16(BM, BN, false, false);
      uint32_t it = 0, tcount = 0;
      HeadTile t;
      for (int tile = blockIdx.x; head_tile(p, tile, t); tile += gridDim.x, ++tcount) {
        const int buf = tcount & 1;
        if (!mbar_wait(&tempty[buf], ((tcount >> 1) & 1) ^ 1, p.status, kTimeoutAccumFree)) { *aborted = 1; break; }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + buf * BN;
        bool ok = true;
        for (int kb = 0; kb < kb_count; ++kb, ++it) {
          const int s = it % kStages;
          if (!mbar_wait(&full[s], (it / kStages) & 1, p.status, kTimeoutFull)) { *aborted = 1; ok = false; break; }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem_a + s * kStageA), sb = smem_u32(smem_b + s * kStageB);
#pragma unroll
          for (int kk = 0; kk < BK / 16; ++kk)
            umma_f16(d_tmem, make_smem_desc_sw128(sa + kk * 32, 16, 1024), make_smem_desc_sw128(sb + kk * 32, 16, 1024),
                     idesc, (kb > 0 || kk > 0) ? 1u : 0u);
          umma_commit(&empty[s]);
        }
        if (!ok) break;
        umma_commit(&tfull[buf]);
      }
    }
  } else {
    const int quarter = warp & 3;  // TMEM lanes this warp may access
    uint8_t* stage = smem_c + quarter * kStageC;
    uint32_t tcount = 0;
    HeadTile t;
    for (int tile = blockIdx.x; head_tile(p, tile, t); tile += gridDim.x, ++tcount) {
      const int buf = tcount & 1;
      const int row = t.m0 + quarter * 32 + lane;
      const bool live = row < p.M;
      const int64_t target = live ? p.targets[row] : -1;
      // the target's column inside this tile, or a column no chunk has
      const int64_t rel = target - t.n0;
      const int hit = rel >= 0 && rel < BN && target < p.N ? static_cast<int>(rel) : -1;
      // dx = 2^y (a + b y) with 1 / (S T) inside a and b; a row without a gradient has y = -inf throughout
      float m = INFINITY, a = 0.f, b = 0.f, bonus = 0.f;
      if (GRAD && live && target != p.ignore_index) {
        const float4 sv = p.saved[row];
        if (sv.y != 0.f) {
          const float g = p.g != nullptr && target >= 0 && target < p.N ? p.g[row] : 0.f;
          const float h = p.h != nullptr ? p.h[row] * kLn2 : 0.f;
          const float scale = p.inv_t * sv.y;
          m = sv.x;
          a = -scale * (g - h * sv.z);
          b = -scale * h;
          bonus = p.inv_t * g;
        }
      }
      if (!mbar_wait(&tfull[buf], (tcount >> 1) & 1, p.status, kTimeoutAccum)) { *aborted = 1; break; }
      tc_fence_after();
      const uint32_t t_addr = tmem_base + buf * BN + (static_cast<uint32_t>(quarter * 32) << 16);
      if (!GRAD) {
        RowStats st;
#pragma unroll 1
        for (int c0 = 0; c0 < BN; c0 += 32) {
          const int left = p.N - t.n0 - c0;  // columns of this chunk inside the vocabulary
          if (left <= 0) break;
          uint32_t raw[32];
          tmem_ld_32x32b_x32(t_addr + c0, raw);
          tmem_ld_wait();
          float top = -INFINITY;
          if (left < 32) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i >= left) raw[i] = __float_as_uint(-INFINITY);
          }
#pragma unroll
          for (int i = 0; i < 32; ++i) top = fmaxf(top, __uint_as_float(raw[i]));
          if (top > st.m) st.rebase(top, p.c2);
          if (st.m != -INFINITY) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
              const float y = (__uint_as_float(raw[i]) - st.m) * p.c2;
              const float e = exp2_fast(y);
              st.s += e;
              st.w += e * fmaxf(y, kMinExponent);
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (__uint_as_float(raw[i]) != __uint_as_float(raw[i])) st.s = NAN;
          }
          const int at = hit - c0;
          if (at >= 0 && at < 32) {
            float x = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i == at) x = __uint_as_float(raw[i]);
            p.target_logit[row] = x;
          }
        }
        if (live) {
          const int64_t o = static_cast<int64_t>(t.nb) * p.M + row;
          p.part_m[o] = st.m;
          p.part_s[o] = st.s;
          p.part_w[o] = st.w;
        }
      } else {
#pragma unroll 1
        for (int c0 = 0; c0 < BN; c0 += 64) {
          uint32_t raw[64];
          tmem_ld_32x32b_x32(t_addr + c0, *reinterpret_cast<uint32_t(*)[32]>(&raw[0]));
          tmem_ld_32x32b_x32(t_addr + c0 + 32, *reinterpret_cast<uint32_t(*)[32]>(&raw[32]));
          tmem_ld_wait();
          if (lane == 0) bulk_wait_group_read0();  // the last chunk's store has read the staging buffer
          __syncwarp();
          uint8_t* my_row = stage + lane * 128;
          const int at = hit - c0;
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float y = fmaxf((__uint_as_float(raw[q * 8 + i]) - m) * p.c2, kMinExponent);
              d[i] = exp2_fast(y) * (a + b * y) + (q * 8 + i == at ? bonus : 0.f);
            }
            uint4 v;
            __nv_bfloat162 pair[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) pair[i] = __floats2bfloat162_rn(d[2 * i], d[2 * i + 1]);
            v = *reinterpret_cast<uint4*>(pair);
            *reinterpret_cast<uint4*>(my_row + ((q ^ (lane & 7)) << 4)) = v;
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0 && t.n0 + c0 < p.N && t.m0 + quarter * 32 < p.M) {
            tma_store_2d(&tma_c, smem_u32(stage), t.n0 + c0, t.m0 + quarter * 32);
            bulk_commit_group();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&tempty[buf]);
    }
    if (GRAD && lane == 0) bulk_wait_group0();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// Joins the column tiles of each row: 32 rows a block, 16 slices of the tiles, merged in slice order.
constexpr int kJoinSlices = 16;
__global__ void __launch_bounds__(32 * kJoinSlices)
    lm_head_join_kernel(const float* __restrict__ part_m, const float* __restrict__ part_s,
                        const float* __restrict__ part_w, const float* __restrict__ target_logit,
                        const int64_t* __restrict__ targets, int64_t ignore_index, int rows, int vocab, int tiles,
                        float c2, float* __restrict__ log_probs, float* __restrict__ entropy,
                        float4* __restrict__ saved, int* status) {
  __shared__ RowStats part[kJoinSlices][32];
  const int lane = threadIdx.x & 31, slice = threadIdx.x >> 5;
  const int r = blockIdx.x * 32 + lane;
  RowStats st;
  if (r < rows) {
    for (int t = slice; t < tiles; t += kJoinSlices) {
      const int64_t o = static_cast<int64_t>(t) * rows + r;
      RowStats u;
      u.m = part_m[o], u.s = part_s[o], u.w = part_w[o];
      st.merge(u, c2);
    }
  }
  part[slice][lane] = st;
  __syncthreads();
  if (slice != 0 || r >= rows) return;
  for (int s = 1; s < kJoinSlices; ++s) st.merge(part[s][lane], c2);
  const int64_t target = targets[r];
  float lp = 0.f, ent = 0.f;
  if (target != ignore_index) {
    const float log2s = log2f(st.s);
    ent = st.s == 0.f ? 0.f : kLn2 * (log2s - st.w / st.s);
    if (target >= 0 && target < vocab) {
      lp = st.s == 0.f ? -INFINITY : kLn2 * ((target_logit[r] - st.m) * c2 - log2s);
    } else {
      lp = NAN;
      report_status(status, kOutOfBounds);
    }
  }
  log_probs[r] = lp;
  entropy[r] = ent;
  saved[r] = saved_stats(st);
}

CUtensorMap head_map(const at::Tensor& t, int64_t row_stride, int box_rows) {
  bind_primary_context();
  TDSV_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (row_stride * 2) % 16 == 0,
             "linear_token_statistics: rows must start on 16-byte boundaries");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(t.size(1)), static_cast<cuuint64_t>(t.size(0))};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_stride) * 2};
  cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUtensorMap map;
  const CUresult r = encode_fn()(&map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, t.data_ptr(), dims, strides, box, estr,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed with code ", static_cast<int>(r));
  return map;
}

void check_head(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets) {
  check_cuda_tensor(hidden, "hidden");
  check_cuda_tensor(weight, "weight");
  check_cuda_tensor(targets, "targets");
  TDSV_CHECK(hidden.dim() == 2 && weight.dim() == 2 && hidden.size(1) == weight.size(1),
             "linear_token_statistics: hidden [rows, K] and weight [V, K]");
  TDSV_CHECK(hidden.scalar_type() == at::kBFloat16 && weight.scalar_type() == at::kBFloat16,
             "linear_token_statistics: bf16 hidden and weight");
  TDSV_CHECK(hidden.size(1) % 8 == 0 && hidden.size(1) > 0, "linear_token_statistics: K must be a multiple of 8");
  TDSV_CHECK(targets.scalar_type() == at::kLong && targets.numel() == hidden.size(0),
             "linear_token_statistics: int64 targets, one per row");
  TDSV_CHECK(weight.size(0) >= 1 && weight.size(0) < (1 << 30) && hidden.size(0) < (1 << 30),
             "linear_token_statistics: size");
}

template <bool GRAD>
void launch_head(const at::Tensor& hidden, const at::Tensor& weight, const CUtensorMap& mc, HeadParams& p) {
  auto kern = lm_head_kernel<GRAD>;
  static std::once_flag once;
  std::call_once(once, [&] {
    TDSV_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  });
  const CUtensorMap ma = head_map(hidden, hidden.size(1), BM), mb = head_map(weight, weight.size(1), BN);
  p.M = static_cast<int>(hidden.size(0));
  p.N = static_cast<int>(weight.size(0));
  p.K = static_cast<int>(hidden.size(1));
  p.status = status_word_ptr();
  const int64_t tiles = static_cast<int64_t>((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  TDSV_CHECK(tiles < (int64_t(1) << 30), "linear_token_statistics: too many tiles");
  const int grid = static_cast<int>(std::min<int64_t>(num_sms(), tiles));
  void* args[] = {const_cast<CUtensorMap*>(&ma), const_cast<CUtensorMap*>(&mb), const_cast<CUtensorMap*>(&mc), &p};
  TDSV_CUDA_CHECK(cudaLaunchKernel(reinterpret_cast<const void*>(kern), dim3(grid), dim3(kThreads), args, kSmemBytes,
                                   stream()));
}

}  // namespace

// (log_probs [M], entropy [M], saved [M, 4])
std::vector<at::Tensor> lm_head_stats_fwd(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                                          double temperature, int64_t ignore_index) {
  check_head(hidden, weight, targets);
  const int64_t rows = hidden.size(0), vocab = weight.size(0);
  c10::cuda::CUDAGuard guard(hidden.device());
  const auto f32 = hidden.options().dtype(at::kFloat);
  auto log_probs = at::empty({rows}, f32), entropy = at::empty({rows}, f32), saved = at::empty({rows, 4}, f32);
  if (rows == 0) return {log_probs, entropy, saved};
  const int64_t tiles = (vocab + BN - 1) / BN;
  auto part = at::empty({3, tiles, rows}, f32);
  auto target_logit = at::empty({rows}, f32);
  HeadParams p{};
  p.c2 = static_cast<float>(1.4426950408889634 / temperature);
  p.targets = targets.data_ptr<int64_t>();
  p.part_m = part.data_ptr<float>();
  p.part_s = p.part_m + tiles * rows;
  p.part_w = p.part_s + tiles * rows;
  p.target_logit = target_logit.data_ptr<float>();
  p.ignore_index = ignore_index;
  const CUtensorMap unused{};
  launch_head<false>(hidden, weight, unused, p);
  lm_head_join_kernel<<<static_cast<unsigned>((rows + 31) / 32), 32 * kJoinSlices, 0, stream()>>>(
      p.part_m, p.part_s, p.part_w, p.target_logit, p.targets, ignore_index, static_cast<int>(rows),
      static_cast<int>(vocab), static_cast<int>(tiles), p.c2, log_probs.data_ptr<float>(), entropy.data_ptr<float>(),
      reinterpret_cast<float4*>(saved.data_ptr<float>()), p.status);
  TDSV_LAUNCH_CHECK();
  return {log_probs, entropy, saved};
}

// bf16 gradient of the logits, [M, V] with rows padded to 16 bytes.
at::Tensor lm_head_stats_bwd(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                             const at::Tensor& saved, double temperature, int64_t ignore_index,
                             const c10::optional<at::Tensor>& g_log_probs, const c10::optional<at::Tensor>& g_entropy) {
  check_head(hidden, weight, targets);
  const int64_t rows = hidden.size(0), vocab = weight.size(0), pitch = (vocab + 7) / 8 * 8;
  c10::cuda::CUDAGuard guard(hidden.device());
  auto dlogits = at::empty({rows, pitch}, hidden.options()).narrow(1, 0, vocab);
  if (rows == 0) return dlogits;
  check_cuda_tensor(saved, "saved");
  TDSV_CHECK(saved.scalar_type() == at::kFloat && saved.numel() == 4 * rows, "linear_token_statistics: saved row statistics");
  auto pointer = [&](const c10::optional<at::Tensor>& t) -> const float* {
    if (!t.has_value() || !t->defined()) return nullptr;
    check_cuda_tensor(*t, "gradient");
    TDSV_CHECK(t->scalar_type() == at::kFloat && t->numel() == rows, "linear_token_statistics: fp32 gradients, one per row");
    return t->data_ptr<float>();
  };
  HeadParams p{};
  p.c2 = static_cast<float>(1.4426950408889634 / temperature);
  p.inv_t = static_cast<float>(1.0 / temperature);
  p.targets = targets.data_ptr<int64_t>();
  p.saved = reinterpret_cast<const float4*>(saved.data_ptr<float>());
  p.g = pointer(g_log_probs);
  p.h = pointer(g_entropy);
  p.ignore_index = ignore_index;
  const CUtensorMap mc = head_map(dlogits, pitch, 32);
  launch_head<true>(hidden, weight, mc, p);
  return dlogits;
}

}  // namespace tdsv
