// Token statistics straight from hidden states and the LM head's weight: for scoring, the logits
//   X[M, N] = hidden[M, K] weight[N, K]^T        (bf16 operands, fp32 accumulators)
// exist only in tensor memory (a backward may keep them, below). One persistent tcgen05 kernel, two epilogues:
//
//   statistics  each 128 x BN tile of X is reduced, row by row, to (m, S, W) of logit_rows.cuh; the column
//               of the row's target is kept. A second kernel joins the tiles of a row in a fixed order.
//   gradient    the tile is recomputed and leaves as  dX = 2^y (a + b y) + d_it g / T  in bf16, with y
//               from the fp32 accumulators and a, b from the saved row statistics (logits rounded to bf16 first
//               would put an error of 2^-9 |x| into ln p). dX feeds the plain GEMMs of dhidden and dweight.
//
// Roundings. Statistics are fp32 throughout. The tensor cores' fp32 sums over K shrink a logit by 1.8e-6 of itself at
// K = 2048 and 4.8e-6 at 5120 (bit for bit what the plain library product of bf16 operands gives); the epilogue adds 6e-8.
// So log-probabilities and entropies are 1.5e-6 to 3.4e-6 from 64 bits, where a product of fp32 operands outside the tensor
// cores has 2e-7 to 8e-7. dX is rounded to bf16 because it is an operand of two tensor-core products whose other operands are bf16, as in the
// cross entropy of this framework: each value is off by 2^-8 of itself at most, 1.65e-3 in the mean, so dhidden and dweight
// are 2.3e-3 from 64 bits where the rounding of an exact result to bf16 alone is 1.65e-3. An exact dX (a high and a low part)
// would take each of the two products twice: 3.7 ms would be about 5.9 at 1023 x 5120 x 129280.
//
// Where a backward will follow and the fp32 logits fit the caller's budget, the statistics' epilogue stores them
// as well (behind the MMAs, which are what the kernel waits for), and the gradient is one pass over them: for
// 1023 x 5120 x 129280 that replaces a product of 1010 us.
//
// When only scores are wanted, rows without a target are left out: the others are gathered first and their
// number stays on the device.
//
// Roles inside a CTA (192 threads, one CTA per SM): warp 0 feeds a ring of 128B-swizzled stages by TMA,
// one thread of warp 1 issues the MMAs into a double-buffered accumulator, warps 2-5 are the epilogue. A
// thread of the epilogue owns one row (its TMEM lane), so the reduction needs no shuffles: 8 instructions a value
// against the 64 cycles that the MMAs of a 256-wide tile take per 16 of K. Every wait is bounded (common.cuh); a
// timeout records a status code and the CTA drains and exits.
//
// Bound by the tensor cores: 4096 x 2048 x 151936 takes 1.80 ms, 1417 TFLOP/s (the plain library product 1.85 ms). One
// row block is bound by the weight's way from memory instead: 16 rows take 105 us, 5.9 TB/s.
#include "logit_rows.cuh"

#include <mutex>

namespace tdsv {

namespace {

constexpr int BM = 128;
constexpr int BN = 256;
constexpr int BK = 64;
constexpr int kThreads = 192;
constexpr int kStageB = BN * BK * 2;
constexpr int kStageC = 32 * 128;

// FEW: at most 32 rows. The weight is then read once, from memory, and what is on its way sets the pace (16 rows: 144 us
// with 4 stages of 208 columns, 200 with 128 columns), so a stage holds 32 rows of hidden and there are six: 105 us. The
// MMA still takes 128 rows: the others are whatever follows in shared memory, and their accumulators are not read.
template <bool FEW>
struct Ring {
  static constexpr int kRows = FEW ? 32 : BM;
  static constexpr int kStages = FEW ? 6 : 4;
  static constexpr int kStageA = kRows * BK * 2;
  static constexpr int kStaging = FEW ? 0 : 4 * kStageC;
  static constexpr int kSmemBytes = kStages * (kStageA + kStageB) + kStaging + 1024 /*align*/ + 256 /*barriers*/;
};

enum Epilogue : int { kStats = 0, kStatsKeep = 1, kGrad = 2 };

struct HeadParams {
  int M, N, K;
  int bn;                  // columns of a tile (kStats: any multiple of 16 up to BN, to share few tiles evenly)
  const int* rows;         // device: the rows that are there, or null: M
  float c2, inv_t;
  const int64_t* targets;  // [M]
  // statistics
  float4* part;                     // [column tiles, M]: m, S, W
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
__device__ __forceinline__ bool head_tile(const HeadParams& p, int rows, int tile, HeadTile& t) {
  const int m_blocks = (rows + BM - 1) / BM, n_blocks = (p.N + p.bn - 1) / p.bn;
  if (tile >= m_blocks * n_blocks) return false;
  t.nb = tile / m_blocks;
  t.m0 = (tile % m_blocks) * BM;
  t.n0 = t.nb * p.bn;
  return true;
}

template <int EPI, bool FEW>
__global__ void __launch_bounds__(kThreads, 1)
    lm_head_kernel(const __grid_constant__ CUtensorMap tma_a, const __grid_constant__ CUtensorMap tma_b,
                   const __grid_constant__ CUtensorMap tma_c, const HeadParams p) {
  using R = Ring<FEW>;
  constexpr int kStages = R::kStages, kStageA = R::kStageA;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* smem_a = smem;
  uint8_t* smem_b = smem + kStages * kStageA;
  uint8_t* smem_c = smem_b + kStages * kStageB;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_c + R::kStaging);
  uint64_t* empty = full + kStages;
  uint64_t* tfull = empty + kStages;  // [2]
  uint64_t* tempty = tfull + 2;       // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  int* aborted = reinterpret_cast<int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rows = p.rows != nullptr ? min(*p.rows, p.M) : p.M;
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
      for (int tile = blockIdx.x; head_tile(p, rows, tile, t); tile += gridDim.x) {
        for (int kb = 0; kb < kb_count; ++kb, ++it) {
          const int s = it % kStages;
          const uint32_t ph = (it / kStages) & 1;
          if (!mbar_wait(&empty[s], ph ^ 1, p.status, kTimeoutEmpty)) { *aborted = 1; break; }
          if (*(volatile int*)aborted) break;
          mbar_arrive_expect_tx(&full[s], kStageA + p.bn * BK * 2);
          tma_load_2d(smem_a + s * kStageA, &tma_a, &full[s], kb * BK, t.m0);
          tma_load_2d(smem_b + s * kStageB, &tma_b, &full[s], kb * BK, t.n0);
        }
        if (*(volatile int*)aborted) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_bf16(BM, p.bn, false, false);
      uint32_t it = 0, tcount = 0;
      HeadTile t;
      for (int tile = blockIdx.x; head_tile(p, rows, tile, t); tile += gridDim.x, ++tcount) {
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
    for (int tile = blockIdx.x; head_tile(p, rows, tile, t); tile += gridDim.x, ++tcount) {
      const int buf = tcount & 1;
      const int row = t.m0 + quarter * 32 + lane;
      const bool live = row < rows;
      const bool some = t.m0 + quarter * 32 < rows;  // (rows of this warp)
      const int64_t target = live ? p.targets[row] : -1;
      // the target's column inside this tile, or a column no chunk has
      const int64_t rel = target - t.n0;
      const int hit = rel >= 0 && rel < p.bn && target < p.N ? static_cast<int>(rel) : -1;
      // dx = 2^y (a + b y) with 1 / (S T) inside a and b; a row without a gradient has y = -inf throughout
      float m = INFINITY, a = 0.f, b = 0.f, bonus = 0.f;
      if (EPI == kGrad && live && target != p.ignore_index) {
        const float4 sv = p.saved[row];
        if (sv.y != 0.f) {
          const float g = p.g != nullptr && target >= 0 && target < p.N ? p.g[row] : 0.f;
          const float h = p.h != nullptr ? p.h[row] * kLn2 : 0.f;
          const float scale = p.inv_t * sv.y;
          m = sv.x;
          a = -scale * (g - h * sv.z);
          b = -scale * h;
          bonus = __fmul_rn(p.inv_t, g);  // (rounded as in a: the two cancel where p = 1)
        }
      }
      if (!mbar_wait(&tfull[buf], (tcount >> 1) & 1, p.status, kTimeoutAccum)) { *aborted = 1; break; }
      tc_fence_after();
      const uint32_t t_addr = tmem_base + buf * BN + (static_cast<uint32_t>(quarter * 32) << 16);
      if (EPI != kGrad && some) {
        RowStats st;
#pragma unroll 1
        for (int c0 = 0; c0 < BN; c0 += 32) {
          const int left = min(p.N - t.n0, p.bn) - c0;  // columns of this chunk inside the tile
          if (left <= 0) break;
          uint32_t raw[32];
          tmem_ld_32x32b_x32(t_addr + c0, raw);
          tmem_ld_wait();
          if (EPI == kStatsKeep) {
            if (lane == 0) bulk_wait_group_read0();  // the last chunk's store has read the staging buffer
            __syncwarp();
            uint8_t* my_row = stage + lane * 128;
#pragma unroll
            for (int q = 0; q < 8; ++q)
              *reinterpret_cast<uint4*>(my_row + ((q ^ (lane & 7)) << 4)) =
                  make_uint4(raw[4 * q], raw[4 * q + 1], raw[4 * q + 2], raw[4 * q + 3]);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && t.m0 + quarter * 32 < p.M) {
              tma_store_2d(&tma_c, smem_u32(stage), t.n0 + c0, t.m0 + quarter * 32);
              bulk_commit_group();
            }
          }
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
          p.part[o] = make_float4(st.m, st.s, st.w, 0.f);
        }
      }
      if (EPI == kGrad) {
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
    if (EPI != kStats && lane == 0) bulk_wait_group0();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 0) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 2 * BN);
  }
}

// Joins the column tiles of each row: 4 rows a block, 128 slices of the tiles. The largest reference first, so that
// no term waits for the one before; the order of the sums is fixed.
constexpr int kJoinRows = 4, kJoinThreads = 512;
__global__ void __launch_bounds__(kJoinThreads)
    lm_head_join_kernel(const HeadParams p, const int* __restrict__ where, int tiles, float* __restrict__ log_probs,
                        float* __restrict__ entropy, float4* __restrict__ saved) {
  __shared__ float part[3][kJoinThreads / 32][kJoinRows];
  constexpr int kSlices = kJoinThreads / kJoinRows;
  const int lane = threadIdx.x % kJoinRows, slice = threadIdx.x / kJoinRows, warp = threadIdx.x >> 5;
  const int i = blockIdx.x * kJoinRows + lane;
  const bool live = i < (p.rows != nullptr ? min(*p.rows, p.M) : p.M);
  const float4* mine = p.part + i;
  float m = -INFINITY;
  if (live)
#pragma unroll 4
    for (int t = slice; t < tiles; t += kSlices) {
      const float4 u = mine[static_cast<int64_t>(t) * p.M];
      m = fmaxf(m, u.y != 0.f ? u.x : -INFINITY);
    }
#pragma unroll
  for (int o = kJoinRows; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) < kJoinRows) part[0][warp][lane] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) m = fmaxf(m, part[0][w][lane]);
  float sum = 0.f, weighted = 0.f;
  if (live)
#pragma unroll 4
    for (int t = slice; t < tiles; t += kSlices) {
      const float4 u = mine[static_cast<int64_t>(t) * p.M];
      const float d = (u.x - m) * p.c2, f = exp2_fast(d);
      sum += u.y != 0.f ? u.y * f : 0.f;
      weighted += u.y != 0.f ? (u.z + u.y * fmaxf(d, kMinExponent)) * f : 0.f;
    }
#pragma unroll
  for (int o = kJoinRows; o < 32; o <<= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
    weighted += __shfl_xor_sync(0xffffffffu, weighted, o);
  }
  if ((threadIdx.x & 31) < kJoinRows) part[1][warp][lane] = sum, part[2][warp][lane] = weighted;
  __syncthreads();
  if (slice != 0 || !live) return;
  RowStats st;
  st.m = m;
#pragma unroll
  for (int w = 0; w < kJoinThreads / 32; ++w) st.s += part[1][w][lane], st.w += part[2][w][lane];
  const int64_t target = p.targets[i];
  const int r = where != nullptr ? where[i] : i;
  float lp = 0.f, ent = 0.f;
  if (target != p.ignore_index) {
    const float log2s = log2f(st.s);
    ent = st.s == 0.f ? 0.f : kLn2 * (log2s - st.w / st.s);
    if (target >= 0 && target < p.N) {
      lp = st.s == 0.f ? -INFINITY : (p.target_logit[i] - st.m) * p.inv_t - kLn2 * log2s;
    } else {
      lp = NAN;
      report_status(p.status, kOutOfBounds);
    }
  }
  log_probs[r] = lp;
  entropy[r] = ent;
  if (saved != nullptr) saved[r] = saved_stats(st);
}

// The rows with a target, in order: where[i] is row i's place, with its target; the others' results are zeros.
__global__ void __launch_bounds__(1024)
    lm_head_rows_kernel(const int64_t* __restrict__ targets, int rows, int64_t ignore_index, int* __restrict__ where,
                        int64_t* __restrict__ kept_targets, int* __restrict__ count, float* __restrict__ log_probs,
                        float* __restrict__ entropy) {
  __shared__ int sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int base = 0;
  for (int r0 = 0; r0 < rows; r0 += 1024) {
    const int r = r0 + static_cast<int>(threadIdx.x);
    const int64_t t = r < rows ? targets[r] : ignore_index;
    const bool keep = t != ignore_index;
    const uint32_t mask = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) sums[warp] = __popc(mask);
    __syncthreads();
    int before = base, all = 0;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) before += sums[w];
      all += sums[w];
    }
    if (keep) {
      const int at = before + __popc(mask & ((1u << lane) - 1u));
      where[at] = r;
      kept_targets[at] = t;
    } else if (r < rows) {
      log_probs[r] = 0.f;
      entropy[r] = 0.f;
    }
    base += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *count = base;
}
__global__ void lm_head_gather_kernel(const uint4* __restrict__ hidden, const int* __restrict__ where,
                                      const int* __restrict__ count, int vecs, uint4* __restrict__ out) {
  const int i = blockIdx.x;
  if (i >= *count) return;
  const int64_t from = static_cast<int64_t>(where[i]) * vecs, to = static_cast<int64_t>(i) * vecs;
  for (int j = threadIdx.x; j < vecs; j += blockDim.x) out[to + j] = hidden[from + j];
}

// The gradient from kept logits: 8 values a thread, rows of both padded to 8 values.
constexpr int kKeptThreads = 256, kKeptVecs = 4;
__global__ void __launch_bounds__(kKeptThreads)
    lm_head_kept_kernel(const float4* __restrict__ logits, const HeadParams p, int parts, int vecs,
                        uint4* __restrict__ dlogits) {
  const int r = static_cast<int>(blockIdx.x / static_cast<unsigned>(parts));
  const int first = static_cast<int>(blockIdx.x - static_cast<unsigned>(r) * static_cast<unsigned>(parts)) * kKeptThreads *
                    kKeptVecs;
  const int64_t target = p.targets[r];
  const float4 sv = p.saved[r];
  uint4* out = dlogits + static_cast<int64_t>(r) * vecs;
  const float4* row = logits + static_cast<int64_t>(r) * vecs * 2;
  const bool live = target != p.ignore_index && sv.y != 0.f;
  const bool has_target = target >= 0 && target < p.N;
  const float g = live && has_target && p.g != nullptr ? p.g[r] : 0.f, h = live && p.h != nullptr ? p.h[r] * kLn2 : 0.f;
  const float scale = p.inv_t * sv.y, a = -scale * (g - h * sv.z), b = -scale * h;
  const float bonus = __fmul_rn(p.inv_t, g);  // (rounded as in a: the two cancel where p = 1)
#pragma unroll
  for (int u = 0; u < kKeptVecs; ++u) {
    const int i = first + u * kKeptThreads + static_cast<int>(threadIdx.x);
    if (i >= vecs) return;
    uint4 o = make_uint4(0, 0, 0, 0);
    if (live) {
      const float4 lo = row[2 * i], hi = row[2 * i + 1];
      float d[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = gradient_one(d[e], sv.x, p.c2, a, b);
      const int64_t hit = has_target ? target - 8 * static_cast<int64_t>(i) : -1;
      if (hit >= 0 && hit < 8) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e == hit) d[e] += bonus;
      }
      o.x = pack_pair<__nv_bfloat16>(d[0], d[1]);
      o.y = pack_pair<__nv_bfloat16>(d[2], d[3]);
      o.z = pack_pair<__nv_bfloat16>(d[4], d[5]);
      o.w = pack_pair<__nv_bfloat16>(d[6], d[7]);
    }
    out[i] = o;
  }
}

CUtensorMap head_map(const at::Tensor& t, int64_t row_stride, int box_rows) {
  bind_primary_context();
  const bool bf16 = t.scalar_type() == at::kBFloat16;
  const int item = bf16 ? 2 : 4;
  TDSV_CHECK(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (row_stride * item) % 16 == 0,
             "linear_token_statistics: rows must start on 16-byte boundaries");
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(t.size(1)), static_cast<cuuint64_t>(t.size(0))};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_stride) * item};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / item), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1, 1};
  CUtensorMap map;
  const CUresult r = encode_fn()(&map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT32, 2, t.data_ptr(), dims, strides, box, estr,
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
  // (every reader of both, the gather of the kept rows among them, moves 16 bytes at a time)
  TDSV_CHECK(reinterpret_cast<uintptr_t>(hidden.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(weight.data_ptr()) % 16 == 0,
             "linear_token_statistics: hidden and weight must start on 16-byte boundaries");
  TDSV_CHECK(targets.scalar_type() == at::kLong && targets.numel() == hidden.size(0),
             "linear_token_statistics: int64 targets, one per row");
  TDSV_CHECK(weight.size(0) >= 1 && weight.size(0) < (1 << 30) && hidden.size(0) < (1 << 30),
             "linear_token_statistics: size");
}

// Columns of a tile: 256, unless the tiles are so few that their last round over the SMs would be mostly empty
// (one row block of 151936 columns: 594 tiles are 4.01 rounds of 148; of 208 columns 731 are 4.94).
int tile_columns(int64_t rows, int64_t vocab) {
  const int64_t m_blocks = (rows + BM - 1) / BM, sms = num_sms();
  if (m_blocks * ((vocab + BN - 1) / BN) >= 8 * sms) return BN;
  int best = BN;
  int64_t least = INT64_MAX;
  for (int bn = BN; bn >= 96; bn -= 16) {
    const int64_t columns = (m_blocks * ((vocab + bn - 1) / bn) + sms - 1) / sms * bn;
    if (columns < least) least = columns, best = bn;
  }
  return best;
}

template <int EPI, bool FEW>
void launch_head(const at::Tensor& hidden, const at::Tensor& weight, const CUtensorMap& mc, HeadParams& p) {
  using R = Ring<FEW>;
  auto kern = lm_head_kernel<EPI, FEW>;
  static std::once_flag once;
  std::call_once(once, [&] {
    TDSV_CUDA_CHECK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, R::kSmemBytes));
  });
  p.M = static_cast<int>(hidden.size(0));
  p.N = static_cast<int>(weight.size(0));
  p.K = static_cast<int>(hidden.size(1));
  p.bn = EPI == kStats ? tile_columns(p.M, p.N) : BN;
  p.status = status_word_ptr();
  const CUtensorMap ma = head_map(hidden, hidden.size(1), R::kRows), mb = head_map(weight, weight.size(1), p.bn);
  const int64_t tiles = static_cast<int64_t>((p.M + BM - 1) / BM) * ((p.N + p.bn - 1) / p.bn);
  TDSV_CHECK(tiles < (int64_t(1) << 30), "linear_token_statistics: too many tiles");
  const int grid = static_cast<int>(std::min<int64_t>(num_sms(), tiles));
  void* args[] = {const_cast<CUtensorMap*>(&ma), const_cast<CUtensorMap*>(&mb), const_cast<CUtensorMap*>(&mc), &p};
  TDSV_CUDA_CHECK(cudaLaunchKernel(reinterpret_cast<const void*>(kern), dim3(grid), dim3(kThreads), args, R::kSmemBytes,
                                   stream()));
}

}  // namespace

// (log_probs [M], entropy [M], saved [M, 4], fp32 logits [M, V] in rows padded to 32 bytes). `saved` is undefined
// without `save`, the logits unless `keep` asks for them.
std::vector<at::Tensor> lm_head_stats_fwd(const at::Tensor& hidden_in, const at::Tensor& weight, const at::Tensor& targets,
                                          double temperature, int64_t ignore_index, bool save, bool keep) {
  check_head(hidden_in, weight, targets);
  const int64_t rows = hidden_in.size(0), vocab = weight.size(0);
  c10::cuda::CUDAGuard guard(hidden_in.device());
  const auto f32 = hidden_in.options().dtype(at::kFloat);
  auto log_probs = at::empty({rows}, f32), entropy = at::empty({rows}, f32);
  at::Tensor saved, logits, hidden = hidden_in, where, kept_targets;
  if (save) saved = at::empty({rows, 4}, f32);
  if (keep) logits = at::empty({rows, (vocab + 7) / 8 * 8}, f32).narrow(1, 0, vocab);
  if (rows == 0) return {log_probs, entropy, saved, logits};
  HeadParams p{};
  p.c2 = static_cast<float>(1.4426950408889634 / temperature);
  p.inv_t = static_cast<float>(1.0 / temperature);
  p.targets = targets.data_ptr<int64_t>();
  p.ignore_index = ignore_index;
  if (!save && rows > 2 * BM) {  // (fewer would hardly save a row block)
    where = at::empty({rows + 1}, f32.dtype(at::kInt));
    kept_targets = at::empty({rows}, targets.options());
    hidden = at::empty_like(hidden_in);
    int* count = where.data_ptr<int>() + rows;
    lm_head_rows_kernel<<<1, 1024, 0, stream()>>>(p.targets, static_cast<int>(rows), ignore_index, where.data_ptr<int>(),
                                                  kept_targets.data_ptr<int64_t>(), count, log_probs.data_ptr<float>(),
                                                  entropy.data_ptr<float>());
    const int vecs = static_cast<int>(hidden.size(1) / 8);
    lm_head_gather_kernel<<<static_cast<unsigned>(rows), 128, 0, stream()>>>(
        static_cast<const uint4*>(hidden_in.data_ptr()), where.data_ptr<int>(), count, vecs,
        static_cast<uint4*>(hidden.data_ptr()));
    TDSV_LAUNCH_CHECK();
    p.rows = count;
    p.targets = kept_targets.data_ptr<int64_t>();
  }
  const int64_t tiles = (vocab + (keep ? BN : tile_columns(rows, vocab)) - 1) / (keep ? BN : tile_columns(rows, vocab));
  auto part = at::empty({4 * tiles + 1, rows}, f32);
  p.part = reinterpret_cast<float4*>(part.data_ptr<float>());
  p.target_logit = part.data_ptr<float>() + 4 * tiles * rows;
  const CUtensorMap unused{};
  if (keep) launch_head<kStatsKeep, false>(hidden, weight, head_map(logits, (vocab + 7) / 8 * 8, 32), p);
  else if (rows <= Ring<true>::kRows) launch_head<kStats, true>(hidden, weight, unused, p);
  else launch_head<kStats, false>(hidden, weight, unused, p);
  lm_head_join_kernel<<<static_cast<unsigned>((rows + kJoinRows - 1) / kJoinRows), kJoinThreads, 0, stream()>>>(
      p, where.defined() ? where.data_ptr<int>() : nullptr, static_cast<int>(tiles), log_probs.data_ptr<float>(),
      entropy.data_ptr<float>(), save ? reinterpret_cast<float4*>(saved.data_ptr<float>()) : nullptr);
  TDSV_LAUNCH_CHECK();
  return {log_probs, entropy, saved, logits};
}

// bf16 gradient of the logits, [M, V] with rows padded to 16 bytes, from the logits that were kept or else from the
// product again.
at::Tensor lm_head_stats_bwd(const at::Tensor& hidden, const at::Tensor& weight, const at::Tensor& targets,
                             const at::Tensor& saved, const c10::optional<at::Tensor>& logits, double temperature,
                             int64_t ignore_index, const c10::optional<at::Tensor>& g_log_probs,
                             const c10::optional<at::Tensor>& g_entropy) {
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
  if (logits.has_value() && logits->defined()) {
    TDSV_CHECK(logits->is_cuda() && logits->scalar_type() == at::kFloat && logits->dim() == 2 && logits->size(0) == rows &&
                   logits->size(1) == vocab && (rows == 1 || logits->stride(0) == pitch),
               "linear_token_statistics: kept logits");
    p.M = static_cast<int>(rows);
    p.N = static_cast<int>(vocab);
    const int vecs = static_cast<int>(pitch / 8), parts = (vecs + kKeptThreads * kKeptVecs - 1) / (kKeptThreads * kKeptVecs);
    TDSV_CHECK(rows * parts < (int64_t(1) << 31), "linear_token_statistics: too many rows");
    lm_head_kept_kernel<<<static_cast<unsigned>(rows * parts), kKeptThreads, 0, stream()>>>(
        reinterpret_cast<const float4*>(logits->data_ptr<float>()), p, parts, vecs, static_cast<uint4*>(dlogits.data_ptr()));
    TDSV_LAUNCH_CHECK();
    return dlogits;
  }
  launch_head<kGrad, false>(hidden, weight, head_map(dlogits, pitch, 32), p);
  return dlogits;
}

}  // namespace tdsv
