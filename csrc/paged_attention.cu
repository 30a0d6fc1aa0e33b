// Attention of new tokens over a paged cache.
//
// Row (i, h) of a sequence is query head h of its new token i, at position length - n + i. With the keys and values of
// h's key head,
//
//     out = sum_j p_j v_j / sum_j p_j,   p_j = 2^(c (q . k_j) - m),   c = scale log2(e)
//
// over the positions j that the row sees: up to its own, or, under the mask of a drafted tree, those before the new
// tokens and the new tokens whose bit is set. m is the running maximum; sums are fp32, p is rounded to the cache's
// type for its product with v (the sum of p is not, so that a row's weights err by their own roundings alone). A row
// that sees nothing gives zeros, as do rows of the call that no sequence has.
//
// The rows of a sequence under one key head are its n tokens times the heads of the group, in tiles of 16. The keys of
// a tile are cut into units of 128, and all units of all tiles stand in one line, of which each block takes an equal
// stretch: a batch of very different lengths fills the SMs as evenly as one of equal ones, and one long sequence as well
// as many short ones. A tile whose units lie in several blocks is joined by a second kernel from its parts. The line
// follows from starts and lengths on the GPU; each block sums them for itself.
//
// Four warps take 32 of a unit's keys each, with their own running maximum and sum, and with their own ring of
// tiles that TMA fills (192 KB of an SM on the way or at work): no warp waits for another until the tile is joined. A key or
// value crosses HBM once for each 16 rows, and the cache's traffic is what bounds a step: 64 sequences of up to 8192 tokens
// (554 MB) take 106 us, 5.2 TB/s, 8 of up to 40960 tokens 92 us, 5.5 TB/s; one of 4001 tokens 9 us and 3 us for the join.
// Where a sequence brings more rows the kernel of paged_rows.cu takes them: at 32 drafted tokens (256 rows) this one needs
// 563 us for what takes 72 there, at 2048 tokens of a prompt 5632 for 501.
#include "paged_attend.cuh"

namespace tdsv {

namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kTileRows = 16;
constexpr int kWarpKeys = 32, kUnitKeys = kWarps * kWarpKeys;
constexpr int kStages = 3;
constexpr int kHalfBytes = kWarpKeys * 128;   // 64 dims of a warp's keys
constexpr int kSideBytes = 2 * kHalfBytes;    // keys, or values
constexpr int kStageBytes = 2 * kSideBytes;

enum : int { kWaitTile = 341 };

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(at)
               : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same_v<T, __half>)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Units of a sequence: key heads x row tiles x units of keys.
struct Line {
  int tiles, units;  // row tiles, units of keys a tile
  __device__ __forceinline__ Line(const PagedSequence& s, int group) {
    tiles = (s.n * group + kTileRows - 1) / kTileRows;
    units = s.n == 0 ? 0 : (s.length + kUnitKeys - 1) / kUnitKeys;
  }
  __device__ __forceinline__ int64_t all(int kv_heads) const { return static_cast<int64_t>(tiles) * units * kv_heads; }
};

// A place in the line.
struct Cursor {
  int b = -1, head = 0, tile = 0, unit = 0;
  PagedSequence s;
  int tiles = 0, units = 0;

  __device__ __forceinline__ void enter(const AttendArgs& a, int seq) {
    b = seq;
    s = paged_sequence(a.batch, b, nullptr);
    const Line l(s, a.group);
    tiles = l.tiles, units = l.units;
    head = tile = unit = 0;
  }
  __device__ __forceinline__ void place(int64_t offset) {
    unit = static_cast<int>(offset % units);
    offset /= units;
    tile = static_cast<int>(offset % tiles);
    head = static_cast<int>(offset / tiles);
  }
  // (the caller knows that there is a next unit)
  __device__ __forceinline__ void next(const AttendArgs& a) {
    if (++unit < units) return;
    unit = 0;
    if (++tile < tiles) return;
    tile = 0;
    if (++head < a.batch.kv_heads) return;
    do enter(a, b + 1);
    while (units == 0 && b + 1 < a.batch.seqs);
  }
};

struct Shared {
  float out[kWarps][kTileRows][kHeadDim];
  float2 stats[kWarps][kTileRows];
  uint64_t full[kWarps][kStages];
  StretchScratch<kThreads> stretch;
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    attend_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                  const T* __restrict__ q, T* __restrict__ out, const __grid_constant__ AttendArgs a) {
  extern __shared__ uint8_t raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
  Shared& sm = *reinterpret_cast<Shared*>(ring + kWarps * kStages * kStageBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedBatch& batch = a.batch;

  if (tid == 0) {
    a.splits[blockIdx.x].rows = 0;
    for (int i = 0; i < kWarps * kStages; ++i) mbar_init(&sm.full[i / kStages][i % kStages], 1);
    fence_barrier_init();
  }
  const Stretch line = block_stretch(a, sm.stretch, [&](const PagedSequence& s) { return Line(s, a.group).all(batch.kv_heads); });
  if (line.begin >= line.end) return;

  Cursor compute;
  compute.enter(a, line.seq);
  compute.place(line.offset);
  Cursor load = compute;
  const int count = static_cast<int>(line.end - line.begin);  // units of this block
  const int rows_per_box = min(1 << batch.page_shift, kWarpKeys);
  const uint32_t my_ring = smem_u32(ring) + warp * kStages * kStageBytes;

  // Loads unit number `i` of this block into its stage: the warp's 32 keys and values, as far as there are any.
  auto issue = [&](int i) {
    const int key0 = load.unit * kUnitKeys + warp * kWarpKeys;
    if (key0 < load.s.length) {
      uint64_t* bar = &sm.full[warp][i % kStages];
      const uint32_t to = my_ring + (i % kStages) * kStageBytes;
      const int boxes = min(kWarpKeys / rows_per_box, (load.s.length - key0 + rows_per_box - 1) / rows_per_box);
      if (lane == 0) mbar_arrive_expect_tx(bar, boxes * rows_per_box * 512);
      __syncwarp();
      if (lane < boxes) {  // a lane each, so that their pages are looked up together
        const int at = key0 + lane * rows_per_box;
        const int page = checked_page(a, batch.tables[load.b * batch.table_stride + (at >> batch.page_shift)]);
        const int row = at & ((1 << batch.page_shift) - 1);
        const uint32_t box = to + lane * rows_per_box * 128;
        tma_load_4d(box, &key_map, bar, 0, row, load.head, page);
        tma_load_4d(box + kHalfBytes, &key_map, bar, 64, row, load.head, page);
        tma_load_4d(box + kSideBytes, &value_map, bar, 0, row, load.head, page);
        tma_load_4d(box + kSideBytes + kHalfBytes, &value_map, bar, 64, row, load.head, page);
      }
    }
    if (i + 1 < count) load.next(a);
  };
  for (int i = 0; i < min(kStages, count); ++i) issue(i);

  const int g = lane >> 2, c2 = (lane & 3) * 2;
  uint32_t phases = 0;  // of this warp's stages
  uint32_t qf[kHeadDim / 16][4];
  float o[kHeadDim / 8][4], m[2], l[2];
  bool ok = true;
  int token[2];
  for (int i = 0; i < count; ++i) {
    const PagedSequence s = compute.s;
    const int prefix = s.length - s.n;
    if (i == 0 || compute.unit == 0) {  // a new tile
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int row = compute.tile * kTileRows + g + 8 * r;
        token[r] = row < s.n * a.group ? row / a.group : -1;
        m[r] = -INFINITY, l[r] = 0.f;
        const int head = compute.head * a.group + row % a.group;
        const T* from = q + (static_cast<int64_t>(s.start + token[r]) * a.hq + head) * kHeadDim + c2;
#pragma unroll
        for (int k = 0; k < kHeadDim / 16; ++k) {
          qf[k][r] = token[r] < 0 ? 0u : *reinterpret_cast<const uint32_t*>(from + k * 16);
          qf[k][2 + r] = token[r] < 0 ? 0u : *reinterpret_cast<const uint32_t*>(from + k * 16 + 8);
        }
      }
#pragma unroll
      for (int k = 0; k < kHeadDim / 8; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[k][j] = 0.f;
    }
    const int key0 = compute.unit * kUnitKeys + warp * kWarpKeys;
    const int stage = i % kStages;
    if (key0 < s.length) {
      ok = ok && warp_wait(&sm.full[warp][stage], (phases >> stage) & 1, a.status, kWaitTile);
      phases ^= 1u << stage;
      const uint32_t ks = my_ring + stage * kStageBytes, vs = ks + kSideBytes;
      const int here = s.length - key0;  // keys of the tile that exist
      if (here < kWarpKeys) {            // what lies behind them may be anything: a weight of 0 does not undo a NaN
        uint8_t* v = ring + (warp * kStages + stage) * kStageBytes + kSideBytes;
        for (int x = here * 8 + lane; x < kWarpKeys * 8; x += 32) {
          *reinterpret_cast<uint4*>(v + x * 16) = make_uint4(0, 0, 0, 0);
          *reinterpret_cast<uint4*>(v + kHalfBytes + x * 16) = make_uint4(0, 0, 0, 0);
        }
        __syncwarp();
      }
      // scores: 16 rows x 32 keys
      float sc[kWarpKeys / 8][4];
#pragma unroll
      for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) sc[n][j] = 0.f;
#pragma unroll
      for (int k = 0; k < kHeadDim / 16; ++k)
#pragma unroll
        for (int n = 0; n < kWarpKeys / 16; ++n) {
          uint32_t b[4];
          const int row = n * 16 + (lane & 7) + ((lane >> 4) & 1) * 8;
          ldmatrix4(b, ks + (k >> 2) * kHalfBytes + swz(row, (k & 3) * 2 + ((lane >> 3) & 1)));
          mma16816<T>(sc[2 * n], qf[k], b[0], b[1]);
          mma16816<T>(sc[2 * n + 1], qf[k], b[2], b[3]);
        }
      // what each row sees
      if (key0 + kWarpKeys > prefix) {
#pragma unroll
        for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int r = j >> 1, key = key0 + n * 8 + c2 + (j & 1), x = key - prefix;
            bool seen = token[r] >= 0 && key < s.length;
            if (seen && x >= 0) {
              if (a.tree_words < 0) seen = x <= token[r];
              else
                seen = x < a.tree_words * 32 &&
                       (a.tree[static_cast<int64_t>(s.start + token[r]) * a.tree_words + (x >> 5)] >> (x & 31) & 1u);
            }
            if (!seen) sc[n][j] = -INFINITY;
          }
      }
      float alpha[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float mx = -INFINITY;
#pragma unroll
        for (int n = 0; n < kWarpKeys / 8; ++n) mx = fmaxf(mx, fmaxf(sc[n][2 * r], sc[n][2 * r + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        mx = fmaxf(m[r], mx * a.scale_log2);
        const float base = mx == -INFINITY ? 0.f : mx;
        alpha[r] = ex2_approx(m[r] - base);
        m[r] = mx;
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < kWarpKeys / 8; ++n)
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float p = ex2_approx(fmaf(sc[n][2 * r + j], a.scale_log2, -base));
            sc[n][2 * r + j] = p;
            sum += p;
          }
        l[r] = l[r] * alpha[r] + sum;  // this lane's columns; the others' are added at the end
      }
#pragma unroll
      for (int n = 0; n < kHeadDim / 8; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][j] *= alpha[j >> 1];
#pragma unroll
      for (int k = 0; k < kWarpKeys / 16; ++k) {
        const uint32_t p[4] = {pack2<T>(sc[2 * k][0], sc[2 * k][1]), pack2<T>(sc[2 * k][2], sc[2 * k][3]),
                               pack2<T>(sc[2 * k + 1][0], sc[2 * k + 1][1]), pack2<T>(sc[2 * k + 1][2], sc[2 * k + 1][3])};
#pragma unroll
        for (int n = 0; n < kHeadDim / 16; ++n) {
          uint32_t b[4];
          const int row = k * 16 + (lane & 15), chunk = n * 2 + (lane >> 4);
          ldmatrix4_t(b, vs + (chunk >> 3) * kHalfBytes + swz(row, chunk & 7));
          mma16816<T>(o[2 * n], p, b[0], b[1]);
          mma16816<T>(o[2 * n + 1], p, b[2], b[3]);
        }
      }
      if (here < kWarpKeys) fence_proxy_async_smem();  // the zeros, before TMA writes there again
      __syncwarp();
    }
    if (i + kStages < count) issue(i + kStages);

    if (compute.unit == compute.units - 1 || i == count - 1) {  // the tile's last unit here: the four warps' parts join
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
        l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
        if ((lane & 3) == 0) sm.stats[warp][g + 8 * r] = make_float2(m[r], l[r]);
#pragma unroll
        for (int n = 0; n < kHeadDim / 8; ++n)
          *reinterpret_cast<float2*>(&sm.out[warp][g + 8 * r][n * 8 + c2]) = make_float2(o[n][2 * r], o[n][2 * r + 1]);
      }
      __syncthreads();
      const int64_t unit0 = line.begin + i - compute.unit;  // the tile's place in the line
      const int first = static_cast<int>(unit0 / line.share), last = static_cast<int>((unit0 + compute.units - 1) / line.share);
      const bool whole = first == last;
      const int64_t slot = a.slot(blockIdx.x, first);
      for (int x = tid; x < kTileRows * kHeadDim / 4; x += kThreads) {
        const int r = x / (kHeadDim / 4), d = x % (kHeadDim / 4) * 4;
        const int row = compute.tile * kTileRows + r;
        if (row >= s.n * a.group) break;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm.stats[w][r].x);
        const float base = mx == -INFINITY ? 0.f : mx;
        float sum = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
          const float2 st = sm.stats[w][r];
          const float f = ex2_approx(st.x - base);
          const float4 part = *reinterpret_cast<const float4*>(&sm.out[w][r][d]);
          sum += f * st.y;
          v.x += f * part.x, v.y += f * part.y, v.z += f * part.z, v.w += f * part.w;
        }
        const int t = s.start + row / a.group;
        if (whole) {
          const float inv = sum == 0.f ? 0.f : 1.f / sum;
          T* to = out + (static_cast<int64_t>(t) * a.hq + compute.head * a.group + row % a.group) * kHeadDim + d;
          *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
        } else {
          *reinterpret_cast<float4*>(a.parts + (slot + r) * kHeadDim + d) = v;
          if (d == 0) a.part_stats[slot + r] = make_float2(mx, sum);
        }
      }
      if (tid == 0 && !whole && first == static_cast<int>(blockIdx.x))
        a.splits[first] = {last, min(kTileRows, s.n * a.group - compute.tile * kTileRows), s.start, compute.tile * kTileRows,
                           compute.head * a.group};
      __syncthreads();
    }
    if (i + 1 < count) compute.next(a);
  }
}

// Rows that no sequence has: zeros, a thread a row.
constexpr int kJoinThreads = 256;
template <typename T>
__device__ __forceinline__ void zero_row(T* out, const AttendArgs& a, int t) {
  if (t >= a.batch.rows) return;
  int lo = 0, hi = a.batch.seqs;  // the sequences whose rows end at or before t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (a.batch.starts[mid + 1] <= t) lo = mid + 1;
    else hi = mid;
  }
  if (lo < a.batch.seqs) {
    const PagedSequence s = paged_sequence(a.batch, lo, nullptr);
    if (t >= s.start && t < s.start + s.n) return;
  }
  uint4* to = reinterpret_cast<uint4*>(out + static_cast<int64_t>(t) * a.hq * kHeadDim);
  for (int i = 0; i < a.hq * kHeadDim / 8; ++i) to[i] = make_uint4(0, 0, 0, 0);
}

// Joins the parts of tiles that lie in several blocks. The first blocks of the grid are for the tiles that begin in each
// block of the attention, `per_tile` of them for each; the others look for rows that no sequence has.
//
// Tiles of 16 rows: WARPS warps a row, each with a share of the parts. (A single sequence's row has 32 of them: one warp took
// 18 us for it, twice as long as the attention itself.)
template <typename T, int WARPS>
__global__ void __launch_bounds__(kJoinThreads) attend_join_kernel(T* __restrict__ out, const __grid_constant__ AttendArgs a,
                                                                   int blocks, int per_tile) {
  constexpr int kRows = kJoinThreads / 32 / WARPS;
  __shared__ float4 sums[kRows][WARPS][32];
  __shared__ float2 stats[kRows][WARPS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (static_cast<int>(blockIdx.x) >= blocks * per_tile) {
    zero_row(out, a, (blockIdx.x - blocks * per_tile) * kJoinThreads + threadIdx.x);
    return;
  }
  const int first = blockIdx.x / per_tile;
  const Split split = a.splits[first];
  const int r = (blockIdx.x - first * per_tile) * kRows + warp / WARPS, w0 = warp % WARPS;
  if (r - warp / WARPS >= split.rows) return;  // (the whole block)
  const bool there = r < split.rows;
  const int row = split.first + r, last = there ? split.last : -1;
  float mx = -INFINITY, sum = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x0 = first + w0; x0 <= last; x0 += 4 * WARPS) {  // four parts at once
    float2 st[4];
    float4 part[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int x = x0 + u * WARPS;
      st[u] = make_float2(-INFINITY, 0.f);
      part[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (x > last) continue;
      const int64_t slot = a.slot(x, first);
      st[u] = a.part_stats[slot + r];
      part[u] = *reinterpret_cast<const float4*>(a.parts + (slot + r) * kHeadDim + 4 * lane);
    }
    const float to_max = fmaxf(fmaxf(fmaxf(st[0].x, st[1].x), fmaxf(st[2].x, st[3].x)), mx);
    const float base = to_max == -INFINITY ? 0.f : to_max, old = ex2_approx(mx - base);
    mx = to_max;
    sum *= old;
    v.x *= old, v.y *= old, v.z *= old, v.w *= old;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float f = ex2_approx(st[u].x - base);
      sum += f * st[u].y;
      v.x += f * part[u].x, v.y += f * part[u].y, v.z += f * part[u].z, v.w += f * part[u].w;
    }
  }
  {
    const int x = warp / WARPS;
    sums[x][w0][lane] = v;
    if (lane == 0) stats[x][w0] = make_float2(mx, sum);
    __syncthreads();
    if (w0 != 0) return;
    mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, stats[x][w].x);
    const float base = mx == -INFINITY ? 0.f : mx;
    sum = 0.f;
    v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const float f = ex2_approx(stats[x][w].x - base);
      const float4 part = sums[x][w][lane];
      sum += f * stats[x][w].y;
      v.x += f * part.x, v.y += f * part.y, v.z += f * part.z, v.w += f * part.w;
    }
  }
  if (!there) return;
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  T* to = out + (static_cast<int64_t>(split.start + row / a.group) * a.hq + split.head + row % a.group) * kHeadDim + 4 * lane;
  *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x * inv, v.y * inv), pack2<T>(v.z * inv, v.w * inv));
}

// Tiles of 256 rows, whose parts lie four dims of all rows after the next four: a warp takes eight rows, a lane one of them
// and every fourth quadruple of dims, so that a part's eight loads a lane are on their way together.
template <typename T>
__global__ void __launch_bounds__(kJoinThreads) attend_join_rows_kernel(T* __restrict__ out, const __grid_constant__ AttendArgs a,
                                                                        int blocks, int per_tile) {
  if (static_cast<int>(blockIdx.x) >= blocks * per_tile) {
    zero_row(out, a, (blockIdx.x - blocks * per_tile) * kJoinThreads + threadIdx.x);
    return;
  }
  const int first = blockIdx.x / per_tile, lane = threadIdx.x & 31;
  const Split split = a.splits[first];
  const int r = (blockIdx.x - first * per_tile) * (kJoinThreads / 4) + (threadIdx.x >> 5) * 8 + (lane & 7), d = lane >> 3;
  if (r >= split.rows) return;
  float mx = -INFINITY;
  for (int x = first; x <= split.last; ++x) mx = fmaxf(mx, a.part_stats[a.slot(x, first) + r].x);
  const float base = mx == -INFINITY ? 0.f : mx;
  float sum = 0.f;
  float4 v[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int x = first; x <= split.last; ++x) {
    const int64_t slot = a.slot(x, first);
    const float4* from = reinterpret_cast<const float4*>(a.parts + slot * kHeadDim) + r;
    float4 part[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) part[i] = from[(d + 4 * i) * kRowsTile];
    const float2 st = a.part_stats[slot + r];
    const float f = ex2_approx(st.x - base);
    sum += f * st.y;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      v[i].x += f * part[i].x, v[i].y += f * part[i].y, v[i].z += f * part[i].z, v[i].w += f * part[i].w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int row = split.first + r;
  T* to = out + (static_cast<int64_t>(split.start + row / a.group) * a.hq + split.head + row % a.group) * kHeadDim + 4 * d;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    *reinterpret_cast<uint2*>(to + 16 * i) = make_uint2(pack2<T>(v[i].x * inv, v[i].y * inv), pack2<T>(v[i].z * inv, v[i].w * inv));
}

CUtensorMap pool_map(const at::Tensor& pool, int box_rows) {
  const PoolStrides s = pool_strides(pool);
  CUtensorMap map;
  const cuuint64_t dims[4] = {kHeadDim, static_cast<cuuint64_t>(pool.size(2)), static_cast<cuuint64_t>(pool.size(1)),
                              static_cast<cuuint64_t>(pool.size(0))};
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(s.row) * 2, static_cast<cuuint64_t>(s.head) * 2,
                                 static_cast<cuuint64_t>(s.page) * 2};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_rows), 1, 1}, steps[4] = {1, 1, 1, 1};
  const CUresult r = encode_fn()(&map, pool.scalar_type() == at::kHalf ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                                 4, pool.data_ptr(), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  TDSV_CHECK(r == CUDA_SUCCESS, "paged_attention: the cache's layout was refused (", static_cast<int>(r), ")");
  return map;
}

}  // namespace

void launch_attend_join(const AttendArgs& a, at::Tensor& out, int blocks) {
  auto launch = [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto go = [&](auto kern, int rows) {  // rows of a tile that a block takes
      const int per_tile = (a.tile_rows + rows - 1) / rows;
      const unsigned grid = static_cast<unsigned>(blocks * per_tile + (a.batch.rows + kJoinThreads - 1) / kJoinThreads);
      kern<<<grid, kJoinThreads, 0, stream()>>>(static_cast<T*>(out.data_ptr()), a, blocks, per_tile);
    };
    if (a.slot_rows > kTileRows) go(attend_join_rows_kernel<T>, kJoinThreads / 4);
    else go(attend_join_kernel<T, 4>, kJoinThreads / 32 / 4);
  };
  if (out.scalar_type() == at::kHalf) launch(static_cast<__half*>(nullptr));
  else launch(static_cast<__nv_bfloat16*>(nullptr));
  TDSV_LAUNCH_CHECK();
}

at::Tensor paged_attention(const at::Tensor& q, const at::Tensor& keys, const at::Tensor& values, const at::Tensor& tables,
                           const at::Tensor& starts, const at::Tensor& lengths, double scale,
                           const c10::optional<at::Tensor>& tree) {
  constexpr const char* what = "paged_attention";
  check_cuda_tensor(q, "q");
  c10::cuda::CUDAGuard guard(q.device());
  TDSV_CHECK(q.dim() == 3 && q.size(2) == kHeadDim && q.size(1) >= 1, what, ": q must be [rows, heads, 128]");
  TDSV_CHECK(keys.device() == q.device() && keys.scalar_type() == q.scalar_type(), what, ": q and the cache must be alike");
  TDSV_CHECK(reinterpret_cast<uintptr_t>(q.data_ptr()) % 16 == 0, what, ": q must start on 16 bytes");
  const int64_t rows = q.size(0), hq = q.size(1);
  AttendArgs a{};
  a.batch = paged_batch(keys, values, tables, starts, lengths, rows, what);
  TDSV_CHECK(hq % a.batch.kv_heads == 0 && rows * hq < (int64_t(1) << 30), what, ": heads must be a multiple of the cache's");
  a.group = static_cast<int>(hq / a.batch.kv_heads);
  a.hq = static_cast<int>(hq);
  a.scale_log2 = static_cast<float>(scale * 1.4426950408889634);
  a.tree_words = -1;
  if (tree.has_value() && tree->defined()) {
    check_cuda_tensor(*tree, "tree");
    TDSV_CHECK(tree->device() == q.device() && tree->scalar_type() == at::kInt && tree->dim() == 2 && tree->size(0) == rows &&
                   tree->size(1) < (1 << 24),
               what, ": tree must be int32 [rows, words]");
    a.tree = reinterpret_cast<const uint32_t*>(tree->data_ptr<int>());
    a.tree_words = static_cast<int>(tree->size(1));
  }
  auto out = at::empty_like(q);
  if (rows == 0) return out;
  a.status = status_word_ptr();
  // A tile of 16 rows reads its keys once for all of a decoding step's rows; where a sequence brings more (on average),
  // tiles of 256 do: 64 sequences of 4000 tokens take 115 us by the one and 131 by the other at 16 rows, 188 and 131 at 24.
  // While SMs are idle another tile of 16 costs less than the other kernel's longer start: a single sequence of 4000
  // tokens takes 18 and 25 us at 16 rows, 23 and 29 at 64, 29 and 29 at 128 (512 rows over all heads).
  const int64_t most_tokens = (static_cast<int64_t>(a.batch.seqs) * a.batch.width) << a.batch.page_shift;
  const bool idle = rows * hq <= 512 && most_tokens <= 8192;
  const bool many = a.group <= kRowsTile && rows * a.group > kTileRows * static_cast<int64_t>(a.batch.seqs) && !idle;
  const int blocks = num_sms();
  a.tile_rows = many ? kRowsTile / a.group * a.group : kTileRows;
  a.slot_rows = many ? kRowsTile : kTileRows;
  a.least = many ? 2 : 1;  // (a tile's end costs that kernel as much as some units)
  const auto f32 = q.options().dtype(at::kFloat);
  // parts, their statistics and the splits, in one allocation
  const int64_t slots = 2 * static_cast<int64_t>(blocks) * a.slot_rows;
  auto workspace = at::empty({slots * (kHeadDim + 2) + blocks * static_cast<int64_t>(sizeof(Split) / sizeof(float))}, f32);
  a.parts = workspace.data_ptr<float>();
  a.part_stats = reinterpret_cast<float2*>(a.parts + slots * kHeadDim);
  a.splits = reinterpret_cast<Split*>(a.parts + slots * (kHeadDim + 2));
  bind_primary_context();
  const int box_rows = std::min(1 << a.batch.page_shift, many ? 128 : kWarpKeys);
  const CUtensorMap key_map = pool_map(keys, box_rows), value_map = pool_map(values, box_rows);
  if (many) {
    launch_attend_rows(a, key_map, value_map, q, out, blocks);
  } else {
    auto launch = [&](auto* tag) {
      using T = std::remove_pointer_t<decltype(tag)>;
      constexpr int smem = kWarps * kStages * kStageBytes + sizeof(Shared) + 1024;
      static_assert(smem <= 227 * 1024, "fits an SM");
      TDSV_CUDA_CHECK(cudaFuncSetAttribute(attend_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
      attend_kernel<T><<<blocks, kThreads, smem, stream()>>>(key_map, value_map, static_cast<const T*>(q.data_ptr()),
                                                             static_cast<T*>(out.data_ptr()), a);
    };
    if (q.scalar_type() == at::kHalf) launch(static_cast<__half*>(nullptr));
    else launch(static_cast<__nv_bfloat16*>(nullptr));
    TDSV_LAUNCH_CHECK();
  }
  launch_attend_join(a, out, blocks);
  return out;
}

}  // namespace tdsv
