// What the two kernels of attention over a paged cache share: the arguments, a block's stretch of the line of units,
// and the join of tiles that lie in several blocks. The mathematics is at the top of paged_attention.cu.
#pragma once

#include "paged.cuh"
#include "tc_util.cuh"

#include <type_traits>

namespace tdsv {

// The tile that begins in a block and goes on behind it, which is the block's last one, if there is one (rows > 0).
struct Split {
  int last, rows;            // the block that it ends in; rows of the tile
  int start, first, head;    // the sequence's first row of the call; the tile's first row in it; the group's first head
};

struct AttendArgs {
  PagedBatch batch;
  const uint32_t* tree;  // [rows, tree_words]
  int tree_words;        // -1: causal
  int group, hq;
  int tile_rows, slot_rows;  // rows of a tile (token x head of the group), and of a slot of `parts`
  int least;             // units of a block, where there are any
  float scale_log2;      // scale log2(e)
  float* parts;          // [2 blocks] slots of slot_rows x kHeadDim sums of tiles that lie in several blocks
  float2* part_stats;    // [2 blocks][slot_rows]: m, sum
  Split* splits;         // [blocks]
  int* status;

  // Where block `block` keeps its part of a tile that begins in block `first`: a block holds at most one part of a
  // tile that began before it and one of a tile that goes on behind it.
  __device__ __forceinline__ int64_t slot(int block, int first) const {
    return static_cast<int64_t>(2 * block + (block == first ? 1 : 0)) * slot_rows;
  }
};

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// A page that is in the pool: one outside is reported and page 0 read in its stead.
__device__ __forceinline__ int checked_page(const AttendArgs& a, int page) {
  if (page >= 0 && page < a.batch.pages) return page;
  report_status(a.status, kOutOfBounds);
  return 0;
}

// This block's stretch of the line of all units, and where it begins. WORK(sequence) is a sequence's units.
struct Stretch {
  int64_t begin, end, share;  // [begin, end); every block has `share`, the last ones less
  int seq;                    // of unit `begin`
  int64_t offset;             // of it among that sequence's units
};
template <int THREADS>
struct StretchScratch {
  int64_t sums[THREADS / 32];
  int64_t offset;
  int seq;
};
// By all threads of the block: thread t sums the sequences [t * per, ...). Ends with a barrier.
template <int THREADS, typename WORK>
__device__ __forceinline__ Stretch block_stretch(const AttendArgs& a, StretchScratch<THREADS>& sm, const WORK& work) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const PagedBatch& batch = a.batch;
  const int per = (batch.seqs + THREADS - 1) / THREADS;
  int64_t mine = 0;
  for (int i = tid * per; i < min(batch.seqs, (tid + 1) * per); ++i) mine += work(paged_sequence(batch, i, a.status));
  int64_t before = mine;  // inclusive, then exclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += v;
  }
  if (lane == 31) sm.sums[warp] = before;
  __syncthreads();
  int64_t total = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) {
    if (w < warp) before += sm.sums[w];
    total += sm.sums[w];
  }
  before -= mine;
  Stretch s;
  s.share = max(static_cast<int64_t>(a.least), (total + gridDim.x - 1) / gridDim.x);
  s.begin = min(total, s.share * blockIdx.x);
  s.end = min(total, s.begin + s.share);
  if (s.begin < s.end && s.begin >= before && s.begin < before + mine) {
    int64_t at = before;
    for (int i = tid * per; i < batch.seqs; ++i) {
      const int64_t units = work(paged_sequence(batch, i, nullptr));
      if (s.begin < at + units) {
        sm.seq = i;
        sm.offset = s.begin - at;
        break;
      }
      at += units;
    }
  }
  __syncthreads();
  s.seq = sm.seq;
  s.offset = sm.offset;
  return s;
}

// Host, in paged_attention.cu.
void launch_attend_join(const AttendArgs& a, at::Tensor& out, int blocks);
// Host, in paged_rows.cu: attention by tiles of up to 256 rows.
constexpr int kRowsTile = 256;
void launch_attend_rows(const AttendArgs& a, const CUtensorMap& key_map, const CUtensorMap& value_map, const at::Tensor& q,
                        at::Tensor& out, int blocks);

}  // namespace tdsv
