// Attention over a paged cache where a sequence brings many rows: chunks of prompts and trees of drafted tokens.
// (The mathematics, and the line of units that the blocks share, are at the top of paged_attention.cu.)
//
// A tile is up to 256 rows of one sequence and key head, whole tokens of them, as two halves of 128 (one of the
// tensor cores' tiles each) that share every key and value. 576 threads:
//   warp 0       producer: the unit's 128 keys, then its 128 values, by TMA through a ring of five slots of 32 KB; a lane
//                a page, so that the pages are looked up together
//   warp 1       issues the products: for each half PV of this unit as its weights arrive, then QK of the next one
//   warps 2-17   softmax, two threads per row, of 64 keys each: scores from tensor memory into registers, the row's mask,
//                the running maximum (agreed on through shared memory; raised only when it grows by more than 2^8, so that
//                the sums in tensor memory are rarely rescaled), the weights back over the scores as the A operand of PV
// While one half's softmax runs, the tensor cores work on the other half. What bounds it is the chain of a half: its
// softmax (2400 cycles: read 400, the rows' maxima agreed on 300, the exponentials and their way back 1700), then its
// products (1100), and a wake-up at either end (250 each): 4000 cycles a unit, of which the tensor cores work 2200. Three
// chunks of prompts (5312 new tokens on 17535 cached, 459 GFLOP) take 0.47 to 0.51 ms, 0.9 to 1.0 PFLOP/s. Tried: one
// thread a row (the scores spill, to L2, as the ring leaves next to nothing of L1: 1313 us), all 64 scores in registers
// (172 bytes spilled: 506 us against 463), a part of the exponentials as polynomials (595 and 654 us against 564: the
// instructions cost more than the special-function unit's time that they save).
//   TMEM: scores 0 [0, 128), scores 1 [128, 256), sums 0 [256, 384), sums 1 [384, 512).
// Commits of QK come behind the half's last PV, so a thread that sees its next scores may touch its sums.
#include "logit_rows.cuh"
#include "paged_attend.cuh"

namespace tdsv {

namespace {

constexpr int kThreads = 576;
constexpr int kHalfRows = 128, kUnitKeys = 128;
constexpr int kAtomBytes = 128 * 128;    // 128 rows of 64 dims, swizzled
constexpr int kSlotBytes = 2 * kAtomBytes;
constexpr int kSlots = 5;
constexpr int kSplitThread = 64;          // of the first half's softmax, which every tile has

enum : int { kWaitEmpty = 351, kWaitQ, kWaitKeys, kWaitValues, kWaitWeights, kWaitScores, kWaitSums, kWaitTail,
              kWaitPair };

// A warp's wait that polls: a suspended one wakes late, and these are on the path from one product to the next (1.5 % of
// a long chunk).
__device__ __forceinline__ bool spin_wait(uint64_t* bar, uint32_t parity, int* status, int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, code));
}

template <typename T>
__device__ __forceinline__ uint32_t product_desc(bool b_mn_major) {
  const uint32_t d = make_idesc_bf16(128, 128, false, b_mn_major);
  return std::is_same_v<T, __half> ? d & ~(1u << 7 | 1u << 10) : d;  // (fp16 is format 0)
}

// sum over 0 <= i < n of floor((a i + b) / m): the lattice points under a line, by Euclid's steps.
__device__ __forceinline__ int64_t floor_sum(uint32_t n, uint32_t m, uint32_t a, uint32_t b) {
  int64_t sum = 0;
  while (n > 0) {
    const uint32_t qa = a / m, qb = b / m;
    sum += static_cast<int64_t>(n) * (n - 1) / 2 * qa + static_cast<int64_t>(n) * qb;
    a -= qa * m;
    b -= qb * m;
    const uint64_t y = static_cast<uint64_t>(a) * n + b;
    if (y < m) break;
    // (a < m <= 256 and n < 2^24 from the first step on, so y fits 32 bits)
    n = static_cast<uint32_t>(y) / m;
    b = static_cast<uint32_t>(y) - n * m;
    const uint32_t x = a;
    a = m;
    m = x;
  }
  return sum;
}

// The units of a sequence's tiles under one key head: a causal tile ends with its last token.
struct Tiles {
  int tokens, prefix, n, tiles;  // tokens of a tile; cached before the new ones; new ones
  bool causal;

  __device__ __forceinline__ Tiles(const AttendArgs& a, const PagedSequence& s)
      : tokens(a.tile_rows / a.group), prefix(s.length - s.n), n(s.n), tiles((s.n + tokens - 1) / tokens),
        causal(a.tree_words < 0) {}
  Tiles() = default;
  __device__ __forceinline__ int units(int t) const {
    return (prefix + (causal ? min(n, (t + 1) * tokens) : n) + kUnitKeys - 1) / kUnitKeys;
  }
  __device__ __forceinline__ int64_t before(int t) const {  // tiles [0, t)
    if (!causal) return static_cast<int64_t>(t) * units(0);
    if (t == 0) return 0;
    const int64_t full = t == tiles ? units(tiles - 1) : 0;
    return full + floor_sum(t == tiles ? t - 1 : t, kUnitKeys, tokens, prefix + tokens + kUnitKeys - 1);
  }
  __device__ __forceinline__ int64_t all() const { return n == 0 ? 0 : before(tiles); }
  // The tile of unit `offset`, which becomes its number within the tile.
  __device__ __forceinline__ int find(int64_t& offset) const {
    if (!causal) {
      const int t = static_cast<int>(static_cast<uint32_t>(offset) / static_cast<uint32_t>(units(0)));
      offset -= before(t);
      return t;
    }
    // before(t) is about (tokens t^2 / 2 + (prefix + 64 + tokens / 2) t) / 128: a guess, and a step or two
    const float half = prefix + 64.f + 0.5f * tokens;
    const float guess = (sqrtf(half * half + 256.f * tokens * static_cast<float>(offset)) - half) / tokens;
    int t = max(0, min(tiles - 1, static_cast<int>(guess)));
    int64_t at = before(t);
    while (t > 0 && at > offset) at -= units(--t);
    while (t < tiles - 1 && at + units(t) <= offset) at += units(t++);
    offset -= at;
    return t;
  }
};

// A tile of the line, and what a block does of it: `count` units from `unit` on.
struct Place {
  int b, head, tile;
};
struct Part {
  PagedSequence s;
  Tiles t;
  int unit, units, count, rows;

  __device__ __forceinline__ Part(const AttendArgs& a, const Place& at, int unit_, int left)
      : s(paged_sequence(a.batch, at.b, nullptr)), t(a, s), unit(unit_), units(t.units(at.tile)),
        count(min(left, units - unit)), rows(min(t.tokens, s.n - at.tile * t.tokens) * a.group) {}
  // (the caller knows that there is a next tile)
  __device__ __forceinline__ void next(const AttendArgs& a, Place& at) const {
    ++at.tile;
    if (at.tile == t.tiles) at.tile = 0, ++at.head;
    if (at.head == a.batch.kv_heads) {
      at.head = 0;
      ++at.b;
      while (at.b + 1 < a.batch.seqs && paged_sequence(a.batch, at.b, nullptr).n == 0) ++at.b;
    }
  }
};

struct Shared {
  uint64_t q_full[2], s_full[2], p_full[2], o_full[2];
  uint64_t kv_full[kSlots], kv_empty[kSlots];
  uint64_t pair[8];           // the two threads of each of a quarter's rows
  float exchange[2][2][kHalfRows];  // [half][part of the keys][row]: maxima, then sums
  StretchScratch<kThreads> stretch;
  Stretch line;
  uint32_t tmem;
};

// 16 columns of this warp's 32 TMEM lanes.
__device__ __forceinline__ void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

// The largest of three.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// 32 columns of a row's mask, from column `x` of the new tokens on (negative: before them).
__device__ __forceinline__ uint32_t tree_columns(const uint32_t* words, int count, int n, int x) {
  auto word = [&](int i) { return i >= 0 && i < count ? words[i] : 0u; };
  uint32_t seen;
  if (x <= -32) return 0xffffffffu;
  if (x < 0) seen = (1u << -x) - 1u | word(0) << -x;
  else seen = __funnelshift_r(word(x >> 5), word((x >> 5) + 1), x & 31);
  const int left = n - x;  // columns that are there
  return left >= 32 ? seen : left <= 0 ? 0u : seen & ((1u << left) - 1u);
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1)
    attend_rows_kernel(const __grid_constant__ CUtensorMap key_map, const __grid_constant__ CUtensorMap value_map,
                       const T* __restrict__ q, T* __restrict__ out, const __grid_constant__ AttendArgs a) {
  extern __shared__ __align__(1024) uint8_t queries[];  // two halves of two atoms, then the ring
  uint8_t* ring = queries + 2 * kSlotBytes;
  Shared& sm = *reinterpret_cast<Shared*>(ring + kSlots * kSlotBytes);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == kSplitThread) a.splits[blockIdx.x].rows = 0;
  if (tid == 0) {
    for (int h = 0; h < 2; ++h) {
      mbar_init(&sm.q_full[h], 2 * kHalfRows);
      mbar_init(&sm.s_full[h], 1);
      mbar_init(&sm.p_full[h], 2 * kHalfRows);
      mbar_init(&sm.o_full[h], 1);
    }
    for (int i = 0; i < 8; ++i) mbar_init(&sm.pair[i], 64);
    for (int i = 0; i < kSlots; ++i) mbar_init(&sm.kv_full[i], 1), mbar_init(&sm.kv_empty[i], 1);
    fence_barrier_init();
  }
  const Stretch line = block_stretch(a, sm.stretch, [&](const PagedSequence& s) {
    return Tiles(a, s).all() * a.batch.kv_heads;
  });
  if (line.begin >= line.end) return;
  if (smem_u32(queries) & 1023u) {  // (the swizzle counts on it)
    report_status(a.status, kBadShape);
    return;
  }
  if (tid == 0) sm.line = line;
  if (warp == 1) {
    tmem_alloc(&sm.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sm.tmem;

  Place at{line.seq, 0, 0};
  int unit;  // where the block's first tile begins for it; later ones begin with their first
  {
    const Tiles t(a, paged_sequence(a.batch, at.b, nullptr));
    const int64_t all = t.all();
    at.head = static_cast<int>(line.offset / all);
    int64_t offset = line.offset - at.head * all;
    at.tile = t.find(offset);
    unit = static_cast<int>(offset);
  }
  int left = static_cast<int>(line.end - line.begin);  // units of this block
  bool ok = true;

  if (warp < 2) {
    if (warp == 0) {
      const int rows_per_box = min(1 << a.batch.page_shift, kUnitKeys);
      int slot = 0, round = 0;
      while (ok && left > 0) {
        const Part p(a, at, unit, left);
        const int* table = a.batch.tables + at.b * a.batch.table_stride;
        // this lane's page of a unit, looked up a unit ahead of its keys and kept for its values
        const auto look = [&](int u) {
          const int place = u * kUnitKeys + lane * rows_per_box;
          return lane < kUnitKeys / rows_per_box && place < p.s.length ? table[place >> a.batch.page_shift] : -1;
        };
        const auto load = [&](const CUtensorMap* map, int u, int page) {
          if (round > 0 && ok) ok = warp_wait(&sm.kv_empty[slot], (round - 1) & 1, a.status, kWaitEmpty);
          if (!ok) return;
          const int place = u * kUnitKeys + lane * rows_per_box;
          const int boxes = min(kUnitKeys / rows_per_box, (p.s.length - u * kUnitKeys + rows_per_box - 1) / rows_per_box);
          if (lane == 0) mbar_arrive_expect_tx(&sm.kv_full[slot], boxes * rows_per_box * 256);
          __syncwarp();
          if (lane < boxes) {
            const int row = place & ((1 << a.batch.page_shift) - 1);
            const uint32_t to = smem_u32(ring) + slot * kSlotBytes + lane * rows_per_box * 128;
            page = checked_page(a, page);
            tma_load_4d(to, map, &sm.kv_full[slot], 0, row, at.head, page);
            tma_load_4d(to + kAtomBytes, map, &sm.kv_full[slot], 64, row, at.head, page);
          }
          if (++slot == kSlots) slot = 0, ++round;
        };
        // keys of a unit before the values of the one before it: their product comes first
        int now = look(unit), next = look(unit + 1);
        load(&key_map, unit, now);
        for (int i = 1; i <= p.count; ++i) {
          const int before = now;
          now = next;
          if (i + 1 < p.count) next = look(unit + i + 1);
          if (i < p.count) load(&key_map, unit + i, now);
          load(&value_map, unit + i - 1, before);
        }
        left -= p.count;
        unit = 0;
        if (left > 0) p.next(a, at);
      }
    } else {
      if (elect_one()) {
        const uint32_t desc_s = product_desc<T>(false), desc_o = product_desc<T>(true);
        const uint32_t qs = smem_u32(queries), rs = smem_u32(ring);
        int slot = 0, slot_round = 0;
        uint32_t q_turn = 0, p_turn = 0;  // parities, a bit for each half
        auto take = [&](int code) {  // the ring's next slot, when it is full
          ok = ok && mbar_wait(&sm.kv_full[slot], slot_round & 1, a.status, code);
          const int s = slot;
          if (++slot == kSlots) slot = 0, ++slot_round;
          return s;
        };
        auto scores = [&](int h, int s) {
#pragma unroll
          for (int k = 0; k < kHeadDim / 16; ++k)
            umma_f16(tmem + h * 128, kmajor_desc(qs + h * kSlotBytes, k, kAtomBytes),
                     kmajor_desc(rs + s * kSlotBytes, k, kAtomBytes), desc_s, k > 0);
          umma_commit(&sm.s_full[h]);
        };
        auto sums = [&](int h, int s, bool more) {
#pragma unroll
          for (int k = 0; k < kUnitKeys / 16; ++k)
            umma_f16_ts(tmem + 256 + h * 128, tmem + h * 128 + (k >> 1) * 32 + (k & 1) * 8, mnmajor_desc(rs + s * kSlotBytes, k, kAtomBytes),
                        desc_o, more || k > 0);
        };
        while (ok && left > 0) {
          const Part p(a, at, unit, left);
          const int halves = p.rows > kHalfRows ? 2 : 1;
          const int first = take(kWaitKeys);
          for (int h = 0; ok && h < halves; ++h) {
            ok = mbar_wait(&sm.q_full[h], q_turn >> h & 1, a.status, kWaitQ);
            q_turn ^= 1u << h;
            if (!ok) break;
            tc_fence_after();
            scores(h, first);
          }
          if (!ok) break;
          umma_commit(&sm.kv_empty[first]);
          for (int i = 0; ok && i < p.count; ++i) {
            const bool more = i + 1 < p.count;
            const int ks = more ? take(kWaitKeys) : 0;
            const int vs = take(kWaitValues);
            for (int h = 0; ok && h < halves; ++h) {
              ok = mbar_wait(&sm.p_full[h], p_turn >> h & 1, a.status, kWaitWeights);
              p_turn ^= 1u << h;
              if (!ok) break;
              tc_fence_after();
              sums(h, vs, i > 0);
              if (more) scores(h, ks);
              else umma_commit(&sm.o_full[h]);
            }
            if (!ok) break;
            umma_commit(&sm.kv_empty[vs]);
            if (more) umma_commit(&sm.kv_empty[ks]);
          }
          left -= p.count;
          unit = 0;
          if (left > 0) p.next(a, at);
        }
      }
      __syncwarp();
    }
  } else {
    const int half = (warp - 2) >> 3, part = (warp - 2) >> 2 & 1, quarter = warp & 3, r = quarter * 32 + lane;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t s_col = lanes + half * 128 + part * 64, o_col = s_col + 256;
    uint8_t* staged = queries + half * kSlotBytes + part * kAtomBytes;  // 64 dims of the half's rows
    uint64_t* pair_bar = &sm.pair[half * 4 + quarter];
    uint32_t pair_turn = 0, s_turn = 0, o_turn = 0;
    while (ok && left > 0) {
      const Part p(a, at, unit, left);
      const int row = half * kHalfRows + r;
      const bool active = p.rows > half * kHalfRows, there = row < p.rows;
      const int token = there ? at.tile * p.t.tokens + row / a.group : 0;
      if (active) {
        // the row's 64 dims in q and out; eight lanes move one row's 128 bytes
        const int64_t to = (static_cast<int64_t>(p.s.start + token) * a.hq + at.head * a.group + row % a.group) * kHeadDim + part * 64;
        const int mine = there ? static_cast<int>(to / 64) : -1, sub = lane >> 3, chunk = lane & 7;
        uint4 v[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) {
          const int from = __shfl_sync(0xffffffffu, mine, x * 4 + sub);
          v[x] = make_uint4(0, 0, 0, 0);
          if (from >= 0) v[x] = *reinterpret_cast<const uint4*>(q + static_cast<int64_t>(from) * 64 + chunk * 8);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) *reinterpret_cast<uint4*>(staged + swz(quarter * 32 + x * 4 + sub, chunk)) = v[x];
        fence_proxy_async_smem();
        tc_fence_before();  // (the sums of the last tile have been read)
        mbar_arrive(&sm.q_full[half]);
        float m = -INFINITY, l = 0.f;
        for (int i = 0; i < p.count; ++i) {
          const int key0 = (unit + i) * kUnitKeys;
          if (half == 0 && key0 + kUnitKeys > p.s.length) {
            // what lies behind the sequence may be anything, and a weight of 0 does not undo a NaN
            // (values of unit i: behind the keys of the next one, where the tile has one here)
            const int n = 2 * (static_cast<int>(sm.line.end - sm.line.begin) - left + i) + (i + 1 < p.count ? 2 : 1), s = n % kSlots;
            if (!(ok = warp_wait(&sm.kv_full[s], (n / kSlots) & 1, a.status, kWaitTail))) break;
            if (key0 + r >= p.s.length) {
              uint8_t* z = ring + s * kSlotBytes + part * kAtomBytes + r * 128;
#pragma unroll
              for (int c = 0; c < 8; ++c) *reinterpret_cast<uint4*>(z + c * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
          }
          if (!(ok = spin_wait(&sm.s_full[half], s_turn & 1, a.status, kWaitScores))) break;
          s_turn ^= 1;
          tc_fence_after();
          // what the row sees; nothing is hidden before the tile's first token
          const int x0 = key0 - p.t.prefix;
          const bool masked = x0 + kUnitKeys > (p.t.causal ? at.tile * p.t.tokens : 0);
          uint32_t seen[2];
          if (masked) {
            const uint32_t* words = a.tree + static_cast<int64_t>(p.s.start + token) * max(a.tree_words, 0);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const int x = x0 + part * 64 + c * 32;
              if (p.t.causal) {
                const int see = token - x + 1;
                seen[c] = see >= 32 ? 0xffffffffu : see <= 0 ? 0u : (1u << see) - 1u;
              } else {
                seen[c] = tree_columns(words, a.tree_words, p.s.n, x);
              }
            }
          }
          // 32 scores at a time, which is what the registers hold: the first ones are read again for their weights
          uint32_t sv[32];
          const auto hide = [&](int c) {
            if (masked) {
#pragma unroll
              for (int j = 0; j < 32; ++j)
                if (!(seen[c] >> j & 1u)) sv[j] = __float_as_uint(-INFINITY);
            }
          };
          float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            tmem_ld_32x32b_x32(s_col + c * 32, sv);
            tmem_ld_wait();
            hide(c);
#pragma unroll
            for (int j = 0; j < 32; j += 2)
              m4[j / 2 & 3] = max3(m4[j / 2 & 3], __uint_as_float(sv[j]), __uint_as_float(sv[j + 1]));
          }
          sm.exchange[half][part][r] = fmaxf(max3(m4[0], m4[1], m4[2]), m4[3]);
          mbar_arrive(pair_bar);
          if (!(ok = spin_wait(pair_bar, pair_turn & 1, a.status, kWaitPair))) break;
          pair_turn ^= 1;
          const float mx = fmaxf(sm.exchange[half][0][r], sm.exchange[half][1][r]) * a.scale_log2;
          float alpha = 1.f;
          if (mx > m + 8.f) {
            alpha = ex2_approx(m - mx);  // (0 from -inf)
            m = mx;
          }
          if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {  // (rare, and the scores hold the registers)
              uint32_t ov[16];
              tmem_ld_32x32b_x16(o_col + c * 16, ov);
              tmem_ld_wait();
#pragma unroll
              for (int j = 0; j < 16; ++j) ov[j] = __float_as_uint(__uint_as_float(ov[j]) * alpha);
              tmem_st_32x32b_x16(o_col + c * 16, ov);
            }
          }
          const float zero = m == -INFINITY ? 0.f : -m;
          const F2 scale = pair(a.scale_log2, a.scale_log2), shift = pair(zero, zero);
          F2 sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
#pragma unroll
          for (int c = 1; c >= 0; --c) {
            if (c == 0) {
              tmem_ld_wait();
              hide(0);
            }
            uint32_t packed[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const F2 e = fma2(pair(__uint_as_float(sv[2 * j]), __uint_as_float(sv[2 * j + 1])), scale, shift);
              const F2 w = pair(ex2_approx(e.f.x), ex2_approx(e.f.y));
              sums[j & 1] = add2(sums[j & 1], w);
              packed[j] = pack2<T>(w.f.x, w.f.y);
            }
            if (c == 1) tmem_ld_32x32b_x32(s_col, sv);  // on its way while these weights leave
            tmem_st_32x32b_x16(s_col + c * 32, packed);   // over these scores alone
          }
          const F2 sum = add2(sums[0], sums[1]);
          l = l * alpha + (sum.f.x + sum.f.y);
          tmem_st_wait();
          tc_fence_before();
          mbar_arrive(&sm.p_full[half]);
        }
        if (!ok || !(ok = warp_wait(&sm.o_full[half], o_turn & 1, a.status, kWaitSums))) break;
        o_turn ^= 1;
        tc_fence_after();
        sm.exchange[half][part][r] = l;
        mbar_arrive(pair_bar);
        if (!(ok = spin_wait(pair_bar, pair_turn & 1, a.status, kWaitPair))) break;
        pair_turn ^= 1;
        l = sm.exchange[half][0][r] + sm.exchange[half][1][r];
        const int64_t unit0 = sm.line.end - left - unit;  // the tile's place in the line
        const int first = static_cast<int>(unit0 / sm.line.share), last = static_cast<int>((unit0 + p.units - 1) / sm.line.share);
        const float inv = l == 0.f ? 0.f : 1.f / l;
        const int64_t slot = a.slot(blockIdx.x, first);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          uint32_t ov[32];
          tmem_ld_32x32b_x32(o_col + c * 32, ov);
          tmem_ld_wait();
          if (first == last) {  // staged where the queries were, so that whole lines leave
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              auto o = [&](int x) { return __uint_as_float(ov[8 * j + x]) * inv; };
              *reinterpret_cast<uint4*>(staged + swz(r, c * 4 + j)) =
                  make_uint4(pack2<T>(o(0), o(1)), pack2<T>(o(2), o(3)), pack2<T>(o(4), o(5)), pack2<T>(o(6), o(7)));
            }
          } else if (there) {  // 16 bytes of each row side by side
#pragma unroll
            for (int j = 0; j < 8; ++j)
              *reinterpret_cast<uint4*>(a.parts + slot * kHeadDim + ((part * 16 + c * 8 + j) * kRowsTile + row) * 4) =
                  make_uint4(ov[4 * j], ov[4 * j + 1], ov[4 * j + 2], ov[4 * j + 3]);
          }
        }
        if (first == last) {
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 8; ++x) {
            const int dst = __shfl_sync(0xffffffffu, mine, x * 4 + sub);
            const uint4 o = *reinterpret_cast<const uint4*>(staged + swz(quarter * 32 + x * 4 + sub, chunk));
            if (dst >= 0) *reinterpret_cast<uint4*>(out + static_cast<int64_t>(dst) * 64 + chunk * 8) = o;
          }
          __syncwarp();
        }
        if (there && part == 0 && first != last) a.part_stats[slot + row] = make_float2(m, l);
        if (tid == kSplitThread && first != last && first == static_cast<int>(blockIdx.x))
          a.splits[first] = {last, p.rows, p.s.start, at.tile * a.tile_rows, at.head * a.group};
      }
      left -= p.count;
      unit = 0;
      if (left > 0) p.next(a, at);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) {
    __syncwarp();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace

void launch_attend_rows(const AttendArgs& a, const CUtensorMap& key_map, const CUtensorMap& value_map, const at::Tensor& q,
                        at::Tensor& out, int blocks) {
  auto launch = [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    constexpr int smem = (2 + kSlots) * kSlotBytes + sizeof(Shared);
    static_assert(smem <= 227 * 1024, "fits an SM");
    TDSV_CUDA_CHECK(cudaFuncSetAttribute(attend_rows_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    attend_rows_kernel<T><<<blocks, kThreads, smem, stream()>>>(key_map, value_map, static_cast<const T*>(q.data_ptr()),
                                                                static_cast<T*>(out.data_ptr()), a);
  };
  if (q.scalar_type() == at::kHalf) launch(static_cast<__half*>(nullptr));
  else launch(static_cast<__nv_bfloat16*>(nullptr));
  TDSV_LAUNCH_CHECK();
}

}  // namespace tdsv
