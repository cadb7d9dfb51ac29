// Attention with a sliding window and first tokens that stay visible, head_dim 128, bf16 in, fp32
// accumulate, grouped key heads. Query i of the call sits at key position p_i = q_start + i and sees key j when
//   j < s_kv  and  (j < sinks  or  p_i - left <= j <= p_i + right)     (causal: and j <= p_i)
//   o_i = sum_j softmax_j(scale q_i . k_j) v_j over those keys; a query that sees none gets zeros.
//
// One pass over the visible keys with a running row maximum and sum, as the full attention kernel:
// tcgen05 S = Q K^T (SS form) and O += P V (TS form) on 128 x 128 tiles, one softmax thread per query
// row, O rescaled only when a row maximum grew by more than 2^8, P rounded to bf16 for the second product
// (the tensor cores' operand type: 2^-8 of a weight at most, averaged over a row's keys; the row sum keeps the
// fp32 weights). Against 64 bits that is 2.3e-3 of the output; token_kernel, whose weights stay in fp32, is off by
// 1.7e-3, the output's own rounding: a single token's error follows the kernel that its call takes.
//
// Tiles: the G = n_heads / n_kv_heads query heads that share a key head are packed into the rows of a Q
// tile (row r = position r / G, head r % G), so a key tile is read once for all of them and a few query
// rows fill as much of the tile as they can. A CTA walks the union of its rows' keys: the first-token run
// [0, sinks) in 128-key tiles, then the window run from its exact first key (TMA rows need no alignment), or
// one run from key 0 where the two touch. Only tiles on a boundary are masked, by per-row bit words.
// Keys that no row of the CTA sees are never loaded, or (behind the end of a run, inside its last
// tile) have their V rows zeroed in shared memory before the product, so whatever a cache
// holds there cannot reach a result through 0 * NaN.
//
// kTiles = 2: 256 packed rows a work item, 12 warps, 5-stage K/V ring, one CTA per SM (the full kernel's schedule). CTAs
// are persistent: the ring runs on across items, the next item's Q loads once the last Q K^T of this one has retired, and
// its first S is issued behind the last P V. An item costs 4.5 us beside its tiles so (the chain of its first tile, the
// last P V, the write-back of O); with a CTA per item a start and an end cost 10 us of a 28 us item (37 heads x 8192,
// window 511 + 512: 227 us, 206 so). kTiles = 1:
// 128 packed rows, 8 warps, 2-stage ring, two CTAs per SM, a CTA per item. Few rows split the tile list over several
// items; each writes (O, m, l) in fp32 to the caller's workspace and join_kernel combines them in a fixed order. A
// single token has a kernel of its own (token_kernel).
//
// Bound: the exponentials and the chain S -> P -> O of a tile, as in the full kernel, at 1.97 us per 256 x 128 tile (the full
// kernel: 1.88 on the same items), 0.09 us more where it is masked, and the 4.5 us an item. 42000 queries x 14 heads,
// window 2048 + 2048, 512 first tokens: 1.34-1.40 ms under the power cap = 0.97-1.0 PFLOP/s of visible pairs, which are 95 %
// of the tiles'; tensor and exponential pipes are 57 % busy on such a walk. 28 heads x 4096, window 511 + 512: 96-103 us,
// pipes 43 % busy: 448 items for 148 CTAs leave one with 36 tiles in four items (71 + 18 us) where the mean is 30. 5 tokens x
// 56 heads over 168000 keys of 8 heads: 113-130 us = 5.3-6.1 TB/s.
#include <algorithm>
#include <cmath>

#include "h3_attn_tile.cuh"

namespace h3 {
namespace window {

using namespace h3::attn;

struct Params {
  int n_heads, group, s_q, s_kv;
  int left, right, sinks, causal, q_start;  // sinks <= s_kv; causal: right = 0
  int tile_pos;                             // query positions per Q tile: 128 / group
  // blocks of queries in the order of launch: those in the middle of the sequence, head by head, then the ones at its
  // ends, whose walks are shorter, from the longest down
  int blocks, first_mid, n_mid, kv_heads, heads_turn;
  int splits, n_items, rounds;  // work items: (block, part); rounds of the grid over them
  float scale_log2;
  __nv_bfloat16* o;
  long long o_rank_rows, o_rank_stride, o_head_stride, o_row_stride;
  float* part_o;  // splits > 1: [split][head][s_q][128], unnormalised; else nullptr
  float* part_ml; // [split][head][s_q][2]: row maximum (log2 units), row sum
  int* status;
};

// The plan of a call (walks, masks, the deal of work items) is written for host and device: h3_window_plan_kat shows it
// to tests without a GPU.
//
// Key tiles of one CTA: a_tiles tiles of the first-token run, then the run that begins at b_start.
struct Walk {
  int a_tiles, a_end, b_start, b_end, n;
  __host__ __device__ __forceinline__ int base(int j) const { return j < a_tiles ? j * kBlockN : b_start + (j - a_tiles) * kBlockN; }
  __host__ __device__ __forceinline__ int end(int j) const { return j < a_tiles ? a_end : b_end; }
};

__host__ __device__ __forceinline__ Walk make_walk(const Params& p, int p_first, int p_last) {
  Walk w;
  const int lo = max(0, p_first - p.left), hi = min(p.s_kv - 1, p_last + p.right);
  const int ns = p.causal ? max(0, min(p.sinks, p_last + 1)) : p.sinks;
  const bool window = lo <= hi;
  const bool joined = window && lo <= ns;
  w.a_tiles = joined ? 0 : (ns + kBlockN - 1) / kBlockN;
  w.a_end = ns;
  w.b_start = joined ? 0 : lo;
  w.b_end = joined ? max(hi + 1, ns) : hi + 1;
  w.n = w.a_tiles + (window ? (w.b_end - w.b_start + kBlockN - 1) / kBlockN : 0);
  return w;
}

// Block of queries and key head of CTA w. The ends: before the middle block first_mid - 1, first_mid - 2, ... and behind
// it first_mid + n_mid, ... in turn, with the head running fastest (heads_turn) or, where that would spread the K and V in
// use beyond the L2, slowest.
__host__ __device__ __forceinline__ void block_of(const Params& p, int w, int& block, int& kvh) {
  const int mid = p.n_mid * p.kv_heads;
  if (w < mid) {
    kvh = w / p.n_mid;
    block = p.first_mid + (w - kvh * p.n_mid);
    return;
  }
  const int ends = p.blocks - p.n_mid, u = w - mid;
  kvh = p.heads_turn ? u % p.kv_heads : u / ends;
  const int k = p.heads_turn ? u / p.kv_heads : u - kvh * ends;
  const int before = p.first_mid, behind = ends - before, both = 2 * min(before, behind);
  const int i = k < both ? k >> 1 : k - (both >> 1);
  const bool front = k < both ? (k & 1) == 0 : before > behind;
  block = front ? before - 1 - i : p.first_mid + p.n_mid + i;
}

// One work item: a block of queries of one key head, and part z of its key tiles, [j_lo, j_lo + n_kv) of the walk.
struct Item {
  int kvh, i0, z;
  int j_lo, n_kv;
};
// Work item of CTA `cta` of `ctas` in round r, or -1. Rounds alternate in direction: items come
// longest first but for the two ends' taking turns, so that a CTA's long and short ones even out.
template <int kTiles>
__host__ __device__ __forceinline__ int rounds_of(const Params& p) {
  return kTiles == 1 ? 1 : p.rounds;  // one Q tile: a CTA per item
}
template <int kTiles>
__host__ __device__ __forceinline__ int item_of(const Params& p, int r, int cta, int ctas) {
  if (kTiles == 1) return cta;
  const int c = (r & 1) ? ctas - 1 - cta : cta;
  const int w = r * ctas + c;
  return w < p.n_items ? w : -1;
}
template <int kTiles>
__host__ __device__ __forceinline__ Item make_item(const Params& p, int w, Walk& walk) {
  Item it;
  int block;
  it.z = w % p.splits;
  block_of(p, w / p.splits, block, it.kvh);
  it.i0 = block * kTiles * p.tile_pos;
  walk = make_walk(p, p.q_start + it.i0, p.q_start + min(it.i0 + kTiles * p.tile_pos, p.s_q) - 1);
  it.j_lo = int((long long)walk.n * it.z / p.splits);
  it.n_kv = int((long long)walk.n * (it.z + 1) / p.splits) - it.j_lo;
  return it;
}
// The CTA's next work item with key tiles, from round r on; r becomes its round, or the number of rounds.
template <int kTiles>
__device__ __forceinline__ Item next_item(const Params& p, int& r, Walk& walk) {
  Item it = {};
  for (; r < rounds_of<kTiles>(p); ++r) {
    const int w = item_of<kTiles>(p, r, int(blockIdx.x), int(gridDim.x));
    if (w < 0) continue;
    it = make_item<kTiles>(p, w, walk);
    if (it.n_kv > 0) break;
  }
  return it;
}

// Bits e of a 32-key word whose keys lie in [a, b] or below n (all relative to the word's first key).
__host__ __device__ __forceinline__ uint32_t visible_bits(int a, int b, int n) {
  const uint32_t ge = a <= 0 ? 0xffffffffu : (a > 31 ? 0u : 0xffffffffu << a);
  const uint32_t le = b < 0 ? 0u : (b >= 31 ? 0xffffffffu : (2u << b) - 1u);
  const uint32_t lt = n <= 0 ? 0u : (n > 31 ? 0xffffffffu : (1u << n) - 1u);
  return (ge & le) | lt;
}

// Keys of [lo, hi] and keys below ns: what the row at position pos sees, or (sees_all) what every row of [first, last] sees.
struct Seen {
  int lo, hi, ns;
};
__host__ __device__ __forceinline__ Seen sees(const Params& p, int pos) {
  return {pos - p.left, min(pos + p.right, p.s_kv - 1), p.causal ? min(p.sinks, pos + 1) : p.sinks};
}
__host__ __device__ __forceinline__ Seen sees_all(const Params& p, int first, int last) {
  return {last - p.left, min(first + p.right, p.s_kv - 1), p.causal ? min(p.sinks, first + 1) : p.sinks};
}
// Whether a key tile of the walk hides a key from some row. A separate first-token run has no window in it.
__host__ __device__ __forceinline__ bool is_masked(const Seen& all, int key, bool first_run) {
  return !(key + kBlockN <= all.ns || (!first_run && key >= all.lo && key + kBlockN - 1 <= all.hi));
}
// The row's window counted from the tile's first key: arguments of visible_bits for its first word.
__host__ __device__ __forceinline__ Seen in_tile(const Seen& row, int key, bool first_run) {
  return {first_run ? 1 << 20 : row.lo - key, row.hi - key, row.ns - key};
}

template <int kTiles>
struct Cfg {
  static constexpr int kThreads = 128 + 128 * kTiles;
  static constexpr int kStages = kTiles == 2 ? 5 : 2;
  // Ring stages come back through kRel release barriers used round robin: release r completes once the
  // last tile's S(r) is ready, i.e. once every MMA reading K_r and V_(r-1) has retired. The producer trails a
  // barrier by less than one phase while 2 * kRel > kStages - 1.
  static constexpr int kRel = kStages;
  static constexpr int kBarQ = 0, kBarKV = 1, kBarRel = kBarKV + kStages, kBarS = kBarRel + kRel,
                       kBarPSplit = kBarS + kTiles, kBarPLast = kBarPSplit + kTiles, kBarO = kBarPLast + kTiles,
                       kBarDrain = kBarO + kTiles, kBarQFree = kBarDrain + 1, kNumBars = kBarQFree + 1;
  static constexpr uint32_t kOffKV = kTiles * kTileBytes;
  static constexpr uint32_t kOffBars = kOffKV + kStages * kTileBytes;
  static constexpr uint32_t kSmem = 1024 + kOffBars + kNumBars * 8 + 16;
  static constexpr int kCtasPerSm = kTiles == 2 ? 1 : 2;
  static constexpr uint32_t kCols = kTiles * 256;  // S_t [128 t, +128), O_t [128 (kTiles + t), +128)
  // registers: the control warpgroup gives back what the softmax warpgroups (a 128-score row a thread) take
  static constexpr int kRegsLaunch = kTiles == 2 ? 168 : 128;
  static constexpr int kRegsControl = kTiles == 2 ? 72 : 40;
  static constexpr int kRegsSoftmax = 216;
  static_assert(128 * kRegsControl + 128 * kTiles * kRegsSoftmax <= kThreads * kRegsLaunch, "register split over budget");
};

constexpr int kSplitChunks = 3;  // P is handed over after 3 of its 4 32-key chunks, then the rest

template <int kTiles>
__global__ void __launch_bounds__(Cfg<kTiles>::kThreads, Cfg<kTiles>::kCtasPerSm)
    window_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                  const __grid_constant__ CUtensorMap tmap_v, const Params p) {
  using C = Cfg<kTiles>;
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(bar(C::kBarQ), 1);
    for (int s = 0; s < C::kStages; ++s) mbar_init(bar(C::kBarKV + s), 1);
    for (int r = 0; r < C::kRel; ++r) mbar_init(bar(C::kBarRel + r), 1);
    for (int t = 0; t < kTiles; ++t) {
      mbar_init(bar(C::kBarS + t), 1);
      mbar_init(bar(C::kBarPSplit + t), 128);
      mbar_init(bar(C::kBarPLast + t), 128);
      mbar_init(bar(C::kBarO + t), 1);
    }
    mbar_init(bar(C::kBarDrain), 1);
    mbar_init(bar(C::kBarQFree), 1);
    *abort_flag = (*reinterpret_cast<volatile int*>(p.status) != 0) ? 1 : 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == 2) {
    tmem_alloc(smem_u32(tmem_slot), C::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const WaitCtx ctx{abort_flag, p.status};
  const bool run = *abort_flag == 0;  // uniform over the CTA
  if (warp < 4) {
    regs_dec<C::kRegsControl>();
    const uint32_t sq = sbase, skv = sbase + C::kOffKV;
    if (warp == 0 && run) {
      // ------------------------------------------------------------ TMA producer: Q, then K_0, V_0, K_1, V_1, ...
      const bool issuer = elect_one();
      int it = 0, q_loads = 0;  // ring items, work items so far
      bool ok = true;
      Walk walk;
      int r = 0;
      for (Item item = next_item<kTiles>(p, r, walk); ok && r < rounds_of<kTiles>(p);
           ++r, item = next_item<kTiles>(p, r, walk)) {
        // Q is free once the last S of the item before is ready
        if (q_loads > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(bar(C::kBarQFree), uint32_t(q_loads - 1) & 1u, ctx,
                                                                    kStatusTimeoutQ))))
          break;
        if (issuer) {
          const uint32_t box = 64u * 2u * uint32_t(p.group * p.tile_pos);  // rows past group * tile_pos stay unused
          mbar_expect_tx(bar(C::kBarQ), kTiles * 2 * box);
          for (int t = 0; t < kTiles; ++t)
            for (int hh = 0; hh < 2; ++hh)
              tma_load_4d(sq + t * kTileBytes + hh * kHalfBytes, &tmap_q, bar(C::kBarQ), hh * 64, 0,
                          item.i0 + t * p.tile_pos, item.kvh);
        }
        __syncwarp();
        ++q_loads;
        for (int j = 0; ok && j < item.n_kv; ++j) {
          const int key = walk.base(item.j_lo + j);
          for (int kv = 0; kv < 2; ++kv, ++it) {
            const int st = it % C::kStages;
            if (it >= C::kStages) {
              // the stage's previous item (it - kStages) is free once release e has completed: K_r (item 2r) after
              // S(r), V_r (item 2r + 1) after S(r + 1); tiles are counted on across work items
              const int e = (it - C::kStages + 1) / 2;
              if (!__all_sync(0xffffffffu, mbar_wait(bar(C::kBarRel + e % C::kRel), uint32_t(e / C::kRel) & 1u, ctx,
                                                     kStatusTimeoutKV))) {
                ok = false;
                break;
              }
            }
            if (issuer) {
              const CUtensorMap* m = kv ? &tmap_v : &tmap_k;
              const uint32_t dst = skv + st * kTileBytes;
              mbar_expect_tx(bar(C::kBarKV + st), kTileBytes);
              tma_load_3d(dst, m, bar(C::kBarKV + st), 0, key, item.kvh);
              tma_load_3d(dst + kHalfBytes, m, bar(C::kBarKV + st), 64, key, item.kvh);
            }
            __syncwarp();
          }
        }
      }
      // every issued copy must land before the CTA may exit
      if (issuer) {
        if (q_loads > 0) drain_wait(bar(C::kBarQ), uint32_t(q_loads - 1) & 1u, p.status);
        for (int st = 0; st < C::kStages; ++st) {
          const int cnt = it / C::kStages + (st < it % C::kStages ? 1 : 0);
          if (cnt > 0) drain_wait(bar(C::kBarKV + st), uint32_t(cnt - 1) & 1u, p.status);
        }
      }
      __syncwarp();
    } else if (warp == 1 && run) {
      // ------------------------------------------------------------ MMA issuer (the whole warp loops, one lane issues)
      const bool issuer = elect_one();
      auto wait_all = [&](uint32_t b, uint32_t par, int code) -> bool {
        return __all_sync(0xffffffffu, mbar_wait(b, par, ctx, code));
      };
      auto wait_full = [&](int it) -> bool {
        return wait_all(bar(C::kBarKV + it % C::kStages), uint32_t(it / C::kStages) & 1u, kStatusTimeoutKV);
      };
      auto commit = [&](int b) {
        if (issuer) mma_commit(bar(b));
        __syncwarp();
      };
      auto col_o = [&](int t) { return tmem + 128u * uint32_t(kTiles + t); };
      auto col_p = [&](int t) { return tmem + 128u * uint32_t(t) + 64u; };
      Walk walk, walk_next;
      int r = 0, items = 0, jg = 0;  // round; work items and key tiles so far
      Item item = next_item<kTiles>(p, r, walk);
      bool ok = r < rounds_of<kTiles>(p);
      if (ok && (ok = wait_all(bar(C::kBarQ), 0, kStatusTimeoutQ) && wait_full(0))) {
        tc_fence_after();
        for (int t = 0; t < kTiles; ++t) {
          if (issuer) issue_qk(tmem + 128u * t, sq + t * kTileBytes, skv);
          __syncwarp();
          commit(C::kBarS + t);
        }
      }
      while (ok) {
        int r_next = r + 1;
        const Item following = next_item<kTiles>(p, r_next, walk_next);
        for (int j = 0; ok && j < item.n_kv; ++j, ++jg) {
          const int it_v = 2 * jg + 1, it_k = 2 * jg + 2;
          const bool last = j + 1 == item.n_kv;
          const bool next = !last || r_next < rounds_of<kTiles>(p);
          if (!(ok = wait_full(it_v))) break;
          const uint32_t sv = skv + (it_v % C::kStages) * kTileBytes;
          const uint32_t sk = skv + (it_k % C::kStages) * kTileBytes;
          const uint32_t ph = uint32_t(jg) & 1u;
          {
            // keys behind the end of the run, inside its last tile: no row sees them, their V rows become zero
            // (rows past s_kv already are: the TMA fill). The 128-byte swizzle permutes within a row only.
            const int key = walk.base(item.j_lo + j);
            const int from = walk.end(item.j_lo + j) - key, to = min(kBlockN, p.s_kv - key);
            if (from < to) {
              for (int c = 8 * from + lane; c < 8 * to; c += 32) {
                st_shared_u4(sv + 16u * uint32_t(c), make_uint4(0, 0, 0, 0));
                st_shared_u4(sv + kHalfBytes + 16u * uint32_t(c), make_uint4(0, 0, 0, 0));
              }
              fence_proxy_async();
              __syncwarp();
            }
          }
          for (int t = 0; t < kTiles; ++t) {
            if (!(ok = wait_all(bar(C::kBarPSplit + t), ph, kStatusTimeoutP))) break;
            tc_fence_after();
            if (issuer) issue_pv_steps<0, 2 * kSplitChunks>(col_o(t), col_p(t), sv, j > 0);
            __syncwarp();
            if (!(ok = wait_all(bar(C::kBarPLast + t), ph, kStatusTimeoutP))) break;
            tc_fence_after();
            if (issuer) issue_pv_steps<2 * kSplitChunks, 8 - 2 * kSplitChunks>(col_o(t), col_p(t), sv, true);
            __syncwarp();
            if (last) commit(C::kBarO + t);
            if (next) {
              if (t == 0 && last && !(ok = wait_all(bar(C::kBarQ), uint32_t(items + 1) & 1u, kStatusTimeoutQ))) break;
              if (t == 0 && !(ok = wait_full(it_k))) break;
              if (issuer) issue_qk(tmem + 128u * t, sq + t * kTileBytes, sk);
              __syncwarp();
              commit(C::kBarS + t);
            }
          }
        }
        if (r_next >= rounds_of<kTiles>(p)) break;
        r = r_next;
        item = following;
        walk = walk_next;
        ++items;
      }
      // every issued MMA must retire before TMEM is released
      if (issuer) {
        mma_commit(bar(C::kBarDrain));
        drain_wait(bar(C::kBarDrain), 0, p.status);
      }
      __syncwarp();
    }
  } else {
    regs_inc<C::kRegsSoftmax>();
    // ------------------------------------------------------------ softmax + epilogue
    const int t = (warp - 4) >> 2;
    const int quad = warp & 3;
    const uint32_t lane_off = uint32_t(quad * 32) << 16;
    const uint32_t tS = tmem + lane_off + 128u * uint32_t(t);
    const uint32_t tP = tS + 64u;
    const uint32_t tO = tmem + lane_off + 128u * uint32_t(kTiles + t);
    const float c = p.scale_log2;
    const uint64_t c2 = f2_pack(c, c);
    const int r_in = quad * 32 + lane;
    const int row_pos = r_in / p.group;              // packed row -> query position in the tile, head in the group
    const int row_head = r_in - row_pos * p.group;
    bool ok = run;
    int jg = 0, items = 0;
    for (int r = 0; ok && r < rounds_of<kTiles>(p); ++r) {
      const int w = item_of<kTiles>(p, r, int(blockIdx.x), int(gridDim.x));
      if (w < 0) continue;
      Walk walk;
      const Item item = make_item<kTiles>(p, w, walk);
      const int it0 = item.i0 + t * p.tile_pos;        // the tile's first query
      const int pos = p.q_start + it0 + row_pos;       // this row's key position
      const Seen row = sees(p, pos), all = sees_all(p, p.q_start + it0, p.q_start + it0 + p.tile_pos - 1);
      float m_run = -INFINITY;
      uint64_t l_a = f2_pack(0.f, 0.f), l_b = f2_pack(0.f, 0.f);

      for (int j = 0; ok && j < item.n_kv; ++j, ++jg) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar(C::kBarS + t), uint32_t(jg) & 1u, ctx, kStatusTimeoutS));
        if (!ok) break;
        if (t == kTiles - 1 && quad == 0) {
          if (lane == 0) {
            mbar_arrive(bar(C::kBarRel + jg % C::kRel));
            if (j + 1 == item.n_kv) mbar_arrive(bar(C::kBarQFree));  // every S of this item is done: Q may be replaced
          }
          __syncwarp();
        }
        tc_fence_after();
        const int key = walk.base(item.j_lo + j);
        const bool first_run = item.j_lo + j < walk.a_tiles;
        const bool masked = is_masked(all, key, first_run);
        uint32_t sa[64], sb[64];
        tmem_ld64_wait(tS, sa);
        tmem_ld64_nowait(tS + 64, sb);
        float s[128];
#pragma unroll
        for (int i = 0; i < 64; ++i) s[i] = __uint_as_float(sa[i]);
        const Seen at = in_tile(row, key, first_run);
        if (masked) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const uint32_t bits = visible_bits(at.lo - 32 * w, at.hi - 32 * w, at.ns - 32 * w);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((bits >> i) & 1u)) s[32 * w + i] = -INFINITY;
          }
        }
        float mx0 = fmax3(s[0], s[1], s[2]), mx1 = fmax3(s[3], s[4], s[5]);
        float mx2 = fmax3(s[6], s[7], s[8]), mx3 = fmax3(s[9], s[10], s[11]);
#pragma unroll
        for (int i = 12; i < 60; i += 8) {
          mx0 = fmax3(mx0, s[i], s[i + 1]);
          mx1 = fmax3(mx1, s[i + 2], s[i + 3]);
          mx2 = fmax3(mx2, s[i + 4], s[i + 5]);
          mx3 = fmax3(mx3, s[i + 6], s[i + 7]);
        }
        mx0 = fmax3(mx0, s[60], s[61]);
        mx1 = fmax3(mx1, s[62], s[63]);
        tmem_ld64_wait_on(sb);
#pragma unroll
        for (int i = 0; i < 64; ++i) s[64 + i] = __uint_as_float(sb[i]);
        if (masked) {
#pragma unroll
          for (int w = 2; w < 4; ++w) {
            const uint32_t bits = visible_bits(at.lo - 32 * w, at.hi - 32 * w, at.ns - 32 * w);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((bits >> i) & 1u)) s[32 * w + i] = -INFINITY;
          }
        }
#pragma unroll
        for (int i = 64; i < 120; i += 8) {
          mx0 = fmax3(mx0, s[i], s[i + 1]);
          mx1 = fmax3(mx1, s[i + 2], s[i + 3]);
          mx2 = fmax3(mx2, s[i + 4], s[i + 5]);
          mx3 = fmax3(mx3, s[i + 6], s[i + 7]);
        }
        mx0 = fmax3(mx0, s[120], s[121]);
        mx1 = fmax3(mx1, s[122], s[123]);
        mx2 = fmax3(mx2, s[124], s[125]);
        mx3 = fmax3(mx3, s[126], s[127]);
        const float m_new = fmaxf(m_run, fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3)) * c);
        if (j == 0) {
          m_run = m_new;
        } else {
          // rows whose running maximum grew by more than 2^8 (or from nothing) rescale O and l; O_t is quiescent
          // here: S_t(j) ready implies every earlier P_t V has retired
          const bool need = m_new > m_run + kRescaleThreshold;
          if (__any_sync(0xffffffffu, need)) {
            const float f = need ? ex2_approx(m_run - m_new) : 1.0f;
            if (need) {
              l_a = f2_fma(l_a, f2_pack(f, f), f2_pack(0.f, 0.f));
              l_b = f2_fma(l_b, f2_pack(f, f), f2_pack(0.f, 0.f));
              m_run = m_new;
            }
            __syncwarp();
#pragma unroll 1
            for (int c16 = 0; c16 < 8; ++c16) {
              uint32_t o[16];
              tmem_ld16_wait(tO + c16 * 16, o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
              tmem_st16(tO + c16 * 16, o);
            }
            tmem_st_wait();
          }
        }
        // exponentials in four 32-key chunks, each stored as bf16 P as soon as it is done. A row that has seen no
        // key yet keeps m_run = -inf: its weights are exp2(-inf - 0) = 0.
        const float m_use = m_run == -INFINITY ? 0.f : m_run;
        const uint64_t nm2 = f2_pack(-m_use, -m_use);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t pk[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int e = 32 * k + 2 * i;
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(s[e], s[e + 1]), c2, nm2), x0, x1);
            s[e] = ex2_approx(x0);
            s[e + 1] = ex2_approx(x1);
            pk[i] = pack_bf16x2(s[e], s[e + 1]);
          }
          tmem_st16(tP + 16 * k, pk);
          if (k == kSplitChunks - 1) {
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(bar(C::kBarPSplit + t));
          }
        }
        tmem_st_wait();
        tc_fence_before();
        mbar_arrive(bar(C::kBarPLast + t));
#pragma unroll
        for (int i = 0; i < 128; i += 4) {
          l_a = f2_add(l_a, f2_pack(s[i], s[i + 1]));
          l_b = f2_add(l_b, f2_pack(s[i + 2], s[i + 3]));
        }
      }
      float la0, la1, lb0, lb1;
      f2_unpack(l_a, la0, la1);
      f2_unpack(l_b, lb0, lb1);
      const float l_run = (la0 + la1) + (lb0 + lb1);
      if (ok && item.n_kv > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(bar(C::kBarO + t), uint32_t(items) & 1u, ctx, kStatusTimeoutO));
        ++items;
      }
      // an item without keys writes its zeros too; an aborted one writes nothing
      if (ok) {
        tc_fence_after();
        const int i = it0 + row_pos;
        const int head = item.kvh * p.group + row_head;
        const bool valid = row_pos < p.tile_pos && i < p.s_q;
        const bool none = item.n_kv == 0 || l_run == 0.f;
        const float inv = 1.0f / l_run;
        const long long ri = valid ? i : 0;
        __nv_bfloat16* dst = p.o + (ri / p.o_rank_rows) * p.o_rank_stride + (long long)head * p.o_head_stride +
                             (ri % p.o_rank_rows) * p.o_row_stride;
        const long long part = ((long long)item.z * p.n_heads + head) * p.s_q + ri;
#pragma unroll
        for (int c4 = 0; c4 < 4; ++c4) {
          uint32_t o[32];
          tmem_ld32_wait(tO + c4 * 32, o);
          if (valid && p.part_o != nullptr) {
            float4* d = reinterpret_cast<float4*>(p.part_o + part * 128 + c4 * 32);
#pragma unroll
            for (int e = 0; e < 8; ++e)
              d[e] = none ? make_float4(0.f, 0.f, 0.f, 0.f)
                          : make_float4(__uint_as_float(o[4 * e]), __uint_as_float(o[4 * e + 1]),
                                        __uint_as_float(o[4 * e + 2]), __uint_as_float(o[4 * e + 3]));
          } else if (valid) {
            uint32_t w[16];
#pragma unroll
            for (int e = 0; e < 16; ++e)
              w[e] = none ? 0u : pack_bf16x2(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
            uint4* d = reinterpret_cast<uint4*>(dst + c4 * 32);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
          }
          __syncwarp();  // the next load of O takes the whole warp
        }
        if (valid && p.part_ml != nullptr)
          reinterpret_cast<float2*>(p.part_ml)[part] = make_float2(m_run, none ? 0.f : l_run);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kCols);
  }
}

// One CTA per output row: its warps take the splits' (O, m, l) in turn, all loads in flight at once; the sums are
// joined in a fixed order, normalised and rounded once.
constexpr int kJoinWarps = 8;

__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const Params p, int splits) {
  __shared__ float4 sh_o[kJoinWarps][32];
  __shared__ float sh_l[kJoinWarps];
  pdl_wait();
  if (*reinterpret_cast<volatile int*>(p.status) != 0) return;
  const long long row = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long rows = (long long)p.n_heads * p.s_q;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml);
  float m = -INFINITY;
  for (int s = lane; s < splits; s += 32) m = fmaxf(m, ml[s * rows + row].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float m_use = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = warp; s < splits; s += kJoinWarps) {
    const float2 v = ml[s * rows + row];
    const float4 o = reinterpret_cast<const float4*>(p.part_o + (s * rows + row) * 128)[lane];
    const float f = ex2_approx(v.x - m_use);
    l += f * v.y;
    acc.x += f * o.x;
    acc.y += f * o.y;
    acc.z += f * o.z;
    acc.w += f * o.w;
  }
  sh_o[warp][lane] = acc;
  if (lane == 0) sh_l[warp] = l;
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWarps; ++w) {
    const float4 o = sh_o[w][lane];
    l += sh_l[w];
    acc.x += o.x;
    acc.y += o.y;
    acc.z += o.z;
    acc.w += o.w;
  }
  const float inv = l == 0.f ? 0.f : 1.0f / l;
  const long long i = row % p.s_q, head = row / p.s_q;
  __nv_bfloat16* dst = p.o + (i / p.o_rank_rows) * p.o_rank_stride + head * p.o_head_stride +
                       (i % p.o_rank_rows) * p.o_row_stride;
  reinterpret_cast<uint2*>(dst)[lane] =
      make_uint2(pack_bf16x2(acc.x * inv, acc.y * inv), pack_bf16x2(acc.z * inv, acc.w * inv));
}

// ---------------------------------------------------------------- single tokens
// One query position and kGroup query heads to a key head (at most 4): every key of the walk is visible to every row,
// so there is nothing to mask, and a 128-row tile would be all padding. A cluster of CTAs takes the keys of one
// key head, one run of them each; a half-warp takes a key (16 bytes of K and of V a lane), kKeys keys at a time in
// flight, with its own running maximum and sums; half-warps join through shared memory, CTAs through distributed
// shared memory. One launch, no workspace, and bound by the latency of the loads: a half-warp asks for its next keys when
// the sums of the ones before are done. 56 heads over 1536 of 42000 keys: three such rounds a CTA, 12 us with the keys in
// the L2 and 14 without (44 MB: 3.1 TB/s); 23 % of the issue slots are used, ten warps wait on loads for each that issues.
constexpr int kTokenWarps = 8;
constexpr int kKeys = 4;  // keys in flight per half-warp
constexpr int kTokenMaxCluster = 8;

struct TokenParams {
  const __nv_bfloat16 *q, *k, *v;
  long long q_head, kv_head, kv_row;
};

template <int kGroup>
__global__ void __launch_bounds__(32 * kTokenWarps) token_kernel(const Params p, const TokenParams tp) {
  constexpr int kHalves = 2 * kTokenWarps;
  __shared__ float sh_m[kHalves][kGroup], sh_l[kHalves][kGroup];
  __shared__ float sh_o[kHalves][kGroup][kHeadDim];
  __shared__ float cta_m[kGroup], cta_l[kGroup], cta_o[kGroup][kHeadDim];
  const int lane = threadIdx.x & 31, sub = lane & 15;
  const int half = threadIdx.x >> 4;
  const int rank = int(cluster_ctarank()), ranks = int(gridDim.x);
  const int kvh = blockIdx.y;
  const bool live = *reinterpret_cast<volatile int*>(p.status) == 0;
  const Walk walk = make_walk(p, p.q_start, p.q_start);
  const bool window = walk.n > walk.a_tiles;
  const int n_first = walk.a_tiles > 0 ? walk.a_end : 0;  // keys of the separate first-token run
  const int total = live ? n_first + (window ? walk.b_end - walk.b_start : 0) : 0;
  const int k0 = int((long long)total * rank / ranks), k1 = int((long long)total * (rank + 1) / ranks);
  const __nv_bfloat16* kb = tp.k + kvh * tp.kv_head + 8 * sub;
  const __nv_bfloat16* vb = tp.v + kvh * tp.kv_head + 8 * sub;

  float q[kGroup][8], acc[kGroup][8], m[kGroup], l[kGroup];
#pragma unroll
  for (int g = 0; g < kGroup; ++g) {
    bf16x8_to_f32(*reinterpret_cast<const uint4*>(tp.q + (long long)(kvh * kGroup + g) * tp.q_head + 8 * sub), q[g]);
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      q[g][e] *= p.scale_log2;
      acc[g][e] = 0.f;
    }
  }
  for (int base = k0 + half * kKeys; base < k1; base += kHalves * kKeys) {
    uint4 ku[kKeys], vu[kKeys];
    bool in[kKeys];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      in[i] = base + i < k1;
      const int at = in[i] ? base + i : base;
      const long long key = at < n_first ? at : walk.b_start + (at - n_first);
      ku[i] = __ldg(reinterpret_cast<const uint4*>(kb + key * tp.kv_row));
      vu[i] = __ldg(reinterpret_cast<const uint4*>(vb + key * tp.kv_row));
    }
    float s[kGroup][kKeys];
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      float kf[8];
      bf16x8_to_f32(ku[i], kf);
#pragma unroll
      for (int g = 0; g < kGroup; ++g) {
        float d = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) d += q[g][e] * kf[e];
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) d += __shfl_xor_sync(half & 1 ? 0xffff0000u : 0x0000ffffu, d, o);
        s[g][i] = in[i] ? d : -INFINITY;
      }
    }
#pragma unroll
    for (int g = 0; g < kGroup; ++g) {
      float top = m[g];
#pragma unroll
      for (int i = 0; i < kKeys; ++i) top = fmaxf(top, s[g][i]);
      const float use = top == -INFINITY ? 0.f : top;
      const float f = ex2_approx(m[g] - use);
      m[g] = top;
      l[g] *= f;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[g][e] *= f;
#pragma unroll
      for (int i = 0; i < kKeys; ++i) {
        s[g][i] = ex2_approx(s[g][i] - use);
        l[g] += s[g][i];
      }
    }
#pragma unroll
    for (int i = 0; i < kKeys; ++i) {
      float vf[8];
      bf16x8_to_f32(vu[i], vf);
      if (in[i]) {  // a key past the share is not added, whatever its V holds
#pragma unroll
        for (int g = 0; g < kGroup; ++g)
#pragma unroll
          for (int e = 0; e < 8; ++e) acc[g][e] += s[g][i] * vf[e];
      }
    }
  }
#pragma unroll
  for (int g = 0; g < kGroup; ++g) {
    if (sub == 0) {
      sh_m[half][g] = m[g];
      sh_l[half][g] = l[g];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sh_o[half][g][8 * sub + e] = acc[g][e];
  }
  __syncthreads();
  // the CTA's half-warps, in ascending order
  for (int t = threadIdx.x; t < kGroup * kHeadDim; t += 32 * kTokenWarps) {
    const int g = t / kHeadDim, d = t % kHeadDim;
    float top = -INFINITY;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) top = fmaxf(top, sh_m[h][g]);
    const float use = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o = 0.f;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const float f = ex2_approx(sh_m[h][g] - use);
      sum += f * sh_l[h][g];
      o += f * sh_o[h][g][d];
    }
    cta_o[g][d] = o;
    if (d == 0) {
      cta_m[g] = top;
      cta_l[g] = sum;
    }
  }
  cluster_sync_all();
  // the cluster's CTAs, in ascending order: each finishes its share of the outputs, two neighbouring elements a thread
  const int pairs = kGroup * kHeadDim / 2;
  for (int t = rank * 32 * kTokenWarps + threadIdx.x; live && t < pairs; t += ranks * 32 * kTokenWarps) {
    const int g = 2 * t / kHeadDim, d = 2 * t % kHeadDim;
    float pm[kTokenMaxCluster], top = -INFINITY;
#pragma unroll
    for (int r = 0; r < kTokenMaxCluster; ++r) {
      pm[r] = r < ranks ? ld_cluster_f32(mapa_shared(smem_u32(&cta_m[g]), r)) : -INFINITY;
      top = fmaxf(top, pm[r]);
    }
    const float use = top == -INFINITY ? 0.f : top;
    float sum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
    for (int r = 0; r < kTokenMaxCluster; ++r) {
      if (r < ranks) {
        const float f = ex2_approx(pm[r] - use);
        sum += f * ld_cluster_f32(mapa_shared(smem_u32(&cta_l[g]), r));
        o0 += f * ld_cluster_f32(mapa_shared(smem_u32(&cta_o[g][d]), r));
        o1 += f * ld_cluster_f32(mapa_shared(smem_u32(&cta_o[g][d + 1]), r));
      }
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    *reinterpret_cast<uint32_t*>(p.o + (long long)(kvh * kGroup + g) * p.o_head_stride + d) =
        pack_bf16x2(o0 * inv, o1 * inv);
  }
  cluster_sync_all();  // no CTA leaves while another reads its shared memory
}

// ---------------------------------------------------------------- host
constexpr int64_t kMaxPos = 1ll << 29;  // lengths and |q_start|: positions lie in [-2^29, 2^30)
constexpr int kMaxSplits = 64;

struct Shape {
  int64_t n_heads, n_kv_heads, s_q, s_kv, left, right, sinks, q_start;
  int32_t causal;
};

static int check_shape(const Shape& s) {
  if (s.n_heads < 1 || s.n_kv_heads < 1 || s.n_heads > 65535 || s.n_heads % s.n_kv_heads ||
      s.n_heads / s.n_kv_heads > 128 || s.s_q < 1 || s.s_kv < 1 || s.s_q > kMaxPos || s.s_kv > kMaxPos ||
      s.sinks < 0 || s.q_start < -kMaxPos || s.q_start > kMaxPos)
    return H3_ERR_SHAPE;
  return H3_OK;
}

// The launch shape of a call.
struct Plan {
  int tiles;    // Q tiles per CTA
  int tile_pos; // query positions per Q tile
  int blocks;    // blocks of queries per key head
  int first_mid, n_mid, heads_turn;  // their order (Params)
  int splits, n_items, ctas;
  int token;     // cluster size of token_kernel, or 0: window_kernel
};

// A single token with at most 4 query heads to a key head and few keys, or with a head of its own over a cache with key
// heads enough that clusters of 8 CTAs fill the SMs three times (fewer do not keep enough loads in flight), is token_kernel,
// a CTA for 128 keys up to 8 of them. One query head to a key head, 1000 keys of 8 / 28 / 56 heads: 7.6 / 8.7 / 10.7 us, by
// tiles 10.6 / 11.8 / 14.8; 2000: 11.9 / 13.2 / 16.4 and 10.9 / 14.6 / 21.0; 4000 of 56 heads: 28.4 and 31.1; 8000: 47.2
// and 47.2 (of 8 heads, with keys in the L2: 31 and 15.6). With 2 to 4 the sums of a key cost as many times the
// arithmetic, and at 92-128 registers a thread only two CTAs fit an SM: a second round of clusters costs more than it
// hides. Groups of 2 / 4, 750 keys of 40 heads (240 CTAs): 9.0 / 11.1 us, by tiles 12.0 / 12.1; 1000 keys of 37 heads (296
// CTAs): 15.1 / 18.9 and 12.5 / 12.6; 8000 of 56: 69 / 87 and 47 / 48. Groups of 4 lose to the tiles from some 12 tiles of
// keys on where they fit (20 heads, 1500 keys 13.0 and 12.0; 2000: 15.6 and 13.4; 4 heads: 8.7 / 10.4 and 10.4 / 10.4).
// Else Q tiles of window_kernel: two per CTA (256 packed rows, one CTA an SM) where the rows fill more than one, else
// one (two CTAs an SM); and splits only when the unsplit grid leaves CTA slots empty: then as many as fill them,
// with at least two key tiles each.
static bool by_tokens(int group, int64_t kv_heads, int64_t key_tiles, int sms) {
  if (group == 1) return key_tiles <= 16 || (key_tiles <= 64 && kv_heads * kTokenMaxCluster >= 3 * sms);
  const int64_t ctas = kv_heads * std::min<int64_t>(kTokenMaxCluster, key_tiles);
  return group <= 4 && key_tiles <= 16 && group * key_tiles <= 48 && 4 * ctas <= 7 * sms;
}
static int make_plan(const Shape& s, int64_t splits_asked, int sms, Plan& pl) {
  const int group = (int)(s.n_heads / s.n_kv_heads);
  pl.tile_pos = 128 / group;
  pl.tiles = s.s_q <= pl.tile_pos ? 1 : 2;
  const int64_t per_cta = (int64_t)pl.tiles * pl.tile_pos;
  const int64_t blocks = (s.s_q + per_cta - 1) / per_cta;
  const int64_t ctas = blocks * s.n_kv_heads, slots = (int64_t)sms * (pl.tiles == 1 ? 2 : 1);
  const int64_t left = s.left < 0 || s.left > kMaxPos ? kMaxPos : s.left;
  const int64_t right = s.causal ? 0 : (s.right < 0 || s.right > kMaxPos ? kMaxPos : s.right);
  if (ctas > (1ll << 30)) return H3_ERR_SHAPE;
  // Blocks of the middle (whole windows) first, the shorter ones at the ends last, longest first, so that the CTAs' shares
  // even out (Params, item_of). Heads turn while the keys that all of them look at fit the L2 twice: causal without a left
  // bound, 28 heads x 8192 (117 MB): 525 us head by head, 478 in turn; 7 x 42000 (150 MB): 2749 and 2558; but 56 x 20000
  // (573 MB): 5.63 ms and 6.14.
  const int64_t p0 = s.q_start;
  int64_t a = left >= kMaxPos ? blocks : (std::max<int64_t>(left - p0, 0) + per_cta - 1) / per_cta;
  a = std::min(a, blocks);
  int64_t b = s.causal || right >= kMaxPos ? blocks : (std::max<int64_t>(s.s_kv - right - p0, 0)) / per_cta;
  b = std::max(a, std::min(b, blocks));
  pl.blocks = (int)blocks;
  pl.first_mid = (int)a;
  pl.n_mid = (int)(b - a);
  const int64_t span = std::min(s.s_kv, left + right + per_cta) + std::min(s.sinks, s.s_kv);
  pl.heads_turn = s.n_kv_heads * std::min(span, s.s_kv) * 512 <= (256ll << 20);
  const int64_t key_tiles = (std::min(span, s.s_kv) + kBlockN - 1) / kBlockN;
  pl.token = 0;
  if (splits_asked == 0 && s.s_q == 1 && by_tokens(group, s.n_kv_heads, key_tiles, sms)) {
    pl.token = (int)std::max<int64_t>(1, std::min<int64_t>(kTokenMaxCluster, key_tiles));
    pl.splits = pl.n_items = pl.ctas = 1;
    return H3_OK;
  }
  int64_t splits = splits_asked;
  if (splits == 0) splits = std::min(slots / std::max<int64_t>(ctas, 1), key_tiles / 2);
  pl.splits = (int)std::max<int64_t>(1, std::min<int64_t>(splits, kMaxSplits));
  if (ctas * pl.splits > (1ll << 30)) return H3_ERR_SHAPE;
  pl.n_items = (int)ctas * pl.splits;
  // two tiles: a CTA per SM walks the items; one tile: a CTA per item (few rows: there are hardly more than fit)
  pl.ctas = pl.tiles == 2 ? std::min(pl.n_items, sms) : pl.n_items;
  return H3_OK;
}

static int sm_count(int& sms) {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess &&
                 cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess
             ? H3_OK
             : H3_ERR_CUDA;
}

// The fields of Params that the plan reads.
static void plan_params(const Shape& s, const Plan& pl, Params& p) {
  p.n_heads = (int)s.n_heads;
  p.group = (int)(s.n_heads / s.n_kv_heads);
  p.s_q = (int)s.s_q;
  p.s_kv = (int)s.s_kv;
  // A side without a bound, or with one beyond every key, reaches from any row of the call (and from the unused rows of
  // its last 256) over all keys: positions plus and minus it stay inside int32 wherever the call's positions lie.
  const int64_t far_left = std::max<int64_t>(0, s.q_start + s.s_q + 2 * kBlockM);
  const int64_t far_right = std::max<int64_t>(0, s.s_kv - s.q_start);
  p.left = (int)(s.left < 0 ? far_left : std::min(s.left, far_left));
  p.right = s.causal ? 0 : (int)(s.right < 0 ? far_right : std::min(s.right, far_right));
  p.sinks = (int)std::min(s.sinks, s.s_kv);
  p.causal = s.causal ? 1 : 0;
  p.q_start = (int)s.q_start;
  p.tile_pos = pl.tile_pos;
  p.blocks = pl.blocks;
  p.first_mid = pl.first_mid;
  p.n_mid = pl.n_mid;
  p.kv_heads = (int)s.n_kv_heads;
  p.heads_turn = pl.heads_turn;
  p.splits = pl.splits;
  p.n_items = pl.n_items;
  p.rounds = (pl.n_items + pl.ctas - 1) / pl.ctas;
}

// Key tiles of every work item, eight int32 a tile: CTA, round, key head, first query, part, first key, end of its run,
// bit 0 first-token run, bits 1 and 2 masked for the block's first and second Q tile. An item without keys has one
// with first key -1.
template <int kTiles>
static int64_t list_tiles(const Params& p, int ctas, int32_t* out, int64_t most) {
  int64_t n = 0;
  for (int r = 0; r < rounds_of<kTiles>(p); ++r)
    for (int c = 0; c < ctas; ++c) {
      const int w = item_of<kTiles>(p, r, c, ctas);
      if (w < 0) continue;
      Walk walk;
      const Item it = make_item<kTiles>(p, w, walk);
      for (int j = 0; j < std::max(it.n_kv, 1); ++j, ++n) {
        if (n >= most) return H3_ERR_WORKSPACE;
        const bool any = it.n_kv > 0, first_run = any && it.j_lo + j < walk.a_tiles;
        const int key = any ? walk.base(it.j_lo + j) : -1;
        int flags = first_run;
        for (int t = 0; any && t < kTiles; ++t) {
          const int first = p.q_start + it.i0 + t * p.tile_pos;
          flags |= int(is_masked(sees_all(p, first, first + p.tile_pos - 1), key, first_run)) << (1 + t);
        }
        const int32_t row[8] = {c, r, it.kvh, it.i0, it.z, key, any ? walk.end(it.j_lo + j) : -1, flags};
        std::copy(row, row + 8, out + 8 * n);
      }
    }
  return n;
}

static int64_t workspace_bytes(const Shape& s, const Plan& pl) {
  return pl.splits == 1 ? 0 : (int64_t)pl.splits * s.n_heads * s.s_q * (128 + 2) * (int64_t)sizeof(float);
}

// [kv_heads][s_q][group][128] view of q: box 64 x group x tile_pos x 1, SW128, zero fill.
static int make_q_map(CUtensorMap* map, const void* q, const Shape& s, int64_t head_stride, int64_t row_stride,
                      int tile_pos) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return H3_ERR_DRIVER;
  const cuuint64_t group = (cuuint64_t)(s.n_heads / s.n_kv_heads);
  const cuuint64_t hs = (cuuint64_t)(s.n_heads > 1 ? head_stride : s.s_q * row_stride);
  cuuint64_t dims[4] = {128, group, (cuuint64_t)s.s_q, (cuuint64_t)s.n_kv_heads};
  cuuint64_t strides[3] = {hs * 2, (cuuint64_t)row_stride * 2, hs * group * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)group, (cuuint32_t)tile_pos, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(q), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? H3_OK : H3_ERR_TENSOR_MAP;
}

template <int kTiles>
static int launch(cudaStream_t st, const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Params& p,
                  const Plan& pl) {
  using C = Cfg<kTiles>;
  auto* kern = window_kernel<kTiles>;
  // setmaxnreg draws on the registers the CTA is launched with: the split must fit them
  static const int regs = [&] {
    cudaFuncAttributes a;
    return cudaFuncGetAttributes(&a, kern) == cudaSuccess ? a.numRegs : 0;
  }();
  if (regs * C::kThreads < 128 * C::kRegsControl + 128 * kTiles * C::kRegsSoftmax) return H3_ERR_UNSUPPORTED;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)C::kSmem) != cudaSuccess)
    return H3_ERR_LAUNCH;
  kern<<<(unsigned)pl.ctas, C::kThreads, C::kSmem, st>>>(q, k, v, p);
  return cudaGetLastError() == cudaSuccess ? H3_OK : H3_ERR_LAUNCH;
}

}  // namespace window
}  // namespace h3

using namespace h3;
using namespace h3::window;

extern "C" int64_t h3_window_attn_workspace(int64_t n_heads, int64_t n_kv_heads, int64_t s_q, int64_t s_kv,
                                            int64_t left, int64_t right, int64_t sinks, int32_t causal,
                                            int64_t q_start, int64_t splits) {
  const Shape s = {n_heads, n_kv_heads, s_q, s_kv, left, right, sinks, q_start, causal};
  int rc;
  if ((rc = check_shape(s)) != H3_OK) return rc;
  if (splits < 0 || splits > kMaxSplits) return H3_ERR_SHAPE;
  Plan pl;
  int sms = 0;
  if ((rc = sm_count(sms)) != H3_OK || (rc = make_plan(s, splits, sms, pl)) != H3_OK) return rc;
  return workspace_bytes(s, pl);
}

extern "C" int64_t h3_window_plan_kat(int64_t n_heads, int64_t n_kv_heads, int64_t s_q, int64_t s_kv, int64_t left,
                                      int64_t right, int64_t sinks, int32_t causal, int64_t q_start, int64_t splits,
                                      int32_t sms, int32_t* tiles, int64_t max_tiles) {
  const Shape s = {n_heads, n_kv_heads, s_q, s_kv, left, right, sinks, q_start, causal};
  int rc;
  if (!tiles) return H3_ERR_NULL;
  if ((rc = check_shape(s)) != H3_OK) return rc;
  if (splits < 0 || splits > kMaxSplits || sms < 1) return H3_ERR_SHAPE;
  Plan pl;
  if ((rc = make_plan(s, splits, sms, pl)) != H3_OK) return rc;
  if (pl.token > 0) return H3_ERR_UNSUPPORTED;
  Params p = {};
  plan_params(s, pl, p);
  return pl.tiles == 2 ? list_tiles<2>(p, pl.ctas, tiles, max_tiles) : list_tiles<1>(p, pl.ctas, tiles, max_tiles);
}

extern "C" int h3_window_mask_kat(int64_t s_kv, int64_t left, int64_t right, int64_t sinks, int32_t causal,
                                  int64_t s_q, int64_t q_start, int64_t query, int64_t key, int32_t first_run,
                                  uint32_t* bits) {
  const Shape s = {1, 1, s_q, s_kv, left, right, sinks, q_start, causal};
  int rc;
  if (!bits) return H3_ERR_NULL;
  if ((rc = check_shape(s)) != H3_OK) return rc;
  if (query < 0 || query >= s_q || key < 0 || key >= s_kv) return H3_ERR_SHAPE;
  Plan pl;
  if ((rc = make_plan(s, 1, 1, pl)) != H3_OK) return rc;
  Params p = {};
  plan_params(s, pl, p);
  const Seen at = in_tile(sees(p, (int)(q_start + query)), (int)key, first_run != 0);
  for (int w = 0; w < kBlockN / 32; ++w) bits[w] = visible_bits(at.lo - 32 * w, at.hi - 32 * w, at.ns - 32 * w);
  return H3_OK;
}

extern "C" int h3_window_attn(const void* q, const void* k, const void* v, void* o, int64_t n_heads,
                              int64_t n_kv_heads, int64_t s_q, int64_t s_kv, int64_t q_head_stride,
                              int64_t q_row_stride, int64_t kv_head_stride, int64_t kv_row_stride, int64_t o_rank_rows,
                              int64_t o_rank_stride, int64_t o_head_stride, int64_t o_row_stride, float softmax_scale,
                              int64_t left, int64_t right, int64_t sinks, int32_t causal, int64_t q_start,
                              int64_t splits, void* workspace, int64_t ws_bytes, int32_t* status, void* stream) {
  if (!q || !k || !v || !o || !status) return H3_ERR_NULL;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(o) || (workspace && !aligned16(workspace)) ||
      (reinterpret_cast<uintptr_t>(status) & 3u))
    return H3_ERR_ALIGN;
  const Shape s = {n_heads, n_kv_heads, s_q, s_kv, left, right, sinks, q_start, causal};
  int rc;
  if ((rc = check_shape(s)) != H3_OK) return rc;
  if (o_rank_rows < 1 || splits < 0 || splits > kMaxSplits) return H3_ERR_SHAPE;
  if (!(softmax_scale > 0.f) || !std::isfinite(softmax_scale)) return H3_ERR_SHAPE;
  if (q_row_stride < 128 || kv_row_stride < 128 || o_row_stride < 128 || (q_row_stride % 8) || (kv_row_stride % 8) ||
      (q_head_stride % 8) || (kv_head_stride % 8) || (o_row_stride % 8) || (o_head_stride % 8) ||
      (o_rank_stride % 8) || q_head_stride < 0 || kv_head_stride < 0 || o_head_stride < 0 || o_rank_stride < 0 ||
      (n_heads > 1 && q_head_stride == 0) || (n_kv_heads > 1 && kv_head_stride == 0))
    return H3_ERR_STRIDE;
  Plan pl;
  int sms = 0;
  if ((rc = sm_count(sms)) != H3_OK || (rc = make_plan(s, splits, sms, pl)) != H3_OK) return rc;
  if (ws_bytes < workspace_bytes(s, pl)) return H3_ERR_WORKSPACE;
  if (pl.splits > 1 && !workspace) return H3_ERR_NULL;

  Params p = {};
  plan_params(s, pl, p);
  p.scale_log2 = (float)((double)softmax_scale * 1.4426950408889634);
  p.o = reinterpret_cast<__nv_bfloat16*>(o);
  p.o_rank_rows = o_rank_rows;
  p.o_rank_stride = o_rank_stride;
  p.o_head_stride = o_head_stride;
  p.o_row_stride = o_row_stride;
  p.part_o = pl.splits > 1 ? reinterpret_cast<float*>(workspace) : nullptr;
  p.part_ml = pl.splits > 1 ? p.part_o + (int64_t)pl.splits * n_heads * s_q * 128 : nullptr;
  p.status = status;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (pl.token > 0) {
    const TokenParams tp = {reinterpret_cast<const __nv_bfloat16*>(q), reinterpret_cast<const __nv_bfloat16*>(k),
                            reinterpret_cast<const __nv_bfloat16*>(v), q_head_stride, kv_head_stride, kv_row_stride};
    auto* kern = p.group == 1 ? token_kernel<1> : p.group == 2 ? token_kernel<2> : p.group == 3 ? token_kernel<3>
                                                                                               : token_kernel<4>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)pl.token, (unsigned)n_kv_heads);
    cfg.blockDim = dim3(32 * kTokenWarps);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)pl.token;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaLaunchKernelEx(&cfg, kern, p, tp) != cudaSuccess) return H3_ERR_LAUNCH;
    return cudaGetLastError() == cudaSuccess ? H3_OK : H3_ERR_LAUNCH;
  }
  CUtensorMap mq, mk, mv;
  const long long kvhs = n_kv_heads > 1 ? kv_head_stride : s_kv * kv_row_stride;
  if ((rc = make_q_map(&mq, q, s, q_head_stride, q_row_stride, pl.tile_pos)) != H3_OK) return rc;
  if ((rc = make_head_map(&mk, k, s_kv, n_kv_heads, kv_row_stride, kvhs)) != H3_OK) return rc;
  if ((rc = make_head_map(&mv, v, s_kv, n_kv_heads, kv_row_stride, kvhs)) != H3_OK) return rc;
  rc = pl.tiles == 2 ? launch<2>(st, mq, mk, mv, p, pl) : launch<1>(st, mq, mk, mv, p, pl);
  if (rc != H3_OK || pl.splits == 1) return rc;
  return launch_dependent(join_kernel, dim3((unsigned)(n_heads * s_q)), 32 * kJoinWarps, 0, st, p, pl.splits);
}
