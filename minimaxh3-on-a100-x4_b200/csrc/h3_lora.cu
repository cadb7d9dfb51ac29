// Low-rank adapters of many requests beside a shared projection:
//   y_t = W x_t + s_a B_a (A_a x_t),   a = row_adapter[t]       (a outside [0, n_adapters): y_t = W x_t)
// bf16 in, fp32 accumulate, one rounding of y (epilogue 1: the SwiGLU of h3_gemm_bf16, with its roundings).
// The adapters are stacked: A rows [a * rank, (a + 1) * rank) of [n_adapters * rank][k], B the same columns of
// [n][n_adapters * rank], so 64 stacked columns (a "chunk") are one k-block of the tensor cores whatever the rank.
//
// Many rows (tile path, two launches). lower_kernel: T = s_a A_a x for each row's own adapter, tcgen05 tiles of
// 128 rows x 64 stacked columns over k, only the chunks that a row of the tile uses; bound by reading x. T is
// rounded once to bf16 (2^-8 of T, the operand type of the second product; against y this is below y's own
// rounding unless the adapter outweighs the projection). adapter_gemm_kernel: the projection GEMM (SM-pair tiles
// of 256 x 256) with, behind a tile's k-blocks of x and W, one more per chunk in use: its A operand is T, written to
// shared memory by four extra warps with zeros outside each row's adapter, its B operand the chunk's columns of
// the stacked B by TMA. So the adapters cost (64 * chunks) / k of the projection's products and no pass
// over y. It is launched as a programmatic dependent: its first tiles run while lower_kernel finishes.
//
// Few rows (row path, three launches): bound by reading W once. The weights are the M = 128 operand and the rows (16 ..
// 64 of them) the N operand. few_lower_kernel: T, a cluster of 8 CTAs per 128 rows of the stacked A in use, an eighth of
// k each, summed through distributed shared memory. stream_kernel: all k-blocks of W and, behind those of each
// 128-row tile, the chunks in use of the same rows of the stacked B against T (as above); they are dealt out
// evenly to two CTAs per SM, and each CTA writes fp32 sums of the piece of a tile that it had. finish_kernel adds a
// column's pieces in a fixed order, rounds and stores. Each launch is a programmatic dependent of the one before:
// W streams while T is made, and a CTA leaves its piece with B for last. (B T by scalar code in finish_kernel took
// 15-25 us at 37 rows x 21504 columns.)
//
// Tile path: a row's bits do not depend on the other rows of the call or on its length. Row path: they do not depend on
// the other rows' values, but where a column's pieces begin follows the chunks in use. A caller that needs the first
// whatever the length (shards of one sequence) asks for tiles with H3_GEMM_ROW_INDEPENDENT.
#include <algorithm>

#include "h3_gemm.cuh"

namespace h3 {
namespace lora {

using namespace h3::gemm;

constexpr int kMaxRank = 256;
constexpr int kMaxChunks = 1024;  // n_adapters * rank <= 65536
// Row path up to here: 5376 -> 21504 with 24 adapters of rank 16, 64 rows 54 us, 65 rows by tiles 85; 7168 -> 5376 with 4,
// 26 and 42. (Its accumulators and partial sums grow with the rows; the tiles cost the same up to 256.)
constexpr int kFewRows = 64;

struct Adapters {
  const int* row_adapter;
  const float* scale;
  int n_adapters, rank;
};
// the adapter of row r, or -1
__device__ __forceinline__ int adapter_of(const Adapters& ad, int m, int r) {
  const int a = r < m ? ad.row_adapter[r] : -1;
  return a >= 0 && a < ad.n_adapters ? a : -1;
}

// ---------------------------------------------------------------- tile path: T = s A x
// k is summed in kQuarters parts, each on its own, and the parts are added in ascending order. With few tiles of rows a
// cluster of kQuarters CTAs takes one part each (kCluster = 4) and the parts meet in distributed shared memory; with many, one
// CTA takes them one after the other (kCluster = 1). Both give the same bits, so a row's T does not depend on the
// call's length. One CTA per SM. 42000 rows of 7168: 99 us = 6.1 TB/s; whole calls of 1000 rows, 7168 -> 5376: 98 us with
// one CTA per tile over all of k, 82 so; 65 rows of 5376 -> 21504, 4 adapters of rank 32: 86 and 77. With many chunks in use
// the launch is what bounds it: a tile's passes come one after the other, 43 us on 4 CTAs for 65 rows with 24 adapters of
// rank 16 (two passes), 332 us on 32 CTAs for 1000 rows with 24 of rank 128 (twelve).
constexpr int kQuarters = 4;
constexpr uint32_t kChunkBytes = 64u * 64u * 2u;
constexpr uint32_t kLowerRing = 192u * 1024u;
constexpr int kLowerMaxStages = 6;
template <int kCluster>
struct Lower {
  // Chunks per pass over k: tensor memory holds kQuarters parts of two, or a cluster's CTA its own part of four.
  static constexpr int kPass = kCluster > 1 ? 4 : 2;
  static constexpr uint32_t kStage = kTileBytes + kPass * kChunkBytes;
  static constexpr int kStages = kLowerRing / kStage;
  static constexpr int kSumRow = 64 * kPass + 4;  // floats of a row of the cluster's sums (padded against bank conflicts)
  static_assert(kStages <= kLowerMaxStages && 128 * kSumRow * 4 <= kLowerRing, "the sums reuse the ring");
};
constexpr int kNoColumn = 1 << 30;
struct LowerSmem {
  uint32_t own[kMaxChunks / 32], both[kMaxChunks / 32];  // chunks in use: these 128 rows, the block of 256
  uint16_t list[kMaxChunks];
  int col0[128];     // first stacked column of each row's adapter, or kNoColumn
  float scale[128];
  int count;
  uint64_t bars[2 * kLowerMaxStages + 3];
  uint32_t tmem;
  int abort;
};
constexpr uint32_t kLowerSmem = 1024 + kLowerRing + sizeof(LowerSmem);

template <int kCluster>
__global__ void __launch_bounds__(192, 1)
    lower_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_a,
                 const Adapters ad, __nv_bfloat16* low, int* chunks, int chunk_stride, int m, int n_kb, int kc_blocks,
                 int* status) {
  constexpr int kPass = Lower<kCluster>::kPass, kLowerStages = Lower<kCluster>::kStages;
  constexpr int kSumRow = Lower<kCluster>::kSumRow;
  constexpr uint32_t kLowerStage = Lower<kCluster>::kStage;
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  LowerSmem& sh = *reinterpret_cast<LowerSmem*>(smem + kLowerRing);
  enum { kF = 0, kE = kLowerStages, kAccF = 2 * kLowerStages, kAccE = kAccF + 1, kD = kAccE + 1 };
  auto bar = [&](int i) { return smem_u32(&sh.bars[i]); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = blockIdx.x / kCluster, m0 = tile * 128;
  const int rank = kCluster > 1 ? int(cluster_ctarank()) : 0;
  const int q_begin = kCluster > 1 ? rank : 0, q_end = kCluster > 1 ? rank + 1 : kQuarters;  // this CTA's parts of k
  auto acc = [&](int q, int i) { return 64u * uint32_t(kCluster > 1 ? i : kPass * q + i); };  // columns of part q, chunk i
  auto part = [&](int q) { return n_kb * q / kQuarters; };                                  // first k-block of part q

  for (int i = threadIdx.x; i < kMaxChunks / 32; i += 192) sh.own[i] = sh.both[i] = 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kLowerStages; ++s) {
      mbar_init(bar(kF + s), 1);
      mbar_init(bar(kE + s), 1);
    }
    mbar_init(bar(kAccF), 1);
    mbar_init(bar(kAccE), 4);
    mbar_init(bar(kD), 1);
    sh.abort = *reinterpret_cast<volatile int*>(status) != 0 ? 1 : 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sh.tmem), 512);
    tmem_relinquish();
  }
  __syncthreads();
  // chunks in use by the 256-row block, and by this tile's 128 rows of it
  for (int r = threadIdx.x; r < 256; r += 192) {
    const int row = (m0 & ~255) + r;
    const int a = adapter_of(ad, m, row);
    if ((row & ~127) == m0) {
      sh.col0[row - m0] = a < 0 ? kNoColumn : a * ad.rank;
      sh.scale[row - m0] = a < 0 ? 0.f : ad.scale[a];
    }
    if (a < 0) continue;
    const int last = (a * ad.rank + ad.rank - 1) / 64;
    for (int c = a * ad.rank / 64; c <= last; ++c) {
      atomicOr(&sh.both[c / 32], 1u << (c & 31));
      if ((row & ~127) == m0) atomicOr(&sh.own[c / 32], 1u << (c & 31));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 2 || (warp == 3 && (tile & 1) == 0 && rank == 0)) {
    // ascending lists: this tile's in shared memory, the block's (its first tile writes it) in global memory
    const uint32_t word = warp == 2 ? sh.own[lane] : sh.both[lane];
    int at = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += up;
    }
    int* out = chunks + (long long)(tile >> 1) * chunk_stride;
    if (lane == 31) {
      if (warp == 2)
        sh.count = at;
      else
        out[0] = at;
    }
    at -= __popc(word);
    for (uint32_t w = word; w != 0; w &= w - 1, ++at) {
      const int c = 32 * lane + __ffs(w) - 1;
      if (warp == 2)
        sh.list[at] = (uint16_t)c;
      else
        out[1 + at] = c;
    }
  }
  __syncthreads();
  const int count = sh.count;
  const uint32_t tmem = sh.tmem;
  const WaitCtx ctx{&sh.abort, status};
  const bool run = sh.abort == 0 && count > 0;
  const int passes = (count + kPass - 1) / kPass;

  const bool issuer = warp < 2 && elect_one();
  const int quad = warp & 3;
  const uint32_t lane_off = uint32_t(quad * 32) << 16;
  float* sums = reinterpret_cast<float*>(smem);  // kCluster > 1: [128 rows][kSumRow] of this CTA's part, between passes
  int it = 0;                                    // ring items so far
  bool ok = run;
  // Whether 8 stacked columns from `col` on are row r_in's adapter's, and where its T goes.
  auto owns = [&](int r_in, int col) { return col >= sh.col0[r_in] && col < sh.col0[r_in] + ad.rank; };
  auto put = [&](int r_in, int col, const float (&v)[8]) {
    const float scale = sh.scale[r_in];
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = pack_bf16x2(v[2 * e] * scale, v[2 * e + 1] * scale);
    *reinterpret_cast<uint4*>(low + (long long)(m0 + r_in) * ad.rank + (col - sh.col0[r_in])) =
        make_uint4(w[0], w[1], w[2], w[3]);
  };

  for (int ps = 0; ps < passes; ++ps) {
    const int nc = min(kPass, count - ps * kPass);
    if (warp == 0) {
      for (int kb = part(q_begin); ok && kb < part(q_end); ++kb, ++it) {
        const int st = it % kLowerStages;
        if (it >= kLowerStages &&
            !(ok = __all_sync(0xffffffffu, mbar_wait(bar(kE + st), uint32_t(it / kLowerStages - 1) & 1u, ctx,
                                                     kStatusTimeoutKV))))
          break;
        if (issuer) {
          const uint32_t dst = sbase + st * kLowerStage;
          mbar_expect_tx(bar(kF + st), kTileBytes + nc * kChunkBytes);
          tma_load_3d(dst, &tmap_x, bar(kF + st), 64 * (kb % kc_blocks), m0, kb / kc_blocks);
          for (int i = 0; i < nc; ++i)
            tma_load_3d(dst + kTileBytes + i * kChunkBytes, &tmap_a, bar(kF + st), 64 * kb,
                        64 * sh.list[ps * kPass + i], 0);
        }
        __syncwarp();
      }
    } else if (warp == 1) {
      constexpr uint32_t idesc = idesc_bf16_f32(128, 64, 0, 0);
      if (ok && ps > 0)  // the pass before has been read out of the accumulators
        ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccE), uint32_t(ps - 1) & 1u, ctx, kStatusTimeoutO));
      tc_fence_after();
      for (int q = q_begin; q < q_end; ++q)
        for (int kb = part(q); ok && kb < part(q + 1); ++kb, ++it) {
          const int st = it % kLowerStages;
          if (!(ok = __all_sync(0xffffffffu,
                                mbar_wait(bar(kF + st), uint32_t(it / kLowerStages) & 1u, ctx, kStatusTimeoutKV))))
            break;
          tc_fence_after();
          if (issuer) {
            const uint32_t x = sbase + st * kLowerStage;
            for (int i = 0; i < nc; ++i)
              for (int ks = 0; ks < 4; ++ks)
                mma_ss(tmem + acc(q, i), smem_desc_sw128(x + 32u * ks, 16, 1024),
                       smem_desc_sw128(x + kTileBytes + i * kChunkBytes + 32u * ks, 16, 1024), idesc,
                       kb > part(q) || ks > 0 ? 1u : 0u);
            mma_commit(bar(kE + st));
          }
          __syncwarp();
        }
      if (ok && issuer) mma_commit(bar(kAccF));
      __syncwarp();
    } else {
      if (ok) ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccF), uint32_t(ps) & 1u, ctx, kStatusTimeoutS));
      tc_fence_after();
      const int r_in = quad * 32 + lane;
      for (int i = 0; i < nc; ++i)
#pragma unroll 1
        for (int c = 0; c < 4; ++c) {
          float v[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = 0.f;
          for (int q = q_begin; q < q_end; ++q) {
            if (!ok || part(q) == part(q + 1)) continue;
            uint32_t r[16];
            tmem_ld16_wait(tmem + lane_off + acc(q, i) + 16u * c, r);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] += __uint_as_float(r[e]);
          }
          if constexpr (kCluster > 1) {
            float4* d = reinterpret_cast<float4*>(sums + r_in * kSumRow + 64 * i + 16 * c);
#pragma unroll
            for (int e = 0; e < 4; ++e) d[e] = make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          } else if (ok) {
            const int col = 64 * sh.list[ps * kPass + i] + 16 * c;
            const float lo[8] = {v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]};
            const float hi[8] = {v[8], v[9], v[10], v[11], v[12], v[13], v[14], v[15]};
            if (owns(r_in, col)) put(r_in, col, lo);
            if (owns(r_in, col + 8)) put(r_in, col + 8, hi);
            __syncwarp();  // the next load of the accumulators takes the whole warp
          }
        }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kAccE));
    }
    if constexpr (kCluster > 1) {
      // the ring is idle: every MMA of the pass has retired (kAccF), and nothing was loaded beyond it. This CTA adds the
      // parts of its 32 rows.
      __syncthreads();
      cluster_sync_all();
      constexpr int kRows = 128 / kCluster;
      for (int i = threadIdx.x; i < kRows * 8 * nc; i += 192) {
        const int r_in = kRows * rank + i / (8 * nc), piece = i % (8 * nc);
        const int col = 64 * sh.list[ps * kPass + piece / 8] + 8 * (piece % 8);
        if (!owns(r_in, col) || sh.abort != 0) continue;
        float4 lo[kCluster], hi[kCluster];
        const uint32_t from = smem_u32(sums + r_in * kSumRow + 8 * piece);
#pragma unroll
        for (int q = 0; q < kCluster; ++q) {
          const uint32_t at = mapa_shared(from, q);
          lo[q] = ld_cluster_f32x4(at);
          hi[q] = ld_cluster_f32x4(at + 16u);
        }
        float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < kCluster; ++q) {
          const float part_v[8] = {lo[q].x, lo[q].y, lo[q].z, lo[q].w, hi[q].x, hi[q].y, hi[q].z, hi[q].w};
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] += part_v[e];
        }
        put(r_in, col, v);
      }
      cluster_sync_all();   // the sums have been read: the ring may be filled again
      fence_proxy_async();  // by the async proxy
    }
  }
  if (warp == 0 && issuer) {
    for (int st = 0; st < kLowerStages; ++st) {
      const int cnt = it / kLowerStages + (st < it % kLowerStages ? 1 : 0);
      if (cnt > 0) drain_wait_cluster(bar(kF + st), uint32_t(cnt - 1) & 1u, status);
    }
  } else if (warp == 1 && issuer) {
    mma_commit(bar(kD));
    drain_wait_cluster(bar(kD), 0, status);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- tile path: y = W x + B T
constexpr int kAdapterThreads = kThreads + 32 * kLowWarps;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kAdapterThreads, 1)
    adapter_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                        const __grid_constant__ CUtensorMap tmap_b, const Params p) {
  gemm_body<true>(tmap_x, tmap_w, tmap_b, p);
}

// ---------------------------------------------------------------- row path: T
constexpr int kRing = 4;  // stages at most
// 72 KB, three to four stages: two CTAs of stream_kernel and one of few_lower_kernel fit an SM, so that no CTA of the
// first waits for the second to leave (with 108 KB rings that cost 4-5 us of 24-51).
constexpr uint32_t kRingBytes = 72u * 1024u;
constexpr int kSplitK = 8;  // CTAs of a cluster, each an eighth of k

struct Few {
  int m, m_pad;         // rows, and rows rounded up to 16
  int n_kb, kc_blocks;  // k-blocks of 64
  int stages;
  int* status;
  __nv_bfloat16* low;   // T [m][rank]
};

struct FewLowerSmem {
  uint64_t bars[2 * kRing + 2];
  uint32_t tmem;
  int abort, used;
};
constexpr uint32_t kFewLowerSmem = 1024 + kRingBytes + sizeof(FewLowerSmem);
static_assert(kRingBytes >= kFewRows * 128 * 4, "the sums reuse the ring");

__global__ void __launch_bounds__(192, 2)
    few_lower_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_x,
                     const Adapters ad, const Few f) {
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  FewLowerSmem& sh = *reinterpret_cast<FewLowerSmem*>(smem + kRingBytes);
  enum { kF = 0, kE = kRing, kAcc = 2 * kRing, kD = kAcc + 1 };
  auto bar = [&](int i) { return smem_u32(&sh.bars[i]); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = int(cluster_ctarank());
  const int tile = blockIdx.x / kSplitK;  // 128 rows of the stacked A
  const uint32_t stage_bytes = kTileBytes + uint32_t(f.m_pad) * 128u;
  const uint32_t cols = f.m_pad <= 32 ? 32u : 64u;
  const int kb0 = f.n_kb * rank / kSplitK, kb1 = f.n_kb * (rank + 1) / kSplitK;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(bar(kF + i), 1);
      mbar_init(bar(kE + i), 1);
    }
    mbar_init(bar(kAcc), 1);
    mbar_init(bar(kD), 1);
    sh.abort = *reinterpret_cast<volatile int*>(f.status) != 0 ? 1 : 0;
    sh.used = 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sh.tmem), cols);
    tmem_relinquish();
  }
  __syncthreads();
  if (threadIdx.x < f.m) {  // does a row use an adapter with rows in this tile?
    const int a = adapter_of(ad, f.m, threadIdx.x);
    if (a >= 0 && a * ad.rank < 128 * (tile + 1) && (a + 1) * ad.rank > 128 * tile) sh.used = 1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const WaitCtx ctx{&sh.abort, f.status};
  const bool used = sh.used != 0;  // the same in every CTA of the cluster
  const bool run = sh.abort == 0 && used && kb1 > kb0;

  if (warp == 0 && run) {
    const bool issuer = elect_one();
    int it = 0;
    for (int kb = kb0; kb < kb1; ++kb, ++it) {
      const int st = it % f.stages;
      if (it >= f.stages &&
          !__all_sync(0xffffffffu, mbar_wait(bar(kE + st), uint32_t(it / f.stages - 1) & 1u, ctx, kStatusTimeoutKV)))
        break;
      if (issuer) {
        const uint32_t dst = sbase + st * stage_bytes;
        mbar_expect_tx(bar(kF + st), stage_bytes);
        tma_load_3d(dst, &tmap_a, bar(kF + st), 64 * kb, 128 * tile, 0);
        tma_load_3d(dst + kTileBytes, &tmap_x, bar(kF + st), 64 * (kb % f.kc_blocks), 0, kb / f.kc_blocks);
      }
      __syncwarp();
    }
    if (issuer)
      for (int st = 0; st < f.stages; ++st) {
        const int cnt = it / f.stages + (st < it % f.stages ? 1 : 0);
        if (cnt > 0) drain_wait_cluster(bar(kF + st), uint32_t(cnt - 1) & 1u, f.status);
      }
    __syncwarp();
  } else if (warp == 1 && run) {
    const bool issuer = elect_one();
    const uint32_t idesc = idesc_bf16_f32(128, f.m_pad, 0, 0);
    int it = 0;
    bool ok = true;
    for (int kb = kb0; kb < kb1; ++kb, ++it) {
      const int st = it % f.stages;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kF + st), uint32_t(it / f.stages) & 1u, ctx, kStatusTimeoutKV))))
        break;
      tc_fence_after();
      if (issuer) {
        const uint32_t w = sbase + st * stage_bytes;
        for (int ks = 0; ks < 4; ++ks)
          mma_ss(tmem, smem_desc_sw128(w + 32u * ks, 16, 1024), smem_desc_sw128(w + kTileBytes + 32u * ks, 16, 1024),
                 idesc, kb > kb0 || ks > 0 ? 1u : 0u);
        mma_commit(bar(kE + st));
      }
      __syncwarp();
    }
    if (issuer) {
      if (ok) mma_commit(bar(kAcc));
      mma_commit(bar(kD));
      drain_wait_cluster(bar(kD), 0, f.status);
    }
    __syncwarp();
  }
  // sums of this CTA's share of k to sums[row of x][row of the tile] (the ring is idle: every MMA has retired)
  float* sums = reinterpret_cast<float*>(smem);
  if (warp >= 2 && used) {
    const int quad = warp & 3;
    const bool ok = run && __all_sync(0xffffffffu, mbar_wait(bar(kAcc), 0, ctx, kStatusTimeoutS));
    tc_fence_after();
    for (int q = 0; q < f.m_pad / 16; ++q) {
      uint32_t r[16];
      if (ok) tmem_ld16_wait(tmem + (uint32_t(quad * 32) << 16) + 16u * q, r);
#pragma unroll
      for (int e = 0; e < 16; ++e) sums[(16 * q + e) * 128 + quad * 32 + lane] = ok ? __uint_as_float(r[e]) : 0.f;
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  if (used && sh.abort == 0) {
    // this CTA's sixteenth-row slices of the tile, over the cluster's sums in ascending order
    constexpr int kMine = 128 / kSplitK;
    for (int i = threadIdx.x; i < f.m * kMine; i += 192) {
      const int row = i / kMine, at = kMine * rank + i % kMine;
      const int g = 128 * tile + at, a = g / ad.rank;
      if (adapter_of(ad, f.m, row) != a) continue;
      float v = 0.f;
#pragma unroll
      for (int c = 0; c < kSplitK; ++c) v += ld_cluster_f32(mapa_shared(smem_u32(sums + row * 128 + at), c));
      f.low[(long long)row * ad.rank + (g - a * ad.rank)] = __float2bfloat16_rn(v * ad.scale[a]);
    }
  }
  cluster_sync_all();  // no CTA leaves while another reads its sums
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// ---------------------------------------------------------------- row path: W and B streamed once
struct Stream {
  Few f;
  int tiles;          // 128-row tiles of W
  int* head;          // [2]: k-blocks per tile (those of W and the chunks in use), k-blocks per CTA
  float* part;        // [piece][m][columns]
  long long columns;  // 128 * tiles
};
// A tile's k-blocks [tile * per_tile, (tile + 1) * per_tile) of the whole list lie in CTAs first .. last; its pieces are
// numbered from the first.
__host__ __device__ inline int first_cta(int tile, int per_tile, int per_cta) {
  return int((long long)tile * per_tile / per_cta);
}
__host__ __device__ inline int last_cta(int tile, int per_tile, int per_cta) {
  return int(((long long)(tile + 1) * per_tile - 1) / per_cta);
}

// The share [begin, end) of CTA `cta` of `ctas` in the list of all tiles' k-blocks.
struct Share {
  int per_cta;
  long long begin, end;
};
__host__ __device__ inline Share share_of(int tiles, int per_tile, int cta, int ctas) {
  const long long total = (long long)tiles * per_tile;
  Share s;
  s.per_cta = int((total + ctas - 1) / ctas);
  const long long from = (long long)cta * s.per_cta;
  s.begin = from < total ? from : total;
  s.end = from + s.per_cta < total ? from + s.per_cta : total;
  return s;
}
// A CTA's pieces, k-blocks [kb0, kb1) of a tile, from the last to the first: the start of a tile, whole ones, the end of one
// with its chunks of B. The piece that ends at g; g becomes its begin.
struct Piece {
  int tile, kb0, kb1;
};
__host__ __device__ inline Piece piece_of(const Share& s, int per_tile, long long& g) {
  Piece q;
  q.tile = int((g - 1) / per_tile);
  const long long base = (long long)q.tile * per_tile;
  q.kb1 = int(g - base);
  q.kb0 = int(s.begin > base ? s.begin - base : 0);
  g = base + q.kb0;
  return q;
}

constexpr int kStreamThreads = 256;  // TMA, MMA, 4 epilogue warps, 2 warps that write T
constexpr int kFewChunks = kFewRows * (kMaxRank / 64);  // chunks in use at most

struct StreamSmem {
  uint32_t bits[kMaxChunks / 32];  // chunks in use
  uint16_t list[kFewChunks];
  int count;
  uint64_t bars[4 * kRing + 5];
  uint32_t tmem;
  int abort;
};
constexpr uint32_t kStreamSmem = 1024 + kRingBytes + sizeof(StreamSmem);

__global__ void __launch_bounds__(kStreamThreads, 2)
    stream_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                  const __grid_constant__ CUtensorMap tmap_b, const Adapters ad, const Stream s) {
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  StreamSmem& sh = *reinterpret_cast<StreamSmem*>(smem + kRingBytes);
  enum { kF = 0, kE = kRing, kLF = 2 * kRing, kLE = 3 * kRing, kAccF = 4 * kRing, kAccE = kAccF + 2, kD = kAccE + 2 };
  auto bar = [&](int i) { return smem_u32(&sh.bars[i]); };
  const Few& f = s.f;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t stage_bytes = kTileBytes + uint32_t(f.m_pad) * 128u;
  // two accumulators of m_pad columns
  const uint32_t cols = f.m_pad <= 16 ? 32u : (f.m_pad <= 32 ? 64u : 128u);

  for (int i = threadIdx.x; i < kMaxChunks / 32; i += kStreamThreads) sh.bits[i] = 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kRing; ++i) {
      mbar_init(bar(kF + i), 1);
      mbar_init(bar(kE + i), 1);
      mbar_init(bar(kLE + i), 1);
      mbar_init(bar(kLF + i), 2);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kAccF + b), 1);
      mbar_init(bar(kAccE + b), 4);
    }
    mbar_init(bar(kD), 1);
    sh.abort = *reinterpret_cast<volatile int*>(f.status) != 0 ? 1 : 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sh.tmem), cols);
    tmem_relinquish();
  }
  __syncthreads();
  if (threadIdx.x < f.m) {
    const int a = adapter_of(ad, f.m, threadIdx.x);
    if (a >= 0) {
      const int last = (a * ad.rank + ad.rank - 1) / 64;
      for (int c = a * ad.rank / 64; c <= last; ++c) atomicOr(&sh.bits[c / 32], 1u << (c & 31));
    }
  }
  __syncthreads();
  if (warp == 2) {  // ascending list of the chunks in use
    const uint32_t word = sh.bits[lane];
    int at = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += up;
    }
    if (lane == 31) sh.count = at;
    at -= __popc(word);
    for (uint32_t w = word; w != 0; w &= w - 1, ++at) sh.list[at] = (uint16_t)(32 * lane + __ffs(w) - 1);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const WaitCtx ctx{&sh.abort, f.status};
  const bool run = sh.abort == 0;
  const int per_tile = f.n_kb + sh.count;
  const Share mine = share_of(s.tiles, per_tile, int(blockIdx.x), int(gridDim.x));
  const int per_cta = mine.per_cta;
  const long long g_begin = mine.begin, g_end = mine.end;
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    s.head[0] = per_tile;
    s.head[1] = per_cta;
  }
  auto piece = [&](long long& g) { return piece_of(mine, per_tile, g); };

  if (warp == 0 && run) {
    const bool issuer = elect_one();
    int it = 0;
    bool ok = true;
    for (long long g = g_end; ok && g > g_begin;) {
      const Piece q = piece(g);
      for (int kb = q.kb0; kb < q.kb1; ++kb, ++it) {
        const int st = it % f.stages;
        if (it >= f.stages && !(ok = __all_sync(0xffffffffu, mbar_wait(bar(kE + st), uint32_t(it / f.stages - 1) & 1u,
                                                                       ctx, kStatusTimeoutKV))))
          break;
        if (issuer) {
          const uint32_t dst = sbase + st * stage_bytes;
          if (kb < f.n_kb) {
            mbar_expect_tx(bar(kF + st), stage_bytes);
            tma_load_3d(dst, &tmap_w, bar(kF + st), 64 * kb, 128 * q.tile, 0);
            tma_load_3d(dst + kTileBytes, &tmap_x, bar(kF + st), 64 * (kb % f.kc_blocks), 0, kb / f.kc_blocks);
          } else {
            mbar_arrive(bar(kLE + st));
            mbar_expect_tx(bar(kF + st), kTileBytes);
            tma_load_3d(dst, &tmap_b, bar(kF + st), 64 * sh.list[kb - f.n_kb], 128 * q.tile, 0);
          }
        }
        __syncwarp();
      }
    }
    if (issuer)
      for (int st = 0; st < f.stages; ++st) {
        const int cnt = it / f.stages + (st < it % f.stages ? 1 : 0);
        if (cnt > 0) drain_wait_cluster(bar(kF + st), uint32_t(cnt - 1) & 1u, f.status);
      }
    __syncwarp();
  } else if (warp == 1 && run) {
    const bool issuer = elect_one();
    const uint32_t idesc = idesc_bf16_f32(128, f.m_pad, 0, 0);
    int it = 0, i = 0;
    uint32_t low_par = 0;  // bit st: parity of the stage's next use for T
    bool ok = true;
    for (long long g = g_end; ok && g > g_begin; ++i) {
      const Piece q = piece(g);
      const int b = i & 1;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccE + b), (uint32_t(i >> 1) & 1u) ^ 1u, ctx, kStatusTimeoutO))))
        break;
      tc_fence_after();
      for (int kb = q.kb0; kb < q.kb1; ++kb, ++it) {
        const int st = it % f.stages;
        if (!(ok = __all_sync(0xffffffffu,
                              mbar_wait(bar(kF + st), uint32_t(it / f.stages) & 1u, ctx, kStatusTimeoutKV))))
          break;
        if (kb >= f.n_kb) {
          if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kLF + st), (low_par >> st) & 1u, ctx, kStatusTimeoutKV))))
            break;
          low_par ^= 1u << st;
        }
        tc_fence_after();
        if (issuer) {
          const uint32_t w = sbase + st * stage_bytes;
          for (int ks = 0; ks < 4; ++ks)
            mma_ss(tmem + uint32_t(b * f.m_pad), smem_desc_sw128(w + 32u * ks, 16, 1024),
                   smem_desc_sw128(w + kTileBytes + 32u * ks, 16, 1024), idesc, kb > q.kb0 || ks > 0 ? 1u : 0u);
          mma_commit(bar(kE + st));
        }
        __syncwarp();
      }
      if (ok && issuer) mma_commit(bar(kAccF + b));
      __syncwarp();
    }
    if (issuer) {
      mma_commit(bar(kD));
      drain_wait_cluster(bar(kD), 0, f.status);
    }
    __syncwarp();
  } else if (warp >= 2 && warp < 6 && run) {
    const int quad = warp & 3;
    const uint32_t lane_off = uint32_t(quad * 32) << 16;
    int i = 0;
    bool ok = true;
    for (long long g = g_end; ok && g > g_begin; ++i) {
      const Piece q = piece(g);
      const int b = i & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccF + b), uint32_t(i >> 1) & 1u, ctx, kStatusTimeoutS));
      if (!ok) break;
      tc_fence_after();
      // lane = column of the tile: a warp stores 32 consecutive columns of a row
      float* dst = s.part + (long long)((int)blockIdx.x - first_cta(q.tile, per_tile, per_cta)) * f.m * s.columns +
                   128ll * q.tile + quad * 32 + lane;
#pragma unroll 1
      for (int c = 0; c < f.m_pad / 16; ++c) {
        uint32_t r[16];
        tmem_ld16_wait(tmem + lane_off + uint32_t(b * f.m_pad + 16 * c), r);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (16 * c + e < f.m) dst[(16 * c + e) * s.columns] = __uint_as_float(r[e]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kAccE + b));
    }
  } else if (warp >= 6 && run && sh.count > 0) {
    // T of a chunk: one thread per row of x, zeros outside the row's own adapter; K-major, 128-byte swizzle
    const int row = (warp - 6) * 32 + lane;
    const int a = adapter_of(ad, f.m, row);
    const int col0 = a >= 0 ? a * ad.rank : -1;
    const int pieces = min(ad.rank, 64) / 8;
    const uint4* src = reinterpret_cast<const uint4*>(f.low + (long long)row * ad.rank);
    const int at = (max(col0, 0) & 63) / 8;  // the row's pieces of 8 columns in its (first) chunk: [at, at + pieces)
    uint32_t free_par = 0;
    int it = 0;
    bool ok = true;
    pdl_wait();  // T comes from the kernel before
    uint4 v[8];  // the pieces of the row's first chunk; with ranks up to 64 it has no other
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = make_uint4(0, 0, 0, 0);
      if (col0 >= 0 && e >= at && e < at + pieces) v[e] = src[e - at];
    }
    for (long long g = g_end; ok && g > g_begin;) {
      const Piece q = piece(g);
      it += max(0, min(q.kb1, f.n_kb) - q.kb0);
      for (int kb = max(q.kb0, f.n_kb); kb < q.kb1; ++kb, ++it) {
        const int st = it % f.stages;
        const int beyond = sh.list[kb - f.n_kb] - max(col0, 0) / 64;  // the chunk, counted from the row's first
        const bool mine = col0 >= 0 && beyond >= 0 && (beyond == 0 || 64 * beyond < ad.rank);
        if (ad.rank > 64) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (mine) v[e] = src[8 * beyond + e];
        }
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kLE + st), (free_par >> st) & 1u, ctx, kStatusTimeoutKV)))) break;
        free_par ^= 1u << st;
        if (row < f.m_pad) {
          const uint32_t dst = sbase + st * stage_bytes + kTileBytes + 128u * uint32_t(row);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            st_shared_u4(dst + (uint32_t(e ^ (row & 7)) << 4), mine ? v[e] : make_uint4(0, 0, 0, 0));
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(kLF + st));
      }
    }
  }
  pdl_wait();  // this grid has not finished before the one that it overlaps with
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// Four neighbouring columns of a row a thread: the pieces in ascending order, rounded once.
__device__ __forceinline__ float4 sum_pieces(const Stream& s, int per_tile, int per_cta, int row, int n) {
  const int tile = n / 128;
  const int count = last_cta(tile, per_tile, per_cta) - first_cta(tile, per_tile, per_cta) + 1;
  const float* at = s.part + row * s.columns + n;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int q = 0; q < count; ++q) {
    const float4 v = *reinterpret_cast<const float4*>(at + (long long)q * s.f.m * s.columns);
    y.x += v.x;
    y.y += v.y;
    y.z += v.z;
    y.w += v.w;
  }
  return y;
}

constexpr int kFinishThreads = 256;

__global__ void __launch_bounds__(kFinishThreads)
    finish_kernel(const Stream s, __nv_bfloat16* c, long long ldc, int n_out, int swiglu) {
  pdl_wait();
  if (*reinterpret_cast<volatile int*>(s.f.status) != 0) return;
  const int per_tile = s.head[0], per_cta = s.head[1];
  const int row = blockIdx.y, n = 4 * (blockIdx.x * kFinishThreads + threadIdx.x);
  if (n >= n_out) return;
  float4 y = sum_pieces(s, per_tile, per_cta, row, n);
  if (swiglu) {
    // out = bf16(bf16(silu(g)) * u), g and u the bf16-rounded gate / up projections
    const float4 u = sum_pieces(s, per_tile, per_cta, row, n_out + n);
    auto gate = [](float g, float up) {
      g = bf16_round(g);
      return bf16_round(g / (1.0f + __expf(-g))) * bf16_round(up);
    };
    y = make_float4(gate(y.x, u.x), gate(y.y, u.y), gate(y.z, u.z), gate(y.w, u.w));
  }
  *reinterpret_cast<uint2*>(c + (long long)row * ldc + n) = make_uint2(pack_bf16x2(y.x, y.y), pack_bf16x2(y.z, y.w));
}

// ---------------------------------------------------------------- host
struct Layout {
  bool few;
  int64_t low_bytes, list_bytes, part_bytes;  // T; chunk lists (tile path) or the two counts (row path); pieces
  int chunk_stride;
  Stream s;
  int ctas, a_tiles;
  int64_t bytes() const { return low_bytes + list_bytes + part_bytes; }
};

static int check_adapters(int64_t rank, int64_t n_adapters) {
  if (n_adapters < 1 || rank < 8 || rank > kMaxRank || (rank < 64 ? 64 % rank : rank % 64)) return H3_ERR_SHAPE;
  return n_adapters * rank > 64ll * kMaxChunks ? H3_ERR_SHAPE : H3_OK;
}

// CTAs of stream_kernel: two per SM, four k-blocks each at least (a CTA's piece costs its write and its read).
static int stream_ctas(int tiles, int64_t n_kb, int sms) {
  return (int)std::max<int64_t>(1, std::min<int64_t>(2 * sms, tiles * n_kb / 4));
}
// Pieces of a tile that the workspace holds, whatever the chunks in use add.
static int64_t most_pieces(int tiles, int ctas) { return (ctas + tiles - 1) / tiles + 2; }

static int make_layout(int64_t m, int64_t n_kb, int64_t kc_blocks, int64_t w_rows, int64_t rank, int64_t n_adapters,
                       bool tiles, Layout& l) {
  l = {};
  const int64_t stacked = rank * n_adapters;
  l.few = !tiles && m <= kFewRows;
  l.low_bytes = (m * rank * 2 + 255) / 256 * 256;
  if (!l.few) {
    l.chunk_stride = 1 + (int)((stacked + 63) / 64);
    l.list_bytes = (m + 255) / 256 * l.chunk_stride * (int64_t)sizeof(int);
    return H3_OK;
  }
  int sms = 0, rc;
  if ((rc = sm_count(sms)) != H3_OK) return rc;
  Stream& s = l.s;
  s.f.m = (int)m;
  s.f.m_pad = (int)((m + 15) / 16 * 16);
  s.f.n_kb = (int)n_kb;
  s.f.kc_blocks = (int)kc_blocks;
  s.f.stages = std::min<int>(kRing, kRingBytes / (kTileBytes + s.f.m_pad * 128));
  s.tiles = (int)((w_rows + 127) / 128);
  s.columns = 128ll * s.tiles;
  l.a_tiles = (int)((stacked + 127) / 128);
  l.ctas = stream_ctas(s.tiles, n_kb, sms);
  l.list_bytes = 256;
  l.part_bytes = most_pieces(s.tiles, l.ctas) * m * s.columns * (int64_t)sizeof(float);
  return H3_OK;
}

// Launch in clusters of `cluster` CTAs along x.
template <typename... P, typename... A>
static int launch_cluster(void (*kern)(P...), dim3 grid, int cluster, int threads, size_t smem, cudaStream_t st,
                          A... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) return H3_ERR_LAUNCH;
  return cudaGetLastError() == cudaSuccess ? H3_OK : H3_ERR_LAUNCH;
}

template <typename K>
static int allow_smem(K* kern, uint32_t bytes) {
  return cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) == cudaSuccess
             ? H3_OK
             : H3_ERR_LAUNCH;
}

}  // namespace lora
}  // namespace h3

using namespace h3;
using namespace h3::lora;

extern "C" int64_t h3_gemm_adapters_workspace(int64_t m, int64_t a_chunks, int64_t a_chunk_cols, int64_t n_out,
                                              int32_t epilogue, int64_t rank, int64_t n_adapters) {
  int rc;
  const bool tiles = (epilogue & H3_GEMM_ROW_INDEPENDENT) != 0;
  epilogue &= ~H3_GEMM_ROW_INDEPENDENT;
  if (m < 1 || m > (1ll << 31) - 256 || a_chunks < 1 || a_chunks > 65535 || a_chunk_cols < 8 || n_out < 8 ||
      a_chunk_cols > (1ll << 24) || a_chunk_cols * a_chunks > (1ll << 24) || n_out > (1ll << 30) ||
      (epilogue != 0 && epilogue != 1) || 2 * n_out * a_chunk_cols * a_chunks > (1ll << 41))
    return H3_ERR_SHAPE;
  if ((rc = check_adapters(rank, n_adapters)) != H3_OK) return rc;
  Layout l;
  const int64_t kc = (a_chunk_cols + 63) / 64;
  if ((rc = make_layout(m, kc * a_chunks, kc, epilogue == 1 ? 2 * n_out : n_out, rank, n_adapters, tiles, l)) != H3_OK)
    return rc;
  return l.bytes();
}

extern "C" int64_t h3_adapters_deal_kat(int64_t w_rows, int64_t n_kb, int64_t chunks, int32_t sms, int32_t* pieces,
                                        int64_t max_pieces, int64_t* tile_pieces) {
  if (!pieces || !tile_pieces) return H3_ERR_NULL;
  if (w_rows < 1 || w_rows > (1ll << 31) || n_kb < 1 || n_kb > (1ll << 21) || chunks < 0 || chunks > kFewChunks || sms < 1)
    return H3_ERR_SHAPE;
  const int tiles = (int)((w_rows + 127) / 128), per_tile = (int)(n_kb + chunks), ctas = stream_ctas(tiles, n_kb, sms);
  *tile_pieces = most_pieces(tiles, ctas);
  int64_t n = 0;
  for (int c = 0; c < ctas; ++c) {
    const Share share = share_of(tiles, per_tile, c, ctas);
    for (long long g = share.end; g > share.begin; ++n) {
      if (n >= max_pieces) return H3_ERR_WORKSPACE;
      const Piece q = piece_of(share, per_tile, g);
      const int first = first_cta(q.tile, per_tile, share.per_cta), last = last_cta(q.tile, per_tile, share.per_cta);
      const int32_t row[6] = {c, q.tile, q.kb0, q.kb1, c - first, last - first + 1};
      std::copy(row, row + 6, pieces + 6 * n);
    }
  }
  return n;
}

extern "C" int h3_gemm_adapters(const void* a, int64_t m, int64_t a_chunks, int64_t a_chunk_cols,
                                int64_t a_chunk_stride, int64_t a_row_stride, const void* w, int64_t n_out,
                                int64_t w_row_stride, const void* lora_a, int64_t lora_a_row_stride,
                                const void* lora_b, int64_t lora_b_row_stride, int64_t rank, int64_t n_adapters,
                                const float* scale, const int32_t* row_adapter, void* c, int64_t c_row_stride,
                                int32_t epilogue, void* workspace, int64_t ws_bytes, int32_t* status, void* stream) {
  const bool tiles = (epilogue & H3_GEMM_ROW_INDEPENDENT) != 0;
  epilogue &= ~H3_GEMM_ROW_INDEPENDENT;
  const Call call = {a, m, a_chunks, a_chunk_cols, a_chunk_stride, a_row_stride, w, n_out, w_row_stride, c,
                     c_row_stride, epilogue, status};
  int rc;
  if ((rc = check_call(call)) != H3_OK) return rc;
  if (!lora_a || !lora_b || !scale || !row_adapter || !workspace) return H3_ERR_NULL;
  if (!aligned16(lora_a) || !aligned16(lora_b) || !aligned16(workspace) || (reinterpret_cast<uintptr_t>(scale) & 3u) ||
      (reinterpret_cast<uintptr_t>(row_adapter) & 3u))
    return H3_ERR_ALIGN;
  if (n_out > (1ll << 30) || call.w_rows() * call.k() > (1ll << 40)) return H3_ERR_SHAPE;
  if ((rc = check_adapters(rank, n_adapters)) != H3_OK) return rc;
  const int64_t stacked = rank * n_adapters, k = call.k(), w_rows = call.w_rows();
  if (lora_a_row_stride % 8 || lora_a_row_stride < k || lora_b_row_stride % 8 || lora_b_row_stride < stacked)
    return H3_ERR_STRIDE;
  Params p = call_params(call);
  Layout l;
  if ((rc = make_layout(m, p.n_kb, p.kc_blocks, w_rows, rank, n_adapters, tiles, l)) != H3_OK) return rc;
  if (ws_bytes < l.bytes()) return H3_ERR_WORKSPACE;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Adapters ad = {row_adapter, scale, (int)n_adapters, (int)rank};
  CUtensorMap tx, tw, ta, tb;
  if ((rc = map_w(&tw, call)) != H3_OK) return rc;
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  __nv_bfloat16* low = reinterpret_cast<__nv_bfloat16*>(ws);
  if ((rc = make_map(&tb, lora_b, stacked, w_rows, 1, lora_b_row_stride, w_rows * lora_b_row_stride)) != H3_OK) return rc;
  if (l.few) {
    Stream& s = l.s;
    s.f.status = status;
    s.f.low = low;
    s.head = reinterpret_cast<int*>(ws + l.low_bytes);
    s.part = reinterpret_cast<float*>(ws + l.low_bytes + l.list_bytes);
    if ((rc = map_a(&tx, call, (unsigned)s.f.m_pad)) != H3_OK) return rc;
    if ((rc = make_map(&ta, lora_a, k, stacked, 1, lora_a_row_stride, stacked * lora_a_row_stride)) != H3_OK) return rc;
    if ((rc = allow_smem(few_lower_kernel, kFewLowerSmem)) != H3_OK) return rc;
    if ((rc = launch_cluster(few_lower_kernel, dim3((unsigned)(l.a_tiles * kSplitK)), kSplitK, 192, kFewLowerSmem, st, ta,
                             tx, ad, s.f)) != H3_OK)
      return rc;
    if ((rc = allow_smem(stream_kernel, kStreamSmem)) != H3_OK) return rc;
    if ((rc = launch_dependent(stream_kernel, dim3((unsigned)l.ctas), kStreamThreads, kStreamSmem, st, tw, tx, tb, ad,
                               s)) != H3_OK)
      return rc;
    const dim3 grid((unsigned)((n_out / 4 + kFinishThreads - 1) / kFinishThreads), (unsigned)m);
    return launch_dependent(finish_kernel, grid, kFinishThreads, 0, st, s, reinterpret_cast<__nv_bfloat16*>(c),
                            (long long)c_row_stride, (int)n_out, (int)epilogue);
  }
  if ((rc = map_a(&tx, call)) != H3_OK) return rc;
  if ((rc = make_map(&ta, lora_a, k, stacked, 1, lora_a_row_stride, stacked * lora_a_row_stride, 64)) != H3_OK) return rc;
  int* chunks = reinterpret_cast<int*>(ws + l.low_bytes);
  int sms = 0;
  if ((rc = sm_count(sms)) != H3_OK) return rc;
  // a cluster per tile of rows while their CTAs fit the SMs at once (see kQuarters)
  const int64_t row_tiles = (m + 127) / 128;
  const int cluster = row_tiles * kQuarters <= sms ? kQuarters : 1;
  auto* lower = cluster > 1 ? lower_kernel<kQuarters> : lower_kernel<1>;
  if ((rc = allow_smem(lower, kLowerSmem)) != H3_OK) return rc;
  if ((rc = launch_cluster(lower, dim3((unsigned)(row_tiles * cluster)), cluster, 192, kLowerSmem, st, tx, ta, ad, low,
                           chunks, l.chunk_stride, (int)m, p.n_kb, p.kc_blocks, status)) != H3_OK)
    return rc;
  p.low = low;
  p.row_adapter = row_adapter;
  p.chunks = chunks;
  p.chunk_stride = l.chunk_stride;
  p.rank = (int)rank;
  p.n_adapters = (int)n_adapters;
  constexpr uint32_t smem = smem_bytes(kNumBarsAdapters);
  if ((rc = allow_smem(adapter_gemm_kernel, smem)) != H3_OK) return rc;
  const int clusters = std::max(1, std::min(p.n_tiles, sms / 2));
  return launch_dependent(adapter_gemm_kernel, dim3(2 * clusters), kAdapterThreads, smem, st, tx, tw, tb, p);
}
