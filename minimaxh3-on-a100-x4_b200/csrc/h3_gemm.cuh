// The projection GEMM's tiles (see h3_gemm.cu), shared by the plain kernel and the one with low-rank
// adapters: ring and barrier layout, the kernel's body, argument checks and tensor maps.
#pragma once
#include "h3_rows.cuh"
#include "h3attn.h"

namespace h3 {
namespace gemm {

constexpr int kThreads = 192;  // warp 0 TMA producer, warp 1 TMEM allocator + MMA issuer, warps 2..5 epilogue
constexpr int kStages = 6;
constexpr uint32_t kTileBytes = 128u * 64u * 2u;  // 128 rows x 64 bf16 (one SW128 block)
constexpr uint32_t kStageBytes = 2 * kTileBytes;  // A tile + W tile
constexpr uint32_t kOffBars = kStages * kStageBytes;
// Every tcgen05.commit drains the tensor pipe (~100 clk), against 512 clk of MMA work per k-block,
// so ring stages are released kRelEvery k-blocks at a time: release e (one commit, reaching both
// CTAs) frees the stages of k-blocks [kRelEvery e, kRelEvery e + kRelEvery). The producer waits
// release (it - kStages) / kRelEvery before reusing a stage; release barriers are used round
// robin, and with kRel > (kStages - 1) / kRelEvery every parity wait stays within one phase.
constexpr int kRelEvery = 2;
constexpr int kRel = 3;
static_assert(kRel * kRelEvery > kStages - 1, "release barriers too few for the ring");
enum : int {
  kFull = 0,                      // leader: both CTAs' A and W tiles of a stage landed
  kRelease = kFull + kStages,     // both: k-block group consumed (multicast commit), round robin
  kAccFull = kRelease + kRel,     // both: accumulator b complete (multicast commit)
  kAccEmpty = kAccFull + 2,       // leader: accumulator b drained by the epilogue warps of both CTAs
  kDrain = kAccEmpty + 2,         // leader: every issued MMA retired
  kNumBars = kDrain + 1,
  // with adapters, per ring stage:
  kLowFree = kNumBars,              // both: the stage may be filled with adapter rows (arrived on by the producer)
  kLowFull = kLowFree + kStages,    // leader: the adapter rows of both CTAs are in place
  kNumBarsAdapters = kLowFull + kStages
};
constexpr uint32_t smem_bytes(int n_bars) { return 1024 + kOffBars + n_bars * 8 + 16; }
constexpr int kLowWarps = 4;  // with adapters: warps 6..9 of each CTA write the adapter rows

struct Params {
  int m, n_out, n_kb, kc_blocks;  // k-block kb reads A chunk kb / kc_blocks at column 64 * (kb % kc_blocks)
  int n_m, n_n, n_tiles;
  int swiglu, f;                  // swiglu: CTA r's W rows start at r * f + 128 * nb
  int group_m;                    // rasterisation: row tiles per group (their A rows stay in L2)
  __nv_bfloat16* c;
  long long ldc;
  int* status;
  // adapters (gemm_body<true>): after the k-blocks of x and W a tile adds, for each 64-column chunk of the stacked
  // adapters that a row of its 256 uses, one k-block of the rows' low[m][rank] (zero outside a row's own adapter)
  // and the chunk's columns of the stacked B
  const __nv_bfloat16* low;
  const int* row_adapter;
  const int* chunks;  // per 256-row block: count, then the chunks in ascending order
  int chunk_stride, rank, n_adapters;
};

__device__ __forceinline__ void tile_coords(const Params& p, int t, int& mb, int& nb) {
  const int per_group = p.group_m * p.n_n;
  const int group = t / per_group;
  const int first_m = group * p.group_m;
  const int gm = min(p.group_m, p.n_m - first_m);
  const int r = t - group * per_group;
  mb = first_m + r % gm;
  nb = r / gm;
}

// One 64-wide k-block: four M=256 N=256 K=16 pair MMAs (descriptors step 32 B along K).
__device__ __forceinline__ void issue_kblock(uint32_t d_tmem, uint32_t a_base, uint32_t b_base, bool accumulate) {
  constexpr uint32_t idesc = idesc_bf16_f32(256, 256, 0, 0);
  const uint64_t ad = smem_desc_sw128(a_base, 16, 1024), bd = smem_desc_sw128(b_base, 16, 1024);
  const uint32_t alo = uint32_t(ad), ahi = uint32_t(ad >> 32), blo = uint32_t(bd), bhi = uint32_t(bd >> 32);
#define H3_GEMM_STEP(O) \
  "add.u32 la, %1, " #O ";\n\t add.u32 lb, %3, " #O ";\n\t" \
  "mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t" \
  "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, pt;\n\t"
  asm volatile(
      "{\n\t.reg .pred pf, pt;\n\t.reg .b32 la, lb;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 pf, %6, 0;\n\t setp.eq.b32 pt, %6, %6;\n\t"
      "mov.b64 da, {%1, %2};\n\t mov.b64 db, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %5, pf;\n\t"
      H3_GEMM_STEP(2) H3_GEMM_STEP(4) H3_GEMM_STEP(6)
      "}\n" ::"r"(d_tmem), "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc), "r"(accumulate ? 1u : 0u)
      : "memory");
#undef H3_GEMM_STEP
}

__device__ __forceinline__ float bf16_round(float x) { return __bfloat162float(__float2bfloat16_rn(x)); }

__device__ __forceinline__ void drain_wait_cluster(uint32_t bar, uint32_t parity, int* status) {
  uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait_acq_cluster(bar, parity)) {
    if (globaltimer_ns() - t0 > H3_WAIT_LIMIT_NS) {
      atomicCAS(status, 0, kStatusTimeoutDrain);
      return;
    }
  }
}

// The kernel's body; kAdapters adds low-rank adapters as extra k-blocks (tmap_b: the stacked B).
template <bool kAdapters>
__device__ __forceinline__ void gemm_body(const CUtensorMap& tmap_a, const CUtensorMap& tmap_w,
                                          const CUtensorMap& tmap_b, const Params& p) {
  constexpr int kBars = kAdapters ? kNumBarsAdapters : kNumBars;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kOffBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int i) { return smem_u32(&bars[i]); };

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cid = blockIdx.x >> 1;
  const int n_clusters = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(bar(kFull + s), 1);
    for (int r = 0; r < kRel; ++r) mbar_init(bar(kRelease + r), 1);
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kAccFull + b), 1);
      mbar_init(bar(kAccEmpty + b), 8);  // 4 epilogue warps in each CTA
    }
    mbar_init(bar(kDrain), 1);
    if constexpr (kAdapters)
      for (int s = 0; s < kStages; ++s) {
        mbar_init(bar(kLowFree + s), 1);
        mbar_init(bar(kLowFull + s), 2 * kLowWarps);
      }
    *abort_flag = (*reinterpret_cast<volatile int*>(p.status) != 0) ? 1 : 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc_pair(smem_u32(tmem_slot), 512);
    tmem_relinquish_pair();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_w);
  }
  tc_fence_before();
  cluster_sync_all();  // barriers and TMEM of both CTAs exist before anything remote touches them
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const WaitCtx ctx{abort_flag, p.status};
  const bool grid_aborted = *abort_flag != 0;

  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer (both CTAs)
    // The whole warp runs the loop and agrees on every wait; one elected lane issues the copies.
    if (!grid_aborted) {
      const bool issuer = elect_one();
      int it = 0;
      bool ok = true;
      for (int t = cid; ok && t < p.n_tiles; t += n_clusters) {
        int mb, nb;
        tile_coords(p, t, mb, nb);
        const int a_row = mb * 256 + 128 * int(rank);
        const int w_row = p.swiglu ? int(rank) * p.f + 128 * nb : nb * 256 + 128 * int(rank);
        for (int kb = 0; kb < p.n_kb; ++kb, ++it) {
          const int st = it % kStages;
          if (it >= kStages) {
            const int e = (it - kStages) / kRelEvery;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kRelease + e % kRel), uint32_t(e / kRel) & 1u, ctx,
                                                        kStatusTimeoutKV))))
              break;
          }
          if (issuer) {
            if (rank == 0) mbar_expect_tx(bar(kFull + st), 2 * kStageBytes);
            const uint32_t full_leader = mapa_shared(bar(kFull + st), 0);
            const uint32_t dst = sbase + st * kStageBytes;
            tma_load_3d_pair(dst, &tmap_a, full_leader, 64 * (kb % p.kc_blocks), a_row, kb / p.kc_blocks);
            tma_load_3d_pair(dst + kTileBytes, &tmap_w, full_leader, 64 * kb, w_row, 0);
          }
          __syncwarp();
        }
        if constexpr (kAdapters) {
          if (t == cid) pdl_wait();  // the chunk lists and low rows come from the kernel before
          const int* list = p.chunks + (long long)mb * p.chunk_stride;
          const int cnt = ok ? list[0] : 0;
          int ids = 0;  // of 32 chunks, one a lane
          for (int i = 0; i < cnt; ++i, ++it) {
            if ((i & 31) == 0) ids = i + lane < cnt ? list[1 + i + lane] : 0;
            const int chunk = __shfl_sync(0xffffffffu, ids, i & 31);
            const int st = it % kStages;
            if (it >= kStages) {
              const int e = (it - kStages) / kRelEvery;
              if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kRelease + e % kRel), uint32_t(e / kRel) & 1u, ctx,
                                                          kStatusTimeoutKV))))
                break;
            }
            if (issuer) {
              mbar_arrive(bar(kLowFree + st));
              if (rank == 0) mbar_expect_tx(bar(kFull + st), 2 * kTileBytes);
              tma_load_3d_pair(sbase + st * kStageBytes + kTileBytes, &tmap_b, mapa_shared(bar(kFull + st), 0),
                               64 * chunk, w_row, 0);
            }
            __syncwarp();
          }
        }
      }
      if (rank == 0 && issuer) {
        // every copy of both CTAs counts on the leader's barriers: drain them before exit
        for (int st = 0; st < kStages; ++st) {
          const int cnt = it / kStages + (st < it % kStages ? 1 : 0);
          if (cnt > 0) drain_wait_cluster(bar(kFull + st), uint32_t(cnt - 1) & 1u, p.status);
        }
      }
      __syncwarp();
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (leader CTA)
    // The whole warp runs the loop and agrees on every wait; one elected lane issues the MMAs and
    // commits (a lane-0-only issuer falls behind when other warps issue at full rate).
    if (rank == 0 && !grid_aborted) {
      const bool issuer = elect_one();
      int it = 0, i = 0;
      [[maybe_unused]] uint32_t low_par = 0;  // bit st: parity of the stage's next adapter use
      bool ok = true;
      for (int t = cid; ok && t < p.n_tiles; t += n_clusters, ++i) {
        const int b = i & 1;
        // accumulator b is free once the epilogue drained the tile that used it two tiles ago
        if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar(kAccEmpty + b), (uint32_t(i >> 1) & 1u) ^ 1u, ctx,
                                                             kStatusTimeoutO))))
          break;
        tc_fence_after();
        const uint32_t d = tmem + 256u * b;
        for (int kb = 0; kb < p.n_kb; ++kb, ++it) {
          const int st = it % kStages;
          if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar(kFull + st), uint32_t(it / kStages) & 1u, ctx,
                                                               kStatusTimeoutKV))))
            break;
          tc_fence_after();
          const uint32_t a_base = sbase + st * kStageBytes;
          if (issuer) {
            issue_kblock(d, a_base, a_base + kTileBytes, kb > 0);
            if (it % kRelEvery == kRelEvery - 1) mma_commit_pair(bar(kRelease + (it / kRelEvery) % kRel), 0x3);
          }
          __syncwarp();
        }
        if constexpr (kAdapters) {
          if (t == cid) pdl_wait();
          int mb, nb;
          tile_coords(p, t, mb, nb);
          const int cnt = ok ? p.chunks[(long long)mb * p.chunk_stride] : 0;
          for (int l = 0; l < cnt; ++l, ++it) {
            const int st = it % kStages;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar(kFull + st), uint32_t(it / kStages) & 1u, ctx,
                                                                 kStatusTimeoutKV))))
              break;
            if (!(ok = __all_sync(0xffffffffu, mbar_wait_cluster(bar(kLowFull + st), (low_par >> st) & 1u, ctx,
                                                                 kStatusTimeoutKV))))
              break;
            low_par ^= 1u << st;
            tc_fence_after();
            const uint32_t a_base = sbase + st * kStageBytes;
            if (issuer) {
              issue_kblock(d, a_base, a_base + kTileBytes, true);
              if (it % kRelEvery == kRelEvery - 1) mma_commit_pair(bar(kRelease + (it / kRelEvery) % kRel), 0x3);
            }
            __syncwarp();
          }
        }
        if (ok && issuer) mma_commit_pair(bar(kAccFull + b), 0x3);
        __syncwarp();
      }
      if (issuer) {
        mma_commit_pair(bar(kDrain), 0x1);
        drain_wait_cluster(bar(kDrain), 0, p.status);
      }
      __syncwarp();
    }
  } else if (!kAdapters || warp < 6) {
    // ------------------------------------------------------------ epilogue (warps 2..5, both CTAs)
    const int quad = warp & 3;  // TMEM lane quarter this warp may access
    const uint32_t lane_off = uint32_t(quad * 32) << 16;
    bool ok = !grid_aborted;
    int i = 0;
    for (int t = cid; ok && t < p.n_tiles; t += n_clusters, ++i) {
      const int b = i & 1;
      int mb, nb;
      tile_coords(p, t, mb, nb);
      ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccFull + b), uint32_t(i >> 1) & 1u, ctx, kStatusTimeoutS));
      if (!ok) break;
      tc_fence_after();
      const int row = mb * 256 + 128 * int(rank) + quad * 32 + lane;
      const bool valid = row < p.m;
      const uint32_t acc = tmem + lane_off + 256u * b;
      if (!p.swiglu) {
        const int n0 = nb * 256;
        __nv_bfloat16* dst = p.c + (long long)(valid ? row : 0) * p.ldc + n0;
#pragma unroll 1
        for (int c32 = 0; c32 < 8; ++c32) {
          uint32_t r[32];
          tmem_ld32_wait(acc + 32 * c32, r);
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) w[e] = pack_bf16x2(__uint_as_float(r[2 * e]), __uint_as_float(r[2 * e + 1]));
          if (valid) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (n0 + 32 * c32 + 8 * q < p.n_out)
                *reinterpret_cast<uint4*>(dst + 32 * c32 + 8 * q) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2],
                                                                                w[4 * q + 3]);
          }
          __syncwarp();  // the next load of the accumulators takes the whole warp
        }
      } else {
        // out = bf16(bf16(silu(g)) * u), g and u the bf16-rounded gate / up projections
        const int n0 = nb * 128;
        __nv_bfloat16* dst = p.c + (long long)(valid ? row : 0) * p.ldc + n0;
#pragma unroll 1
        for (int c32 = 0; c32 < 4; ++c32) {
          uint32_t g[32], u[32];
          tmem_ld32_wait(acc + 32 * c32, g);
          tmem_ld32_wait(acc + 128 + 32 * c32, u);
          uint32_t w[16];
#pragma unroll
          for (int e = 0; e < 16; ++e) {
            float v[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float gx = bf16_round(__uint_as_float(g[2 * e + h]));
              const float ux = bf16_round(__uint_as_float(u[2 * e + h]));
              const float sx = bf16_round(gx / (1.0f + __expf(-gx)));
              v[h] = sx * ux;
            }
            w[e] = pack_bf16x2(v[0], v[1]);
          }
          if (valid) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<uint4*>(dst + 32 * c32 + 8 * q) = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2],
                                                                              w[4 * q + 3]);
          }
          __syncwarp();
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_remote(mapa_shared(bar(kAccEmpty + b), 0));
    }
  } else if constexpr (kAdapters) {
    // ------------------------------------------------------------ adapter rows (warps 6..9, both CTAs)
    // One thread per A row: the row's share of a chunk's 64 columns, written K-major with the 128-byte swizzle
    // (16-byte piece c of row r at c ^ (r & 7)), as the TMA writes the tiles of x.
    bool ok = !grid_aborted;
    int it = 0;
    uint32_t free_par = 0;
    const int r_in = (warp - 6) * 32 + lane;
    const int pieces = min(p.rank, 64) / 8;
    pdl_wait();
    for (int t = cid; ok && t < p.n_tiles; t += n_clusters) {
      int mb, nb;
      tile_coords(p, t, mb, nb);
      it += p.n_kb;
      const int* list = p.chunks + (long long)mb * p.chunk_stride;
      const int cnt = list[0];
      if (cnt == 0) continue;
      const int row = mb * 256 + 128 * int(rank) + r_in;
      const int ad = row < p.m ? p.row_adapter[row] : -1;
      const int col0 = ad >= 0 && ad < p.n_adapters ? ad * p.rank : -1;  // first stacked column of the row's adapter
      const uint4* src = reinterpret_cast<const uint4*>(p.low + (long long)row * p.rank);
      const int at = (max(col0, 0) & 63) / 8;  // the row's pieces of 8 columns in its (first) chunk: [at, at + pieces)
      int held = col0 >= 0 ? col0 / 64 : -1;   // the chunk whose pieces v holds, loaded before they are needed
      uint4 v[8];
      auto hold = [&] {
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          v[q] = make_uint4(0, 0, 0, 0);
          if (held >= 0 && q >= at && q < at + pieces) v[q] = src[8 * (held - col0 / 64) + q - at];
        }
      };
      hold();
      int ids = 0;  // of 32 chunks, one a lane
      for (int l = 0; l < cnt; ++l, ++it) {
        if ((l & 31) == 0) ids = l + lane < cnt ? list[1 + l + lane] : 0;
        const int st = it % kStages;
        const bool mine = __shfl_sync(0xffffffffu, ids, l & 31) == held;
        if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kLowFree + st), (free_par >> st) & 1u, ctx, kStatusTimeoutKV))))
          break;
        free_par ^= 1u << st;
        const uint32_t dst = sbase + st * kStageBytes + 128u * uint32_t(r_in);
#pragma unroll
        for (int q = 0; q < 8; ++q)
          st_shared_u4(dst + (uint32_t(q ^ (r_in & 7)) << 4), mine ? v[q] : make_uint4(0, 0, 0, 0));
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive_remote_release(mapa_shared(bar(kLowFull + st), 0));
        if (mine && 64 * (held + 1) < col0 + p.rank) {  // ranks above 64: the row's next chunk
          ++held;
          hold();
        }
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // the leader's MMAs into this CTA's TMEM have retired; nothing remote is pending
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------- host
// [outer][rows][inner] bf16 with element strides; box 64 x box_rows x 1, SW128, zero fill out of range.
inline int make_map(CUtensorMap* map, const void* base, long long inner, long long rows, long long outer,
                    long long row_stride, long long outer_stride, unsigned box_rows = 128) {
  const EncodeTiledFn enc = get_encode_fn();
  if (!enc) return H3_ERR_DRIVER;
  cuuint64_t dims[3] = {(cuuint64_t)inner, (cuuint64_t)rows, (cuuint64_t)outer};
  cuuint64_t strides[2] = {(cuuint64_t)row_stride * 2, (cuuint64_t)outer_stride * 2};
  cuuint32_t box[3] = {64, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(
      map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? H3_OK : H3_ERR_TENSOR_MAP;
}


// A projection call's arguments, their checks, and the fields of Params that do not depend on adapters.
struct Call {
  const void* a;
  int64_t m, a_chunks, a_chunk_cols, a_chunk_stride, a_row_stride;
  const void* w;
  int64_t n_out, w_row_stride;
  void* c;
  int64_t c_row_stride;
  int32_t epilogue;
  int32_t* status;
  int64_t k() const { return a_chunk_cols * a_chunks; }
  int64_t w_rows() const { return epilogue == 1 ? 2 * n_out : n_out; }
};

inline int check_call(const Call& q) {
  if (!q.a || !q.w || !q.c || !q.status) return H3_ERR_NULL;
  if (!aligned16(q.a) || !aligned16(q.w) || !aligned16(q.c)) return H3_ERR_ALIGN;
  if (q.m < 1 || q.a_chunks < 1 || q.a_chunk_cols < 8 || q.n_out < 8 || (q.epilogue != 0 && q.epilogue != 1))
    return H3_ERR_SHAPE;
  if (q.m > (1ll << 31) - 256 || q.a_chunks > 65535 || q.a_chunk_cols * q.a_chunks > (1ll << 24)) return H3_ERR_SHAPE;
  if (q.a_chunk_cols % 8 || (q.a_chunks > 1 && q.a_chunk_cols % 64) || q.n_out % 8) return H3_ERR_SHAPE;
  if (q.epilogue == 1 && q.n_out % 128) return H3_ERR_SHAPE;
  if (q.a_row_stride % 8 || q.a_row_stride < q.a_chunk_cols || q.w_row_stride % 8 || q.c_row_stride % 8 ||
      q.w_row_stride < q.k() || q.c_row_stride < q.n_out)
    return H3_ERR_STRIDE;
  if (q.a_chunks > 1 && (q.a_chunk_stride % 8 || q.a_chunk_stride < q.m * q.a_row_stride)) return H3_ERR_STRIDE;
  return H3_OK;
}

inline int map_a(CUtensorMap* map, const Call& q, unsigned box_rows = 128) {
  return make_map(map, q.a, q.a_chunk_cols, q.m, q.a_chunks, q.a_row_stride,
                  q.a_chunks > 1 ? q.a_chunk_stride : q.m * q.a_row_stride, box_rows);
}
inline int map_w(CUtensorMap* map, const Call& q) {
  return make_map(map, q.w, q.k(), q.w_rows(), 1, q.w_row_stride, q.w_rows() * q.w_row_stride);
}

inline Params call_params(const Call& q) {
  Params p = {};
  p.m = (int)q.m;
  p.n_out = (int)q.n_out;
  p.kc_blocks = (int)((q.a_chunk_cols + 63) / 64);
  p.n_kb = p.kc_blocks * (int)q.a_chunks;
  p.n_m = (int)((q.m + 255) / 256);
  p.n_n = q.epilogue == 1 ? (int)(q.n_out / 128) : (int)((q.n_out + 255) / 256);
  p.n_tiles = p.n_m * p.n_n;
  p.swiglu = q.epilogue;
  p.f = (int)q.n_out;
  p.c = reinterpret_cast<__nv_bfloat16*>(q.c);
  p.ldc = q.c_row_stride;
  p.status = q.status;
  // Consecutive tiles walk every column tile of a group of 16 row tiles: the group's A rows are
  // reused from L2 while W streams past, and W is read from DRAM once per group. Under the power
  // cap less DRAM traffic means a higher clock: at M=42000, groups of 16 run the qkv / fc1 / fc2
  // shapes 5-11 % faster than groups of 8 (4 and 24 are slower; column-major groups are equal).
  p.group_m = 16;
  return p;
}

inline int sm_count(int& sms) {
  int dev = 0;
  return cudaGetDevice(&dev) == cudaSuccess &&
                 cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess
             ? H3_OK
             : H3_ERR_CUDA;
}

}  // namespace gemm
}  // namespace h3
