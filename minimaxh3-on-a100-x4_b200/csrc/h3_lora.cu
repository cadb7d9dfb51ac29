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
// Few rows (row path, two launches): bound by reading W once. stream_kernel: W and the stacked A are the M = 128
// operand, the rows of x (16 .. 64 of them) the N operand; all their k-blocks, tile after tile, are dealt out
// evenly to two CTAs per SM, and each CTA writes fp32 sums of the piece of a tile that it had. finish_kernel adds a
// column's pieces in a fixed order, then s_a B_a T with T in fp32, rounds and stores. Adapter tiles that no
// row uses are neither read nor written.
//
// A row's value does not depend on the other rows of a call in either path (the paths differ in summation order).
#include <algorithm>

#include "h3_gemm.cuh"

namespace h3 {
namespace lora {

using namespace h3::gemm;

constexpr int kMaxRank = 256;
constexpr int kMaxChunks = 1024;  // n_adapters * rank <= 65536
constexpr int kFewRows = 64;      // row path up to here

struct Adapters {
  const int* row_adapter;
  const float* scale;
  int n_adapters, rank, n_chunks;
};
// the adapter of row r, or -1
__device__ __forceinline__ int adapter_of(const Adapters& ad, int m, int r) {
  const int a = r < m ? ad.row_adapter[r] : -1;
  return a >= 0 && a < ad.n_adapters ? a : -1;
}

// ---------------------------------------------------------------- tile path: T = s A x
constexpr int kLowerStages = 3;
constexpr int kPass = 2;  // chunks per pass over k: 16 KB of x and 2 x 8 KB of A per stage, two CTAs per SM
constexpr uint32_t kChunkBytes = 64u * 64u * 2u;
constexpr uint32_t kLowerStage = kTileBytes + kPass * kChunkBytes;
struct LowerSmem {
  uint32_t own[kMaxChunks / 32], both[kMaxChunks / 32];  // chunks in use: these 128 rows, the block of 256
  uint16_t list[kMaxChunks];
  int count;
  uint64_t bars[2 * kLowerStages + 5];
  uint32_t tmem;
  int abort;
};
constexpr uint32_t kLowerSmem = 1024 + kLowerStages * kLowerStage + sizeof(LowerSmem);

__global__ void __launch_bounds__(192, 2)
    lower_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_a,
                 const Adapters ad, __nv_bfloat16* low, int* chunks, int chunk_stride, int m, int n_kb, int kc_blocks,
                 int* status) {
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  LowerSmem& sh = *reinterpret_cast<LowerSmem*>(smem + kLowerStages * kLowerStage);
  enum { kF = 0, kE = kLowerStages, kAccF = 2 * kLowerStages, kAccE = kAccF + 2, kD = kAccE + 2 };
  auto bar = [&](int i) { return smem_u32(&sh.bars[i]); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int m0 = blockIdx.x * 128;

  for (int i = threadIdx.x; i < kMaxChunks / 32; i += 192) sh.own[i] = sh.both[i] = 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kLowerStages; ++s) {
      mbar_init(bar(kF + s), 1);
      mbar_init(bar(kE + s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kAccF + b), 1);
      mbar_init(bar(kAccE + b), 4);
    }
    mbar_init(bar(kD), 1);
    sh.abort = *reinterpret_cast<volatile int*>(status) != 0 ? 1 : 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sh.tmem), 256);
    tmem_relinquish();
  }
  __syncthreads();
  // chunks in use by the 256-row block, and by this tile's 128 rows of it
  for (int r = threadIdx.x; r < 256; r += 192) {
    const int row = (m0 & ~255) + r;
    const int a = adapter_of(ad, m, row);
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
  if (warp == 2 || (warp == 3 && (blockIdx.x & 1) == 0)) {
    // ascending lists: this tile's in shared memory, the block's (its first tile writes it) in global memory
    const uint32_t word = warp == 2 ? sh.own[lane] : sh.both[lane];
    int at = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += up;
    }
    int* out = chunks + (long long)(blockIdx.x >> 1) * chunk_stride;
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

  if (warp == 0 && run) {
    const bool issuer = elect_one();
    int it = 0;
    bool ok = true;
    for (int ps = 0; ok && ps < passes; ++ps) {
      const int nc = min(kPass, count - ps * kPass);
      for (int kb = 0; kb < n_kb; ++kb, ++it) {
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
    }
    if (issuer)
      for (int st = 0; st < kLowerStages; ++st) {
        const int cnt = it / kLowerStages + (st < it % kLowerStages ? 1 : 0);
        if (cnt > 0) drain_wait_cluster(bar(kF + st), uint32_t(cnt - 1) & 1u, status);
      }
    __syncwarp();
  } else if (warp == 1 && run) {
    const bool issuer = elect_one();
    constexpr uint32_t idesc = idesc_bf16_f32(128, 64, 0, 0);
    int it = 0;
    bool ok = true;
    for (int ps = 0; ok && ps < passes; ++ps) {
      const int b = ps & 1, nc = min(kPass, count - ps * kPass);
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccE + b), (uint32_t(ps >> 1) & 1u) ^ 1u, ctx, kStatusTimeoutO))))
        break;
      tc_fence_after();
      for (int kb = 0; kb < n_kb; ++kb, ++it) {
        const int st = it % kLowerStages;
        if (!(ok = __all_sync(0xffffffffu,
                              mbar_wait(bar(kF + st), uint32_t(it / kLowerStages) & 1u, ctx, kStatusTimeoutKV))))
          break;
        tc_fence_after();
        if (issuer) {
          const uint32_t x = sbase + st * kLowerStage;
          for (int i = 0; i < nc; ++i)
            for (int ks = 0; ks < 4; ++ks)
              mma_ss(tmem + 128u * b + 64u * i, smem_desc_sw128(x + 32u * ks, 16, 1024),
                     smem_desc_sw128(x + kTileBytes + i * kChunkBytes + 32u * ks, 16, 1024), idesc,
                     kb > 0 || ks > 0 ? 1u : 0u);
          mma_commit(bar(kE + st));
        }
        __syncwarp();
      }
      if (ok && issuer) mma_commit(bar(kAccF + b));
      __syncwarp();
    }
    if (issuer) {
      mma_commit(bar(kD));
      drain_wait_cluster(bar(kD), 0, status);
    }
    __syncwarp();
  } else if (warp >= 2 && run) {
    const int quad = warp & 3;
    const uint32_t lane_off = uint32_t(quad * 32) << 16;
    const int row = m0 + quad * 32 + lane;
    const int a = adapter_of(ad, m, row);
    const float scale = a >= 0 ? ad.scale[a] : 0.f;
    const int lo = a >= 0 ? a * ad.rank : 0, hi = a >= 0 ? lo + ad.rank : 0;  // the row's stacked columns
    bool ok = true;
    for (int ps = 0; ok && ps < passes; ++ps) {
      const int b = ps & 1, nc = min(kPass, count - ps * kPass);
      ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccF + b), uint32_t(ps >> 1) & 1u, ctx, kStatusTimeoutS));
      if (!ok) break;
      tc_fence_after();
      for (int i = 0; i < nc; ++i) {
        const int first = 64 * sh.list[ps * kPass + i];
#pragma unroll 1
        for (int q = 0; q < 4; ++q) {
          uint32_t r[16];
          tmem_ld16_wait(tmem + lane_off + 128u * b + 64u * i + 16u * q, r);
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = first + 16 * q + 8 * h;
            if (col >= lo && col < hi) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e)
                w[e] = pack_bf16x2(__uint_as_float(r[8 * h + 2 * e]) * scale,
                                   __uint_as_float(r[8 * h + 2 * e + 1]) * scale);
              *reinterpret_cast<uint4*>(low + (long long)row * ad.rank + (col - lo)) = make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kAccE + b));
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// ---------------------------------------------------------------- tile path: y = W x + B T
constexpr int kAdapterThreads = kThreads + 32 * kLowWarps;

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kAdapterThreads, 1)
    adapter_gemm_kernel(const __grid_constant__ CUtensorMap tmap_x, const __grid_constant__ CUtensorMap tmap_w,
                        const __grid_constant__ CUtensorMap tmap_b, const Params p) {
  gemm_body<true>(tmap_x, tmap_w, tmap_b, p);
}

// ---------------------------------------------------------------- row path: W and A streamed once
struct Stream {
  int m, m_pad;           // rows, and rows rounded up to 16
  int n_kb, kc_blocks;    // k-blocks of 64
  int w_tiles, a_tiles;   // 128-row tiles of W, of the stacked A
  int per_cta;            // k-blocks per CTA
  int stages;
  float* part;            // [piece][m][columns]: column c of tile t at 128 t + c
  long long columns;      // 128 * (w_tiles + a_tiles)
  int* status;
};
// The CTA that has k-block g of the tile list, and the first of a tile's CTAs: piece = cta - first_cta(tile).
__device__ __forceinline__ int first_cta(const Stream& s, int tile) {
  return int((long long)tile * s.n_kb / s.per_cta);
}
__device__ __forceinline__ int pieces_of(const Stream& s, int tile) {
  return int(((long long)(tile + 1) * s.n_kb - 1) / s.per_cta) - first_cta(s, tile) + 1;
}

constexpr int kMaxStreamStages = 6;
constexpr uint32_t kStreamRing = 6u * (kTileBytes + 16u * 128u);  // 108 KB: two CTAs per SM

struct StreamSmem {
  uint32_t used[kMaxChunks / 2 / 32];  // tiles of the stacked A that a row uses
  uint64_t bars[2 * kMaxStreamStages + 5];
  uint32_t tmem;
  int abort;
};
constexpr uint32_t kStreamSmem = 1024 + kStreamRing + sizeof(StreamSmem);

__global__ void __launch_bounds__(192, 2)
    stream_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_a,
                  const __grid_constant__ CUtensorMap tmap_x, const Adapters ad, const Stream s) {
  pdl_launch_dependents();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sbase = smem_u32(smem);
  StreamSmem& sh = *reinterpret_cast<StreamSmem*>(smem + kStreamRing);
  enum { kF = 0, kE = kMaxStreamStages, kAccF = 2 * kMaxStreamStages, kAccE = kAccF + 2, kD = kAccE + 2 };
  auto bar = [&](int i) { return smem_u32(&sh.bars[i]); };
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t x_bytes = uint32_t(s.m_pad) * 128u, stage_bytes = kTileBytes + x_bytes;
  // two accumulators of m_pad columns
  const uint32_t cols = s.m_pad <= 16 ? 32u : (s.m_pad <= 32 ? 64u : 128u);

  for (int i = threadIdx.x; i < kMaxChunks / 2 / 32; i += 192) sh.used[i] = 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMaxStreamStages; ++i) {
      mbar_init(bar(kF + i), 1);
      mbar_init(bar(kE + i), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar(kAccF + b), 1);
      mbar_init(bar(kAccE + b), 4);
    }
    mbar_init(bar(kD), 1);
    sh.abort = *reinterpret_cast<volatile int*>(s.status) != 0 ? 1 : 0;
    fence_mbar_init();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(&sh.tmem), cols);
    tmem_relinquish();
  }
  __syncthreads();
  if (threadIdx.x < s.m) {
    const int a = adapter_of(ad, s.m, threadIdx.x);
    if (a >= 0) {
      const int last = (a * ad.rank + ad.rank - 1) / 128;
      for (int t = a * ad.rank / 128; t <= last; ++t) atomicOr(&sh.used[t / 32], 1u << (t & 31));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  const WaitCtx ctx{&sh.abort, s.status};
  const bool run = sh.abort == 0;
  const long long total = (long long)(s.w_tiles + s.a_tiles) * s.n_kb;
  const long long g_end = min(total, (long long)(blockIdx.x + 1) * s.per_cta);
  auto skipped = [&](int tile) {
    const int t = tile - s.w_tiles;
    return t >= 0 && !((sh.used[t / 32] >> (t & 31)) & 1u);
  };

  if (warp == 0 && run) {
    const bool issuer = elect_one();
    int it = 0;
    bool ok = true;
    for (long long g = (long long)blockIdx.x * s.per_cta; ok && g < g_end;) {
      const int tile = int(g / s.n_kb), kb0 = int(g - (long long)tile * s.n_kb);
      const int kb1 = int(min((long long)s.n_kb, kb0 + (g_end - g)));
      g += kb1 - kb0;
      if (skipped(tile)) continue;
      const bool is_w = tile < s.w_tiles;
      const int row = 128 * (is_w ? tile : tile - s.w_tiles);
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int st = it % s.stages;
        if (it >= s.stages && !(ok = __all_sync(0xffffffffu, mbar_wait(bar(kE + st), uint32_t(it / s.stages - 1) & 1u,
                                                                       ctx, kStatusTimeoutKV))))
          break;
        if (issuer) {
          const uint32_t dst = sbase + st * stage_bytes;
          mbar_expect_tx(bar(kF + st), stage_bytes);
          tma_load_3d(dst, is_w ? &tmap_w : &tmap_a, bar(kF + st), 64 * kb, row, 0);
          tma_load_3d(dst + kTileBytes, &tmap_x, bar(kF + st), 64 * (kb % s.kc_blocks), 0, kb / s.kc_blocks);
        }
        __syncwarp();
      }
    }
    if (issuer)
      for (int st = 0; st < s.stages; ++st) {
        const int cnt = it / s.stages + (st < it % s.stages ? 1 : 0);
        if (cnt > 0) drain_wait_cluster(bar(kF + st), uint32_t(cnt - 1) & 1u, s.status);
      }
    __syncwarp();
  } else if (warp == 1 && run) {
    const bool issuer = elect_one();
    const uint32_t idesc = idesc_bf16_f32(128, s.m_pad, 0, 0);
    int it = 0, i = 0;
    bool ok = true;
    for (long long g = (long long)blockIdx.x * s.per_cta; ok && g < g_end;) {
      const int tile = int(g / s.n_kb), kb0 = int(g - (long long)tile * s.n_kb);
      const int kb1 = int(min((long long)s.n_kb, kb0 + (g_end - g)));
      g += kb1 - kb0;
      if (skipped(tile)) continue;
      const int b = i & 1;
      if (!(ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccE + b), (uint32_t(i >> 1) & 1u) ^ 1u, ctx, kStatusTimeoutO))))
        break;
      tc_fence_after();
      for (int kb = kb0; kb < kb1; ++kb, ++it) {
        const int st = it % s.stages;
        if (!(ok = __all_sync(0xffffffffu,
                              mbar_wait(bar(kF + st), uint32_t(it / s.stages) & 1u, ctx, kStatusTimeoutKV))))
          break;
        tc_fence_after();
        if (issuer) {
          const uint32_t w = sbase + st * stage_bytes;
          for (int ks = 0; ks < 4; ++ks)
            mma_ss(tmem + uint32_t(b * s.m_pad), smem_desc_sw128(w + 32u * ks, 16, 1024),
                   smem_desc_sw128(w + kTileBytes + 32u * ks, 16, 1024), idesc, kb > kb0 || ks > 0 ? 1u : 0u);
          mma_commit(bar(kE + st));
        }
        __syncwarp();
      }
      if (ok && issuer) mma_commit(bar(kAccF + b));
      __syncwarp();
      ++i;
    }
    if (issuer) {
      mma_commit(bar(kD));
      drain_wait_cluster(bar(kD), 0, s.status);
    }
    __syncwarp();
  } else if (warp >= 2 && run) {
    const int quad = warp & 3;
    const uint32_t lane_off = uint32_t(quad * 32) << 16;
    int i = 0;
    bool ok = true;
    for (long long g = (long long)blockIdx.x * s.per_cta; ok && g < g_end;) {
      const int tile = int(g / s.n_kb), kb0 = int(g - (long long)tile * s.n_kb);
      const int kb1 = int(min((long long)s.n_kb, kb0 + (g_end - g)));
      g += kb1 - kb0;
      if (skipped(tile)) continue;
      const int b = i & 1;
      ok = __all_sync(0xffffffffu, mbar_wait(bar(kAccF + b), uint32_t(i >> 1) & 1u, ctx, kStatusTimeoutS));
      if (!ok) break;
      tc_fence_after();
      // lane = column of the tile: a warp stores 32 consecutive columns of a row
      float* dst = s.part + (long long)(blockIdx.x - first_cta(s, tile)) * s.m * s.columns + 128ll * tile + quad * 32 + lane;
#pragma unroll 1
      for (int q = 0; q < s.m_pad / 16; ++q) {
        uint32_t r[16];
        tmem_ld16_wait(tmem + lane_off + uint32_t(b * s.m_pad + 16 * q), r);
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (16 * q + e < s.m) dst[(16 * q + e) * s.columns] = __uint_as_float(r[e]);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(kAccE + b));
      ++i;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, cols);
  }
}

// One row and 256 columns a CTA, two neighbouring columns a thread: the pieces of W x in ascending order, plus B_a T.
// The first kAhead * 8 columns of B are loaded before the wait for stream_kernel (they do not depend on it).
constexpr int kAhead = 4;

struct Finish {
  const __nv_bfloat16* b;  // stacked B
  long long b_row;
  __nv_bfloat16* c;
  long long ldc;
  int n_out, swiglu;
};

// Columns n and n + 1 of a row.
struct FinishPair {
  uint4 b0[kAhead], b1[kAhead];
  const __nv_bfloat16* from;

  __device__ __forceinline__ void load(const Finish& f, int col0, int rank, int n) {
    from = f.b + n * f.b_row + col0;
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (col0 >= 0 && 8 * q < rank) {
        b0[q] = __ldg(reinterpret_cast<const uint4*>(from + 8 * q));
        b1[q] = __ldg(reinterpret_cast<const uint4*>(from + f.b_row + 8 * q));
      }
  }
  __device__ __forceinline__ float2 pieces(const Stream& s, int row, int n) const {
    const int count = pieces_of(s, n / 128);
    const float* at = s.part + row * s.columns + n;
    float2 y = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int q = 0; q < count; ++q) {
      const float2 v = *reinterpret_cast<const float2*>(at + (long long)q * s.m * s.columns);
      y.x += v.x;
      y.y += v.y;
    }
    return y;
  }
  static __device__ __forceinline__ void dot8(const uint4& u0, const uint4& u1, const float* t, float2& d) {
    float w0[8], w1[8];
    bf16x8_to_f32(u0, w0);
    bf16x8_to_f32(u1, w1);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d.x += w0[e] * t[e];
      d.y += w1[e] * t[e];
    }
  }
  __device__ __forceinline__ float2 low(const Finish& f, const float* t, int rank) const {
    float2 d = make_float2(0.f, 0.f);
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
      if (8 * q < rank) dot8(b0[q], b1[q], t + 8 * q, d);
    for (int j = 8 * kAhead; j < rank; j += 8)
      dot8(__ldg(reinterpret_cast<const uint4*>(from + j)), __ldg(reinterpret_cast<const uint4*>(from + f.b_row + j)),
           t + j, d);
    return d;
  }
};

__global__ void __launch_bounds__(128) finish_kernel(const Adapters ad, const Stream s, const Finish f) {
  __shared__ float t[kMaxRank];
  const int row = blockIdx.y;
  const int a = adapter_of(ad, s.m, row);
  const int col0 = a < 0 ? -1 : a * ad.rank;
  const int n = blockIdx.x * 256 + 2 * threadIdx.x;
  const bool mine = n < f.n_out;
  FinishPair y, u;
  if (mine) y.load(f, col0, ad.rank, n);
  if (mine && f.swiglu) u.load(f, col0, ad.rank, f.n_out + n);
  pdl_wait();
  if (*reinterpret_cast<volatile int*>(s.status) != 0) return;
  if (a >= 0) {
    for (int j = threadIdx.x; j < ad.rank; j += 128) {
      const int col = 128 * s.w_tiles + col0 + j;
      const int count = pieces_of(s, col / 128);
      float v = 0.f;
#pragma unroll 4
      for (int q = 0; q < count; ++q) v += s.part[((long long)q * s.m + row) * s.columns + col];
      t[j] = v * ad.scale[a];
    }
  }
  float2 gy = make_float2(0.f, 0.f), gu = gy;
  if (mine) gy = y.pieces(s, row, n);
  if (mine && f.swiglu) gu = u.pieces(s, row, f.n_out + n);
  __syncthreads();
  if (!mine) return;
  if (a >= 0) {
    const float2 d = y.low(f, t, ad.rank);
    gy.x += d.x;
    gy.y += d.y;
  }
  if (f.swiglu) {
    if (a >= 0) {
      const float2 d = u.low(f, t, ad.rank);
      gu.x += d.x;
      gu.y += d.y;
    }
    // out = bf16(bf16(silu(g)) * u), g and u the bf16-rounded gate / up projections
    const float g0 = bf16_round(gy.x), g1 = bf16_round(gy.y);
    gy.x = bf16_round(g0 / (1.0f + __expf(-g0))) * bf16_round(gu.x);
    gy.y = bf16_round(g1 / (1.0f + __expf(-g1))) * bf16_round(gu.y);
  }
  *reinterpret_cast<uint32_t*>(f.c + (long long)row * f.ldc + n) = pack_bf16x2(gy.x, gy.y);
}

// ---------------------------------------------------------------- host
struct Layout {
  bool few;
  int64_t low_bytes, list_bytes, part_bytes;  // tile path: T, chunk lists; row path: pieces
  int chunk_stride;
  Stream s;
  int ctas;
  int64_t bytes() const { return few ? part_bytes : low_bytes + list_bytes; }
};

static int check_adapters(int64_t rank, int64_t n_adapters) {
  if (n_adapters < 1 || rank < 8 || rank > kMaxRank || (rank < 64 ? 64 % rank : rank % 64)) return H3_ERR_SHAPE;
  return n_adapters * rank > 64ll * kMaxChunks ? H3_ERR_SHAPE : H3_OK;
}

static int make_layout(int64_t m, int64_t n_kb, int64_t kc_blocks, int64_t w_rows, int64_t rank, int64_t n_adapters,
                       Layout& l) {
  l = {};
  const int64_t stacked = rank * n_adapters;
  l.few = m <= kFewRows;
  if (!l.few) {
    l.chunk_stride = 1 + (int)((stacked + 63) / 64);
    l.low_bytes = (m * rank * 2 + 255) / 256 * 256;
    l.list_bytes = (m + 255) / 256 * l.chunk_stride * (int64_t)sizeof(int);
    return H3_OK;
  }
  int sms = 0, rc;
  if ((rc = sm_count(sms)) != H3_OK) return rc;
  Stream& s = l.s;
  s.m = (int)m;
  s.m_pad = (int)((m + 15) / 16 * 16);
  s.n_kb = (int)n_kb;
  s.kc_blocks = (int)kc_blocks;
  s.w_tiles = (int)((w_rows + 127) / 128);
  s.a_tiles = (int)((stacked + 127) / 128);
  const int64_t total = (int64_t)(s.w_tiles + s.a_tiles) * n_kb;
  s.per_cta = (int)((total + 2 * sms - 1) / (2 * sms));
  l.ctas = (int)((total + s.per_cta - 1) / s.per_cta);
  s.stages = std::min<int>(kMaxStreamStages, kStreamRing / (kTileBytes + s.m_pad * 128));
  s.columns = 128ll * (s.w_tiles + s.a_tiles);
  const int64_t most = (n_kb + s.per_cta - 2) / s.per_cta + 1;  // pieces of one tile
  l.part_bytes = most * m * s.columns * (int64_t)sizeof(float);
  return H3_OK;
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
  if (m < 1 || m > (1ll << 31) - 256 || a_chunks < 1 || a_chunks > 65535 || a_chunk_cols < 8 || n_out < 8 ||
      a_chunk_cols > (1ll << 24) || a_chunk_cols * a_chunks > (1ll << 24) || n_out > (1ll << 30) || (epilogue != 0 && epilogue != 1) ||
      2 * n_out * a_chunk_cols * a_chunks > (1ll << 41))
    return H3_ERR_SHAPE;
  if ((rc = check_adapters(rank, n_adapters)) != H3_OK) return rc;
  Layout l;
  const int64_t kc = (a_chunk_cols + 63) / 64;
  if ((rc = make_layout(m, kc * a_chunks, kc, epilogue == 1 ? 2 * n_out : n_out, rank, n_adapters, l)) != H3_OK) return rc;
  return l.bytes();
}

extern "C" int h3_gemm_adapters(const void* a, int64_t m, int64_t a_chunks, int64_t a_chunk_cols,
                                int64_t a_chunk_stride, int64_t a_row_stride, const void* w, int64_t n_out,
                                int64_t w_row_stride, const void* lora_a, int64_t lora_a_row_stride,
                                const void* lora_b, int64_t lora_b_row_stride, int64_t rank, int64_t n_adapters,
                                const float* scale, const int32_t* row_adapter, void* c, int64_t c_row_stride,
                                int32_t epilogue, void* workspace, int64_t ws_bytes, int32_t* status, void* stream) {
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
  if ((rc = make_layout(m, p.n_kb, p.kc_blocks, w_rows, rank, n_adapters, l)) != H3_OK) return rc;
  if (ws_bytes < l.bytes()) return H3_ERR_WORKSPACE;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const Adapters ad = {row_adapter, scale, (int)n_adapters, (int)rank, (int)((stacked + 63) / 64)};
  CUtensorMap tx, tw, ta, tb;
  if ((rc = map_w(&tw, call)) != H3_OK) return rc;
  if (l.few) {
    if ((rc = map_a(&tx, call, (unsigned)l.s.m_pad)) != H3_OK) return rc;
    if ((rc = make_map(&ta, lora_a, k, stacked, 1, lora_a_row_stride, stacked * lora_a_row_stride)) != H3_OK) return rc;
    l.s.part = reinterpret_cast<float*>(workspace);
    l.s.status = status;
    if ((rc = allow_smem(stream_kernel, kStreamSmem)) != H3_OK) return rc;
    stream_kernel<<<(unsigned)l.ctas, 192, kStreamSmem, st>>>(tw, ta, tx, ad, l.s);
    if (cudaGetLastError() != cudaSuccess) return H3_ERR_LAUNCH;
    const Finish f = {reinterpret_cast<const __nv_bfloat16*>(lora_b), lora_b_row_stride,
                      reinterpret_cast<__nv_bfloat16*>(c), c_row_stride, (int)n_out, epilogue};
    const dim3 grid((unsigned)((n_out + 255) / 256), (unsigned)m);
    return launch_dependent(finish_kernel, grid, 128, 0, st, ad, l.s, f);
  }
  if ((rc = map_a(&tx, call)) != H3_OK) return rc;
  if ((rc = make_map(&ta, lora_a, k, stacked, 1, lora_a_row_stride, stacked * lora_a_row_stride, 64)) != H3_OK) return rc;
  if ((rc = make_map(&tb, lora_b, stacked, w_rows, 1, lora_b_row_stride, w_rows * lora_b_row_stride)) != H3_OK) return rc;
  __nv_bfloat16* low = reinterpret_cast<__nv_bfloat16*>(workspace);
  int* chunks = reinterpret_cast<int*>(reinterpret_cast<uint8_t*>(workspace) + l.low_bytes);
  if ((rc = allow_smem(lower_kernel, kLowerSmem)) != H3_OK) return rc;
  lower_kernel<<<(unsigned)((m + 127) / 128), 192, kLowerSmem, st>>>(tx, ta, ad, low, chunks, l.chunk_stride, (int)m,
                                                                     p.n_kb, p.kc_blocks, status);
  if (cudaGetLastError() != cudaSuccess) return H3_ERR_LAUNCH;
  p.low = low;
  p.row_adapter = row_adapter;
  p.chunks = chunks;
  p.chunk_stride = l.chunk_stride;
  p.rank = (int)rank;
  p.n_adapters = (int)n_adapters;
  int sms = 0;
  if ((rc = sm_count(sms)) != H3_OK) return rc;
  constexpr uint32_t smem = smem_bytes(kNumBarsAdapters);
  if ((rc = allow_smem(adapter_gemm_kernel, smem)) != H3_OK) return rc;
  const int clusters = std::max(1, std::min(p.n_tiles, sms / 2));
  return launch_dependent(adapter_gemm_kernel, dim3(2 * clusters), kAdapterThreads, smem, st, tx, tw, tb, p);
}
