// Pieces shared by the attention kernels (full and windowed): 128 x 128 tile geometry, the
// tcgen05 issue of S = Q K^T and O += P V for one tile, the drain wait, and the tensor map of
// [heads][rows][128] bf16.
#pragma once
#include "h3_rows.cuh"
#include "h3attn.h"

namespace h3 {
namespace attn {

constexpr int kBlockM = 128;
constexpr int kBlockN = 128;
constexpr uint32_t kHalfBytes = 128u * 64u * 2u;  // 128 rows x 64 bf16: one 128-B swizzle column block
constexpr uint32_t kTileBytes = 2u * kHalfBytes;  // 128 rows x 128 bf16
constexpr float kRescaleThreshold = 8.0f;  // log2 units

// Every 8-MMA group below is ONE asm block with the smem descriptors formed by immediate
// adds on the low word: the single MMA-issuing thread shares its SM sub-partition with two
// busy softmax warps, and the tensor pipe queue is shallow, so the instructions it spends
// per MMA directly become tensor-core idle time. Start addresses stay below 256 KB, so the
// low-word adds never carry out of the 14-bit start-address field.

// S = Q K^T for one 128x128 tile pair: both operands K-major, SW128, two 64-column blocks
// 16 KB apart; K steps of 16 elements advance 32 B inside a block.
__device__ __forceinline__ void issue_qk(uint32_t d_tmem, uint32_t a_base, uint32_t b_base) {
  constexpr uint32_t idesc = idesc_bf16_f32(128, 128, 0, 0);
  const uint64_t ad = smem_desc_sw128(a_base, 16, 1024), bd = smem_desc_sw128(b_base, 16, 1024);
  const uint32_t alo = uint32_t(ad), ahi = uint32_t(ad >> 32), blo = uint32_t(bd), bhi = uint32_t(bd >> 32);
#define H3_QK_STEP(OFF) \
  "add.u32 la, %1, " #OFF ";\n\t add.u32 lb, %3, " #OFF ";\n\t" \
  "mov.b64 da, {la, %2};\n\t mov.b64 db, {lb, %4};\n\t" \
  "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, pt;\n\t"
  asm volatile(
      "{\n\t.reg .pred pf, pt;\n\t.reg .b32 la, lb;\n\t.reg .b64 da, db;\n\t"
      "setp.ne.b32 pf, %0, %0;\n\t setp.eq.b32 pt, %0, %0;\n\t"
      "mov.b64 da, {%1, %2};\n\t mov.b64 db, {%3, %4};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, pf;\n\t"
      H3_QK_STEP(2) H3_QK_STEP(4) H3_QK_STEP(6) H3_QK_STEP(1024) H3_QK_STEP(1026) H3_QK_STEP(1028) H3_QK_STEP(1030)
      "}\n" ::"r"(d_tmem), "r"(alo), "r"(ahi), "r"(blo), "r"(bhi), "r"(idesc)
      : "memory");
#undef H3_QK_STEP
}

// Bounded wait that ignores the abort flag: used while draining copies/MMAs before exit.
__device__ __forceinline__ void drain_wait(uint32_t bar, uint32_t parity, int* status) {
  uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait_sleep(bar, parity)) {
    if (globaltimer_ns() - t0 > H3_WAIT_LIMIT_NS) {
      atomicCAS(status, 0, kStatusTimeoutDrain);
      return;
    }
  }
}

// O (+)= P V over K steps [kFirst, kFirst + kSteps) of one tile (16 keys per step): P from
// TMEM at 8 columns per step, V in shared memory 2 KB per step. One asm block per call.
template <int kFirst, int kSteps>
__device__ __forceinline__ void issue_pv_steps(uint32_t d_tmem, uint32_t p_tmem, uint32_t v_base, bool accumulate) {
  static_assert(kFirst >= 0 && kSteps >= 0 && kFirst + kSteps <= 8, "8 K steps per tile");
  if constexpr (kSteps > 0) {
    constexpr uint32_t idesc = idesc_bf16_f32(128, 128, 0, 1);
    // steps 0-3 sit in the first 64-key block of V's rows, 4-7 in the second (8 KB on); the two
    // 64-wide d blocks are 16 KB apart (LBO), 8-key groups 1 KB apart (SBO)
    const uint64_t bd = smem_desc_sw128(v_base + uint32_t(kFirst) * 2048u, kHalfBytes, 1024);
    const uint32_t blo = uint32_t(bd), bhi = uint32_t(bd >> 32);
    const uint32_t pa = p_tmem + uint32_t(kFirst) * 8u;
#define H3_PV_STEP(KK) \
  "add.u32 ta, %1, " #KK "*8;\n\t add.u32 lb, %2, " #KK "*128;\n\t mov.b64 db, {lb, %3};\n\t" \
  "tcgen05.mma.cta_group::1.kind::f16 [%0], [ta], db, %4, pt;\n\t"
#define H3_PV_HEAD \
  "{\n\t.reg .pred pf, pt;\n\t.reg .b32 ta, lb;\n\t.reg .b64 db;\n\t" \
  "setp.ne.b32 pf, %5, 0;\n\t setp.eq.b32 pt, %5, %5;\n\t mov.b64 db, {%2, %3};\n\t" \
  "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, pf;\n\t"
#define H3_PV_ARGS ::"r"(d_tmem), "r"(pa), "r"(blo), "r"(bhi), "r"(idesc), "r"(accumulate ? 1u : 0u) : "memory"
    if constexpr (kSteps == 1) {
      asm volatile(H3_PV_HEAD "}\n" H3_PV_ARGS);
    } else if constexpr (kSteps == 2) {
      asm volatile(H3_PV_HEAD H3_PV_STEP(1) "}\n" H3_PV_ARGS);
    } else if constexpr (kSteps == 4) {
      asm volatile(H3_PV_HEAD H3_PV_STEP(1) H3_PV_STEP(2) H3_PV_STEP(3) "}\n" H3_PV_ARGS);
    } else if constexpr (kSteps == 6) {
      asm volatile(H3_PV_HEAD H3_PV_STEP(1) H3_PV_STEP(2) H3_PV_STEP(3) H3_PV_STEP(4) H3_PV_STEP(5) "}\n" H3_PV_ARGS);
    } else if constexpr (kSteps == 8) {
      asm volatile(H3_PV_HEAD H3_PV_STEP(1) H3_PV_STEP(2) H3_PV_STEP(3) H3_PV_STEP(4) H3_PV_STEP(5) H3_PV_STEP(6)
                       H3_PV_STEP(7) "}\n" H3_PV_ARGS);
    } else {
      static_assert(kSteps == 1 || kSteps == 2 || kSteps == 4 || kSteps == 6 || kSteps == 8, "step count");
    }
#undef H3_PV_ARGS
#undef H3_PV_HEAD
#undef H3_PV_STEP
  }
}

// [n_heads][rows][128] bf16 with element strides (row_stride, head_stride); box 64 x box_rows x 1, SW128.
inline int make_head_map(CUtensorMap* map, const void* base, long long rows, long long n_heads,
                         long long row_stride, long long head_stride, unsigned box_rows = 128) {
  EncodeTiledFn enc = get_encode_fn();
  if (!enc) return H3_ERR_DRIVER;
  cuuint64_t dims[3] = {128, (cuuint64_t)rows, (cuuint64_t)n_heads};
  cuuint64_t strides[2] = {(cuuint64_t)row_stride * 2, (cuuint64_t)head_stride * 2};
  cuuint32_t box[3] = {64, box_rows, 1};
  cuuint32_t estr[3] = {1, 1, 1};
  CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, estr,
                   CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                   CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? H3_OK : H3_ERR_TENSOR_MAP;
}

}  // namespace attn
}  // namespace h3
