// Token-sharded projection GEMM for the attention layer and the SwiGLU FFN:
//   C[m][n] = sum_k A[m][k] * W[n][k]      (bf16 in, fp32 accumulate, bf16 out)
// W is an nn.Linear weight ([out][in], K contiguous). It replaces the qkv_proj / out_proj calls
// of the reference's attention forward (harness/sp_runtime.py:93, :126) and the FFN's fc1 and
// swiglu-into-fc2 linears (harness/sp_blockloop.py:169-170).
//
// Every output row is computed by exactly one tile with one fixed K order (64-wide k-blocks in
// ascending order, four K=16 MMAs each, no split-K), so a row's result does not depend on how
// many rows the call has or where the row sits: token-sharded calls on W ranks give the same
// bits as the 1-GPU call, which is what makes the W-way layer bit-exact.
//
// Layout: persistent clusters of two CTAs (one per SM). A pair tile is 256 rows x 256 columns:
// CTA r stages A rows [128r, 128r+128) and W rows for columns [128r, 128r+128), and the leader's
// single thread issues tcgen05.mma.cta_group::2 (M=256, N=256, K=16), leaving each CTA a
// 128 x 256 fp32 accumulator in TMEM. Two accumulators (512 columns) alternate between tiles so
// the epilogue of one tile overlaps the main loop of the next. A is read through a 3-D tensor
// map [chunks][rows][chunk_cols]: plain row-major A is one chunk; the head->seq receive buffer
// [H][rows][128] is read in place as A[rows][H*128] (out_proj without an unpack pass).
// SwiGLU epilogue: W holds [gate; up] (2F rows); CTA 0 stages gate rows, CTA 1 the matching up
// rows, so accumulator column c (gate) and c + 128 (up) of a row sit in the same thread.
#include <algorithm>

#include "h3_gemm.cuh"

namespace h3 {
namespace gemm {

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    gemm_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_w,
                const Params p) {
  gemm_body<false>(tmap_a, tmap_w, tmap_w, p);
}

}  // namespace gemm
}  // namespace h3

using namespace h3;
using namespace h3::gemm;

extern "C" int h3_gemm_bf16(const void* a, int64_t m, int64_t a_chunks, int64_t a_chunk_cols, int64_t a_chunk_stride,
                            int64_t a_row_stride, const void* w, int64_t n_out, int64_t w_row_stride, void* c,
                            int64_t c_row_stride, int32_t epilogue, int32_t* status, void* stream) {
  const Call call = {a, m, a_chunks, a_chunk_cols, a_chunk_stride, a_row_stride, w, n_out, w_row_stride, c,
                     c_row_stride, epilogue, status};
  int rc;
  if ((rc = check_call(call)) != H3_OK) return rc;
  CUtensorMap ta, tw;
  if ((rc = map_a(&ta, call)) != H3_OK) return rc;
  if ((rc = map_w(&tw, call)) != H3_OK) return rc;
  const Params p = call_params(call);
  int sms = 0;
  if ((rc = sm_count(sms)) != H3_OK) return rc;
  const int clusters = std::max(1, std::min(p.n_tiles, sms / 2));
  constexpr uint32_t smem = smem_bytes(kNumBars);
  if (cudaFuncSetAttribute(gemm_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
    return H3_ERR_LAUNCH;
  gemm_kernel<<<2 * clusters, kThreads, smem, reinterpret_cast<cudaStream_t>(stream)>>>(ta, tw, p);
  return cudaGetLastError() == cudaSuccess ? H3_OK : H3_ERR_LAUNCH;
}
