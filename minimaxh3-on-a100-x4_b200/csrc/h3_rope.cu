// Rotary positions over several axes (time, height, width, ...), computed from the positions:
//   theta_i = pos[token][axis_i] * inv_freq_i                       (64 pairs i of a 128-element head)
//   y_i = cos(theta_i) x_i - sin(theta_i) x_(i+64),  y_(i+64) = sin(theta_i) x_i + cos(theta_i) x_(i+64)
// A pair whose axis is outside [0, n_axes) keeps its finite values (it is turned by 0: an infinity makes its partner NaN,
// 0 * inf, as it does in every pair). Two forms:
//   * rope_axes: rotates [tokens][heads][128] (inverse: the transposed rotation, its gradient)
//   * pack_axes: per-head RMSNorm of q and k, rotation and the seq->head send layout in one pass, as
//     qknorm_rope_pack does with a table of 2x2 matrices (1 KB per token, which this form does not read)
//
// Angles: the product is taken in fp64 and reduced to a fraction of a turn before it is rounded to
// fp32, so a position of 10^5 is as exact as position 1 (an fp32 product would be off by 2^-24 of
// the angle, 6e-3 rad there). sm_100 multiplies fp64 at half the fp32 rate and a token needs 64
// products for all of its heads, so this costs no time that the row traffic does not hide. Rows are
// fp32 from the load to the one rounding at the store.
//
// Both kernels are bound by HBM: every row is read once and written once. One warp walks one token
// (or a share of its rows, when there are fewer tokens than warps): each lane evaluates two of the
// 64 sine/cosine pairs, the warp exchanges them through shared memory, and its four 8-lane groups
// take one head row each (16 elements a lane, 16-byte accesses, both halves of a pair in one lane),
// two (pack) or four rows a group in flight. rope_axes: 92 us at 40868 tokens x 28 heads = 6.4 TB/s, 0.97 of the
// copy rate.
#include "h3_rows.cuh"
#include "h3attn.h"

#include <cmath>

namespace h3 {
namespace rope {

constexpr int kWarps = 8;        // warps per CTA
constexpr int kRows = 4;         // head rows in flight per 8-lane group
constexpr int kStep = 4 * kRows; // head rows per warp step
constexpr double kTurn = 0.15915494309189533577;  // 1 / (2 pi)

struct Axes {
  const void* pos;  // [tokens][n_axes], int32 or fp32
  int is_float;
  int n_axes;
  const double* inv_freq;  // [64], radians per unit position
  const int32_t* axis;     // [64]
  float sign;              // -1: the inverse rotation
};

// The two pairs of one lane: turns per unit position and the axis (-1: not rotated).
struct LanePairs {
  double f[2];
  int a[2];
};
__device__ __forceinline__ LanePairs lane_pairs(const Axes& ax, int lane) {
  LanePairs lp;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int a = ax.axis[lane + 32 * i];
    lp.a[i] = a >= 0 && a < ax.n_axes ? a : -1;
    lp.f[i] = ax.inv_freq[lane + 32 * i] * kTurn;
  }
  return lp;
}

// cos / sin of the token's 64 angles into the warp's 64 float2 of shared memory.
__device__ __forceinline__ void token_angles(const Axes& ax, const LanePairs& lp, long long tok, int lane, float2* sh) {
  __syncwarp();  // the previous token's pairs have been read
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float2 cs = make_float2(1.f, 0.f);
    if (lp.a[i] >= 0) {
      const long long at = tok * ax.n_axes + lp.a[i];
      const double p = ax.is_float ? (double)reinterpret_cast<const float*>(ax.pos)[at]
                                   : (double)reinterpret_cast<const int32_t*>(ax.pos)[at];
      const double t = p * lp.f[i];
      sincospif(2.0f * (float)(t - rint(t)), &cs.y, &cs.x);
      cs.y *= ax.sign;
    }
    sh[lane + 32 * i] = cs;
  }
  __syncwarp();
}

// This lane's eight pairs (8g .. 8g+7) of them.
__device__ __forceinline__ void lane_angles(const float2* sh, int g, float (&c)[8], float (&s)[8]) {
  const float4* src = reinterpret_cast<const float4*>(sh + 8 * g);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 v = src[i];
    c[2 * i] = v.x;
    s[2 * i] = v.y;
    c[2 * i + 1] = v.z;
    s[2 * i + 1] = v.w;
  }
}

__device__ __forceinline__ void rotate(float (&x)[16], const float (&c)[8], const float (&s)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float a = x[i], b = x[8 + i];
    x[i] = c[i] * a - s[i] * b;
    x[8 + i] = s[i] * a + c[i] * b;
  }
}

__global__ void __launch_bounds__(32 * kWarps, 3)
    rope_axes_kernel(const __nv_bfloat16* x, long long x_row, long long x_head, const Axes ax, __nv_bfloat16* out,
                     long long o_row, long long o_head, long long tokens, int n_heads, int parts, int part_heads) {
  __shared__ float2 sh_cs[kWarps][64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane & 7, grp = lane >> 3;
  const LanePairs lp = lane_pairs(ax, lane);
  const long long items = tokens * parts;
  for (long long it = (long long)blockIdx.x * kWarps + warp; it < items; it += (long long)gridDim.x * kWarps) {
    const long long tok = it / parts;
    const int h0 = int(it - tok * parts) * part_heads;
    const int h1 = min(h0 + part_heads, n_heads);
    float c[8], s[8];
    token_angles(ax, lp, tok, lane, sh_cs[warp]);
    lane_angles(sh_cs[warp], g, c, s);
    for (int base = h0; base < h1; base += kStep) {
      uint4 u[kRows][2];
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int h = base + 4 * i + grp;
        if (h < h1) {
          const __nv_bfloat16* src = x + tok * x_row + (long long)h * x_head + 8 * g;
          u[i][0] = *reinterpret_cast<const uint4*>(src);
          u[i][1] = *reinterpret_cast<const uint4*>(src + 64);
        }
      }
#pragma unroll
      for (int i = 0; i < kRows; ++i) {
        const int h = base + 4 * i + grp;
        if (h < h1) {
          float v[16];
          bf16x8_to_f32(u[i][0], v);
          bf16x8_to_f32(u[i][1], v + 8);
          rotate(v, c, s);
          __nv_bfloat16* dst = out + tok * o_row + (long long)h * o_head + 8 * g;
          *reinterpret_cast<uint4*>(dst) = f32_to_bf16x8(v);
          *reinterpret_cast<uint4*>(dst + 64) = f32_to_bf16x8(v + 8);
        }
      }
    }
  }
}

// One head row of an 8-lane group in place: y = x / sqrt(mean(x^2) + eps) * w, then the rotation. Lane g holds elements
// [8g, 8g + 8) and [64 + 8g, ...); weights and angles stay packed (bf16 words, shared memory), so that the row itself is
// all that a thread keeps in fp32.
__device__ __forceinline__ void norm_turn_row(uint4& u0, uint4& u1, const uint4& w0, const uint4& w1, const float4* cs,
                                              float eps) {
  float v[16];
  bf16x8_to_f32(u0, v);
  bf16x8_to_f32(u1, v + 8);
  float q = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) q += v[e] * v[e];
  q += __shfl_xor_sync(0xffffffffu, q, 4);
  q += __shfl_xor_sync(0xffffffffu, q, 2);
  q += __shfl_xor_sync(0xffffffffu, q, 1);
  const float r = 1.0f / sqrtf(q * (1.0f / kHeadDim) + eps);
  const uint32_t wa[4] = {w0.x, w0.y, w0.z, w0.w}, wb[4] = {w1.x, w1.y, w1.z, w1.w};
  uint32_t oa[4], ob[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float4 t = cs[j];
    const float a0 = v[2 * j] * r * __uint_as_float(wa[j] << 16);
    const float a1 = v[2 * j + 1] * r * __uint_as_float(wa[j] & 0xFFFF0000u);
    const float b0 = v[8 + 2 * j] * r * __uint_as_float(wb[j] << 16);
    const float b1 = v[9 + 2 * j] * r * __uint_as_float(wb[j] & 0xFFFF0000u);
    oa[j] = pack_bf16x2(t.x * a0 - t.y * b0, t.z * a1 - t.w * b1);
    ob[j] = pack_bf16x2(t.y * a0 + t.x * b0, t.w * a1 + t.z * b1);
  }
  u0 = make_uint4(oa[0], oa[1], oa[2], oa[3]);
  u1 = make_uint4(ob[0], ob[1], ob[2], ob[3]);
}

struct PackOut {
  __nv_bfloat16* base[3];  // q, k, v (one local send buffer)
  long long rank_stride, head_stride;
  const unsigned long long* rank_base;  // or one buffer per destination rank (peer memory)
  long long tensor_stride, row_offset;
  int heads_per_rank;
  unsigned rank_magic;  // ceil(2^32 / heads_per_rank): h / heads_per_rank = h * magic >> 32, h < 2^16, from 2 a rank on
};
__host__ __device__ __forceinline__ int rank_of_head(const PackOut& o, int h) {
  return o.heads_per_rank == 1 ? h : int((unsigned long long)(unsigned)h * o.rank_magic >> 32);
}
__host__ __device__ __forceinline__ void split_heads(PackOut& o, int heads_per_rank) {
  o.heads_per_rank = heads_per_rank;
  o.rank_magic = (unsigned)(((1ull << 32) + heads_per_rank - 1) / heads_per_rank);
}
template <int kTensor>
__device__ __forceinline__ __nv_bfloat16* pack_row(const PackOut& o, int h, long long tok) {
  const int r = rank_of_head(o, h), hl = h - r * o.heads_per_rank;
  return o.rank_base != nullptr
             ? reinterpret_cast<__nv_bfloat16*>(o.rank_base[r]) + kTensor * o.tensor_stride +
                   (long long)hl * o.head_stride + (o.row_offset + tok) * kHeadDim
             : o.base[kTensor] + (long long)r * o.rank_stride + (long long)hl * o.head_stride + tok * kHeadDim;
}

// in[0..2]: q, k, v rows; w[0..1]: the RMSNorm weights of q and k or nullptr.
struct PackIn {
  const __nv_bfloat16* in[3];
  long long row_stride;
  const __nv_bfloat16* w[2];
  float eps;
};

// Two rows in flight a group and three CTAs (24 warps) an SM, 80 registers without spills: 588 us at 42000 tokens x 56
// heads = 6.14 TB/s, 0.94 of the copy rate (605-613 on boxes whose copies are as much slower). Four rows at two CTAs: 639 us, two rows at four CTAs (spills): 585 us there
// but 92 against 83 us at 5250 tokens, one row at five: 634 us. (Weights and angles in registers as fp32, four rows:
// 720 us; parameter arrays indexed by a runtime tensor number, which go through local memory: 690 us.)
constexpr int kPackRows = 2;                // head rows in flight per 8-lane group
constexpr int kPackStep = 4 * kPackRows;
constexpr int kPackCtas = 3;                // CTAs per SM

// Heads [h0, h1) of one token and one of q, k, v (0, 1, 2; v is copied).
template <int kTensor>
__device__ __forceinline__ void pack_heads(const PackIn& in, const PackOut& out, const float4* cs, long long tok, int h0,
                                           int h1, int g, int grp) {
  uint4 w0 = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u), w1 = w0;  // bf16 ones
  if constexpr (kTensor < 2) {
    if (in.w[kTensor] != nullptr) {
      w0 = __ldg(reinterpret_cast<const uint4*>(in.w[kTensor] + 8 * g));
      w1 = __ldg(reinterpret_cast<const uint4*>(in.w[kTensor] + 64 + 8 * g));
    }
  }
  const __nv_bfloat16* src0 = in.in[kTensor] + tok * in.row_stride + 8 * g;
#pragma unroll 1
  for (int base = h0; base < h1; base += kPackStep) {
    uint4 u[kPackRows][2];
#pragma unroll
    for (int i = 0; i < kPackRows; ++i) {
      const int h = min(base + 4 * i + grp, h1 - 1);  // every lane joins the shuffles below
      const __nv_bfloat16* src = src0 + h * kHeadDim;
      u[i][0] = __ldg(reinterpret_cast<const uint4*>(src));
      u[i][1] = __ldg(reinterpret_cast<const uint4*>(src + 64));
    }
#pragma unroll
    for (int i = 0; i < kPackRows; ++i) {
      if constexpr (kTensor < 2) norm_turn_row(u[i][0], u[i][1], w0, w1, cs, in.eps);
      const int h = base + 4 * i + grp;
      if (h < h1) {
        __nv_bfloat16* dst = pack_row<kTensor>(out, h, tok) + 8 * g;
        *reinterpret_cast<uint4*>(dst) = u[i][0];
        *reinterpret_cast<uint4*>(dst + 64) = u[i][1];
      }
    }
  }
}

__global__ void __launch_bounds__(32 * kWarps, kPackCtas)
    pack_axes_kernel(const __grid_constant__ PackIn in, const __grid_constant__ Axes ax,
                     const __grid_constant__ PackOut out, long long tokens, int n_heads, int parts, int part_heads) {
  __shared__ float2 sh_cs[kWarps][64];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane & 7, grp = lane >> 3;
  const LanePairs lp = lane_pairs(ax, lane);
  const long long items = tokens * parts;
  for (long long it = (long long)blockIdx.x * kWarps + warp; it < items; it += (long long)gridDim.x * kWarps) {
    const long long tok = it / parts;
    const int h0 = int(it - tok * parts) * part_heads;
    const int h1 = min(h0 + part_heads, n_heads);
    token_angles(ax, lp, tok, lane, sh_cs[warp]);
    const float4* cs = reinterpret_cast<const float4*>(sh_cs[warp] + 8 * g);  // (cos, sin) of pairs 8g + 2j, 8g + 2j + 1
    pack_heads<0>(in, out, cs, tok, h0, h1, g, grp);
    pack_heads<1>(in, out, cs, tok, h0, h1, g, grp);
    pack_heads<2>(in, out, cs, tok, h0, h1, g, grp);
  }
  if (out.rank_base != nullptr) __threadfence_system();  // peer stores visible before the host-side barrier
}

// Checks shared by the entry points; fills ax.
static int make_axes(const void* pos, int32_t pos_type, int64_t n_axes, const double* inv_freq, const int32_t* axis,
                     int inverse, Axes& ax) {
  if (!pos || !inv_freq || !axis) return H3_ERR_NULL;
  if ((reinterpret_cast<uintptr_t>(pos) & 3u) || (reinterpret_cast<uintptr_t>(inv_freq) & 7u) ||
      (reinterpret_cast<uintptr_t>(axis) & 3u))
    return H3_ERR_ALIGN;
  if ((pos_type != H3_POS_INT32 && pos_type != H3_POS_FLOAT32) || n_axes < 1 || n_axes > 64) return H3_ERR_SHAPE;
  ax.pos = pos;
  ax.is_float = pos_type == H3_POS_FLOAT32;
  ax.n_axes = (int)n_axes;
  ax.inv_freq = inv_freq;
  ax.axis = axis;
  ax.sign = inverse ? -1.f : 1.f;
  return H3_OK;
}

// One warp a token; below 64 tokens an SM a token's heads are split over several warps, so that the SMs' resident warps
// (24 an SM) come round two or three times and the last round is short: 5250 tokens x 56 heads, 90 us without, 80
// with; 1500 tokens, 27 us, 43 with twice as many parts. Four heads a part at least (a warp's rows at a time).
static int head_parts(int64_t tokens, int64_t n_heads, int& parts, int& part_heads) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return H3_ERR_CUDA;
  const int64_t warps = (int64_t)sms * 64;
  const int64_t want = tokens >= warps ? 1 : (warps + tokens - 1) / tokens;
  int64_t heads = ((n_heads + want - 1) / want + 3) / 4 * 4;
  if (heads > kPackStep) heads = (heads + kPackStep - 1) / kPackStep * kPackStep;  // whole steps
  part_heads = (int)heads;
  parts = (int)((n_heads + heads - 1) / heads);
  return H3_OK;
}

static int pack_impl(const void* q, const void* k, const void* v, int64_t in_row_stride, const Axes& ax,
                     const void* q_weight, const void* k_weight, float eps, PackOut& o, int64_t s_l, int64_t n_heads,
                     int64_t heads_per_rank, void* stream) {
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || (q_weight && !aligned16(q_weight)) ||
      (k_weight && !aligned16(k_weight)))
    return H3_ERR_ALIGN;
  if (s_l < 1 || n_heads < 1 || heads_per_rank < 1 || n_heads % heads_per_rank) return H3_ERR_SHAPE;
  if (s_l > (1ll << 31) || n_heads > 65535 || s_l * 3 * n_heads > (1ll << 40)) return H3_ERR_SHAPE;
  if (in_row_stride < n_heads * kHeadDim || (in_row_stride % 8) || (o.head_stride % 8)) return H3_ERR_STRIDE;
  if (!(eps >= 0.f)) return H3_ERR_SHAPE;
  PackIn in;
  in.in[0] = reinterpret_cast<const __nv_bfloat16*>(q);
  in.in[1] = reinterpret_cast<const __nv_bfloat16*>(k);
  in.in[2] = reinterpret_cast<const __nv_bfloat16*>(v);
  in.row_stride = in_row_stride;
  in.w[0] = reinterpret_cast<const __nv_bfloat16*>(q_weight);
  in.w[1] = reinterpret_cast<const __nv_bfloat16*>(k_weight);
  in.eps = eps;
  split_heads(o, (int)heads_per_rank);
  int parts = 1, part_heads = 1, rc;
  if ((rc = head_parts(s_l, n_heads, parts, part_heads)) != H3_OK) return rc;
  pack_axes_kernel<<<grid_for(s_l * parts, kWarps, 1 << 20), 32 * kWarps, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      in, ax, o, s_l, (int)n_heads, parts, part_heads);
  return cudaGetLastError() == cudaSuccess ? H3_OK : H3_ERR_LAUNCH;
}

}  // namespace rope
}  // namespace h3

using namespace h3;
using namespace h3::rope;

extern "C" int h3_rope_axes(const void* x, int64_t x_row_stride, int64_t x_head_stride, const void* pos,
                            int32_t pos_type, int64_t n_axes, const double* inv_freq, const int32_t* axis,
                            int32_t inverse, void* out, int64_t out_row_stride, int64_t out_head_stride, int64_t s,
                            int64_t n_heads, void* stream) {
  if (!x || !out) return H3_ERR_NULL;
  Axes ax;
  int rc;
  if ((rc = make_axes(pos, pos_type, n_axes, inv_freq, axis, inverse, ax)) != H3_OK) return rc;
  if (!aligned16(x) || !aligned16(out)) return H3_ERR_ALIGN;
  if (s < 1 || n_heads < 1 || s > (1ll << 31) || n_heads > 65535 || s * n_heads > (1ll << 40)) return H3_ERR_SHAPE;
  if ((x_row_stride % 8) || (x_head_stride % 8) || (out_row_stride % 8) || (out_head_stride % 8) ||
      x_row_stride < 0 || x_head_stride < 0 || (s > 1 && out_row_stride < kHeadDim) ||
      (n_heads > 1 && out_head_stride < kHeadDim))
    return H3_ERR_STRIDE;
  int parts = 1, part_heads = 1;
  if ((rc = head_parts(s, n_heads, parts, part_heads)) != H3_OK) return rc;
  rope_axes_kernel<<<grid_for(s * parts, kWarps, 1 << 20), 32 * kWarps, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      reinterpret_cast<const __nv_bfloat16*>(x), x_row_stride, x_head_stride, ax,
      reinterpret_cast<__nv_bfloat16*>(out), out_row_stride, out_head_stride, s, (int)n_heads, parts, part_heads);
  return cudaGetLastError() == cudaSuccess ? H3_OK : H3_ERR_LAUNCH;
}

extern "C" int h3_pack_ranks_kat(int64_t n_heads, int64_t heads_per_rank, int32_t* ranks) {
  if (!ranks) return H3_ERR_NULL;
  if (n_heads < 1 || n_heads > 65535 || heads_per_rank < 1 || heads_per_rank > n_heads) return H3_ERR_SHAPE;
  PackOut o = {};
  split_heads(o, (int)heads_per_rank);
  for (int h = 0; h < n_heads; ++h) ranks[h] = rank_of_head(o, h);
  return H3_OK;
}

extern "C" int h3_qknorm_rope_pack_axes(const void* q, const void* k, const void* v, int64_t in_row_stride,
                                        const void* pos, int32_t pos_type, int64_t n_axes, const double* inv_freq,
                                        const int32_t* axis, const void* q_weight, const void* k_weight, float eps,
                                        void* q_out, void* k_out, void* v_out, int64_t s_l, int64_t n_heads,
                                        int64_t heads_per_rank, int64_t out_rank_stride, int64_t out_head_stride,
                                        void* stream) {
  if (!q || !k || !v || !q_out || !k_out || !v_out) return H3_ERR_NULL;
  Axes ax;
  int rc;
  if ((rc = make_axes(pos, pos_type, n_axes, inv_freq, axis, 0, ax)) != H3_OK) return rc;
  if (!aligned16(q_out) || !aligned16(k_out) || !aligned16(v_out)) return H3_ERR_ALIGN;
  if (out_rank_stride % 8) return H3_ERR_STRIDE;
  PackOut o = {{reinterpret_cast<__nv_bfloat16*>(q_out), reinterpret_cast<__nv_bfloat16*>(k_out),
                reinterpret_cast<__nv_bfloat16*>(v_out)},
               out_rank_stride, out_head_stride, nullptr, 0, 0, 1, 0};
  return pack_impl(q, k, v, in_row_stride, ax, q_weight, k_weight, eps, o, s_l, n_heads, heads_per_rank, stream);
}

extern "C" int h3_qknorm_rope_pack_axes_peer(const void* q, const void* k, const void* v, int64_t in_row_stride,
                                             const void* pos, int32_t pos_type, int64_t n_axes,
                                             const double* inv_freq, const int32_t* axis, const void* q_weight,
                                             const void* k_weight, float eps, const uint64_t* rank_base,
                                             int64_t n_ranks, int64_t tensor_stride, int64_t head_stride,
                                             int64_t row_offset, int64_t s_l, int64_t n_heads, int64_t heads_per_rank,
                                             void* stream) {
  if (!q || !k || !v || !rank_base) return H3_ERR_NULL;
  Axes ax;
  int rc;
  if ((rc = make_axes(pos, pos_type, n_axes, inv_freq, axis, 0, ax)) != H3_OK) return rc;
  if (reinterpret_cast<uintptr_t>(rank_base) & 7u) return H3_ERR_ALIGN;
  // the kernel indexes rank_base[head / heads_per_rank]: the table must cover every destination
  if (row_offset < 0 || heads_per_rank < 1 || n_ranks < 1 || n_heads / heads_per_rank > n_ranks) return H3_ERR_SHAPE;
  if ((tensor_stride % 8) || tensor_stride < 0 || head_stride < 0) return H3_ERR_STRIDE;
  PackOut o = {{nullptr, nullptr, nullptr}, 0, head_stride, reinterpret_cast<const unsigned long long*>(rank_base),
               tensor_stride, row_offset, 1, 0};
  return pack_impl(q, k, v, in_row_stride, ax, q_weight, k_weight, eps, o, s_l, n_heads, heads_per_rank, stream);
}
