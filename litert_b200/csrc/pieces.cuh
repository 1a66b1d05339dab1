// Attention cut into equal pieces: the cached tokens of all (sequence, KV head) pairs form one row of 16-token units, every
// CTA takes an equal piece of it and leaves one partial record (un-normalised output, maximum, sum) per pair that it
// touches; a second kernel merges a pair's records. What sdpa_split.cu and kv4_sdpa.cu share of this.
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace b200 {
namespace {

constexpr int kUnit = 16;  // tokens per unit: the rows of one MMA tile and of one copy box

__device__ __forceinline__ int units_of(int len) { return (len + kUnit - 1) / kUnit; }

// How `total` units are cut: `ctas` pieces, the first `rest` of them one unit longer than the others. No piece is
// shorter than min_units, so that short caches are not scattered over more records than they are worth.
struct Pieces {
  int ctas, size, rest;
  __device__ __forceinline__ Pieces(int total, int grid, int min_units) {
    ctas = max(1, min(grid, (total + min_units - 1) / min_units));
    size = total / ctas;
    rest = total - size * ctas;
  }
  __device__ __forceinline__ int begin(int c) const { return c * size + min(c, rest); }
  __device__ __forceinline__ int owner(int u) const {
    const int longer = rest * (size + 1);
    return u < longer ? u / (size + 1) : rest + (u - longer) / size;
  }
};

// Weights exp2((m_record - m) * to_log2) of a head's records, from their (maximum, sum) pairs at `ml` (to_log2: 1 for maxima
// in powers of two, log2 e for natural ones); returns the softmax denominator, or kLostRecord where a record is one. Whole
// warp; the first 64 pairs in one round trip.
__device__ __forceinline__ float record_weights(const float* ml, size_t stride, int count, int lane, float* weights, float to_log2 = 1.0f) {
  const float2 none = make_float2(-CUDART_INF_F, 0.0f);
  const float2 a = lane < count ? __ldcg(reinterpret_cast<const float2*>(ml + lane * stride)) : none;
  const float2 b = lane + 32 < count ? __ldcg(reinterpret_cast<const float2*>(ml + (lane + 32) * stride)) : none;
  float mm = fmaxf(a.x, b.x);
  for (int c = lane + 64; c < count; c += 32) mm = fmaxf(mm, __ldcg(ml + c * stride));
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  const float muse = mm == -CUDART_INF_F ? 0.0f : mm;
  const float fa = exp2f((a.x - muse) * to_log2), fb = exp2f((b.x - muse) * to_log2);
  float l = fa * a.y + fb * b.y;
  bool lost = a.y == kLostRecord || b.y == kLostRecord;
  if (lane < count) weights[lane] = fa;
  if (lane + 32 < count) weights[lane + 32] = fb;
  for (int c = lane + 64; c < count; c += 32) {
    const float2 v = __ldcg(reinterpret_cast<const float2*>(ml + c * stride));
    const float f = exp2f((v.x - muse) * to_log2);
    weights[c] = f;
    l += f * v.y;
    lost = lost || v.y == kLostRecord;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  return __any_sync(0xffffffffu, lost) ? kLostRecord : l;
}

// Sum of a head's records, weighted, for the four outputs d4 .. d4 + 3: records grp, grp + groups, ...
// (`first`: the first kBatch of them, requested earlier).
template <int kBatch>
__device__ __forceinline__ float4 merge_quad(const float* base, size_t stride, int count, int grp, int groups, const float* weights,
                                             const float4 (&first)[kBatch]) {
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  auto add = [&](float w, const float4& v) {
    acc.x += w * v.x;
    acc.y += w * v.y;
    acc.z += w * v.z;
    acc.w += w * v.w;
  };
#pragma unroll
  for (int j = 0; j < kBatch; ++j) {
    const int c = grp + j * groups;
    if (c < count) add(weights[c], first[j]);
  }
  for (int c0 = grp + kBatch * groups; c0 < count; c0 += 4 * groups) {
    float4 v[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j * groups < count) v[j] = __ldcg(reinterpret_cast<const float4*>(base + (size_t)(c0 + j * groups) * stride));
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (c0 + j * groups < count) add(weights[c0 + j * groups], v[j]);
  }
  return acc;
}
template <int kBatch>
__device__ __forceinline__ void request_quads(float4 (&v)[kBatch], const float* base, size_t stride, int count, int grp, int groups) {
#pragma unroll
  for (int j = 0; j < kBatch; ++j) {
    const int c = grp + j * groups;
    v[j] = c < count ? __ldcg(reinterpret_cast<const float4*>(base + (size_t)c * stride)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
}

}  // namespace
}  // namespace b200
