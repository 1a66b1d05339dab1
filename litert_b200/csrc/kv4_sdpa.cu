// Attention over a key/value cache held in 4 bits (layout in kv4.h).
//
// For query row r (query token i of t, head n) and the attended slots s of its KV head:
//   x_s = scale * q . k_s [cap * tanh(x / cap)] [+ mask],  out = sum_s softmax(x)_s v_s,  scores_s += softmax(x)_s
// With nibbles u and pairs (a, m) per block g of channels, the dequantized rows never exist:
//   q . k_s = sum_g a_sg (sum_c u_sc q_c) + m_sg (sum_c q_c)
//   out_c   = sum_s (p_s a_sg) u_sc + sum_s p_s m_sg
// Products of a nibble and an fp16 number are exact and are added in fp32.
#include <math_constants.h>

#include "common.cuh"
#include "kernels.h"
#include "kv4.h"

namespace b200 {

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// ---- any head size --------------------------------------------------------------------------------------
// One CTA per query row: logits to the workspace, then the softmax, then a thread per channel. For head sizes that the
// tensor-core kernel does not take.
struct RowsWorkspace {
  float* logits;  // [b, t, n, s]
  float2* stats;  // [b, t, n]: maximum, sum
};
__host__ __device__ inline RowsWorkspace rows_workspace(float* ws, int b, int t, int n, int s) {
  const size_t rows = (size_t)b * t * n;
  return {ws + 2 * rows, reinterpret_cast<float2*>(ws)};
}

constexpr int kRowsThreads = 256;

__device__ __forceinline__ float block_reduce(float v, bool max, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float y = __shfl_xor_sync(0xffffffffu, v, o);
    v = max ? fmaxf(v, y) : v + y;
  }
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < kRowsThreads / 32; ++w) v = max ? fmaxf(v, red[w]) : v + red[w];
  return v;
}

__global__ void __launch_bounds__(kRowsThreads) kv4_sdpa_rows_kernel(const Kv4Sdpa p) {
  __shared__ float q[512];
  __shared__ float q_sum[16];
  __shared__ float red[kRowsThreads / 32];
  pdl_enter();
  const int head = blockIdx.x, i = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int h = p.cache.h, s = p.cache.s, nkv = p.cache.nkv, block = p.cache.block, groups = h / block, words = h / 8;
  const int kvh = head / (p.n / nkv);
  const size_t row = ((size_t)b * p.t + i) * p.n + head;
  const RowsWorkspace ws = rows_workspace(p.ws, p.cache.b, p.t, p.n, s);
  float* logits = ws.logits + row * s;
  for (int c = tid; c < h; c += kRowsThreads)
    q[c] = p.f32 ? static_cast<const float*>(p.q)[row * h + c] : __half2float(static_cast<const __half*>(p.q)[row * h + c]);
  __syncthreads();
  if (tid < groups) {
    float sum = 0.0f;
    for (int c = 0; c < block; ++c) sum += q[tid * block + c];
    q_sum[tid] = sum;
  }
  __syncthreads();
  const int limit = kv4_limit(p.lengths ? p.lengths[b] : s, s, p.t, i);
  const float* mask = p.mask ? p.mask + ((size_t)b * p.t + i) * s : nullptr;
  float top = -CUDART_INF_F;
  for (int slot = tid; slot < limit; slot += kRowsThreads) {
    const size_t at = ((size_t)b * s + slot) * nkv + kvh;
    const uint32_t* nib = reinterpret_cast<const uint32_t*>(p.cache.k) + at * words;
    float x = 0.0f;
    for (int g = 0; g < groups; ++g) {
      float dot = 0.0f;
      for (int w = g * block / 8; w < (g + 1) * block / 8; ++w) {
        const uint32_t bits = nib[w];
#pragma unroll
        for (int e = 0; e < 8; ++e) dot = fmaf((float)((bits >> (4 * e)) & 15u), q[8 * w + e], dot);
      }
      const float2 am = __half22float2(p.cache.k_pairs[at * groups + g]);
      x = fmaf(am.x, dot, fmaf(am.y, q_sum[g], x));
    }
    x *= p.scale;
    if (p.logit_cap > 0.0f) x = p.logit_cap * tanhf(x / p.logit_cap);
    if (mask) {
      const float m = mask[slot];
      x = m == -CUDART_INF_F ? m : x + m;  // (whatever the slot holds)
    }
    logits[slot] = x;
    top = fmaxf(top, x);
  }
  top = block_reduce(top, true, red);
  const float use = top == -CUDART_INF_F ? 0.0f : top;
  float sum = 0.0f;
  for (int slot = tid; slot < limit; slot += kRowsThreads) sum += exp2f((logits[slot] - use) * kLog2e);
  sum = block_reduce(sum, false, red);
  if (tid == 0) ws.stats[row] = make_float2(use, sum);
  __syncthreads();
  const bool empty = sum == 0.0f;
  for (int c = tid; c < h; c += kRowsThreads) {
    float acc = 0.0f;
    for (int slot = 0; slot < limit; ++slot) {
      const float w = exp2f((logits[slot] - use) * kLog2e);
      const size_t at = ((size_t)b * s + slot) * nkv + kvh;
      const uint32_t bits = reinterpret_cast<const uint32_t*>(p.cache.v)[at * words + c / 8];
      const float2 am = __half22float2(p.cache.v_pairs[at * groups + c / block]);
      if (w != 0.0f) acc = fmaf(w, fmaf((float)((bits >> (4 * (c % 8))) & 15u), am.x, am.y), acc);
    }
    const float o = empty ? 0.0f : acc / sum;
    if (p.f32) {
      static_cast<float*>(p.out)[row * h + c] = o;
    } else {
      static_cast<__half*>(p.out)[row * h + c] = __float2half_rn(o);
    }
  }
}

__global__ void __launch_bounds__(kRowsThreads) kv4_rows_scores_kernel(const Kv4Sdpa p) {
  pdl_enter();
  const int s = p.cache.s, nkv = p.cache.nkv, group = p.n / nkv, b = blockIdx.z, kvh = blockIdx.y;
  const int slot = blockIdx.x * kRowsThreads + threadIdx.x;
  const int length = kv4_limit(p.lengths ? p.lengths[b] : s, s, p.t, p.t - 1);
  if (slot >= length) return;
  const RowsWorkspace ws = rows_workspace(p.ws, p.cache.b, p.t, p.n, s);
  float sum = 0.0f;
  for (int i = 0; i < p.t; ++i) {
    if (slot >= kv4_limit(length, s, p.t, i)) continue;
    for (int j = 0; j < group; ++j) {
      const size_t row = ((size_t)b * p.t + i) * p.n + kvh * group + j;
      const float2 st = ws.stats[row];
      if (st.y != 0.0f) sum += exp2f((ws.logits[row * s + slot] - st.x) * kLog2e) / st.y;
    }
  }
  p.scores[((size_t)b * nkv + kvh) * s + slot] += sum;
}

cudaError_t launch_rows(const Kv4Sdpa& p, cudaStream_t s) {
  cudaError_t e = launch_chained(kv4_sdpa_rows_kernel, dim3(p.n, p.t, p.cache.b), dim3(kRowsThreads), 0, s, p);
  if (e != cudaSuccess || !p.scores) return e;
  return launch_chained(kv4_rows_scores_kernel, dim3((p.cache.s + kRowsThreads - 1) / kRowsThreads, p.cache.nkv, p.cache.b),
                        dim3(kRowsThreads), 0, s, p);
}

}  // namespace

size_t kv4_sdpa_workspace_bytes(int b, int t, int n, int nkv, int h, int s, int block, int scores) {
  const size_t rows = (size_t)b * t * n;
  return (2 * rows + rows * s) * sizeof(float);
}

cudaError_t launch_kv4_sdpa(const Kv4Sdpa& p, cudaStream_t s) { return launch_rows(p, s); }

}  // namespace b200
