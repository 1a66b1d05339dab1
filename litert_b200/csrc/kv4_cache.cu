// A key/value cache held in 4 bits: storing tokens, reading slots back, evicting by accumulated attention weight
// (layout in kv4.h). Attention over it is in kv4_sdpa.cu.
#include <cooperative_groups.h>
#include <math_constants.h>

#include "common.cuh"
#include "kernels.h"
#include "kv4.h"

namespace b200 {

namespace {

namespace cg = cooperative_groups;

constexpr int kRowThreads = 256;

// ---- storing ---------------------------------------------------------------------------------------------
// Per block of channels: least = fp16(min), scale = fp16((max - least) / 15) with difference and quotient rounded to
// fp32, u = the integer nearest to (x - least) / scale (ties to even), clamped to 0 .. 15. Both roundings to fp16 happen
// before the nibbles are chosen, so that these are the best ones for the pair that is kept.
// Which integer is nearest is decided exactly: the fp32 quotient is off by 15 * 3 * 2^-24 at most, so only quotients that
// near to a border are looked at again, in 64 bits where difference and border are exact.
__device__ __forceinline__ uint32_t nearest_nibble(float x, float least, float scale, float inverse) {
  const float f = (x - least) * inverse;
  const float below = floorf(f);
  float u = rintf(f);
  if (fabsf(f - below - 0.5f) < 1e-5f) {
    const double d = (double)x - (double)least, border = ((double)below + 0.5) * (double)scale;
    u = d > border ? below + 1.0f : d < border ? below : u;
    if (d == border) u = 2.0f * rintf(0.5f * (below + 0.5f));  // the even neighbour
  }
  return (uint32_t)fminf(fmaxf(u, 0.0f), 15.0f);
}

// A thread takes 8 channels (one word of nibbles), block / 8 neighbouring lanes one block. Memory-bound.
template <bool F32>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(const Kv4Append p, const long long items, const int vec) {
  pdl_enter();
  const long long item = (long long)blockIdx.x * kRowThreads + threadIdx.x;
  const int words = p.cache.h / 8, lanes = p.cache.block / 8;
  const bool is_v = blockIdx.y != 0;
  bool live = item < items;
  long long row = live ? item / words : 0;  // (sequence, token, head)
  const int word = live ? (int)(item % words) : 0;
  const int kvh = (int)(row % p.cache.nkv);
  row /= p.cache.nkv;
  const int i = (int)(row % p.t), b = (int)(row / p.t);
  const long long slot = (long long)p.positions[b] + i;
  live = live && slot >= 0 && slot < p.cache.s && (!p.counts || i < p.counts[b]);
  float x[8];
  if (live) {
    const long long at = (is_v ? b * p.v_batch + i * p.v_token : b * p.k_batch + i * p.k_token) + (long long)kvh * p.cache.h + 8 * word;
    if constexpr (F32) {
      const float* src = static_cast<const float*>(is_v ? p.v : p.k) + at;
      if (vec) {
        const float4 lo = __ldg(reinterpret_cast<const float4*>(src)), hi = __ldg(reinterpret_cast<const float4*>(src) + 1);
        x[0] = lo.x, x[1] = lo.y, x[2] = lo.z, x[3] = lo.w, x[4] = hi.x, x[5] = hi.y, x[6] = hi.z, x[7] = hi.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __ldg(src + e);
      }
    } else {
      const __half* src = static_cast<const __half*>(is_v ? p.v : p.k) + at;
      if (vec) {
        const uint4 r = __ldg(reinterpret_cast<const uint4*>(src));
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[e]));
          x[2 * e] = f.x, x[2 * e + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = __half2float(src[e]);
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  }
  float lo = x[0], hi = x[0], bad = 0.0f;  // bad: NaN once any element is infinite or NaN
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    lo = fminf(lo, x[e]);
    hi = fmaxf(hi, x[e]);
    bad = fmaf(0.0f, x[e], bad);
  }
  for (int o = 1; o < lanes; o <<= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    bad += __shfl_xor_sync(0xffffffffu, bad, o);
  }
  __half least_h = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
  const float least = __half2float(least_h);
  __half scale_h = __float2half_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(hi, least), 15.0f), 0.0f), 65504.0f));
  const float scale = __half2float(scale_h);
  uint32_t bits = 0;
  if (bad != bad) {  // an infinity or NaN is not hidden: the block reads back as NaN
    least_h = scale_h = __ushort_as_half(0x7fff);
  } else if (scale > 0.0f) {
    const float inverse = 1.0f / scale;
#pragma unroll
    for (int e = 0; e < 8; ++e) bits |= nearest_nibble(x[e], least, scale, inverse) << (4 * e);
  }
  if (!live) return;
  const size_t to = ((size_t)b * p.cache.s + (size_t)slot) * p.cache.nkv + kvh;
  reinterpret_cast<uint32_t*>(is_v ? p.cache.v : p.cache.k)[to * words + word] = bits;
  if (word % lanes == 0) (is_v ? p.cache.v_pairs : p.cache.k_pairs)[to * (p.cache.h / p.cache.block) + word / lanes] = __halves2half2(scale_h, least_h);
}

// ---- reading back ----------------------------------------------------------------------------------------
template <bool F32>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(const Kv4Read p, const long long items) {
  pdl_enter();
  const long long item = (long long)blockIdx.x * kRowThreads + threadIdx.x;
  if (item >= items) return;
  const int words = p.cache.h / 8, lanes = p.cache.block / 8;
  const bool is_v = blockIdx.y != 0;
  long long row = item / words;
  const int word = (int)(item % words), kvh = (int)(row % p.cache.nkv);
  row /= p.cache.nkv;
  const int i = (int)(row % p.t), b = (int)(row / p.t);
  const long long slot = (p.positions ? (long long)p.positions[b] : 0) + i;
  const bool there = slot >= 0 && slot < p.cache.s && (!p.counts || i < p.counts[b]);
  float x[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
  if (there) {
    const size_t from = ((size_t)b * p.cache.s + (size_t)slot) * p.cache.nkv + kvh;
    const uint32_t bits = __ldg(reinterpret_cast<const uint32_t*>(is_v ? p.cache.v : p.cache.k) + from * words + word);
    const float2 sm = __half22float2(__ldg((is_v ? p.cache.v_pairs : p.cache.k_pairs) + from * (p.cache.h / p.cache.block) + word / lanes));
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = fmaf((float)((bits >> (4 * e)) & 15u), sm.x, sm.y);
  }
  if constexpr (F32) {
    float4* dst = reinterpret_cast<float4*>(static_cast<float*>(is_v ? p.v : p.k) + item * 8);
    dst[0] = make_float4(x[0], x[1], x[2], x[3]);
    dst[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const __half2 h = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
      w[e] = *reinterpret_cast<const uint32_t*>(&h);
    }
    *reinterpret_cast<uint4*>(static_cast<__half*>(is_v ? p.v : p.k) + item * 8) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// ---- eviction --------------------------------------------------------------------------------------------
// Order of scores as unsigned integers: larger score, larger key; the two zeros alike, NaN below everything.
__device__ __forceinline__ uint32_t score_key(float score) {
  if (score != score) return 0u;
  const uint32_t bits = __float_as_uint(score + 0.0f);  // -0 + 0 = +0
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}

constexpr int kEvictThreads = 512;
constexpr int kEvictWarps = kEvictThreads / 32;
constexpr int kEvictRowSmem = 160 * 1024;  // rows on their way

struct EvictShared {
  uint32_t hist[2][256];
  uint32_t digit, above;       // the digit that the threshold has, and how many keys lie above it
  uint32_t more, equal;        // this CTA's keys above / at the threshold
  uint32_t scan[2][kEvictWarps];
};

// One cluster per (sequence, KV head): its CTAs share the slots between them. The slots that neither the first `sinks`
// nor the last `recent` protect are ranked by a radix selection, 8 bits of the key a time: every CTA counts its slots'
// digits, the cluster adds the counts through distributed shared memory, and after four rounds the threshold and the
// number of slots at the threshold that stay (the lowest) are known. The kept slots' list is made by a scan in slot
// order.
// In place, rows move down (slot kept[j] >= j), so a pass of the cluster reads the rows of as many destinations as fit
// into its CTAs' shared memory, waits for the cluster, and writes them: what it overwrites has been read in this pass or
// an earlier one.
__global__ void __launch_bounds__(kEvictThreads, 1) kv4_evict_kernel(const Kv4Evict p, const int in_place) {
  extern __shared__ __align__(16) uint8_t rows_smem[];
  __shared__ EvictShared sh;
  cg::cluster_group cluster = cg::this_cluster();
  const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int pair = blockIdx.x / ctas, b = pair / p.from.nkv, kvh = pair % p.from.nkv;
  pdl_enter();
  const int length = max(0, min(p.lengths[b], p.from.s));
  const int left = min(length, p.budget);
  const float* scores = p.scores + (size_t)pair * p.from.s;
  float* scores_out = p.scores_out + (size_t)pair * p.to.s;
  int32_t* kept = p.kept + (size_t)pair * p.budget;
  if (kvh == 0 && rank == 0 && tid == 0) p.lengths_out[b] = left;
  // behind the kept slots
  for (int j = left + rank * kEvictThreads + tid; j < p.to.s; j += ctas * kEvictThreads) scores_out[j] = 0.0f;
  for (int j = left + rank * kEvictThreads + tid; j < p.budget; j += ctas * kEvictThreads) kept[j] = -1;
  const bool choose = length > p.budget;
  const int first = choose ? p.sinks : 0, behind = choose ? length - p.recent : 0;
  // protected slots (all of them where nothing is evicted)
  if (choose) {
    for (int j = rank * kEvictThreads + tid; j < p.sinks + p.recent; j += ctas * kEvictThreads) {
      const int slot = j < p.sinks ? j : behind + (j - p.sinks), to = j < p.sinks ? j : p.budget - p.recent + (j - p.sinks);
      kept[to] = slot;
      scores_out[to] = scores[slot];
    }
  } else {
    for (int j = rank * kEvictThreads + tid; j < left; j += ctas * kEvictThreads) {
      kept[j] = j;
      scores_out[j] = scores[j];
    }
  }
  const int wanted = choose ? p.budget - p.sinks - p.recent : 0;
  if (wanted > 0) {  // (uniform over the cluster)
    const int n = behind - first, share = (n + ctas - 1) / ctas;
    const int begin = first + min(n, rank * share), end = first + min(n, (rank + 1) * share);
    uint32_t prefix = 0, to_find = (uint32_t)wanted;  // the threshold is the to_find-th largest of the keys with this prefix
    for (int round = 0; round < 4; ++round) {
      const int shift = 24 - 8 * round;
      uint32_t* hist = sh.hist[round & 1];
      for (int i = tid; i < 256; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      for (int i = begin + tid; i < end; i += kEvictThreads) {
        const uint32_t key = score_key(__ldg(scores + i));
        if (round == 0 || (key >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(key >> shift) & 255u], 1u);
      }
      cluster.sync();
      if (warp == 0) {
        // lane l holds the digits 255 - 8 l .. 248 - 8 l: counts from the largest digit down
        uint32_t mine[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          mine[e] = 0;
          for (int c = 0; c < ctas; ++c) mine[e] += cluster.map_shared_rank(hist, c)[255 - 8 * lane - e];
          sum += mine[e];
        }
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
          if (lane >= o) upto += y;
        }
        uint32_t above = upto - sum;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (above < to_find && to_find <= above + mine[e]) {
            sh.digit = 255u - 8u * lane - e;
            sh.above = above;
          }
          above += mine[e];
        }
      }
      __syncthreads();
      prefix |= sh.digit << shift;
      to_find -= sh.above;
    }
    // slots above and at the threshold, here and in the CTAs before
    uint32_t more = 0, equal = 0;
    for (int i = begin + tid; i < end; i += kEvictThreads) {
      const uint32_t key = score_key(__ldg(scores + i));
      more += key > prefix;
      equal += key == prefix;
    }
    more = __reduce_add_sync(0xffffffffu, more);
    equal = __reduce_add_sync(0xffffffffu, equal);
    if (lane == 0) {
      sh.scan[0][warp] = more;
      sh.scan[1][warp] = equal;
    }
    __syncthreads();
    if (tid == 0) {
      more = equal = 0;
      for (int w = 0; w < kEvictWarps; ++w) {
        more += sh.scan[0][w];
        equal += sh.scan[1][w];
      }
      sh.more = more;
      sh.equal = equal;
    }
    cluster.sync();
    uint32_t more_before = 0, equal_before = 0;
    for (int c = 0; c < rank; ++c) {
      const EvictShared* other = cluster.map_shared_rank(&sh, c);
      more_before += other->more;
      equal_before += other->equal;
    }
    // (of the equal ones the first to_find stay)
    uint32_t taken = (uint32_t)first + more_before + min(equal_before, to_find);
    uint32_t equals = equal_before;
    for (int i0 = begin; i0 < end; i0 += kEvictThreads) {
      const int i = i0 + tid;
      const float score = i < end ? __ldg(scores + i) : 0.0f;
      const uint32_t key = i < end ? score_key(score) : 0u;
      const bool is_equal = i < end && key == prefix, is_more = i < end && key > prefix;
      const uint32_t eq_mask = __ballot_sync(0xffffffffu, is_equal), more_mask = __ballot_sync(0xffffffffu, is_more);
      __syncthreads();
      if (lane == 0) {
        sh.scan[0][warp] = __popc(more_mask);
        sh.scan[1][warp] = __popc(eq_mask);
      }
      __syncthreads();
      uint32_t m_before = 0, e_before = 0, m_all = 0, e_all = 0;
#pragma unroll
      for (int w = 0; w < kEvictWarps; ++w) {
        if (w == warp) m_before = m_all, e_before = e_all;
        m_all += sh.scan[0][w];
        e_all += sh.scan[1][w];
      }
      const uint32_t lower = (1u << lane) - 1u;
      m_before += __popc(more_mask & lower);
      e_before += __popc(eq_mask & lower);
      const uint32_t room = to_find > equals ? to_find - equals : 0u;  // equal ones that may still stay
      if (is_more || (is_equal && e_before < room)) {
        const uint32_t to = taken + m_before + min(e_before, room);
        kept[to] = i;
        scores_out[to] = score;
      }
      taken += m_all + min(e_all, room);
      equals += e_all;
    }
  }
  if (in_place && !choose) return;  // (uniform over the cluster, and before any barrier of it)
  __threadfence();
  cluster.sync();  // the list is complete; no CTA's shared memory is read any more
  // ---- rows ----
  const int nibbles = p.from.h / 2, groups = p.from.h / p.from.block;
  const int row_bytes = 2 * nibbles + 8 * groups, row_pad = (row_bytes + 15) / 16 * 16;
  const int chunks = nibbles / 16, parts = 2 * chunks + 2 * groups;  // 16-byte pieces of nibbles, then 4-byte pairs
  const int fit = kEvictRowSmem / row_pad;
  for (int j0 = in_place ? p.sinks : 0; j0 < left; j0 += ctas * fit) {
    const int r0 = j0 + rank * fit, rows = max(0, min(fit, left - r0));
    for (int e = tid; e < rows * parts; e += kEvictThreads) {
      const int r = e / parts, part = e % parts;
      const size_t at = ((size_t)b * p.from.s + (size_t)__ldcg(kept + r0 + r)) * p.from.nkv + kvh;
      uint8_t* dst = rows_smem + (size_t)r * row_pad;
      if (part < 2 * chunks) {
        const uint8_t* src = (part < chunks ? p.from.k : p.from.v) + at * nibbles + (part % chunks) * 16;
        *reinterpret_cast<uint4*>(dst + part * 16) = __ldcg(reinterpret_cast<const uint4*>(src));
      } else {
        const int g = part - 2 * chunks;
        const uint32_t* src = reinterpret_cast<const uint32_t*>(g < groups ? p.from.k_pairs : p.from.v_pairs) + at * groups + g % groups;
        *reinterpret_cast<uint32_t*>(dst + 2 * nibbles + 4 * g) = __ldcg(src);
      }
    }
    if (in_place) {
      cluster.sync();
    } else {
      __syncthreads();
    }
    for (int e = tid; e < rows * parts; e += kEvictThreads) {
      const int r = e / parts, part = e % parts;
      const size_t at = ((size_t)b * p.to.s + (size_t)(r0 + r)) * p.to.nkv + kvh;
      const uint8_t* src = rows_smem + (size_t)r * row_pad;
      if (part < 2 * chunks) {
        uint8_t* dst = (part < chunks ? p.to.k : p.to.v) + at * nibbles + (part % chunks) * 16;
        *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src + part * 16);
      } else {
        const int g = part - 2 * chunks;
        reinterpret_cast<uint32_t*>(g < groups ? p.to.k_pairs : p.to.v_pairs)[at * groups + g % groups] =
            *reinterpret_cast<const uint32_t*>(src + 2 * nibbles + 4 * g);
      }
    }
    __syncthreads();
  }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4Append& p, cudaStream_t s) {
  const long long items = (long long)p.cache.b * p.t * p.cache.nkv * (p.cache.h / 8);
  if (items == 0) return cudaSuccess;
  const int elem = p.f32 ? 4 : 2, per = 16 / elem;  // elements of a 16-byte load
  const bool vec = ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) == 0 &&
                   p.k_batch % per == 0 && p.k_token % per == 0 && p.v_batch % per == 0 && p.v_token % per == 0;
  const dim3 grid((unsigned)((items + kRowThreads - 1) / kRowThreads), 2);
  return p.f32 ? launch_chained(kv4_append_kernel<true>, grid, dim3(kRowThreads), 0, s, p, items, vec ? 1 : 0)
               : launch_chained(kv4_append_kernel<false>, grid, dim3(kRowThreads), 0, s, p, items, vec ? 1 : 0);
}

cudaError_t launch_kv4_read(const Kv4Read& p, cudaStream_t s) {
  const long long items = (long long)p.cache.b * p.t * p.cache.nkv * (p.cache.h / 8);
  if (items == 0) return cudaSuccess;
  const dim3 grid((unsigned)((items + kRowThreads - 1) / kRowThreads), 2);
  return p.f32 ? launch_chained(kv4_read_kernel<true>, grid, dim3(kRowThreads), 0, s, p, items)
               : launch_chained(kv4_read_kernel<false>, grid, dim3(kRowThreads), 0, s, p, items);
}

cudaError_t launch_kv4_evict(const Kv4Evict& p, cudaStream_t s) {
  const int pairs = p.from.b * p.from.nkv;
  if (pairs == 0) return cudaSuccess;
  static bool done[64] = {false};
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kv4_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictRowSmem);
    if (e != cudaSuccess) return e;
    done[dev] = true;
  }
  int ctas = 8;
  while (ctas > 1 && (long long)pairs * ctas > 2ll * device_sm_count()) ctas /= 2;
  return launch_chained_cluster(kv4_evict_kernel, dim3((unsigned)(pairs * ctas)), dim3(kEvictThreads), (size_t)kEvictRowSmem, ctas, s, p,
                                p.from.k == p.to.k ? 1 : 0);
}

}  // namespace b200
