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

// n / d for n below 2^31: a product and a shift, the factor made on the host.
struct Divisor {
  uint32_t d, factor, shift;
};
Divisor divisor(uint32_t d) {
  uint32_t bits = 0;
  while ((1ull << bits) < d) ++bits;
  return {d, (uint32_t)(((1ull << (31 + bits)) + d - 1) / d), 31 + bits};
}
__device__ __forceinline__ uint32_t operator/(uint32_t n, const Divisor& by) { return (uint32_t)(((uint64_t)n * by.factor) >> by.shift); }

// ---- storing ---------------------------------------------------------------------------------------------
// Per block of channels: least = fp16(min), scale = fp16((max - least) / 15) with difference and quotient rounded to
// fp32, u = the integer nearest to (x - least) / scale (ties to even), clamped to 0 .. 15. Both roundings to fp16 happen
// before the nibbles are chosen, so that these are the best ones for the pair that is kept.
// Which integer is nearest is decided exactly: y = (x - least) / (15 scale), clamped for free by the product's saturation,
// is off by 3 x 2^-23 of itself at most (the reciprocal 2 of them, difference and product half of one each), so 15 y by 5.4e-6;
// only what comes within 1e-5 of a border is looked at again, against the border itself: least + (k + 1/2) scale is a multiple
// of 2^-25 below 2^21, exact in 64 bits. (The difference x - least need not be.)
//
// Memory-bound by its bytes, but really by instruction issue: 67 M elements at 36 T lane operations per second leave 12
// operations for each in the time that HBM takes, and it has 19. So 16 channels per thread (block / 16 neighbouring lanes have
// one block), the minimum and the negated maximum of fp16 rows as one pair of halves, nibbles put together by fused products.
// 16 x 8192 rows of 256 in fp16: 53 us of the 26 that their bytes take (issue slots 75 % busy); 16 x 4096 in float32 32 of 23.
__device__ __forceinline__ float nearest_float(float n, float x, float least, float scale) {
  const float below = n * scale > x - least ? n - 1.0f : n;  // the border lies above it
  const double border = (double)least + ((double)below + 0.5) * (double)scale;
  const float u = x > border ? below + 1.0f : x < border ? below : 2.0f * rintf(0.5f * (below + 0.5f));  // (ties: the even neighbour)
  return fminf(fmaxf(u, 0.0f), 15.0f);
}
__device__ __forceinline__ float min_nan(float a, float b) {  // NaN if either is
  float y;
  asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {
  float y;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
  return y;
}

template <bool F32>
struct Sixteen {  // channels, as they lie in memory
  uint32_t w[F32 ? 16 : 8];
};

// One block's nibbles of a thread's 16 channels, and the block's pair. `lanes_log2`: log2 of the lanes that have the block.
template <bool F32>
__device__ __forceinline__ void quantize_sixteen(const Sixteen<F32>& in, int lanes_log2, uint2& word, __half2& pair) {
  float x[16], lo, hi;
  if constexpr (F32) {
#pragma unroll
    for (int e = 0; e < 16; ++e) x[e] = __uint_as_float(in.w[e]);
    lo = hi = x[0];
#pragma unroll
    for (int e = 1; e < 16; ++e) {
      lo = min_nan(lo, x[e]);
      hi = max_nan(hi, x[e]);
    }
    for (int o = 1; o < 1 << lanes_log2; o <<= 1) {
      lo = min_nan(lo, __shfl_xor_sync(0xffffffffu, lo, o));
      hi = max_nan(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
  } else {
    __half2 least2 = *reinterpret_cast<const __half2*>(&in.w[0]), most2 = least2;
#pragma unroll
    for (int e = 1; e < 8; ++e) {
      least2 = __hmin2_nan(least2, *reinterpret_cast<const __half2*>(&in.w[e]));
      most2 = __hmax2_nan(most2, *reinterpret_cast<const __half2*>(&in.w[e]));
    }
    // (minimum, -maximum)
    __half2 both = __halves2half2(__hmin_nan(__low2half(least2), __high2half(least2)), __hneg(__hmax_nan(__low2half(most2), __high2half(most2))));
    for (int o = 1; o < 1 << lanes_log2; o <<= 1) {
      const uint32_t other = __shfl_xor_sync(0xffffffffu, *reinterpret_cast<const uint32_t*>(&both), o);
      both = __hmin2_nan(both, *reinterpret_cast<const __half2*>(&other));
    }
    lo = __low2float(both);
    hi = -__high2float(both);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&in.w[e]));
      x[2 * e] = f.x, x[2 * e + 1] = f.y;
    }
  }
  const bool bad = !(fabsf(lo) < CUDART_INF_F && fabsf(hi) < CUDART_INF_F);  // an infinity or NaN is not hidden: the block reads back as NaN
  __half least_h = __float2half_rn(fminf(fmaxf(lo, -65504.0f), 65504.0f));
  const float least = __half2float(least_h);
  __half scale_h = __float2half_rn(fminf(fmaxf(__fdiv_rn(__fsub_rn(hi, least), 15.0f), 0.0f), 65504.0f));
  const float scale = __half2float(scale_h);
  if (bad) least_h = scale_h = __ushort_as_half(0x7fff);
  pair = __halves2half2(scale_h, least_h);
  // (a factor of zero, and whatever it meets, saturates to zero)
  const float inverse = bad || scale == 0.0f ? 0.0f : __fdividef(1.0f, 15.0f * scale);
  float n[16], far = 0.0f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float y = __saturatef((x[e] - least) * inverse);
    n[e] = fmaf(y, 15.0f, 12582912.0f) - 12582912.0f;  // rounded by the sum's last place
    far = fmaxf(far, fabsf(fmaf(y, 15.0f, -n[e])));
  }
  if (far > 0.49999f) {  // (a quarter of the warps of fp16 rows: exact ties among 512 elements; each of them seldom)
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float y = __saturatef((x[e] - least) * inverse);
      if (fabsf(fmaf(y, 15.0f, -n[e])) > 0.49999f) n[e] = nearest_float(n[e], x[e], least, scale);
    }
  }
  uint32_t out[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const float* m = n + 8 * e;
    // (sums below 2^16, exact; a number added to 2^23 is its low bits)
    const float low = fmaf(fmaf(m[3], 16.0f, m[2]), 256.0f, fmaf(m[1], 16.0f, m[0])) + 8388608.0f;
    const float high = fmaf(fmaf(m[7], 16.0f, m[6]), 256.0f, fmaf(m[5], 16.0f, m[4])) + 8388608.0f;
    out[e] = __byte_perm(__float_as_uint(low), __float_as_uint(high), 0x5410);
  }
  word = make_uint2(out[0], out[1]);
}

// A thread walks over a sequence's pieces of 16 channels, the next one asked for before this one is used: what does not
// depend on the piece is a third of the instructions otherwise.
template <bool F32>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(const Kv4Append p, const uint32_t items, const Divisor per_token, const int lanes_log2,
                                                                 const int vec) {
  constexpr int kElem = F32 ? 4 : 2;
  pdl_enter();
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const uint8_t* src = static_cast<const uint8_t*>(is_v ? p.v : p.k) + (is_v ? p.v_batch : p.k_batch) * b * kElem;
  const long long token = (is_v ? p.v_token : p.k_token) * kElem;
  const long long position = p.positions[b];
  const int count = p.counts ? min(p.counts[b], p.t) : p.t;
  // tokens that have a slot
  const int first = (int)max(0ll, min((long long)INT32_MAX, -position)), behind = (int)max(0ll, min((long long)count, (long long)p.cache.s - position));
  uint8_t* nibbles = (is_v ? p.cache.v : p.cache.k) + ((long long)b * p.cache.s + position) * per_token.d * 8;
  __half2* pairs = (is_v ? p.cache.v_pairs : p.cache.k_pairs) + ((((long long)b * p.cache.s + position) * per_token.d) >> lanes_log2);
  auto ask = [&](uint32_t item, Sixteen<F32>& in) {
    const uint32_t i = item / per_token, rest = item - i * per_token.d;
    const bool live = item < items && (int)i >= first && (int)i < behind;  // (alike for the lanes of a block)
    if (live) {
      const uint8_t* at = src + i * token + (size_t)rest * 16 * kElem;
      if (vec) {
#pragma unroll
        for (int e = 0; e < (F32 ? 4 : 2); ++e) {
          const uint4 v = __ldg(reinterpret_cast<const uint4*>(at) + e);
          in.w[4 * e] = v.x, in.w[4 * e + 1] = v.y, in.w[4 * e + 2] = v.z, in.w[4 * e + 3] = v.w;
        }
      } else if constexpr (F32) {
#pragma unroll
        for (int e = 0; e < 16; ++e) in.w[e] = __ldg(reinterpret_cast<const uint32_t*>(at) + e);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          in.w[e] = __ldg(reinterpret_cast<const unsigned short*>(at) + 2 * e) | (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(at) + 2 * e + 1) << 16;
      }
    }
    return live;
  };
  const uint32_t step = gridDim.x * kRowThreads;
  uint32_t item = blockIdx.x * kRowThreads + threadIdx.x;
  Sixteen<F32> next;
#pragma unroll
  for (int e = 0; e < (F32 ? 16 : 8); ++e) next.w[e] = 0;
  bool next_live = ask(item, next);
  for (uint32_t front = blockIdx.x * kRowThreads; front < items; front += step) {  // (the block's first: all lanes stay)
    const Sixteen<F32> in = next;
    const bool live = next_live;
    const uint32_t now = item;
    item += step;
    next_live = ask(item, next);
    uint2 word;
    __half2 pair;
    quantize_sixteen<F32>(in, lanes_log2, word, pair);
    if (live) {
      *reinterpret_cast<uint2*>(nibbles + (size_t)now * 8) = word;
      if ((now & ((1u << lanes_log2) - 1)) == 0) pairs[now >> lanes_log2] = pair;
    }
  }
}

// ---- reading back ----------------------------------------------------------------------------------------
// A thread takes two words of nibbles, 256 apart, so that a warp's stores of fp16 rows are whole lines. fp16 values are fused
// products of halves: one rounding. fp16 is bound by HBM: 16 x 8192 rows of 256 29.3 us (26 for the bytes). float32 is not: a lane's
// two stores of 16 bytes lie 32 apart from its neighbour's, so each fills half of every sector; 16 x 4096 rows 35 us (23).
template <bool F32>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(const Kv4Read p, const uint32_t items, const Divisor per_token, const int words_log2) {
  pdl_enter();
  const int b = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const uint32_t* nibbles = reinterpret_cast<const uint32_t*>(is_v ? p.cache.v : p.cache.k);
  const __half2* pairs = is_v ? p.cache.v_pairs : p.cache.k_pairs;
  const long long position = p.positions ? (long long)p.positions[b] : 0;
  const int count = p.counts ? p.counts[b] : p.t;
  uint32_t w[2];
  __half2 pair[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t item = blockIdx.x * (2 * kRowThreads) + e * kRowThreads + threadIdx.x;
    const uint32_t i = item / per_token, rest = item - i * per_token.d;
    const long long slot = position + i;
    w[e] = 0;
    pair[e] = __float2half2_rn(0.0f);
    if (item < items && slot >= 0 && slot < p.cache.s && (int)i < count) {
      const size_t from = ((size_t)b * p.cache.s + (size_t)slot) * per_token.d + rest;
      w[e] = __ldg(nibbles + from);
      pair[e] = __ldg(pairs + (from >> words_log2));
    }
  }
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    const uint32_t item = blockIdx.x * (2 * kRowThreads) + e * kRowThreads + threadIdx.x;
    if (item >= items) return;
    const size_t to = ((size_t)b * items + item) * 8;
    if constexpr (F32) {
      const float2 sm = __half22float2(pair[e]);
      float x[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) x[k] = fmaf(__uint_as_float(((w[e] >> (4 * k)) & 15u) | 0x4b000000u) - 8388608.0f, sm.x, sm.y);
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(is_v ? p.v : p.k) + to);
      dst[0] = make_float4(x[0], x[1], x[2], x[3]);
      dst[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      const __half2 s2 = __low2half2(pair[e]), m2 = __high2half2(pair[e]), bias = __float2half2_rn(1024.0f);
      uint32_t v[4];  // nibbles k and k + 4
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t bits = ((w[e] >> (4 * k)) & 0x000f000fu) | 0x64006400u;
        const __half2 y = __hfma2(__hsub2(*reinterpret_cast<const __half2*>(&bits), bias), s2, m2);
        v[k] = *reinterpret_cast<const uint32_t*>(&y);
      }
      *reinterpret_cast<uint4*>(static_cast<__half*>(is_v ? p.v : p.k) + to) =
          make_uint4(__byte_perm(v[0], v[1], 0x5410), __byte_perm(v[2], v[3], 0x5410), __byte_perm(v[0], v[1], 0x7632), __byte_perm(v[2], v[3], 0x7632));
    }
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
constexpr int kEvictSmem = 104 * 1024, kEvictMostSmem = 216 * 1024;  // rows on their way; before that two histograms
constexpr int kDigitBits = 11, kDigits = 1 << kDigitBits, kPerThread = kDigits / kEvictThreads;
constexpr int kWholeSlots = 8192;

struct EvictShared {
  uint32_t digit, above;       // the digit that the threshold has, and how many keys lie above it
  uint32_t more, equal;        // this CTA's keys above / at the threshold
  uint32_t scan[2][kEvictWarps];
};

// One cluster per (sequence, KV head): its CTAs share the slots between them. The slots that neither the first `sinks`
// nor the last `recent` protect are ranked by a radix selection, 11 bits of the key a time (the first digit is sign,
// exponent and two bits more: scores of one order of magnitude do not all count in one word): every CTA counts its slots'
// digits, adds the cluster's counts of a share of the digits through distributed shared memory and hands the sums round,
// and after three rounds the threshold and the number of slots at the threshold that stay (the lowest) are known. (All
// digits' counts read from all CTAs by everybody: 20 us a round.) Up to 8192 slots every CTA counts all of them instead:
// they stay in its L1, and no round waits for the cluster. The kept slots' list is made by a scan in slot order.
// In place, rows move down (slot kept[j] >= j), so a pass of the cluster reads the rows of as many destinations as fit
// into its CTAs' shared memory, waits for the cluster, and writes them: what it overwrites has been read in this pass or
// an earlier one.
// Bound by round trips and barriers, not by its bytes. 16 pairs of 4352 slots cut to 4096 in place: 19.0 us on clusters of 6 (the
// kept rows, read and written, are 5.8 us of HBM time); the counts end at 5.7 us, the list at 8, the rows' reading at 13.5.
// 32 pairs of 32768 to 2048 into another cache: 23.5 us on clusters of 4, counts to 11 us, list to 14.5.
__global__ void __launch_bounds__(kEvictThreads, 2) kv4_evict_kernel(const Kv4Evict p, const int in_place, const int row_log2, const int smem_bytes) {
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
    const int begin = first + min(n, rank * share), end = first + min(n, (rank + 1) * share);  // this CTA's slots
    const bool whole = n <= kWholeSlots || ctas == 1;
    const int count_begin = whole ? first : begin, count_end = whole ? behind : end;
    // the first count leaves the keys in shared memory for the others, where they fit
    uint32_t* keys = reinterpret_cast<uint32_t*>(rows_smem) + 2 * kDigits;
    const bool keep = 4 * (long long)(count_end - count_begin) + 8 * kDigits <= smem_bytes;
    auto key_of = [&](int i) { return keep ? keys[i - count_begin] : score_key(__ldg(scores + i)); };
    uint32_t prefix = 0, to_find = (uint32_t)wanted;  // the threshold is the to_find-th largest of the keys with this prefix
    int shift = 32;
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
      const int above = shift;
      shift = max(0, shift - kDigitBits);
      const uint32_t mask = (1u << (above - shift)) - 1u;
      uint32_t *hist = reinterpret_cast<uint32_t*>(rows_smem), *sums = hist + kDigits;
      for (int i = tid; i < kDigits; i += kEvictThreads) hist[i] = 0;
      __syncthreads();
      if (round == 0) {
#pragma unroll 4
        for (int i = count_begin + tid; i < count_end; i += kEvictThreads) {
          const uint32_t key = score_key(__ldg(scores + i));
          if (keep) keys[i - count_begin] = key;
          atomicAdd(&hist[key >> shift], 1u);
        }
      } else {
#pragma unroll 4
        for (int i = count_begin + tid; i < count_end; i += kEvictThreads) {
          const uint32_t key = key_of(i);  // (a thread's own)
          if ((key ^ prefix) >> above == 0) atomicAdd(&hist[(key >> shift) & mask], 1u);
        }
      }
      if (whole) {
        __syncthreads();
        sums = hist;
      } else {
        cluster.sync();
        const int slice = (kDigits + ctas - 1) / ctas;
        for (int i = rank * slice + tid; i < min(kDigits, (rank + 1) * slice); i += kEvictThreads) {
          uint32_t all = 0;
          for (int c = 0; c < ctas; ++c) all += cluster.map_shared_rank(hist, c)[i];
          for (int c = 0; c < ctas; ++c) cluster.map_shared_rank(sums, c)[i] = all;
        }
        cluster.sync();
      }
      // thread t holds the digits 2047 - 4 t .. 2044 - 4 t: counts from the largest digit down
      uint32_t mine[kPerThread], sum = 0;
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) mine[e] = sums[kDigits - 1 - kPerThread * tid - e];
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) sum += mine[e];
      uint32_t upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      if (lane == 31) sh.scan[0][warp] = upto;
      __syncthreads();
      uint32_t greater = upto - sum;
#pragma unroll
      for (int w = 0; w < kEvictWarps; ++w) greater += w < warp ? sh.scan[0][w] : 0u;
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) {
        if (greater < to_find && to_find <= greater + mine[e]) {
          sh.digit = (uint32_t)(kDigits - 1 - kPerThread * tid - e);
          sh.above = greater;
        }
        greater += mine[e];
      }
      __syncthreads();
      prefix |= sh.digit << shift;
      to_find -= sh.above;
    }
    // slots above and at the threshold: this CTA's (whole: those in front of its own)
    uint32_t more = 0, equal = 0;
#pragma unroll 4
    for (int i = (whole ? first : begin) + tid; i < (whole ? begin : end); i += kEvictThreads) {
      const uint32_t key = key_of(i);
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
    more = equal = 0;
#pragma unroll
    for (int w = 0; w < kEvictWarps; ++w) {
      more += sh.scan[0][w];
      equal += sh.scan[1][w];
    }
    if (!whole) {
      if (tid == 0) {
        sh.more = more;
        sh.equal = equal;
      }
      cluster.sync();
      more = equal = 0;
      for (int c = 0; c < rank; ++c) {
        const EvictShared* other = cluster.map_shared_rank(&sh, c);
        more += other->more;
        equal += other->equal;
      }
    }
    // (of the equal ones the first to_find stay)
    uint32_t taken = (uint32_t)first + more + min(equal, to_find);
    uint32_t equals = equal;
    // four neighbouring slots per thread; counts of slots above (low half) and at the threshold (high half) as one number
    for (int i0 = begin; i0 < end; i0 += 4 * kEvictThreads) {
      const int mine = i0 + 4 * tid;
      float score[4];
      uint32_t kind[4], sum = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        score[e] = mine + e < end ? __ldg(scores + mine + e) : 0.0f;
        const uint32_t key = score_key(score[e]);
        kind[e] = mine + e >= end ? 0u : key > prefix ? 1u : key == prefix ? 0x10000u : 0u;
        sum += kind[e];
      }
      uint32_t upto = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      __syncthreads();
      if (lane == 31) sh.scan[0][warp] = upto;
      __syncthreads();
      uint32_t before = upto - sum, all = 0;
#pragma unroll
      for (int w = 0; w < kEvictWarps; ++w) {
        const uint32_t v = sh.scan[0][w];
        before += w < warp ? v : 0u;
        all += v;
      }
      const uint32_t room = to_find > equals ? to_find - equals : 0u;  // equal ones that may still stay
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t m_before = before & 0xffffu, e_before = before >> 16;
        if (kind[e] == 1u || (kind[e] != 0u && e_before < room)) {
          const uint32_t to = taken + m_before + min(e_before, room);
          kept[to] = mine + e;
          scores_out[to] = score[e];
        }
        before += kind[e];
      }
      taken += (all & 0xffffu) + min(all >> 16, room);
      equals += all >> 16;
    }
  }
  if (in_place && !choose) return;  // (uniform over the cluster, and before any barrier of it)
  __threadfence();
  cluster.sync();  // the list is complete; no CTA's shared memory is read any more
  // ---- rows ----
  // A row's 16-byte pieces of nibbles and its 4-byte pairs lie side by side over 2^row_log2 lanes (row_log2 may be 6: two
  // turns of a warp); all of a pass are asked for before the first is put down.
  const int nibbles = p.from.h / 2, groups = p.from.h / p.from.block;
  const int row_bytes = 2 * nibbles + 8 * groups, row_pad = (row_bytes + 15) / 16 * 16;
  const int chunks = nibbles / 16, parts = 2 * chunks + 2 * groups;
  const int part = tid & ((1 << row_log2) - 1), row_of = tid >> row_log2, rows_at_once = kEvictThreads >> row_log2;
  const bool is_pair = part >= 2 * chunks, is_v = is_pair ? part - 2 * chunks >= groups : part >= chunks;
  const int within = is_pair ? (part - 2 * chunks) % groups * 4 : part % chunks * 16, pitch = is_pair ? 4 * groups : nibbles;
  const uint8_t* from = is_pair ? reinterpret_cast<const uint8_t*>(is_v ? p.from.v_pairs : p.from.k_pairs) : is_v ? p.from.v : p.from.k;
  uint8_t* to = is_pair ? reinterpret_cast<uint8_t*>(is_v ? p.to.v_pairs : p.to.k_pairs) : is_v ? p.to.v : p.to.k;
  const size_t from_step = (size_t)p.from.nkv * pitch, to_step = (size_t)p.to.nkv * pitch;
  from += ((size_t)b * p.from.s * p.from.nkv + kvh) * pitch + within;
  to += ((size_t)b * p.to.s * p.to.nkv + kvh) * pitch + within;
  const int fit = smem_bytes / (row_pad + 4);  // rows, and their slots
  int32_t* slots = reinterpret_cast<int32_t*>(rows_smem + (size_t)fit * row_pad);
  const uint32_t mine = smem_u32(rows_smem) + (uint32_t)(is_pair ? 2 * nibbles + (part - 2 * chunks) * 4 : part * 16);
  const bool live = part < parts;
  const int j_first = in_place ? p.sinks : 0, each = min(fit, (left - j_first + ctas - 1) / ctas);
  for (int j0 = j_first; j0 < left; j0 += ctas * each) {
    const int r0 = j0 + rank * each, rows = max(0, min(each, left - r0));
    __syncthreads();  // (the slots of the pass before have been used)
    for (int r = tid; r < rows; r += kEvictThreads) slots[r] = __ldcg(kept + r0 + r);
    __syncthreads();
    if (live) {
      for (int r = row_of; r < rows; r += rows_at_once) {
        const uint8_t* src = from + slots[r] * from_step;
        const uint32_t dst = mine + (uint32_t)(r * row_pad);
        if (is_pair) {
          asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
        } else {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
        }
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");  // (a thread puts down what it asked for)
    if (in_place) cluster.sync();                      // every row of this pass has been read
    for (int r = row_of; r < rows && live; r += rows_at_once) {
      const uint8_t* src = rows_smem + (mine - smem_u32(rows_smem)) + (size_t)r * row_pad;
      uint8_t* at = to + (size_t)(r0 + r) * to_step;
      if (is_pair) {
        *reinterpret_cast<uint32_t*>(at) = *reinterpret_cast<const uint32_t*>(src);
      } else {
        *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(src);
      }
    }
  }
}

}  // namespace

cudaError_t launch_kv4_append(const Kv4Append& p, cudaStream_t s) {
  const uint32_t per_token = (uint32_t)p.cache.nkv * (p.cache.h / 16), items = (uint32_t)p.t * per_token;
  const int elem = p.f32 ? 4 : 2, per = 16 / elem;  // elements of a 16-byte load
  const bool vec = ((reinterpret_cast<uintptr_t>(p.k) | reinterpret_cast<uintptr_t>(p.v)) & 15) == 0 &&
                   p.k_batch % per == 0 && p.k_token % per == 0 && p.v_batch % per == 0 && p.v_token % per == 0;
  const unsigned blocks = (items + kRowThreads - 1) / kRowThreads, enough = (unsigned)(6 * device_sm_count() + 2 * p.cache.b - 1) / (2 * p.cache.b);
  const dim3 grid(blocks < enough ? blocks : enough, p.cache.b, 2);  // three blocks per SM
  const int lanes_log2 = p.cache.block == 64 ? 2 : 1;
  return p.f32 ? launch_chained(kv4_append_kernel<true>, grid, dim3(kRowThreads), 0, s, p, items, divisor(per_token), lanes_log2, vec ? 1 : 0)
               : launch_chained(kv4_append_kernel<false>, grid, dim3(kRowThreads), 0, s, p, items, divisor(per_token), lanes_log2, vec ? 1 : 0);
}

cudaError_t launch_kv4_read(const Kv4Read& p, cudaStream_t s) {
  const uint32_t per_token = (uint32_t)p.cache.nkv * (p.cache.h / 8), items = (uint32_t)p.t * per_token;
  const dim3 grid((items + 2 * kRowThreads - 1) / (2 * kRowThreads), p.cache.b, 2);
  const int words_log2 = p.cache.block == 64 ? 3 : 2;
  return p.f32 ? launch_chained(kv4_read_kernel<true>, grid, dim3(kRowThreads), 0, s, p, items, divisor(per_token), words_log2)
               : launch_chained(kv4_read_kernel<false>, grid, dim3(kRowThreads), 0, s, p, items, divisor(per_token), words_log2);
}

// Clusters of `ctas` CTAs with an SM each that fit on the current device at once.
static int evict_clusters_alone(int ctas) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)ctas);
  cfg.blockDim = dim3(kEvictThreads);
  cfg.dynamicSmemBytes = kEvictMostSmem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  int n = 0;
  return cudaOccupancyMaxActiveClusters(&n, kv4_evict_kernel, &cfg) == cudaSuccess ? n : 0;
}

cudaError_t launch_kv4_evict(const Kv4Evict& p, cudaStream_t s) {
  const int pairs = p.from.b * p.from.nkv;
  if (pairs == 0) return cudaSuccess;
  static bool done[64] = {false};
  static int alone[64][9];
  int dev = 0;
  cudaGetDevice(&dev);
  if (dev < 0 || dev >= 64) dev = 0;
  if (!done[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(kv4_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kEvictMostSmem);
    if (e != cudaSuccess) return e;
    for (int c = 1; c <= 8; ++c) alone[dev][c] = evict_clusters_alone(c);
    done[dev] = true;
  }
  const int parts = 2 * (p.from.h / 32) + 2 * (p.from.h / p.from.block);
  int row_log2 = 0;
  while ((1 << row_log2) < parts) ++row_log2;
  // The largest clusters that find an SM for each CTA: two CTAs on one SM share its way to memory while others idle, and a
  // second turn of clusters waits for the first (16 x 4352 to 4096 in place on clusters of 8, for which 15 find room: 33 us).
  int ctas = 8;
  while (ctas > 1 && pairs > alone[dev][ctas]) --ctas;
  const int smem = pairs <= alone[dev][ctas] ? kEvictMostSmem : kEvictSmem;
  return launch_chained_cluster(kv4_evict_kernel, dim3((unsigned)(pairs * ctas)), dim3(kEvictThreads), (size_t)smem, ctas, s, p,
                                p.from.k == p.to.k ? 1 : 0, row_log2, smem);
}

}  // namespace b200
