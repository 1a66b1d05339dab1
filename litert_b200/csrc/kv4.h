// The key/value cache held in 4 bits: what its kernels share.
//
// Keys and values each are nibbles [b, s, nkv, h / 2] (channel 2 i in the low half of byte i, so that a 32-bit word holds
// channels 8 j .. 8 j + 7 from its lowest nibble up) and fp16 pairs (scale, least) [b, s, nkv, h / block, 2]: nibble u of
// a block of channels stands for scale * u + least.
#pragma once

#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace b200 {

struct Kv4Cache {
  uint8_t* k;
  uint8_t* v;
  __half2* k_pairs;
  __half2* v_pairs;
  int b, s, nkv, h, block;
};

struct Kv4Append {
  Kv4Cache cache;
  const void* k;  // [b, t, nkv, h] f16 or f32; heads and channels contiguous
  const void* v;
  long long k_batch, k_token, v_batch, v_token;  // strides in elements
  const int32_t* positions;                      // [b]
  const int32_t* counts;                         // [b] or null (= t)
  int t, f32;
};
cudaError_t launch_kv4_append(const Kv4Append& p, cudaStream_t s);

struct Kv4Read {
  Kv4Cache cache;
  void* k;  // [b, t, nkv, h] f16 or f32
  void* v;
  const int32_t* positions;  // [b] or null (= 0)
  const int32_t* counts;     // [b] or null (= t)
  int t, f32;
};
cudaError_t launch_kv4_read(const Kv4Read& p, cudaStream_t s);

struct Kv4Evict {
  Kv4Cache from, to;           // the same cache, or two that do not overlap
  const float* scores;         // [b, nkv, from.s]
  const int32_t* lengths;      // [b]
  int budget, sinks, recent;   // sinks + recent <= budget <= to.s
  int32_t* kept;               // [b, nkv, budget]
  float* scores_out;           // [b, nkv, to.s]
  int32_t* lengths_out;        // [b]
};
cudaError_t launch_kv4_evict(const Kv4Evict& p, cudaStream_t s);

struct Kv4Sdpa {
  Kv4Cache cache;
  const void* q;           // [b, t, n, h] f16 or f32
  void* out;               // like q
  const int32_t* lengths;  // [b] or null (= cache.s)
  const float* mask;       // [b, 1, t, cache.s] additive or null
  float* scores;           // [b, nkv, cache.s] or null: += the weights of the KV head's queries
  int t, n, f32;
  float scale, logit_cap;
  float* ws;
};
size_t kv4_sdpa_workspace_bytes(int b, int t, int n, int nkv, int h, int s, int scores);
cudaError_t launch_kv4_sdpa(const Kv4Sdpa& p, cudaStream_t s);

// Attended slots of query i of t: all that are cached but the last t - 1 - i.
__host__ __device__ inline int kv4_limit(int length, int s, int t, int i) {
  length = length < 0 ? 0 : (length > s ? s : length);
  const int limit = length - (t - 1 - i);
  return limit < 0 ? 0 : limit;
}

}  // namespace b200
