// C-ABI entry points of the cache held in 4 bits (include/litert_b200.h, "key/value cache in 4 bits"): argument checks
// and launches.
#include <cmath>
#include <cstdarg>
#include <cstdio>

#include "../../include/litert_b200.h"
#include "kernels.h"
#include "kv4.h"

namespace {

thread_local char g_error[512] = "";

int fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_error, sizeof(g_error), fmt, ap);
  va_end(ap);
  return code;
}
int done(cudaError_t e, const char* what) {
  return e == cudaSuccess ? B200_OK : fail(B200_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

bool aligned(const void* p, uintptr_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// The cache's shape and tensors. Row indexes of the kernels' grids are 32 bits, offsets 64; slots are counted in 32 bits, up to
// a cluster's threads past the last.
int check_cache(const char* name, const void* k, const void* v, const void* kp, const void* vp, int b, int s, int nkv, int h, int block) {
  if (b != 0 && (!k || !v || !kp || !vp)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: a cache tensor is null", name);
  if (b < 0 || s <= 0 || nkv <= 0 || h <= 0)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: bad cache shape b=%d s=%d nkv=%d h=%d", name, b, s, nkv, h);
  if ((block != 32 && block != 64) || h % block != 0 || h > 512)
    return fail(B200_ERR_UNSUPPORTED, "%s: blocks of 32 or 64 channels that divide a head size up to 512 (block %d, head size %d)", name, block, h);
  if (s > 1 << 30) return fail(B200_ERR_UNSUPPORTED, "%s: at most 2^30 slots, got %d", name, s);
  if (b > 65535 || nkv > 65535) return fail(B200_ERR_UNSUPPORTED, "%s: at most 65535 sequences and KV heads", name);
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(kp, 4) || !aligned(vp, 4))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: nibbles lie on 16-byte boundaries, pairs on 4-byte boundaries", name);
  return B200_OK;
}

b200::Kv4Cache cache_of(void* k, void* v, void* kp, void* vp, int b, int s, int nkv, int h, int block) {
  return {static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), static_cast<__half2*>(kp), static_cast<__half2*>(vp), b, s, nkv, h, block};
}

bool float_type(int dtype) { return dtype == B200_DTYPE_F16 || dtype == B200_DTYPE_F32; }

// Whether [p, p + bytes) and [q, q + more) share a byte.
bool overlap(const void* p, size_t bytes, const void* q, size_t more) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), c = reinterpret_cast<uintptr_t>(q);
  return a < c + more && c < a + bytes;
}

}  // namespace

extern "C" {

const char* b200_kv4_last_error(void) { return g_error; }

int b200_kv4_append(const void* d_k, const void* d_v, int dtype, long long k_batch_stride, long long k_token_stride,
                    long long v_batch_stride, long long v_token_stride, const int32_t* d_positions, const int32_t* d_counts,
                    int b, int t, int nkv, int h, int block, int s_max, void* d_k_cache, void* d_v_cache, void* d_k_scale,
                    void* d_v_scale, void* stream) {
  const char* name = "b200_kv4_append";
  if (int rc = check_cache(name, d_k_cache, d_v_cache, d_k_scale, d_v_scale, b, s_max, nkv, h, block)) return rc;
  if (t < 0) return fail(B200_ERR_INVALID_ARGUMENT, "%s: %d tokens", name, t);
  if (!float_type(dtype)) return fail(B200_ERR_UNSUPPORTED, "%s: keys and values are f16 or f32 (dtype %d)", name, dtype);
  if (b == 0 || t == 0) return B200_OK;
  if (!d_k || !d_v || !d_positions) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(d_k, dtype == B200_DTYPE_F32 ? 4 : 2) || !aligned(d_v, dtype == B200_DTYPE_F32 ? 4 : 2))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: keys and values lie on boundaries of their elements", name);
  if ((long long)t * nkv * (h / 8) > INT32_MAX - 1024)
    return fail(B200_ERR_UNSUPPORTED, "%s: too many tokens of a sequence for one call", name);
  b200::Kv4Append p;
  p.cache = cache_of(d_k_cache, d_v_cache, d_k_scale, d_v_scale, b, s_max, nkv, h, block);
  p.k = d_k, p.v = d_v;
  p.k_batch = k_batch_stride, p.k_token = k_token_stride, p.v_batch = v_batch_stride, p.v_token = v_token_stride;
  p.positions = d_positions, p.counts = d_counts;
  p.t = t, p.f32 = dtype == B200_DTYPE_F32;
  return done(b200::launch_kv4_append(p, static_cast<cudaStream_t>(stream)), name);
}

int b200_kv4_read(const void* d_k_cache, const void* d_v_cache, const void* d_k_scale, const void* d_v_scale, int b, int s_max,
                  int nkv, int h, int block, const int32_t* d_positions, const int32_t* d_counts, int t, int dtype, void* d_k,
                  void* d_v, void* stream) {
  const char* name = "b200_kv4_read";
  if (int rc = check_cache(name, d_k_cache, d_v_cache, d_k_scale, d_v_scale, b, s_max, nkv, h, block)) return rc;
  if (t < 0) return fail(B200_ERR_INVALID_ARGUMENT, "%s: %d tokens", name, t);
  if (!float_type(dtype)) return fail(B200_ERR_UNSUPPORTED, "%s: rows are read as f16 or f32 (dtype %d)", name, dtype);
  if (b == 0 || t == 0) return B200_OK;
  if (!d_k || !d_v) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(d_k, 16) || !aligned(d_v, 16)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: outputs lie on 16-byte boundaries", name);
  if ((long long)t * nkv * (h / 8) > INT32_MAX - 1024)
    return fail(B200_ERR_UNSUPPORTED, "%s: too many tokens of a sequence for one call", name);
  b200::Kv4Read p;
  p.cache = cache_of(const_cast<void*>(d_k_cache), const_cast<void*>(d_v_cache), const_cast<void*>(d_k_scale),
                     const_cast<void*>(d_v_scale), b, s_max, nkv, h, block);
  p.k = d_k, p.v = d_v;
  p.positions = d_positions, p.counts = d_counts;
  p.t = t, p.f32 = dtype == B200_DTYPE_F32;
  return done(b200::launch_kv4_read(p, static_cast<cudaStream_t>(stream)), name);
}

int b200_kv4_evict(void* d_k_cache, void* d_v_cache, void* d_k_scale, void* d_v_scale, int b, int s_max, int nkv, int h, int block,
                   const float* d_scores, const int32_t* d_lengths, int budget, int sinks, int recent, void* d_k_to, void* d_v_to,
                   void* d_k_scale_to, void* d_v_scale_to, int s_to, int32_t* d_kept, float* d_scores_out, int32_t* d_lengths_out,
                   void* stream) {
  const char* name = "b200_kv4_evict";
  if (int rc = check_cache(name, d_k_cache, d_v_cache, d_k_scale, d_v_scale, b, s_max, nkv, h, block)) return rc;
  if (int rc = check_cache(name, d_k_to, d_v_to, d_k_scale_to, d_v_scale_to, b, s_to, nkv, h, block)) return rc;
  if (sinks < 0 || recent < 0 || budget <= 0 || sinks > budget - recent || budget > s_to)
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: budget %d has to hold sinks %d and recent %d and fit into %d slots", name, budget, sinks, recent, s_to);
  if (b == 0) return B200_OK;
  if (!d_scores || !d_lengths || !d_kept || !d_scores_out || !d_lengths_out) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if ((long long)b * nkv > (1 << 26)) return fail(B200_ERR_UNSUPPORTED, "%s: more than 2^26 sequences x KV heads", name);
  const size_t rows = (size_t)b * s_max * nkv, rows_to = (size_t)b * s_to * nkv;
  const void* from[4] = {d_k_cache, d_v_cache, d_k_scale, d_v_scale};
  const void* to[4] = {d_k_to, d_v_to, d_k_scale_to, d_v_scale_to};
  const size_t bytes[4] = {(size_t)h / 2, (size_t)h / 2, 4 * (size_t)(h / block), 4 * (size_t)(h / block)};
  const bool in_place = from[0] == to[0];
  for (int i = 0; i < 4; ++i) {
    if (in_place && (from[i] != to[i] || s_to != s_max))
      return fail(B200_ERR_INVALID_ARGUMENT, "%s: in place means the same four tensors of the same length", name);
    for (int j = 0; j < 4; ++j)
      if (!(in_place && i == j) && overlap(from[i], rows * bytes[i], to[j], rows_to * bytes[j]))
        return fail(B200_ERR_INVALID_ARGUMENT, "%s: the two caches overlap", name);
  }
  if (overlap(d_scores, sizeof(float) * (size_t)b * nkv * s_max, d_scores_out, sizeof(float) * (size_t)b * nkv * s_to) ||
      overlap(d_lengths, sizeof(int32_t) * (size_t)b, d_lengths_out, sizeof(int32_t) * (size_t)b))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: the new scores and lengths have tensors of their own", name);
  b200::Kv4Evict p;
  p.from = cache_of(d_k_cache, d_v_cache, d_k_scale, d_v_scale, b, s_max, nkv, h, block);
  p.to = cache_of(d_k_to, d_v_to, d_k_scale_to, d_v_scale_to, b, s_to, nkv, h, block);
  p.scores = d_scores, p.lengths = d_lengths;
  p.budget = budget, p.sinks = sinks, p.recent = recent;
  p.kept = d_kept, p.scores_out = d_scores_out, p.lengths_out = d_lengths_out;
  return done(b200::launch_kv4_evict(p, static_cast<cudaStream_t>(stream)), name);
}

size_t b200_kv4_sdpa_workspace_bytes(int b, int t, int n, int nkv, int h, int block, int s_max, int with_scores) {
  if (b <= 0 || t <= 0 || n <= 0 || nkv <= 0 || h <= 0 || s_max <= 0 || block <= 0) return 0;
  return b200::kv4_sdpa_workspace_bytes(b, t, n, nkv, h, s_max, with_scores);
}

int b200_kv4_sdpa(const void* d_q, const void* d_k_cache, const void* d_v_cache, const void* d_k_scale, const void* d_v_scale,
                  const int32_t* d_lengths, const float* d_mask, float* d_scores, void* d_out, int b, int t, int n, int nkv, int h,
                  int block, int s_max, int q_dtype, float scale, float logit_cap, void* d_workspace, size_t workspace_bytes,
                  void* stream) {
  const char* name = "b200_kv4_sdpa";
  if (int rc = check_cache(name, d_k_cache, d_v_cache, d_k_scale, d_v_scale, b, s_max, nkv, h, block)) return rc;
  if (t <= 0 || n <= 0 || n % nkv != 0 || t > 65535 || (long long)b * t * n > (1 << 26))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: bad shape b=%d t=%d n=%d nkv=%d", name, b, t, n, nkv);
  if (!float_type(q_dtype)) return fail(B200_ERR_UNSUPPORTED, "%s: queries are f16 or f32 (dtype %d)", name, q_dtype);
  if (!(logit_cap >= 0.0f) || !(scale >= 0.0f)) return fail(B200_ERR_INVALID_ARGUMENT, "%s: scale and logit cap are positive, or 0", name);
  if (b == 0) return B200_OK;
  if (!d_q || !d_out) return fail(B200_ERR_INVALID_ARGUMENT, "%s: null pointer", name);
  if (!aligned(d_q, 16) || !aligned(d_out, q_dtype == B200_DTYPE_F32 ? 4 : 2))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: queries lie on a 16-byte boundary, outputs on boundaries of their elements", name);
  const size_t need = b200::kv4_sdpa_workspace_bytes(b, t, n, nkv, h, s_max, d_scores != nullptr);
  if (!d_workspace || workspace_bytes < need || !aligned(d_workspace, 16))
    return fail(B200_ERR_INVALID_ARGUMENT, "%s: workspace of %zu bytes on a 16-byte boundary needed (b200_kv4_sdpa_workspace_bytes), got %zu", name,
                need, workspace_bytes);
  b200::Kv4Sdpa p;
  p.cache = cache_of(const_cast<void*>(d_k_cache), const_cast<void*>(d_v_cache), const_cast<void*>(d_k_scale),
                     const_cast<void*>(d_v_scale), b, s_max, nkv, h, block);
  p.q = d_q, p.out = d_out, p.lengths = d_lengths, p.mask = d_mask, p.scores = d_scores;
  p.t = t, p.n = n, p.f32 = q_dtype == B200_DTYPE_F32;
  p.scale = scale > 0.0f ? scale : 1.0f / sqrtf((float)h);
  p.logit_cap = logit_cap;
  p.ws = static_cast<float*>(d_workspace);
  return done(b200::launch_kv4_sdpa(p, static_cast<cudaStream_t>(stream)), name);
}

}  // extern "C"
