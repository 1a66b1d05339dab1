// Attention over a key/value cache held in 4 bits (layout in kv4.h).
//
// For query row r (query token i of t, head n) and the attended slots s of its KV head:
//   x_s = scale * q . k_s [cap * tanh(x / cap)] [+ mask],  out = sum_s softmax(x)_s v_s,  scores_s += softmax(x)_s
// With nibbles u and pairs (a, m) per block g of channels, the dequantized rows never exist:
//   q . k_s = sum_g a_sg (sum_c u_sc q_c) + m_sg (sum_c q_c)
//   out_c   = sum_s (p_s a_sg) u_sc + sum_s p_s m_sg
// Products of a nibble and an fp16 number are exact and are added in fp32.
#include <math_constants.h>

#include <cfloat>

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

// ---- head sizes 64, 128 and 256: tensor cores -------------------------------------------------------------
// Up to eight query rows of a KV head (query heads x query tokens) are the 8-wide side of mma.m16n8k16; a tile is 16 slots.
// Every (sequence, KV head, eight rows) pair is cut into pieces of a common greatest length, one per warp. A warp walks
// through its piece without meeting another one; at the end the warps of a CTA add their states of a common pair to one
// partial record (un-normalised outputs, maximum, sum), and a second kernel merges a pair's records. A pair of few tiles
// belongs to one CTA, which writes the outputs itself.
//
// What bounds a launch of a few microseconds is code that runs once: it is fetched, cold, at about eight cycles per
// instruction, so loops outside the main one are rolled. Measured with 16 ragged sequences of up to 8192 tokens, 8 heads x
// 256, replayed: the CTA that completes a pair (a counter) merges it 20.1 us, second kernel 16.1; pieces that run on from one
// pair to the next (all of one length) 17.5, 4 of them in the warps that had parts of two pairs; such pieces per CTA 19.4; a
// record for every warp 20.3 (9.8 MB to merge).
constexpr int kSlots = 16;
__host__ __device__ inline int tiles_of(int slots) { return (slots + kSlots - 1) / kSlots; }

__host__ __device__ constexpr int kv4_warps(int h) { return h == 256 ? 8 : 16; }

template <int H, int BLOCK, bool QF32>
struct Kv4Tile {
  static constexpr int kG = H / BLOCK;                 // blocks of a row
  static constexpr int kNibbleBytes = kSlots * H / 2;  // of the keys (or values) of a tile
  static constexpr int kPairBytes = kSlots * kG * 4;
  static constexpr int kBytes = 2 * (kNibbleBytes + kPairBytes);
  static constexpr int kQueryBytes = H / 32 * 512 * (QF32 ? 2 : 1);  // a warp's query fragments
  static constexpr int kWarps = kv4_warps(H);
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRec = H + 4;  // floats of a record per row: outputs, maximum, sum, padding
  static constexpr int kFit = (220 * 1024 / kWarps - kQueryBytes) / kBytes;
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kWarpBytes = kQueryBytes + kStages * kBytes;
  static constexpr int kSmem = kWarps * kWarpBytes + 128;
  static_assert(8 * kRec * 4 <= kWarpBytes, "a warp's state fits into its part");
  static_assert(kBytes % 128 == 0 && kStages >= 3 && kSmem <= 221 * 1024, "layout");
};

struct Kv4Rows {
  int group, rows, chunks;  // query heads per KV head; query rows per KV head; of eight rows each
};
__host__ __device__ inline Kv4Rows kv4_rows(int t, int n, int nkv) {
  const int group = n / nkv, rows = t * group;
  return {group, rows, (rows + 7) / 8};
}

// Workspace of the tensor-core kernels: a record per piece (of which the first of a pair in each CTA is used), then, where
// scores are wanted, the rows' {maximum, 1 / sum} [pair][8 rows] of pairs that have a CTA to themselves, and the logits [pair][slot (rounded up to a tile)][8 rows].
constexpr int kFewRecords = 16;
__host__ __device__ inline size_t kv4_records_floats(long long pieces, int h) { return (size_t)pieces * 8 * (h + 4); }

__device__ __forceinline__ int kv4_length(const Kv4Sdpa& p, int b) {
  return p.lengths ? max(0, min(p.lengths[b], p.cache.s)) : p.cache.s;
}

// a / b for a below 2^22, given 1 / b. (The divisions stand in chains of dependent instructions at the kernels' start.)
__device__ __forceinline__ int divide(int a, int b, float inverse) {
  int q = (int)((float)a * inverse);
  const int r = a - q * b;
  q += (r >= b ? 1 : 0) - (r < 0 ? 1 : 0);
  return q;
}

__device__ __forceinline__ float reciprocal(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// How the pairs are cut: into pieces of up to about `size` tiles, each pair's of equal lengths (to a tile), the smallest size
// that needs no more pieces than there are warps. Every CTA gets an equal number of the pieces (to one).
// Few tiles are not scattered over more CTAs than they are worth: where every pair has at most four tiles per warp of a CTA, it
// gets a CTA to itself; up to four tiles per warp of sixteen CTAs, it gets about these.
struct Kv4Cut {
  bool own_cta;            // a pair is a CTA's, in pieces of equal lengths
  int size, each, longer;  // otherwise: the first `longer` CTAs have one piece more than `each`
  float inverse;           // 1 / size
  int len;                 // attended slots of sequence `lane`
  __device__ __forceinline__ int pieces_of(int slots) const {
    const int tiles = tiles_of(slots);
    return tiles == 0 ? 0 : max(1, min(tiles, (int)((float)(tiles + size - 1) * inverse)));
  }
  __device__ __forceinline__ int begin(int cta) const { return cta * each + min(cta, longer); }
  __device__ __forceinline__ int owner(int piece) const {
    const int front = longer * (each + 1);
    return piece < front ? divide(piece, each + 1, reciprocal((float)(each + 1))) : longer + divide(piece - front, each, reciprocal((float)each));
  }
};
__device__ __forceinline__ Kv4Cut kv4_cut(const Kv4Sdpa& p, int per, int ctas, int warps, int lane) {
  const int pairs = p.cache.b * per;
  Kv4Cut c;
  c.len = lane < p.cache.b ? kv4_length(p, lane) : 0;
  int total = tiles_of(c.len) * per, most = tiles_of(c.len);
#pragma unroll 1
  for (int i = lane + 32; i < p.cache.b; i += 32) {
    const int tiles = tiles_of(kv4_length(p, i));
    total += tiles * per;
    most = max(most, tiles);
  }
  total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
  most = (int)__reduce_max_sync(0xffffffffu, (unsigned)most);
  c.own_cta = pairs <= ctas && most <= 4 * warps;
  c.size = c.each = c.longer = 1;
  c.inverse = 1.0f;
  if (c.own_cta) return c;
  if (total <= 4 * kFewRecords * pairs * warps) ctas = min(ctas, kFewRecords * pairs);
  const int room = ctas * warps;
  c.size = max(1, (int)ceilf((float)total * reciprocal((float)room)));
  int n;
#pragma unroll 1
  while (true) {  // (ends: there is room for twice the pairs, and a large enough size makes a piece of each)
    c.inverse = reciprocal((float)c.size);
    n = c.pieces_of(c.len) * per;
#pragma unroll 1
    for (int i = lane + 32; i < p.cache.b; i += 32) n += c.pieces_of(kv4_length(p, i)) * per;
    n = (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
    if (n <= room) break;
    c.size += 1 + c.size / 16;
  }
  c.each = divide(n, ctas, reciprocal((float)ctas));
  c.longer = n - c.each * ctas;
  return c;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4_or_zero(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void sts128(uint32_t a, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
__device__ __forceinline__ void lds128(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
// Four 8 x 8 matrices of 16-bit elements, lane l naming row l % 8 of matrix l / 8: thread (g, t) receives elements 2 t and
// 2 t + 1 of row g; transposed, elements g of rows 2 t and 2 t + 1.
__device__ __forceinline__ void load_matrices(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(a));
}
__device__ __forceinline__ void load_matrices_transposed(uint32_t a, uint32_t (&v)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
               : "r"(a));
}
// D(16 x 8) += A(16 x 16) B(16 x 8). (Not volatile: products of different chains may be interleaved.)
__device__ __forceinline__ void product(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void first_product(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
// Two floats as one operand.
__device__ __forceinline__ uint64_t packed(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpacked(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// p + j * step in one instruction.
__device__ __forceinline__ const void* advance(const void* p, int j, uint32_t step) {
  uint64_t r;
  asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(j), "r"(step), "l"(p));
  return reinterpret_cast<const void*>(r);
}
// 2^x; results below 2^-126 are zero.
__device__ __forceinline__ float power2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t transposed8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ float2 pair_floats(uint32_t bits) { return __half22float2(*reinterpret_cast<const __half2*>(&bits)); }
__device__ __forceinline__ uint32_t halves(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// a and b as fp16, and what that leaves as fp16: 22 bits of each.
__device__ __forceinline__ void split_halves(float a, float b, uint32_t& high, uint32_t& low) {
  high = halves(a, b);
  const float2 r = pair_floats(high);
  low = halves(a - r.x, b - r.y);
}

// Where in a tile's nibbles the 16-byte piece c (32 channels) of a row lies. Rows follow one another; within each 128 bytes
// the pieces are exchanged by an XOR such that piece c of rows 8 i .. 8 i + 7 touches 32 banks. Rows r and r + 8 are
// exchanged alike, and c only enters through an XOR of bits 4 to 6.
template <int H>
__device__ __forceinline__ uint32_t piece_at(int row, int c) {
  constexpr int kRows = 256 / H;  // per 128 bytes
  const int line = row / kRows, pos = (row % kRows) * (H / 32) + c;
  const int x = H == 256 ? row & 7 : H == 128 ? ((line & 1) << 1) | ((line >> 1) & 1) : line & 1;
  return (uint32_t)(line * 128 + ((pos ^ x) << 4));
}

// For fp16 queries key nibbles become operands by a mask alone: in the low bits of a half, nibble u is the subnormal number u 2^-24,
// one place up u 2^-20. So a word of eight nibbles is four pairs after one shift and four masks, exactly; the factor 16
// between the two kinds goes into the queries of those channels, 2^-24 into the logits' factor. For float32 queries they are
// centred like the values' (8 x scale joins the least value's factor), and the queries' low halves come first, while the sums
// are small: the products truncate (weights' error against 64 bits, 2000 tokens of 128: 1.05e-6 -> 3.7e-7, where torch's float32
// has 1.2e-6; + 0.3 us at 4 x 2000).
// Value nibbles are centred, u - 8, by way of the exponents that make a nibble's place the unit (1024) or an eighth of it
// (64): sums of weights times values that are all positive lose to the tensor core's truncation (float32 outputs were
// 3e-5 off; 8 x scale joins the least value instead).
// A weight times a value scale is two fp16 numbers, 22 bits, for either type of query. As one number it is off by 2^-12 on
// average, times |u - 8| x scale: outputs 2.8e-4 off 64 bits where an fp16 output's own rounding is 2.1e-4.
// A tile's sums begin at zero, the second numbers' products first, and are added in fp32 with rounding. In the tensor core's
// accumulators every product would cut off the sum of all tiles before it: 1.5e-6 off after a tile, 1.4e-5 after 65, 2e-5 after 256
// (float32 queries, normal values; now 0.6e-6 and 1.2 .. 1.5e-6, plain float32 0.4e-6), ten times that in one direction where
// nibbles are only positive. (64 x 32768 of 8 heads x 256, replayed: one number each 71.5 us, with a second one and the unit below
// 83.5, with the sums 86.4; 16 x 8192 15.4, 16.4, 15.8. Half of the slots as complements, 15 - u, to save the centring: 75.9 and
// 85.5 us, but sums about zero only if both halves have weight: 3e-4 off behind a mask that hides one. Uncentred, with - 8 w as
// the sums' beginning: 91.6.)
// What a second number leaves is 2^-25 at least, fp16's last place, however small the product. So a row's weights are counted in
// units of 2^-units such that the largest product of a weight and a scale so far lies in 2^9 .. 2^10, up to 60000 before that is
// put right: rescaling the outputs at every new maximum would happen in most tiles while a warp has seen few. The unit goes by
// what slots contribute, not by their scales alone, so hidden slots, and slots or tiles that end up without weight, do not coarsen
// the others. A scale of zero counts as kLeastScale, which keeps the weights themselves within fp32.
// A unit of the largest scale took 1.4 us less at 64 x 32768, 0.2 at 16 x 8192.
constexpr float kMostOperand = 60000.0f, kLeastScale = 0x1p-40f, kMostUnits = 49.0f;
constexpr int kUnitBits = 9;
constexpr uint32_t kLowNibbles = 0x000f000fu, kHighNibbles = 0x00f000f0u;
__device__ __forceinline__ uint32_t half2_sub(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// (w & mask) | exponent in one instruction: the exponents stay in registers.
struct Centred {
  uint32_t unit, eighth;
  __device__ __forceinline__ Centred() {
    asm volatile("mov.b32 %0, 0x64006400;" : "=r"(unit));
    asm volatile("mov.b32 %0, 0x54005400;" : "=r"(eighth));
  }
  __device__ __forceinline__ static uint32_t splice(uint32_t w, uint32_t mask, uint32_t exponent) {
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(r) : "r"(w), "r"(mask), "r"(exponent));
    return r;
  }
  __device__ __forceinline__ uint32_t low(uint32_t w) const { return half2_sub(splice(w, kLowNibbles, unit), 0x64086408u); }      // - 1032
  __device__ __forceinline__ uint32_t high(uint32_t w) const { return half2_sub(splice(w, kHighNibbles, eighth), 0x54805480u); }  // - 72
};

// Four channels of a query row's result, from its sums; with the first ones, what the scores need of the row.
template <int H, bool QF32>
__device__ __forceinline__ void kv4_output(const Kv4Sdpa& p, float2* stats_ws, int b, int i, int head, int pair, int row, int d, float top, float sum,
                                           const float4& acc) {
  const float inverse = sum != 0.0f ? 1.0f / sum : 0.0f;  // (0: no slot, and zeros)
  const size_t at = (((size_t)b * p.t + i) * p.n + head) * H + d;
  if constexpr (QF32) {
    float* o = static_cast<float*>(p.out) + at;
    o[0] = acc.x * inverse, o[1] = acc.y * inverse, o[2] = acc.z * inverse, o[3] = acc.w * inverse;
  } else {
    __half* o = static_cast<__half*>(p.out) + at;
    o[0] = __float2half_rn(acc.x * inverse), o[1] = __float2half_rn(acc.y * inverse);
    o[2] = __float2half_rn(acc.z * inverse), o[3] = __float2half_rn(acc.w * inverse);
  }
  if (stats_ws && d == 0) stats_ws[(size_t)pair * 8 + row] = make_float2(top == -CUDART_INF_F ? 0.0f : top, inverse);
}

template <int H, int BLOCK, bool QF32>
__global__ void __launch_bounds__(Kv4Tile<H, BLOCK, QF32>::kThreads, 1) kv4_sdpa_kernel(const Kv4Sdpa p, float2* stats_ws, float* logits_ws) {
  using T = Kv4Tile<H, BLOCK, QF32>;
  constexpr int G = T::kG;
  constexpr int P = H / 32;         // 16-byte pieces of a row
  constexpr int kPer = BLOCK / 32;  // of them in a block
  constexpr int kWarps = T::kWarps;
  extern __shared__ uint8_t kv4_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv4_smem_raw) + 127) & ~uintptr_t(127));
  __shared__ int s_pair[kWarps];                       // whose the warps' states are
  __shared__ float s_m[kWarps][8], s_l[kWarps][8];     // their maxima and sums
  __shared__ float s_f[kWarps][8];                     // and factors in the sum
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int nkv = p.cache.nkv, s_max = p.cache.s;
  const Kv4Rows rw = kv4_rows(p.t, p.n, nkv);
  const int per = nkv * rw.chunks;  // pairs per sequence
  // this warp's part of the shared memory; where a lane's copies come from and go to (16-byte piece `lane % P` of rows
  // lane / P + 32 / P j)
  const uint32_t part_at = smem_u32(smem) + (uint32_t)(w * T::kWarpBytes), ring = part_at + T::kQueryBytes;
  const uint32_t row_pitch = (uint32_t)nkv * (H / 2), pair_pitch = (uint32_t)nkv * G * 4;  // bytes
  const int copy_row = lane / P, copy_piece = lane % P;
  const uint32_t copy_from = (uint32_t)copy_row * row_pitch + copy_piece * 16, pair_from = (uint32_t)(lane / G) * pair_pitch + lane % G * 4;
  const uint32_t row_step = row_pitch * (32 / P), pair_step = pair_pitch * (32 / G);
  constexpr int kCopies = kSlots * P / 32, kPairCopies = (kSlots * G + 31) / 32;
  // the row that this lane names for a load of matrices: of two pieces, rows 0 .. 15
  const uint32_t matrix_at = piece_at<H>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
  const float inverse_chunks = reciprocal((float)rw.chunks), inverse_group = reciprocal((float)rw.group), inverse_per = reciprocal((float)per);
  pdl_wait();
  // (only now: what a dependent kernel does ahead of its own wait may then read this kernel's inputs)
  pdl_launch_dependents();
  // this warp's piece: seg tiles from `unit` on of pair in_b of sequence b
  const Kv4Cut cut = kv4_cut(p, per, gridDim.x, kWarps, lane);
  int seg = 0, b = 0, in_b = 0, unit = 0, len = cut.len;
  int pair = -1;
  if (cut.own_cta) {
    if ((int)blockIdx.x < p.cache.b * per) {
      b = divide(blockIdx.x, per, inverse_per);
      in_b = blockIdx.x - b * per;
      len = p.cache.b <= 32 ? __shfl_sync(0xffffffffu, len, b) : kv4_length(p, b);
      const int tiles = tiles_of(len), each = tiles / kWarps, longer = tiles - each * kWarps;
      unit = w * each + min(w, longer);
      seg = each + (w < longer ? 1 : 0);
      if (w == 0 || seg > 0) pair = blockIdx.x;  // (a pair without a slot has zeros to write)
    }
  } else if (w < cut.each + ((int)blockIdx.x < cut.longer ? 1 : 0)) {
    const int piece = cut.begin(blockIdx.x) + w;
#pragma unroll 1
    for (int b0 = 0, base = 0; b0 < p.cache.b; b0 += 32) {
      if (b0 > 0) len = b0 + lane < p.cache.b ? kv4_length(p, b0 + lane) : 0;
      int n = cut.pieces_of(len), upto = n * per;  // inclusive prefix sum over the lanes
#pragma unroll 1
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint32_t here = __ballot_sync(0xffffffffu, base + upto > piece);
      if (here) {
        const int src = __ffs(here) - 1;
        const int rest = piece - __shfl_sync(0xffffffffu, base + upto - n * per, src);
        len = __shfl_sync(0xffffffffu, len, src);
        n = __shfl_sync(0xffffffffu, n, src);
        b = b0 + src;
        const float inverse = reciprocal((float)n);
        in_b = divide(rest, n, inverse);
        const int part = rest - in_b * n, tiles = tiles_of(len), each = divide(tiles, n, inverse), longer = tiles - each * n;
        unit = part * each + min(part, longer);
        seg = each + (part < longer ? 1 : 0);
        pair = b * per + in_b;
        break;
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
  }

  if (seg > 0) {
    const int kvh = divide(in_b, rw.chunks, inverse_chunks), chunk = in_b - kvh * rw.chunks;
    // the queries are asked for first, the tiles arrive meanwhile
    uint4 q_bits[QF32 ? 2 * P : P];
    {
      const int q_row = min(chunk * 8 + g, rw.rows - 1);  // (columns without a row repeat the last one and are dropped)
      const int i = divide(q_row, rw.group, inverse_group);
      const size_t at = (((size_t)b * p.t + i) * p.n + kvh * rw.group + (q_row - i * rw.group)) * H + 8 * t;
#pragma unroll
      for (int sl = 0; sl < P; ++sl) {
        if constexpr (QF32) {
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(p.q) + at + 32 * sl);
          q_bits[2 * sl] = __ldg(src);
          q_bits[2 * sl + 1] = __ldg(src + 1);
        } else {
          q_bits[sl] = __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(p.q) + at + 32 * sl));
        }
      }
    }
    // Requests this warp's next tile: rows behind the length arrive as zeros.
    const size_t row0 = ((size_t)b * s_max + (size_t)unit * kSlots) * nkv + kvh;
    const uint8_t* k_next = p.cache.k + row0 * (H / 2);
    const uint8_t* v_next = p.cache.v + row0 * (H / 2);
    const __half2* kp_next = p.cache.k_pairs + row0 * G;
    const __half2* vp_next = p.cache.v_pairs + row0 * G;
    int asked = 0;
    uint32_t to = ring;
    auto request = [&]() {
      if (asked < seg) {
        const int there = len - (unit + asked) * kSlots;
        if (there >= kSlots) {
          const void* ks = k_next + copy_from;
          const void* vs = v_next + copy_from;
          const void* kps = reinterpret_cast<const uint8_t*>(kp_next) + pair_from;
          const void* vps = reinterpret_cast<const uint8_t*>(vp_next) + pair_from;
#pragma unroll
          for (int j = 0; j < kCopies; ++j) {
            cp_async16(to + piece_at<H>(copy_row + j * (32 / P), copy_piece), advance(ks, j, row_step));
            cp_async16(to + T::kNibbleBytes + piece_at<H>(copy_row + j * (32 / P), copy_piece), advance(vs, j, row_step));
          }
#pragma unroll
          for (int j = 0; j < kPairCopies; ++j) {
            if (lane + 32 * j < kSlots * G) {
              cp_async4(to + 2 * T::kNibbleBytes + (lane + 32 * j) * 4, advance(kps, j, pair_step));
              cp_async4(to + 2 * T::kNibbleBytes + T::kPairBytes + (lane + 32 * j) * 4, advance(vps, j, pair_step));
            }
          }
        } else {  // (one tile of a pair at most)
#pragma unroll 1
          for (int j = 0; j < kCopies; ++j) {
            const int row = copy_row + j * (32 / P);
            const bool ok = row < there;
            const uint32_t from = ok ? copy_from + j * row_step : 0u;
            cp_async16_or_zero(to + piece_at<H>(row, copy_piece), k_next + from, ok);
            cp_async16_or_zero(to + T::kNibbleBytes + piece_at<H>(row, copy_piece), v_next + from, ok);
          }
#pragma unroll 1
          for (int e = lane; e < kSlots * G; e += 32) {
            const bool ok = e / G < there;
            const uint32_t from = ok ? (uint32_t)(e / G) * pair_pitch + e % G * 4 : 0u;
            cp_async4_or_zero(to + 2 * T::kNibbleBytes + e * 4, reinterpret_cast<const uint8_t*>(kp_next) + from, ok);
            cp_async4_or_zero(to + 2 * T::kNibbleBytes + T::kPairBytes + e * 4, reinterpret_cast<const uint8_t*>(vp_next) + from, ok);
          }
        }
        k_next += (size_t)kSlots * row_pitch;
        v_next += (size_t)kSlots * row_pitch;
        kp_next += (size_t)kSlots * nkv * G;
        vp_next += (size_t)kSlots * nkv * G;
        to = to + T::kBytes == ring + T::kStages * T::kBytes ? ring : to + T::kBytes;
        ++asked;
      }
      cp_async_commit();
    };
#pragma unroll 1
    for (int k = 0; k < T::kStages - 1; ++k) request();

    // Queries: thread (g, t) makes row g's elements at its words of a key, as the B operand: channels 0, 4 | 2, 6 of a word
    // meet low nibbles, 1, 5 | 3, 7 high ones. They are scaled by a power of two that brings the row's largest to 2^5 ..
    // 2^6: dividing by 16 (fp16 queries) then loses nothing above 2^-26 of it, and a float32 query is two fp16 numbers to 22 bits.
    // They are kept in shared memory, [piece][lane][4 words] (and again for the low halves).
    const uint32_t query_at = part_at + lane * 16;
    float q_sum[G][2], factor[2];  // of the rows 2 t and 2 t + 1 (the products' columns)
    {
      float top;
      if constexpr (QF32) {
        top = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * P; ++i)
          top = fmaxf(fmaxf(fmaxf(top, fabsf(__uint_as_float(q_bits[i].x))), fabsf(__uint_as_float(q_bits[i].y))),
                      fmaxf(fabsf(__uint_as_float(q_bits[i].z)), fabsf(__uint_as_float(q_bits[i].w))));
      } else {
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < P; ++i)
          most = __vmaxu2(__vmaxu2(__vmaxu2(most, q_bits[i].x & 0x7fff7fffu), q_bits[i].y & 0x7fff7fffu),
                          __vmaxu2(q_bits[i].z & 0x7fff7fffu, q_bits[i].w & 0x7fff7fffu));
        const float2 f = pair_floats(most);
        top = fmaxf(f.x, f.y);
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int field = __float_as_int(top) >> 23;
      const int up = field == 255 ? 0 : min(132 - field, QF32 ? 126 : 29);  // (an infinite query stays what it is)
      const float scale_up = __int_as_float((127 + up) << 23), scale_down = __int_as_float((127 - up) << 23);
      // 2^up as a product of two halves
      const __half2 one = __float2half2_rn(__int_as_float((127 + min(up, 15)) << 23)), two = __float2half2_rn(__int_as_float((127 + max(up - 15, 0)) << 23));
      const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int sl = gr * kPer; sl < (gr + 1) * kPer; ++sl) {
          uint32_t high[4], low[4];
          if constexpr (QF32) {
            const uint4 lo = q_bits[2 * sl], hi = q_bits[2 * sl + 1];
            split_halves(__uint_as_float(lo.x) * scale_up, __uint_as_float(hi.x) * scale_up, high[0], low[0]);
            split_halves(__uint_as_float(lo.z) * scale_up, __uint_as_float(hi.z) * scale_up, high[1], low[1]);
            split_halves(__uint_as_float(lo.y) * scale_up, __uint_as_float(hi.y) * scale_up, high[2], low[2]);
            split_halves(__uint_as_float(lo.w) * scale_up, __uint_as_float(hi.w) * scale_up, high[3], low[3]);
            sts128(query_at + (P + sl) * 512, low);
          } else {
            uint32_t v[4] = {q_bits[sl].x, q_bits[sl].y, q_bits[sl].z, q_bits[sl].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __half2 y = __hmul2(__hmul2(*reinterpret_cast<const __half2*>(&v[e]), one), two);
              v[e] = *reinterpret_cast<const uint32_t*>(&y);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              high[e] = __byte_perm(v[e], v[e + 2], 0x5410);
              const uint32_t odd = __byte_perm(v[e], v[e + 2], 0x7632);
              const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&odd), sixteenth);
              high[2 + e] = *reinterpret_cast<const uint32_t*>(&y);
            }
          }
          sts128(query_at + sl * 512, high);
          // the blocks' sums: products with ones (and sixteens)
#pragma unroll
          for (int odd = 0; odd < 2; ++odd) {
            const uint32_t ones = odd && !QF32 ? 0x4c004c00u : 0x3c003c00u;
            product(sum, ones, ones, ones, ones, high[2 * odd], high[2 * odd + 1]);
            if constexpr (QF32) product(sum, ones, ones, ones, ones, low[2 * odd], low[2 * odd + 1]);
          }
        }
        q_sum[gr][0] = QF32 ? sum[0] : sum[0] * 0x1p-24f;
        q_sum[gr][1] = QF32 ? sum[1] : sum[1] * 0x1p-24f;
      }
      const float f = scale_down * p.scale;
      // (in two steps: 2^24 times a small scale stays within fp32 either way)
      factor[0] = __shfl_sync(0xffffffffu, f, 8 * t) * (QF32 ? 1.0f : 0x1p24f);
      factor[1] = __shfl_sync(0xffffffffu, f, 8 * t + 4) * (QF32 ? 1.0f : 0x1p24f);
    }
    int limit[2];
    const float* mask[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int i = divide(min(chunk * 8 + 2 * t + e, rw.rows - 1), rw.group, inverse_group);
      limit[e] = kv4_limit(len, s_max, p.t, i);
      mask[e] = p.mask ? p.mask + ((size_t)b * p.t + i) * s_max : nullptr;
    }
    const int least_limit = kv4_limit(len, s_max, p.t, divide(chunk * 8, rw.group, inverse_group));  // of any row
    // masks are requested a tile ahead of their use
    float next_mask[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    auto ask_masks = [&](int first) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int slot = first + g + 8 * (e >> 1);
        if (slot < limit[e & 1]) next_mask[e] = __ldg(mask[e & 1] + slot);
      }
    };
    if (p.mask) ask_masks(unit * kSlots);
    const bool guard = p.mask != nullptr || p.t > 1;
    float* logits = logits_ws ? logits_ws + (size_t)pair * ((size_t)tiles_of(s_max) * kSlots * 8) : nullptr;

    // outputs: of piece i and its channels 4 g + {0, 1} and 4 g + {2, 3}, rows 2 t and 2 t + 1
    uint64_t o[P][2][2];  // pairs of rows
    float least_sum[G];
#pragma unroll
    for (int gr = 0; gr < G; ++gr) least_sum[gr] = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) o[i][0][e] = o[i][1][e] = packed(0.0f, 0.0f);
    // the rows' weights are e^(x - m_run) in units of 2^-units (integers; see kMostUnits). The first x that is a number makes a
    // weight of infinity, or, at the type's lowest value, of one: m_run need not be the largest x.
    float m_run[2] = {-FLT_MAX, -FLT_MAX}, l_run[2] = {0.0f, 0.0f}, units[2] = {kMostUnits, kMostUnits};

    const Centred centred;
    // The logits of a tile's slots g and g + 8, rows 2 t and 2 t + 1, without factor, cap and mask.
    auto dot = [&](uint32_t at, float (&x)[4]) {
      const uint32_t pairs_at = at + 2 * T::kNibbleBytes;
      // One product of each chain after the other: a warp waits for a chain's last product before its next.
      constexpr int kAtOnce = P, kChains = kAtOnce / kPer, kApart = kChains < 4 ? 2 : 1;
      x[0] = x[1] = x[2] = x[3] = 0.0f;
#pragma unroll
      for (int i0 = 0; i0 < P; i0 += kAtOnce) {
        uint32_t words[kAtOnce / 2][4];
#pragma unroll
        for (int i = 0; i < kAtOnce; i += 2) load_matrices(at + (matrix_at ^ (uint32_t)((i0 + i) * 16)), words[i / 2]);
        float acc[kChains][kApart][4];  // (few chains: low and high nibbles apart)
// (the low halves of float32 queries first, while the sums are small: the tensor core truncates)
#pragma unroll
        for (int half = QF32 ? 1 : 0; half >= 0; --half) {
#pragma unroll
          for (int j = 0; j < kPer; ++j) {
            uint32_t qs[kChains][4];
#pragma unroll
            for (int c = 0; c < kChains; ++c) lds128(query_at + (half * P + i0 + c * kPer + j) * 512, qs[c]);
#pragma unroll
            for (int odd = 0; odd < 2; ++odd) {
#pragma unroll
              for (int c = 0; c < kChains; ++c) {
                const int i = c * kPer + j;
                const uint32_t (&q)[4] = qs[c];
                const uint32_t wa = words[i / 2][2 * (i & 1)], wb = words[i / 2][2 * (i & 1) + 1];
                uint32_t k[4] = {wa, wb, wa >> 8, wb >> 8};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  if constexpr (QF32) {
                    k[e] = odd ? centred.high(k[e]) : centred.low(k[e]);
                  } else {
                    k[e] &= odd ? kHighNibbles : kLowNibbles;
                  }
                }
                float (&to_acc)[4] = acc[c][odd % kApart];
                if (j == 0 && odd < kApart && half == (QF32 ? 1 : 0)) {
                  first_product(to_acc, k[0], k[1], k[2], k[3], q[2 * odd], q[2 * odd + 1]);
                } else {
                  product(to_acc, k[0], k[1], k[2], k[3], q[2 * odd], q[2 * odd + 1]);
                }
              }
            }
          }
        }
#pragma unroll
        for (int c = 0; c < kChains; ++c) {
          const int gr = i0 / kPer + c;
          const float2 fa = pair_floats(lds32(pairs_at + (uint32_t)((g * G + gr) * 4)));
          const float2 fb = pair_floats(lds32(pairs_at + (uint32_t)(((g + 8) * G + gr) * 4)));
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 f = e < 2 ? fa : fb;
            x[e] = fmaf(f.x, kApart == 2 ? acc[c][0][e] + acc[c][kApart - 1][e] : acc[c][0][e],
                        fmaf(QF32 ? fmaf(8.0f, f.x, f.y) : f.y, q_sum[gr][e & 1], x[e]));
          }
        }
      }
    };
    auto finish = [&](int first, float (&x)[4]) {
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] *= factor[e & 1];
      if (p.logit_cap > 0.0f) {
#pragma unroll 1
        for (int k = 0; k < 4; ++k) {  // (the four values in turn: one copy of the function's code)
          const float y = p.logit_cap * tanhf(x[0] / p.logit_cap);
          x[0] = x[1], x[1] = x[2], x[2] = x[3], x[3] = y;
        }
      }
      if (p.mask) {
        float m[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) m[e] = next_mask[e];
        ask_masks(first + kSlots);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = m[e] == -CUDART_INF_F ? m[e] : x[e] + m[e];
      }
      if (first + kSlots > least_limit) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = first + g + 8 * (e >> 1) < limit[e & 1] ? x[e] : -CUDART_INF_F;
      }
      if (logits) {
        float* to_ws = logits + (size_t)(first + g) * 8 + 2 * t;
        *reinterpret_cast<float2*>(to_ws) = make_float2(x[0], x[1]);
        *reinterpret_cast<float2*>(to_ws + 64) = make_float2(x[2], x[3]);
      }

    };
    // A tile's largest value scales of this thread's slots g and g + 8, compared as halves by the threads that share them, and
    // whether any is infinite or NaN (or a least value is). Found a tile ahead of their use.
    float largest[2];
    bool infinite;
    auto find_largest = [&](uint32_t at) {
      uint32_t scales = 0, either = 0;
#pragma unroll
      for (int j = 0; j < (G + 3) / 4; ++j) {
        const uint32_t from = at + 2 * T::kNibbleBytes + T::kPairBytes + (uint32_t)((g * G + (t + 4 * j) % G) * 4);
        const uint32_t a = lds32(from) & 0x7fff7fffu, c = lds32(from + 8 * G * 4) & 0x7fff7fffu;
        scales = __vmaxu2(scales, __byte_perm(a, c, 0x5410));
        either = __vmaxu2(either, __vmaxu2(a, c));
      }
#pragma unroll
      for (int d = 1; d < (G < 4 ? G : 4); d <<= 1) scales = __vmaxu2(scales, __shfl_xor_sync(0xffffffffu, scales, d));
      const float2 f = pair_floats(scales);
      largest[0] = fmaxf(f.x, kLeastScale);
      largest[1] = fmaxf(f.y, kLeastScale);
      infinite = guard && __any_sync(0xffffffffu, __vcmpgeu2(either, 0x7c007c00u) != 0u);
    };
    // A tile's weights and outputs stand in one block of code with the next tile's products with the queries, so that the
    // chains of the one fill the waits of the other.
    uint32_t at = ring;
    int first = unit * kSlots;
    const int behind = first + seg * kSlots;
    float x[4];
    cp_async_wait<T::kStages - 2>();
    __syncwarp();
    find_largest(at);
    dot(at, x);
    finish(first, x);
#pragma unroll 1
    for (; first < behind; first += kSlots) {
      cp_async_wait<T::kStages - 3>();
      __syncwarp();  // the next tile is there, and everybody is done with the one before this, whose place the next request takes
      request();
      const uint32_t pairs_at = at + 2 * T::kNibbleBytes, next_at = at + T::kBytes == ring + T::kStages * T::kBytes ? ring : at + T::kBytes;
      // -- running maximum and unit; both rarely change --
      float pr[4];
      auto weigh = [&]() {
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = power2(fmaf(x[e] - m_run[e & 1], kLog2e, units[e & 1]));
      };
      weigh();
      // (no maximum is NaN)
      const float operand = fmaxf(fmaxf(pr[0], pr[1]) * largest[0], fmaxf(pr[2], pr[3]) * largest[1]);
      if (__any_sync(0xffffffffu, operand > kMostOperand)) {
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = fmaxf(x[e], x[2 + e]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          top = fmaxf(m_run[e], top);
          alpha[e] = power2((m_run[e] - top) * kLog2e);
          m_run[e] = top;
          // the largest product so far: of this tile, and by its unit of those before
          float most = fmaxf(fmaxf(power2((x[e] - top) * kLog2e) * largest[0], power2((x[2 + e] - top) * kLog2e) * largest[1]),
                             alpha[e] * __int_as_float((127 + kUnitBits - (int)units[e]) << 23));
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
          // (a weight is 1 at most here and a finite scale below 2^16, so -6 at least; with an infinite one nothing stays finite)
          const float now = fmaxf(fminf((float)(127 + kUnitBits - (__float_as_int(most) >> 23)), kMostUnits), -6.0f);
          alpha[e] *= __int_as_float((127 + (int)(now - units[e])) << 23);
          units[e] = now;
        }
        weigh();
        // (a least-value sum belongs to row g: its factor is with the threads of column g)
        const float even = __shfl_sync(0xffffffffu, alpha[0], g >> 1), odd = __shfl_sync(0xffffffffu, alpha[1], g >> 1);
        const float mine_alpha = (g & 1) ? odd : even;
        l_run[0] *= alpha[0];
        l_run[1] *= alpha[1];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) least_sum[gr] *= mine_alpha;
        const uint64_t both = packed(alpha[0], alpha[1]);
#pragma unroll
        for (int i = 0; i < 4 * P; ++i) o[i >> 2][(i >> 1) & 1][i & 1] = mul2(o[i >> 2][(i >> 1) & 1][i & 1], both);
      }
      // slots by rows -> rows by slots: row g, slots 2 t, 2 t + 1, 2 t + 8, 2 t + 9
      float pw[4];
      {
        l_run[0] += pr[0] + pr[2];
        l_run[1] += pr[1] + pr[3];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t c0 = __float_as_uint(pr[2 * e]), c1 = __float_as_uint(pr[2 * e + 1]);
          const uint32_t lo = transposed8x8(__byte_perm(c0, c1, 0x5410)), hi = transposed8x8(__byte_perm(c0, c1, 0x7632));
          pw[2 * e] = __uint_as_float(__byte_perm(lo, hi, 0x5410));
          pw[2 * e + 1] = __uint_as_float(__byte_perm(lo, hi, 0x7632));
        }
      }
      float y[4];
      // slots that some row does not see may hold anything: their weights are zero, and so must be their share
      const bool careful = infinite;
      find_largest(next_at);  // (behind the last tile: of whatever lies there, and not used; so are the logits)
      dot(next_at, y);
      // -- outputs: channels by slots times slots by rows; a weight is two fp16 numbers --
      uint32_t high[2], low[2], words[4];
#pragma unroll
      for (int i = 0; i < P; ++i) {
        if (i % kPer == 0) {
          const int gr = i / kPer;
          float ps[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t bits = lds32(pairs_at + T::kPairBytes + (uint32_t)(((2 * t + (j & 1) + 8 * (j >> 1)) * G + gr) * 4));
            const float2 f = pair_floats(bits);
            ps[j] = pw[j] * f.x;
            if (careful && pw[j] == 0.0f) {
              ps[j] = 0.0f;
            } else {
              least_sum[gr] = fmaf(pw[j], fmaf(8.0f, f.x, f.y), least_sum[gr]);
            }
          }
          split_halves(ps[0], ps[1], high[0], low[0]);
          split_halves(ps[2], ps[3], high[1], low[1]);
        }
        if (i % 2 == 0) load_matrices_transposed(at + T::kNibbleBytes + (matrix_at ^ (uint32_t)(i * 16)), words);
        uint32_t e[2][4];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t a = j ? words[2 * (i & 1)] >> 8 : words[2 * (i & 1)], c = j ? words[2 * (i & 1) + 1] >> 8 : words[2 * (i & 1) + 1];
          e[j][0] = centred.low(a), e[j][1] = centred.high(a), e[j][2] = centred.low(c), e[j][3] = centred.high(c);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float sum[4];
          first_product(sum, e[j][0], e[j][1], e[j][2], e[j][3], low[0], low[1]);
          product(sum, e[j][0], e[j][1], e[j][2], e[j][3], high[0], high[1]);
          o[i][j][0] = add2(o[i][j][0], packed(sum[0], sum[1]));
          o[i][j][1] = add2(o[i][j][1], packed(sum[2], sum[3]));
        }
      }
      at = next_at;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = y[e];
      if (first + kSlots < behind) finish(first + kSlots, x);
    }
    cp_async_wait<0>();

    // -- the warp's state, as a record: thread (g, t) has channels 4 g .. 4 g + 3 of every piece for rows 2 t and 2 t + 1 --
    const float from_units[2] = {__int_as_float((127 - (int)units[0]) << 23), __int_as_float((127 - (int)units[1]) << 23)};
    float* state = reinterpret_cast<float*>(smem + w * T::kWarpBytes);
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], d);
    __syncwarp();  // (the ring is not read any more)
#pragma unroll
    for (int gr = 0; gr < G; ++gr) {
      float sum = least_sum[gr];
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      const float least[2] = {__shfl_sync(0xffffffffu, sum, 8 * t), __shfl_sync(0xffffffffu, sum, 8 * t + 4)};
#pragma unroll
      for (int i = gr * kPer; i < (gr + 1) * kPer; ++i) {
        const float2 c0 = unpacked(o[i][0][0]), c1 = unpacked(o[i][0][1]), c2 = unpacked(o[i][1][0]), c3 = unpacked(o[i][1][1]);
        float* to_state = state + 2 * t * T::kRec + i * 32 + g * 4;
        *reinterpret_cast<float4*>(to_state) = make_float4((c0.x + least[0]) * from_units[0], (c1.x + least[0]) * from_units[0],
                                                           (c2.x + least[0]) * from_units[0], (c3.x + least[0]) * from_units[0]);
        *reinterpret_cast<float4*>(to_state + T::kRec) = make_float4((c0.y + least[1]) * from_units[1], (c1.y + least[1]) * from_units[1],
                                                                     (c2.y + least[1]) * from_units[1], (c3.y + least[1]) * from_units[1]);
      }
    }
    if (g < 2) {
      s_m[w][2 * t + g] = g ? m_run[1] : m_run[0];
      s_l[w][2 * t + g] = g ? l_run[1] * from_units[1] : l_run[0] * from_units[0];
    }
  } else if (lane < 8) {  // (no slot)
    s_m[w][lane] = -CUDART_INF_F;
    s_l[w][lane] = 0.0f;
  }
  if (lane == 0) s_pair[w] = pair;

  // -- the states of a CTA's pairs become records, or outputs --
  __syncthreads();
  if (threadIdx.x < 8 * kWarps) {
    const int j = threadIdx.x >> 3, row = threadIdx.x & 7, mine = s_pair[j];
    float top = -CUDART_INF_F;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) top = fmaxf(top, s_pair[i] == mine ? s_m[i][row] : -CUDART_INF_F);
    s_f[j][row] = power2((s_m[j][row] - (top == -CUDART_INF_F ? 0.0f : top)) * kLog2e);
  }
  __syncthreads();
#pragma unroll 1
  for (int first = 0; first < kWarps;) {
    const int mine = s_pair[first];
    if (mine < 0) break;  // (pieces are in order: behind a warp without one there is none)
    int end = first + 1;
#pragma unroll 1
    while (end < kWarps && s_pair[end] == mine) ++end;
    const int of_b = divide(mine, per, inverse_per), of_in_b = mine - of_b * per, of_kvh = divide(of_in_b, rw.chunks, inverse_chunks);
    const int row0 = (of_in_b - of_kvh * rw.chunks) * 8, rows = min(8, rw.rows - row0);
    float* rec = p.ws + (size_t)(cut.begin(blockIdx.x) + first) * 8 * T::kRec;
#pragma unroll 1
    for (int i = threadIdx.x; i < rows * (H / 4); i += T::kThreads) {
      const int row = i / (H / 4), d = i % (H / 4) * 4;
      float sum = 0.0f, top = -CUDART_INF_F;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        const bool here = j >= first && j < end && s_l[j][row] != 0.0f;  // (else there is no state, or nothing in it)
        const float f = s_f[j][row];
        const float4 v = *reinterpret_cast<const float4*>(smem + j * T::kWarpBytes + (row * T::kRec + d) * 4);
        top = fmaxf(top, here ? s_m[j][row] : -CUDART_INF_F);
        acc.x += here ? f * v.x : 0.0f;
        acc.y += here ? f * v.y : 0.0f;
        acc.z += here ? f * v.z : 0.0f;
        acc.w += here ? f * v.w : 0.0f;
        sum += here ? f * s_l[j][row] : 0.0f;
      }
      if (!cut.own_cta) {
        *reinterpret_cast<float4*>(rec + row * T::kRec + d) = acc;
        if (d == 0) *reinterpret_cast<float2*>(rec + row * T::kRec + H) = make_float2(top, sum);
      } else {
        const int i_q = divide(row0 + row, rw.group, inverse_group), head = of_kvh * rw.group + (row0 + row - i_q * rw.group);
        kv4_output<H, QF32>(p, stats_ws, of_b, i_q, head, mine, row, d, top, sum, acc);
      }
    }
    first = end;
  }
}

constexpr int kMergeThreads = 128;
constexpr int kScoreSlots = 256, kStatChunks = 16;

// Adds the weights that kScoreSlots slots of a KV head got to the scores. A row's maximum and sum come from its pair's records
// (or from the CTA that has the pair), again in every CTA: a kernel of its own behind the merge, which left them there, took
// 21.0 us in all instead of 20.3 at 16 x 8192 (16 heads of 128 over 2), and 21.7 instead of 17.9 for drafts of four tokens at
// 8 x 4096. (128 slots: 21.3 and 18.3 us; 512: 21.2 and 19.3; 1024: 23.3 and 22.4.)
template <int H>
__device__ void kv4_add_scores(const Kv4Sdpa& p, const Kv4Cut& cut, const Kv4Rows& rw, int b, int index, int below, int pieces, const float2* stats_ws,
                               const float* logits_ws) {
  constexpr int kRec = H + 4, kPerThread = kScoreSlots / kMergeThreads, kAtOnce = 4;
  __shared__ float2 s_stat[kStatChunks][8];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, row = lane & 7;
  const int parts = (p.cache.s + kScoreSlots - 1) / kScoreSlots, kvh = index / parts, slot0 = (index - kvh * parts) * kScoreSlots + tid;
  const int length = kv4_length(p, b);
  if (slot0 - tid >= length) return;
  const size_t pitch = (size_t)tiles_of(p.cache.s) * kSlots * 8;
  const size_t pair0 = ((size_t)b * p.cache.nkv + kvh) * rw.chunks;
  float4 next[kPerThread][2];
  auto ask = [&](int c) {
    const float* logits = logits_ws + (pair0 + c) * pitch;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
      const int slot = slot0 + j * kMergeThreads;
      const float4* from = reinterpret_cast<const float4*>(logits + (size_t)slot * 8);
      next[j][0] = next[j][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (slot < length) next[j][0] = __ldcg(from), next[j][1] = __ldcg(from + 1);
    }
  };
  ask(0);
  float sums[kPerThread];
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) sums[j] = 0.0f;
#pragma unroll 1
  for (int c = 0; c < rw.chunks; ++c) {
    if (c % kStatChunks == 0) {
      __syncthreads();
#pragma unroll 1
      for (int k = warp; k < min(kStatChunks, rw.chunks - c); k += kMergeThreads / 32) {
        const bool there = row < rw.rows - 8 * (c + k);
        float2 st = make_float2(0.0f, 0.0f);
        if (cut.own_cta) {
          if (there) st = __ldcg(stats_ws + (pair0 + c + k) * 8 + row);
        } else {
          const int first = below + (kvh * rw.chunks + c + k) * pieces, cta = cut.owner(first), count = cut.owner(first + pieces - 1) - cta + 1;
          float top = -CUDART_INF_F, sum = 0.0f;
#pragma unroll 1
          for (int j0 = lane >> 3; j0 < count; j0 += 4 * kAtOnce) {
            float2 ml[kAtOnce];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) {
              const int at = j0 + 4 * j;
              const float* rec = p.ws + (size_t)(at == 0 ? first : cut.begin(cta + min(at, count - 1))) * (8 * kRec);
              ml[j] = make_float2(-CUDART_INF_F, 0.0f);
              if (there && at < count) ml[j] = __ldcg(reinterpret_cast<const float2*>(rec + row * kRec + H));
            }
            float now = top;
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) now = fmaxf(now, ml[j].x);
            const float use = now == -CUDART_INF_F ? 0.0f : now;
            sum *= power2((top - use) * kLog2e);
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) sum = fmaf(power2((ml[j].x - use) * kLog2e), ml[j].y, sum);
            top = now;
          }
#pragma unroll
          for (int o = 8; o < 32; o <<= 1) {
            const float top2 = __shfl_xor_sync(0xffffffffu, top, o), sum2 = __shfl_xor_sync(0xffffffffu, sum, o);
            const float now = fmaxf(top, top2), use = now == -CUDART_INF_F ? 0.0f : now;
            // (the same sum in both lanes: a + b = b + a)
            sum = __fadd_rn(__fmul_rn(power2((top - use) * kLog2e), sum), __fmul_rn(power2((top2 - use) * kLog2e), sum2));
            top = now;
          }
          st = make_float2(top == -CUDART_INF_F ? 0.0f : top, sum != 0.0f ? 1.0f / sum : 0.0f);
        }
        if (lane < 8) s_stat[k][row] = st;
      }
      __syncthreads();
    }
    float4 x[kPerThread][2];
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) x[j][0] = next[j][0], x[j][1] = next[j][1];
    if (c + 1 < rw.chunks) ask(c + 1);
    const int rows = rw.rows - 8 * c;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 st = s_stat[c % kStatChunks][e];
#pragma unroll
      for (int j = 0; j < kPerThread; ++j) {
        const float4 y = x[j][e / 4];
        const float v = e % 4 == 0 ? y.x : e % 4 == 1 ? y.y : e % 4 == 2 ? y.z : y.w;
        if (e < rows) sums[j] = fmaf(power2((v - st.x) * kLog2e), st.y, sums[j]);
      }
    }
  }
  float* scores = p.scores + ((size_t)b * p.cache.nkv + kvh) * p.cache.s;
#pragma unroll
  for (int j = 0; j < kPerThread; ++j) {
    const int slot = slot0 + j * kMergeThreads;
    if (slot < length) scores[slot] += sums[j];
  }
}

// Merges the records of one query row, H >> part_log2 channels per CTA. What it costs are its start and L2 round trips, so
// there is one for all records up to 32 (12 for fp16 rows of 256; twice and four times as many where the channels are parted),
// requested before their weights are known. fp16 rows of up to 128 channels: 64 registers, so that more CTAs, those of the
// scores too, are resident (16 heads of 128 over 2 with scores, 16 x 8192: 1.4 us less of 22.6; of 256 channels 0.8 more of 15.2 without
// scores, and 0.8 more at 64 x 32768, so not those). (The main kernel at 224 registers, to leave room for these CTAs beside it: 82.6 us where
// it took 78 at 64 x 32768.)
// The CTAs behind the first `merge_ctas` of a sequence add to the scores.
template <int H, bool QF32>
__global__ void __launch_bounds__(kMergeThreads, QF32 || H == 256 ? 1 : 8) kv4_merge_kernel(const Kv4Sdpa p, const int ctas, const int merge_ctas, const int part_log2,
                                                                 const float2* stats_ws, const float* logits_ws) {
  constexpr int kRec = H + 4, kBatch = H == 256 && !QF32 ? 6 : H / 16;
  __shared__ float4 s_part[kMergeThreads];
  __shared__ float s_sum[kMergeThreads];
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
  const Kv4Rows rw = kv4_rows(p.t, p.n, p.cache.nkv);
  const int per = p.cache.nkv * rw.chunks;
  const int row = blockIdx.x >> part_log2, part = blockIdx.x & ((1 << part_log2) - 1);
  const int i = row / p.n, head = row - i * p.n, kvh = head / rw.group, r = i * rw.group + head - kvh * rw.group;
  const int quads = (H / 4) >> part_log2, groups = kMergeThreads / quads;  // powers of two
  const int quad = tid & (quads - 1), grp = tid / quads, d = 4 * (part * quads + quad);
  // what does not depend on the kernel before: it has waited for whatever wrote the lengths
  const Kv4Cut cut = kv4_cut(p, per, ctas, kv4_warps(H), lane);
  int below = 0, pieces = 0;  // pieces of the sequences before b, and of each pair of b
#pragma unroll 1
  for (int j = lane; j < b; j += 32) below += cut.pieces_of(j == lane ? cut.len : kv4_length(p, j)) * per;
  below = (int)__reduce_add_sync(0xffffffffu, (unsigned)below);
  pieces = cut.pieces_of(kv4_length(p, b));
  const int in_b = kvh * rw.chunks + (r >> 3), first = below + in_b * pieces, cta = cut.owner(first);
  const int count = pieces == 0 ? 0 : cut.owner(first + pieces - 1) - cta + 1;  // under the first piece, and that of every further CTA
  const float* base = p.ws + (r & 7) * kRec;
  pdl_launch_dependents();
  pdl_wait();
  if ((int)blockIdx.x >= merge_ctas) return kv4_add_scores<H>(p, cut, rw, b, blockIdx.x - merge_ctas, below, pieces, stats_ws, logits_ws);
  if (cut.own_cta) return;
  float sum = 0.0f, top = -CUDART_INF_F;
  float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
  for (int j0 = 0; j0 < count; j0 += kBatch * groups) {
    float2 ml[kBatch];
    float4 v[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {  // (all in flight at once; without a weight where there are fewer)
      const int at = j0 + grp + j * groups, to = min(at, count - 1);
      const float* rec = base + (size_t)(to == 0 ? first : cut.begin(cta + to)) * (8 * kRec);
      ml[j] = __ldcg(reinterpret_cast<const float2*>(rec + H));
      v[j] = __ldcg(reinterpret_cast<const float4*>(rec + d));
    }
    float now = top;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) now = fmaxf(now, ml[j].x);
    const float use = now == -CUDART_INF_F ? 0.0f : now;
    const float keep = top == -CUDART_INF_F ? 0.0f : power2((top - use) * kLog2e);
    top = now;
    acc.x *= keep, acc.y *= keep, acc.z *= keep, acc.w *= keep;
    sum *= keep;
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const float f = j0 + grp + j * groups < count ? power2((ml[j].x - use) * kLog2e) : 0.0f;
      acc.x = fmaf(f, v[j].x, acc.x);
      acc.y = fmaf(f, v[j].y, acc.y);
      acc.z = fmaf(f, v[j].z, acc.z);
      acc.w = fmaf(f, v[j].w, acc.w);
      sum = fmaf(f, ml[j].y, sum);
    }
  }
  // the groups' sums, each under its own maximum
  __shared__ float s_top[kMergeThreads];
  s_part[tid] = acc;
  s_sum[tid] = sum;
  s_top[tid] = top;
  __syncthreads();
  if (grp > 0) return;
#pragma unroll 1
  for (int j = 1; j < groups; ++j) top = fmaxf(top, s_top[j * quads + quad]);
  const float use = top == -CUDART_INF_F ? 0.0f : top;
  acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  sum = 0.0f;
#pragma unroll 1
  for (int j = 0; j < groups; ++j) {
    const int at = j * quads + quad;
    const float f = power2((s_top[at] - use) * kLog2e);
    const float4 v = s_part[at];
    acc.x = fmaf(f, v.x, acc.x);
    acc.y = fmaf(f, v.y, acc.y);
    acc.z = fmaf(f, v.z, acc.z);
    acc.w = fmaf(f, v.w, acc.w);
    sum = fmaf(f, s_sum[at], sum);
  }
  kv4_output<H, QF32>(p, nullptr, b, i, head, b * per + in_b, r & 7, d, top, sum, acc);
}

// CTAs of a launch: one per SM, fewer when even full caches leave some without a tile, more where the pairs are so many that
// their pieces would not find warps.
int kv4_ctas(long long pairs, int s, int h) {
  const long long most = pairs * tiles_of(s), room = (2 * pairs + kv4_warps(h) - 1) / kv4_warps(h);
  const long long n = room > device_sm_count() ? room : device_sm_count();
  return (int)(most < n ? most : n);
}

bool kv4_tensor_shape(int b, int t, int n, int nkv, int h, int s) {
  const long long pairs = (long long)b * nkv * kv4_rows(t, n, nkv).chunks;
  return (h == 64 || h == 128 || h == 256) && pairs * tiles_of(s) <= INT32_MAX / 2 && pairs <= (1 << 19) && tiles_of(s) < (1 << 22);
}

template <int H, int BLOCK, bool QF32>
cudaError_t launch_tensor(const Kv4Sdpa& p, cudaStream_t s) {
  using T = Kv4Tile<H, BLOCK, QF32>;
  const long long pairs = (long long)p.cache.b * p.cache.nkv * kv4_rows(p.t, p.n, p.cache.nkv).chunks;
  const int ctas = kv4_ctas(pairs, p.cache.s, H);
  float* behind = p.ws + kv4_records_floats((long long)ctas * T::kWarps, H);
  float2* stats = p.scores ? reinterpret_cast<float2*>(behind) : nullptr;
  float* logits = p.scores ? behind + 16 * pairs : nullptr;
  static bool done[64] = {false};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 0 || device >= 64) device = 0;
  if (!done[device]) {
    const cudaError_t e = cudaFuncSetAttribute(kv4_sdpa_kernel<H, BLOCK, QF32>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem);
    if (e != cudaSuccess) return e;
    done[device] = true;
  }
  cudaError_t e = launch_chained(kv4_sdpa_kernel<H, BLOCK, QF32>, dim3(ctas), dim3(T::kThreads), (size_t)T::kSmem, s, p, stats, logits);
  if (e != cudaSuccess) return e;
  const bool merge = pairs > ctas || tiles_of(p.cache.s) > 4 * T::kWarps;  // (else every pair is a CTA's: kv4_cut)
  int part_log2 = 0;  // few rows are cut by channels too: their records are many
  while (part_log2 < 2 && ((long long)p.cache.b * p.n * p.t << part_log2) < 2 * device_sm_count()) ++part_log2;
  const int merge_ctas = merge ? (p.n * p.t) << part_log2 : 0;
  const int score_ctas = p.scores ? (p.cache.s + kScoreSlots - 1) / kScoreSlots * p.cache.nkv : 0;
  if (merge_ctas + score_ctas == 0) return cudaSuccess;
  return launch_chained(kv4_merge_kernel<H, QF32>, dim3(merge_ctas + score_ctas, p.cache.b), dim3(kMergeThreads), 0, s, p, ctas, merge_ctas, part_log2,
                        (const float2*)stats, (const float*)logits);
}
template <int H, int BLOCK>
cudaError_t launch_tensor_q(const Kv4Sdpa& p, cudaStream_t s) {
  return p.f32 ? launch_tensor<H, BLOCK, true>(p, s) : launch_tensor<H, BLOCK, false>(p, s);
}
template <int H>
cudaError_t launch_tensor_block(const Kv4Sdpa& p, cudaStream_t s) {
  return p.cache.block == 64 ? launch_tensor_q<H, 64>(p, s) : launch_tensor_q<H, 32>(p, s);
}

}  // namespace

size_t kv4_sdpa_workspace_bytes(int b, int t, int n, int nkv, int h, int s, int scores) {
  const size_t rows = (size_t)b * t * n;
  if (!kv4_tensor_shape(b, t, n, nkv, h, s)) return (2 * rows + rows * s) * sizeof(float);
  const long long pairs = (long long)b * nkv * kv4_rows(t, n, nkv).chunks;
  const size_t tensor = kv4_records_floats((long long)kv4_ctas(pairs, s, h) * kv4_warps(h), h) +
                        (scores ? 16 * (size_t)pairs + (size_t)pairs * tiles_of(s) * kSlots * 8 : 0);
  return tensor * sizeof(float);
}

cudaError_t launch_kv4_sdpa(const Kv4Sdpa& p, cudaStream_t s) {
  const Kv4Cache& c = p.cache;
  if (!kv4_tensor_shape(c.b, p.t, p.n, c.nkv, c.h, c.s)) return launch_rows(p, s);
  return c.h == 256 ? launch_tensor_block<256>(p, s) : c.h == 128 ? launch_tensor_block<128>(p, s) : launch_tensor_block<64>(p, s);
}

}  // namespace b200
