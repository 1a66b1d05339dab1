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

// ---- head sizes 64, 128 and 256: tensor cores -------------------------------------------------------------
// Up to eight query rows of a KV head (query heads x query tokens) are the 8-wide side of mma.m16n8k16; a tile is 32 slots,
// two 16-row sides of it whose chains of products and exponentials run side by side. Every (sequence, KV head, eight rows)
// pair is cut into pieces of a common greatest length, one per warp. A warp walks through its piece without meeting another
// one; at the end the warps of a CTA add their states of a common pair to one partial record (un-normalised outputs, maximum,
// sum), and a second kernel merges a pair's records.
// Measured with 16 ragged sequences of up to 8192 tokens, 8 heads x 256, replayed: pieces that run on from one pair to the
// next (all of one length) 17.5 us, 4 of them in the warps that had parts of two pairs; such pieces per CTA 19.4; a record
// for every warp 20.3 (the second kernel reads 9.8 MB then).
constexpr int kSlots = 32;
__host__ __device__ inline int tiles_of(int slots) { return (slots + kSlots - 1) / kSlots; }

__host__ __device__ constexpr int kv4_warps(int h) { return h == 256 ? 8 : h == 128 ? 12 : 16; }

template <int H, int BLOCK>
struct Kv4Tile {
  static constexpr int kG = H / BLOCK;                 // blocks of a row
  static constexpr int kNibbleBytes = kSlots * H / 2;  // of the keys (or values) of a tile
  static constexpr int kPairBytes = kSlots * kG * 4;
  static constexpr int kBytes = 2 * (kNibbleBytes + kPairBytes);
  static constexpr int kWarps = kv4_warps(H);
  static constexpr int kThreads = 32 * kWarps;
  static constexpr int kRec = H + 4;  // floats of a record per row: outputs, maximum, sum, padding
  static constexpr int kFit = 220 * 1024 / (kWarps * kBytes);
  static constexpr int kStages = kFit > 6 ? 6 : kFit;
  static constexpr int kRing = kWarps * kStages * kBytes;
  static constexpr int kSmem = kRing + 128;
  static_assert(8 * kRec * 4 <= kStages * kBytes, "a warp's state fits into its ring");
  static_assert(kBytes % 128 == 0 && kStages >= 2 && kSmem <= 221 * 1024, "layout");
};

struct Kv4Rows {
  int group, rows, chunks;  // query heads per KV head; query rows per KV head; of eight rows each
};
__host__ __device__ inline Kv4Rows kv4_rows(int t, int n, int nkv) {
  const int group = n / nkv, rows = t * group;
  return {group, rows, (rows + 7) / 8};
}

// Workspace of the tensor-core kernels: a record per piece (of which the first of a pair in each CTA is written), then the
// logits [pair][slot (rounded up to a tile)][8 rows] where scores are wanted.
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

// How the pairs are cut: into pieces of up to about `size` tiles, each pair's of equal lengths (to a tile), the smallest size
// that needs no more pieces than there are warps. Every CTA gets an equal number of the pieces (to one). What is rounded
// here is so in both kernels.
struct Kv4Cut {
  int size, each, longer;  // the first `longer` CTAs have one piece more than `each`
  float inverse;           // 1 / size
  int len;                 // attended slots of sequence `lane`
  __device__ __forceinline__ int pieces_of(int slots) const {
    const int tiles = tiles_of(slots);
    return tiles == 0 ? 0 : max(1, min(tiles, (int)((float)(tiles + size - 1) * inverse)));
  }
  __device__ __forceinline__ int begin(int cta) const { return cta * each + min(cta, longer); }
  __device__ __forceinline__ int owner(int piece) const {
    const int front = longer * (each + 1);
    return piece < front ? divide(piece, each + 1, __frcp_rn((float)(each + 1))) : longer + divide(piece - front, each, __frcp_rn((float)each));
  }
};
// Pieces of the sequences below `upto`, all pairs. Whole warp.
__device__ __forceinline__ int count_pieces(const Kv4Sdpa& p, int per, const Kv4Cut& c, int lane, int upto) {
  int n = lane < upto ? c.pieces_of(c.len) * per : 0;
  for (int i = lane + 32; i < upto; i += 32) n += c.pieces_of(kv4_length(p, i)) * per;
  return (int)__reduce_add_sync(0xffffffffu, (unsigned)n);
}
__device__ __forceinline__ Kv4Cut kv4_cut(const Kv4Sdpa& p, int per, int ctas, int warps, int lane) {
  const int room = ctas * warps;
  const float inverse_room = __frcp_rn((float)room), inverse_ctas = __frcp_rn((float)ctas);
  Kv4Cut c;
  c.len = lane < p.cache.b ? kv4_length(p, lane) : 0;
  int total = tiles_of(c.len) * per;
  for (int i = lane + 32; i < p.cache.b; i += 32) total += tiles_of(kv4_length(p, i)) * per;
  total = (int)__reduce_add_sync(0xffffffffu, (unsigned)total);
  c.size = max(1, (int)ceilf((float)total * inverse_room));
  int n;
  while (true) {  // (ends: there is room for twice the pairs, and a large enough size makes a piece of each)
    c.inverse = __frcp_rn((float)c.size);
    n = count_pieces(p, per, c, lane, p.cache.b);
    if (n <= room) break;
    c.size += 1 + c.size / 16;
  }
  c.each = divide(n, ctas, inverse_ctas);
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
template <int N>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&v)[N]) {
  if constexpr (N == 1) {
    v[0] = lds32(a);
  } else if constexpr (N == 2) {
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(a));
  } else {
#pragma unroll
    for (int i = 0; i < N; i += 4)
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3]) : "r"(a + 4 * i));
  }
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

// Key nibbles become fp16 operands by a mask alone: in the low bits of a half, nibble u is the subnormal number u 2^-24,
// one place up u 2^-20. So a word of eight nibbles is four pairs after one shift and four masks, exactly; the factor 16
// between the two kinds goes into the queries of those channels, 2^-24 into the logits' factor.
// Value nibbles are centred, u - 8, by way of the exponents that make a nibble's place the unit (1024) or an eighth of it
// (64): sums of weights times values that are all positive lose to the tensor core's truncation (float32 outputs were
// 3e-5 off; 8 x scale joins the least value instead).
constexpr uint32_t kLowNibbles = 0x000f000fu, kHighNibbles = 0x00f000f0u;
__device__ __forceinline__ uint32_t half2_sub(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t centred_low(uint32_t w) { return half2_sub((w & kLowNibbles) | 0x64006400u, 0x64086408u); }    // - 1032
__device__ __forceinline__ uint32_t centred_high(uint32_t w) { return half2_sub((w & kHighNibbles) | 0x54005400u, 0x54805480u); }  // - 72

template <int H, int BLOCK, bool QF32>
__global__ void __launch_bounds__(Kv4Tile<H, BLOCK>::kThreads, 1) kv4_sdpa_kernel(const Kv4Sdpa p, float* logits_ws) {
  using T = Kv4Tile<H, BLOCK>;
  constexpr int G = T::kG;
  constexpr int P = H / 32;           // 16-byte pieces of a row
  constexpr int kPer = BLOCK / 32;    // of them in a block
  extern __shared__ uint8_t kv4_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(kv4_smem_raw) + 127) & ~uintptr_t(127));
  __shared__ float s_m[T::kWarps][8], s_l[T::kWarps][8];  // maxima and sums of the warps' states
  __shared__ int s_pair[T::kWarps];                       // and whose these are
  __shared__ int s_rows[T::kWarps];
  const int w = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int nkv = p.cache.nkv, s_max = p.cache.s;
  const Kv4Rows rw = kv4_rows(p.t, p.n, nkv);
  const int per = nkv * rw.chunks;  // pairs per sequence
  // this warp's ring; where a lane's copies come from and go to (16-byte piece `lane % P` of rows lane / P + 32 / P j)
  const uint32_t ring = smem_u32(smem) + (uint32_t)(w * T::kStages * T::kBytes);
  const uint32_t row_pitch = (uint32_t)nkv * (H / 2), pair_pitch = (uint32_t)nkv * G * 4;  // bytes
  const int copy_row = lane / P, copy_piece = lane % P;
  const uint32_t copy_from = (uint32_t)copy_row * row_pitch + copy_piece * 16, pair_from = (uint32_t)(lane / G) * pair_pitch + lane % G * 4;
  const uint32_t row_step = row_pitch * (32 / P), pair_step = pair_pitch * (32 / G);
  // the row that this lane names for a load of matrices: of two pieces, rows 0 .. 15
  const uint32_t matrix_at = piece_at<H>((lane & 7) + ((lane >> 3) & 1) * 8, lane >> 4);
  const float inverse_chunks = __frcp_rn((float)rw.chunks), inverse_group = __frcp_rn((float)rw.group);
  pdl_wait();
  // (only now: what a dependent kernel does ahead of its own wait may then read this kernel's inputs)
  pdl_launch_dependents();
  // this warp's piece
  const Kv4Cut cut = kv4_cut(p, per, gridDim.x, T::kWarps, lane);
  const int first_piece = cut.begin(blockIdx.x), piece = first_piece + w;
  int seg = 0, b = 0, in_b = 0, unit = 0, len = cut.len;  // seg tiles from `unit` on of pair in_b of sequence b
  if (w < cut.each + ((int)blockIdx.x < cut.longer ? 1 : 0)) {
    for (int b0 = 0, base = 0; b0 < p.cache.b; b0 += 32) {
      if (b0 > 0) len = b0 + lane < p.cache.b ? kv4_length(p, b0 + lane) : 0;
      int n = cut.pieces_of(len), upto = n * per;  // inclusive prefix sum over the lanes
#pragma unroll
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
        const float inverse = __frcp_rn((float)n);
        in_b = divide(rest, n, inverse);
        const int part = rest - in_b * n, tiles = tiles_of(len), each = divide(tiles, n, inverse), longer = tiles - each * n;
        unit = part * each + min(part, longer);
        seg = each + (part < longer ? 1 : 0);
        break;
      }
      base += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  if (lane == 0) s_pair[w] = -1;  // no state yet

  if (seg > 0) {
    const int kvh = divide(in_b, rw.chunks, inverse_chunks), chunk = in_b - kvh * rw.chunks;
    const int pair = b * per + in_b;
    // the queries are asked for first, the tiles arrive meanwhile
    const int q_row = chunk * 8 + g;
    uint4 q_bits[QF32 ? 2 * P : P];
    {
      const int i = divide(q_row, rw.group, inverse_group);
      const size_t at = (((size_t)b * p.t + i) * p.n + kvh * rw.group + (q_row - i * rw.group)) * H + 8 * t;
#pragma unroll
      for (int sl = 0; sl < P; ++sl) {
        if constexpr (QF32) {
          const uint4* src = reinterpret_cast<const uint4*>(static_cast<const float*>(p.q) + at + 32 * sl);
          q_bits[2 * sl] = q_row < rw.rows ? __ldg(src) : make_uint4(0, 0, 0, 0);
          q_bits[2 * sl + 1] = q_row < rw.rows ? __ldg(src + 1) : make_uint4(0, 0, 0, 0);
        } else {
          q_bits[sl] = q_row < rw.rows ? __ldg(reinterpret_cast<const uint4*>(static_cast<const __half*>(p.q) + at + 32 * sl)) : make_uint4(0, 0, 0, 0);
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
          for (int j = 0; j < P; ++j) {
            cp_async16(to + piece_at<H>(copy_row + j * (32 / P), copy_piece), advance(ks, j, row_step));
            cp_async16(to + T::kNibbleBytes + piece_at<H>(copy_row + j * (32 / P), copy_piece), advance(vs, j, row_step));
          }
#pragma unroll
          for (int j = 0; j < G; ++j) {
            cp_async4(to + 2 * T::kNibbleBytes + (lane + 32 * j) * 4, advance(kps, j, pair_step));
            cp_async4(to + 2 * T::kNibbleBytes + T::kPairBytes + (lane + 32 * j) * 4, advance(vps, j, pair_step));
          }
        } else {  // (one tile of a pair at most)
#pragma unroll 1
          for (int j = 0; j < P; ++j) {
            const int row = copy_row + j * (32 / P);
            const bool ok = row < there;
            const uint32_t from = ok ? copy_from + j * row_step : 0u;
            cp_async16_or_zero(to + piece_at<H>(row, copy_piece), k_next + from, ok);
            cp_async16_or_zero(to + T::kNibbleBytes + piece_at<H>(row, copy_piece), v_next + from, ok);
          }
#pragma unroll 1
          for (int j = 0; j < G; ++j) {
            const bool ok = (lane + 32 * j) / G < there;
            const uint32_t from = ok ? pair_from + j * pair_step : 0u;
            cp_async4_or_zero(to + 2 * T::kNibbleBytes + (lane + 32 * j) * 4, reinterpret_cast<const uint8_t*>(kp_next) + from, ok);
            cp_async4_or_zero(to + 2 * T::kNibbleBytes + T::kPairBytes + (lane + 32 * j) * 4, reinterpret_cast<const uint8_t*>(vp_next) + from, ok);
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

    // Queries: thread (g, t) holds row g's elements at its words of a key, as the B operand. They are scaled by a power of
    // two that brings the row's largest to 2^10 .. 2^11: dividing by 16 then loses nothing above 2^-36 of it, and a float32
    // query is two fp16 numbers to 22 bits.
    uint32_t q_high[P][4], q_low[QF32 ? P : 1][4];
    float q_sum[G][2], factor[2];  // of the rows 2 t and 2 t + 1 (the products' columns)
    int limit[2];
    {
      float raw[P][8], top = 0.0f;
#pragma unroll
      for (int sl = 0; sl < P; ++sl) {
        if constexpr (QF32) {
          const uint4 lo = q_bits[2 * sl], hi = q_bits[2 * sl + 1];
          raw[sl][0] = __uint_as_float(lo.x), raw[sl][1] = __uint_as_float(lo.y), raw[sl][2] = __uint_as_float(lo.z), raw[sl][3] = __uint_as_float(lo.w);
          raw[sl][4] = __uint_as_float(hi.x), raw[sl][5] = __uint_as_float(hi.y), raw[sl][6] = __uint_as_float(hi.z), raw[sl][7] = __uint_as_float(hi.w);
        } else {
          const uint4 v = q_bits[sl];
          const float2 f0 = pair_floats(v.x), f1 = pair_floats(v.y), f2 = pair_floats(v.z), f3 = pair_floats(v.w);
          raw[sl][0] = f0.x, raw[sl][1] = f0.y, raw[sl][2] = f1.x, raw[sl][3] = f1.y;
          raw[sl][4] = f2.x, raw[sl][5] = f2.y, raw[sl][6] = f3.x, raw[sl][7] = f3.y;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(raw[sl][e]));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int exponent = __float_as_int(top) >> 23;
      const int up = exponent == 255 ? 127 : min(264 - exponent, 253);  // (an infinite query stays what it is)
      const float scale_up = __int_as_float(up << 23), scale_down = __int_as_float((254 - up) << 23);
      float sums[G];
#pragma unroll
      for (int gr = 0; gr < G; ++gr) sums[gr] = 0.0f;
#pragma unroll
      for (int sl = 0; sl < P; ++sl) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          raw[sl][e] *= scale_up;
          sums[sl / kPer] += raw[sl][e];
        }
        // channels 0, 4 | 2, 6 meet low nibbles, 1, 5 | 3, 7 high ones
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int c = e < 2 ? 2 * e : 2 * (e - 2) + 1;
          const float f = e < 2 ? 1.0f : 0.0625f;
          if constexpr (QF32) {
            split_halves(raw[sl][c] * f, raw[sl][c + 4] * f, q_high[sl][e], q_low[sl][e]);
          } else {
            q_high[sl][e] = halves(raw[sl][c] * f, raw[sl][c + 4] * f);
          }
        }
      }
#pragma unroll
      for (int gr = 0; gr < G; ++gr) {
        sums[gr] += __shfl_xor_sync(0xffffffffu, sums[gr], 1);
        sums[gr] += __shfl_xor_sync(0xffffffffu, sums[gr], 2);
        sums[gr] *= 0x1p-24f;
        q_sum[gr][0] = __shfl_sync(0xffffffffu, sums[gr], 8 * t);
        q_sum[gr][1] = __shfl_sync(0xffffffffu, sums[gr], 8 * t + 4);
      }
      const float f = scale_down * p.scale;
      // (in two steps: 2^24 times a small scale stays within fp32 either way)
      factor[0] = __shfl_sync(0xffffffffu, f, 8 * t) * 0x1p24f;
      factor[1] = __shfl_sync(0xffffffffu, f, 8 * t + 4) * 0x1p24f;
    }
    const float* mask[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = chunk * 8 + 2 * t + e, i = divide(r, rw.group, inverse_group);
      limit[e] = r < rw.rows ? kv4_limit(len, s_max, p.t, i) : len;  // (columns without a row are computed and dropped)
      mask[e] = p.mask && r < rw.rows ? p.mask + ((size_t)b * p.t + i) * s_max : nullptr;
    }
    const int least_limit = kv4_limit(len, s_max, p.t, divide(chunk * 8, rw.group, inverse_group));  // of any row
    // masks are requested a tile ahead of their use
    auto masks = [&](int k, float (&m)[2][4]) {
      const int first = (unit + k) * kSlots;
#pragma unroll
      for (int side = 0; side < 2; ++side)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int slot = first + 16 * side + g + 8 * (e >> 1);
          m[side][e] = mask[e & 1] && k < seg && slot < limit[e & 1] ? __ldg(mask[e & 1] + slot) : 0.0f;
        }
    };
    float next_mask[2][4];
    masks(0, next_mask);
    const bool guard = p.mask != nullptr || p.t > 1;  // slots that some row does not see may hold anything
    float* logits = logits_ws ? logits_ws + (size_t)pair * ((size_t)tiles_of(s_max) * kSlots * 8) : nullptr;

    // outputs: of piece i and its channels 4 g + {0, 1} and 4 g + {2, 3}, rows 2 t and 2 t + 1
    float o[P][2][4], least_sum[G];
#pragma unroll
    for (int gr = 0; gr < G; ++gr) least_sum[gr] = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[i][0][e] = o[i][1][e] = 0.0f;
    float m_run[2] = {-CUDART_INF_F, -CUDART_INF_F}, m_use[2] = {0.0f, 0.0f}, l_run[2] = {0.0f, 0.0f};
    uint32_t exponent = 1;  // fp16 exponent field of the largest value scale so far: weights are in units of 2^(exponent - 23)

    uint32_t at = ring;
#pragma unroll 1
    for (int k = 0; k < seg; ++k, at = at + T::kBytes == ring + T::kStages * T::kBytes ? ring : at + T::kBytes) {
      cp_async_wait<T::kStages - 2>();
      __syncwarp();  // the tile is there, and everybody is done with the one whose place the next request takes
      request();
      const uint32_t pairs_at = at + 2 * T::kNibbleBytes;
      const int first = (unit + k) * kSlots;

      // -- logits of slots g, g + 8 (+ 16), rows 2 t and 2 t + 1 --
      float x[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
      // Four pieces and both sides at a time, one product of each chain after the other: a warp waits for a chain's last
      // product before its next.
      constexpr int kAtOnce = P < 4 ? P : 4, kChains = kAtOnce / kPer;
#pragma unroll
      for (int i0 = 0; i0 < P; i0 += kAtOnce) {
        uint32_t words[2][kAtOnce / 2][4];
#pragma unroll
        for (int i = 0; i < kAtOnce; i += 2)
#pragma unroll
          for (int side = 0; side < 2; ++side)
            load_matrices(at + (matrix_at ^ (uint32_t)((i0 + i) * 16)) + side * 8 * H, words[side][i / 2]);
        float acc[2][kChains][4];
#pragma unroll
        for (int j = 0; j < kPer; ++j) {
#pragma unroll
          for (int odd = 0; odd < 2; ++odd)
#pragma unroll
            for (int c = 0; c < kChains; ++c)
#pragma unroll
              for (int side = 0; side < 2; ++side) {
                const int i = c * kPer + j;
                const uint32_t wa = words[side][i / 2][2 * (i & 1)], wb = words[side][i / 2][2 * (i & 1) + 1];
                const uint32_t keep = odd ? kHighNibbles : kLowNibbles;
                const uint32_t a0 = wa & keep, a1 = wb & keep, a2 = (wa >> 8) & keep, a3 = (wb >> 8) & keep;
                if (j == 0 && odd == 0) {
                  first_product(acc[side][c], a0, a1, a2, a3, q_high[i0 + i][0], q_high[i0 + i][1]);
                } else {
                  product(acc[side][c], a0, a1, a2, a3, q_high[i0 + i][2 * odd], q_high[i0 + i][2 * odd + 1]);
                }
                if constexpr (QF32) product(acc[side][c], a0, a1, a2, a3, q_low[i0 + i][2 * odd], q_low[i0 + i][2 * odd + 1]);
              }
        }
#pragma unroll
        for (int c = 0; c < kChains; ++c)
#pragma unroll
          for (int side = 0; side < 2; ++side) {
            const int gr = i0 / kPer + c;
            const float2 fa = pair_floats(lds32(pairs_at + (uint32_t)(((16 * side + g) * G + gr) * 4)));
            const float2 fb = pair_floats(lds32(pairs_at + (uint32_t)(((16 * side + g + 8) * G + gr) * 4)));
            x[side][0] = fmaf(fa.x, acc[side][c][0], fmaf(fa.y, q_sum[gr][0], x[side][0]));
            x[side][1] = fmaf(fa.x, acc[side][c][1], fmaf(fa.y, q_sum[gr][1], x[side][1]));
            x[side][2] = fmaf(fb.x, acc[side][c][2], fmaf(fb.y, q_sum[gr][0], x[side][2]));
            x[side][3] = fmaf(fb.x, acc[side][c][3], fmaf(fb.y, q_sum[gr][1], x[side][3]));
          }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] *= factor[e & 1];
      if (p.logit_cap > 0.0f) {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e >> 2][e & 3] = p.logit_cap * tanhf(x[e >> 2][e & 3] / p.logit_cap);
      }
      if (p.mask) {
        float m[2][4];
#pragma unroll
        for (int e = 0; e < 8; ++e) m[e >> 2][e & 3] = next_mask[e >> 2][e & 3];
        masks(k + 1, next_mask);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float a = m[e >> 2][e & 3];
          x[e >> 2][e & 3] = a == -CUDART_INF_F ? a : x[e >> 2][e & 3] + a;
        }
      }
      if (first + kSlots > least_limit) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int slot = first + 16 * (e >> 2) + g + 8 * ((e >> 1) & 1);
          x[e >> 2][e & 3] = slot < limit[e & 1] ? x[e >> 2][e & 3] : -CUDART_INF_F;
        }
      }
      if (logits) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          *reinterpret_cast<float2*>(logits + (size_t)(first + g + 8 * e) * 8 + 2 * t) = make_float2(x[e >> 1][2 * (e & 1)], x[e >> 1][2 * (e & 1) + 1]);
      }

      // -- running maximum and unit; both rarely change --
      // A weight may exceed 1 by e^kSlack: rescaling the outputs at every new maximum would happen in most tiles while a
      // warp has seen few. The largest value scale of the tile: pairs compared as halves.
      constexpr float kSlack = 4.0f;
      __half2 largest = __float2half2_rn(0.0f);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const uint32_t pw_ = lds32(pairs_at + T::kPairBytes + (uint32_t)(lane + 32 * j) * 4);
        largest = __hmax2(largest, *reinterpret_cast<const __half2*>(&pw_));
      }
      const uint32_t largest_bits = *reinterpret_cast<const uint32_t*>(&largest) & 0x7fffu;
      const uint32_t now = max(exponent, min(__reduce_max_sync(0xffffffffu, largest_bits) >> 10, 30u));
      float tops[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) tops[e] = fmaxf(fmaxf(x[0][e], x[0][2 + e]), fmaxf(x[1][e], x[1][2 + e]));
      const bool grows = tops[0] > m_run[0] + kSlack || tops[1] > m_run[1] + kSlack;
      if (__any_sync(0xffffffffu, grows) || now != exponent) {
        float alpha[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = tops[e];
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
          top = fmaxf(m_run[e], top);
          const float use = top == -CUDART_INF_F ? 0.0f : top;
          alpha[e] = m_run[e] == -CUDART_INF_F ? 0.0f : power2((m_run[e] - use) * kLog2e);
          m_run[e] = top;
          m_use[e] = use;
        }
        const float shrink = __int_as_float((int)(127 + exponent - now) << 23);
        exponent = now;
        // (a least-value sum belongs to row g: its factor is with the threads of column g)
        const float even = __shfl_sync(0xffffffffu, alpha[0], g >> 1), odd = __shfl_sync(0xffffffffu, alpha[1], g >> 1);
        const float mine_alpha = ((g & 1) ? odd : even) * shrink;
        alpha[0] *= shrink;
        alpha[1] *= shrink;
        l_run[0] *= alpha[0];
        l_run[1] *= alpha[1];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) least_sum[gr] *= mine_alpha;
#pragma unroll
        for (int i = 0; i < 2 * P; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i >> 1][i & 1][e] *= alpha[e & 1];
      }
      // slots by rows -> rows by slots: row g, slots 2 t, 2 t + 1, 2 t + 8, 2 t + 9 (+ 16), in units of the value scales
      float pw[2][4];
      const float to_units = 23.0f - (float)exponent;
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        float pr[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pr[e] = power2(fmaf(x[side][e] - m_use[e & 1], kLog2e, to_units));
        l_run[0] += pr[0] + pr[2];
        l_run[1] += pr[1] + pr[3];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t c0 = __float_as_uint(pr[2 * e]), c1 = __float_as_uint(pr[2 * e + 1]);
          const uint32_t lo = transposed8x8(__byte_perm(c0, c1, 0x5410)), hi = transposed8x8(__byte_perm(c0, c1, 0x7632));
          pw[side][2 * e] = __uint_as_float(__byte_perm(lo, hi, 0x5410));
          pw[side][2 * e + 1] = __uint_as_float(__byte_perm(lo, hi, 0x7632));
        }
      }
      // -- outputs: channels by slots times slots by rows; a weight is two fp16 numbers --
#pragma unroll
      for (int side = 0; side < 2; ++side) {
        uint32_t vp[4][G];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          lds_words(pairs_at + T::kPairBytes + (uint32_t)((16 * side + 2 * t + (j & 1) + 8 * (j >> 1)) * G * 4), vp[j]);
        if (guard) {
#pragma unroll
          for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int gr = 0; gr < G; ++gr) vp[j][gr] = pw[side][j] == 0.0f ? 0u : vp[j][gr];
        }
        uint32_t high[G][2], low[G][2];
#pragma unroll
        for (int gr = 0; gr < G; ++gr) {
          float ps[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = pair_floats(vp[j][gr]);
            ps[j] = pw[side][j] * f.x;
            least_sum[gr] = fmaf(pw[side][j], fmaf(8.0f, f.x, f.y), least_sum[gr]);
          }
          split_halves(ps[0], ps[1], high[gr][0], low[gr][0]);
          split_halves(ps[2], ps[3], high[gr][1], low[gr][1]);
        }
#pragma unroll
        for (int i = 0; i < P; i += 2) {
          uint32_t words[4], e[4][4];
          load_matrices_transposed(at + T::kNibbleBytes + (matrix_at ^ (uint32_t)(i * 16)) + side * 8 * H, words);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t a = j & 1 ? words[j & 2] >> 8 : words[j & 2], c = j & 1 ? words[(j & 2) + 1] >> 8 : words[(j & 2) + 1];
            e[j][0] = centred_low(a), e[j][1] = centred_high(a), e[j][2] = centred_low(c), e[j][3] = centred_high(c);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int gr = (i + (j >> 1)) / kPer;
            product(o[i + (j >> 1)][j & 1], e[j][0], e[j][1], e[j][2], e[j][3], high[gr][0], high[gr][1]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int gr = (i + (j >> 1)) / kPer;
            product(o[i + (j >> 1)][j & 1], e[j][0], e[j][1], e[j][2], e[j][3], low[gr][0], low[gr][1]);
          }
        }
      }
    }
    cp_async_wait<0>();

    // -- this pair's state: thread (g, t) has channels 4 g .. 4 g + 3 of every piece for rows 2 t and 2 t + 1 --
    const float from_units = __int_as_float((int)(104 + exponent) << 23);  // 2^(exponent - 23)
    const int rows = min(8, rw.rows - chunk * 8);
    float* state = reinterpret_cast<float*>(smem + w * T::kStages * T::kBytes);
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
      for (int i = gr * kPer; i < (gr + 1) * kPer; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (2 * t + e < rows)
            *reinterpret_cast<float4*>(state + (2 * t + e) * T::kRec + i * 32 + g * 4) =
                make_float4((o[i][0][e] + least[e]) * from_units, (o[i][0][2 + e] + least[e]) * from_units, (o[i][1][e] + least[e]) * from_units,
                            (o[i][1][2 + e] + least[e]) * from_units);
    }
    if (g < 2) {
      s_m[w][2 * t + g] = g ? m_run[1] : m_run[0];
      s_l[w][2 * t + g] = (g ? l_run[1] : l_run[0]) * from_units;
    }
    if (lane == 0) {
      s_pair[w] = pair;
      s_rows[w] = rows;
    }
  }

  // -- neighbouring warps of one pair: one record, under the first one's piece --
  __syncthreads();
  for (int first = 0; first < T::kWarps;) {
    const int pair = s_pair[first];
    if (pair < 0) break;  // (pieces are in order: behind a warp without one there is none)
    int end = first + 1;
    while (end < T::kWarps && s_pair[end] == pair) ++end;
    float* rec = p.ws + (size_t)(first_piece + first) * 8 * T::kRec;
    for (int i = threadIdx.x; i < s_rows[first] * (H / 4); i += T::kThreads) {
      const int row = i / (H / 4), d = i % (H / 4) * 4;
      float top = -CUDART_INF_F, sum = 0.0f;
      float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int j = 0; j < T::kWarps; ++j)
        if (j >= first && j < end) top = fmaxf(top, s_m[j][row]);
      const float use = top == -CUDART_INF_F ? 0.0f : top;
#pragma unroll
      for (int j = 0; j < T::kWarps; ++j) {
        if (j >= first && j < end) {
          const float f = power2((s_m[j][row] - use) * kLog2e);
          const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + j * T::kStages * T::kBytes) + row * T::kRec + d);
          acc.x = fmaf(f, v.x, acc.x);
          acc.y = fmaf(f, v.y, acc.y);
          acc.z = fmaf(f, v.z, acc.z);
          acc.w = fmaf(f, v.w, acc.w);
          sum = fmaf(f, s_l[j][row], sum);
        }
      }
      *reinterpret_cast<float4*>(rec + row * T::kRec + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(rec + row * T::kRec + H) = make_float2(top, sum);
    }
    first = end;
  }
}

// Merges the records of one query row, H >> part_log2 channels per CTA (the first n t << part_log2 CTAs of a sequence), or
// adds the weights that 1024 slots of a KV head got to the scores (the others). What it costs are L2 round trips, so the
// records are requested before their weights are known.
constexpr int kMergeThreads = 256;
constexpr int kScoreSlots = 1024;

__device__ __forceinline__ float merge_reduce(float v, bool max, float* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float y = __shfl_xor_sync(0xffffffffu, v, o);
    v = max ? fmaxf(v, y) : v + y;
  }
  if (lane == 0) red[warp] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int i = 1; i < kMergeThreads / 32; ++i) v = max ? fmaxf(v, red[i]) : v + red[i];
  return v;
}

template <int H, bool QF32>
__global__ void __launch_bounds__(kMergeThreads) kv4_merge_kernel(const Kv4Sdpa p, const int ctas, const int part_log2, const float* logits_ws) {
  constexpr int kRec = H + 4, kBatch = 8;
  constexpr size_t kStride = 8 * (size_t)kRec;
  extern __shared__ float merge_w[];  // per record a weight, then per record a sum
  __shared__ float4 s_part[kMergeThreads];
  __shared__ float s_stat[16];
  pdl_launch_dependents();
  const int b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Kv4Rows rw = kv4_rows(p.t, p.n, p.cache.nkv);
  const int per = p.cache.nkv * rw.chunks;
  // what does not depend on the kernel before: it has waited for whatever wrote the lengths
  const Kv4Cut cut = kv4_cut(p, per, ctas, kv4_warps(H), lane);
  const int length = kv4_length(p, b), pieces = cut.pieces_of(length), below = count_pieces(p, per, cut, lane, b);
  // Records of a pair: under its first piece, and under the first piece of every further CTA.
  struct Records {
    const float* base;  // of piece 0
    int first, cta, count;
  };
  auto records = [&](int in_b) {
    const int first = below + in_b * pieces;
    if (pieces == 0) return Records{p.ws, 0, 0, 0};
    const int cta = cut.owner(first);
    return Records{p.ws, first, cta, cut.owner(first + pieces - 1) - cta + 1};
  };
  auto record_at = [&](const Records& r, int j) { return r.base + (j == 0 ? r.first : cut.begin(r.cta + j)) * kStride; };
  if ((int)blockIdx.x < (p.n * p.t) << part_log2) {
    const int row = blockIdx.x >> part_log2, part = blockIdx.x & ((1 << part_log2) - 1);
    const int i = row / p.n, head = row % p.n, kvh = head / rw.group, r = i * rw.group + head % rw.group;
    const int quads = (H / 4) >> part_log2, groups = kMergeThreads / quads;
    const int quad = tid % quads, grp = tid / quads, channel = 4 * (part * quads + quad);
    const Records rec = records(kvh * rw.chunks + r / 8);
    const int count = rec.count, in_rec = (r % 8) * kRec;
    pdl_wait();
    float4 first[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int c = grp + j * groups;
      first[j] = c < count ? __ldcg(reinterpret_cast<const float4*>(record_at(rec, c) + in_rec + channel)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    float* sums = merge_w + ctas;
    float top = -CUDART_INF_F, l = 0.0f;
    for (int c = tid; c < count; c += kMergeThreads) {
      const float2 v = __ldcg(reinterpret_cast<const float2*>(record_at(rec, c) + in_rec + H));
      merge_w[c] = v.x;
      sums[c] = v.y;
      top = fmaxf(top, v.x);
    }
    top = merge_reduce(top, true, s_stat);
    top = top == -CUDART_INF_F ? 0.0f : top;
    for (int c = tid; c < count; c += kMergeThreads) {
      const float f = exp2f((merge_w[c] - top) * kLog2e);
      merge_w[c] = f;
      l += f * sums[c];
    }
    l = merge_reduce(l, false, s_stat + 8);  // (its barrier also publishes the weights)
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int c0 = grp; c0 < count; c0 += kBatch * groups) {
      if (c0 > grp) {
#pragma unroll
        for (int j = 0; j < kBatch; ++j)
          if (c0 + j * groups < count) first[j] = __ldcg(reinterpret_cast<const float4*>(record_at(rec, c0 + j * groups) + in_rec + channel));
      }
#pragma unroll
      for (int j = 0; j < kBatch; ++j) {
        if (c0 + j * groups < count) {
          const float f = merge_w[c0 + j * groups];
          acc.x = fmaf(f, first[j].x, acc.x);
          acc.y = fmaf(f, first[j].y, acc.y);
          acc.z = fmaf(f, first[j].z, acc.z);
          acc.w = fmaf(f, first[j].w, acc.w);
        }
      }
    }
    s_part[tid] = acc;
    __syncthreads();
    if (grp > 0) return;
#pragma unroll 4
    for (int j = 1; j < groups; ++j) {
      const float4 v = s_part[j * quads + quad];
      acc.x += v.x;
      acc.y += v.y;
      acc.z += v.z;
      acc.w += v.w;
    }
    if (l == 0.0f) {
      acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // no slot
    } else {
      acc = make_float4(acc.x / l, acc.y / l, acc.z / l, acc.w / l);
    }
    const size_t at = (((size_t)b * p.t + i) * p.n + head) * H + channel;
    if constexpr (QF32) {
      float* o = static_cast<float*>(p.out) + at;
      o[0] = acc.x, o[1] = acc.y, o[2] = acc.z, o[3] = acc.w;
    } else {
      __half* o = static_cast<__half*>(p.out) + at;
      o[0] = __float2half_rn(acc.x), o[1] = __float2half_rn(acc.y), o[2] = __float2half_rn(acc.z), o[3] = __float2half_rn(acc.w);
    }
    return;
  }
  const int ranges = (p.cache.s + kScoreSlots - 1) / kScoreSlots;
  const int at = blockIdx.x - ((p.n * p.t) << part_log2), kvh = at / ranges, slot0 = at % ranges * kScoreSlots;
  pdl_wait();
  if (slot0 >= length) return;
  const size_t pitch = (size_t)tiles_of(p.cache.s) * kSlots * 8;
  float sums[kScoreSlots / kMergeThreads];
#pragma unroll
  for (int j = 0; j < kScoreSlots / kMergeThreads; ++j) sums[j] = 0.0f;
  for (int c = 0; c < rw.chunks; ++c) {
    const int in_b = kvh * rw.chunks + c, rows = min(8, rw.rows - 8 * c);
    const Records rec = records(in_b);
    const int in_rec = warp * kRec + H;
    __syncthreads();
    if (warp < rows) {
      float top = -CUDART_INF_F, l = 0.0f;
      for (int j = lane; j < rec.count; j += 32) top = fmaxf(top, __ldcg(record_at(rec, j) + in_rec));
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      top = top == -CUDART_INF_F ? 0.0f : top;
      for (int j = lane; j < rec.count; j += 32) {
        const float2 v = __ldcg(reinterpret_cast<const float2*>(record_at(rec, j) + in_rec));
        l += exp2f((v.x - top) * kLog2e) * v.y;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
      if (lane == 0) {
        s_stat[warp] = top;
        s_stat[8 + warp] = l == 0.0f ? 0.0f : 1.0f / l;
      }
    } else if (lane == 0) {
      s_stat[warp] = 0.0f;
      s_stat[8 + warp] = 0.0f;
    }
    __syncthreads();
    const float* logits = logits_ws + ((size_t)b * per + in_b) * pitch;
#pragma unroll
    for (int j = 0; j < kScoreSlots / kMergeThreads; ++j) {
      const int slot = slot0 + threadIdx.x + j * kMergeThreads;
      if (slot < length) {
        const float4 x = __ldcg(reinterpret_cast<const float4*>(logits + (size_t)slot * 8)), y = __ldcg(reinterpret_cast<const float4*>(logits + (size_t)slot * 8) + 1);
        const float v[8] = {x.x, x.y, x.z, x.w, y.x, y.y, y.z, y.w};
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < rows) sums[j] = fmaf(exp2f((v[e] - s_stat[e]) * kLog2e), s_stat[8 + e], sums[j]);
      }
    }
  }
  float* scores = p.scores + ((size_t)b * p.cache.nkv + kvh) * p.cache.s;
#pragma unroll
  for (int j = 0; j < kScoreSlots / kMergeThreads; ++j) {
    const int slot = slot0 + threadIdx.x + j * kMergeThreads;
    if (slot < length) scores[slot] += sums[j];
  }
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
  return (h == 64 || h == 128 || h == 256) && pairs * tiles_of(s) <= INT32_MAX / 2 && pairs <= (1 << 19) && tiles_of(s) < (1 << 22) &&
         4ll * n * t + (long long)nkv * ((s + kScoreSlots - 1) / kScoreSlots) <= INT32_MAX;
}

template <int H, int BLOCK, bool QF32>
cudaError_t launch_tensor(const Kv4Sdpa& p, cudaStream_t s) {
  using T = Kv4Tile<H, BLOCK>;
  const long long pairs = (long long)p.cache.b * p.cache.nkv * kv4_rows(p.t, p.n, p.cache.nkv).chunks;
  const int ctas = kv4_ctas(pairs, p.cache.s, H);
  float* logits = p.scores ? p.ws + kv4_records_floats((long long)ctas * T::kWarps, H) : nullptr;
  static bool done[64] = {false};
  int device = 0;
  cudaGetDevice(&device);
  if (device < 0 || device >= 64) device = 0;
  if (!done[device]) {
    const cudaError_t e = cudaFuncSetAttribute(kv4_sdpa_kernel<H, BLOCK, QF32>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::kSmem);
    if (e != cudaSuccess) return e;
    done[device] = true;
  }
  const cudaError_t e = launch_chained(kv4_sdpa_kernel<H, BLOCK, QF32>, dim3(ctas), dim3(T::kThreads), (size_t)T::kSmem, s, p, logits);
  if (e != cudaSuccess) return e;
  const int scores = p.scores ? p.cache.nkv * ((p.cache.s + kScoreSlots - 1) / kScoreSlots) : 0;
  // few rows are cut by channels too: their records are many
  int part_log2 = 0;
  while (part_log2 < 2 && ((long long)p.cache.b * p.n * p.t << part_log2) < device_sm_count()) ++part_log2;
  return launch_chained(kv4_merge_kernel<H, QF32>, dim3(((p.n * p.t) << part_log2) + scores, p.cache.b), dim3(kMergeThreads),
                        2 * sizeof(float) * (size_t)ctas, s, p, ctas, part_log2, (const float*)logits);
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
  const size_t any = 2 * rows + rows * s;  // (also what queries off a 16-byte boundary need)
  if (!kv4_tensor_shape(b, t, n, nkv, h, s)) return any * sizeof(float);
  const long long pairs = (long long)b * nkv * kv4_rows(t, n, nkv).chunks;
  const size_t tensor = kv4_records_floats((long long)kv4_ctas(pairs, s, h) * kv4_warps(h), h) +
                        (scores ? (size_t)pairs * tiles_of(s) * kSlots * 8 : 0);
  return (any > tensor ? any : tensor) * sizeof(float);
}

cudaError_t launch_kv4_sdpa(const Kv4Sdpa& p, cudaStream_t s) {
  const Kv4Cache& c = p.cache;
  if (!kv4_tensor_shape(c.b, p.t, p.n, c.nkv, c.h, c.s) || (reinterpret_cast<uintptr_t>(p.q) & 15) != 0) return launch_rows(p, s);
  return c.h == 256 ? launch_tensor_block<256>(p, s) : c.h == 128 ? launch_tensor_block<128>(p, s) : launch_tensor_block<64>(p, s);
}

}  // namespace b200
