// Cross attention: queries of one sequence over the keys and values of another length.
//
//   o = softmax(scale q k^T + bias) v,   q [B, Sq, H, D], k and v [B, Skv, Hkv, D], Hkv | H
//
// bias is per key (a boolean or additive mask, lengths of padded sequences); -inf excludes a key,
// whatever stands in its k and v, and a row without keys is 0. Scores, the running maximum and the
// sum of the softmax are fp32; logits are kept in base 2 (scale * log2 e folded into one factor).
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>
#include <type_traits>

#include "../../include/slimdit_b200.h"
#include "slim_kernels.h"
#include "slim_ptx.cuh"

namespace slim {
namespace xattn {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int MAX_DIM = 128;
constexpr int KEY_TILE = 128;

// Which keys take part. A boolean mask and lengths are read by the attention kernel itself; an additive
// mask goes through bias_kernel first (then lengths are in n_keys, and mask and lengths are null).
struct Keys {
  const uint8_t* mask;        // boolean mask or null
  int64_t mask_b, mask_k;
  const void* lengths;        // [batch] or null
  int lengths64;
  const float* bias;          // [batch, bias_pitch] base-2 bias per key, or null
  int64_t bias_pitch;
  const int* n_keys;          // [batch] keys in use (with bias), or null
};

struct Params {
  slim_view q, k, v, out;
  int64_t batch, q_len, kv_len;
  int heads, kv_heads, dim;
  float scale2;               // scale * log2 e
  Keys keys;
};

__device__ __forceinline__ int64_t clamp_length(const void* lengths, int lengths64, int64_t b, int64_t kv_len) {
  const int64_t l = lengths64 ? static_cast<const int64_t*>(lengths)[b] : static_cast<const int32_t*>(lengths)[b];
  return l < 0 ? 0 : l < kv_len ? l : kv_len;
}

// ---------------------------------------------------------------- additive mask -> base-2 bias per key
__device__ __forceinline__ float mask_value(const void* mask, int type, int64_t i) {
  if (type == kF32) return static_cast<const float*>(mask)[i];
  if (type == kBF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(mask)[i]);
  return __half2float(static_cast<const __half*>(mask)[i]);
}

// One block per sequence: bias[b, i] = (mask[b, i] - max over the sequence) * log2 e, -inf for excluded
// keys and the padding of the row; n_keys[b] = 1 + the last key not excluded. A softmax does not change
// under the shift, which keeps rows whose keys all carry the type's lowest value apart from rows
// without keys: a finite bias stays finite.
__global__ void __launch_bounds__(1024) bias_kernel(const void* __restrict__ mask, int type, int64_t stride_b,
                                                    int64_t stride_k, const void* __restrict__ lengths,
                                                    int lengths64, int64_t kv_len, int64_t pitch,
                                                    float* __restrict__ bias, int* __restrict__ n_keys) {
  __shared__ float s_max[32];
  __shared__ int s_last[32];
  const int64_t b = blockIdx.x;
  const int64_t len = lengths != nullptr ? clamp_length(lengths, lengths64, b, kv_len) : kv_len;
  float top = -INFINITY;
  int last = 0;
  for (int64_t i = threadIdx.x; i < len; i += blockDim.x) {
    const float m = mask_value(mask, type, b * stride_b + i * stride_k);
    if (m != -INFINITY) {
      top = fmaxf(top, m);
      last = static_cast<int>(i) + 1;
    }
  }
  for (int o = 16; o >= 1; o >>= 1) {
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
  }
  if ((threadIdx.x & 31) == 0) {
    s_max[threadIdx.x >> 5] = top;
    s_last[threadIdx.x >> 5] = last;
  }
  __syncthreads();
  top = -INFINITY;
  last = 0;
  for (int w = 0; w < static_cast<int>(blockDim.x >> 5); ++w) {
    top = fmaxf(top, s_max[w]);
    last = max(last, s_last[w]);
  }
  if (threadIdx.x == 0) n_keys[b] = last;
  for (int64_t i = threadIdx.x; i < pitch; i += blockDim.x) {
    float y = -INFINITY;
    if (i < len) {
      const float m = mask_value(mask, type, b * stride_b + i * stride_k);
      if (m != -INFINITY) {
        y = (m - top) * kLog2e;
        if (y == -INFINITY) y = -FLT_MAX;
      }
    }
    bias[b * pitch + i] = y;
  }
}

// ---------------------------------------------------------------- shared by both kernels
constexpr int BM = 128, BN = KEY_TILE;  // rows and keys of a tile
constexpr float GROWTH = 8.0f;          // base-2 growth of a row's maximum that is let stand
// What is kept as a row's maximum, the m of its weights 2^(y - m), is less than the true one by HEADROOM. The
// weights of the largest keys are then up to 2^(HEADROOM + GROWTH), which is 2^15 in fp16 (largest 65504), and the
// smallest that fp16 can hold is 2^-24 / 2^HEADROOM of the largest: with m the maximum itself, a tail of 10^5 keys that
// are 2^-25 of one dominant key each was lost from the second product while the sum still had it. bf16 has the
// exponents of fp32 and needs none. Sums and output carry the same factor 2^HEADROOM, pieces too, and it divides out.
template <typename T>
constexpr float HEADROOM = std::is_same<T, __half>::value ? 7.0f : 0.0f;
constexpr int SOFTMAX_WARPS = 16;
constexpr int WARPS = SOFTMAX_WARPS + 4, THREADS = 32 * WARPS;
// Registers: 96 a thread at launch, of which the softmax warps take 104 and the last warpgroup leaves
// all but 64: 4 x 104 + 64 = 5 x 96.
constexpr int REGS = 96, REGS_SOFTMAX = 104, REGS_OTHER = 64;
static_assert(4 * REGS_SOFTMAX + REGS_OTHER <= 5 * REGS, "the register shares exceed the launch's allocation");

// Shared-memory tiles of 128 rows: DP / 64 blocks of 64 elements (128 bytes) a row, 128-byte swizzle.
template <int DP>
struct Tile {
  static constexpr int BLOCKS = DP / 64;
  static constexpr int BLOCK_BYTES = 128 * 128;
  static constexpr int BYTES = BLOCKS * BLOCK_BYTES;
};

// A row is a (token, query head of the group) pair, the head running fastest, so that the heads that share
// keys share their loads; `tokens` tokens make a tile of up to 128 rows.
struct TileParams {
  slim_view out;
  int64_t q_len, kv_len;
  int kv_heads, dim;
  int group, tokens;          // query heads per key head, tokens per row tile
  uint32_t group_inv;         // ceil(2^16 / group): row / group = row * group_inv >> 16 for rows below 128
  int kb, kh, vb, vh;         // 0 for a k / v that is the same for every sequence / head
  float scale2;
  Keys keys;
  int items, per_head;        // items in all, and of one (sequence, key head)
  int splits, per;            // split: pieces of the keys of a row tile, key tiles of each
  int rows;                   // split: rows of a tile that exist
  float* partial;             // split: results of the pieces
};

__device__ __forceinline__ int token_of(const TileParams& p, int row) { return row * p.group_inv >> 16; }

template <bool BIAS>
__device__ __forceinline__ int keys_of(const TileParams& p, int b) {
  if (BIAS) return p.keys.n_keys[b];
  return static_cast<int>(p.keys.lengths != nullptr ? clamp_length(p.keys.lengths, p.keys.lengths64, b, p.kv_len) : p.kv_len);
}

// TMA loads of a tile of 128 keys (rows past the end come as zeros).
template <int DP>
__device__ __forceinline__ void load_keys(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int head, int key_tile, int b) {
  for (int c = 0; c < Tile<DP>::BLOCKS; ++c)
    tma_load_4d(dst + c * Tile<DP>::BLOCK_BYTES, map, bar, c * 64, head, key_tile * BN, b);
}

// S[tmem] = Q K^T and O[tmem] (+)= P[tmem] V of one tile, by one thread. V is read as it lies (keys x head
// elements): an MN-major operand.
template <int DP, bool BF16>
__device__ __forceinline__ void mma_scores(uint32_t s, uint64_t q_desc, uint64_t k_desc) {
  constexpr uint32_t IDESC = idesc_f16(BM, BN, BF16, false);
#pragma unroll
  for (int k = 0; k < DP / 16; ++k) {
    const uint32_t off = (k >> 2) * Tile<DP>::BLOCK_BYTES + (k & 3) * 32;
    mma_f16(s, smem_desc_at(q_desc, off), smem_desc_at(k_desc, off), IDESC, k != 0);
  }
}
template <int DP, bool BF16>
__device__ __forceinline__ void mma_values(uint32_t o, uint32_t weights, uint64_t v_desc, bool accumulate) {
  constexpr uint32_t IDESC = idesc_f16(BM, DP, BF16, true);
  const uint32_t more = accumulate;
#pragma unroll
  for (int k = 0; k < BN / 16; ++k)
    mma_f16_ta(o, weights + k * 8, smem_desc_at(v_desc, k * 2048), IDESC, k != 0 ? 1u : more);
}

__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Logits so large that their steps in fp32 come near 1. The weights' exponent y sc - m is formed in one rounding, while
// m = y sc of the largest key was rounded by itself: its weight is 2^0 only up to half a step of m, which from 2^30 on
// leaves the range of fp32. There the logits are rounded before m is taken off, as by a product and a subtraction.
constexpr float LARGE = 4194304.0f;  // 2^22: half a step is a quarter
template <int N>
__device__ __forceinline__ float scale_if_large(float (&y)[N], float peak, bool real, float& sc) {
  const bool large = real && fabsf(peak) * sc > LARGE && peak != -INFINITY;
  if (__any_sync(0xffffffffu, large)) {
    const float factor = large ? sc : 1.0f;  // this thread's row goes by its own scores
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] *= factor;
    peak *= factor;
    if (large) sc = 1.0f;
  }
  return peak;
}

// Base-2 weights of 32 keys: w = 2^(y sc + off), summed in fp32, packed to the type of v: both operands of a
// 16-bit MMA have one type, and weights of 32 bits would take a tf32 copy of v, or a second product for what the
// rounding leaves. It costs half a step of a weight, 2^-9 (bf16) or 2^-12 (fp16) of it, independent from key to key:
// the error against 64 bits is 2.2e-3 instead of the 1.7e-3 of the result's own rounding in bf16, 2.4e-4 instead of
// 2.1e-4 in fp16 (2-norm, normal inputs).
template <typename T>
__device__ __forceinline__ float2 weights(const float* y, float sc, float off, uint32_t (&w)[16]) {
  const float2 sc2 = make_float2(sc, sc), off2 = make_float2(off, off);
  float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float2 x = fma2(make_float2(y[2 * e], y[2 * e + 1]), sc2, off2);
    const float2 g = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    sum = add2(sum, g);
    w[e] = pack2<T>(g.x, g.y);
  }
  return sum;
}

template <int N>
__device__ __forceinline__ float max_of(const float* y) {
  float mx[4] = {y[0], y[1], y[2], y[3]};
#pragma unroll
  for (int e = 4; e < N - 4; e += 8) {
#pragma unroll
    for (int u = 0; u < 4; ++u) mx[u] = fmax3(mx[u], y[e + u], y[e + 4 + u]);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) mx[u] = fmaxf(mx[u], y[N - 4 + u]);
  return fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]);
}

// The largest score of some keys as a row's maximum is kept, and whether it has outgrown the maximum m in use. The
// latter is the exponent of its weight, rounded as there: no weight passes 2^(HEADROOM + GROWTH) even where the
// logits are so large that their own steps count.
template <typename T>
__device__ __forceinline__ float as_top(float peak, float sc) { return fmaf(peak, sc, -HEADROOM<T>); }
template <typename T>
__device__ __forceinline__ bool outgrown(float peak, float sc, float m) {
  return fmaf(peak, sc, -m) > HEADROOM<T> + GROWTH;
}

// Which of the keys key0 + [first, first + 32 W) take part, one bit each, and whether key0 + row does. With
// a bias only what lies behind the last key is left out here.
template <bool BIAS, int W>
__device__ __forceinline__ bool key_bits(const TileParams& p, int b, int key0, int left, int first, int row, int lane,
                                         uint32_t (&bits)[W]) {
  bool used = row < left;
#pragma unroll
  for (int w = 0; w < W; ++w) {
    const int n = left - first - 32 * w;
    bits[w] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
  }
  if (BIAS) {
    used = used && __ldg(p.keys.bias + b * p.keys.bias_pitch + key0 + row) != -INFINITY;
  } else if (p.keys.mask != nullptr) {
    const uint8_t* mask = p.keys.mask + b * p.keys.mask_b + key0 * p.keys.mask_k;
    used = used && __ldg(mask + row * p.keys.mask_k) != 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int i = first + 32 * w + lane;
      bits[w] = __ballot_sync(0xffffffffu, i < left && __ldg(mask + i * p.keys.mask_k) != 0);
    }
  }
  return used;
}

// Scores of N keys from key first of a tile on: -inf where the bit is not set, or (BIAS) s scale2 + bias.
template <bool BIAS, int N>
__device__ __forceinline__ void mask_scores(const TileParams& p, int b, int key0, int first, const uint32_t (&bits)[N / 32],
                                            float (&y)[N]) {
  if (BIAS) {
    const float4* bias4 = reinterpret_cast<const float4*>(p.keys.bias + b * p.keys.bias_pitch + key0 + first);
#pragma unroll
    for (int e = 0; e < N; e += 4) {
      // an excluded key's score may be NaN; behind the last key the bias row may have ended
      const float4 a = (bits[e / 32] >> (e & 31)) & 1 ? __ldg(bias4 + e / 4)
                                                      : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
      y[e + 0] = a.x == -INFINITY ? -INFINITY : fmaf(y[e + 0], p.scale2, a.x);
      y[e + 1] = a.y == -INFINITY ? -INFINITY : fmaf(y[e + 1], p.scale2, a.y);
      y[e + 2] = a.z == -INFINITY ? -INFINITY : fmaf(y[e + 2], p.scale2, a.z);
      y[e + 3] = a.w == -INFINITY ? -INFINITY : fmaf(y[e + 3], p.scale2, a.w);
    }
    return;
  }
  uint32_t all = bits[0];
#pragma unroll
  for (int w = 1; w < N / 32; ++w) all &= bits[w];
  if (all != 0xffffffffu) {
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = (bits[e / 32] >> (e & 31)) & 1 ? y[e] : -INFINITY;
  }
}

// O *= alpha for COLS columns of this thread's row.
template <int COLS>
__device__ __forceinline__ void rescale(uint32_t t_o, float alpha) {
#pragma unroll 1
  for (int c = 0; c < COLS; c += 16) {
    uint32_t o[16];
    tmem_ld_32x32b_x16(t_o + c, o);
    tmem_ld_wait();
    reg_dep16(o);
#pragma unroll
    for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
    tmem_st_32x32b_x16(t_o + c, o);
  }
}

}  // namespace xattn
}  // namespace slim
