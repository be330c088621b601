// Cross attention: queries of one sequence over the keys and values of another length.
//
//   o = softmax(scale q k^T + bias) v,   q [B, Sq, H, D], k and v [B, Skv, Hkv, D], Hkv | H
//
// bias is per key (a boolean or additive mask, lengths of padded sequences); -inf excludes a key,
// whatever stands in its k and v, and a row without keys is 0. Scores, the running maximum and the
// sum of the softmax are fp32; logits are kept in base 2 (scale * log2 e folded into one factor).
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

enum MaskType : int { kMaskF32 = kF32, kMaskBF16 = kBF16, kMaskF16 = kF16, kMaskBool = 3, kMaskNone = -1 };

struct Params {
  slim_view q, k, v, out;
  int64_t batch, q_len, kv_len;
  int heads, kv_heads, dim;
  float scale2;               // scale * log2 e
  const float* bias;          // [batch, bias_pitch] base-2 bias per key, or null
  int64_t bias_pitch;
  const int* n_keys;          // [batch] keys in use (with bias), or null
};

// ---------------------------------------------------------------- mask -> base-2 bias per key
__device__ __forceinline__ float mask_value(const void* mask, int type, int64_t i) {
  switch (type) {
    case kMaskF32: return static_cast<const float*>(mask)[i];
    case kMaskBF16: return __bfloat162float(static_cast<const __nv_bfloat16*>(mask)[i]);
    case kMaskF16: return __half2float(static_cast<const __half*>(mask)[i]);
    case kMaskBool: return static_cast<const uint8_t*>(mask)[i] ? 0.0f : -INFINITY;
    default: return 0.0f;
  }
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
  int64_t len = kv_len;
  if (lengths != nullptr) {
    const int64_t l = lengths64 ? static_cast<const int64_t*>(lengths)[b] : static_cast<const int32_t*>(lengths)[b];
    len = l < 0 ? 0 : l < kv_len ? l : kv_len;
  }
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

// ---------------------------------------------------------------- tile kernel
// One CTA takes 256 rows of one (sequence, key head): two tiles of 128 rows, a row being a (token,
// query head of the group) pair with the head running fastest, so the heads that share keys share
// their loads. 10 warps:
//   warps 0..3, 4..7  softmax of tile 0 / 1, one row a thread: the scores are read from TMEM twice
//                     (row maximum, then weights 2^(s scale2 + bias - m)), the weights go back packed
//                     to 16 bits over the scores they came from, where the second product reads them.
//                     O is rescaled only when a maximum grows by more than 2^8 over the one in use
//                     (the weights stay below 2^8, sums and O are fp32), which is rare after the
//                     first tile.
//   warp 8            TMA: both Q tiles, then K_0 V_0 K_1 V_1 ... through one ring of tiles
//   warp 9            TMEM, and the MMAs: S_t = Q_t K_j^T, then per tile O_t += P_t V_j followed at
//                     once by S_t = Q_t K_{j+1}^T: while one tile is in the softmax the tensor cores
//                     work on the other.
// V is read as it lies (keys x head elements): an MN-major operand. Excluded keys have weight 0; their
// rows of V are cleared in shared memory, as 0 * NaN is not 0.
namespace tile {
constexpr int BM = 128, BN = KEY_TILE;
constexpr int WARPS = 10, THREADS = 32 * WARPS;
__device__ __forceinline__ constexpr uint32_t col_s(int t) { return t * 128u; }         // scores, then weights
__device__ __forceinline__ constexpr uint32_t col_o(int t) { return 256u + t * 128u; }  // output accumulator
constexpr float GROWTH = 8.0f;  // base-2 growth of a maximum that is let stand

template <int DP>
struct Layout {
  static constexpr int BLOCKS = DP / 64;               // 64-element (128-byte) column blocks of a tile
  static constexpr int BLOCK_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = BLOCKS * BLOCK_BYTES;
  static constexpr int STAGES = DP == 128 ? 5 : 8;
  static constexpr int OFF_KV = 2 * TILE_BYTES;
  static constexpr int OFF_SH = OFF_KV + STAGES * TILE_BYTES;
};

template <int STAGES>
struct Shared {
  uint64_t q_full[2];
  uint64_t full[STAGES], empty[STAGES];
  uint64_t s_full[2], p_full[2], o_full[2];
  uint64_t drain;
  uint32_t tmem_base;
  volatile int abort;
};

template <int DP>
constexpr size_t smem_bytes() {
  return 1024 + Layout<DP>::OFF_SH + sizeof(Shared<Layout<DP>::STAGES>);
}

struct TileParams {
  int64_t q_len, kv_len;
  int group, tokens;          // query heads per key head, tokens per 128-row tile
  int kb, kh, vb, vh;         // 0 for a k / v that is the same for every sequence / head
  float scale2;
  const float* bias;
  int64_t bias_pitch;
  const int* n_keys;
};

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

// 32 scores of one row from TMEM as base-2 logits without the row's offset: s, or s scale2 + bias.
template <bool MASK>
__device__ __forceinline__ void load_scores(uint32_t taddr, int c, const float4* bias4, float scale2, int valid,
                                            float (&y)[32]) {
  uint32_t r[32];
  tmem_ld_32x32b_x32(taddr + c, r);
  tmem_ld_wait();
  reg_dep32(r);
#pragma unroll
  for (int e = 0; e < 32; ++e) y[e] = __uint_as_float(r[e]);
  if (MASK) {
#pragma unroll
    for (int e = 0; e < 32; e += 4) {
      const float4 b = __ldg(bias4 + (c + e) / 4);
      // an excluded key's score may be NaN
      y[e + 0] = b.x == -INFINITY ? -INFINITY : fmaf(y[e + 0], scale2, b.x);
      y[e + 1] = b.y == -INFINITY ? -INFINITY : fmaf(y[e + 1], scale2, b.y);
      y[e + 2] = b.z == -INFINITY ? -INFINITY : fmaf(y[e + 2], scale2, b.z);
      y[e + 3] = b.w == -INFINITY ? -INFINITY : fmaf(y[e + 3], scale2, b.w);
    }
  } else if (valid < BN) {
#pragma unroll
    for (int e = 0; e < 32; ++e) y[e] = c + e < valid ? y[e] : -INFINITY;
  }
}

template <typename T, int DP, bool MASK>
__global__ void __launch_bounds__(THREADS, 1)
tile_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
            const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to, const TileParams p) {
  using L = Layout<DP>;
  using Sh = Shared<L::STAGES>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_QK = idesc_f16(BM, BN, BF16, false);
  constexpr uint32_t IDESC_PV = idesc_f16(BM, DP, BF16, true);
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw_addr = smem_u32(smem_raw);
  uint8_t* smem = smem_raw + (((raw_addr + 1023) & ~1023u) - raw_addr);
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + L::OFF_KV;
  Sh& sh = *reinterpret_cast<Sh*>(smem + L::OFF_SH);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.z, hk = blockIdx.y;
  const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * 2 * p.tokens;
  const int tiles = tok0 + p.tokens < p.q_len ? 2 : 1;
  const int64_t keys = MASK ? p.n_keys[b] : p.kv_len;
  const int nk = static_cast<int>((keys + BN - 1) / BN);

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh.q_full[t], 1);
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.p_full[t], BM);
      mbar_init(&sh.o_full[t], 1);
    }
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    mbar_init(&sh.drain, 1);
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;

  if (warp == 8) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && nk > 0) {
      const uint32_t q_bytes = static_cast<uint32_t>(L::BLOCKS * 128 * p.group * p.tokens);
      for (int t = 0; t < tiles; ++t) {
        mbar_arrive_expect_tx(&sh.q_full[t], q_bytes);
        for (int c = 0; c < L::BLOCKS; ++c)
          tma_load_4d(sQ + t * L::TILE_BYTES + c * L::BLOCK_BYTES, &tq, &sh.q_full[t], c * 64, hk * p.group,
                      static_cast<int32_t>(tok0 + t * p.tokens), b);
      }
      uint32_t issued = 0, last_parity = 0;
      for (int i = 0; i < 2 * nk && !sh.abort; ++i) {  // K_0 V_0 K_1 V_1 ...
        const int s = i % L::STAGES;
        const uint32_t ph = (i / L::STAGES) & 1;
        if (!mbar_wait(&sh.empty[s], ph ^ 1, kErrWaitTimeoutProducer)) {
          sh.abort = 1;
          break;
        }
        const bool is_v = i & 1;
        mbar_arrive_expect_tx(&sh.full[s], L::TILE_BYTES);
        for (int c = 0; c < L::BLOCKS; ++c)
          tma_load_4d(sKV + s * L::TILE_BYTES + c * L::BLOCK_BYTES, is_v ? &tv : &tk, &sh.full[s], c * 64,
                      hk * (is_v ? p.vh : p.kh), (i >> 1) * BN, b * (is_v ? p.vb : p.kb));
        issued |= 1u << s;
        last_parity = (last_parity & ~(1u << s)) | (ph << s);
      }
      // every load issued by this thread lands before the CTA may exit
      for (int t = 0; t < tiles; ++t) mbar_wait(&sh.q_full[t], 0, kErrWaitTimeoutDrain);
      for (int s = 0; s < L::STAGES; ++s)
        if (issued & (1u << s)) mbar_wait(&sh.full[s], (last_parity >> s) & 1, kErrWaitTimeoutDrain);
    }
  } else if (warp == 9) {
    // ------------------------------------------------------------ MMA issue
    if (lane == 0 && nk > 0) {
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        ok = ok && mbar_wait(bar, parity, kErrWaitTimeoutMma) && !sh.abort;
        return ok;
      };
      auto full = [&](int i) { return wait(&sh.full[i % L::STAGES], (i / L::STAGES) & 1); };
      auto qk = [&](int t, int i) {
        const uint32_t qa = smem_u32(sQ + t * L::TILE_BYTES);
        const uint32_t ka = smem_u32(sKV + (i % L::STAGES) * L::TILE_BYTES);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k) {
          const uint32_t off = (k >> 2) * L::BLOCK_BYTES + (k & 3) * 32;
          mma_f16(tmem + col_s(t), smem_desc_sw128(qa + off), smem_desc_sw128(ka + off), IDESC_QK, k != 0);
        }
        mma_commit(&sh.s_full[t]);
        if (t == tiles - 1) mma_commit(&sh.empty[i % L::STAGES]);
      };
      auto pv = [&](int t, int i, bool first) {
        const uint32_t va = smem_u32(sKV + (i % L::STAGES) * L::TILE_BYTES);
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          mma_f16_ta(tmem + col_o(t), tmem + col_s(t) + k * 8, smem_desc_mn_sw128(va + k * 2048, L::BLOCK_BYTES),
                     IDESC_PV, !(first && k == 0));
        mma_commit(&sh.o_full[t]);
        if (t == tiles - 1) mma_commit(&sh.empty[i % L::STAGES]);
      };
      if (full(0)) {
        for (int t = 0; t < tiles && wait(&sh.q_full[t], 0); ++t) {
          tc_fence_after();
          qk(t, 0);
        }
      }
      for (int j = 0; ok && j < nk; ++j) {
        for (int t = 0; t < tiles; ++t) {
          if (t == 0 && !full(2 * j + 1)) break;
          if (!wait(&sh.p_full[t], j & 1)) break;
          tc_fence_after();
          pv(t, 2 * j + 1, j == 0);
          if (j + 1 < nk) {
            if (t == 0 && !full(2 * j + 2)) break;
            tc_fence_after();
            qk(t, 2 * j + 2);
          }
        }
      }
      if (!ok) sh.abort = 1;
      mma_commit(&sh.drain);
      mbar_wait(&sh.drain, 0, kErrWaitTimeoutDrain);
    }
    __syncwarp();
  } else if ((warp >> 2) < tiles) {
    // ------------------------------------------------------------ softmax of one row, output
    const int t = warp >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_s = t_lane + col_s(t), t_o = t_lane + col_o(t);
    const float scale2 = p.scale2;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      bool ok = mbar_wait(bar, parity, kErrWaitTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok) && !sh.abort;
      if (!ok) sh.abort = 1;
      return ok;
    };
    bool good = true;
    float m = -INFINITY;
    float2 l2 = make_float2(0.0f, 0.0f);
    for (int j = 0; j < nk; ++j) {
      const float4* bias4 = MASK ? reinterpret_cast<const float4*>(p.bias + b * p.bias_pitch + static_cast<int64_t>(j) * BN) : nullptr;
      const int64_t left = keys - static_cast<int64_t>(j) * BN;
      const int valid = left < BN ? static_cast<int>(left) : BN;
      if (MASK && t == 0) {
        // tile 0's weights gate the second product of both tiles
        const bool clear = __ldg(reinterpret_cast<const float*>(bias4) + row) == -INFINITY;
        if (__any_sync(0xffffffffu, clear)) {
          const int i = 2 * j + 1;
          if (!(good = wait(&sh.full[i % L::STAGES], (i / L::STAGES) & 1))) break;
          if (clear) {
            uint4* v = reinterpret_cast<uint4*>(sKV + (i % L::STAGES) * L::TILE_BYTES + row * 128);
#pragma unroll
            for (int c = 0; c < L::BLOCKS; ++c)
#pragma unroll
              for (int e = 0; e < 8; ++e) v[c * (L::BLOCK_BYTES / 16) + e] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
      }
      if (!(good = wait(&sh.s_full[t], j & 1))) break;
      tc_fence_after();
      float top = -INFINITY;
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        float y[32];
        load_scores<MASK>(t_s, c, bias4, scale2, valid, y);
        float mx[4] = {y[0], y[1], y[2], y[3]};
#pragma unroll
        for (int e = 4; e < 28; e += 8) {
#pragma unroll
          for (int u = 0; u < 4; ++u) mx[u] = fmax3(mx[u], y[e + u], y[e + 4 + u]);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) mx[u] = fmaxf(mx[u], y[28 + u]);
        top = fmaxf(top, fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]));
      }
      const float m_new = fmaxf(m, MASK ? top : top * scale2);
      if (j == 0) {
        m = m_new;
      } else if (__any_sync(0xffffffffu, m_new > m + GROWTH)) {
        const float alpha = m_new == -INFINITY ? 1.0f : ex2_approx(m - m_new);
        m = m_new;
        l2 = mul2(l2, make_float2(alpha, alpha));
        if (!(good = wait(&sh.o_full[t], (j - 1) & 1))) break;
        tc_fence_after();
#pragma unroll 1
        for (int c = 0; c < DP; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t_o + c, r);
          tmem_ld_wait();
          reg_dep32(r);
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = __float_as_uint(__uint_as_float(r[e]) * alpha);
          tmem_st_32x32b_x32(t_o + c, r);
        }
      }
      const float off = m == -INFINITY ? 0.0f : -m;
      const float2 off2 = make_float2(off, off), sc2 = make_float2(scale2, scale2);
#pragma unroll 1
      for (int c = 0; c < BN; c += 32) {
        float y[32];
        load_scores<MASK>(t_s, c, bias4, scale2, valid, y);
        uint32_t w[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float2 a = make_float2(y[2 * e], y[2 * e + 1]);
          const float2 x = MASK ? add2(a, off2) : fma2(a, sc2, off2);
          const float2 g = make_float2(ex2_approx(x.x), ex2_approx(x.y));
          l2 = add2(l2, g);
          w[e] = pack2<T>(g.x, g.y);
        }
        tmem_st_32x32b_x16(t_s + c / 2, w);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(&sh.p_full[t]);
    }
    // the tile's rows leave through the shared memory of its queries
    uint8_t* stage = sQ + t * L::TILE_BYTES;
    const float l = l2.x + l2.y;
    if (good && nk > 0) {
      good = wait(&sh.o_full[t], (nk - 1) & 1);
      tc_fence_after();
    }
    if (good) {
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll 1
      for (int c = 0; c < DP; c += 32) {
        uint32_t r[32];
        if (nk > 0) {
          tmem_ld_32x32b_x32(t_o + c, r);
          tmem_ld_wait();
          reg_dep32(r);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) r[e] = 0;
        }
        uint8_t* dst = stage + (c >> 6) * L::BLOCK_BYTES + row * 128;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = pack2<T>(__uint_as_float(r[8 * u + 2 * e]) * inv, __uint_as_float(r[8 * u + 2 * e + 1]) * inv);
          const int chunk = ((c & 63) >> 3) + u;
          *reinterpret_cast<uint4*>(dst + ((chunk ^ (row & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
      fence_proxy_async_smem();
    }
    named_barrier(1 + t, BM);  // reached on every path
    if (good && !sh.abort && quarter == 0 && lane == 0) {
      for (int c = 0; c < L::BLOCKS; ++c)
        tma_store_4d(&to, stage + c * L::BLOCK_BYTES, c * 64, hk * p.group, static_cast<int32_t>(tok0 + t * p.tokens), b);
      bulk_commit_group();
      bulk_wait_group<0>();
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// [batch, seq, heads, dim] view of 16-bit elements as a 4-D map with boxes of 64 elements x box_heads x
// box_tokens; dimensions of size 1 or stride 0 become size 1.
static bool make_map(CUtensorMap* map, bool bf16, const slim_view& v, int64_t batch, int64_t seq, int heads, int dim,
                     int box_heads, int box_tokens) {
  PFN_encodeTiledAttn enc = attn_encode_fn();
  if (enc == nullptr) return false;
  const int64_t sizes[3] = {heads, seq, batch}, strides_el[3] = {v.stride_h, v.stride_s, v.stride_b};
  cuuint64_t dims[4] = {static_cast<cuuint64_t>(dim)}, strides[3];
  for (int i = 0; i < 3; ++i) {
    const bool single = sizes[i] == 1 || strides_el[i] == 0;
    dims[i + 1] = single ? 1 : static_cast<cuuint64_t>(sizes[i]);
    strides[i] = single ? 256 : static_cast<cuuint64_t>(strides_el[i]) * 2;
  }
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(box_heads), static_cast<cuuint32_t>(box_tokens), 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return enc(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, v.data, dims, strides,
             box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int DP, bool MASK>
cudaError_t launch(const Params& p, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  const int group = p.heads / p.kv_heads, tokens = BM / group;
  CUtensorMap mq, mk, mv, mo;
  // without keys k and v may be null: their maps are never used
  const slim_view& k = p.kv_len > 0 ? p.k : p.q;
  const slim_view& v = p.kv_len > 0 ? p.v : p.q;
  if (!make_map(&mq, BF16, p.q, p.batch, p.q_len, p.heads, p.dim, group, tokens) ||
      !make_map(&mo, BF16, p.out, p.batch, p.q_len, p.heads, p.dim, group, tokens) ||
      !make_map(&mk, BF16, k, p.batch, p.kv_len > 0 ? p.kv_len : 1, p.kv_len > 0 ? p.kv_heads : 1, p.dim, 1, BN) ||
      !make_map(&mv, BF16, v, p.batch, p.kv_len > 0 ? p.kv_len : 1, p.kv_len > 0 ? p.kv_heads : 1, p.dim, 1, BN))
    return cudaErrorInvalidValue;
  int dev = 0;
  cudaGetDevice(&dev);
  static PerDeviceOnce once;
  const cudaError_t e = once.run(dev, [] {
    return cudaFuncSetAttribute(tile_kernel<T, DP, MASK>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem_bytes<DP>()));
  });
  if (e != cudaSuccess) return e;
  const TileParams tp{p.q_len, p.kv_len, group, tokens, p.k.stride_b != 0, p.k.stride_h != 0, p.v.stride_b != 0,
                      p.v.stride_h != 0, p.scale2, p.bias, p.bias_pitch, p.n_keys};
  const dim3 grid(static_cast<unsigned>((p.q_len + 2 * tokens - 1) / (2 * tokens)), static_cast<unsigned>(p.kv_heads),
                  static_cast<unsigned>(p.batch));
  tile_kernel<T, DP, MASK><<<grid, THREADS, smem_bytes<DP>(), st>>>(mq, mk, mv, mo, tp);
  return cudaGetLastError();
}

template <typename T>
cudaError_t launch(const Params& p, cudaStream_t st) {
  if (p.bias != nullptr) return p.dim > 64 ? launch<T, 128, true>(p, st) : launch<T, 64, true>(p, st);
  return p.dim > 64 ? launch<T, 128, false>(p, st) : launch<T, 64, false>(p, st);
}
}  // namespace tile

struct Workspace {
  int64_t bias, n_keys, total, pitch;
};

static Workspace workspace(int64_t batch, int64_t kv_len, bool masked) {
  Workspace w{};
  w.pitch = (kv_len + KEY_TILE - 1) / KEY_TILE * KEY_TILE;
  if (masked) {
    w.bias = 0;
    w.n_keys = (batch * w.pitch * 4 + 255) / 256 * 256;
    w.total = w.n_keys + (batch * 4 + 255) / 256 * 256;
  }
  return w;
}

static int checks(int64_t batch, int64_t q_len, int64_t kv_len, int heads, int kv_heads, int dim) {
  if (batch < 0 || q_len < 0 || kv_len < 0 || heads <= 0 || kv_heads <= 0)
    return fail(SLIM_ERR_SHAPE, "bad attention shape batch=%lld q_len=%lld kv_len=%lld heads=%d/%d",
                static_cast<long long>(batch), static_cast<long long>(q_len), static_cast<long long>(kv_len), heads, kv_heads);
  if (dim <= 0 || dim > MAX_DIM || dim % 8)
    return fail(SLIM_ERR_SHAPE, "head dim must be a multiple of 8 up to %d, got %d", MAX_DIM, dim);
  if (heads % kv_heads || heads / kv_heads > 128)
    return fail(SLIM_ERR_SHAPE, "%d query heads do not group over %d key heads (at most 128 each)", heads, kv_heads);
  if (batch >= (int64_t{1} << 16) || q_len >= (int64_t{1} << 31) - 256 || kv_len >= (int64_t{1} << 31) - 256 || heads >= (1 << 16))
    return fail(SLIM_ERR_SHAPE, "attention shape too large");
  return SLIM_OK;
}

// Strides that a tensor map takes: 16-byte multiples below 2^40 bytes, and 0 only for the sequences
// and heads of k and v.
static bool view_ok(const slim_view* v, int64_t batch, int64_t seq, int heads, bool shared) {
  auto ok = [](int64_t n, int64_t stride, bool zero) {
    return n == 1 || (stride % 8 == 0 && stride < (int64_t{1} << 39) && (stride > 0 || (zero && stride == 0)));
  };
  return aligned16(v->data) && ok(batch, v->stride_b, shared) && ok(seq, v->stride_s, false) && ok(heads, v->stride_h, shared);
}

}  // namespace xattn
}  // namespace slim

using namespace slim;

extern "C" {

int slim_cross_attn_workspace_bytes(int64_t batch, int64_t q_len, int64_t kv_len, int heads, int kv_heads, int dim,
                                    int masked, uint64_t* bytes) {
  const int rc = xattn::checks(batch, q_len, kv_len, heads, kv_heads, dim);
  if (rc != SLIM_OK) return rc;
  if (bytes == nullptr) return fail(SLIM_ERR_NULL, "bytes is NULL");
  *bytes = static_cast<uint64_t>(xattn::workspace(batch, kv_len, masked != 0).total);
  return SLIM_OK;
}

int slim_cross_attn(const slim_view* q, const slim_view* k, const slim_view* v, const slim_view* out, int dtype,
                    int64_t batch, int64_t q_len, int64_t kv_len, int heads, int kv_heads, int dim, const void* mask,
                    int mask_type, int64_t mask_stride_b, int64_t mask_stride_k, const void* kv_lengths,
                    int lengths_bits, float scale, void* ws, uint64_t workspace_bytes, void* stream) {
  SLIM_NVTX("slim_cross_attn");
  int rc;
  if (dtype != kBF16 && dtype != kF16) return fail(SLIM_ERR_DTYPE, "cross attention takes bf16 or fp16, got dtype code %d", dtype);
  if ((rc = xattn::checks(batch, q_len, kv_len, heads, kv_heads, dim)) != SLIM_OK) return rc;
  if (mask != nullptr && mask_type != kF32 && mask_type != kBF16 && mask_type != kF16 && mask_type != SLIM_MASK_BOOL)
    return fail(SLIM_ERR_DTYPE, "unsupported mask type %d", mask_type);
  if (kv_lengths != nullptr && lengths_bits != 32 && lengths_bits != 64)
    return fail(SLIM_ERR_DTYPE, "lengths must be 32- or 64-bit integers");
  if (!(scale > 0.0f) || !(scale <= FLT_MAX)) return fail(SLIM_ERR_SHAPE, "scale must be positive and finite");
  if (batch == 0 || q_len == 0) return SLIM_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || q->data == nullptr || out->data == nullptr ||
      (kv_len > 0 && (k->data == nullptr || v->data == nullptr)))
    return fail(SLIM_ERR_NULL, "q/k/v/out is NULL");
  if (!xattn::view_ok(q, batch, q_len, heads, false) || !xattn::view_ok(out, batch, q_len, heads, false) ||
      (kv_len > 0 && (!xattn::view_ok(k, batch, kv_len, kv_heads, true) || !xattn::view_ok(v, batch, kv_len, kv_heads, true))))
    return fail(SLIM_ERR_ALIGN, "rows of q/k/v/out must be 16-byte aligned with positive strides (0 for shared k/v)");
  const bool masked = kv_len > 0 && (mask != nullptr || kv_lengths != nullptr);
  const xattn::Workspace w = xattn::workspace(batch, kv_len, masked);
  if (workspace_bytes < static_cast<uint64_t>(w.total))
    return fail(SLIM_ERR_SHAPE, "workspace of %llu bytes is smaller than the %lld needed",
                static_cast<unsigned long long>(workspace_bytes), static_cast<long long>(w.total));
  if (w.total > 0 && ws == nullptr) return fail(SLIM_ERR_NULL, "workspace is NULL");
  if (!aligned16(ws)) return fail(SLIM_ERR_ALIGN, "workspace must be 16-byte aligned");
  if ((rc = check_arch()) != SLIM_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  xattn::Params p{*q, *k, *v, *out, batch, q_len, kv_len, heads, kv_heads, dim, scale * xattn::kLog2e, nullptr, 0, nullptr};
  cudaError_t e;
  if (masked) {
    float* bias = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + w.bias);
    int* n_keys = reinterpret_cast<int*>(static_cast<uint8_t*>(ws) + w.n_keys);
    xattn::bias_kernel<<<static_cast<unsigned>(batch), 1024, 0, st>>>(
        mask, mask != nullptr ? mask_type : xattn::kMaskNone, mask_stride_b, mask_stride_k, kv_lengths,
        lengths_bits == 64, kv_len, w.pitch, bias, n_keys);
    if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "attention mask launch");
    note_launch();
    p.bias = bias;
    p.bias_pitch = w.pitch;
    p.n_keys = n_keys;
  }
  e = dtype == kBF16 ? xattn::tile::launch<__nv_bfloat16>(p, st) : xattn::tile::launch<__half>(p, st);
  if (e != cudaSuccess) return cuda_fail(e, "cross attention launch");
  note_launch();
  return SLIM_OK;
}

}  // extern "C"
