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
  float* partial;             // split results (see split_floats), or null
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

// ---------------------------------------------------------------- tile kernel
// A row is a (token, query head of the group) pair, the head running fastest, so the heads that share
// keys share their loads; 128 rows are a tile. Two tiles share a CTA, in one of two ways:
//   wide   256 rows of one (sequence, key head), every key tile loaded once for both
//   SPLIT  for few rows: one tile of rows, its keys cut over several CTAs and within a CTA over the
//          two tiles (even and odd key tiles); partial sums go to memory and split_kernel joins them
// 20 warps (the last idle):
//   warps 0..7, 8..15  softmax of tile 0 / 1, half a row (64 keys) a thread: the scores come from TMEM, the
//                     row maximum of both halves through shared memory, the weights 2^(s scale2 + bias
//                     - m) go back packed to 16 bits over the scores, where the second product reads
//                     them. O is rescaled only when a maximum grows by more than 2^8 over the one in use
//                     (the weights stay below 2^8, sums and O are fp32), which is rare after the first
//                     tile. With a whole row a thread one warp per scheduler worked on a tile, issued
//                     its exponentials at half the unit's rate, and a step took XX cycles instead of XX.
//   warp 16           TMA: the Q tiles, then key and value tiles in the order of their use, one ring
//   warps 17, 18      the MMAs of tile 0 / 1: S_t = Q_t K_0^T, then per step O_t += P_t V_j followed at
//                     once by S_t = Q_t K_{j+1}^T: while one tile is in the softmax the tensor cores
//                     work on the other.
// V is read as it lies (keys x head elements): an MN-major operand. Excluded keys have weight 0; their
// rows of V are cleared in shared memory, as 0 * NaN is not 0.
namespace tile {
constexpr int BM = 128, BN = KEY_TILE;
constexpr int SOFTMAX_WARPS = 16, WARP_TMA = 16, WARP_MMA = 17, WARP_RELAY = 19;
constexpr int WARPS = 20, THREADS = 32 * WARPS;
// Registers: 96 a thread at launch, of which the softmax warps take 104 and the last warpgroup leaves
// all but 64: 4 x 104 + 64 = 5 x 96.
constexpr int REGS = 96, REGS_SOFTMAX = 104, REGS_OTHER = 64;
static_assert(4 * REGS_SOFTMAX + REGS_OTHER <= 5 * REGS, "the register shares exceed the launch's allocation");
__device__ __forceinline__ constexpr uint32_t col_s(int t) { return t * 128u; }         // scores, then weights
__device__ __forceinline__ constexpr uint32_t col_o(int t) { return 256u + t * 128u; }  // output accumulator
constexpr float GROWTH = 8.0f;  // base-2 growth of a maximum that is let stand

template <int DP, bool SPLIT>
struct Layout {
  static constexpr int BLOCKS = DP / 64;               // 64-element (128-byte) column blocks of a tile
  static constexpr int BLOCK_BYTES = 128 * 128;
  static constexpr int TILE_BYTES = BLOCKS * BLOCK_BYTES;
  static constexpr int Q_TILES = SPLIT ? 1 : 2;
  static constexpr int STAGES = DP == 64 ? 8 : SPLIT ? 6 : 4;
  static constexpr int STAGING_BYTES = SPLIT ? 0 : 2048;  // a softmax warp's: 32 rows x 32 columns of the output
  static constexpr int OFF_KV = Q_TILES * TILE_BYTES;
  static constexpr int OFF_STAGING = OFF_KV + STAGES * TILE_BYTES;
  static constexpr int OFF_SH = OFF_STAGING + SOFTMAX_WARPS * STAGING_BYTES;
};

template <int STAGES>
struct Shared {
  uint64_t q_full[2], q_free[2];
  uint64_t full[STAGES], empty[STAGES];
  uint64_t s_full[2], p_full[2], o_full[2], o_free[2];
  uint64_t turn[2];   // wide: the tile whose MMAs may be issued
  uint64_t drain[2];
  uint32_t tmem_base;
  volatile int abort;
  float x[2][2][BM];  // a row's maxima over both halves of the keys: [tile][half][row]
};

template <int DP, bool SPLIT>
constexpr size_t smem_bytes() {
  static_assert(Layout<DP, SPLIT>::OFF_SH + sizeof(Shared<Layout<DP, SPLIT>::STAGES>) <= 232448, "shared memory");
  return Layout<DP, SPLIT>::OFF_SH + sizeof(Shared<Layout<DP, SPLIT>::STAGES>);
}

struct TileParams {
  slim_view out;
  int64_t q_len, kv_len;
  int kv_heads, dim;
  int group, tokens;          // query heads per key head, tokens per 128-row tile
  int kb, kh, vb, vh;         // 0 for a k / v that is the same for every sequence / head
  float scale2;
  Keys keys;
  int items, per_head;        // items in all, and of one (sequence, key head)
  // SPLIT
  int splits, per;            // items per tile of rows, key tiles of each (even)
  int rows;                   // rows of a tile that exist
  float* partial;
};

// One piece of work: a pair of row tiles (SPLIT: one row tile and a range of the keys) of a (sequence, head).
struct Item {
  int b, hk, split, tiles;
  int64_t q_tile, tok0, keys;
  int j0, steps;              // SPLIT: first key tile; steps over key tiles
};

template <bool BIAS, bool SPLIT>
__device__ __forceinline__ Item item_at(const TileParams& p, int index) {
  Item it;
  const int head = index / p.per_head, x = index - head * p.per_head;
  it.b = head / p.kv_heads;
  it.hk = head - it.b * p.kv_heads;
  it.split = SPLIT ? x % p.splits : 0;
  it.q_tile = SPLIT ? x / p.splits : 2 * static_cast<int64_t>(x);
  it.tok0 = it.q_tile * p.tokens;
  it.tiles = SPLIT || it.tok0 + p.tokens < p.q_len ? 2 : 1;
  it.keys = BIAS ? p.keys.n_keys[it.b]
            : p.keys.lengths != nullptr ? clamp_length(p.keys.lengths, p.keys.lengths64, it.b, p.kv_len)
                                        : p.kv_len;
  const int nk = static_cast<int>((it.keys + BN - 1) / BN);
  it.j0 = SPLIT ? it.split * p.per : 0;
  it.steps = !SPLIT ? nk : nk <= it.j0 ? 0 : ((nk - it.j0 < p.per ? nk - it.j0 : p.per) + 1) / 2;
  return it;
}

// Partial results of `parts` pieces of `items` tiles of `rows` rows: (m, l) pairs, then O rows.
__host__ __device__ inline int64_t split_floats(int64_t parts, int64_t items, int64_t rows, int dp) {
  return parts * items * rows * (2 + dp);
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

// Base-2 weights of 32 keys: w = 2^(y sc + off), summed in fp32, packed to the type of v.
template <typename T>
__device__ __forceinline__ void weights(const float* y, float2 sc2, float2 off2, float2& l2, uint32_t (&w)[16]) {
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float2 x = fma2(make_float2(y[2 * e], y[2 * e + 1]), sc2, off2);
    const float2 g = make_float2(ex2_approx(x.x), ex2_approx(x.y));
    l2 = add2(l2, g);
    w[e] = pack2<T>(g.x, g.y);
  }
}

__device__ __forceinline__ float row_max(const float* y) {
  float mx[4] = {y[0], y[1], y[2], y[3]};
#pragma unroll
  for (int e = 4; e < 60; e += 8) {
#pragma unroll
    for (int u = 0; u < 4; ++u) mx[u] = fmax3(mx[u], y[e + u], y[e + 4 + u]);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) mx[u] = fmaxf(mx[u], y[60 + u]);
  return fmaxf(fmax3(mx[0], mx[1], mx[2]), mx[3]);
}

template <typename T, int DP, bool BIAS, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
tile_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
            const __grid_constant__ CUtensorMap tv, const TileParams p) {
  using L = Layout<DP, SPLIT>;
  using Sh = Shared<L::STAGES>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr uint32_t IDESC_QK = idesc_f16(BM, BN, BF16, false);
  constexpr uint32_t IDESC_PV = idesc_f16(BM, DP, BF16, true);
  constexpr int STEP_LOADS = SPLIT ? 4 : 2;
  extern __shared__ __align__(1024) uint8_t tile_smem[];
  uint8_t* smem = tile_smem;
  if (smem_u32(smem) & 1023) {  // the swizzled tiles need it; there is no room to round up
    record_error(kErrSmemAlign);
    return;
  }
  uint8_t* sQ = smem;
  uint8_t* sKV = smem + L::OFF_KV;
  Sh& sh = *reinterpret_cast<Sh*>(smem + L::OFF_SH);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  // key tile of a step: wide, j for both tiles; SPLIT, j0 + 2 j + t. Position of a tile's K and V in the
  // order of a step's loads: wide K V, SPLIT K_0 K_1 V_0 V_1
  auto k_load = [](int t) { return SPLIT ? t : 0; };
  auto v_load = [](int t) { return SPLIT ? 2 + t : 1; };

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh.q_full[t], 1);
      mbar_init(&sh.q_free[t], SPLIT ? 2 : 1);
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.p_full[t], 2 * BM / 32);
      mbar_init(&sh.o_full[t], 1);
      mbar_init(&sh.o_free[t], 2 * BM / 32);
      mbar_init(&sh.turn[t], 1);
      mbar_init(&sh.drain[t], 1);
    }
    for (int s = 0; s < L::STAGES; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], SPLIT ? 1 : 2);  // wide: both tiles have used it
    }
    sh.abort = 0;
    fence_mbar_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(&sh.tmem_base, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem_base;

  if (warp >= SOFTMAX_WARPS) {
    regs_dec<REGS_OTHER>();
    if (warp == WARP_TMA) {
      // ---------------------------------------------------------- TMA producer
      if (lane == 0) {
        const uint32_t q_bytes = static_cast<uint32_t>(L::BLOCKS * 128 * p.group * p.tokens);
        uint32_t issued = 0, last_parity = 0;   // per slot
        uint32_t q_loads[2] = {0, 0};
        int slot = 0, parity = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t ph) {
          ok = ok && mbar_wait_abort(bar, ph, kErrWaitTimeoutProducer, &sh.abort);
          return ok;
        };
        auto load = [&](const Item& it, int i) {
          if (!wait(&sh.empty[slot], parity ^ 1)) return;
          const bool is_v = SPLIT ? (i & 2) != 0 : (i & 1) != 0;
          const int kt = SPLIT ? it.j0 + 2 * (i >> 2) + (i & 1) : i >> 1;
          mbar_arrive_expect_tx(&sh.full[slot], L::TILE_BYTES);
          for (int c = 0; c < L::BLOCKS; ++c)  // rows past the end come as zeros
            tma_load_4d(sKV + slot * L::TILE_BYTES + c * L::BLOCK_BYTES, is_v ? &tv : &tk, &sh.full[slot], c * 64,
                        it.hk * (is_v ? p.vh : p.kh), kt * BN, it.b * (is_v ? p.vb : p.kb));
          issued |= 1u << slot;
          last_parity = (last_parity & ~(1u << slot)) | (static_cast<uint32_t>(parity) << slot);
          if (++slot == L::STAGES) {
            slot = 0;
            parity ^= 1;
          }
        };
        for (int index = blockIdx.x; ok && index < p.items; index += gridDim.x) {
          const Item it = item_at<BIAS, SPLIT>(p, index);
          if (it.steps == 0) continue;
          // the first keys do not have to wait for the last item's queries to be done with
          load(it, 0);
          const int q_tiles = SPLIT ? 1 : it.tiles;
          for (int t = 0; ok && t < q_tiles; ++t) {
            if (q_loads[t] > 0 && !wait(&sh.q_free[t], (q_loads[t] - 1) & 1)) break;
            mbar_arrive_expect_tx(&sh.q_full[t], q_bytes);
            for (int c = 0; c < L::BLOCKS; ++c)
              tma_load_4d(sQ + t * L::TILE_BYTES + c * L::BLOCK_BYTES, &tq, &sh.q_full[t], c * 64, it.hk * p.group,
                          static_cast<int32_t>(it.tok0 + t * p.tokens), it.b);
            ++q_loads[t];
          }
          for (int i = 1; ok && i < STEP_LOADS * it.steps; ++i) load(it, i);
        }
        // every load issued by this thread lands before the CTA may exit
        for (int t = 0; t < 2; ++t)
          if (q_loads[t] > 0) mbar_wait(&sh.q_full[t], (q_loads[t] - 1) & 1, kErrWaitTimeoutDrain);
        for (int s = 0; s < L::STAGES; ++s)
          if (issued & (1u << s)) mbar_wait(&sh.full[s], (last_parity >> s) & 1, kErrWaitTimeoutDrain);
      }
    } else if (warp - WARP_MMA < 2) {
      // ---------------------------------------------------------- MMA issue of tile t
      const int t = warp - WARP_MMA;
      if (lane == 0) {
        // the ring position of a load, carried along as (slot, parity)
        struct Ring {
          int slot, parity;
          __device__ __forceinline__ Ring at(int n) const {
            const int s = slot + n;
            return s >= L::STAGES ? Ring{s - L::STAGES, parity ^ 1} : Ring{s, parity};
          }
        };
        const uint64_t q_desc = smem_desc_sw128(smem_u32(sQ + (SPLIT ? 0 : t * L::TILE_BYTES)));
        const uint32_t kv_addr = smem_u32(sKV);
        const uint32_t t_s = tmem + col_s(t), t_o = tmem + col_o(t);
        Ring base{0, 0};        // of the step's first load
        uint32_t items = 0;     // of this tile so far
        uint32_t steps = 0;     // of this tile so far
        uint32_t batches = 0;   // of MMAs issued in turn so far
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t ph) {
          ok = ok && mbar_poll_abort(bar, ph, kErrWaitTimeoutMma, &sh.abort);
          return ok;
        };
        auto full = [&](Ring r) { return wait(&sh.full[r.slot], r.parity); };
        for (int index = blockIdx.x; ok && index < p.items; index += gridDim.x) {
          const Item it = item_at<BIAS, SPLIT>(p, index);
          if (it.steps == 0) continue;
          if (t >= it.tiles) {  // the other tile's loads
            const int n = base.slot + STEP_LOADS * it.steps;
            base = Ring{n % L::STAGES, base.parity ^ (n / L::STAGES & 1)};
            continue;
          }
          // Both tiles' MMAs share the tensor cores. Issued as they come they interleave, both tiles finish
          // late and their softmaxes run in step (3.90 instead of 2.77 ms at 16384 x 16111 x 24 heads of
          // 128); so the batches (second product, next scores) take turns. The turn passes on before a batch's
          // last MMAs are issued: they cover the time until the other tile's thread has noticed.
          auto my_turn = [&] { return it.tiles == 1 || wait(&sh.turn[t], t == 0 ? (batches & 1) ^ 1 : batches & 1); };
          auto pass_turn = [&] {
            if (it.tiles == 2) {
              mbar_arrive(&sh.turn[t ^ 1]);
              ++batches;
            }
          };
          auto qk = [&](Ring r) {
            const uint64_t kd = smem_desc_sw128(kv_addr + r.slot * L::TILE_BYTES);
#pragma unroll
            for (int k = 0; k < DP / 16; ++k) {
              if (k == DP / 32) pass_turn();
              const uint32_t off = (k >> 2) * L::BLOCK_BYTES + (k & 3) * 32;
              mma_f16(t_s, smem_desc_at(q_desc, off), smem_desc_at(kd, off), IDESC_QK, k != 0);
            }
            mma_commit(&sh.s_full[t]);
          };
          if (!full(base.at(k_load(t))) || !wait(&sh.q_full[SPLIT ? 0 : t], items & 1) || !my_turn()) break;
          tc_fence_after();
          qk(base.at(k_load(t)));
          for (int j = 0; j < it.steps; ++j) {
            const Ring next = base.at(STEP_LOADS), v = base.at(v_load(t)), k = next.at(k_load(t));
            const bool more = j + 1 < it.steps;
            if (!full(v) || (more && !full(k)) || !my_turn()) break;
            // the last item's output has been read
            if (j == 0 && items > 0 && !wait(&sh.o_free[t], (items - 1) & 1)) break;
            if (!wait(&sh.p_full[t], (steps + j) & 1)) break;
            tc_fence_after();
            const uint64_t vd = smem_desc_mn_sw128(kv_addr + v.slot * L::TILE_BYTES, L::BLOCK_BYTES);
#pragma unroll
            for (int c = 0; c < BN / 16; ++c)
              mma_f16_ta(t_o, t_s + c * 8, smem_desc_at(vd, c * 2048), IDESC_PV, j != 0 || c != 0);
            if (more) {
              qk(k);
            } else {
              mma_commit(&sh.o_full[t]);
              pass_turn();
            }
            base = next;
          }
          steps += it.steps;
          ++items;
        }
        mma_commit(&sh.drain[t]);
        mbar_wait(&sh.drain[t], 0, kErrWaitTimeoutDrain);
      }
    }
    else if (warp == WARP_RELAY && lane == 0) {
      // ---------------------------------------------------------- tiles handed back to the producer
      // A tcgen05.commit holds the tensor cores up for about 120 cycles, so there is one a step (S_j ready,
      // hence Q K_j done, and before it P_{j-1} V_{j-1}: one thread issued them in order) instead of one
      // for each tile of keys and values that is done with; this thread passes it on.
      uint32_t loads = 0, steps[2] = {0, 0}, items[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t ph) {
        ok = ok && mbar_wait_abort(bar, ph, kErrWaitTimeoutMma, &sh.abort);
        return ok;
      };
      for (int index = blockIdx.x; ok && index < p.items; index += gridDim.x) {
        const Item it = item_at<BIAS, SPLIT>(p, index);
        auto release = [&](uint32_t i) {
          mbar_arrive(&sh.empty[i % L::STAGES]);
          if (it.tiles == 1) mbar_arrive(&sh.empty[i % L::STAGES]);
        };
        for (int j = 0; ok && j < it.steps; ++j) {
          for (int t = 0; t < it.tiles && wait(&sh.s_full[t], (steps[t] + j) & 1); ++t) {
            release(loads + STEP_LOADS * j + k_load(t));
            if (j > 0) release(loads + STEP_LOADS * (j - 1) + v_load(t));
            if (j + 1 == it.steps) mbar_arrive(&sh.q_free[SPLIT ? 0 : t]);
          }
        }
        for (int t = 0; it.steps > 0 && t < it.tiles && wait(&sh.o_full[t], items[t] & 1); ++t) {
          release(loads + STEP_LOADS * (it.steps - 1) + v_load(t));
          steps[t] += it.steps;
          ++items[t];
        }
        loads += STEP_LOADS * it.steps;
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax of half a row, output
    regs_inc<REGS_SOFTMAX>();
    const int t = warp >> 3;
    const int half = (warp >> 2) & 1;  // of the keys of a tile, of the columns of O
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_s = t_lane + col_s(t), t_o = t_lane + col_o(t) + half * (DP / 2);
    const float scale2 = p.scale2;
    // few rows: warps whose rows do not exist only keep step
    const bool live = !SPLIT || quarter * 32 < p.rows;
    // 128 rows need not be a whole number of tokens: what is left in the others has no say in rescaling
    const bool real = row < p.group * p.tokens;
    // After a wait that failed the warp goes through its steps without work (every further wait fails at
    // once), so that both halves meet at each of their barriers.
    bool good = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      good = __all_sync(0xffffffffu, mbar_wait_abort(bar, parity, kErrWaitTimeoutEpilogue, &sh.abort)) != 0 && good;
    };
    uint32_t step0 = 0;   // steps of this tile before the item
    uint32_t loads0 = 0;  // loads of both tiles before the item
    uint32_t items0 = 0;  // items of this tile before the item
#pragma unroll 1
    for (int index = blockIdx.x; index < p.items; index += gridDim.x) {
      const Item it = item_at<BIAS, SPLIT>(p, index);
      const int b = it.b;
      if (t >= it.tiles) {
        loads0 += STEP_LOADS * it.steps;
        continue;
      }
      float m = -INFINITY;
      float2 l2 = make_float2(0.0f, 0.0f);
#pragma unroll 1
      for (int j = 0; j < it.steps; ++j) {
        const int64_t key0 = static_cast<int64_t>(SPLIT ? it.j0 + 2 * j + t : j) * BN;
        const float4* bias4 =
            BIAS ? reinterpret_cast<const float4*>(p.keys.bias + b * p.keys.bias_pitch + key0 + 64 * half) : nullptr;
        const int64_t left64 = it.keys - key0;
        const int left = left64 < BN ? static_cast<int>(left64) : BN;  // keys of this tile up to the last one
        // one bit per key of this half that takes part (with a bias: per key up to the last one)
        uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
        bool used = row < left;  // the key of this row's number
        if (left < BN) {
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int n = left - 64 * half - 32 * w;
            bits[w] = n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u;
          }
        }
        if (BIAS) {
          used = used && __ldg(p.keys.bias + b * p.keys.bias_pitch + key0 + row) != -INFINITY;
        } else if (p.keys.mask != nullptr) {
          const uint8_t* mask = p.keys.mask + b * p.keys.mask_b;
          used = used && __ldg(mask + (key0 + row) * p.keys.mask_k) != 0;
#pragma unroll
          for (int w = 0; w < 2; ++w) {
            const int i = 64 * half + 32 * w + lane;
            bits[w] = __ballot_sync(0xffffffffu, i < left && __ldg(mask + (key0 + i) * p.keys.mask_k) != 0);
          }
        }
        const bool clear = !used && key0 + row < p.kv_len;
        if (__any_sync(0xffffffffu, clear)) {
          // wide: both tiles clear the same rows, each before its own second product
          const uint32_t i = loads0 + STEP_LOADS * j + v_load(t), slot = i % L::STAGES;
          wait(&sh.full[slot], (i / L::STAGES) & 1);
          if (clear && good) {
            uint4* v = reinterpret_cast<uint4*>(sKV + slot * L::TILE_BYTES + row * 128 +
                                                half * (DP == 128 ? L::BLOCK_BYTES : 64));
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) v[e] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        wait(&sh.s_full[t], (step0 + j) & 1);
        tc_fence_after();
        if (live) {
          uint32_t r[64];
          tmem_ld_32x32b_x32(t_s + 64 * half, *reinterpret_cast<uint32_t(*)[32]>(r));
          tmem_ld_32x32b_x32(t_s + 64 * half + 32, *reinterpret_cast<uint32_t(*)[32]>(r + 32));
          tmem_ld_wait();
          reg_dep32(*reinterpret_cast<uint32_t(*)[32]>(r));
          reg_dep32(*reinterpret_cast<uint32_t(*)[32]>(r + 32));
          float* y = reinterpret_cast<float*>(r);
          if (BIAS) {
#pragma unroll
            for (int e = 0; e < 64; e += 4) {
              // an excluded key's score may be NaN; behind the last key the bias row may have ended
              const float4 a = (bits[e / 32] >> (e & 31)) & 1 ? __ldg(bias4 + e / 4)
                                                              : make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
              y[e + 0] = a.x == -INFINITY ? -INFINITY : fmaf(y[e + 0], scale2, a.x);
              y[e + 1] = a.y == -INFINITY ? -INFINITY : fmaf(y[e + 1], scale2, a.y);
              y[e + 2] = a.z == -INFINITY ? -INFINITY : fmaf(y[e + 2], scale2, a.z);
              y[e + 3] = a.w == -INFINITY ? -INFINITY : fmaf(y[e + 3], scale2, a.w);
            }
          } else if ((bits[0] & bits[1]) != 0xffffffffu) {
#pragma unroll
            for (int e = 0; e < 64; ++e) y[e] = (bits[e / 32] >> (e & 31)) & 1 ? y[e] : -INFINITY;
          }
          // Weights 2^(y sc - m). From the second step on they are taken with the m in use, and only if some
          // row's maximum then turns out to have grown too far are they taken again: that keeps the maxima
          // off the way from the scores to the weights.
          const float sc = BIAS ? 1.0f : scale2;
          const int pair = 1 + 4 * t + quarter;  // barrier of both halves
          float2 add = make_float2(0.0f, 0.0f);
          auto store_weights = [&] {
            const float off = m == -INFINITY ? 0.0f : -m;
            const float2 off2 = make_float2(off, off), sc2 = make_float2(sc, sc);
            add = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < 64; c += 32) {
              uint32_t w[16];
              weights<T>(y + c, sc2, off2, add, w);
              tmem_st_32x32b_x16(t_s + 32 * half + c / 2, w);
            }
          };
          if (j > 0) {
            named_barrier(pair, 64);  // both halves have read the scores that the weights go over
            store_weights();
          }
          const float own = row_max(y) * sc;
          if (j == 0 || named_barrier_any(pair, 64, real && own > m + GROWTH)) {
            sh.x[t][half][row] = own;
            named_barrier(pair, 64);
            const float m_new = fmaxf(m, fmaxf(own, sh.x[t][half ^ 1][row]));
            named_barrier(pair, 64);  // both have read it before it is written again
            if (j > 0) {
              // O holds P_0 V_0 + ... + P_{j-1} V_{j-1} (done before S_j)
              const float alpha = m_new == -INFINITY ? 1.0f : ex2_approx(m - m_new);
              l2 = mul2(l2, make_float2(alpha, alpha));
#pragma unroll 1
              for (int c = 0; c < DP / 2; c += 16) {
                uint32_t o[16];
                tmem_ld_32x32b_x16(t_o + c, o);
                tmem_ld_wait();
                reg_dep16(o);
#pragma unroll
                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * alpha);
                tmem_st_32x32b_x16(t_o + c, o);
              }
            }
            m = m_new;
            store_weights();
          }
          l2 = add2(l2, add);
          tmem_st_wait();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[t]);
      }
      if (it.steps > 0) {
        wait(&sh.o_full[t], items0 & 1);
        tc_fence_after();
        ++items0;
      }
      // the sum over both halves
      sh.x[t][half][row] = l2.x + l2.y;
      named_barrier(1 + 4 * t + quarter, 64);
      const float l = sh.x[t][0][row] + sh.x[t][1][row];
      named_barrier(1 + 4 * t + quarter, 64);  // both have read it before the next item's maxima
      if (SPLIT) {
        // (m, l) and O of this piece; O stays unwritten where no key took part
        if (good && live) {
          const int64_t parts = 2 * p.splits, row_tiles = p.items / p.splits;
          const int64_t at = ((2 * it.split + t) * row_tiles + index / p.splits) * p.rows + row;
          const bool exists = row < p.rows;
          if (exists && half == 0) reinterpret_cast<float2*>(p.partial)[at] = make_float2(m, l);
          if (it.steps > 0) {
            float* o = p.partial + 2 * parts * row_tiles * p.rows + at * DP + half * (DP / 2);
#pragma unroll 1
            for (int c = 0; c < DP / 2; c += 32) {
              uint32_t r[32];
              tmem_ld_32x32b_x32(t_o + c, r);
              tmem_ld_wait();
              reg_dep32(r);
              if (exists) {
#pragma unroll
                for (int u = 0; u < 8; ++u)
                  reinterpret_cast<uint4*>(o + c)[u] = make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]);
              }
            }
          }
        }
        if (it.steps > 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.o_free[t]);
        }
      } else {
        // 32 columns of the warp's 32 rows at a time through its own shared memory (16-byte chunk u of row
        // r at u ^ (r >> 1 & 3)), then 64-byte pieces of 8 rows a store
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        uint8_t* stage = smem + L::OFF_STAGING + warp * L::STAGING_BYTES;
#pragma unroll 1
        for (int c = 0; c < DP / 2; c += 32) {
          uint32_t r[32];
          if (it.steps > 0) {
            tmem_ld_32x32b_x32(t_o + c, r);
            tmem_ld_wait();
            reg_dep32(r);
            if (c + 32 == DP / 2) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(&sh.o_free[t]);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) r[e] = 0;
          }
          __syncwarp();
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = pack2<T>(__uint_as_float(r[8 * u + 2 * e]) * inv, __uint_as_float(r[8 * u + 2 * e + 1]) * inv);
            *reinterpret_cast<uint4*>(stage + lane * 64 + ((u ^ (lane >> 1 & 3)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
          const int chunk = lane & 3, col = half * (DP / 2) + c + chunk * 8;
          if (good && col < p.dim) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int sr = i * 8 + (lane >> 2), tr = quarter * 32 + sr;
              const int tok = tr / p.group, h = it.hk * p.group + tr - tok * p.group;
              const int64_t token = it.tok0 + t * p.tokens + tok;
              if (tok < p.tokens && token < p.q_len)
                *reinterpret_cast<uint4*>(static_cast<T*>(p.out.data) + b * p.out.stride_b + token * p.out.stride_s +
                                          h * p.out.stride_h + col) =
                    *reinterpret_cast<const uint4*>(stage + sr * 64 + ((chunk ^ (sr >> 1 & 3)) << 4));
            }
          }
        }
      }
      step0 += it.steps;
      loads0 += STEP_LOADS * it.steps;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------- joining the pieces of a split
// One block per row: 8 warps take every 8th piece, a lane DP / 32 columns; pieces in a fixed order.
// out = sum_i 2^(m_i - M) O_i / sum_i 2^(m_i - M) l_i, pieces without keys left unread.
template <typename T, int DP>
__global__ void __launch_bounds__(256) split_kernel(const float* __restrict__ partial, slim_view out, int64_t q_len,
                                                    int group, int tokens, int rows, int q_tiles, int kv_heads,
                                                    int parts, int64_t items, int dim) {
  constexpr int E = DP / 32;
  __shared__ float s_o[8][DP];
  __shared__ float s_l[8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t item = blockIdx.x / rows;
  const int row = static_cast<int>(blockIdx.x - item * rows);
  const int64_t token = item % q_tiles * tokens + row / group;
  if (token >= q_len) return;  // whole blocks
  const float2* ml = reinterpret_cast<const float2*>(partial) + item * rows + row;
  const float* o = partial + 2 * parts * items * rows + (item * rows + row) * DP + lane * E;
  const int64_t step = items * rows;
  float top = -INFINITY;
  for (int i = lane; i < parts; i += 32) top = fmaxf(top, ml[i * step].x);
#pragma unroll
  for (int sft = 16; sft >= 1; sft >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sft));
  const float off = top == -INFINITY ? 0.0f : top;
  float acc[E] = {}, l = 0.0f;
#pragma unroll 4
  for (int i = warp; i < parts; i += 8) {
    const float2 a = ml[i * step];
    if (a.y == 0.0f) continue;
    const float w = exp2f(a.x - off);
    l = fmaf(w, a.y, l);
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(w, o[i * step * DP + e], acc[e]);
  }
#pragma unroll
  for (int e = 0; e < E; ++e) s_o[warp][lane * E + e] = acc[e];
  if (lane == 0) s_l[warp] = l;
  __syncthreads();
  const int d = threadIdx.x;
  if (d < dim) {
    float x = 0.0f;
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      x += s_o[w][d];
      l += s_l[w];
    }
    const int64_t b = item / q_tiles / kv_heads;
    const int h = static_cast<int>(item / q_tiles % kv_heads) * group + row % group;
    T* dst = static_cast<T*>(out.data) + b * out.stride_b + token * out.stride_s + h * out.stride_h;
    store_f(dst + d, l == 0.0f ? 0.0f : x / l);
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

// How a problem is laid over the SMs: splits = 0 for the wide form.
struct Plan {
  int group, tokens;
  int64_t q_tiles;
  int splits, per;            // per: key tiles of a split, even
  int rows;
  int64_t floats;             // of partial results
};

// The wide form takes 2 row tiles x 1 key tile a step, SPLIT 1 row tile x 2 key tiles, which moves twice
// the keys and values through L2 for the same work (a step takes 1.35 times as long at 16384 x 16111 x
// 24 heads of 128). Costs in wide steps (about 2 us): an item's ends cost 0.7, a launch 2, joining the
// pieces 1.5. The cheapest wins: few rows are split, many waves of items are not.
inline Plan make_plan(int64_t batch, int64_t q_len, int64_t kv_len, int heads, int kv_heads, int dim) {
  Plan p{};
  p.group = heads / kv_heads;
  p.tokens = BM / p.group;
  p.q_tiles = (q_len + p.tokens - 1) / p.tokens;
  const int64_t nk = (kv_len + BN - 1) / BN, base = batch * kv_heads, sms = sm_count();
  auto waves = [&](int64_t ctas) { return (ctas + sms - 1) / sms; };
  double best = static_cast<double>(waves(base * ((p.q_tiles + 1) / 2))) * (0.7 + static_cast<double>(nk)) + 2.0;
  for (int64_t s = 1; s <= 64 && 2 * (s - 1) < nk; ++s) {
    const int64_t per = (nk + 2 * s - 1) / (2 * s) * 2;
    if ((s - 1) * per >= nk) continue;  // the last CTAs would have nothing
    const double cost = static_cast<double>(waves(base * p.q_tiles * s)) * (0.7 + 1.35 * static_cast<double>(per) / 2) + 3.5;
    if (cost < best && base * p.q_tiles * s < (int64_t{1} << 24)) {
      best = cost;
      p.splits = static_cast<int>(s);
      p.per = static_cast<int>(per);
    }
  }
  if (p.splits > 0) {
    p.rows = p.group * static_cast<int>(q_len < p.tokens ? q_len : p.tokens);
    p.floats = split_floats(2 * p.splits, base * p.q_tiles, p.rows, dim > 64 ? 128 : 64);
  }
  return p;
}

template <typename T, int DP, bool BIAS, bool SPLIT>
cudaError_t launch(const Params& p, const Plan& plan, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mq, mk, mv;
  // without keys k and v may be null: their maps are never used
  const bool any = p.kv_len > 0;
  if (!make_map(&mq, BF16, p.q, p.batch, p.q_len, p.heads, p.dim, plan.group, plan.tokens) ||
      !make_map(&mk, BF16, any ? p.k : p.q, p.batch, any ? p.kv_len : 1, any ? p.kv_heads : 1, p.dim, 1, BN) ||
      !make_map(&mv, BF16, any ? p.v : p.q, p.batch, any ? p.kv_len : 1, any ? p.kv_heads : 1, p.dim, 1, BN))
    return cudaErrorInvalidValue;
  int dev = 0;
  cudaGetDevice(&dev);
  static PerDeviceOnce once;
  constexpr size_t smem = smem_bytes<DP, SPLIT>();
  cudaError_t e = once.run(dev, [] {
    cudaFuncAttributes attr;
    cudaError_t err = cudaFuncGetAttributes(&attr, tile_kernel<T, DP, BIAS, SPLIT>);
    if (err == cudaSuccess && attr.numRegs < REGS) err = cudaErrorInvalidConfiguration;  // the shares would not fit
    if (err != cudaSuccess) return err;
    return cudaFuncSetAttribute(tile_kernel<T, DP, BIAS, SPLIT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem));
  });
  if (e != cudaSuccess) return e;
  const int64_t per_head = SPLIT ? plan.q_tiles * plan.splits : (plan.q_tiles + 1) / 2;
  const int64_t items = per_head * p.kv_heads * p.batch;
  TileParams tp{p.out, p.q_len, p.kv_len, p.kv_heads, p.dim, plan.group, plan.tokens, p.k.stride_b != 0,
                p.k.stride_h != 0, p.v.stride_b != 0, p.v.stride_h != 0, p.scale2, p.keys, static_cast<int>(items),
                static_cast<int>(per_head), plan.splits, plan.per, plan.rows, p.partial};
  const int64_t sms = sm_count();
  tile_kernel<T, DP, BIAS, SPLIT><<<static_cast<unsigned>(items < sms ? items : sms), THREADS, smem, st>>>(mq, mk, mv, tp);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  note_launch();
  if (SPLIT) {
    const int64_t tiles = items / plan.splits;
    split_kernel<T, DP><<<static_cast<unsigned>(tiles * plan.rows), 256, 0, st>>>(
        p.partial, p.out, p.q_len, plan.group, plan.tokens, plan.rows, static_cast<int>(plan.q_tiles), p.kv_heads,
        2 * plan.splits, tiles, p.dim);
    if ((e = cudaGetLastError()) != cudaSuccess) return e;
    note_launch();
  }
  return cudaSuccess;
}

template <typename T, int DP>
cudaError_t launch(const Params& p, const Plan& plan, cudaStream_t st) {
  if (plan.splits > 0)
    return p.keys.bias != nullptr ? launch<T, DP, true, true>(p, plan, st) : launch<T, DP, false, true>(p, plan, st);
  return p.keys.bias != nullptr ? launch<T, DP, true, false>(p, plan, st) : launch<T, DP, false, false>(p, plan, st);
}
}  // namespace tile

struct Workspace {
  int64_t bias, n_keys, partial, total, pitch;
};

static Workspace workspace(int64_t batch, int64_t kv_len, bool additive, const tile::Plan& plan) {
  auto up = [](int64_t v) { return (v + 255) / 256 * 256; };
  Workspace w{};
  w.pitch = (kv_len + KEY_TILE - 1) / KEY_TILE * KEY_TILE;
  if (additive) {
    w.n_keys = up(batch * w.pitch * 4);
    w.total = w.n_keys + up(batch * 4);
  }
  w.partial = w.total;
  w.total += up(plan.floats * 4);
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
  const int64_t tokens = 128 / (heads / kv_heads);
  if (batch >= (int64_t{1} << 16) || q_len >= (int64_t{1} << 31) - 256 || kv_len >= (int64_t{1} << 31) - 256 || heads >= (1 << 16) ||
      (q_len + tokens - 1) / tokens * kv_heads * (batch < 1 ? 1 : batch) >= (int64_t{1} << 31))
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
                                    int additive, uint64_t* bytes) {
  const int rc = xattn::checks(batch, q_len, kv_len, heads, kv_heads, dim);
  if (rc != SLIM_OK) return rc;
  if (bytes == nullptr) return fail(SLIM_ERR_NULL, "bytes is NULL");
  const xattn::tile::Plan plan = xattn::tile::make_plan(batch, q_len, kv_len, heads, kv_heads, dim);
  *bytes = static_cast<uint64_t>(xattn::workspace(batch, kv_len, additive != 0, plan).total);
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
  const bool additive = kv_len > 0 && mask != nullptr && mask_type != SLIM_MASK_BOOL;
  const xattn::tile::Plan plan = xattn::tile::make_plan(batch, q_len, kv_len, heads, kv_heads, dim);
  const xattn::Workspace w = xattn::workspace(batch, kv_len, additive, plan);
  if (workspace_bytes < static_cast<uint64_t>(w.total))
    return fail(SLIM_ERR_SHAPE, "workspace of %llu bytes is smaller than the %lld needed",
                static_cast<unsigned long long>(workspace_bytes), static_cast<long long>(w.total));
  if (w.total > 0 && ws == nullptr) return fail(SLIM_ERR_NULL, "workspace is NULL");
  if (!aligned16(ws)) return fail(SLIM_ERR_ALIGN, "workspace must be 16-byte aligned");
  if ((rc = check_arch()) != SLIM_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* base = static_cast<uint8_t*>(ws);
  xattn::Params p{*q, *k, *v, *out, batch, q_len, kv_len, heads, kv_heads, dim, scale * xattn::kLog2e, {}, nullptr};
  if (plan.floats > 0) p.partial = reinterpret_cast<float*>(base + w.partial);
  cudaError_t e;
  if (additive) {
    float* bias = reinterpret_cast<float*>(base + w.bias);
    int* n_keys = reinterpret_cast<int*>(base + w.n_keys);
    xattn::bias_kernel<<<static_cast<unsigned>(batch), 1024, 0, st>>>(mask, mask_type, mask_stride_b, mask_stride_k,
                                                                      kv_lengths, lengths_bits == 64, kv_len, w.pitch,
                                                                      bias, n_keys);
    if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "attention mask launch");
    note_launch();
    p.keys.bias = bias;
    p.keys.bias_pitch = w.pitch;
    p.keys.n_keys = n_keys;
  } else if (kv_len > 0) {
    p.keys.mask = static_cast<const uint8_t*>(mask);
    p.keys.mask_b = mask_stride_b;
    p.keys.mask_k = mask_stride_k;
    p.keys.lengths = kv_lengths;
    p.keys.lengths64 = lengths_bits == 64;
  }
  if (dtype == kBF16)
    e = dim > 64 ? xattn::tile::launch<__nv_bfloat16, 128>(p, plan, st) : xattn::tile::launch<__nv_bfloat16, 64>(p, plan, st);
  else
    e = dim > 64 ? xattn::tile::launch<__half, 128>(p, plan, st) : xattn::tile::launch<__half, 64>(p, plan, st);
  if (e != cudaSuccess) return cuda_fail(e, "cross attention launch");
  return SLIM_OK;
}

}  // extern "C"
