// Cross attention, many rows: 256 rows of one (sequence, key head) a CTA.
#pragma once

#include "cross_attn.cuh"

namespace slim {
namespace xattn {
namespace wide {

// Persistent CTAs, one per SM. An item is a pair of row tiles with all its keys; both tiles use every tile
// of keys and values that is loaded. 20 warps:
//   warps 0..7, 8..15  softmax of tile 0 / 1, half a row (64 keys) a thread: scores from TMEM, weights
//                2^(s scale2 + bias - m) packed to 16 bits over the scores, where the second product reads
//                them. m is only changed, and O and the sums rescaled, when some row's maximum has grown by
//                more than 2^8 over it (so weights stay in their type's range; sums and O are fp32), which is
//                rare after an item's first step.
//   warp 16      TMA: queries, keys and values in the order of their use
//   warp 17      the MMAs: S_t = Q_t K_0^T, then per step and tile O_t += P_t V_j followed at once by
//                S_t = Q_t K_{j+1}^T: while one tile is in the softmax the tensor cores work on the other.
//                (Two warps that issue for a tile each let the tiles' MMAs interleave: both finish late and
//                their softmaxes run in step, 3.90 instead of 2.77 ms at 16384 x 16111 x 24 heads of 128.)
//   warp 18      hands loads that are done with back to the producer
// Excluded keys have weight 0; their rows of V are cleared in shared memory, as 0 * NaN is not 0.
//
// 16384 x 16111 x 24 heads of 128, bf16: 2.66 to 2.78 ms in single launches (1170 to 1220 TFLOP/s, by the card), 3.1 ms
// (1050) one after the other under the power cap. A step (both tiles) takes 3900 cycles: the
// products alone 2700 of them (their operands come through shared memory), the exponentials alone 2050,
// and a tile's scores -> weights -> second product -> next scores chain 3900, which bounds it now. A row a
// thread instead of half a row: 2.79 ms.
constexpr int WARP_TMA = 16, WARP_MMA = 17, WARP_RELAY = 18;
__device__ __forceinline__ constexpr uint32_t col_s(int t) { return t * 128u; }         // scores, then weights
__device__ __forceinline__ constexpr uint32_t col_o(int t) { return 256u + t * 128u; }  // output accumulator

template <int DP>
struct Layout {
  static constexpr int TILE = Tile<DP>::BYTES;
  static constexpr int PAIRS = DP == 64 ? 4 : 2;  // ring places of a V and a K tile
  static constexpr int STAGING = 32 * 32 * 2;     // a softmax warp's: 32 rows x 32 columns of the output
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int OFF_STAGING = OFF_KV + PAIRS * 2 * TILE;
  static constexpr int OFF_SH = OFF_STAGING + SOFTMAX_WARPS * STAGING;
};

template <int PAIRS>
struct Shared {
  uint64_t q_full[2], q_free[2];
  uint64_t full[PAIRS], empty[PAIRS];
  uint64_t s_full[2], p_full[2], o_full[2], o_free[2];
  uint64_t drain;
  uint32_t tmem_base;
  volatile int abort;
  float x[2][2][BM];  // a row's maxima over both halves of the keys: [tile][half][row]
};

template <int DP>
constexpr size_t smem_bytes() {
  static_assert(Layout<DP>::OFF_SH + sizeof(Shared<Layout<DP>::PAIRS>) <= 232448, "shared memory");
  return Layout<DP>::OFF_SH + sizeof(Shared<Layout<DP>::PAIRS>);
}

struct Item {
  int b, hk, tiles, keys, steps;
  int64_t tok0;
};

template <bool BIAS>
__device__ __forceinline__ Item item_at(const TileParams& p, int index) {
  Item it;
  const int head = index / p.per_head;
  it.b = head / p.kv_heads;
  it.hk = head - it.b * p.kv_heads;
  it.tok0 = static_cast<int64_t>(index - head * p.per_head) * 2 * p.tokens;
  it.tiles = it.tok0 + p.tokens < p.q_len ? 2 : 1;
  it.keys = keys_of<BIAS>(p, it.b);
  it.steps = (it.keys + BN - 1) / BN;
  return it;
}

template <typename T, int DP, bool BIAS>
__global__ void __launch_bounds__(THREADS, 1)
wide_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
            const __grid_constant__ CUtensorMap tv, const __grid_constant__ TileParams p) {
  using L = Layout<DP>;
  using Sh = Shared<L::PAIRS>;
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
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

  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&sh.q_full[t], 1);
      mbar_init(&sh.q_free[t], 1);
      mbar_init(&sh.s_full[t], 1);
      mbar_init(&sh.p_full[t], SOFTMAX_WARPS / 2 + 1);  // and the relay: S_t cannot overtake it
      mbar_init(&sh.o_full[t], 1);
      mbar_init(&sh.o_free[t], SOFTMAX_WARPS / 2);
    }
    mbar_init(&sh.drain, 1);
    for (int s = 0; s < L::PAIRS; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
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

  // Steps are numbered through all items of the CTA (h). Keys and values travel in pairs: place h % PAIRS of
  // the ring takes V_{h-1} and K_h, which are used one after the other (P_{h-1} V_{h-1}, then S_h) and, once
  // S_h is there, are done with together.
  if (warp >= SOFTMAX_WARPS) {
    regs_dec<REGS_OTHER>();
    if (warp == WARP_TMA) {
      // ---------------------------------------------------------- TMA producer
      if (lane == 0) {
        const uint32_t q_bytes = static_cast<uint32_t>(Tile<DP>::BLOCKS * 128 * p.group * p.tokens);
        uint32_t q_loads[2] = {0, 0}, h = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t ph) {
          ok = ok && mbar_wait_abort(bar, ph, kErrWaitTimeoutProducer, &sh.abort);
          return ok;
        };
        Item prev{};
        bool any = false;
        // one pair: the values of the step before (prev, step v_step) and the keys of this one
        auto pair = [&](const Item* it, int j, int v_step) {
          const uint32_t slot = h % L::PAIRS;
          if (!wait(&sh.empty[slot], (h / L::PAIRS & 1) ^ 1)) return;
          mbar_arrive_expect_tx(&sh.full[slot], (any ? L::TILE : 0) + (it != nullptr ? L::TILE : 0));
          uint8_t* dst = sKV + slot * 2 * L::TILE;
          if (any) load_keys<DP>(dst, &tv, &sh.full[slot], prev.hk * p.vh, v_step, prev.b * p.vb);
          if (it != nullptr) load_keys<DP>(dst + L::TILE, &tk, &sh.full[slot], it->hk * p.kh, j, it->b * p.kb);
          ++h;
        };
        for (int index = blockIdx.x; ok && index < p.items; index += gridDim.x) {
          const Item it = item_at<BIAS>(p, index);
          for (int j = 0; ok && j < it.steps; ++j) {
            pair(&it, j, j > 0 ? j - 1 : any ? prev.steps - 1 : 0);
            if (j > 0) continue;
            prev = it;
            any = true;
            // (after the pair: who has seen an item's queries knows that the ring has come to its keys)
            for (int t = 0; ok && t < it.tiles; ++t) {
              if (q_loads[t] > 0 && !wait(&sh.q_free[t], (q_loads[t] - 1) & 1)) break;
              mbar_arrive_expect_tx(&sh.q_full[t], q_bytes);
              for (int c = 0; c < Tile<DP>::BLOCKS; ++c)
                tma_load_4d(sQ + t * L::TILE + c * Tile<DP>::BLOCK_BYTES, &tq, &sh.q_full[t], c * 64, it.hk * p.group,
                            static_cast<int32_t>(it.tok0 + t * p.tokens), it.b);
              ++q_loads[t];
            }
          }
        }
        if (ok && any) pair(nullptr, 0, prev.steps - 1);
        // every load issued by this thread lands before the CTA may exit
        for (int t = 0; t < 2; ++t)
          if (q_loads[t] > 0) mbar_wait(&sh.q_full[t], (q_loads[t] - 1) & 1, kErrWaitTimeoutDrain);
        for (uint32_t i = 0; i < L::PAIRS && i < h; ++i)
          mbar_wait(&sh.full[(h - 1 - i) % L::PAIRS], ((h - 1 - i) / L::PAIRS) & 1, kErrWaitTimeoutDrain);
      }
    } else if (warp == WARP_MMA) {
      // ---------------------------------------------------------- MMA issue
      // The whole warp goes through the steps and one lane issues: what the MMAs take as operands is then
      // uniform in the warp.
      const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0);
      const bool leader = elect_one();
      const uint64_t q_desc = smem_desc_sw128(smem_u32(sQ));
      const uint64_t k_desc = smem_desc_sw128(smem_u32(sKV) + L::TILE);
      const uint64_t v_desc = smem_desc_mn_sw128(smem_u32(sKV), Tile<DP>::BLOCK_BYTES);
      // steps in all, and of each tile steps, items whose queries are in use, items whose output is begun
      uint32_t h = 0, steps[2] = {0, 0}, q_items[2] = {0, 0}, o_items[2] = {0, 0};
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t ph) {
        const bool done = mbar_poll_abort(bar, ph, kErrWaitTimeoutMma, &sh.abort);
        ok = __all_sync(0xffffffffu, done) != 0 && ok;
        return ok;
      };
      auto full = [&](uint32_t n) { return wait(&sh.full[n % L::PAIRS], n / L::PAIRS & 1); };
      auto place = [](uint32_t n) { return n % L::PAIRS * (2 * L::TILE); };
      auto next_item = [&](int index, Item& it) {  // the first one from index on that has keys
        for (; index < p.items; index += gridDim.x) {
          it = item_at<BIAS>(p, index);
          if (it.steps > 0) break;
        }
        return index;
      };
      // S_t = Q_t K^T of an item's first step, from place n
      auto first_scores = [&](int t, uint32_t n) {
        if (!wait(&sh.q_full[t], q_items[t]++ & 1)) return;
        tc_fence_after();
        if (leader) {
          mma_scores<DP, BF16>(tm + col_s(t), smem_desc_at(q_desc, t * L::TILE), smem_desc_at(k_desc, place(n)));
          mma_commit(&sh.s_full[t]);
        }
        __syncwarp();
      };
      Item it, next;
      int index = next_item(blockIdx.x, it);
      if (index < p.items && full(0)) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (t < it.tiles) first_scores(t, 0);
      }
      while (ok && index < p.items) {
        index = next_item(index + gridDim.x, next);
        const int next_tiles = index < p.items ? next.tiles : 0;
        for (int j = 0; ok && j < it.steps; ++j, ++h) {
          const bool more = j + 1 < it.steps;
          if (!full(h + 1)) break;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (t < it.tiles) {
              // the last item's output has been read
              if (j == 0 && o_items[t]++ > 0 && !wait(&sh.o_free[t], o_items[t] & 1)) break;
              if (!wait(&sh.p_full[t], steps[t]++ & 1)) break;
              tc_fence_after();
              if (leader) {
                mma_values<DP, BF16>(tm + col_o(t), tm + col_s(t), smem_desc_at(v_desc, place(h + 1)), j != 0);
                if (more)
                  mma_scores<DP, BF16>(tm + col_s(t), smem_desc_at(q_desc, t * L::TILE), smem_desc_at(k_desc, place(h + 1)));
                mma_commit(more ? &sh.s_full[t] : &sh.o_full[t]);
              }
              __syncwarp();
            }
            if (!more && t < next_tiles) first_scores(t, h + 1);
          }
        }
        it = next;
      }
      if (leader) {
        mma_commit(&sh.drain);
        mbar_wait(&sh.drain, 0, kErrWaitTimeoutDrain);
      }
    } else if (warp == WARP_RELAY && lane == 0) {
      // ---------------------------------------------------------- pairs handed back to the producer
      // A tcgen05.commit holds the tensor cores up for about 120 cycles, so there is one a step (S_t ready,
      // hence Q K_h done, and before it P V_{h-1}: one thread issued them in order) instead of one for each
      // thing that is done with; this thread passes it on.
      uint32_t h = 0, steps[2] = {0, 0}, items[2] = {0, 0};
      int before = 0;  // tiles of the item before
      bool ok = true;
      for (int index = blockIdx.x; ok && index < p.items; index += gridDim.x) {
        const Item it = item_at<BIAS>(p, index);
        for (int j = 0; ok && j < it.steps; ++j, ++h) {
          if (j == 0) {  // the item before may have had a tile that this one does not have
            for (int t = 0; ok && t < before; ++t)
              ok = mbar_wait_abort(&sh.o_full[t], items[t]++ & 1, kErrWaitTimeoutMma, &sh.abort);
            before = it.tiles;
          }
          for (int t = 0; ok && t < it.tiles; ++t) {
            ok = mbar_wait_abort(&sh.s_full[t], steps[t]++ & 1, kErrWaitTimeoutMma, &sh.abort);
            mbar_arrive(&sh.p_full[t]);
            if (j + 1 == it.steps) mbar_arrive(&sh.q_free[t]);
          }
          if (ok) mbar_arrive(&sh.empty[h % L::PAIRS]);
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax of half a row, output
    regs_inc<REGS_SOFTMAX>();
    const int t = warp >> 3;
    const int half = (warp >> 2) & 1;  // of the keys of a tile, of the columns of O
    const int quarter = warp & 3;      // of the rows: the lanes of TMEM that the warp reaches
    const int row = quarter * 32 + lane;
    const int pair = 1 + 4 * t + quarter;  // barrier of a row's two halves
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_s = t_lane + col_s(t), t_o = t_lane + col_o(t) + half * (DP / 2);
    const float scale = BIAS ? 1.0f : p.scale2;
    // 128 rows need not be a whole number of tokens: what is left in the others has no say in what is done for all
    const bool real = row < p.group * p.tokens;
    // After a wait that failed the warp goes through its steps without work (every further wait fails at
    // once), so that both halves meet at each of their barriers.
    bool good = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool ok = mbar_wait_abort(bar, parity, kErrWaitTimeoutEpilogue, &sh.abort);
      good = __all_sync(0xffffffffu, ok) != 0 && good;
      tc_fence_after();
    };
    // The larger, or the sum, of a value of both halves of the rows.
    auto other = [&](float v) {
      sh.x[t][half][row] = v;
      named_barrier(pair, 64);
      v = sh.x[t][half ^ 1][row];
      named_barrier(pair, 64);  // both have read it before it is written again
      return v;
    };
    uint32_t steps = 0;  // of this tile before the item
    uint32_t h = 0;      // of both tiles before the item
    uint32_t items = 0;  // of this tile before the item
    Item next{};
    if (blockIdx.x < p.items) next = item_at<BIAS>(p, blockIdx.x);
#pragma unroll 1
    for (int index = blockIdx.x; index < p.items; index += gridDim.x) {
      const Item it = next;
      if (t >= it.tiles) {
        if (index + gridDim.x < p.items) next = item_at<BIAS>(p, index + gridDim.x);
        h += it.steps;
        continue;
      }
      float m = -INFINITY;
      float2 l2 = make_float2(0.0f, 0.0f);
#pragma unroll 1
      for (int j = 0; j < it.steps; ++j) {
        const int key0 = j * BN, left = it.keys - key0;
        uint32_t bits[2] = {0xffffffffu, 0xffffffffu};
        bool clear = false;
        if (BIAS || left < BN || p.keys.mask != nullptr)
          clear = !key_bits<BIAS, 2>(p, it.b, key0, left, 64 * half, row, lane, bits) && key0 + row < p.kv_len;
        wait(&sh.s_full[t], (steps + j) & 1);
        uint32_t r[64];
        tmem_ld_32x32b_x32(t_s + 64 * half, *reinterpret_cast<uint32_t(*)[32]>(r));
        tmem_ld_32x32b_x32(t_s + 64 * half + 32, *reinterpret_cast<uint32_t(*)[32]>(r + 32));
        tmem_ld_wait();
        reg_dep32(*reinterpret_cast<uint32_t(*)[32]>(r));
        reg_dep32(*reinterpret_cast<uint32_t(*)[32]>(r + 32));
        float(&y)[64] = reinterpret_cast<float(&)[64]>(r);
        mask_scores<BIAS, 64>(p, it.b, key0, 64 * half, bits, y);
        float sc = scale;
        const float peak = BIAS ? max_of<64>(y) : scale_if_large(y, max_of<64>(y), real, sc);
        // (the barrier also tells that both halves have read the scores that the weights go over)
        tc_fence_before();
        if (j == 0 || named_barrier_any(pair, 64, real && outgrown<T>(peak, sc, m))) {
          const float own = as_top<T>(peak, sc);
          const float m_new = fmaxf(m, fmaxf(own, other(own)));
          if (j > 0) {  // O holds P_0 V_0 + ... + P_{j-1} V_{j-1} (done before S_j)
            const float alpha = m_new == -INFINITY ? 1.0f : ex2_approx(m - m_new);
            l2 = mul2(l2, make_float2(alpha, alpha));
            rescale<DP / 2>(t_o, alpha);
          }
          m = m_new;
        }
        tc_fence_after();
        const float off = m == -INFINITY ? 0.0f : -m;
#pragma unroll
        for (int c = 0; c < 64; c += 32) {
          uint32_t w[16];
          l2 = add2(l2, weights<T>(y + c, sc, off, w));
          tmem_st_32x32b_x16(t_s + 32 * half + c / 2, w);
        }
        tmem_st_wait();
        if (__any_sync(0xffffffffu, clear)) {
          // Both tiles clear the same rows, each before its own second product. (After S_j, so that the
          // place's earlier pair is known to have come: a parity tells only two apart.)
          const uint32_t n = h + j + 1;
          wait(&sh.full[n % L::PAIRS], n / L::PAIRS & 1);
          if (clear && good) {
            uint4* v = reinterpret_cast<uint4*>(sKV + n % L::PAIRS * (2 * L::TILE) + row * 128 +
                                                half * (DP == 128 ? Tile<DP>::BLOCK_BYTES : 64));
#pragma unroll
            for (int e = 0; e < DP / 16; ++e) v[e] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[t]);
      }
      if (index + gridDim.x < p.items) next = item_at<BIAS>(p, index + gridDim.x);  // ahead of its use: it loads
      const float own_l = l2.x + l2.y, l = own_l + other(own_l);
      if (it.steps > 0) wait(&sh.o_full[t], items++ & 1);
      // 32 columns of the warp's 32 rows at a time through its own shared memory (16-byte chunk u of row
      // r at u ^ (r >> 1 & 3)), then 64-byte pieces of 8 rows a store
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint8_t* stage = smem + L::OFF_STAGING + warp * L::STAGING;
      const int64_t token0 = it.tok0 + t * p.tokens;
      const int tokens = p.q_len - token0 < p.tokens ? static_cast<int>(p.q_len - token0) : p.tokens;
      T* out = static_cast<T*>(p.out.data) + it.b * p.out.stride_b + token0 * p.out.stride_s + it.hk * p.group * p.out.stride_h;
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
            const int tok = token_of(p, tr);
            if (tok < tokens)
              *reinterpret_cast<uint4*>(out + tok * p.out.stride_s + (tr - tok * p.group) * p.out.stride_h + col) =
                  *reinterpret_cast<const uint4*>(stage + sr * 64 + ((chunk ^ (sr >> 1 & 3)) << 4));
          }
        }
      }
      steps += it.steps;
      h += it.steps;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == WARP_MMA) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

}  // namespace wide
}  // namespace xattn
}  // namespace slim
