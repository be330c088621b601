// Cross attention, few row tiles: one a CTA, and if there are still too few of them (SPLIT) the keys of
// a row tile cut into pieces that lie on several SMs; the pieces' sums go to memory and join_kernel
// joins them.
#pragma once

#include "cross_attn.cuh"

namespace slim {
namespace xattn {
namespace narrow {

// Persistent CTAs, one per SM. An item is a row tile with its keys or, SPLIT, a range of them; a CTA runs
// its items' steps (key tiles of 128) as one stream, so that the next item's loads and scores overlap the
// last one's end. With many keys bound by reading them: a step's 64 KB (128 elements) may take 1.5 us, its
// work takes 1.25 (one token over 131071 keys, 8 x 4 heads: 104 us with the join,
// 5.2 TB/s).
// 20 warps, S and the weights P twice in TMEM (steps g and g + 1), O once:
//   warps 0..15  softmax, a quarter row (32 keys) a thread; weights and maxima as in the wide kernel. An
//                item's sums leave after the next item's first step, when its last product is long done.
//   warp 16      TMA: queries (two buffers), keys and values in the order of their use
//   warp 17      the MMAs: S_0, S_1, then O += P_g V_g and S_{g+2} = Q K_{g+2}^T; one commit a step
//   warp 18      hands what S_g's commit shows to be done (Q K_g, P_{g-2} V_{g-2}) back to the producer
constexpr int WARP_TMA = 16, WARP_MMA = 17, WARP_RELAY = 18;
__device__ __forceinline__ constexpr uint32_t col_s(uint32_t g) { return (g & 1) * 128u; }        // scores
__device__ __forceinline__ constexpr uint32_t col_p(uint32_t g) { return 256u + (g & 1) * 64u; }  // weights
constexpr uint32_t COL_O = 384;                                                                  // output

template <int DP>
struct Layout {
  static constexpr int TILE = Tile<DP>::BYTES;
  static constexpr int PAIRS = DP == 64 ? 4 : 2;  // ring places of a V and a K tile
  static constexpr int OUT_COLS = DP / 4;         // columns of the output a softmax warp writes
  static constexpr int OFF_KV = 2 * TILE;
  static constexpr int STAGING = 32 * 16 * 2;     // a softmax warp's: 32 rows x 16 columns of the output
  static constexpr int OFF_STAGING = OFF_KV + PAIRS * 2 * TILE;
  static constexpr int OFF_SH = OFF_STAGING + SOFTMAX_WARPS * STAGING;
};

template <int PAIRS>
struct Shared {
  uint64_t q_full[2], q_free[2];
  uint64_t full[PAIRS], empty[PAIRS];
  uint64_t s_full[2], p_full[2], o_free;
  uint64_t drain;
  uint32_t tmem_base;
  volatile int abort;
  float x[2][4][BM];  // values of a row's four quarters, two exchanges
};

template <int DP>
constexpr size_t smem_bytes() {
  static_assert(Layout<DP>::OFF_SH + sizeof(Shared<Layout<DP>::PAIRS>) <= 232448, "shared memory");
  return Layout<DP>::OFF_SH + sizeof(Shared<Layout<DP>::PAIRS>);
}

struct Item {
  int b, hk, split, tile0, steps, keys;  // steps over key tiles from tile0 on
  int64_t tok0;
};

template <bool BIAS>
__device__ __forceinline__ Item item_at(const TileParams& p, int index) {
  Item it;
  const int head = index / p.per_head, x = index - head * p.per_head;
  it.b = head / p.kv_heads;
  it.hk = head - it.b * p.kv_heads;
  const int q_tile = x / p.splits;
  it.split = x - q_tile * p.splits;
  it.tok0 = static_cast<int64_t>(q_tile) * p.tokens;
  it.keys = keys_of<BIAS>(p, it.b);
  const int nk = (it.keys + BN - 1) / BN;
  it.tile0 = it.split * p.per;
  it.steps = nk <= it.tile0 ? 0 : nk - it.tile0 < p.per ? nk - it.tile0 : p.per;
  return it;
}

// A position in the stream of this CTA's steps.
template <bool BIAS>
struct Cursor {
  const TileParams& p;
  int index, j = 0;
  uint32_t items = 0;  // items with steps before this one
  Item it;
  bool valid;
  __device__ __forceinline__ explicit Cursor(const TileParams& params) : p(params), index(blockIdx.x) { find(); }
  __device__ __forceinline__ void find() {
    valid = false;
    for (; index < p.items; index += gridDim.x) {
      it = item_at<BIAS>(p, index);
      if (it.steps > 0) {
        valid = true;
        return;
      }
    }
  }
  __device__ __forceinline__ void next() {
    if (++j < it.steps) return;
    j = 0;
    ++items;
    index += gridDim.x;
    find();
  }
};

// Partial results of `parts` pieces of `tiles` tiles of `rows` rows, in floats: (m, l) pairs, then from
// split_o() on (a multiple of 16 bytes) the O rows.
__host__ __device__ inline int64_t split_o(int64_t parts, int64_t tiles, int64_t rows) {
  return (2 * parts * tiles * rows + 3) & ~int64_t{3};
}
__host__ __device__ inline int64_t split_floats(int64_t parts, int64_t tiles, int64_t rows, int dp) {
  return split_o(parts, tiles, rows) + parts * tiles * rows * dp;
}

template <typename T, int DP, bool BIAS, bool SPLIT>
__global__ void __launch_bounds__(THREADS, 1)
narrow_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
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
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sh.q_full[i], 1);
      mbar_init(&sh.q_free[i], 1);
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.p_full[i], SOFTMAX_WARPS + 1);  // and the relay: S_{g+2} cannot overtake it
    }
    for (int s = 0; s < L::PAIRS; ++s) {
      mbar_init(&sh.full[s], 1);
      mbar_init(&sh.empty[s], 1);
    }
    mbar_init(&sh.o_free, SOFTMAX_WARPS);
    mbar_init(&sh.drain, 1);
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
    // Keys and values travel in pairs: place h % PAIRS of the ring takes V_{h-2} and K_h, which are used one
    // after the other (P_{h-2} V_{h-2}, S_h) and, once S_h is there, are done with together.
    if (warp == WARP_TMA) {
      // ---------------------------------------------------------- TMA producer
      if (lane == 0) {
        const uint32_t q_bytes = static_cast<uint32_t>(Tile<DP>::BLOCKS * 128 * p.group * p.tokens);
        uint32_t q_loads = 0, h = 0;
        bool ok = true;
        auto wait = [&](uint64_t* bar, uint32_t ph) {
          ok = ok && mbar_wait_abort(bar, ph, kErrWaitTimeoutProducer, &sh.abort);
          return ok;
        };
        Cursor<BIAS> kc(p), vc(p);
        for (; kc.valid || vc.valid; ++h) {
          const uint32_t slot = h % L::PAIRS;
          const bool with_v = h >= 2, with_k = kc.valid;
          if (h >= 2 && !vc.valid) break;
          if (with_k && kc.j == 0) {
            const uint32_t i = kc.items & 1;
            if (kc.items > 1 && !wait(&sh.q_free[i], ((kc.items >> 1) - 1) & 1)) break;
            mbar_arrive_expect_tx(&sh.q_full[i], q_bytes);
            for (int c = 0; c < Tile<DP>::BLOCKS; ++c)
              tma_load_4d(sQ + i * L::TILE + c * Tile<DP>::BLOCK_BYTES, &tq, &sh.q_full[i], c * 64, kc.it.hk * p.group,
                          static_cast<int32_t>(kc.it.tok0), kc.it.b);
            ++q_loads;
          }
          if (!wait(&sh.empty[slot], (h / L::PAIRS & 1) ^ 1)) break;
          mbar_arrive_expect_tx(&sh.full[slot], (with_v ? L::TILE : 0) + (with_k ? L::TILE : 0));
          uint8_t* dst = sKV + slot * 2 * L::TILE;
          if (with_v) {
            load_keys<DP>(dst, &tv, &sh.full[slot], vc.it.hk * p.vh, vc.it.tile0 + vc.j, vc.it.b * p.vb);
            vc.next();
          }
          if (with_k) {
            load_keys<DP>(dst + L::TILE, &tk, &sh.full[slot], kc.it.hk * p.kh, kc.it.tile0 + kc.j, kc.it.b * p.kb);
            kc.next();
          }
        }
        // every load issued by this thread lands before the CTA may exit
        for (uint32_t i = 0; i < 2 && i < q_loads; ++i)
          mbar_wait(&sh.q_full[(q_loads - 1 - i) & 1], ((q_loads - 1 - i) >> 1) & 1, kErrWaitTimeoutDrain);
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
      bool ok = true;
      auto wait = [&](uint64_t* bar, uint32_t ph) {
        const bool done = mbar_poll_abort(bar, ph, kErrWaitTimeoutMma, &sh.abort);
        ok = __all_sync(0xffffffffu, done) != 0 && ok;
        return ok;
      };
      Cursor<BIAS> qc(p), pc(p);
      auto ready = [&](uint32_t h) {  // the pair, and the queries of a new item
        return wait(&sh.full[h % L::PAIRS], h / L::PAIRS & 1) &&
               (!qc.valid || qc.j > 0 || wait(&sh.q_full[qc.items & 1], qc.items >> 1 & 1));
      };
      auto qk = [&](uint32_t h) {
        if (leader) {
          mma_scores<DP, BF16>(tm + col_s(h), smem_desc_at(q_desc, (qc.items & 1) * L::TILE),
                               smem_desc_at(k_desc, h % L::PAIRS * (2 * L::TILE)));
          mma_commit(&sh.s_full[h & 1]);
        }
        __syncwarp();
        qc.next();
      };
      for (uint32_t h = 0; h < 2 && qc.valid && ready(h); ++h) {
        tc_fence_after();
        qk(h);
      }
      for (uint32_t g = 0; ok && pc.valid; ++g) {
        if (!ready(g + 2)) break;
        // the last item's output has been read
        if (pc.j == 0 && pc.items > 0 && !wait(&sh.o_free, (pc.items - 1) & 1)) break;
        if (!wait(&sh.p_full[g & 1], g >> 1 & 1)) break;
        tc_fence_after();
        if (leader) {
          mma_values<DP, BF16>(tm + COL_O, tm + col_p(g), smem_desc_at(v_desc, (g + 2) % L::PAIRS * (2 * L::TILE)), pc.j != 0);
          if (!qc.valid) mma_commit(&sh.s_full[g & 1]);  // S_{g+2} stands for P_g V_g being done in any case
        }
        __syncwarp();
        if (qc.valid) qk(g + 2);
        pc.next();
      }
      if (leader) {
        mma_commit(&sh.drain);
        mbar_wait(&sh.drain, 0, kErrWaitTimeoutDrain);
      }
    } else if (warp == WARP_RELAY) {
      // ---------------------------------------------------------- pairs handed back to the producer
      // A tcgen05.commit holds the tensor cores up for about 120 cycles, so there is one a step instead of
      // one for each thing that is done with.
      if (lane == 0) {
        Cursor<BIAS> c(p);
        for (uint32_t g = 0; c.valid; ++g) {
          if (!mbar_wait_abort(&sh.s_full[g & 1], g >> 1 & 1, kErrWaitTimeoutMma, &sh.abort)) break;
          mbar_arrive(&sh.empty[g % L::PAIRS]);
          if (c.j + 1 == c.it.steps) mbar_arrive(&sh.q_free[c.items & 1]);
          mbar_arrive(&sh.p_full[g & 1]);
          c.next();
        }
      }
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax of a quarter row, output
    regs_inc<REGS_SOFTMAX>();
    const int quarter = warp & 3;  // of the rows: the lanes of TMEM that the warp reaches
    const int part = warp >> 2;    // of the keys of a tile, of the columns of O
    const int row = quarter * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quarter * 32) << 16);
    const uint32_t t_o = t_lane + COL_O + part * L::OUT_COLS;
    const float scale = BIAS ? 1.0f : p.scale2;
    // few rows: warps whose rows do not exist only keep step
    const bool live = quarter * 32 < p.rows;
    // 128 rows need not be a whole number of tokens: what is left in the others has no say in what is done for all
    const bool real = row < p.group * p.tokens;
    // After a wait that failed the warp goes through its steps without work (every further wait fails at
    // once), so that a row's four warps meet at each of their barriers.
    bool good = true;
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      const bool ok = mbar_wait_abort(bar, parity, kErrWaitTimeoutEpilogue, &sh.abort);
      good = __all_sync(0xffffffffu, ok) != 0 && good;
    };
    // S_g, or (g beyond the last step) P_{g-2} V_{g-2} done
    auto wait_s = [&](uint32_t g) {
      wait(&sh.s_full[g & 1], (g >> 1) & 1);
      tc_fence_after();
    };
    // A value of each of the row's four quarters; two buffers, as a warp can be one exchange ahead.
    uint32_t exchanges = 0;
    auto exchange = [&](float v) {
      float(*x)[BM] = sh.x[exchanges++ & 1];
      x[part][row] = v;
      named_barrier(1 + quarter, 128);
      return make_float4(x[0][row], x[1][row], x[2][row], x[3][row]);
    };

    // Items without keys: zeros, or a piece with nothing in it.
#pragma unroll 1
    for (int index = blockIdx.x; index < p.items; index += gridDim.x) {
      const Item it = item_at<BIAS>(p, index);
      if (it.steps > 0) continue;
      const int tok = row / p.group, head = it.hk * p.group + row - tok * p.group;
      const int64_t token = it.tok0 + tok;
      if (SPLIT) {
        const int64_t at = (it.split * static_cast<int64_t>(p.items / p.splits) + index / p.splits) * p.rows + row;
        if (part == 0 && row < p.rows) reinterpret_cast<float2*>(p.partial)[at] = make_float2(-INFINITY, 0.0f);
      } else if (tok < p.tokens && token < p.q_len) {
        T* out = static_cast<T*>(p.out.data) + it.b * p.out.stride_b + token * p.out.stride_s + head * p.out.stride_h;
        for (int k = part * L::OUT_COLS; k < (part + 1) * L::OUT_COLS && k < p.dim; k += 8)
          *reinterpret_cast<uint4*>(out + k) = make_uint4(0, 0, 0, 0);
      }
    }

    // The sums of an item whose last step was g.
    auto finish = [&](const Item& it, int index, uint32_t g, float m, float2 l2) {
      const float4 ls = exchange(l2.x + l2.y);
      wait_s(g + 2);
      uint32_t r[L::OUT_COLS];
      if constexpr (DP == 128) {
        tmem_ld_32x32b_x32(t_o, r);
      } else {
        tmem_ld_32x32b_x16(t_o, r);
      }
      tmem_ld_wait();
#pragma unroll
      for (int c = 0; c < L::OUT_COLS; c += 16) reg_dep16(*reinterpret_cast<uint32_t(*)[16]>(r + c));
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.o_free);
      const float l = (ls.x + ls.y) + (ls.z + ls.w);
      if (SPLIT) {
        if (!good || row >= p.rows) return;
        const int64_t row_tiles = p.items / p.splits;
        const int64_t at = (it.split * row_tiles + index / p.splits) * p.rows + row;
        if (part == 0) reinterpret_cast<float2*>(p.partial)[at] = make_float2(m, l);
        uint4* o = reinterpret_cast<uint4*>(p.partial + split_o(p.splits, row_tiles, p.rows) + at * DP + part * L::OUT_COLS);
#pragma unroll
        for (int u = 0; u < L::OUT_COLS / 4; ++u) o[u] = make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]);
        return;
      }
      // 16 columns of the warp's 32 rows at a time through its own shared memory (16-byte chunk u of row r
      // at u ^ (r >> 2 & 1)), then 32-byte pieces of 16 rows a store
      const float inv = l == 0.0f ? 0.0f : 1.0f / l;
      uint8_t* stage = smem + L::OFF_STAGING + warp * L::STAGING;
      const int tokens = p.q_len - it.tok0 < p.tokens ? static_cast<int>(p.q_len - it.tok0) : p.tokens;
      T* out = static_cast<T*>(p.out.data) + it.b * p.out.stride_b + it.tok0 * p.out.stride_s + it.hk * p.group * p.out.stride_h;
#pragma unroll
      for (int c = 0; c < L::OUT_COLS; c += 16) {
        __syncwarp();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          uint32_t w[4];
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = pack2<T>(__uint_as_float(r[c + 8 * u + 2 * e]) * inv, __uint_as_float(r[c + 8 * u + 2 * e + 1]) * inv);
          *reinterpret_cast<uint4*>(stage + lane * 32 + ((u ^ (lane >> 2 & 1)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        __syncwarp();
        const int chunk = lane & 1, col = part * L::OUT_COLS + c + chunk * 8;
        if (good && col < p.dim) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int sr = i * 16 + (lane >> 1), tr = quarter * 32 + sr;
            const int tok = token_of(p, tr);
            if (tok < tokens)
              *reinterpret_cast<uint4*>(out + tok * p.out.stride_s + (tr - tok * p.group) * p.out.stride_h + col) =
                  *reinterpret_cast<const uint4*>(stage + sr * 32 + ((chunk ^ (sr >> 2 & 1)) << 4));
          }
        }
      }
    };

    bool pending = false;      // an item whose output is still to leave
    Item last;
    int last_index = 0;
    float last_m = 0.0f, m = -INFINITY;
    float2 last_l = make_float2(0.0f, 0.0f), l2 = make_float2(0.0f, 0.0f);
    Cursor<BIAS> c(p);
#pragma unroll 1
    for (uint32_t g = 0;; ++g) {
      if (c.valid) {
        const int key0 = (c.it.tile0 + c.j) * BN, left = c.it.keys - key0;
        uint32_t bits[1] = {0xffffffffu};
        bool clear = false;
        if (BIAS || left < BN || p.keys.mask != nullptr)
          clear = !key_bits<BIAS, 1>(p, c.it.b, key0, left, 32 * part, row, lane, bits) && key0 + row < p.kv_len;
        if (c.j == 0) {
          m = -INFINITY;
          l2 = make_float2(0.0f, 0.0f);
        }
        wait_s(g);  // also: P_{g-2} V_{g-2} is done and its weights may be overwritten
        if (live) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(t_lane + col_s(g) + 32 * part, r);
          tmem_ld_wait();
          reg_dep32(r);
          float(&y)[32] = reinterpret_cast<float(&)[32]>(r);
          mask_scores<BIAS, 32>(p, c.it.b, key0, 32 * part, bits, y);
          float sc = scale;
          const float peak = BIAS ? max_of<32>(y) : scale_if_large(y, max_of<32>(y), real, sc);
          // Weights with the maximum in use, and once more with a new one if some row's has grown too far
          // (an item's first step has none to start with).
          bool fresh = c.j == 0;
          float2 add;
#pragma unroll 1
          while (true) {
            if (fresh) {
              const float4 tops = exchange(as_top<T>(peak, sc));
              const float m_new = fmaxf(m, fmaxf(fmaxf(tops.x, tops.y), fmaxf(tops.z, tops.w)));
              if (c.j > 0) {
                wait_s(g + 1);  // P_{g-1} V_{g-1} done
                const float alpha = m_new == -INFINITY ? 1.0f : ex2_approx(m - m_new);
                l2 = mul2(l2, make_float2(alpha, alpha));
                rescale<L::OUT_COLS>(t_o, alpha);
              }
              m = m_new;
            }
            uint32_t w[16];
            add = weights<T>(y, sc, m == -INFINITY ? 0.0f : -m, w);
            tmem_st_32x32b_x16(t_lane + col_p(g) + 16 * part, w);
            if (fresh) break;
            fresh = named_barrier_any(1 + quarter, 128, real && outgrown<T>(peak, sc, m));
            if (!fresh) break;
            tmem_st_wait();  // stores are not ordered: these weights have landed before the next go over them
          }
          l2 = add2(l2, add);
          tmem_st_wait();
        }
        // (after S_g, so that the place's earlier pair is known to have come: a parity tells two apart)
        if (__any_sync(0xffffffffu, clear)) {
          wait(&sh.full[(g + 2) % L::PAIRS], (g + 2) / L::PAIRS & 1);
          if (clear && good) {
            uint4* v = reinterpret_cast<uint4*>(sKV + (g + 2) % L::PAIRS * (2 * L::TILE) + row * 128 +
                                                (DP == 128 ? (part >> 1) * Tile<DP>::BLOCK_BYTES + (part & 1) * 64 : part * 32));
#pragma unroll
            for (int e = 0; e < DP / 32; ++e) v[e] = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[g & 1]);
      }
      if (pending && (!c.valid || c.j == 0)) {
        finish(last, last_index, g - 1, last_m, last_l);
        pending = false;
      }
      if (!c.valid) break;
      if (c.j + 1 == c.it.steps) {
        pending = true;
        last = c.it;
        last_index = c.index;
        last_m = m;
        last_l = l2;
      }
      c.next();
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
__global__ void __launch_bounds__(256) join_kernel(const float* __restrict__ partial, slim_view out, int64_t q_len,
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
  const float* o = partial + split_o(parts, items, rows) + (item * rows + row) * DP + lane * E;
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

}  // namespace narrow
}  // namespace xattn
}  // namespace slim
