// Cross attention: argument checks, the choice of kernel and the launches.
#include <cfloat>

#include "cross_attn_narrow.cuh"
#include "cross_attn_wide.cuh"

namespace slim {
namespace xattn {

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

// How a problem is laid over the SMs.
struct Plan {
  int group, tokens;
  int64_t q_tiles;
  int splits, per;            // 0: the wide kernel; else pieces of a row tile's keys, key tiles of each
  int rows;
  int64_t floats;             // of the pieces' results
};

// The cheapest layout by a count of steps, one row tile x one key tile in the narrow kernel (1.23 us).
// The wide kernel takes two row tiles x one key tile in 1.6 of them and moves half the keys and values: it
// wins as soon as there are enough pairs of row tiles for the SMs. An item's ends cost 1.
//
// Pieces cost join_kernel: 2.5 steps, 1 for every 700 rows (a block each) and 1 for every 4 MB of their sums, taken from
// captured calls at 80 shapes of 1 to 200 queries over 500 to 20000 keys, heads 8 to 32 of 64 and 128. A call outside of
// a graph also pays a second launch on the host, so they count 6 at least. At 4 x 1 query over 1500 keys x 16 heads of
// 64 that keeps one launch: 20 us on the device instead of 16 in two pieces, but 20 us a call instead of 26 when calls
// are issued one by one. 2 x 200 queries over 4000 keys x 24 heads: 47 us unsplit, 58 in three pieces.
inline double pieces_cost(int64_t s, int64_t tiles, int rows, int dp) {
  const double join = 2.5 + static_cast<double>(tiles * rows) / 700 +
                      static_cast<double>(narrow::split_floats(s, tiles, rows, dp)) / (1 << 20);
  return join > 6.0 ? join : 6.0;
}

inline Plan make_plan(int64_t batch, int64_t q_len, int64_t kv_len, int heads, int kv_heads, int dim) {
  Plan p{};
  p.group = heads / kv_heads;
  p.tokens = BM / p.group;
  p.q_tiles = (q_len + p.tokens - 1) / p.tokens;
  p.rows = p.group * static_cast<int>(q_len < p.tokens ? q_len : p.tokens);
  const int64_t nk = (kv_len + BN - 1) / BN, base = batch * kv_heads, tiles = base * p.q_tiles, sms = sm_count();
  const int64_t pairs = base * ((p.q_tiles + 1) / 2);
  const int dp = dim > 64 ? 128 : 64;
  double best = static_cast<double>((pairs + sms - 1) / sms) * (1.0 + 1.6 * static_cast<double>(nk));
  // The narrow kernel is considered up to 4 row tiles an SM, and for any number of them where a key head has a
  // single one, as the wide kernel's second tile would then be empty: one query over 2048 keys, 75 sequences of
  // 32 / 8 heads of 128, 131 us (wide 154); 100 queries over 300, 100 sequences of 8 heads, 47 us (55). With three row
  // tiles a key head it is no rule: 300 queries over 1000 keys x 296 heads 84 us (90), over 4000 x 2 x 148 heads of
  // 64 256 us (227).
  const int64_t most = p.q_tiles == 1 && tiles > 4 * sms ? tiles : 4 * sms;
  for (int64_t s = 1; s <= 128 && s <= (nk > 0 ? nk : 1) && tiles * s <= most; ++s) {
    const int64_t per = (nk + s - 1) / s;
    if (s > 1 && (s - 1) * per >= nk) continue;  // the last pieces would be empty
    double cost = static_cast<double>((tiles * s + sms - 1) / sms * (per + 1));
    if (s > 1) cost += pieces_cost(s, tiles, p.rows, dp);
    if (cost < best) {
      best = cost;
      p.splits = static_cast<int>(s);
      p.per = static_cast<int>(per);
    }
  }
  if (p.splits > 1) p.floats = narrow::split_floats(p.splits, tiles, p.rows, dp);
  return p;
}

template <typename Kernel>
cudaError_t prepare(Kernel kernel, size_t smem, PerDeviceOnce& once) {
  int dev = 0;
  cudaGetDevice(&dev);
  return once.run(dev, [=] {
    cudaFuncAttributes attr;
    cudaError_t e = cudaFuncGetAttributes(&attr, kernel);
    if (e == cudaSuccess && attr.numRegs < REGS) e = cudaErrorInvalidConfiguration;  // the shares would not fit
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
  });
}

template <typename T, int DP, bool BIAS>
cudaError_t launch(const Params& p, const Plan& plan, float* partial, cudaStream_t st) {
  constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
  CUtensorMap mq, mk, mv;
  // without keys k and v may be null: their maps are never used
  const bool any = p.kv_len > 0;
  if (!make_map(&mq, BF16, p.q, p.batch, p.q_len, p.heads, p.dim, plan.group, plan.tokens) ||
      !make_map(&mk, BF16, any ? p.k : p.q, p.batch, any ? p.kv_len : 1, any ? p.kv_heads : 1, p.dim, 1, BN) ||
      !make_map(&mv, BF16, any ? p.v : p.q, p.batch, any ? p.kv_len : 1, any ? p.kv_heads : 1, p.dim, 1, BN))
    return cudaErrorInvalidValue;
  const int64_t per_head = plan.splits > 0 ? plan.q_tiles * plan.splits : (plan.q_tiles + 1) / 2;
  const int64_t items = per_head * p.kv_heads * p.batch;
  const TileParams tp{p.out, p.q_len, p.kv_len, p.kv_heads, p.dim, plan.group, plan.tokens,
                      static_cast<uint32_t>((65536 + plan.group - 1) / plan.group), p.k.stride_b != 0,
                      p.k.stride_h != 0, p.v.stride_b != 0, p.v.stride_h != 0, p.scale2, p.keys,
                      static_cast<int>(items), static_cast<int>(per_head), plan.splits, plan.per, plan.rows, partial};
  const int64_t sms = sm_count();
  const unsigned grid = static_cast<unsigned>(items < sms ? items : sms);
  static PerDeviceOnce once[3];
  cudaError_t e;
  auto run = [&](auto kernel, size_t smem, PerDeviceOnce& o) {
    cudaError_t err = prepare(kernel, smem, o);
    if (err != cudaSuccess) return err;
    kernel<<<grid, THREADS, smem, st>>>(mq, mk, mv, tp);
    err = cudaGetLastError();
    if (err == cudaSuccess) note_launch();
    return err;
  };
  if (plan.splits == 0) return run(wide::wide_kernel<T, DP, BIAS>, wide::smem_bytes<DP>(), once[0]);
  if (plan.splits == 1) return run(narrow::narrow_kernel<T, DP, BIAS, false>, narrow::smem_bytes<DP>(), once[1]);
  if ((e = run(narrow::narrow_kernel<T, DP, BIAS, true>, narrow::smem_bytes<DP>(), once[2])) != cudaSuccess) return e;
  const int64_t tiles = items / plan.splits;
  narrow::join_kernel<T, DP><<<static_cast<unsigned>(tiles * plan.rows), 256, 0, st>>>(
      partial, p.out, p.q_len, plan.group, plan.tokens, plan.rows, static_cast<int>(plan.q_tiles), p.kv_heads,
      plan.splits, tiles, p.dim);
  if ((e = cudaGetLastError()) != cudaSuccess) return e;
  note_launch();
  return cudaSuccess;
}

template <typename T, int DP>
cudaError_t launch(const Params& p, const Plan& plan, float* partial, cudaStream_t st) {
  return p.keys.bias != nullptr ? launch<T, DP, true>(p, plan, partial, st) : launch<T, DP, false>(p, plan, partial, st);
}

struct Workspace {
  int64_t bias, n_keys, partial, total, pitch;
};

static Workspace workspace(int64_t batch, int64_t kv_len, bool additive, const Plan& plan) {
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
      (q_len + tokens - 1) / tokens * kv_heads * (batch < 1 ? 1 : batch) >= (int64_t{1} << 31) - 1024)
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
  const xattn::Plan plan = xattn::make_plan(batch, q_len, kv_len, heads, kv_heads, dim);
  *bytes = static_cast<uint64_t>(xattn::workspace(batch, kv_len, additive != 0, plan).total);
  return SLIM_OK;
}

int slim_cross_attn_layout(int64_t batch, int64_t q_len, int64_t kv_len, int heads, int kv_heads, int dim, int* pieces,
                           int* key_tiles) {
  const int rc = xattn::checks(batch, q_len, kv_len, heads, kv_heads, dim);
  if (rc != SLIM_OK) return rc;
  if (pieces == nullptr || key_tiles == nullptr) return fail(SLIM_ERR_NULL, "pieces/key_tiles is NULL");
  const xattn::Plan plan = xattn::make_plan(batch, q_len, kv_len, heads, kv_heads, dim);
  *pieces = plan.splits;
  *key_tiles = plan.splits > 0 ? plan.per : static_cast<int>((kv_len + xattn::KEY_TILE - 1) / xattn::KEY_TILE);
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
  if (!(scale > 0.0f) || !(scale * xattn::kLog2e <= FLT_MAX)) return fail(SLIM_ERR_SHAPE, "scale must be positive and finite");
  if (batch == 0 || q_len == 0) return SLIM_OK;
  if (q == nullptr || k == nullptr || v == nullptr || out == nullptr || q->data == nullptr || out->data == nullptr ||
      (kv_len > 0 && (k->data == nullptr || v->data == nullptr)))
    return fail(SLIM_ERR_NULL, "q/k/v/out is NULL");
  if (!xattn::view_ok(q, batch, q_len, heads, false) || !xattn::view_ok(out, batch, q_len, heads, false) ||
      (kv_len > 0 && (!xattn::view_ok(k, batch, kv_len, kv_heads, true) || !xattn::view_ok(v, batch, kv_len, kv_heads, true))))
    return fail(SLIM_ERR_ALIGN, "rows of q/k/v/out must be 16-byte aligned with positive strides (0 for shared k/v)");
  const bool additive = kv_len > 0 && mask != nullptr && mask_type != SLIM_MASK_BOOL;
  const xattn::Plan plan = xattn::make_plan(batch, q_len, kv_len, heads, kv_heads, dim);
  const xattn::Workspace w = xattn::workspace(batch, kv_len, additive, plan);
  if (workspace_bytes < static_cast<uint64_t>(w.total))
    return fail(SLIM_ERR_SHAPE, "workspace of %llu bytes is smaller than the %lld needed",
                static_cast<unsigned long long>(workspace_bytes), static_cast<long long>(w.total));
  if (w.total > 0 && ws == nullptr) return fail(SLIM_ERR_NULL, "workspace is NULL");
  if (!aligned16(ws)) return fail(SLIM_ERR_ALIGN, "workspace must be 16-byte aligned");
  if ((rc = check_arch()) != SLIM_OK) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint8_t* base = static_cast<uint8_t*>(ws);
  xattn::Params p{*q, *k, *v, *out, batch, q_len, kv_len, heads, kv_heads, dim, scale * xattn::kLog2e, {}};
  float* partial = plan.floats > 0 ? reinterpret_cast<float*>(base + w.partial) : nullptr;
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
    e = dim > 64 ? xattn::launch<__nv_bfloat16, 128>(p, plan, partial, st) : xattn::launch<__nv_bfloat16, 64>(p, plan, partial, st);
  else
    e = dim > 64 ? xattn::launch<__half, 128>(p, plan, partial, st) : xattn::launch<__half, 64>(p, plan, partial, st);
  if (e != cudaSuccess) return cuda_fail(e, "cross attention launch");
  return SLIM_OK;
}

}  // extern "C"
