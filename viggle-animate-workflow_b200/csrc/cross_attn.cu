// Cross attention: queries of one sequence over the keys and values of another length.
//
//   o = softmax(scale q k^T + bias) v,   q [B, Sq, H, D], k and v [B, Skv, Hkv, D], Hkv | H
//
// bias is per key (a boolean or additive mask, lengths of padded sequences); -inf excludes a key,
// whatever stands in its k and v, and a row without keys is 0. Scores, the running maximum and the
// sum of the softmax are fp32; logits are kept in base 2 (scale * log2 e folded into one factor).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cfloat>

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

// ---------------------------------------------------------------- one warp per query row
template <typename T>
__device__ __forceinline__ float load_f(const T* p);
template <>
__device__ __forceinline__ float load_f(const __nv_bfloat16* p) { return __bfloat162float(*p); }
template <>
__device__ __forceinline__ float load_f(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store_f(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_f(__half* p, float v) { *p = __float2half_rn(v); }

template <typename T>
__global__ void __launch_bounds__(256) row_kernel(const Params p) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = p.batch * p.q_len * p.heads;
  const int64_t step = static_cast<int64_t>(gridDim.x) * (blockDim.x >> 5);
  for (int64_t r = static_cast<int64_t>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); r < rows; r += step) {
    const int h = static_cast<int>(r % p.heads);
    const int64_t s = r / p.heads % p.q_len;
    const int64_t b = r / p.heads / p.q_len;
    const int hk = h / (p.heads / p.kv_heads);
    const T* q = static_cast<const T*>(p.q.data) + b * p.q.stride_b + s * p.q.stride_s + h * p.q.stride_h;
    const T* k = static_cast<const T*>(p.k.data) + b * p.k.stride_b + hk * p.k.stride_h;
    const T* v = static_cast<const T*>(p.v.data) + b * p.v.stride_b + hk * p.v.stride_h;
    T* out = static_cast<T*>(p.out.data) + b * p.out.stride_b + s * p.out.stride_s + h * p.out.stride_h;
    const int64_t keys = p.n_keys != nullptr ? p.n_keys[b] : p.kv_len;
    float x[MAX_DIM / 32], o[MAX_DIM / 32] = {};
    for (int e = 0; e < MAX_DIM / 32; ++e) x[e] = lane + 32 * e < p.dim ? load_f<T>(q + lane + 32 * e) : 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int64_t i = 0; i < keys; ++i) {
      const float add = p.bias != nullptr ? p.bias[b * p.bias_pitch + i] : 0.0f;
      if (add == -INFINITY) continue;
      float y = 0.0f;
      for (int e = 0; e < MAX_DIM / 32; ++e)
        if (lane + 32 * e < p.dim) y = fmaf(x[e], load_f<T>(k + i * p.k.stride_s + lane + 32 * e), y);
      for (int sh = 16; sh >= 1; sh >>= 1) y += __shfl_xor_sync(0xffffffffu, y, sh);
      y = fmaf(y, p.scale2, add);
      const float top = fmaxf(m, y);
      const float keep = exp2f(m - top), w = exp2f(y - top);
      l = fmaf(l, keep, w);
      m = top;
      for (int e = 0; e < MAX_DIM / 32; ++e)
        if (lane + 32 * e < p.dim) o[e] = fmaf(o[e], keep, w * load_f<T>(v + i * p.v.stride_s + lane + 32 * e));
    }
    for (int e = 0; e < MAX_DIM / 32; ++e)
      if (lane + 32 * e < p.dim) store_f(out + lane + 32 * e, l == 0.0f ? 0.0f : o[e] / l);
  }
}

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

static bool view_ok(const slim_view* v, int64_t batch, int64_t seq, int heads) {
  return aligned16(v->data) && (batch == 1 || v->stride_b % 8 == 0) && (seq == 1 || v->stride_s % 8 == 0) &&
         (heads == 1 || v->stride_h % 8 == 0);
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
  if (!xattn::view_ok(q, batch, q_len, heads) || !xattn::view_ok(out, batch, q_len, heads) ||
      (kv_len > 0 && (!xattn::view_ok(k, batch, kv_len, kv_heads) || !xattn::view_ok(v, batch, kv_len, kv_heads))))
    return fail(SLIM_ERR_ALIGN, "rows of q/k/v/out must be 16-byte aligned");
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
  const int64_t blocks = (batch * q_len * heads + 7) / 8;
  const unsigned grid = static_cast<unsigned>(blocks < (1 << 20) ? blocks : (1 << 20));
  if (dtype == kBF16)
    xattn::row_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>(p);
  else
    xattn::row_kernel<__half><<<grid, 256, 0, st>>>(p);
  if ((e = cudaGetLastError()) != cudaSuccess) return cuda_fail(e, "cross attention launch");
  note_launch();
  return SLIM_OK;
}

}  // extern "C"
