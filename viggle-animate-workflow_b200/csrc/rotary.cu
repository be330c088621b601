// Rotary positions applied to queries and keys (strided views, in place or not).
//
// Token t turns pair j of its first `rot` elements by the angle a = pos[t] * inv_freq[j]:
//   (x, y) -> magnitude * (x cos a - y sin a, x sin a + y cos a)
// with the pair at elements (j, j + rot/2) ("half") or (2j, 2j + 1) ("interleaved"); elements
// from `rot` on pass through. With several position axes pair j takes the axis of its section.
//
// Six flops a pair against 8 (bf16) or 16 (fp32) bytes: bound by HBM. One block takes a few
// tokens: it computes their cos and sin once into shared memory (the angle reduced to turns in
// fp64, because pos * inv_freq in fp32 is off by up to 2^-24 of the whole angle, not of a turn),
// then all heads of q and k go through in 16-byte accesses. The products and sums are fp32,
// rounded once to the element type. 30026 tokens x 112 heads x 128, 96 of them turned, bf16 rows of
// a packed buffer: 272 us in a single launch (6.3 TB/s), 275 to 281 one call after the other (6.1 to
// 6.3), 256 in place; by single elements instead of words a single launch took 293 us, as the kernel is then close
// to being bound by instruction issue (70 % of the slots, by words 63 %).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/slimdit_b200.h"
#include "slim_kernels.h"

namespace slim {
namespace rope {

constexpr int THREADS = 256;
constexpr int BLOCKS = 8;           // blocks per SM: 32 registers a thread
constexpr int MAX_TOKENS = 16;      // tokens per block
constexpr int MAX_TABLE = 1024;     // (token, pair) entries of cos/sin in shared memory

struct Params {
  slim_view q, q_out, k, k_out;
  int heads_q, heads;               // heads of q, heads of q and k together
  int64_t batch, seq;
  int dim, rot, pairs;              // pairs = rot / 2
  const void* pos;
  int pos32;
  int64_t pos_b, pos_s, pos_a;
  const float* inv_freq;
  int section_end[SLIM_ROTARY_MAX_AXES];
  int axes;
  float magnitude;
  int inverse;
  int tokens;                       // tokens per block
  int chunks;                       // work items per (token, head): rotated, then passed through
  int rot_chunks;
};

template <typename T>
__device__ __forceinline__ float to_f(T v);
template <>
__device__ __forceinline__ float to_f(float v) { return v; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_f(float v);
template <>
__device__ __forceinline__ float from_f(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }

// Written out so that every access width and layout rounds alike. a = (cos, sin).
__device__ __forceinline__ float turn_x(float x, float y, float2 a) { return __fmaf_rn(x, a.x, -__fmul_rn(y, a.y)); }
__device__ __forceinline__ float turn_y(float x, float y, float2 a) { return __fmaf_rn(x, a.y, __fmul_rn(y, a.x)); }

template <typename T, int P>
struct alignas(sizeof(T) * P) Vec {
  T e[P];
};

// Two 16-bit elements of a word as fp32, and back.
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
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

// P pairs: partners in u and v (HALF), or neighbours in u then v. cs[e * step]: (cos, sin) of pair e.
template <typename T, int P, bool HALF>
__device__ __forceinline__ void turn(Vec<T, P>& u, Vec<T, P>& v, const float2* cs, int step) {
  if constexpr (sizeof(T) == 2 && P >= 2) {  // by words: the kernel is not far from being bound by issue
    uint32_t* uw = reinterpret_cast<uint32_t*>(&u);
    uint32_t* vw = reinterpret_cast<uint32_t*>(&v);
    if constexpr (HALF) {
#pragma unroll
      for (int w = 0; w < P / 2; ++w) {
        const float2 x = unpack2<T>(uw[w]), y = unpack2<T>(vw[w]);
        const float2 a = cs[2 * w * step], b = cs[(2 * w + 1) * step];
        uw[w] = pack2<T>(turn_x(x.x, y.x, a), turn_x(x.y, y.y, b));
        vw[w] = pack2<T>(turn_y(x.x, y.x, a), turn_y(x.y, y.y, b));
      }
    } else {
#pragma unroll
      for (int e = 0; e < P; ++e) {
        uint32_t& word = e < P / 2 ? uw[e % (P / 2)] : vw[e % (P / 2)];
        const float2 z = unpack2<T>(word), a = cs[e * step];
        word = pack2<T>(turn_x(z.x, z.y, a), turn_y(z.x, z.y, a));
      }
    }
  } else {
#pragma unroll
    for (int e = 0; e < P; ++e) {
      T& xe = HALF || P == 1 ? u.e[e] : 2 * e < P ? u.e[2 * e % P] : v.e[2 * e % P];
      T& ye = HALF || P == 1 ? v.e[e] : 2 * e < P ? u.e[(2 * e + 1) % P] : v.e[(2 * e + 1) % P];
      const float2 a = cs[e * step];
      const float x = to_f<T>(xe), y = to_f<T>(ye);
      xe = from_f<T>(turn_x(x, y, a));
      ye = from_f<T>(turn_y(x, y, a));
    }
  }
}

// P pairs per item: two accesses of P elements (a half pair's partners, or the two halves of
// 2P neighbours), P * sizeof(T) bytes each.
template <typename T, int P, bool HALF>
__global__ void __launch_bounds__(THREADS, BLOCKS) rotary_kernel(const Params p) {
  using V = Vec<T, P>;
  __shared__ float2 table[MAX_TABLE];
  __shared__ void* rows[MAX_TOKENS][4];  // a token's rows in q, k, q_out, k_out
  const int64_t total = p.batch * p.seq;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * p.tokens;
  const int n_tok = static_cast<int>(total - first < p.tokens ? total - first : p.tokens);

  if (threadIdx.x < n_tok * 4) {
    const int t = threadIdx.x >> 2, w = threadIdx.x & 3;
    const slim_view& v = w == 0 ? p.q : w == 1 ? p.k : w == 2 ? p.q_out : p.k_out;
    const uint32_t token = static_cast<uint32_t>(first) + t, b = token / static_cast<uint32_t>(p.seq);
    const uint32_t s = token - b * static_cast<uint32_t>(p.seq);
    rows[t][w] = static_cast<T*>(v.data) + b * v.stride_b + s * v.stride_s;
  }
  for (int i = threadIdx.x; i < n_tok * p.pairs; i += THREADS) {
    const int t = i / p.pairs;
    const int j = i - t * p.pairs;
    const uint32_t token = static_cast<uint32_t>(first) + t, b = token / static_cast<uint32_t>(p.seq);
    const uint32_t s = token - b * static_cast<uint32_t>(p.seq);
    int axis = 0;
    while (axis + 1 < p.axes && j >= p.section_end[axis]) ++axis;
    const int64_t at = b * p.pos_b + s * p.pos_s + axis * p.pos_a;
    const double pos = p.pos32 ? static_cast<double>(static_cast<const int32_t*>(p.pos)[at])
                               : static_cast<double>(static_cast<const int64_t*>(p.pos)[at]);
    // turns = pos * f / (2 pi) as the unevaluated sum of two doubles, so that the fraction of a turn
    // is good to fp32 whatever the position: 1/(2 pi) = kTurn + kTurnLo
    constexpr double kTurn = 0.15915494309189535, kTurnLo = -9.839338337591243e-18;
    const double f = p.inv_freq[j];
    const double g = f * kTurn, g_lo = fma(f, kTurn, -g) + f * kTurnLo;
    const double turns = pos * g, turns_lo = fma(pos, g, -turns) + pos * g_lo;
    // sin and cos of the fraction rounded to fp32, then moved by what the rounding left
    const double part = (turns - rint(turns)) + turns_lo;
    const float near = static_cast<float>(part), left = 6.2831853f * static_cast<float>(part - near);
    float s0, c0;
    sincospif(2.0f * near, &s0, &c0);
    const float cs = fmaf(-left, s0, c0), sn = p.inverse ? -fmaf(left, c0, s0) : fmaf(left, c0, s0);
    // the pairs of a work item lie rot_chunks apart: its neighbours' are next to them
    table[t * p.pairs + j % P * p.rot_chunks + j / P] = make_float2(cs * p.magnitude, sn * p.magnitude);
  }
  __syncthreads();

  // Rows of this block: (token, head); this thread takes chunk c of every rows_step-th. (Two or four rows
  // in flight a thread cost more in registers, hence threads, than they gain: 293, 381, 625 us at 30026
  // tokens x 112 heads x 128, in the form by single elements.)
  const int rows_step = THREADS / p.chunks > 0 ? THREADS / p.chunks : 1;
  for (int c = threadIdx.x % p.chunks; c < p.chunks; c += THREADS) {
    const int row0 = threadIdx.x / p.chunks;
    if (row0 >= rows_step) break;
    const bool turns = c < p.rot_chunks;
    const int lo = turns ? (HALF ? c * P : 2 * c * P) : p.rot + (c - p.rot_chunks) * P;
    const int hi = HALF ? c * P + p.pairs : 2 * c * P + P;
    int t = row0 / p.heads;
    int h = row0 - t * p.heads;
    while (t < n_tok) {
      const bool is_k = h >= p.heads_q;
      const int hh = is_k ? h - p.heads_q : h;
      const T* src = static_cast<const T*>(rows[t][is_k]) + hh * (is_k ? p.k.stride_h : p.q.stride_h);
      T* dst = static_cast<T*>(rows[t][2 + is_k]) + hh * (is_k ? p.k_out.stride_h : p.q_out.stride_h);
      const float2* cs = table + t * p.pairs + c;
      V u = *reinterpret_cast<const V*>(src + lo), v;
      if (turns) v = *reinterpret_cast<const V*>(src + hi);
      h += rows_step;
      while (h >= p.heads) {
        h -= p.heads;
        ++t;
      }
      if (turns) {
        turn<T, P, HALF>(u, v, cs, p.rot_chunks);
        *reinterpret_cast<V*>(dst + hi) = v;
      }
      *reinterpret_cast<V*>(dst + lo) = u;
    }
  }
}

template <typename T, int P>
cudaError_t launch_p(const Params& p, bool half, cudaStream_t st) {
  const int64_t total = p.batch * p.seq;
  const unsigned grid = static_cast<unsigned>((total + p.tokens - 1) / p.tokens);
  if (half)
    rotary_kernel<T, P, true><<<grid, THREADS, 0, st>>>(p);
  else
    rotary_kernel<T, P, false><<<grid, THREADS, 0, st>>>(p);
  return cudaGetLastError();
}

static bool view_fits(const slim_view& v, int64_t batch, int64_t seq, int heads, int size, int bytes) {
  if (reinterpret_cast<uintptr_t>(v.data) % bytes) return false;
  return (batch == 1 || v.stride_b * size % bytes == 0) && (seq == 1 || v.stride_s * size % bytes == 0) &&
         (heads == 1 || v.stride_h * size % bytes == 0);
}

template <typename T>
cudaError_t launch(Params& p, bool half, bool copies, cudaStream_t st) {
  // The widest access (16 bytes down to one element) that every address allows and that divides
  // the rotated half and the part passed through.
  int P = 16 / static_cast<int>(sizeof(T));
  const int hk = p.heads - p.heads_q;
  for (; P > 1; P >>= 1) {
    const int bytes = P * static_cast<int>(sizeof(T));
    const bool ok = p.pairs % P == 0 && (!copies || (p.dim - p.rot) % P == 0) &&
                    view_fits(p.q, p.batch, p.seq, p.heads_q, sizeof(T), bytes) &&
                    view_fits(p.q_out, p.batch, p.seq, p.heads_q, sizeof(T), bytes) &&
                    (hk == 0 || (view_fits(p.k, p.batch, p.seq, hk, sizeof(T), bytes) &&
                                 view_fits(p.k_out, p.batch, p.seq, hk, sizeof(T), bytes)));
    if (ok) break;
  }
  p.rot_chunks = p.pairs / P;
  p.chunks = p.rot_chunks + (copies ? (p.dim - p.rot) / P : 0);
  // Tokens per block: up to twelve rounds of its threads, so that the table's latency is a small part (65537 tokens x
  // 10 heads of 64 in fp32: 57 us with sixteen, 139 with one; 30026 tokens x 112 heads of 128, bf16: 268 us with three,
  // 287 with eight), within the table; fewer where that leaves SMs idle, or a second round of blocks with few in it
  // (8198 tokens x 48 heads of 128: 40 us with two tokens a block, 42 with five).
  const int64_t items = static_cast<int64_t>(p.heads) * p.chunks;
  int64_t tokens = (12 * THREADS + items - 1) / items;
  if (tokens > MAX_TOKENS) tokens = MAX_TOKENS;
  if (tokens > MAX_TABLE / p.pairs) tokens = MAX_TABLE / p.pairs;
  const int64_t total = p.batch * p.seq;
  const int64_t sms = sm_count(), full = sms * BLOCKS;
  auto uneven = [&](int64_t blocks) { return blocks < sms * 4 || (blocks > full && blocks < 2 * full); };
  while (tokens > 1 && uneven(total / tokens)) tokens >>= 1;
  p.tokens = static_cast<int>(tokens < 1 ? 1 : tokens);
  if constexpr (sizeof(T) == 2)
    if (P == 8) return launch_p<T, 8>(p, half, st);
  switch (P) {
    case 4: return launch_p<T, 4>(p, half, st);
    case 2: return launch_p<T, 2>(p, half, st);
    default: return launch_p<T, 1>(p, half, st);
  }
}

}  // namespace rope
}  // namespace slim

using namespace slim;

extern "C" int slim_rotary(const slim_view* q, const slim_view* q_out, int heads_q, const slim_view* k,
                           const slim_view* k_out, int heads_k, int dtype, int64_t batch, int64_t seq, int dim, int rot,
                           int layout, const void* pos, int pos_bits, int64_t pos_stride_b, int64_t pos_stride_s,
                           int64_t pos_stride_a, const float* inv_freq, const int* sections, int axes, float magnitude,
                           int inverse, void* stream) {
  SLIM_NVTX("slim_rotary");
  int rc;
  if ((rc = check_dtype(dtype)) != SLIM_OK) return rc;
  if (batch < 0 || seq < 0 || heads_q <= 0 || heads_k < 0 || dim <= 0)
    return fail(SLIM_ERR_SHAPE, "bad rotary shape batch=%lld seq=%lld heads=%d/%d dim=%d", static_cast<long long>(batch),
                static_cast<long long>(seq), heads_q, heads_k, dim);
  if (dim > 2 * rope::MAX_TABLE) return fail(SLIM_ERR_SHAPE, "head dim %d is above %d", dim, 2 * rope::MAX_TABLE);
  if (rot < 2 || rot % 2 || rot > dim)
    return fail(SLIM_ERR_SHAPE, "the rotated part must be even and within the head dim %d, got %d", dim, rot);
  if (layout != SLIM_ROTARY_HALF && layout != SLIM_ROTARY_INTERLEAVED) return fail(SLIM_ERR_DTYPE, "unknown rotary layout %d", layout);
  if (pos_bits != 32 && pos_bits != 64) return fail(SLIM_ERR_DTYPE, "positions must be 32- or 64-bit integers");
  if (axes < 1 || axes > SLIM_ROTARY_MAX_AXES || (axes > 1 && sections == nullptr))
    return fail(SLIM_ERR_SHAPE, "1 to %d position axes, got %d", SLIM_ROTARY_MAX_AXES, axes);
  if (batch > (int64_t{1} << 31) || seq > (int64_t{1} << 31) || batch * seq > (int64_t{1} << 31) - 1 ||
      heads_q > (1 << 20) || heads_k > (1 << 20))
    return fail(SLIM_ERR_SHAPE, "rotary shape too large");
  rope::Params p{};
  int end = 0;
  for (int a = 0; a < axes; ++a) {
    const int n = sections != nullptr ? sections[a] : rot / 2;
    if (n < 0 || n > rot / 2 - end) return fail(SLIM_ERR_SHAPE, "the sections do not add up to the %d pairs", rot / 2);
    p.section_end[a] = end += n;
  }
  if (end != rot / 2) return fail(SLIM_ERR_SHAPE, "the sections add up to %d of %d pairs", end, rot / 2);
  if (batch == 0 || seq == 0) return SLIM_OK;
  if (q == nullptr || q_out == nullptr || q->data == nullptr || q_out->data == nullptr || pos == nullptr || inv_freq == nullptr)
    return fail(SLIM_ERR_NULL, "q/q_out/pos/inv_freq is NULL");
  if (heads_k > 0 && (k == nullptr || k_out == nullptr || k->data == nullptr || k_out->data == nullptr))
    return fail(SLIM_ERR_NULL, "k/k_out is NULL");
  if ((rc = check_arch()) != SLIM_OK) return rc;
  p.q = *q;
  p.q_out = *q_out;
  bool copies = q->data != q_out->data;
  if (heads_k > 0) {
    p.k = *k;
    p.k_out = *k_out;
    copies = copies || k->data != k_out->data;
  }
  copies = copies && rot < dim;
  p.heads_q = heads_q;
  p.heads = heads_q + heads_k;
  p.batch = batch;
  p.seq = seq;
  p.dim = dim;
  p.rot = rot;
  p.pairs = rot / 2;
  p.pos = pos;
  p.pos32 = pos_bits == 32;
  p.pos_b = pos_stride_b;
  p.pos_s = pos_stride_s;
  p.pos_a = pos_stride_a;
  p.inv_freq = inv_freq;
  p.axes = axes;
  p.magnitude = magnitude;
  p.inverse = inverse;
  const bool half = layout == SLIM_ROTARY_HALF;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = dtype == kF32    ? rope::launch<float>(p, half, copies, st)
                        : dtype == kBF16 ? rope::launch<__nv_bfloat16>(p, half, copies, st)
                                         : rope::launch<__half>(p, half, copies, st);
  if (e != cudaSuccess) return cuda_fail(e, "rotary launch");
  note_launch();
  return SLIM_OK;
}
