// qk_rope.cu -- per-head RMSNorm of q and k, rotary embedding and the append
// of k and v to a paged cache, in one pass over a batch of tokens.
//
// For every token and head (x the head's D values, w its norm weight):
//   y = x / sqrt(mean(x^2) + eps) * (w + offset)      (left out without weights)
//   for i < r/2:  a = position * inv_freq[i]
//     y[i], y[i + r/2] = y[i] cos a - y[i + r/2] sin a, y[i + r/2] cos a + y[i] sin a
// with r = rope_dim <= D (the rest of the head is not rotated); q goes to
// q_out, k to the cache row of the token's slot (and / or k_out), v to its
// cache row unchanged.  Everything is f32 from the load to the one rounding
// of the store.
//
// Angles: a position of 1e5 times a frequency near 1 has no fraction of a turn
// left to speak of in f32 (its last bit is 8e-3 rad).  The host turns each
// frequency into 64-bit fixed point, f = round(2^64 * inv_freq / 2 pi) mod
// 2^64; position * f modulo 2^64 is then the exact fraction of a turn (error
// position * 2^-65), reduced to an eighth of a turn in integers before the
// one rounding to f32.
//
// Bound by memory: T*D*((2H+2KV)*act + 2KV*cache) bytes, each once.  One CTA
// takes one token and up to kWarps * IT head groups: D/8 lanes hold a head
// (16 or 32 bytes each, so every access is a full 128-bit one), 32*8/D heads
// per warp and group.  A warp first issues the loads of all its groups; while
// they are in flight one thread per rotated pair computes cos and sin, which
// the CTA's heads share through shared memory.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_common.cuh"
#include "serve_common.h"

namespace {

constexpr int kWarps = 8, kMaxHalf = 128;

struct QkLaunch {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  void *q_out, *k_out;
  int64_t qo_stride, ko_stride;
  const float *q_weight, *k_weight;
  float offset, eps;
  const int32_t* positions;
  int32_t half;  // rotated pairs (rope_dim / 2)
  int32_t H, KV, heads;  // heads: H + 2 KV, or H + KV without a cache
  void *k_cache, *v_cache;
  const int64_t* slots;
  int64_t cache_rows;
  int32_t groups_per_cta;
  uint64_t turn[kMaxHalf];  // 2^64 * inv_freq / (2 pi), modulo 2^64
};

template <typename T>
CHPE_DEV void load8(const T* p, float (&x)[8]);
template <>
CHPE_DEV void load8<float>(const float* p, float (&x)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}
template <>
CHPE_DEV void load8<__half>(const __half* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    x[2 * i] = f.x, x[2 * i + 1] = f.y;
  }
}
template <>
CHPE_DEV void load8<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[8]) {
  const uint4 a = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
  }
}
template <typename T>
CHPE_DEV void store8(T* p, const float (&x)[8]);
template <>
CHPE_DEV void store8<float>(float* p, const float (&x)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <>
CHPE_DEV void store8<__half>(__half* p, const float (&x)[8]) {
  uint4 a;
  uint32_t* w = &a.x;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = a;
}
template <>
CHPE_DEV void store8<__nv_bfloat16>(__nv_bfloat16* p, const float (&x)[8]) {
  uint4 a;
  uint32_t* w = &a.x;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = a;
}

// cos and sin of a fraction of a turn given in units of 2^-64 turns.
CHPE_DEV float2 cos_sin_turn(uint64_t f) {
  const uint64_t up = f + (1ull << 61);             // + 1/8 turn
  const uint32_t quad = (uint32_t)(up >> 62);       // nearest quarter turn
  const int64_t r = (int64_t)(up & ((1ull << 62) - 1)) - (int64_t)(1ull << 61);  // [-1/8, 1/8) turn
  float s, c;
  sincospif(__ll2float_rn(r) * 0x1p-63f, &s, &c);  // half turns
  const float cc = (quad & 1u) ? s : c, ss = (quad & 1u) ? c : s;
  return make_float2((quad == 1u || quad == 2u) ? -cc : cc, quad >= 2u ? -ss : ss);
}

// TA: type of q, k, v and the outputs; TC: type of the cache; D: head dim;
// IT: head groups a warp holds at once.
template <typename TA, typename TC, int D, int IT>
__global__ void __launch_bounds__(32 * kWarps) qk_rope_kernel(const __grid_constant__ QkLaunch P) {
  constexpr int LPH = D / 8, HPW = 32 / LPH;  // lanes per head, heads per warp and group
  __shared__ float2 cs[kMaxHalf];
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane % LPH, hl = lane / LPH;
  const int heads = P.heads;
  const int g0 = blockIdx.y * P.groups_per_cta;
  const int g1 = min(g0 + P.groups_per_cta, (heads + HPW - 1) / HPW);

  float x[IT][8];
#pragma unroll
  for (int u = 0; u < IT; u++) {
    const int g = g0 + warp + u * kWarps, h = g * HPW + hl;
    if (g < g1 && h < heads) {
      const TA* src = h < P.H ? static_cast<const TA*>(P.q) + t * P.q_stride + (int64_t)h * D
                      : h < P.H + P.KV ? static_cast<const TA*>(P.k) + t * P.k_stride + (int64_t)(h - P.H) * D
                                       : static_cast<const TA*>(P.v) + t * P.v_stride + (int64_t)(h - P.H - P.KV) * D;
      load8(src + 8 * sub, x[u]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) x[u][e] = 0.f;
    }
  }
  const int64_t slot = P.slots ? P.slots[t] : -1;
  if ((int)threadIdx.x < P.half)
    cs[threadIdx.x] = cos_sin_turn((uint64_t)(int64_t)P.positions[t] * P.turn[threadIdx.x]);
  __syncthreads();

  const int sh = P.half / 8;  // lanes per rotated half
  float2 r[8];
  {
    const int i0 = 8 * (sub < sh ? sub : sub - sh);
    const bool rot = sub < 2 * sh;
#pragma unroll
    for (int e = 0; e < 8; e++) r[e] = rot ? cs[i0 + e] : make_float2(1.f, 0.f);
    if (sub < sh)  // the lower half subtracts
#pragma unroll
      for (int e = 0; e < 8; e++) r[e].y = -r[e].y;
  }
  const int partner = sub < sh ? sub + sh : sub < 2 * sh ? sub - sh : sub;
#pragma unroll
  for (int u = 0; u < IT; u++) {
    const int g = g0 + warp + u * kWarps, h = g * HPW + hl;
    if (g >= g1) break;  // uniform over the warp
    const bool is_q = h < P.H, is_k = !is_q && h < P.H + P.KV;
    const float* w = is_q ? P.q_weight : is_k ? P.k_weight : nullptr;
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) ss = fmaf(x[u][e], x[u][e], ss);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w) {
      const float inv = 1.0f / sqrtf(ss / (float)D + P.eps);
      float wv[8];
      load8(w + 8 * sub, wv);
#pragma unroll
      for (int e = 0; e < 8; e++) x[u][e] = x[u][e] * inv * (wv[e] + P.offset);
    }
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; e++) {
      const float p = __shfl_sync(0xffffffffu, x[u][e], partner, LPH);
      y[e] = is_q || is_k ? fmaf(x[u][e], r[e].x, p * r[e].y) : x[u][e];
    }
    if (h >= heads) continue;
    if (is_q) {
      store8(static_cast<TA*>(P.q_out) + t * P.qo_stride + (int64_t)h * D + 8 * sub, y);
      continue;
    }
    const int kvh = is_k ? h - P.H : h - P.H - P.KV;
    if (is_k && P.k_out) store8(static_cast<TA*>(P.k_out) + t * P.ko_stride + (int64_t)kvh * D + 8 * sub, y);
    if (slot >= 0 && slot < P.cache_rows) {
      TC* c = static_cast<TC*>(is_k ? P.k_cache : P.v_cache);
      store8(c + (slot * P.KV + kvh) * D + 8 * sub, y);
    }
  }
}

template <typename TA, typename TC, int D>
cudaError_t launch(QkLaunch& P, uint32_t tokens, cudaStream_t s) {
  constexpr int HPW = 32 / (D / 8);
  // without a cache the v heads have nowhere to go
  P.heads = P.H + (P.k_cache ? 2 : 1) * P.KV;
  const int groups = (P.heads + HPW - 1) / HPW;
  constexpr int IT = 4;
  int ctas = (groups + kWarps * IT - 1) / (kWarps * IT);
  P.groups_per_cta = (groups + ctas - 1) / ctas;
  qk_rope_kernel<TA, TC, D, IT><<<dim3(tokens, ctas), 32 * kWarps, 0, s>>>(P);
  return cudaGetLastError();
}

template <typename TA, typename TC>
cudaError_t launch_d(QkLaunch& P, uint32_t head_dim, uint32_t tokens, cudaStream_t s) {
  if (head_dim == 64) return launch<TA, TC, 64>(P, tokens, s);
  if (head_dim == 128) return launch<TA, TC, 128>(P, tokens, s);
  return launch<TA, TC, 256>(P, tokens, s);
}

}  // namespace

extern "C" int chpe_qk_norm_rope(const void* q, const void* k, const void* v, int dtype, int64_t q_stride,
                                 int64_t k_stride, int64_t v_stride, uint32_t num_tokens, uint32_t num_heads,
                                 uint32_t num_kv_heads, uint32_t head_dim, const float* q_weight,
                                 const float* k_weight, float weight_offset, float eps,
                                 const int32_t* positions, const double* inv_freq, uint32_t rope_dim, void* q_out,
                                 int64_t q_out_stride, void* k_out, int64_t k_out_stride, void* k_cache,
                                 void* v_cache, int cache_dtype, uint64_t cache_rows, const int64_t* slots,
                                 void* stream) {
  chpe::ServeCall c("chpe_qk_norm_rope");
  const size_t es = chpe::dtype_size(dtype);
  if (!es) return c.fail(-1, "unknown dtype %lld", dtype), c.done();
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return c.fail(-1, "head_dim must be 64, 128 or 256"), c.done();
  if (num_heads == 0 || num_kv_heads == 0 || num_heads > 65535 || num_kv_heads > 65535)
    return c.fail(-1, "num_heads and num_kv_heads must be 1..65535"), c.done();
  if (rope_dim > head_dim || rope_dim % 16 != 0)
    return c.fail(-1, "rope_dim must be a multiple of 16 up to head_dim"), c.done();
  if (num_tokens > 0x7fffffffu) return c.fail(-1, "too many tokens"), c.done();
  if (!k_cache != !v_cache) return c.fail(-1, "k_cache and v_cache go together"), c.done();
  if (!k_cache && !k_out) return c.fail(-1, "neither a cache nor k_out to write k to"), c.done();
  if (k_cache && cache_dtype != CHPE_F16 && cache_dtype != CHPE_BF16)
    return c.fail(-1, "the cache must be FP16 or BF16"), c.done();
  if (k_cache && dtype != CHPE_F32 && dtype != cache_dtype)
    return c.fail(-1, "the cache must have the type of q, k and v unless those are float"), c.done();
  if (k_cache && cache_rows > (uint64_t)INT64_MAX) return c.fail(-1, "cache_rows is too large"), c.done();
  if (num_tokens == 0) return c.done();
  const int64_t lane = 16 / (int64_t)es;  // elements of a 16-byte access
  const int64_t hq = (int64_t)num_heads * head_dim, hk = (int64_t)num_kv_heads * head_dim;
  const int64_t strides[5] = {q_stride, k_stride, k_cache ? v_stride : hk, q_out_stride, k_out ? k_out_stride : hk};
  const int64_t least[5] = {hq, hk, hk, hq, hk};
  static const char* const names[5] = {"q_stride", "k_stride", "v_stride", "q_out_stride", "k_out_stride"};
  for (int i = 0; i < 5; i++)
    if (num_tokens > 1 && (strides[i] < least[i] || strides[i] % lane != 0 || strides[i] > INT64_MAX / 4 / num_tokens)) {
      snprintf(c.msg, sizeof(c.msg), "%s must be at least the token's size and a multiple of 16 bytes", names[i]);
      c.rc = -1;
      return c.done();
    }
  QkLaunch P{};
  if (rope_dim && !inv_freq) return c.fail(-1, "inv_freq is NULL"), c.done();
  for (uint32_t i = 0; i < rope_dim / 2; i++) {
    // a fraction of a turn, exact to 2^-64: an 80-bit product with 1 / 2 pi
    const double f = inv_freq[i];
    if (!(fabs(f) <= 16.0)) return c.fail(-1, "inv_freq[%lld] is not a number within 16", i), c.done();
    long double turns = (long double)f * 0.159154943091895335768883763372514362L;
    turns -= floorl(turns);
    const long double scaled = turns * 18446744073709551616.0L + 0.5L;
    P.turn[i] = scaled >= 18446744073709551616.0L ? 0u : (uint64_t)scaled;
  }
  c.ptr(q, "q", 16);
  c.ptr(k, "k", 16);
  c.ptr(q_out, "q_out", 16);
  c.ptr_or_null(k_out, "k_out", 16);
  if (k_cache) {
    c.ptr(v, "v", 16);
    c.ptr(k_cache, "k_cache", 16);
    c.ptr(v_cache, "v_cache", 16);
    c.ptr(slots, "slots", 8);
  }
  if (rope_dim) c.ptr(positions, "positions", 4);
  c.ptr_or_null(q_weight, "q_weight", 16);
  c.ptr_or_null(k_weight, "k_weight", 16);
  if (c.rc) return c.done();

  P.q = q, P.k = k, P.v = v;
  P.q_stride = q_stride, P.k_stride = k_stride, P.v_stride = v_stride;
  P.q_out = q_out, P.k_out = k_out, P.qo_stride = q_out_stride, P.ko_stride = k_out_stride;
  P.q_weight = q_weight, P.k_weight = k_weight, P.offset = weight_offset, P.eps = eps;
  P.positions = positions, P.half = (int32_t)rope_dim / 2;
  P.H = (int32_t)num_heads, P.KV = (int32_t)num_kv_heads;
  P.k_cache = k_cache, P.v_cache = v_cache, P.slots = k_cache ? slots : nullptr;
  P.cache_rows = (int64_t)cache_rows;
  chpe::DeviceScope scope(c.device);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool half = !k_cache ? dtype != CHPE_BF16 : cache_dtype == CHPE_F16;
  cudaError_t e;
  if (dtype == CHPE_F32) e = half ? launch_d<float, __half>(P, head_dim, num_tokens, s)
                                  : launch_d<float, __nv_bfloat16>(P, head_dim, num_tokens, s);
  else if (dtype == CHPE_F16) e = launch_d<__half, __half>(P, head_dim, num_tokens, s);
  else e = launch_d<__nv_bfloat16, __nv_bfloat16>(P, head_dim, num_tokens, s);
  if (e != cudaSuccess) {
    snprintf(c.msg, sizeof(c.msg), "launch: %s", cudaGetErrorString(e));
    c.rc = -3;
  }
  return c.done();
}
