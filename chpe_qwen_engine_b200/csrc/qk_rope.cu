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
// Bound by memory: T*D*((2H+2KV)*act + 2KV*cache) bytes, each once.  A lane
// holds both halves of its rotated pairs, 8 values each (two full 128-bit
// accesses of 16-bit values), so the rotation needs no exchange between lanes;
// D/16 lanes make a head, 512/D heads a group.  A warp takes one token and a run of
// its groups: it computes the token's cos and sin once (two to four pairs per lane,
// passed around through shared memory), keeps the norm weights in registers,
// and issues the loads of U groups before it works on the first.  How long the runs
// are goes by the number of tokens: one group per warp when there are few (a
// single token of the 72B's heads is 20 warps), all of a token's when the tokens alone fill
// the GPU and the angles are worth sharing.  16384 tokens of 64/8 heads of 128 in
// BF16: 115 us, 5.8 TB/s, 90 % of the copy rate (a plain copy of q, k and v alone takes 102);
// one token: 2.9 us, a launch and three dependent loads.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "device_common.cuh"
#include "serve_common.h"

namespace {

constexpr int kWarps = 2, kMaxHalf = 128;

struct QkLaunch {
  const void *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;  // elements between tokens
  void *q_out, *k_out;
  int64_t qo_stride, ko_stride;
  const float *q_weight, *k_weight;
  float offset, eps;
  const int32_t* positions;
  int32_t half;  // rotated pairs (rope_dim / 2)
  int32_t H, KV;
  int32_t gq, gkv, groups;  // groups of q, of k (and of v), of all
  int32_t runs;             // warps per token
  uint32_t warps;           // tokens * runs
  void *k_cache, *v_cache;
  const int64_t* slots;
  int64_t cache_rows;
  uint64_t turn[kMaxHalf];  // 2^64 * inv_freq / (2 pi), modulo 2^64
};

// Eight values as they lie in memory, and as f32.
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  CHPE_DEV void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  CHPE_DEV void zero() {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; i++) w[i] = make_uint4(0, 0, 0, 0);
  }
  CHPE_DEV void get(float (&x)[8]) const {
    const uint32_t* u = &w[0].x;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = __uint_as_float(i < 4 ? (&w[0].x)[i] : (&w[sizeof(T) / 2 - 1].x)[i - 4]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(u[i] << 16);
        x[2 * i + 1] = __uint_as_float(u[i] & 0xFFFF0000u);
      }
    }
  }
};
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
  const int64_t r = (int64_t)(up & ((1ull << 62) - 1)) - (1ll << 61);  // [-1/8, 1/8) turn
  float s, c;
  sincospif((float)r * 0x1p-63f, &s, &c);  // half turns
  const float cc = (quad & 1u) ? s : c, ss = (quad & 1u) ? c : s;
  return make_float2((quad == 1u || quad == 2u) ? -cc : cc, quad >= 2u ? -ss : ss);
}

// TA: type of q, k, v and the outputs; TC: type of the cache; D: head dim; U:
// groups a warp has in flight.
template <typename TA, typename TC, int D, int U>
__global__ void __launch_bounds__(32 * kWarps) qk_rope_kernel(const __grid_constant__ QkLaunch P) {
  constexpr int LPH = D / 16, HPG = 32 / LPH;  // lanes per head, heads per group
  __shared__ float2 cs[kWarps][kMaxHalf];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t id = blockIdx.x * kWarps + warp;
  if (id >= P.warps) return;
  const int64_t t = id / (uint32_t)P.runs;
  const int run = (int)(id % (uint32_t)P.runs);
  const int g_begin = (int)((int64_t)run * P.groups / P.runs), g_end = (int)((int64_t)(run + 1) * P.groups / P.runs);
  const int sub = lane % LPH, hl = lane / LPH;
  const int sh = P.half / 8;  // lanes that hold rotated pairs
  // this lane's two chunks of 8: a rotated pair's halves, or two neighbours of the rest
  const int ca = 8 * (sub < sh ? sub : 2 * sub), cb = 8 * (sub < sh ? sub + sh : 2 * sub + 1);

  Raw8<TA> ra[U], rb[U];
  auto head_of = [&](int g) {  // head of its kind and the kind: 0 q, 1 k, 2 v
    const int kind = g < P.gq ? 0 : g < P.gq + P.gkv ? 1 : 2;
    return make_int2((g - (kind == 0 ? 0 : kind == 1 ? P.gq : P.gq + P.gkv)) * HPG + hl, kind);
  };
  auto fetch = [&](int u, int g) {
    const int2 h = head_of(g);
    if (g < g_end && h.x < (h.y == 0 ? P.H : P.KV)) {
      const TA* src = h.y == 0 ? static_cast<const TA*>(P.q) + t * P.q_stride
                      : h.y == 1 ? static_cast<const TA*>(P.k) + t * P.k_stride
                                 : static_cast<const TA*>(P.v) + t * P.v_stride;
      ra[u].load(src + h.x * D + ca);
      rb[u].load(src + h.x * D + cb);
    } else {
      ra[u].zero();
      rb[u].zero();
    }
  };
#pragma unroll
  for (int u = 0; u < U; u++) fetch(u, g_begin + u);
  const int64_t slot = P.slots ? P.slots[t] : -1;
  const bool keep = slot >= 0 && slot < P.cache_rows;

  float2 r[8];
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = make_float2(1.f, 0.f);
  if (P.half) {
    const uint64_t pos = (uint64_t)(int64_t)P.positions[t];
    for (int i = lane; i < P.half; i += 32) cs[warp][(i & 7) * sh + (i >> 3)] = cos_sin_turn(pos * P.turn[i]);
    __syncwarp();
    if (sub < sh)
#pragma unroll
      for (int e = 0; e < 8; e++) r[e] = cs[warp][e * sh + sub];
  }

  float wa[8], wb[8];
  int have = -1;  // kind whose weights are held
  for (int g0 = g_begin; g0 < g_end; g0 += U) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      const int g = g0 + u;
      if (g >= g_end) break;
      const int2 h = head_of(g);
      float a[8], b[8];
      ra[u].get(a);
      rb[u].get(b);
      fetch(u, g + U);
      if (h.y < 2) {
        const float* w = h.y == 0 ? P.q_weight : P.k_weight;
        if (w) {
          if (have != h.y) {
            have = h.y;
#pragma unroll
            for (int e = 0; e < 8; e++) {
              wa[e] = w[ca + e] + P.offset;
              wb[e] = w[cb + e] + P.offset;
            }
          }
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; e++) ss = fmaf(a[e], a[e], fmaf(b[e], b[e], ss));
#pragma unroll
          for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const float inv = rsqrtf(ss * (1.0f / D) + P.eps);  // within 2 ulp; an exact root and quotient took 5 us of 121
#pragma unroll
          for (int e = 0; e < 8; e++) {
            a[e] = a[e] * inv * wa[e];
            b[e] = b[e] * inv * wb[e];
          }
        }
        if (sub < sh) {  // the others' values stay as they are, infinities and signs of zero too
#pragma unroll
          for (int e = 0; e < 8; e++) {
            const float x = a[e], y = b[e];
            a[e] = fmaf(x, r[e].x, -y * r[e].y);
            b[e] = fmaf(y, r[e].x, x * r[e].y);
          }
        }
      }
      if (h.x >= (h.y == 0 ? P.H : P.KV)) continue;
      if (h.y == 0) {
        TA* o = static_cast<TA*>(P.q_out) + t * P.qo_stride + h.x * D;
        store8(o + ca, a);
        store8(o + cb, b);
        continue;
      }
      if (h.y == 1 && P.k_out) {
        TA* o = static_cast<TA*>(P.k_out) + t * P.ko_stride + h.x * D;
        store8(o + ca, a);
        store8(o + cb, b);
      }
      if (keep) {
        TC* o = static_cast<TC*>(h.y == 1 ? P.k_cache : P.v_cache) + (slot * P.KV + h.x) * D;
        store8(o + ca, a);
        store8(o + cb, b);
      }
    }
  }
}

template <typename TA, typename TC, int D>
cudaError_t launch(QkLaunch& P, uint32_t tokens, cudaStream_t s) {
  constexpr int HPG = 512 / D, U = sizeof(TA) == 4 ? 2 : 4;
  P.gq = (P.H + HPG - 1) / HPG;
  P.gkv = (P.KV + HPG - 1) / HPG;
  P.groups = P.gq + (P.k_cache ? 2 : 1) * P.gkv;  // without a cache the v heads have nowhere to go
  // about 8 warps for each of 148 SMs, at most one per group and at least one per
  // token: more of them only work out more angles (300 tokens of 64/8 heads: 6.2 us
  // with 8, 8.9 with 16, 9.8 with 32)
  const int64_t want = (148 * 8 + (int64_t)tokens - 1) / tokens;
  P.runs = (int32_t)(want < 1 ? 1 : want > P.groups ? P.groups : want);
  // (more warps than 32 bits can count: whole tokens)
  if ((uint64_t)tokens * P.runs > 0xffffff00u) P.runs = 1;
  P.warps = tokens * (uint32_t)P.runs;
  chpe::ServeLaunch L(dim3((P.warps + kWarps - 1) / kWarps), 32 * kWarps, 0, s);
  return cudaLaunchKernelEx(&L.cfg, qk_rope_kernel<TA, TC, D, U>, P);
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
  if (num_tokens == 0) return c.done();
  if (!k_cache != !v_cache) return c.fail(-1, "k_cache and v_cache go together"), c.done();
  if (!k_cache && !k_out) return c.fail(-1, "neither a cache nor k_out to write k to"), c.done();
  if (k_cache && cache_dtype != CHPE_F16 && cache_dtype != CHPE_BF16)
    return c.fail(-1, "the cache must be FP16 or BF16"), c.done();
  if (k_cache && dtype != CHPE_F32 && dtype != cache_dtype)
    return c.fail(-1, "the cache must have the type of q, k and v unless those are float"), c.done();
  if (k_cache && cache_rows > (uint64_t)INT64_MAX) return c.fail(-1, "cache_rows is too large"), c.done();
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
    if (turns < 0.0L || turns >= 1.0L) turns -= floorl(turns);  // a library call, 1 us for 64 of them
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
  c.ptr_or_null(q_weight, "q_weight", 4);  // (read value by value, once per warp)
  c.ptr_or_null(k_weight, "k_weight", 4);
  if (c.rc) return c.done();
  {
    // q_out may be q and k_out k, row by row; else what is written meets nothing
    using chpe::Rows;
    const int64_t n = num_tokens, b = (int64_t)es, w = head_dim * (int64_t)sizeof(float);
    const Rows in[] = {{"q", q, hq * b, n, q_stride, b}, {"k", k, hk * b, n, k_stride, b},
                       {"v", k_cache ? v : nullptr, hk * b, n, v_stride, b}, {"q_weight", q_weight, w}, {"k_weight", k_weight, w},
                       {"positions", rope_dim ? positions : nullptr, 4 * n}, {"slots", k_cache ? slots : nullptr, 8 * n}};
    const Rows out[] = {{"q_out", q_out, hq * b, n, q_out_stride, b}, {"k_out", k_out, hk * b, n, k_out_stride, b},
                        chpe::pool("k_cache", k_cache, cache_rows, hk * 2), chpe::pool("v_cache", v_cache, cache_rows, hk * 2)};
    for (int o = 0; o < 4; o++) {
      for (int i = 0; i < 7; i++)
        if (!(o == i && out[o].p == in[i].p && (n == 1 || out[o].stride == in[i].stride) && o < 2)) c.apart(out[o], in[i]);
      for (int i = 0; i < o; i++) c.apart(out[o], out[i]);
    }
    if (c.rc) return c.done();
  }

  P.q = q, P.k = k, P.v = v;
  P.q_stride = q_stride, P.k_stride = k_stride, P.v_stride = v_stride;
  P.q_out = q_out, P.k_out = k_out, P.qo_stride = q_out_stride, P.ko_stride = k_out_stride;
  P.q_weight = q_weight, P.k_weight = k_weight, P.offset = weight_offset, P.eps = eps;
  P.positions = positions, P.half = (int32_t)rope_dim / 2;
  P.H = (int32_t)num_heads, P.KV = (int32_t)num_kv_heads;
  P.k_cache = k_cache, P.v_cache = v_cache, P.slots = k_cache ? slots : nullptr;
  P.cache_rows = (int64_t)cache_rows;
  chpe::DeviceScope scope(c.launch_device());
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
