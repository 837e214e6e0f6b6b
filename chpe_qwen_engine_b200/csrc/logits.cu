// logits.cu -- penalties for repeated tokens, biases and a grammar's mask on the
// logits of a batch, and the token that wins.
//
// For row b and token v, x = logits[b][v], every step rounded to f32 on its own
// (no fused multiply-add), so results equal the same steps done one by one:
//   v in the history at all:               x = x > 0 ? x / repetition : x * repetition
//   v written c > 0 times after the prompt: x = (x - frequency * c) - presence
//   a bias entry for v (the last of them):  x = x + value
//   mask bit of v is 0:                     x = -inf
// argmax: the lowest index of the largest x; NaN never wins; -1 when nothing
// is above -inf.
//
// Bound by memory: the logits in, the f32 logits out.  A cluster of 8 CTAs takes
// one row, a slice of the vocabulary each.  A CTA counts its slice's tokens of the
// history in shared memory (one word per token: bit 31 seen in the prompt, the
// rest the count after it) with integer atomics, whose order does not matter,
// then streams its slice once, four tokens per thread and step.  The CTAs join
// their best tokens through distributed shared memory: no workspace, no second
// launch.  Without history and biases no table is made.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>

#include "device_common.cuh"
#include "serve_common.h"

namespace cg = cooperative_groups;

namespace {

constexpr int kCluster = 8, kThreads = 512;
constexpr uint32_t kChunk = 32768;  // tokens of a slice counted at a time (6 bytes each with biases)

struct LogitsLaunch {
  const void* logits;
  int64_t stride;
  uint32_t vocab, slice, chunk;  // slice: tokens per CTA; chunk: per pass over them (both multiples of 32)
  const int32_t* history;
  int64_t history_stride;
  uint32_t history_len;
  const int32_t *prompt_lens, *total_lens;
  const float *repetition, *frequency, *presence;
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t bias_stride;
  uint32_t max_bias;
  const uint32_t* mask;
  int64_t mask_stride;
  float* out;
  int64_t out_stride;
  int32_t* argmax;
};

CHPE_DEV unsigned long long order_key(float v, uint32_t idx) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 and +0 are equal
  const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)o << 32) | (unsigned long long)(0xFFFFFFFFu - idx);
}

template <typename T>
CHPE_DEV float to_float(T v);
template <>
CHPE_DEV float to_float<float>(float v) { return v; }
template <>
CHPE_DEV float to_float<__half>(__half v) { return __half2float(v); }
template <>
CHPE_DEV float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T>
CHPE_DEV void load4(const T* p, float (&x)[4]);
template <>
CHPE_DEV void load4<float>(const float* p, float (&x)[4]) {
  const float4 a = *reinterpret_cast<const float4*>(p);
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
}
template <>
CHPE_DEV void load4<__half>(const __half* p, float (&x)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a.x));
  const float2 g = __half22float2(*reinterpret_cast<const __half2*>(&a.y));
  x[0] = f.x, x[1] = f.y, x[2] = g.x, x[3] = g.y;
}
template <>
CHPE_DEV void load4<__nv_bfloat16>(const __nv_bfloat16* p, float (&x)[4]) {
  const uint2 a = *reinterpret_cast<const uint2*>(p);
  x[0] = __uint_as_float(a.x << 16), x[1] = __uint_as_float(a.x & 0xFFFF0000u);
  x[2] = __uint_as_float(a.y << 16), x[3] = __uint_as_float(a.y & 0xFFFF0000u);
}

// VEC: rows and the output start at multiples of four tokens' bytes.
template <typename T, bool HIST, bool BIAS, bool VEC>
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kThreads)
    logits_kernel(const __grid_constant__ LogitsLaunch P) {
  extern __shared__ __align__(16) unsigned char smem[];
  uint32_t* const counts = reinterpret_cast<uint32_t*>(smem);                       // [chunk]
  uint32_t* const which = reinterpret_cast<uint32_t*>(smem + (HIST ? 4 * P.chunk : 0));  // [chunk] 16-bit entries
  __shared__ unsigned long long best_of[kThreads / 32];
  __shared__ unsigned long long cta_best;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t tid = threadIdx.x, rank = cluster.block_rank();
  const int64_t row = blockIdx.x / kCluster;
  const uint32_t v_begin = min(rank * P.slice, P.vocab), v_end = min(v_begin + P.slice, P.vocab);
  const T* const x_row = static_cast<const T*>(P.logits) + row * P.stride;
  float* const out = P.out ? P.out + row * P.out_stride : nullptr;
  const uint32_t* const mask = P.mask ? P.mask + row * P.mask_stride : nullptr;
  const float* const bias_values = BIAS ? P.bias_values + row * P.bias_stride : nullptr;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  uint32_t total = 0, prompt = 0;
  if (HIST) {
    if (P.repetition) rep = P.repetition[row];
    if (P.frequency) freq = P.frequency[row];
    if (P.presence) pres = P.presence[row];
    const int n = P.total_lens ? P.total_lens[row] : (int)P.history_len;
    total = n < 0 ? 0u : min((uint32_t)n, P.history_len);
    const int p = P.prompt_lens ? P.prompt_lens[row] : 0;
    prompt = p < 0 ? 0u : (uint32_t)p;
  }

  float best = -INFINITY;
  uint32_t best_v = 0;
  auto rule = [&](float x, uint32_t v, uint32_t word, uint32_t entry) {
    if (HIST && word) {
      if (P.repetition) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
      const uint32_t n = word & 0x7FFFFFFFu;
      if (n) {
        if (P.frequency) x = __fsub_rn(x, __fmul_rn(freq, (float)n));
        if (P.presence) x = __fsub_rn(x, pres);
      }
    }
    if (BIAS && entry) x = __fadd_rn(x, bias_values[entry - 1]);
    return x;
  };
  auto offer = [&](float x, uint32_t v) {
    if (x > best) {
      best = x;
      best_v = v;
    }
  };

  for (uint32_t c0 = v_begin; c0 < v_end; c0 += P.chunk) {
    const uint32_t n = min(P.chunk, v_end - c0);
    if constexpr (HIST || BIAS) {
      if (c0 != v_begin) __syncthreads();  // the previous chunk's table is read
      const uint32_t words = (HIST ? P.chunk : 0) + (BIAS ? P.chunk / 2 : 0);
      for (uint32_t i = tid; i < words / 4; i += kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
      __syncthreads();
      if (HIST) {
        const int32_t* const h = P.history + row * P.history_stride;
        for (uint32_t i = tid; i < total; i += kThreads) {
          const uint32_t o = (uint32_t)h[i] - c0;  // ids outside the slice, negative ones too, are large
          if (o < n) {
            if (i < prompt) atomicOr(&counts[o], 0x80000000u);
            else atomicAdd(&counts[o], 1u);
          }
        }
      }
      if (BIAS) {
        const int32_t* const ids = P.bias_ids + row * P.bias_stride;
        for (uint32_t i = tid; i < P.max_bias; i += kThreads) {
          const uint32_t o = (uint32_t)ids[i] - c0;
          if (o < n) {  // the largest entry number of the token stays
            const uint32_t sh = (o & 1u) * 16u;
            uint32_t old = which[o >> 1];
            while (((old >> sh) & 0xFFFFu) < i + 1) {
              const uint32_t seen = atomicCAS(&which[o >> 1], old, (old & ~(0xFFFFu << sh)) | ((i + 1) << sh));
              if (seen == old) break;
              old = seen;
            }
          }
        }
      }
      __syncthreads();
    }
    if (VEC) {
      const uint32_t full = n & ~3u;
#pragma unroll 2
      for (uint32_t i = 4 * tid; i < full; i += 4 * kThreads) {
        const uint32_t v = c0 + i;
        float x[4];
        load4(x_row + v, x);
        const uint32_t bits = mask ? mask[v >> 5] >> (v & 31u) : 0xFu;
        uint4 w = make_uint4(0, 0, 0, 0);
        uint2 e = make_uint2(0, 0);
        if (HIST) w = *reinterpret_cast<const uint4*>(counts + i);
        if (BIAS) e = *reinterpret_cast<const uint2*>(which + (i >> 1));
        if ((HIST && (w.x | w.y | w.z | w.w)) || (BIAS && (e.x | e.y))) {
          x[0] = rule(x[0], v, w.x, e.x & 0xFFFFu);
          x[1] = rule(x[1], v + 1, w.y, e.x >> 16);
          x[2] = rule(x[2], v + 2, w.z, e.y & 0xFFFFu);
          x[3] = rule(x[3], v + 3, w.w, e.y >> 16);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
          if (!(bits >> j & 1u)) x[j] = -INFINITY;
          offer(x[j], v + j);
        }
        if (out) *reinterpret_cast<float4*>(out + v) = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
    for (uint32_t i = (VEC ? (n & ~3u) : 0u) + tid; i < n; i += kThreads) {
      const uint32_t v = c0 + i;
      float x = to_float<T>(x_row[v]);
      x = rule(x, v, HIST ? counts[i] : 0u, BIAS ? (which[i >> 1] >> ((i & 1u) * 16u)) & 0xFFFFu : 0u);
      if (mask && !(mask[v >> 5] >> (v & 31u) & 1u)) x = -INFINITY;
      offer(x, v);
      if (out) out[v] = x;
    }
  }
  if (!P.argmax) return;  // uniform over the grid

  unsigned long long key = best > -INFINITY ? order_key(best, best_v) : 0ull;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long k = __shfl_xor_sync(0xffffffffu, key, o);
    key = k > key ? k : key;
  }
  if ((tid & 31u) == 0) best_of[tid >> 5] = key;
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kThreads / 32; w++) key = best_of[w] > key ? best_of[w] : key;
    cta_best = key;
  }
  cluster.sync();
  if (rank == 0 && tid < 32) {
    key = tid < kCluster ? *cluster.map_shared_rank(&cta_best, tid) : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, key, o);
      key = k > key ? k : key;
    }
    if (tid == 0) P.argmax[row] = key ? (int32_t)(0xFFFFFFFFu - (uint32_t)(key & 0xFFFFFFFFull)) : -1;
  }
  cluster.sync();  // the other CTAs' shared memory stays until it is read
}

template <typename T, bool HIST, bool BIAS, bool VEC>
cudaError_t launch(const LogitsLaunch& P, uint32_t batch, int device, cudaStream_t s) {
  const int bytes = (int)(P.chunk * ((HIST ? 4 : 0) + (BIAS ? 2 : 0)));
  if (bytes > 48 * 1024) {
    static int set[64] = {};  // per device: done once
    const int dev = device >= 0 && device < 64 ? device : -1;
    if (dev < 0 || !__atomic_load_n(&set[dev], __ATOMIC_RELAXED)) {
      const cudaError_t e = cudaFuncSetAttribute(logits_kernel<T, HIST, BIAS, VEC>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)(kChunk * ((HIST ? 4 : 0) + (BIAS ? 2 : 0))));
      if (e != cudaSuccess) return e;
      if (dev >= 0) __atomic_store_n(&set[dev], 1, __ATOMIC_RELAXED);
    }
  }
  logits_kernel<T, HIST, BIAS, VEC><<<batch * kCluster, kThreads, bytes, s>>>(P);
  return cudaGetLastError();
}

template <typename T, bool VEC>
cudaError_t launch_rules(const LogitsLaunch& P, uint32_t batch, int device, cudaStream_t s) {
  if (P.history && P.bias_ids) return launch<T, true, true, VEC>(P, batch, device, s);
  if (P.history) return launch<T, true, false, VEC>(P, batch, device, s);
  if (P.bias_ids) return launch<T, false, true, VEC>(P, batch, device, s);
  return launch<T, false, false, VEC>(P, batch, device, s);
}

template <typename T>
cudaError_t launch_type(const LogitsLaunch& P, uint32_t batch, bool vec, int device, cudaStream_t s) {
  return vec ? launch_rules<T, true>(P, batch, device, s) : launch_rules<T, false>(P, batch, device, s);
}

}  // namespace

extern "C" int chpe_logits_process(const void* logits, int dtype, int64_t logits_stride, uint32_t batch,
                                   uint32_t vocab, const int32_t* history, int64_t history_stride,
                                   uint32_t history_len, const int32_t* prompt_lens, const int32_t* total_lens,
                                   const float* repetition, const float* frequency, const float* presence,
                                   const int32_t* bias_ids, const float* bias_values, int64_t bias_stride,
                                   uint32_t max_bias, const uint32_t* mask, int64_t mask_stride, float* out,
                                   int64_t out_stride, int32_t* argmax, void* stream) {
  chpe::ServeCall c("chpe_logits_process");
  const size_t es = chpe::dtype_size(dtype);
  if (!es) return c.fail(-1, "unknown dtype %lld", dtype), c.done();
  if (vocab == 0 || vocab > 0x7fffffffu) return c.fail(-1, "vocab must be 1..2^31-1"), c.done();
  if (batch > (1u << 24)) return c.fail(-1, "batch must be at most 2^24"), c.done();
  if (!out && !argmax) return c.fail(-1, "neither out nor argmax to write"), c.done();
  if ((prompt_lens || total_lens || repetition || frequency || presence) && !history)
    return c.fail(-1, "lengths or penalties without a history"), c.done();
  if (!bias_ids != !bias_values) return c.fail(-1, "bias_ids and bias_values go together"), c.done();
  if (bias_ids && max_bias > 65535) return c.fail(-1, "at most 65535 biases per row"), c.done();
  if (history_len > 0x7fffffffu) return c.fail(-1, "history_len must be below 2^31"), c.done();
  const int64_t words = ((int64_t)vocab + 31) / 32;
  if (batch > 1) {
    const int64_t most = INT64_MAX / 8 / batch;
    if (logits_stride < (int64_t)vocab || logits_stride > most) return c.fail(-1, "logits_stride must be at least vocab"), c.done();
    if (out && (out_stride < (int64_t)vocab || out_stride > most)) return c.fail(-1, "out_stride must be at least vocab"), c.done();
    if (history && (history_stride < (int64_t)history_len || history_stride > most))
      return c.fail(-1, "history_stride must be at least history_len"), c.done();
    // a stride of 0 gives every row the same list or mask
    if (bias_ids && bias_stride != 0 && (bias_stride < (int64_t)max_bias || bias_stride > most))
      return c.fail(-1, "bias_stride must be 0 or at least max_bias"), c.done();
    if (mask && mask_stride != 0 && (mask_stride < words || mask_stride > most))
      return c.fail(-1, "mask_stride must be 0 or at least %lld words", words), c.done();
  }
  if (batch == 0) return c.done();
  c.ptr(logits, "logits", es);
  if (history && history_len) c.ptr(history, "history", 4);
  c.ptr_or_null(prompt_lens, "prompt_lens", 4);
  c.ptr_or_null(total_lens, "total_lens", 4);
  c.ptr_or_null(repetition, "repetition", 4);
  c.ptr_or_null(frequency, "frequency", 4);
  c.ptr_or_null(presence, "presence", 4);
  if (bias_ids && max_bias) {
    c.ptr(bias_ids, "bias_ids", 4);
    c.ptr(bias_values, "bias_values", 4);
  }
  c.ptr_or_null(mask, "mask", 4);
  c.ptr_or_null(out, "out", 4);
  c.ptr_or_null(argmax, "argmax", 4);
  if (c.rc) return c.done();

  LogitsLaunch P{};
  P.logits = logits, P.stride = logits_stride, P.vocab = vocab;
  const uint32_t each = (uint32_t)(((uint64_t)vocab + kCluster - 1) / kCluster);
  P.slice = (each + 31u) & ~31u;
  P.chunk = P.slice < kChunk ? P.slice : kChunk;
  if (history_len) P.history = history, P.history_stride = history_stride, P.history_len = history_len;
  P.prompt_lens = prompt_lens, P.total_lens = total_lens;
  P.repetition = repetition, P.frequency = frequency, P.presence = presence;
  if (max_bias) P.bias_ids = bias_ids, P.bias_values = bias_values, P.bias_stride = bias_stride, P.max_bias = max_bias;
  P.mask = mask, P.mask_stride = mask_stride;
  P.out = out, P.out_stride = out_stride, P.argmax = argmax;
  const bool vec = reinterpret_cast<uintptr_t>(logits) % (4 * es) == 0 && (batch == 1 || logits_stride % 4 == 0) &&
                   (!out || (reinterpret_cast<uintptr_t>(out) % 16 == 0 && (batch == 1 || out_stride % 4 == 0)));
  chpe::DeviceScope scope(c.device);
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (dtype == CHPE_F32) e = launch_type<float>(P, batch, vec, c.device, s);
  else if (dtype == CHPE_F16) e = launch_type<__half>(P, batch, vec, c.device, s);
  else e = launch_type<__nv_bfloat16>(P, batch, vec, c.device, s);
  if (e != cudaSuccess) {
    snprintf(c.msg, sizeof(c.msg), "launch: %s", cudaGetErrorString(e));
    c.rc = -3;
  }
  return c.done();
}
