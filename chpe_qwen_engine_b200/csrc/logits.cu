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
// Bound by memory: the logits in, the f32 logits out.  A cluster of 8 or 16 CTAs
// takes one row; tiles of 128 tokens (a warp's four per lane) go to the CTAs in turn, so
// that the frequent tokens, which have low ids, are spread over them.  Three steps:
//   1. table: the CTA's tokens of the history are counted in shared memory (one
//      entry per token: the top bit seen in the prompt, the rest the count after it;
//      16-bit entries unless the history is longer than they count), its biases
//      entered.  Integer atomics, whose order does not matter; the prompt's bits are read
//      before they are set, since many threads meet at the frequent tokens;
//   2. stream: the CTA's tokens once, four per thread and step, kAhead steps' loads in
//      flight (the first ones issued before step 1), the mask applied; tokens with an
//      entry are left out of the comparison;
//   3. rules: the tokens with an entry, which step 2 put on a list, one per thread
//      whatever their place: their logits are worked out and written over what step 2
//      left there.
// The CTAs join their best tokens through distributed shared memory: no
// workspace, no second launch.  Without history and biases only step 2 is left.
// 256 rows of 151936 BF16 logits: 55 us as they are (4.2 TB/s; a plain cast of
// them to f32 by the library takes 103), 70 with histories of up to 8191.  In
// place, only what changes is written.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "device_common.cuh"
#include "serve_common.h"

namespace {

constexpr uint32_t kMaxCluster = 16;
constexpr int kMaxThreads = 512;
constexpr uint32_t kTile = 128;
constexpr uint32_t kChunk = 28672;  // most tokens of a CTA counted at a time (up to 8 bytes each)
constexpr int kAhead = 4;  // steps of the stream, and
constexpr int kIds = 4;    // ids of the history, whose loads a thread has in flight

struct LogitsLaunch {
  const void* logits;
  int64_t stride;
  uint32_t lg;  // log2 of the CTAs of a row
  uint32_t vocab, chunk;  // chunk: tokens a CTA takes at a time (a multiple of kTile)
  const int32_t* history;
  int64_t history_stride;
  uint32_t history_len;
  const int32_t *prompt_lens, *total_lens;
  const float *repetition, *frequency, *presence;
  const int32_t* bias_ids;
  const float* bias_values;
  int64_t bias_stride;
  uint32_t max_bias;
  uint32_t slots, slot_shift;  // places for bias entries: chunk (one per token), or 2^(32 - slot_shift)
  const uint32_t* mask;
  int64_t mask_stride;
  float* out;
  int64_t out_stride;
  int32_t in_place;  // out is the logits: what the mask leaves as it is need not be written
  int32_t* argmax;
};

CHPE_DEV unsigned long long order_key(float v, uint32_t idx) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 and +0 are equal
  const uint32_t o = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)o << 32) | (unsigned long long)(0xFFFFFFFFu - idx);
}

// ---- cluster: rank, barrier in two halves, a store to another CTA's shared memory
CHPE_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
CHPE_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
CHPE_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
CHPE_DEV void put_cluster(unsigned long long* p, uint32_t rank, unsigned long long v) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}

template <typename T>
CHPE_DEV float to_float(T v);
template <>
CHPE_DEV float to_float<float>(float v) { return v; }
template <>
CHPE_DEV float to_float<__half>(__half v) { return __half2float(v); }
template <>
CHPE_DEV float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }

// Four logits as they lie in memory, and as f32.
template <typename T>
struct Raw4 {
  uint32_t w[sizeof(T)];
  CHPE_DEV void load(const T* p) {
    if constexpr (sizeof(T) == 4) {
      const uint4 a = *reinterpret_cast<const uint4*>(p);
      w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    } else {
      const uint2 a = *reinterpret_cast<const uint2*>(p);
      w[0] = a.x, w[1] = a.y;
    }
  }
  CHPE_DEV void get(float (&x)[4]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < 4; i++) x[i] = __uint_as_float(w[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
      }
    }
  }
};

// E: bytes of a table entry (0: neither history nor biases).  VEC: rows and the
// output start at multiples of four tokens' bytes.
// At most 64 registers, so that four CTAs of 256 threads share an SM (with 68, 64 rows
// with a history took 27.9 us instead of 20.0).
template <typename T, int E, bool BIAS, bool VEC>
__global__ void __launch_bounds__(kMaxThreads, 2) logits_kernel(const __grid_constant__ LogitsLaunch P) {
  constexpr uint32_t kSeen = E == 2 ? 0x8000u : 0x80000000u, kBiased = kSeen >> 1;
  extern __shared__ __align__(16) unsigned char smem[];
  uint32_t* const table = reinterpret_cast<uint32_t*>(smem);  // [chunk] entries of E bytes
  uint32_t* const which = table + P.chunk / 4 * E;            // [slots] entry numbers of 16 bits
  uint16_t* const list = reinterpret_cast<uint16_t*>(which + (BIAS ? P.slots / 2 : 0));  // tokens with an entry
  __shared__ uint32_t listed;
  __shared__ unsigned long long best_of[kMaxThreads / 32];
  __shared__ unsigned long long cta_best[kMaxCluster];
  const uint32_t tid = threadIdx.x, rank = cluster_rank(), nt = blockDim.x;
  pdl_wait();
  pdl_launch_dependents();
  if (P.argmax) cluster_arrive();  // every CTA of the cluster has started: waited for at the end
  const int64_t row = blockIdx.x >> P.lg;
  const T* const x_row = static_cast<const T*>(P.logits) + row * P.stride;
  float* const out = P.out ? P.out + row * P.out_stride : nullptr;
  const uint32_t* const mask = P.mask ? P.mask + row * P.mask_stride : nullptr;
  // the CTA's i-th token, and the place of token v among them (0xFFFFFFFF: another CTA's, or none)
  auto token = [&](uint32_t i) { return (((i / kTile) << P.lg) + rank) * kTile + i % kTile; };
  auto place = [&](uint32_t v) {
    const uint32_t tile = v / kTile;
    return v < P.vocab && (tile & ((1u << P.lg) - 1u)) == rank ? (tile >> P.lg) * kTile + v % kTile : 0xFFFFFFFFu;
  };
  // where the search for a biased token's entry begins
  auto slot_of = [&](uint32_t o) { return P.slots == P.chunk ? o : (o * 0x9E3779B1u) >> P.slot_shift; };
  const uint32_t tiles = (P.vocab + kTile - 1) / kTile;
  const uint32_t mine = rank < tiles ? (((tiles - rank - 1) >> P.lg) + 1) * kTile : 0;  // the last may be cut

  float best = -INFINITY;
  uint32_t best_v = 0;
  auto offer = [&](float x, uint32_t v) {  // in any order: of equals the lowest
    if (x > best || (x == best && v < best_v && x > -INFINITY)) {
      best = x;
      best_v = v;
    }
  };
  // what the later steps wait for is asked for first: the row's lengths and penalties,
  // the first ids of its history and its first bias
  uint32_t total = 0, prompt = 0, first_id[kIds], first_bias = 0xFFFFFFFFu;
  float rep = 1.f, freq = 0.f, pres = 0.f;
  const int32_t* const hist = P.history ? P.history + row * P.history_stride : nullptr;
  const int32_t* const ids = BIAS ? P.bias_ids + row * P.bias_stride : nullptr;
  if constexpr (E != 0) {
    if (hist) {
#pragma unroll
      for (int j = 0; j < kIds; j++) first_id[j] = tid + j * nt < P.history_len ? (uint32_t)hist[tid + j * nt] : 0xFFFFFFFFu;
      const int m = P.total_lens ? P.total_lens[row] : (int)P.history_len;
      total = m < 0 ? 0u : min((uint32_t)m, P.history_len);
      const int p = P.prompt_lens ? P.prompt_lens[row] : 0;
      prompt = p < 0 ? 0u : (uint32_t)p;
      if (P.repetition) rep = P.repetition[row];
      if (P.frequency) freq = P.frequency[row];
      if (P.presence) pres = P.presence[row];
    }
    if (BIAS && tid < P.max_bias) first_bias = (uint32_t)ids[tid];
  }
  for (uint32_t c0 = 0; c0 < mine; c0 += P.chunk) {
    const uint32_t n = min(P.chunk, mine - c0);
    Raw4<T> raw[kAhead];
    uint32_t bits[kAhead];
    auto fetch = [&](int u, uint32_t i) {
      const uint32_t v = token(c0 + i);
      if (i < n && v + 4 <= P.vocab) {
        raw[u].load(x_row + v);
        if (mask) bits[u] = mask[v >> 5];
      }
    };
    if constexpr (VEC)
#pragma unroll
      for (int u = 0; u < kAhead; u++) fetch(u, 4 * (tid + u * nt));

    if constexpr (E != 0) {
      if (c0) __syncthreads();  // the previous chunk's table is read
      const uint32_t words = P.chunk / 4 * E + (BIAS ? P.slots / 2 : 0);
      for (uint32_t i = tid; i < words / 4; i += nt) reinterpret_cast<uint4*>(table)[i] = make_uint4(0, 0, 0, 0);
      if (tid == 0) listed = 0;
      __syncthreads();
      auto flag = [&](uint32_t o, uint32_t f) {
        const uint32_t sh = E == 2 ? (o & 1u) * 16u : 0u;
        uint32_t* const at = table + (E == 2 ? o >> 1 : o);
        if (!(*reinterpret_cast<volatile uint32_t*>(at) & f << sh)) atomicOr(at, f << sh);
      };
      for (uint32_t i0 = tid; i0 < total; i0 += kIds * nt) {
        uint32_t id[kIds];
#pragma unroll
        for (int j = 0; j < kIds; j++)
          id[j] = i0 + j * nt >= total ? 0xFFFFFFFFu : i0 == tid ? first_id[j] : (uint32_t)hist[i0 + j * nt];
#pragma unroll
        for (int j = 0; j < kIds; j++) {
          const uint32_t o = place(id[j]) - c0;
          if (o >= n) continue;
          if (i0 + j * nt < prompt) flag(o, kSeen);
          else atomicAdd(table + (E == 2 ? o >> 1 : o), 1u << (E == 2 ? (o & 1u) * 16u : 0u));
        }
      }
      if constexpr (BIAS) {
        for (uint32_t i = tid; i < P.max_bias; i += nt) {
          const uint32_t id = i == tid ? first_bias : (uint32_t)ids[i], o = place(id) - c0;
          if (o >= n) continue;
          flag(o, kBiased);
          uint32_t k = slot_of(o);  // at most half of the slots are taken: the search ends before it is back
          for (uint32_t tries = 0; tries < P.slots; tries++, k = k + 1 < P.slots ? k + 1 : 0) {
            const uint32_t sh = (k & 1u) * 16u;
            uint32_t* const at = which + (k >> 1);
            uint32_t old = *reinterpret_cast<volatile uint32_t*>(at);
            bool done = false;
            // an empty slot, or the token's own with a smaller number: the largest number stays
            for (;;) {
              const uint32_t e = old >> sh & 0xFFFFu;
              if (e && (uint32_t)ids[e - 1] != id) break;
              done = true;
              if (e > i) break;
              const uint32_t seen = atomicCAS(at, old, (old & ~(0xFFFFu << sh)) | ((i + 1) << sh));
              if (seen == old) break;
              done = false;
              old = seen;
            }
            if (done) break;
          }
        }
      }
      __syncthreads();
    }
    // bit j: token i + j of the chunk has an entry
    auto entries4 = [&](uint32_t i) {
      uint32_t b = 0;
      if constexpr (E == 2) {
        const uint2 c = *reinterpret_cast<const uint2*>(table + i / 2);
        if (c.x | c.y) b = (c.x & 0xFFFFu ? 1u : 0u) | (c.x >> 16 ? 2u : 0u) | (c.y & 0xFFFFu ? 4u : 0u) | (c.y >> 16 ? 8u : 0u);
      } else if constexpr (E == 4) {
        const uint4 c = *reinterpret_cast<const uint4*>(table + i);
        if (c.x | c.y | c.z | c.w) b = (c.x ? 1u : 0u) | (c.y ? 2u : 0u) | (c.z ? 4u : 0u) | (c.w ? 8u : 0u);
      }
      return b;
    };

    if constexpr (VEC) {
      for (uint32_t i0 = 4 * tid; i0 < n; i0 += 4 * kAhead * nt) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
          const uint32_t i = i0 + 4 * u * nt, v = token(c0 + i);
          if (i >= n || v + 4 > P.vocab) break;  // later ones are larger
          float x[4];
          raw[u].get(x);
          const uint32_t allowed = bits[u] >> (i & 31u);
          fetch(u, i + 4 * kAhead * nt);
          if (mask) {
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = allowed >> j & 1u ? x[j] : -INFINITY;
          }
          if (out && !(P.in_place && (!mask || (allowed & 0xFu) == 0xFu))) *reinterpret_cast<float4*>(out + v) = make_float4(x[0], x[1], x[2], x[3]);
          if constexpr (E != 0) {  // tokens that step 3 comes back to
            const uint32_t later = entries4(i);
            if (later) {
              uint32_t at = atomicAdd(&listed, __popc(later));
#pragma unroll
              for (int j = 0; j < 4; j++)
                if (later >> j & 1u) {
                  x[j] = -INFINITY;
                  list[at++] = (uint16_t)(i + j);
                }
            }
          }
          const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));  // passes over NaN
          if (top > best) {  // a thread's tokens come in ascending order
            best = top;
            best_v = v + (x[0] == top ? 0u : x[1] == top ? 1u : x[2] == top ? 2u : 3u);
          }
        }
      }
    }
    // one by one: all tokens, or those behind the last whole four
    for (uint32_t i = VEC ? n - min(n, kTile) + tid : tid; i < n; i += nt) {
      const uint32_t v = token(c0 + i);
      if (v >= P.vocab || (VEC && v < (P.vocab & ~3u))) continue;
      float x = to_float<T>(x_row[v]);
      const bool banned = mask && !(mask[v >> 5] >> (v & 31u) & 1u);
      if (banned) x = -INFINITY;
      if (out && (banned || !P.in_place)) out[v] = x;
      bool open = true;
      if constexpr (E != 0) open = !(entries4(i & ~3u) >> (i & 3u) & 1u);
      if (open) offer(x, v);
      else list[atomicAdd(&listed, 1u)] = (uint16_t)i;
    }

    if constexpr (E != 0) {
      __syncthreads();  // step 3 writes over what other threads wrote
      for (uint32_t k = tid; k < listed; k += nt) {
        const uint32_t o = list[k], v = token(c0 + o);
        float x = to_float<T>(x_row[v]);  // in place a forbidden token's logit is gone: it is -inf whatever it was
        const uint32_t allowed = mask ? mask[v >> 5] >> (v & 31u) & 1u : 1u;
        const uint32_t word = E == 2 ? table[o >> 1] >> ((o & 1u) * 16u) & 0xFFFFu : table[o];
        if (word & ~kBiased && P.repetition) x = x > 0.f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
        const uint32_t c = word & (kBiased - 1u);
        if (c && P.frequency) x = __fsub_rn(x, __fmul_rn(freq, (float)c));
        if (c && P.presence) x = __fsub_rn(x, pres);
        if constexpr (BIAS) {
          if (word & kBiased) {
            uint32_t k = slot_of(o);
            for (uint32_t tries = 0; tries < P.slots; tries++, k = k + 1 < P.slots ? k + 1 : 0) {
              const uint32_t e = which[k >> 1] >> ((k & 1u) * 16u) & 0xFFFFu;
              if (e && (uint32_t)ids[e - 1] != v) continue;  // another token's
              if (e) x = __fadd_rn(x, P.bias_values[row * P.bias_stride + e - 1]);
              break;
            }
          }
        }
        if (!allowed) x = -INFINITY;
        if (out) out[v] = x;
        offer(x, v);
      }
    }
  }
  if (!P.argmax) return;  // uniform over the grid

  unsigned long long key = best > -INFINITY ? order_key(best, best_v) : 0ull;
  auto warp_key = [&] {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long k = __shfl_xor_sync(0xffffffffu, key, o);
      key = k > key ? k : key;
    }
  };
  warp_key();
  if ((tid & 31u) == 0) best_of[tid >> 5] = key;
  __syncthreads();
  if (tid >= 32) return;  // one warp closes the CTA; the others count as arrived
  key = tid < nt / 32 ? best_of[tid] : 0ull;
  warp_key();
  cluster_wait();
  if (tid == 0) put_cluster(&cta_best[rank], 0, key);
  cluster_arrive();  // rank 0 alone stays for the others' keys
  if (rank != 0) return;
  cluster_wait();
  key = tid < 1u << P.lg ? *reinterpret_cast<volatile unsigned long long*>(&cta_best[tid]) : 0ull;
  warp_key();
  if (tid == 0) P.argmax[row] = key ? (int32_t)(0xFFFFFFFFu - (uint32_t)(key & 0xFFFFFFFFull)) : -1;
}

template <typename T, int E, bool BIAS, bool VEC>
cudaError_t launch(LogitsLaunch P, uint32_t batch, int device, cudaStream_t s) {
  if (BIAS) {
    // twice as many slots as entries, hashed; or, where that is as much, one per token
    P.slots = 32, P.slot_shift = 27;
    while (P.slots < 2 * P.max_bias) P.slots *= 2, P.slot_shift--;
    if (P.slots >= P.chunk) P.slots = P.chunk;
  }
  // table, slots, and room on the list for every token that can have an entry
  uint64_t entries = (P.history ? P.history_len : 0u) + (uint64_t)(BIAS ? P.max_bias : 0u);
  if (entries > P.chunk) entries = P.chunk;
  const int bytes = E ? (int)(P.chunk * E + (BIAS ? 2 * P.slots : 0) + 2 * entries) : 0;
  auto kernel = logits_kernel<T, E, BIAS, VEC>;
  static int set[64] = {};  // per device: done once
  const int dev = device >= 0 && device < 64 ? device : -1;
  if (dev < 0 || !__atomic_load_n(&set[dev], __ATOMIC_RELAXED)) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               (int)(kChunk * (E + (BIAS ? 2 : 0) + 2)));
    if (e != cudaSuccess) return e;
    if (dev >= 0) __atomic_store_n(&set[dev], 1, __ATOMIC_RELAXED);
  }
  chpe::ServeLaunch L(dim3(batch << P.lg), batch <= 32 ? 512 : 256, bytes, s, 1u << P.lg);
  return cudaLaunchKernelEx(&L.cfg, kernel, P);
}

template <typename T, bool VEC>
cudaError_t launch_rules(const LogitsLaunch& P, uint32_t batch, int device, cudaStream_t s) {
  if (!P.history && !P.bias_ids) return launch<T, 0, false, VEC>(P, batch, device, s);
  if (P.history && P.history_len > 0x3FFFu)  // more than 14 bits count
    return P.bias_ids ? launch<T, 4, true, VEC>(P, batch, device, s) : launch<T, 4, false, VEC>(P, batch, device, s);
  return P.bias_ids ? launch<T, 2, true, VEC>(P, batch, device, s) : launch<T, 2, false, VEC>(P, batch, device, s);
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
  if (batch == 0) return c.done();
  if (!out && !argmax) return c.fail(-1, "neither out nor argmax to write"), c.done();
  if ((prompt_lens || total_lens || repetition || frequency || presence) && !history)
    return c.fail(-1, "lengths or penalties without a history"), c.done();
  if (!bias_ids != !bias_values) return c.fail(-1, "bias_ids and bias_values go together"), c.done();
  if (bias_ids && max_bias > 65535) return c.fail(-1, "at most 65535 biases per row"), c.done();
  if (history_len > 0x3fffffffu) return c.fail(-1, "history_len must be below 2^30"), c.done();
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
  const bool in_place = dtype == CHPE_F32 && out == logits && (batch == 1 || out_stride == logits_stride);
  {
    using chpe::Rows;
    const int64_t n = batch, v = vocab;
    const Rows in[] = {{"history", history, 4ll * history_len, n, history_stride, 4},
                       {"logits", logits, v * (int64_t)es, n, logits_stride, (int64_t)es},
                       {"bias_ids", bias_ids, 4ll * max_bias, n, bias_stride, 4}, {"bias_values", bias_values, 4ll * max_bias, n, bias_stride, 4},
                       {"mask", mask, 4 * words, n, mask_stride, 4}, {"prompt_lens", prompt_lens, 4 * n},
                       {"total_lens", total_lens, 4 * n}, {"repetition", repetition, 4 * n},
                       {"frequency", frequency, 4 * n}, {"presence", presence, 4 * n}};
    const Rows x("out", out, 4 * v, n, out_stride, 4), t("argmax", argmax, 4 * n);
    for (int i = 0; i < 10; i++) {
      if (!(i == 1 && in_place)) c.apart(x, in[i]);
      // (one row's token may go behind its history: it is written when all has been read)
      if (!(i == 0 && n == 1)) c.apart(t, in[i]);
    }
    c.apart(x, t);
    if (c.rc) return c.done();
  }

  LogitsLaunch P{};
  P.logits = logits, P.stride = logits_stride, P.vocab = vocab;
  // Few rows are waited for by their loads: 16 CTAs of 512 threads each.  Many
  // overlap one another's phases best when the CTAs are small.  All rules, rows of 152064,
  // us with 16 x 512 / 8 x 512 / 8 x 256: 5 rows 7.4 / 9.6 / 12.0, 14 rows 9.8 / 9.9 /
  // 12.4, 18 rows 15.2 / 12.5 / 14.1, 32 rows 25 / 14.1 / 16.6, 48 rows 34 / 24.5 / 19.3.
  P.lg = batch <= 14 ? 4 : 3;
  const uint32_t tiles = (vocab + kTile - 1) / kTile, each = (tiles + (1u << P.lg) - 1) >> P.lg;
  P.chunk = each < kChunk / kTile ? each * kTile : kChunk;
  if (history_len) P.history = history, P.history_stride = history_stride, P.history_len = history_len;
  P.prompt_lens = prompt_lens, P.total_lens = total_lens;
  P.repetition = repetition, P.frequency = frequency, P.presence = presence;
  if (max_bias) P.bias_ids = bias_ids, P.bias_values = bias_values, P.bias_stride = bias_stride, P.max_bias = max_bias;
  P.mask = mask, P.mask_stride = mask_stride;
  P.out = out, P.out_stride = out_stride, P.argmax = argmax;
  P.in_place = in_place;
  const bool vec = reinterpret_cast<uintptr_t>(logits) % (4 * es) == 0 && (batch == 1 || logits_stride % 4 == 0) &&
                   (!out || (reinterpret_cast<uintptr_t>(out) % 16 == 0 && (batch == 1 || out_stride % 4 == 0)));
  chpe::DeviceScope scope(c.launch_device());
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
