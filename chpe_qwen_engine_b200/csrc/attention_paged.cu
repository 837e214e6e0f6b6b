// attention_paged.cu -- decode attention of a batch of sequences over a paged
// K/V cache: one new token per sequence, page tables and lengths on the device.
//
//   out[b,h] = sum_t p[t] v[t],  p = softmax over t < len[b] of scale * q[b,h].k[t]
//   lse[b,h] = log sum_t exp(scale * q[b,h].k[t])
//
// with position t of sequence b in row t % page of page table[b][t / page].
// Query heads h*G .. h*G+G-1 share kv head h.  Bound by memory: every K and V
// row is read once, 4*H/KV flops for each 2 elements.
//
// Work split.  A CTA takes several kv heads of the same positions at once, a warp
// each, because a position's heads lie side by side in the cache: what a CTA reads
// is then whole pages, not a 256-byte row of every 2 KB (one head per CTA
// took 162 us instead of 124, all else alike, for a batch of 64 on 64/8 heads of 128).  Where there are
// fewer heads than warps the remaining warps take further 16-position units of
// the tile.  The work is a line of tiles: sequence by sequence, group of heads by
// group, tile by tile, and CTA c of C takes the c-th of C equal stretches,
// whatever sequences lie in it.  A batch of very different lengths, one long
// sequence and many short ones all fill the GPU alike, and the host never learns
// a length (a captured graph stays valid as sequences grow).  A sequence's group that
// lies in one CTA is finished there; of one cut between CTAs each writes partial
// records (values, maximum, sum per query head) and combine_kernel, launched behind with
// programmatic dependent launch, joins them in the order of the positions: results do
// not depend on timing.
//
// Each warp has a ring of its own in shared memory (cp.async, 16-byte chunks
// XOR-swizzled by row so that ldmatrix is free of bank conflicts) that runs
// ahead across the ends of sequences, a running maximum and sums in registers, and
// waits for no other warp; only warps that share a head meet, at the end of a part.
//
// Measured (device time, replayed from a graph): 131071 positions of one sequence on 64/8
// heads of 128 in BF16: 93 us, 89 % of the copy rate; 64 sequences of up to 8192 there: 122 us, 92 %, with
// float queries 120; 37 of up to 4093 on 16/4 heads of 256: 43.5 us, 75 %; one of 77 on 16/2 heads: 8 us.
// What is left: SMs get bandwidth unevenly, so that CTAs with equal shares end
// 10 % before and after the mean, and the records' join, 3 us behind a gap of 2.
// Handing a fifth of the line out to whoever is done evened the ends out but cost as
// much in more, shorter parts.
//
// Matrix instructions: mma.sync m16n8k16 on the transposed products, S^T = K Q^T
// and O^T = V^T P^T: the cache's rows fill the instruction's 16-row operand and
// the 8 query heads of a kv head its 8 columns, so that nothing is padded, and the
// sums take half the registers of the untransposed form (D=256: 64 instead of 128 per
// lane).  P^T comes out of S^T by movmatrix.  Queries of the cache's type go in as
// they are; float ones as two FP16 or three BF16 parts (22 and 24 bits), each a
// column operand of its own, and so do the probabilities, held times 2^14 over
// FP16, which keeps the small ones.  A tile's products are summed from zero and then
// added to the running sums in f32, because the instruction cuts what it adds to its
// accumulator: over 131071 positions the output was off by 3.2e-6 of its norm, now by 4.5e-7
// (f32 products by the library: 5.8e-7), for 93 us instead of 92.  tcgen05.mma would need its operands in shared memory or TMEM in
// layouts of 128 rows for 8 columns of work; the tensor pipe is busy 14 to 19 % of the time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "device_common.cuh"
#include "serve_common.h"

namespace {

constexpr int kUnit = 16;          // positions a warp takes at a time
constexpr int kHeads = 8;          // query heads of a column operand
constexpr int kBegin = 3;          // tiles that beginning a sequence's group costs (its query, records, refill)
// Probabilities are held times 2^kPShift: over FP16, whose parts end at 2^-24, so that small
// ones are kept; over BF16 as they are (times 2^14, values above 2^113 of a single
// position went beyond f32).
template <typename T>
constexpr float kPShift = std::is_same<T, __half>::value ? 14.f : 0.f;

struct PagedLaunch {
  const void* q;
  int64_t q_stride;
  const void *kc, *vc;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* lens;
  uint32_t n_pages, page_shift;
  int32_t cap;  // positions a table row can hold
  int32_t B, H, KV, G, HT;  // HT: virtual heads (of up to 8 N query heads) per kv head
  int32_t HW, groups;       // virtual heads of a CTA (a power of two); groups of them
  int32_t tile_shift;       // log2 of a tile's positions: 16 for each warp that shares a head
  float scale;
  void* out;
  int64_t out_stride;
  float* lse;
  float* part;  // records [2 * grid][HW]
  int4* desc;   // cuts: sequence, group, number of CTAs (0: not cut), the first of them
  float p_shift;   // kPShift of the cache's type
  int32_t by_seq;  // a desc entry for each sequence and group (they are at most `grid`); else for each CTA
};

template <typename T>
CHPE_DEV uint32_t pack2(float a, float b);
template <>
CHPE_DEV uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
CHPE_DEV uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <typename T>
CHPE_DEV float2 unpack2(uint32_t w);
template <>
CHPE_DEV float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <>
CHPE_DEV float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

template <typename T>
CHPE_DEV void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
CHPE_DEV void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
CHPE_DEV void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CHPE_DEV void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The 8x8 matrix of a warp's register (row lane / 4, two columns each), transposed.
CHPE_DEV uint32_t transpose8(uint32_t a) {
  uint32_t d;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
CHPE_DEV void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// 16 bytes global -> shared; zeros when !on (the address is not read)
CHPE_DEV void cp16_if(uint32_t dst, const void* src, bool on) {
  const int n = on ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
CHPE_DEV void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
CHPE_DEV void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
CHPE_DEV void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Two neighbours of a query row (their address is a multiple of their size).
template <typename T>
CHPE_DEV float2 load2(const T* p) {
  if constexpr (std::is_same<T, float>::value) return *reinterpret_cast<const float2*>(p);
  else return unpack2<T>(*reinterpret_cast<const uint32_t*>(p));
}
template <typename T>
CHPE_DEV void store2(T* p, float a, float b) {
  if constexpr (std::is_same<T, float>::value) *reinterpret_cast<float2*>(p) = make_float2(a, b);
  else *reinterpret_cast<uint32_t*>(p) = pack2<T>(a, b);
}
template <typename T>
CHPE_DEV void store1(T* p, float v) {
  if constexpr (std::is_same<T, float>::value) *p = v;
  else if constexpr (std::is_same<T, __half>::value) *p = __float2half_rn(v);
  else *p = __float2bfloat16_rn(v);
}

CHPE_DEV int seq_len(const PagedLaunch& P, int b) {
  const int n = P.lens[b];
  return max(0, min(n, P.cap));
}
CHPE_DEV int tiles_of(const PagedLaunch& P, int len) { return (len + (1 << P.tile_shift) - 1) >> P.tile_shift; }
// Places of one sequence's group on the line: its tiles, behind kBegin that stand
// for what beginning it costs (without them, 64 sequences of up to 1024 took 32.0 us
// instead of 25.6: the CTAs with the short ones were last).
CHPE_DEV int places_of(int tiles) { return tiles ? tiles + kBegin : 0; }

// N: column operands of a warp, 8 query heads each.
template <int D, int N>
struct Cfg {
  static constexpr int kWarps = D == 256 ? 4 : 8;
  static constexpr int kRow = D * 2;                    // bytes of a cache row of one head
  static constexpr int kStageBytes = 2 * kUnit * kRow;  // K and V of one unit
  static constexpr int kStages = 3;
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kSums = D * 8 + 16;              // floats that a warp hands to another of its head
  static constexpr int kWarpHeads = N * kHeads;         // query heads of a warp (a "virtual" kv head)
  static constexpr int kRec = kWarpHeads * (D + 2);     // floats of a warp's record: values, then (max, sum) of each head
  static constexpr int kMaxCtas = D == 64 ? 320 : 160;  // grid limit, sizes the workspace
};

// A place on the line of tiles, and the stretch of one sequence's group that
// begins there.
struct Cursor {
  int t;        // next place of the line
  int b, base;  // sequence, its first place
  int group, tile0, n_tiles, tiles, len;

  CHPE_DEV bool next(const PagedLaunch& P, int t_end) {
    do {
      if (t >= t_end) return false;
      int places = places_of(tiles);
      while (t >= base + places * P.groups) {  // the next sequence that has tiles
        base += places * P.groups;
        len = seq_len(P, ++b);
        tiles = tiles_of(P, len);
        places = places_of(tiles);
      }
      group = P.groups == 1 ? 0 : (int)((uint32_t)(t - base) / (uint32_t)places);
      const int at = t - base - group * places, n = min(places - at, t_end - t);
      tile0 = max(at - kBegin, 0);
      n_tiles = at + n - kBegin - tile0;
      t += n;
    } while (n_tiles <= 0);  // the stretch ends before the first tile
    return true;
  }
};

// T: type of the cache; TQ: of q and out.
template <typename T, typename TQ, int D, int N>
__global__ void __launch_bounds__(32 * Cfg<D, N>::kWarps) paged_kernel(const __grid_constant__ PagedLaunch P) {
  using C = Cfg<D, N>;
  constexpr bool SAME = std::is_same<T, TQ>::value;  // the query is its own only part
  // parts of the probabilities, of the query: FP16 has 22 bits in two, BF16 24 in three
  constexpr int PP = std::is_same<T, __nv_bfloat16>::value ? 3 : 2, QP = SAME ? 1 : PP;
  constexpr int KS = D / 16, CH = D / 8;  // 16-dimension steps, 16-byte chunks per row
  constexpr int W = C::kWarps, THREADS = 32 * W;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ int strip_sum[W];
  __shared__ int s_base, s_seq;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int row = lane >> 2, quad = lane & 3;
  const int cta = blockIdx.x, n_cta = gridDim.x;
  const int hw = warp & (P.HW - 1), sub = warp >> (31 - __clz(P.HW)), subs = 1 << (P.tile_shift - 4);

  pdl_wait();
  // ---- this CTA's stretch of the line of tiles
  const int per = (P.B + THREADS - 1) / THREADS;
  const int b_lo = min(tid * per, P.B), b_hi = min(b_lo + per, P.B);
  int mine = 0;
  for (int b = b_lo; b < b_hi; b++) mine += places_of(tiles_of(P, seq_len(P, b)));
  mine *= P.groups;
  int incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += up;
  }
  if (lane == 31) strip_sum[warp] = incl;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int w = 0; w < W; w++) {
    incl += w < warp ? strip_sum[w] : 0;
    total += strip_sum[w];
  }
  const int share = (int)((uint32_t)total / (uint32_t)n_cta), more = total - share * n_cta;
  const int t_begin = cta * share + min(cta, more), t_end = t_begin + share + (cta < more ? 1 : 0);
  if (t_begin < t_end && t_begin >= incl - mine && t_begin < incl) {  // one thread
    int base = incl - mine, b = b_lo;
    for (; b < b_hi - 1; b++) {
      const int n = places_of(tiles_of(P, seq_len(P, b))) * P.groups;
      if (t_begin < base + n) break;
      base += n;
    }
    s_seq = b;
    s_base = base;
  }
  // sequences without a position: nothing else writes their outputs
  for (int b = cta; b < P.B; b += n_cta) {
    if (seq_len(P, b) > 0) continue;
    for (int i = tid; i < P.H * D; i += THREADS) store1(static_cast<TQ*>(P.out) + b * P.out_stride + i, 0.f);
    if (P.lse)
      for (int i = tid; i < P.H; i += THREADS) P.lse[(int64_t)b * P.H + i] = -INFINITY;
    if (P.by_seq)
      for (int g = tid; g < P.groups; g += THREADS) P.desc[b * P.groups + g] = make_int4(0, 0, 0, 0);
  }
  __syncthreads();
  int4 cut = make_int4(0, 0, 0, 0);
  if (t_begin >= t_end) {
    if (tid == 0 && !P.by_seq) P.desc[cta] = cut;
    return;
  }
  Cursor at;  // the stretch that is worked on
  at.t = t_begin, at.b = s_seq, at.base = s_base;
  at.len = seq_len(P, at.b), at.tiles = tiles_of(P, at.len);

  const uint32_t ring = smem_u32(smem) + warp * (C::kStages * C::kStageBytes);
  const size_t row_stride = (size_t)P.KV * D;  // elements between positions
  const T* const kc = static_cast<const T*>(P.kc);
  const T* const vc = static_cast<const T*>(P.vc);

  // ---- the units this warp will come to, copied kStages - 1 ahead across the
  // ends of stretches: one step each time, one group of copies per step
  Cursor ahead = at;
  bool some = ahead.next(P, t_end);
  int a_it = 0, a_st = 0, a_p = 0, page_val = -1;
  const int32_t* a_row = nullptr;
  size_t a_head = 0;
  uint32_t ok_bits = 0;  // by stage: the unit's page is there
  auto step_ahead = [&] {
    if (some) {
      if (a_it == 0) {
        a_row = P.table + ahead.b * P.table_stride;
        a_head = (size_t)((ahead.group * P.HW + hw) / P.HT) * D;
        a_p = (ahead.tile0 << P.tile_shift) + sub * kUnit;
      }
      if ((a_it & 31) == 0) {  // lanes hold 32 units' pages at a time
        const int64_t p = a_p + ((int64_t)lane << P.tile_shift);
        page_val = p < ahead.len ? a_row[p >> P.page_shift] : -1;
      }
      const int pg = __shfl_sync(0xffffffffu, page_val, a_it & 31);
      const bool there = (uint32_t)pg < P.n_pages;
      ok_bits = (ok_bits & ~(1u << a_st)) | ((there ? 1u : 0u) << a_st);
      const size_t r0 = ((size_t)(there ? pg : 0) << P.page_shift) + (a_p & ((1 << P.page_shift) - 1));
      const uint32_t dst = ring + a_st * C::kStageBytes;
      // a warp's instruction copies RPI rows; lane: row `hi` of them, chunk `ch`
      constexpr int RPI = 32 / CH;
      const int hi = lane / CH, ch = lane % CH;
      const T* k_at = kc + (r0 + hi) * row_stride + a_head + ch * 8;
      const T* v_at = vc + (r0 + hi) * row_stride + a_head + ch * 8;
      if (there && a_p + kUnit <= ahead.len) {
        const uint32_t d0 = dst + hi * C::kRow;
#pragma unroll
        for (int i = 0; i < kUnit / RPI; i++) {
          const uint32_t d = d0 + i * RPI * C::kRow + (((ch ^ hi) ^ ((i * RPI) & 7)) << 4);
          cp16(d, k_at);
          cp16(d + kUnit * C::kRow, v_at);
          k_at += RPI * row_stride;
          v_at += RPI * row_stride;
        }
      } else {  // the sequence ends in this unit, or its page is not there: zeros
#pragma unroll 1
        for (int i = 0; i < kUnit / RPI; i++) {
          const int r = i * RPI + hi;
          const bool on = there && a_p + r < ahead.len;
          const uint32_t d = dst + r * C::kRow + ((ch ^ (r & 7)) << 4);
          cp16_if(d, on ? k_at + i * RPI * row_stride : kc, on);
          cp16_if(d + kUnit * C::kRow, on ? v_at + i * RPI * row_stride : vc, on);
        }
      }
      a_st = a_st + 1 < C::kStages ? a_st + 1 : 0;
      a_p += 1 << P.tile_shift;
      if (++a_it == ahead.n_tiles) {
        a_it = 0;
        some = ahead.next(P, t_end);
      }
    }
    cp_commit();
  };
  int st = 0;  // stage of the unit that is worked on
  bool started = false;

  while (at.next(P, t_end)) {
    const int vh = at.group * P.HW + hw, kvh = vh / P.HT, h0 = kvh * P.G + (vh % P.HT) * C::kWarpHeads;
    const int nh = min(C::kWarpHeads, (kvh + 1) * P.G - h0);

    // ---- the query's parts as column operands: lane holds heads `row` of each
    uint32_t qb[N][QP][KS][2];
    float2 x[N][SAME ? 1 : KS][2];
#pragma unroll
    for (int c = 0; c < N; c++) {
      const int head = c * kHeads + row;
      const TQ* const q_row = static_cast<const TQ*>(P.q) + at.b * P.q_stride + (int64_t)(h0 + head) * D + 2 * quad;
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          if constexpr (SAME) qb[c][0][k][h] = head < nh ? *reinterpret_cast<const uint32_t*>(q_row + k * 16 + h * 8) : 0u;
          else x[c][k][h] = head < nh ? load2(q_row + k * 16 + h * 8) : make_float2(0.f, 0.f);
        }
    }
    if (!started) {  // the first copies, behind the query's loads
#pragma unroll 1
      for (int i = 0; i < C::kStages - 1; i++) step_ahead();
      started = true;
    }
    float scale[N][2];
#pragma unroll
    for (int c = 0; c < N; c++) {
      float mine = P.scale * 1.44269504088896340736f;  // scores in powers of two
      if constexpr (!SAME) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
          for (int h = 0; h < 2; h++) top = fmaxf(top, fmaxf(fabsf(x[c][k][h].x), fabsf(x[c][k][h].y)));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // a power of two that brings the largest |q| of the head to [2^TOP, 2^(TOP + 1)).  Two
        // FP16 parts are off by 2^-23 of the value, but never by less than 2^-25: from the top of
        // FP16's range, what is above 2^-16 of the largest keeps its 22 bits (from [1, 2), what
        // is above a quarter did, and scores beside a dimension of 4e4 were off by 0.02)
        constexpr int TOP = std::is_same<T, __half>::value ? 14 : 0;
        const int e = top < INFINITY ? max(TOP - 126, min(TOP + 126, (int)(__float_as_uint(top) >> 23) - 127)) - TOP : 0;
        const float down = __uint_as_float((uint32_t)(127 - e) << 23);
        mine *= __uint_as_float((uint32_t)(127 + e) << 23);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float2 y = make_float2(x[c][k][h].x * down, x[c][k][h].y * down);
#pragma unroll
            for (int part = 0; part < QP; part++) {
              const uint32_t w = pack2<T>(y.x, y.y);
              qb[c][part][k][h] = w;
              const float2 f = unpack2<T>(w);
              y.x -= f.x;
              y.y -= f.y;
            }
          }
      }
      // from here on a lane holds two heads of each operand, 2 * quad and 2 * quad + 1
      scale[c][0] = __shfl_sync(0xffffffffu, mine, 8 * quad);
      scale[c][1] = __shfl_sync(0xffffffffu, mine, 8 * quad + 4);
    }

    float o[N][KS][4];  // [16 dimensions][dimension row, head], [.. + 8]
    float m[N][2], l[N][2];
#pragma unroll
    for (int c = 0; c < N; c++) {
#pragma unroll
      for (int t = 0; t < KS; t++)
#pragma unroll
        for (int e = 0; e < 4; e++) o[c][t][e] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; h++) m[c][h] = -INFINITY, l[c][h] = 0.f;
    }

    // ldmatrix rows.  K: matrices (positions 0-7, dimensions 0-7), (8-15, 0-7), (0-7,
    // 8-15), (8-15, 8-15).  V, transposed: (positions 0-7, dimensions 0-7), (0-7,
    // 8-15), (8-15, 0-7), (8-15, 8-15).
    const int mat = lane >> 3, mr = lane & 7;
    const int k_row = (mat & 1) * 8 + mr, k_ch = mat >> 1;
    const int v_row = (mat >> 1) * 8 + mr, v_ch = mat & 1;

    int p = (at.tile0 << P.tile_shift) + sub * kUnit;
    for (int it = 0; it < at.n_tiles; it++, p += 1 << P.tile_shift) {
      step_ahead();
      cp_wait<C::kStages - 1>();
      __syncwarp();
      if (p < at.len && (ok_bits >> st & 1u)) {
        const uint32_t kb = ring + st * C::kStageBytes, vb = kb + kUnit * C::kRow;
        float acc[N][2][4] = {};  // two chains: even and odd steps
#pragma unroll
        for (int k = 0; k < KS; k++) {
          uint32_t kf[4];
          ldsm4(kf, kb + k_row * C::kRow + (((2 * k + k_ch) ^ (k_row & 7)) << 4));
#pragma unroll
          for (int c = 0; c < N; c++)
#pragma unroll
            for (int part = 0; part < QP; part++) mma16816<T>(acc[c][k & 1], kf, qb[c][part][k][0], qb[c][part][k][1]);
        }
        // scores of positions p + row and p + row + 8, heads 2 quad and 2 quad + 1
        const bool in0 = p + row < at.len, in1 = p + row + 8 < at.len;
        uint32_t pb[N][PP][2];
#pragma unroll
        for (int c = 0; c < N; c++) {
          float sc[4], mn[2];
#pragma unroll
          for (int e = 0; e < 4; e++)
            sc[e] = (e < 2 ? in0 : in1) ? (acc[c][0][e] + acc[c][1][e]) * scale[c][e & 1] : -INFINITY;
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float mx = fmaxf(sc[h], sc[h + 2]);
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            mn[h] = fmaxf(m[c][h], mx);
          }
          if (__any_sync(0xffffffffu, mn[0] != m[c][0] || mn[1] != m[c][1])) {
            float corr[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
              corr[h] = mn[h] == -INFINITY ? 1.f : exp2f(m[c][h] - mn[h]);
              l[c][h] *= corr[h];
              m[c][h] = mn[h];
            }
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
              for (int e = 0; e < 4; e++) o[c][t][e] *= corr[e & 1];
          }
          float y[4];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            y[e] = exp2f(sc[e] - ((m[c][e & 1] == -INFINITY ? 0.f : m[c][e & 1]) - kPShift<T>));
            l[c][e & 1] += y[e];
          }
#pragma unroll
          for (int part = 0; part < PP; part++)
#pragma unroll
            for (int i = 0; i < 2; i++) {  // positions 0-7 and 8-15
              const uint32_t w = pack2<T>(y[2 * i], y[2 * i + 1]);
              pb[c][part][i] = transpose8(w);
              const float2 f = unpack2<T>(w);
              y[2 * i] -= f.x;
              y[2 * i + 1] -= f.y;
            }
        }
#pragma unroll
        for (int t = 0; t < KS; t++) {
          uint32_t vf[4];
          ldsm4t(vf, vb + v_row * C::kRow + (((2 * t + v_ch) ^ (v_row & 7)) << 4));
#pragma unroll
          for (int c = 0; c < N; c++) {
            float add[4] = {};  // the smallest parts first
#pragma unroll
            for (int part = PP - 1; part >= 0; part--) mma16816<T>(add, vf, pb[c][part][0], pb[c][part][1]);
#pragma unroll
            for (int e = 0; e < 4; e++) o[c][t][e] += add[e];
          }
        }
      }
      __syncwarp();  // the stage may be filled again
      st = st + 1 < C::kStages ? st + 1 : 0;
    }
#pragma unroll
    for (int c = 0; c < N; c++) {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        l[c][h] += __shfl_xor_sync(0xffffffffu, l[c][h], 4);
        l[c][h] += __shfl_xor_sync(0xffffffffu, l[c][h], 8);
        l[c][h] += __shfl_xor_sync(0xffffffffu, l[c][h], 16);
      }
      if (subs > 1) {  // warps that share the head: the first one takes the others' sums
        float* const sums = reinterpret_cast<float*>(smem + C::kRing) + hw * C::kSums;
        __syncthreads();  // the sums handed over before are taken
        if (sub > 0) {
          float* const to = sums + (sub - 1) * P.HW * C::kSums;  // four per lane and 16 dimensions, then m and l
#pragma unroll
          for (int t = 0; t < KS; t++)
            *reinterpret_cast<float4*>(to + t * 128 + 4 * lane) = make_float4(o[c][t][0], o[c][t][1], o[c][t][2], o[c][t][3]);
          if (row == 0) *reinterpret_cast<float4*>(to + D * 8 + 4 * quad) = make_float4(m[c][0], m[c][1], l[c][0], l[c][1]);
        }
        __syncthreads();
        if (sub == 0) {
          for (int w = 0; w < subs - 1; w++) {
            const float* const from = sums + w * P.HW * C::kSums;
            const float4 ml = *reinterpret_cast<const float4*>(from + D * 8 + 4 * quad);
            float fa[2], fb[2];
#pragma unroll
            for (int h = 0; h < 2; h++) {
              const float mb = h ? ml.y : ml.x, top = fmaxf(m[c][h], mb);
              fa[h] = m[c][h] == -INFINITY ? 0.f : exp2f(m[c][h] - top);
              fb[h] = mb == -INFINITY ? 0.f : exp2f(mb - top);
              l[c][h] = l[c][h] * fa[h] + (h ? ml.w : ml.z) * fb[h];
              m[c][h] = top;
            }
#pragma unroll
            for (int t = 0; t < KS; t++) {
              const float4 v = *reinterpret_cast<const float4*>(from + t * 128 + 4 * lane);
              o[c][t][0] = o[c][t][0] * fa[0] + v.x * fb[0];
              o[c][t][1] = o[c][t][1] * fa[1] + v.y * fb[1];
              o[c][t][2] = o[c][t][2] * fa[0] + v.z * fb[0];
              o[c][t][3] = o[c][t][3] * fa[1] + v.w * fb[1];
            }
          }
        }
      }
    }
    if (sub == 0) {
      const bool whole = at.n_tiles == at.tiles;
      float* const rec = P.part + (((size_t)2 * cta + (at.tile0 == 0 ? 1 : 0)) * P.HW + hw) * C::kRec;
      TQ* const out = static_cast<TQ*>(P.out) + at.b * P.out_stride + (int64_t)h0 * D;
#pragma unroll
      for (int c = 0; c < N; c++) {
        float inv[2];
#pragma unroll
        for (int h = 0; h < 2; h++) inv[h] = !whole ? 1.f : l[c][h] == 0.f ? 0.f : 1.f / l[c][h];
        // lanes of neighbouring rows swap a value, so that each has two dimensions of one head
        const int head = c * kHeads + 2 * quad + (row & 1), dim = row & ~1;
#pragma unroll
        for (int t = 0; t < KS; t++)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            const float v0 = o[c][t][e] * inv[0], v1 = o[c][t][e + 1] * inv[1];
            const float got = __shfl_xor_sync(0xffffffffu, row & 1 ? v0 : v1, 4);
            o[c][t][e] = row & 1 ? got : v0;
            o[c][t][e + 1] = row & 1 ? v1 : got;
          }
        if (head < nh) {
          if (whole) {
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
              for (int e = 0; e < 4; e += 2) store2(out + head * D + t * 16 + e * 4 + dim, o[c][t][e], o[c][t][e + 1]);
          } else {
#pragma unroll
            for (int t = 0; t < KS; t++)
#pragma unroll
              for (int e = 0; e < 4; e += 2)
                *reinterpret_cast<float2*>(rec + head * D + t * 16 + e * 4 + dim) = make_float2(o[c][t][e], o[c][t][e + 1]);
          }
        }
        if (row < 2 && head < nh) {
          const float mh = row ? m[c][1] : m[c][0], lh = row ? l[c][1] : l[c][0];
          if (!whole) *reinterpret_cast<float2*>(rec + C::kWarpHeads * D + 2 * head) = make_float2(mh, lh);
          else if (P.lse)
            P.lse[(int64_t)at.b * P.H + h0 + head] =
                lh == 0.f ? -INFINITY : 0.693147180559945309417f * (mh + (log2f(lh) - kPShift<T>));
        }
      }
    }
    if (at.tile0 == 0) {
      cut = make_int4(0, 0, 0, 0);
      if (at.n_tiles < at.tiles) {  // the CTAs that hold the rest of the group's tiles follow without a gap
        const int last = at.base + (at.group + 1) * places_of(at.tiles) - 1;
        const int big = (share + 1) * more;  // places of the CTAs with one more
        const int owner = last < big ? last / (share + 1) : more + (last - big) / share;
        cut = make_int4(at.b, at.group, owner - cta + 1, cta);
      }
      if (tid == 0 && P.by_seq) P.desc[at.b * P.groups + at.group] = cut;
    }
  }
  pdl_launch_dependents();  // (at the start, the joining CTAs were in the way: 47.3 us instead of 45.1 on 37 mixed sequences)
  if (tid == 0 && !P.by_seq) P.desc[cta] = cut;
}

// Joins the records of a cut group: blockIdx.x the desc entry, blockIdx.y the
// query head within the group and the DB of its D values, JW warps.  The records' weights
// are worked out once, side by side; 4 * DB bytes of a record take DB/4 lanes, and every
// lane has kBatch records' loads in flight.
template <typename TQ, int D, int N, int DB, int JW>
__global__ void __launch_bounds__(32 * JW) combine_kernel(const __grid_constant__ PagedLaunch P) {
  using C = Cfg<D, N>;
  constexpr int kLanes = DB / 4, kRows = 32 * JW / kLanes;  // lanes of a record, records side by side
  constexpr int kBatch = 8, kMax = C::kMaxCtas;
  static_assert(32 * JW % kLanes == 0, "");
  __shared__ float weight[kMax];
  __shared__ float sv[kRows][DB];
  __shared__ float red[2][JW];
  pdl_wait();
  pdl_launch_dependents();
  const int4 cut = P.desc[blockIdx.x];
  const int n = cut.z;  // at most one record per CTA
  if (n == 0) return;
  const int slice = blockIdx.y % (D / DB), hh = blockIdx.y / (D / DB);
  const int hw = hh / C::kWarpHeads, h = hh % C::kWarpHeads, vh = cut.y * P.HW + hw;
  const int kvh = vh / P.HT, head = kvh * P.G + (vh % P.HT) * C::kWarpHeads + h;
  if (head >= (kvh + 1) * P.G) return;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int my_row = tid / kLanes, col = slice * DB + 4 * (tid % kLanes);
  // record i: the beginning lies in slot 1 of the first CTA, the others in slot 0 of theirs
  auto rec = [&](int i) { return P.part + (((size_t)2 * (cut.w + i) + (i == 0 ? 1 : 0)) * P.HW + hw) * C::kRec; };
  float4 x[kBatch];
  auto fetch = [&](int j, int i) {
    x[j] = i < n ? *reinterpret_cast<const float4*>(rec(i) + h * D + col) : make_float4(0.f, 0.f, 0.f, 0.f);
  };
#pragma unroll
  for (int j = 0; j < kBatch; j++) fetch(j, my_row + j * kRows);

  constexpr int PER = (kMax + 32 * JW - 1) / (32 * JW);
  float2 ml[PER];
  float M = -INFINITY;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int i = tid + j * 32 * JW;
    ml[j] = i < n ? *reinterpret_cast<const float2*>(rec(i) + C::kWarpHeads * D + 2 * h) : make_float2(-INFINITY, 0.f);
    M = fmaxf(M, ml[j].x);
  }
  M = warp_max(M);
  if (lane == 0) red[0][warp] = M;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < JW; w++) M = fmaxf(M, red[0][w]);
  float L = 0.f;
#pragma unroll
  for (int j = 0; j < PER; j++) {
    const int i = tid + j * 32 * JW;
    const float w = ml[j].x == -INFINITY ? 0.f : exp2f(ml[j].x - M);
    if (i < n) weight[i] = w;
    L = fmaf(ml[j].y, w, L);  // a NaN sum stays
  }
  L = warp_sum(L);
  if (lane == 0) red[1][warp] = L;
  __syncthreads();
  L = 0.f;
#pragma unroll
  for (int w = 0; w < JW; w++) L += red[1][w];

  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = my_row; i0 < n; i0 += kBatch * kRows) {
#pragma unroll
    for (int j = 0; j < kBatch; j++) {
      const int i = i0 + j * kRows;
      if (i >= n) break;
      const float w = weight[i];
      v.x = fmaf(x[j].x, w, v.x);
      v.y = fmaf(x[j].y, w, v.y);
      v.z = fmaf(x[j].z, w, v.z);
      v.w = fmaf(x[j].w, w, v.w);
      fetch(j, i + kBatch * kRows);
    }
  }
  *reinterpret_cast<float4*>(&sv[my_row][4 * (tid % kLanes)]) = v;
  __syncthreads();
  for (int d = tid; d < DB; d += 32 * JW) {
    float y = 0.f;
    for (int w = 0; w < min(n, kRows); w++) y += sv[w][d];
    store1(static_cast<TQ*>(P.out) + cut.x * P.out_stride + (int64_t)head * D + slice * DB + d, L == 0.f ? 0.f : y / L);
  }
  if (P.lse && tid == 0 && slice == 0)
    P.lse[(int64_t)cut.x * P.H + head] = L == 0.f ? -INFINITY : 0.693147180559945309417f * (M + (log2f(L) - P.p_shift));
}

// The same where a group is cut into a few records only: a warp per query head, a
// record's heads to a CTA, no barrier.  blockIdx.x the desc entry, blockIdx.y the head's warp of
// the main kernel.
template <typename TQ, int D, int N>
__global__ void __launch_bounds__(32 * N * kHeads) combine_few_kernel(const __grid_constant__ PagedLaunch P) {
  using C = Cfg<D, N>;
  constexpr int PER = D / 64, kBatch = D == 256 ? 4 : 8;  // pairs of a lane, records in flight
  pdl_wait();
  pdl_launch_dependents();
  const int4 cut = P.desc[blockIdx.x];
  const int n = cut.z;
  if (n == 0) return;
  const int hw = blockIdx.y, h = threadIdx.x >> 5, lane = threadIdx.x & 31, vh = cut.y * P.HW + hw;
  const int kvh = vh / P.HT, head = kvh * P.G + (vh % P.HT) * C::kWarpHeads + h;
  if (head >= (kvh + 1) * P.G) return;
  auto rec = [&](int i) { return P.part + (((size_t)2 * (cut.w + i) + (i == 0 ? 1 : 0)) * P.HW + hw) * C::kRec; };
  float2 x[kBatch][PER];
  auto fetch = [&](int j, int i) {
#pragma unroll
    for (int e = 0; e < PER; e++)
      x[j][e] = i < n ? *reinterpret_cast<const float2*>(rec(i) + h * D + 64 * e + 2 * lane) : make_float2(0.f, 0.f);
  };
#pragma unroll
  for (int j = 0; j < kBatch; j++) fetch(j, j);
  float M = -INFINITY;
  for (int i = lane; i < n; i += 32) M = fmaxf(M, rec(i)[C::kWarpHeads * D + 2 * h]);
  M = warp_max(M);
  float2 v[PER];
#pragma unroll
  for (int e = 0; e < PER; e++) v[e] = make_float2(0.f, 0.f);
  float L = 0.f;
  for (int c = 0; c < n; c += 32) {  // 32 records' weights at a time
    float w = 0.f;
    if (c + lane < n) {
      const float2 ml = *reinterpret_cast<const float2*>(rec(c + lane) + C::kWarpHeads * D + 2 * h);
      w = ml.x == -INFINITY ? 0.f : exp2f(ml.x - M);
      L = fmaf(ml.y, w, L);  // a NaN sum stays
    }
    const int end = min(32, n - c);
    for (int i0 = 0; i0 < end; i0 += kBatch) {
#pragma unroll
      for (int j = 0; j < kBatch; j++) {
        const float wi = __shfl_sync(0xffffffffu, w, (i0 + j) & 31);  // 0 behind the last
#pragma unroll
        for (int e = 0; e < PER; e++) {
          v[e].x = fmaf(x[j][e].x, wi, v[e].x);
          v[e].y = fmaf(x[j][e].y, wi, v[e].y);
        }
        fetch(j, c + i0 + j + kBatch);
      }
    }
  }
  L = warp_sum(L);
  const float inv = L == 0.f ? 0.f : 1.f / L;
  TQ* const out = static_cast<TQ*>(P.out) + cut.x * P.out_stride + (int64_t)head * D + 2 * lane;
#pragma unroll
  for (int e = 0; e < PER; e++) store2(out + 64 * e, v[e].x * inv, v[e].y * inv);
  if (P.lse && lane == 0)
    P.lse[(int64_t)cut.x * P.H + head] = L == 0.f ? -INFINITY : 0.693147180559945309417f * (M + (log2f(L) - P.p_shift));
}

template <int D>
constexpr size_t workspace_bytes_of() {
  using C = Cfg<D, D == 128 ? 2 : 1>;
  return C::kMaxCtas * sizeof(int4) + (size_t)2 * C::kMaxCtas * C::kWarps * C::kRec * sizeof(float);
}

template <typename T, typename TQ, int D, int N>
cudaError_t launch(PagedLaunch P, void* workspace, int device, cudaStream_t s) {
  using C = Cfg<D, N>;
  // per device: SMs times resident CTAs of this kernel (one query, then kept)
  static int grid_of[64] = {};
  const int dev = device >= 0 && device < 64 ? device : -1;
  int grid = dev >= 0 ? __atomic_load_n(&grid_of[dev], __ATOMIC_RELAXED) : 0;
  if (grid == 0) {
    int sms = 0, res = 0;
    const int most = C::kRing + (C::kWarps - 1) * C::kSums * (int)sizeof(float);  // one head: all other warps hand over
    cudaError_t e = cudaFuncSetAttribute(paged_kernel<T, TQ, D, N>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
    if (e == cudaSuccess)
      e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&res, paged_kernel<T, TQ, D, N>, 32 * C::kWarps, most);
    if (e != cudaSuccess) return e;
    grid = sms * (res < 1 ? 1 : res);
    if (grid > C::kMaxCtas) grid = C::kMaxCtas;
    if (dev >= 0) __atomic_store_n(&grid_of[dev], grid, __ATOMIC_RELAXED);
  }
  const int subs = C::kWarps / P.HW;
  P.p_shift = kPShift<T>;
  P.by_seq = (int64_t)P.B * P.groups <= grid;
  P.desc = static_cast<int4*>(workspace);
  P.part = reinterpret_cast<float*>(P.desc + C::kMaxCtas);
  chpe::ServeLaunch main(dim3(grid), 32 * C::kWarps, C::kRing + (subs - 1) * P.HW * C::kSums * sizeof(float), s);
  const cudaError_t e = cudaLaunchKernelEx(&main.cfg, paged_kernel<T, TQ, D, N>, P);
  if (e != cudaSuccess) return e;
  const int cuts = P.by_seq ? P.B * P.groups : grid;
  // The records that a group of an even batch is cut into; which kernel joins them goes by
  // that, and each joins any number.  Many: 16 warps for 64 values of a query head (two
  // sequences of 2048 on 64/8 heads, 76 records each: 10.6 us, with four warps per head
  // 10.8, with one 16.8).  Some: four warps per query head (eight sequences, 20 records:
  // 21.0 us, with 16 warps 27.3, with one 21.7).  Few: one warp each (64 sequences of up to
  // 1024, two or three records: 25.8 us, with four warps 29.0, with 16 66.2).  An uneven
  // batch pays for the estimate: one sequence of 131071 among 63 of ten, some 140 records,
  // takes 104 us where four warps per head take 98.
  const int64_t records = (P.cap >> P.tile_shift) < grid / cuts + 2 ? (P.cap >> P.tile_shift) : grid / cuts + 2;
  if (records > 64) {
    chpe::ServeLaunch join(dim3(cuts, P.HW * C::kWarpHeads * (D / 64)), 32 * 16, 0, s);
    return cudaLaunchKernelEx(&join.cfg, combine_kernel<TQ, D, N, 64, 16>, P);
  }
  if (records > 8) {
    chpe::ServeLaunch join(dim3(cuts, P.HW * C::kWarpHeads), 32 * 4, 0, s);
    return cudaLaunchKernelEx(&join.cfg, combine_kernel<TQ, D, N, D, 4>, P);
  }
  chpe::ServeLaunch join(dim3(cuts, P.HW), 32 * C::kWarpHeads, 0, s);
  return cudaLaunchKernelEx(&join.cfg, combine_few_kernel<TQ, D, N>, P);
}

template <typename T, typename TQ>
cudaError_t launch_d(const PagedLaunch& P, void* workspace, uint32_t d, int operands, int device, cudaStream_t s) {
  if (d == 64) return launch<T, TQ, 64, 1>(P, workspace, device, s);
  if (d == 256) return launch<T, TQ, 256, 1>(P, workspace, device, s);
  return operands == 2 ? launch<T, TQ, 128, 2>(P, workspace, device, s) : launch<T, TQ, 128, 1>(P, workspace, device, s);
}

}  // namespace

extern "C" size_t chpe_attention_decode_paged_workspace(uint32_t head_dim) {
  return head_dim == 64    ? workspace_bytes_of<64>()
         : head_dim == 128 ? workspace_bytes_of<128>()
         : head_dim == 256 ? workspace_bytes_of<256>()
                           : 0;
}

extern "C" int chpe_attention_decode_paged(const void* q, int dtype, int64_t q_stride, const void* k_cache,
                                           const void* v_cache, int cache_dtype, uint32_t num_pages,
                                           uint32_t page_size, const int32_t* page_table, int64_t table_stride,
                                           uint32_t max_pages, const int32_t* seq_lens, uint32_t batch, uint32_t num_heads,
                                           uint32_t num_kv_heads, uint32_t head_dim, float scale, void* out,
                                           int64_t out_stride, float* lse, void* workspace,
                                           size_t workspace_bytes, void* stream) {
  chpe::ServeCall c("chpe_attention_decode_paged");
  const size_t es = chpe::dtype_size(dtype);
  if (!es) return c.fail(-1, "unknown dtype %lld", dtype), c.done();
  if (cache_dtype != CHPE_F16 && cache_dtype != CHPE_BF16) return c.fail(-1, "the cache must be FP16 or BF16"), c.done();
  if (dtype != CHPE_F32 && dtype != cache_dtype)
    return c.fail(-1, "the cache must have the type of q unless q is float"), c.done();
  if (head_dim != 64 && head_dim != 128 && head_dim != 256) return c.fail(-1, "head_dim must be 64, 128 or 256"), c.done();
  if (num_heads == 0 || num_kv_heads == 0 || num_heads > 65535 || num_heads % num_kv_heads != 0)
    return c.fail(-1, "num_heads must be a multiple of num_kv_heads, at most 65535"), c.done();
  if (page_size < 16 || page_size > 65536 || (page_size & (page_size - 1)))
    return c.fail(-1, "page_size must be a power of two from 16 to 65536"), c.done();
  if (batch > 65535) return c.fail(-1, "batch must be at most 65535"), c.done();
  if (batch > 1 && (table_stride < 0 || table_stride > INT64_MAX / 8 / batch ||
                    (table_stride != 0 && table_stride < (int64_t)max_pages)))
    return c.fail(-1, "table_stride must be 0 (one table for all) or at least max_pages"), c.done();
  if (!(fabsf(scale) <= 1e6f)) return c.fail(-1, "scale is not a number within 1e6"), c.done();
  const int64_t least = (int64_t)num_heads * head_dim;
  if (batch > 1 && (q_stride < least || out_stride < least || q_stride > INT64_MAX / 8 / batch ||
                    out_stride > INT64_MAX / 8 / batch))
    return c.fail(-1, "q_stride and out_stride must be at least num_heads * head_dim"), c.done();
  if (batch > 1 && (q_stride * es % 16 != 0 || out_stride * es % 16 != 0))
    return c.fail(-1, "q_stride and out_stride must be multiples of 16 bytes"), c.done();
  if (batch == 0) return c.done();
  if (workspace_bytes < chpe_attention_decode_paged_workspace(head_dim))
    return c.fail(-2, "needs a workspace of %lld bytes, got %lld",
                  (long long)chpe_attention_decode_paged_workspace(head_dim), (long long)workspace_bytes),
           c.done();
  c.ptr(q, "q", 16);
  c.ptr(out, "out", 16);
  c.ptr(seq_lens, "seq_lens", 4);
  c.ptr(workspace, "workspace", 16);
  c.ptr_or_null(lse, "lse", 4);
  if (num_pages && max_pages) {
    c.ptr(k_cache, "k_cache", 16);
    c.ptr(v_cache, "v_cache", 16);
    c.ptr(page_table, "page_table", 4);
  }
  if (c.rc) return c.done();
  {
    using chpe::Rows;
    const int64_t n = batch, b = (int64_t)es;
    const uint64_t rows = num_pages && max_pages ? (uint64_t)num_pages * page_size : 0, row = 2ull * num_kv_heads * head_dim;
    const Rows in[] = {{"q", q, least * b, n, q_stride, b}, chpe::pool("k_cache", k_cache, rows, row),
                       chpe::pool("v_cache", v_cache, rows, row),
                       {"page_table", rows ? page_table : nullptr, 4ll * max_pages, n, table_stride, 4}, {"seq_lens", seq_lens, 4 * n}};
    const Rows to[] = {{"out", out, least * b, n, out_stride, b}, {"lse", lse, 4 * n * num_heads},
                        {"workspace", workspace, (int64_t)chpe_attention_decode_paged_workspace(head_dim)}};
    for (int o = 0; o < 3; o++) {
      for (const Rows& i : in) c.apart(to[o], i);
      for (int i = 0; i < o; i++) c.apart(to[o], to[i]);
    }
    if (c.rc) return c.done();
  }

  PagedLaunch P{};
  P.q = q, P.q_stride = q_stride;
  P.kc = k_cache, P.vc = v_cache;
  P.table = page_table, P.table_stride = table_stride, P.lens = seq_lens;
  P.n_pages = num_pages;
  while ((1u << P.page_shift) < page_size) P.page_shift++;
  const int64_t cap = num_pages ? (int64_t)max_pages * page_size : 0;  // an empty pool holds no position
  P.cap = (int32_t)(cap < INT32_MAX - 1024 ? cap : INT32_MAX - 1024);
  P.B = (int32_t)batch, P.H = (int32_t)num_heads, P.KV = (int32_t)num_kv_heads;
  P.G = P.H / P.KV;
  // More than 8 query heads per kv head: two operands per warp, so that the rows copied
  // serve 16, or two warps that copy the same rows.  At heads of 128 the former takes 72
  // instead of 86 us for 64 sequences of up to 8192 on 64/4 heads in BF16, but 11.1 instead
  // of 9.8 for one of 4000 on 32/2, so it is taken where the tables have room for 64 MB of
  // entries; at 64 they are even (26.9 us), and at 256 the registers are lacking.
  const double room = 4.0 * batch * P.cap * num_kv_heads * head_dim;
  const int operands = head_dim == 128 && P.G > kHeads && room >= 64.0 * (1 << 20) ? 2 : 1;
  const int per_warp = operands * kHeads;
  P.HT = (P.G + per_warp - 1) / per_warp;
  const int vh = P.KV * P.HT, warps = head_dim == 256 ? Cfg<256, 1>::kWarps : Cfg<128, 1>::kWarps;
  static_assert(Cfg<64, 1>::kWarps == Cfg<128, 1>::kWarps, "");
  P.HW = warps;
  while (vh % P.HW != 0) P.HW /= 2;
  P.groups = vh / P.HW;
  P.tile_shift = 4;
  while ((kUnit * warps / P.HW) >> P.tile_shift > 1) P.tile_shift++;
  if ((int64_t)((P.cap >> P.tile_shift) + 1 + kBegin) * P.groups > INT32_MAX / P.B)
    return c.fail(-1, "batch * max_pages * page_size is too large"), c.done();
  P.scale = scale;
  P.out = out, P.out_stride = out_stride, P.lse = lse;
  chpe::DeviceScope scope(c.launch_device());
  const cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (cache_dtype == CHPE_F16) e = dtype == CHPE_F32 ? launch_d<__half, float>(P, workspace, head_dim, operands, c.device, s)
                                                     : launch_d<__half, __half>(P, workspace, head_dim, operands, c.device, s);
  else e = dtype == CHPE_F32 ? launch_d<__nv_bfloat16, float>(P, workspace, head_dim, operands, c.device, s)
                             : launch_d<__nv_bfloat16, __nv_bfloat16>(P, workspace, head_dim, operands, c.device, s);
  if (e != cudaSuccess) {
    snprintf(c.msg, sizeof(c.msg), "launch: %s", cudaGetErrorString(e));
    c.rc = -3;
  }
  return c.done();
}
