// Key and value rows in 4 bits on gfx950: conversion into the cache and back, and eviction
// by accumulated attention weight.
//
// Format (include/deltaattn_cache.h): groups of 32 dims, elements E2M1 (sign, two exponent
// bits, one mantissa bit) times one power of two a group.  A power of two makes every value
// exact in bf16 and lets v_cvt_scalef32_pk_* convert a byte of two codes, scale included, in
// one instruction.
#include "da_common.hpp"
#include "../../include/deltaattn_cache.h"

namespace da {

// ------------------------------------------------------------------------------------
// rows -> 4 bits
// ------------------------------------------------------------------------------------
struct Quant4Args {
  const void* x[2];  // k, v
  int64_t s_b[2], s_h[2], s_n[2];
  uint8_t* codes[2];
  uint8_t* scales[2];
  const int32_t* counts;
  const int32_t* ts;
  const float* mass;
  const int32_t* lengths;
  const int32_t* index;
  int32_t* o_counts;
  int32_t* o_ts;
  float* o_mass;
  int32_t* o_lengths;
  int64_t N, M, capacity;
  int B, H, D;
};

// Eight consecutive elements of a row, as fp32.  The rows are read once: they pass the caches by.
template <int DT>
__device__ __forceinline__ void load8(const void* row, int64_t at, float (&x)[8]) {
  if constexpr (DT == DA_F32) {
    const f32x4 a = __builtin_nontemporal_load((const f32x4*)((const float*)row + at));
    const f32x4 b = __builtin_nontemporal_load((const f32x4*)((const float*)row + at + 4));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = a[i];
      x[4 + i] = b[i];
    }
  } else {
    const u32x4 w = __builtin_nontemporal_load((const u32x4*)((const uint16_t*)row + at));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = E16<DT>::lo(w[i]);
      x[2 * i + 1] = E16<DT>::hi(w[i]);
    }
  }
}

__device__ __forceinline__ uint32_t quad_umax(uint32_t v) {
  const uint32_t a = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppXor1, 0xF, 0xF, false);
  v = v > a ? v : a;
  const uint32_t b = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppXor2, 0xF, 0xF, false);
  return v > b ? v : b;
}

// The exponent byte of a group whose largest magnitude has fp32 bits `top`: with top = 1.f x
// 2^(E - 127), 4 x 1.f <= 6 exactly where the fraction is at most one half.  Magnitudes are
// compared as integers, so a NaN is the largest.
__device__ __forceinline__ uint32_t group_exponent(uint32_t top) {
  const int E = (int)(top >> 23);
  if (E == 255) return 255u;
  int x = E - 2 + ((top & 0x7fffffu) > 0x400000u ? 1 : 0);
  x = x < 2 ? 2 : x;
  return (uint32_t)(x > 252 ? 252 : x);
}

// A lane takes 8 dims: 16 bytes of a 16-bit row (32 of an fp32 one), 4 bytes of codes; the
// four lanes of a quad are one group, whose largest magnitude is two quad permutes away.
// Lanes per row: 4 NG.  Each thread takes kQuantItems of them, a block's width apart, with
// all of its loads in flight (64K tokens of 8 heads of 128 bf16 dims, as projections lay them out:
// 65 us, 5.3 TB/s; one item a thread 74, four 65).  blockIdx.z = key, value or the rows' small fields.
constexpr int kQuantItems = 2;
template <int DT, int NG>
__global__ __launch_bounds__(256) void quantize4_kernel(Quant4Args a) {
  constexpr uint32_t kLpr = 4 * NG;
  const int bh = blockIdx.y, z = blockIdx.z;
  const int b = bh / a.H, h = bh - b * a.H;
  const uint32_t M = (uint32_t)a.M;
  uint32_t len = M;
  if (a.lengths) {
    const int n = a.lengths[bh];
    len = n < 0 ? 0 : ((uint32_t)n > M ? M : (uint32_t)n);
  }
  if (z == 2) {  // the rows' small fields, a lane each
    for (uint32_t m = blockIdx.x * 256 + threadIdx.x; m < M; m += gridDim.x * 256) {
      int s = m < len ? (a.index ? a.index[(int64_t)bh * M + m] : (int)m) : -1;
      const bool real = s >= 0 && s < a.N;
      const int64_t row = bh * a.capacity + m, from = bh * a.N + (real ? s : 0);
      a.o_counts[row] = real ? (a.counts ? a.counts[from] : 1) : 0;
      a.o_ts[row] = real ? (a.ts ? a.ts[from] : s) : 0;
      if (a.o_mass) a.o_mass[row] = real && a.mass ? a.mass[from] : 0.0f;
      if (m == 0) a.o_lengths[bh] = (int32_t)len;
    }
    return;
  }
  const char* base = (const char*)a.x[z] + (b * a.s_b[z] + h * a.s_h[z]) * (DT == DA_F32 ? 4 : 2);
  const uint32_t first = blockIdx.x * 256 * kQuantItems + threadIdx.x;  // below 2^31: capacity <= 2^26
  float x[kQuantItems][8];
  int src[kQuantItems];
#pragma unroll
  for (int u = 0; u < kQuantItems; ++u) {
    const uint32_t m = (first + u * 256) / kLpr;
    int s = -1;
    if (m < len) {
      s = (int)m;
      if (a.index) {
        s = a.index[(int64_t)bh * M + m];
        if (s >= a.N) s = -1;
      }
    }
    src[u] = s;
  }
#pragma unroll
  for (int u = 0; u < kQuantItems; ++u) {
    const int d = 8 * (int)((first + u * 256) % kLpr);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[u][i] = 0.0f;
    if (src[u] >= 0 && d < a.D) load8<DT>(base, src[u] * a.s_n[z] + d, x[u]);
  }
#pragma unroll
  for (int u = 0; u < kQuantItems; ++u) {
    const uint32_t it = first + u * 256, m = it / kLpr;
    const int c = (int)(it - m * kLpr);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = __float_as_uint(x[u][i]) & 0x7fffffffu;
      top = top > w ? top : w;
    }
    top = quad_umax(top);
    const uint32_t e = group_exponent(top);
    uint32_t codes = 0;
    if (e != 255u) {
      // multiplying by a power of two is exact (results below the smallest normal are far
      // below the first rounding border, 0.25); the conversion rounds to nearest even and
      // saturates, which only the largest exponent reaches
      const float inv = __uint_as_float((254u - e) << 23);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[u][i] *= inv;
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[u][0], x[u][1], 1.0f, 0);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[u][2], x[u][3], 1.0f, 1);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[u][4], x[u][5], 1.0f, 2);
      codes = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(codes, x[u][6], x[u][7], 1.0f, 3);
    }
    if (m < M) {
      const int64_t row = bh * a.capacity + m;
      ((uint32_t*)a.codes[z])[row * kLpr + c] = codes;
      if ((c & 3) == 0) a.scales[z][row * NG + (c >> 2)] = (uint8_t)(src[u] < 0 ? 0u : e);
    }
  }
}

// ------------------------------------------------------------------------------------
// 4 bits -> rows
// ------------------------------------------------------------------------------------
struct Dequant4Args {
  const uint8_t* codes[2];
  const uint8_t* scales[2];
  void* x[2];
  const int32_t* lengths;
  int64_t N, capacity;
  int D;
};

// A lane turns 4 bytes of codes into 8 elements; kQuantItems of them in flight a thread.
template <int DT, int NG>
__global__ __launch_bounds__(256) void dequantize4_kernel(Dequant4Args a) {
  constexpr uint32_t kLpr = 4 * NG;
  const int bh = blockIdx.y, z = blockIdx.z;
  const int n = a.lengths[bh];
  const uint32_t len = n < 0 ? 0 : (n > a.N ? (uint32_t)a.N : (uint32_t)n);
  const uint32_t first = blockIdx.x * 256 * kQuantItems + threadIdx.x;
  uint32_t w[kQuantItems], e[kQuantItems];
#pragma unroll
  for (int u = 0; u < kQuantItems; ++u) {
    const uint32_t it = first + u * 256, m = it / kLpr;
    const int c = (int)(it - m * kLpr);
    const int64_t row = bh * a.capacity + m;
    w[u] = e[u] = 0;
    if (m < len) {
      w[u] = ((const uint32_t*)a.codes[z])[row * kLpr + c];
      e[u] = a.scales[z][row * NG + (c >> 2)];
    }
  }
#pragma unroll
  for (int u = 0; u < kQuantItems; ++u) {
    const uint32_t it = first + u * 256, m = it / kLpr;
    const int d = 8 * (int)(it - m * kLpr);
    if (m >= (uint32_t)a.N || d >= a.D) continue;
    const float s = __uint_as_float(e[u] << 23);
    const f32x2 p0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 0);
    const f32x2 p1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 1);
    const f32x2 p2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 2);
    const f32x2 p3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w[u], s, 3);
    const int64_t at = (bh * a.N + m) * a.D + d;
    if constexpr (DT == DA_F32) {
      float* o = (float*)a.x[z] + at;
      *(f32x4*)o = f32x4{p0[0], p0[1], p1[0], p1[1]};
      *(f32x4*)(o + 4) = f32x4{p2[0], p2[1], p3[0], p3[1]};
    } else {
      *(u32x4*)((uint16_t*)a.x[z] + at) = u32x4{E16<DT>::pack(p0[0], p0[1]), E16<DT>::pack(p1[0], p1[1]),
                                                E16<DT>::pack(p2[0], p2[1]), E16<DT>::pack(p3[0], p3[1])};
    }
  }
}

// ------------------------------------------------------------------------------------
// one decode token
// ------------------------------------------------------------------------------------
struct Update4Args {
  const void* new_k;
  const void* new_v;
  int64_t sn_b, sn_h;
  void* kx;
  void* vx;
  int64_t sx_b, sx_h, sx_s;
  DaKv4 kv;
  void* k_last;  // [B, Hkv, D]
  int64_t exact_len, total_len, window;
  int B, H, D;
  float thr;
};

// The largest magnitude (fp32 bits) of a lane's row of 16 lanes, which hold one group.
__device__ __forceinline__ uint32_t row16_umax(uint32_t v) {
  v = quad_umax(v);
  uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppHalfMirror, 0xF, 0xF, false);
  v = v > o ? v : o;
  o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, kDppMirror, 0xF, 0xF, false);
  return v > o ? v : o;
}

// One wave a (sequence, KV head), lane l dims 2 l and 2 l + 1: decode_update_kernel's step with the
// packed rows in 4 bits.  The test whether the evicted token merges looks at the last anchor's key as
// it was, kept beside the rows, so the decisions are those of a cache at full width.
template <bool COS, int DT>
__global__ __launch_bounds__(256) void update4_kernel(Update4Args a) {
  using PT = DecPair<DT>;
  using E = typename PT::Elem;
  using Word = typename PT::Word;
  const int lane = threadIdx.x & 63;
  const int w = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= a.B * a.H) return;
  const int b = w / a.H, h = w - b * a.H;
  const bool act = 2 * lane < a.D;
  const int groups = (a.D + 31) / 32;
  const int64_t widx = a.exact_len % a.window;
  E* const ring_k = (E*)a.kx + b * a.sx_b + h * a.sx_h + widx * a.sx_s + 2 * lane;
  E* const ring_v = (E*)a.vx + b * a.sx_b + h * a.sx_h + widx * a.sx_s + 2 * lane;
  E* const last = (E*)a.k_last + (int64_t)w * a.D + 2 * lane;
  if (a.exact_len >= a.window) {
    const Word ek = act ? *(const Word*)ring_k : Word{};
    const Word ev = act ? *(const Word*)ring_v : Word{};
    int n = a.kv.lengths[w];
    n = n < 0 ? 0 : (n > a.kv.capacity ? (int)a.kv.capacity : n);
    const int64_t row0 = (int64_t)w * a.kv.capacity;
    bool merge = false;
    if (n > 0) {
      const Word lk = act ? *(const Word*)last : Word{};
      merge = evict_merges<COS, DT>(ek, lk, a.thr);
    }
    if (merge) {
      if (lane == 0) a.kv.counts[row0 + n - 1] += 1;
    } else if (n < a.kv.capacity) {
      const int64_t row = row0 + n;
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        const Word x = z == 0 ? ek : ev;
        const float x0 = PT::lo(x), x1 = PT::hi(x);
        const uint32_t m0 = __float_as_uint(x0) & 0x7fffffffu, m1 = __float_as_uint(x1) & 0x7fffffffu;
        const uint32_t e = group_exponent(row16_umax(m0 > m1 ? m0 : m1));
        uint32_t code = 0;
        if (e != 255u) {
          const float inv = __uint_as_float((254u - e) << 23);
          code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x0 * inv, x1 * inv, 1.0f, 0);
        }
        uint8_t* const codes = z == 0 ? a.kv.k_codes : a.kv.v_codes;
        uint8_t* const scales = z == 0 ? a.kv.k_scales : a.kv.v_scales;
        if (lane < 16 * groups) codes[row * 16 * groups + lane] = (uint8_t)code;
        if ((lane & 15) == 0 && lane < 16 * groups) scales[row * groups + (lane >> 4)] = (uint8_t)e;
      }
      if (act) *(Word*)last = ek;
      if (lane == 0) {
        a.kv.counts[row] = 1;
        a.kv.timestamps[row] = (int32_t)(a.total_len - a.window);
        if (a.kv.mass) a.kv.mass[row] = 0.0f;
        a.kv.lengths[w] = n + 1;
      }
    }
  }
  if (act) {
    const Word nk = *(const Word*)((const E*)a.new_k + b * a.sn_b + h * a.sn_h + 2 * lane);
    const Word nv = *(const Word*)((const E*)a.new_v + b * a.sn_b + h * a.sn_h + 2 * lane);
    *(Word*)ring_k = nk;
    *(Word*)ring_v = nv;
  }
}

// ------------------------------------------------------------------------------------
// eviction: the rows kept
// ------------------------------------------------------------------------------------
struct HeavyArgs {
  const float* mass;
  const int32_t* lengths;
  int64_t capacity;  // rows a head's mass array holds
  int budget, sinks, recent;
  int32_t* index;  // [bh][budget]
  int32_t* kept;   // [bh]
};

// Masses in an order of unsigned integers (-0 as 0; every NaN, of either sign, as one largest).
__device__ __forceinline__ uint32_t mass_order(float m) {
  const uint32_t u = opaque_bits(m);
  if ((u << 1) == 0) return 0x80000000u;
  if ((u << 1) > 0xff000000u) return 0xffffffffu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kHeavyThreads = 1024, kHeavyWaves = kHeavyThreads / 64, kHeavyBins = 2048;
constexpr int kHeavyPer = 16;                              // masses a thread of heavy_rows_kernel holds
constexpr int kHeavyShort = kHeavyThreads * kHeavyPer;     // rows of a head that one workgroup sorts out

// One more row of `bin` for the lanes that are `in`: lanes that share the first one's bin (rows of
// no weight at all, often most of them) add together, the others one by one.
__device__ __forceinline__ void count_bin(uint32_t* hist, bool in, uint32_t bin, int lane) {
  const uint64_t act = __ballot(in);
  if (act) {
    const uint32_t lead = (uint32_t)__builtin_amdgcn_readlane((int)bin, __ffsll((unsigned long long)act) - 1);
    const uint64_t same = __ballot(in && bin == lead);
    if (lane == 0) atomicAdd(&hist[lead], (uint32_t)__popcll(same));
    if (in && bin != lead) atomicAdd(&hist[bin], 1u);
  }
}

// The highest bin such that it and those above hold at least `need` rows, and how many of its own
// rows are needed.  Thread t brings the counts of bins 2 t and 2 t + 1; called by all threads, the
// counts' writes already waited for.
__device__ __forceinline__ void pick_bin(uint32_t c0, uint32_t c1, uint32_t& need, uint32_t& bin, uint32_t* s_wave,
                                         uint32_t* s_pick, int tid) {
  const int lane = tid & 63, wid = tid >> 6;
  uint32_t suf = c0 + c1;  // becomes the sum over this thread's bins and those above
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t up = (uint32_t)__shfl_down((int)suf, d, 64);
    suf += lane + d < 64 ? up : 0;
  }
  if (lane == 0) s_wave[wid] = suf;
  __syncthreads();
  for (int w = wid + 1; w < kHeavyWaves; ++w) suf += s_wave[w];
  const uint32_t after1 = suf - c0 - c1;  // rows in bins above 2 t + 1
  if (after1 < need && after1 + c1 >= need) {
    s_pick[0] = 2 * tid + 1;
    s_pick[1] = need - after1;
  } else if (after1 + c1 < need && suf >= need) {
    s_pick[0] = 2 * tid;
    s_pick[1] = need - after1 - c1;
  }
  __syncthreads();
  bin = s_pick[0];
  need = s_pick[1];
}

__device__ __forceinline__ int heavy_length(const HeavyArgs& a, int bh) {
  const int n = a.lengths ? a.lengths[bh] : (int)a.capacity;
  return n < 0 ? 0 : (n > a.capacity ? (int)a.capacity : n);
}

// Heads of at most kHeavyShort rows, one workgroup each, every mass read once and kept in
// registers.  The border (the need-th largest mass between the protected ends) comes from three
// histogram passes over 11, 11 and 10 bits of the order; then the rows above it are written, and as
// many of its equals as still fit, lowest row first, in row order.
__device__ __forceinline__ void heavy_choose(const HeavyArgs& a, int32_t* out) {
  __shared__ uint32_t s_hist[kHeavyBins];
  __shared__ uint32_t s_wave[kHeavyWaves];
  __shared__ uint32_t s_cnt[2][kHeavyPer * kHeavyWaves];  // rows above / at the border, in row order
  __shared__ uint32_t s_pick[2];
  const int bh = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int n = heavy_length(a, bh);
  if (tid == 0) a.kept[bh] = n < a.budget ? n : a.budget;
  if (n <= a.budget) {
    for (int i = tid; i < a.budget; i += kHeavyThreads) out[i] = i < n ? i : -1;
    return;
  }
  const float* const mass = a.mass + (int64_t)bh * a.capacity;
  const int lo = a.sinks, hi = n - a.recent;  // the rows that compete
  uint32_t u[kHeavyPer];
  {
    float m[kHeavyPer];
#pragma unroll
    for (int j = 0; j < kHeavyPer; ++j) {
      const int i = lo + j * kHeavyThreads + tid;
      m[j] = i < hi ? mass[i] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kHeavyPer; ++j) u[j] = mass_order(m[j]);
  }
  for (int i = tid; i < a.sinks; i += kHeavyThreads) out[i] = i;
  for (int i = tid; i < a.recent; i += kHeavyThreads) out[a.budget - a.recent + i] = hi + i;
  uint32_t need = (uint32_t)(a.budget - a.sinks - a.recent);
  if (need == 0) return;
  uint32_t prefix = 0, mask = 0;  // bits of the border found so far
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
    const uint32_t bits = pass == 2 ? 1023u : 2047u;
    s_hist[tid] = 0;
    s_hist[tid + kHeavyThreads] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kHeavyPer; ++j) {
      const int row = lo + j * kHeavyThreads;
      if (row < hi) count_bin(s_hist, row + tid < hi && (u[j] & mask) == prefix, (u[j] >> shift) & bits, lane);
    }
    __syncthreads();
    uint32_t bin;
    pick_bin(s_hist[2 * tid], s_hist[2 * tid + 1], need, bin, s_wave, s_pick, tid);
    prefix |= bin << shift;
    mask |= bits << shift;
  }
  uint64_t bg[kHeavyPer], be[kHeavyPer];
#pragma unroll
  for (int j = 0; j < kHeavyPer; ++j) {
    const bool in = lo + j * kHeavyThreads + tid < hi;
    bg[j] = __ballot(in && u[j] > prefix);
    be[j] = __ballot(in && u[j] == prefix);
    if (lane == 0) {
      s_cnt[0][j * kHeavyWaves + wid] = (uint32_t)__popcll(bg[j]);
      s_cnt[1][j * kHeavyWaves + wid] = (uint32_t)__popcll(be[j]);
    }
  }
  __syncthreads();
  if (wid < 2) {  // prefix sums of the 256 counts, four a lane: wave 0 above, wave 1 at the border
    uint32_t c[4], run = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      c[j] = s_cnt[wid][4 * lane + j];
      run += c[j];
    }
    uint32_t inc = run;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t dn = (uint32_t)__shfl_up((int)inc, d, 64);
      inc += lane >= d ? dn : 0;
    }
    uint32_t at = inc - run;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      s_cnt[wid][4 * lane + j] = at;
      at += c[j];
    }
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int j = 0; j < kHeavyPer; ++j) {
    const uint32_t g = s_cnt[0][j * kHeavyWaves + wid] + (uint32_t)__popcll(bg[j] & below);
    const uint32_t e = s_cnt[1][j * kHeavyWaves + wid] + (uint32_t)__popcll(be[j] & below);
    const bool gt = (bg[j] >> lane) & 1, eq = (be[j] >> lane) & 1;
    if (gt || (eq && e < need)) out[a.sinks + g + (e < need ? e : need)] = lo + j * kHeavyThreads + tid;
  }
}

__global__ __launch_bounds__(kHeavyThreads) void heavy_rows_kernel(HeavyArgs a) {
  heavy_choose(a, a.index + (int64_t)blockIdx.x * a.budget);
}

// Longer heads in chunks of kChunk rows, a workgroup each, in five launches that take the chip:
// histogram of the top 11 bits a chunk; the border's bin a head; the rows of that bin, listed a
// chunk; the border itself from the lists, and what every chunk keeps; the rows' numbers.  (One
// workgroup a head took 120 us for 131072 rows, where these take a quarter.)
constexpr int kChunkPer = 4, kChunk = kHeavyThreads * kChunkPer;

struct HeavyWork {      // per head and chunk, in the workspace
  uint32_t* hist;       // [bh][chunks][kHeavyBins]
  uint32_t* list;       // [bh][chunks][kChunk]: orders of the rows of the border's bin
  uint32_t* count;      // [bh][chunks][4]: rows in the list; rows above (first: in higher bins) and at the border
  uint32_t* border;     // [bh][4]: bin, rows needed of it; border, equals needed
  int chunks;
};

__device__ __forceinline__ void chunk_masses(const HeavyArgs& a, int bh, int first, int lo, int hi,
                                             uint32_t (&u)[kChunkPer], bool (&in)[kChunkPer]) {
  const float* const mass = a.mass + (int64_t)bh * a.capacity;
  float m[kChunkPer];
#pragma unroll
  for (int j = 0; j < kChunkPer; ++j) {
    const int i = first + j * kHeavyThreads + (int)threadIdx.x;
    in[j] = i >= lo && i < hi;
    m[j] = in[j] ? mass[i] : 0.0f;
  }
#pragma unroll
  for (int j = 0; j < kChunkPer; ++j) u[j] = mass_order(m[j]);
}

__global__ __launch_bounds__(kHeavyThreads) void heavy_hist_kernel(HeavyArgs a, HeavyWork w) {
  __shared__ uint32_t s_hist[kHeavyBins];
  const int bh = blockIdx.x / w.chunks, c = blockIdx.x - bh * w.chunks, tid = threadIdx.x;
  const int n = heavy_length(a, bh);
  if (n <= a.budget) return;
  s_hist[tid] = 0;
  s_hist[tid + kHeavyThreads] = 0;
  uint32_t u[kChunkPer];
  bool in[kChunkPer];
  chunk_masses(a, bh, c * kChunk, a.sinks, n - a.recent, u, in);
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kChunkPer; ++j) count_bin(s_hist, in[j], u[j] >> 21, tid & 63);
  __syncthreads();
  uint32_t* const h = w.hist + (int64_t)blockIdx.x * kHeavyBins;
  h[tid] = s_hist[tid];
  h[tid + kHeavyThreads] = s_hist[tid + kHeavyThreads];
}

__global__ __launch_bounds__(kHeavyThreads) void heavy_bin_kernel(HeavyArgs a, HeavyWork w) {
  __shared__ uint32_t s_wave[kHeavyWaves];
  __shared__ uint32_t s_pick[2];
  const int bh = blockIdx.x, tid = threadIdx.x;
  const int n = heavy_length(a, bh);
  if (tid == 0) a.kept[bh] = n < a.budget ? n : a.budget;
  uint32_t need = (uint32_t)(a.budget - a.sinks - a.recent), bin = kHeavyBins;  // none: no row competes for a place
  if (n > a.budget && need > 0) {
    uint32_t c0 = 0, c1 = 0;
    const u32x2* h = (const u32x2*)(const void*)(w.hist + (int64_t)bh * w.chunks * kHeavyBins) + tid;
#pragma unroll 16
    for (int c = 0; c < w.chunks; ++c) {
      const u32x2 v = h[(int64_t)c * (kHeavyBins / 2)];
      c0 += v[0];
      c1 += v[1];
    }
    pick_bin(c0, c1, need, bin, s_wave, s_pick, tid);
  }
  if (tid == 0) {
    w.border[4 * bh] = bin;
    w.border[4 * bh + 1] = need;
  }
}

__global__ __launch_bounds__(kHeavyThreads) void heavy_list_kernel(HeavyArgs a, HeavyWork w) {
  __shared__ uint32_t s_fill, s_above;
  const int bh = blockIdx.x / w.chunks, c = blockIdx.x - bh * w.chunks, tid = threadIdx.x, lane = tid & 63;
  const int n = heavy_length(a, bh);
  if (n <= a.budget) return;
  const uint32_t bin = w.border[4 * bh];
  if (tid == 0) s_fill = s_above = 0;
  uint32_t u[kChunkPer];
  bool in[kChunkPer];
  chunk_masses(a, bh, c * kChunk, a.sinks, n - a.recent, u, in);
  __syncthreads();
  uint32_t* const list = w.list + (int64_t)blockIdx.x * kChunk;
  uint32_t above = 0;  // of this wave
#pragma unroll
  for (int j = 0; j < kChunkPer; ++j) {
    const bool hit = in[j] && (u[j] >> 21) == bin;
    above += (uint32_t)__popcll(__ballot(in[j] && (u[j] >> 21) > bin));
    const uint64_t act = __ballot(hit);
    if (act) {
      uint32_t at = 0;
      if (lane == 0) at = atomicAdd(&s_fill, (uint32_t)__popcll(act));
      at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + (uint32_t)__popcll(act & ((1ull << lane) - 1));
      if (hit) list[at] = u[j];
    }
  }
  if (lane == 0 && above) atomicAdd(&s_above, above);
  __syncthreads();
  if (tid == 0) {
    w.count[4 * blockIdx.x] = s_fill;
    w.count[4 * blockIdx.x + 1] = s_above;
  }
}

__global__ __launch_bounds__(kHeavyThreads) void heavy_border_kernel(HeavyArgs a, HeavyWork w) {
  __shared__ uint32_t s_hist[kHeavyBins];
  __shared__ uint32_t s_wave[kHeavyWaves];
  __shared__ uint32_t s_pick[2];
  const int bh = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int n = heavy_length(a, bh);
  if (n <= a.budget) return;
  const uint32_t bin = w.border[4 * bh];
  uint32_t need = w.border[4 * bh + 1];
  uint32_t prefix = bin << 21, mask = 2047u << 21;
  uint32_t* const count = w.count + (int64_t)bh * w.chunks * 4;
  const uint32_t* const list = w.list + (int64_t)bh * w.chunks * kChunk;
  const bool any = bin < kHeavyBins;
  if (any) {
    for (int pass = 1; pass < 3; ++pass) {
      const int shift = pass == 1 ? 10 : 0;
      const uint32_t bits = pass == 1 ? 2047u : 1023u;
      s_hist[tid] = 0;
      s_hist[tid + kHeavyThreads] = 0;
      __syncthreads();
      for (int c = wid; c < w.chunks; c += kHeavyWaves) {
        const uint32_t fill = count[4 * c];
        for (uint32_t i0 = 0; i0 < fill; i0 += 256) {
          uint32_t v[4];
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j) v[j] = i0 + 64 * j + lane < fill ? list[(int64_t)c * kChunk + i0 + 64 * j + lane] : 0;
#pragma unroll
          for (uint32_t j = 0; j < 4; ++j)
            count_bin(s_hist, i0 + 64 * j + lane < fill && (v[j] & mask) == prefix, (v[j] >> shift) & bits, lane);
        }
      }
      __syncthreads();
      uint32_t b2;
      pick_bin(s_hist[2 * tid], s_hist[2 * tid + 1], need, b2, s_wave, s_pick, tid);
      prefix |= b2 << shift;
      mask |= bits << shift;
    }
  }
  if (tid == 0) {
    w.border[4 * bh + 2] = any ? prefix : 0xffffffffu;
    w.border[4 * bh + 3] = any ? need : 0;
  }
  // rows of each chunk above the border (the list kernel counted those of higher bins) and at it
  for (int c = wid; c < w.chunks; c += kHeavyWaves) {
    uint32_t g = 0, e = 0;
    if (any) {
      const uint32_t fill = count[4 * c];
      g = lane == 0 ? count[4 * c + 1] : 0;
#pragma unroll 4
      for (uint32_t i = lane; i < fill; i += 64) {
        const uint32_t v = list[(int64_t)c * kChunk + i];
        g += v > prefix ? 1 : 0;
        e += v == prefix ? 1 : 0;
      }
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        g += (uint32_t)__shfl_xor((int)g, d, 64);
        e += (uint32_t)__shfl_xor((int)e, d, 64);
      }
    }
    if (lane == 0) {
      count[4 * c + 1] = g;
      count[4 * c + 2] = e;
    }
  }
}

__global__ __launch_bounds__(kHeavyThreads) void heavy_index_kernel(HeavyArgs a, HeavyWork w) {
  __shared__ uint32_t s_cnt[2][kChunkPer * kHeavyWaves];
  __shared__ uint32_t s_before[2];
  const int bh = blockIdx.x / w.chunks, c = blockIdx.x - bh * w.chunks;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int n = heavy_length(a, bh);
  int32_t* const out = a.index + (int64_t)bh * a.budget;
  const int first = c * kChunk;
  if (n <= a.budget) {  // all rows, then -1 (the last chunk's workgroup writes what is past the chunks)
    const int end = c == w.chunks - 1 ? a.budget : min(first + kChunk, a.budget);
    for (int i = first + tid; i < end; i += kHeavyThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int lo = a.sinks, hi = n - a.recent;
  const uint32_t border = w.border[4 * bh + 2], need = w.border[4 * bh + 3];
  uint32_t u[kChunkPer];
  bool in[kChunkPer];
  chunk_masses(a, bh, first, lo, hi, u, in);
  if (wid < 2) {  // rows above / at the border in the chunks before
    uint32_t v = 0;
    for (int i = lane; i < c; i += 64) v += w.count[((int64_t)bh * w.chunks + i) * 4 + 1 + wid];
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += (uint32_t)__shfl_xor((int)v, d, 64);
    if (lane == 0) s_before[wid] = v;
  }
  uint64_t bg[kChunkPer], be[kChunkPer];
#pragma unroll
  for (int j = 0; j < kChunkPer; ++j) {
    bg[j] = __ballot(in[j] && u[j] > border);
    be[j] = __ballot(in[j] && u[j] == border);
    if (lane == 0) {
      s_cnt[0][j * kHeavyWaves + wid] = (uint32_t)__popcll(bg[j]);
      s_cnt[1][j * kHeavyWaves + wid] = (uint32_t)__popcll(be[j]);
    }
  }
  __syncthreads();
  if (wid < 2) {
    const uint32_t own = s_cnt[wid][lane];
    uint32_t inc = own;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t dn = (uint32_t)__shfl_up((int)inc, d, 64);
      inc += lane >= d ? dn : 0;
    }
    s_cnt[wid][lane] = inc - own + s_before[wid];
  }
  __syncthreads();
  const uint64_t below = (1ull << lane) - 1;
#pragma unroll
  for (int j = 0; j < kChunkPer; ++j) {
    const int row = first + j * kHeavyThreads + tid;
    const uint32_t g = s_cnt[0][j * kHeavyWaves + wid] + (uint32_t)__popcll(bg[j] & below);
    const uint32_t e = s_cnt[1][j * kHeavyWaves + wid] + (uint32_t)__popcll(be[j] & below);
    const bool gt = (bg[j] >> lane) & 1, eq = (be[j] >> lane) & 1;
    if (gt || (eq && e < need)) out[a.sinks + g + (e < need ? e : need)] = row;
    else if (row < lo) out[row] = row;
    else if (row >= hi && row < n) out[a.budget - n + row] = row;
  }
}
static_assert(kChunkPer * kHeavyWaves == 64, "one count a lane");

// ------------------------------------------------------------------------------------
// eviction: the rows moved
// ------------------------------------------------------------------------------------
struct Move4Args {
  const uint8_t* codes[2];
  const uint8_t* scales[2];
  uint8_t* o_codes[2];
  uint8_t* o_scales[2];
  const int32_t* counts;
  const int32_t* ts;
  const float* mass;
  int32_t* o_counts;
  int32_t* o_ts;
  float* o_mass;
  const int32_t* index;
  int64_t capacity, o_capacity;
  int budget;
};

// A row's exponent bytes, as one access where they are 1, 2 or 4.
template <int NG>
__device__ __forceinline__ uint32_t load_scales(const uint8_t* p) {
  if constexpr (NG == 4) return *(const uint32_t*)p;
  else if constexpr (NG == 2) return *(const uint16_t*)p;
  else if constexpr (NG == 1) return *p;
  else return p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16;
}
template <int NG>
__device__ __forceinline__ void store_scales(uint8_t* p, uint32_t v) {
  if constexpr (NG == 4) *(uint32_t*)p = v;
  else if constexpr (NG == 2) *(uint16_t*)p = (uint16_t)v;
  else if constexpr (NG == 1) *p = (uint8_t)v;
  else {
    p[0] = (uint8_t)v;
    p[1] = (uint8_t)(v >> 8);
    p[2] = (uint8_t)(v >> 16);
  }
}

// Row m's exponents, count, timestamp and mass from row src, zero where there is none.
template <int NG>
__device__ __forceinline__ void move_fields(const Move4Args& a, int bh, int m, int src) {
  const int64_t to = bh * a.o_capacity + m, from = bh * a.capacity + src;
  uint32_t ks = 0, vs = 0;
  int c = 0, t = 0;
  float w = 0.0f;
  if (src >= 0) {
    ks = load_scales<NG>(a.scales[0] + from * NG);
    vs = load_scales<NG>(a.scales[1] + from * NG);
    c = a.counts[from];
    t = a.ts[from];
    w = a.mass[from];
  }
  store_scales<NG>(a.o_scales[0] + to * NG, ks);
  store_scales<NG>(a.o_scales[1] + to * NG, vs);
  a.o_counts[to] = c;
  a.o_ts[to] = t;
  a.o_mass[to] = w;
}

// blockIdx.z = 0: a lane moves 16 bytes of codes (2 NG lanes a row, keys then values), read once and
// past the caches; z = 1: a lane moves a row's small fields.  (With the fields on the codes' lanes the
// memory instructions a row were three times as many: 131072 rows x 8 heads to 32768
// took 29 us against 22, a ragged batch of 16 47 against 31, 4.9 TB/s.)
constexpr int kMoveItems = 2;
template <int NG>
__global__ __launch_bounds__(256) void move4_kernel(Move4Args a) {
  constexpr uint32_t kLpr = 2 * NG;
  const int bh = blockIdx.y;
  const int32_t* const index = a.index + (int64_t)bh * a.budget;
  if (blockIdx.z == 1) {
    for (int m = blockIdx.x * 256 + threadIdx.x; m < a.budget; m += gridDim.x * 256)
      move_fields<NG>(a, bh, m, index[m]);
    return;
  }
  const uint32_t first = blockIdx.x * 256 * kMoveItems + threadIdx.x;
  u32x4 w[kMoveItems];
  int src[kMoveItems];
#pragma unroll
  for (int u = 0; u < kMoveItems; ++u) {
    const uint32_t m = (first + u * 256) / kLpr;
    src[u] = m < (uint32_t)a.budget ? index[m] : -1;
  }
#pragma unroll
  for (int u = 0; u < kMoveItems; ++u) {
    const int c = (int)((first + u * 256) % kLpr), z = c >= NG ? 1 : 0;
    w[u] = u32x4{0, 0, 0, 0};
    if (src[u] >= 0)
      w[u] = __builtin_nontemporal_load((const u32x4*)(a.codes[z] + ((bh * a.capacity + src[u]) * NG + (c - z * NG)) * 16));
  }
#pragma unroll
  for (int u = 0; u < kMoveItems; ++u) {
    const uint32_t it = first + u * 256, m = it / kLpr;
    if (m >= (uint32_t)a.budget) continue;
    const int c = (int)(it - m * kLpr), z = c >= NG ? 1 : 0, cc = c - z * NG;
    *(u32x4*)(a.o_codes[z] + ((bh * a.o_capacity + m) * NG + cc) * 16) = w[u];
  }
}

// A small budget's choice and move in one launch, the rows' numbers in LDS (8 heads of 60 rows to 40:
// 12.1 us against 13.2, of 300 to 256 12.6 / 13.2, and 3.4 us less of the caller's time; of 600 to 512
// 13.6 / 13.4, of 2111 to 2048 24.6 / 15.2: one workgroup a head moves slowly).
constexpr int kSmallBudget = 256;
template <int NG>
__global__ __launch_bounds__(kHeavyThreads) void evict_small_kernel(HeavyArgs h, Move4Args a) {
  __shared__ int32_t s_index[kSmallBudget];
  const int bh = blockIdx.x, tid = threadIdx.x;
  heavy_choose(h, s_index);
  __syncthreads();
  for (int m = tid; m < a.budget; m += kHeavyThreads) {
    move_fields<NG>(a, bh, m, s_index[m]);
    if (h.index) h.index[(int64_t)bh * a.budget + m] = s_index[m];
  }
  for (int it = tid; it < a.budget * 2 * NG; it += kHeavyThreads) {
    const int m = it / (2 * NG), c = it - m * (2 * NG), z = c >= NG ? 1 : 0, cc = c - z * NG, src = s_index[m];
    u32x4 w = u32x4{0, 0, 0, 0};
    if (src >= 0) w = __builtin_nontemporal_load((const u32x4*)(a.codes[z] + ((bh * a.capacity + src) * NG + cc) * 16));
    *(u32x4*)(a.o_codes[z] + ((bh * a.o_capacity + m) * NG + cc) * 16) = w;
  }
}

static int check_kv4(const DaKv4* kv, int64_t B, int64_t Hkv, int64_t D, bool mass, const char* who) {
  DA_REQUIRE(kv, "%s: null cache", who);
  DA_REQUIRE(kv->k_codes && kv->k_scales && kv->v_codes && kv->v_scales && kv->counts && kv->timestamps &&
                 kv->lengths && (!mass || kv->mass),
             "%s: null pointer in the cache", who);
  if (D <= 0 || D > 128 || (D & 7))
    return set_error(DA_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 in [8, 128]", who);
  DA_REQUIRE(B > 0 && Hkv > 0 && kv->capacity > 0, "%s: empty shape", who);
  DA_REQUIRE(B * Hkv <= 65535, "%s: at most 65535 (sequence, head) pairs", who);
  if (kv->capacity > (1 << 26)) return set_error(DA_ERR_UNSUPPORTED, "%s: capacity above 2^26 rows", who);
  DA_REQUIRE((((uintptr_t)kv->k_codes | (uintptr_t)kv->v_codes) & 15) == 0, "%s: codes must be 16-byte aligned", who);
  DA_REQUIRE((((uintptr_t)kv->k_scales | (uintptr_t)kv->v_scales) & 3) == 0, "%s: exponents must be 4-byte aligned", who);
  return DA_OK;
}

template <int DT>
static void launch_quantize(const Quant4Args& a, int groups, dim3 grid, hipStream_t st) {
  switch (groups) {
    case 1: hipLaunchKernelGGL((quantize4_kernel<DT, 1>), grid, dim3(256), 0, st, a); break;
    case 2: hipLaunchKernelGGL((quantize4_kernel<DT, 2>), grid, dim3(256), 0, st, a); break;
    case 3: hipLaunchKernelGGL((quantize4_kernel<DT, 3>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((quantize4_kernel<DT, 4>), grid, dim3(256), 0, st, a); break;
  }
}
template <int DT>
static void launch_dequantize(const Dequant4Args& a, int groups, dim3 grid, hipStream_t st) {
  switch (groups) {
    case 1: hipLaunchKernelGGL((dequantize4_kernel<DT, 1>), grid, dim3(256), 0, st, a); break;
    case 2: hipLaunchKernelGGL((dequantize4_kernel<DT, 2>), grid, dim3(256), 0, st, a); break;
    case 3: hipLaunchKernelGGL((dequantize4_kernel<DT, 3>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((dequantize4_kernel<DT, 4>), grid, dim3(256), 0, st, a); break;
  }
}

static int check_budget(int64_t budget, int64_t sinks, int64_t recent, const char* who) {
  DA_REQUIRE(budget > 0 && budget <= (1 << 26) && sinks >= 0 && recent >= 0 && sinks <= budget &&
                 recent <= budget - sinks,
             "%s: needs sinks + recent <= budget, budget in [1, 2^26]", who);
  return DA_OK;
}

static bool evict_small(int64_t capacity, int64_t budget) { return capacity <= kHeavyShort && budget <= kSmallBudget; }

// The choice's scratch for heads that may be longer than kHeavyShort rows, after `at`.
static HeavyWork heavy_work(int64_t BH, int64_t capacity, uint32_t* at, int64_t* bytes) {
  HeavyWork w = {};
  w.chunks = capacity > kHeavyShort ? (int)((capacity + kChunk - 1) / kChunk) : 0;
  const int64_t n = BH * w.chunks;
  w.hist = at;
  w.list = w.hist + n * kHeavyBins;
  w.count = w.list + n * kChunk;
  w.border = w.count + n * 4;
  *bytes = (n * (kHeavyBins + kChunk + 4) + (n ? BH * 4 : 0)) * (int64_t)sizeof(uint32_t);
  return w;
}

static int launch_heavy(const float* mass, const int32_t* lengths, int64_t BH, int64_t capacity, int64_t budget,
                        int64_t sinks, int64_t recent, int32_t* index, int32_t* kept, void* workspace, hipStream_t st,
                        const char* who) {
  HeavyArgs a = {};
  a.mass = mass; a.lengths = lengths; a.capacity = capacity;
  a.budget = (int)budget; a.sinks = (int)sinks; a.recent = (int)recent;
  a.index = index; a.kept = kept;
  int64_t bytes;
  const HeavyWork w = heavy_work(BH, capacity, (uint32_t*)workspace, &bytes);
  if (w.chunks == 0) {
    hipLaunchKernelGGL(heavy_rows_kernel, dim3((unsigned)BH), dim3(kHeavyThreads), 0, st, a);
    return check_launch(who);
  }
  // a launch holds fewer than 2^32 threads
  if (BH * w.chunks >= (1ll << 22)) return set_error(DA_ERR_UNSUPPORTED, "%s: too many rows for one call", who);
  const dim3 all((unsigned)(BH * w.chunks)), heads((unsigned)BH);
  hipLaunchKernelGGL(heavy_hist_kernel, all, dim3(kHeavyThreads), 0, st, a, w);
  hipLaunchKernelGGL(heavy_bin_kernel, heads, dim3(kHeavyThreads), 0, st, a, w);
  hipLaunchKernelGGL(heavy_list_kernel, all, dim3(kHeavyThreads), 0, st, a, w);
  hipLaunchKernelGGL(heavy_border_kernel, heads, dim3(kHeavyThreads), 0, st, a, w);
  hipLaunchKernelGGL(heavy_index_kernel, all, dim3(kHeavyThreads), 0, st, a, w);
  return check_launch(who);
}

}  // namespace da

using namespace da;

extern "C" int da_kv4_quantize(const void* k, const void* v, int dtype, int64_t B, int64_t Hkv, int64_t N, int64_t D,
                               int64_t sk_b, int64_t sk_h, int64_t sk_n, int64_t sv_b, int64_t sv_h, int64_t sv_n,
                               const int32_t* counts, const int32_t* timestamps, const float* mass,
                               const int32_t* lengths, const int32_t* index, int64_t M, const DaKv4* out,
                               void* stream) {
  const char* who = "da_kv4_quantize";
  DA_REQUIRE(k && v, "%s: null pointer", who);
  if (int rc = check_kv4(out, B, Hkv, D, false, who)) return rc;
  if (dtype != DA_BF16 && dtype != DA_F16 && dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: rows must be bf16, fp16 or fp32", who);
  DA_REQUIRE(N > 0 && N <= (1 << 26) && M > 0 && M <= out->capacity && (index || M == N),
             "%s: needs 0 < M <= capacity, and M = N without an index", who);
  const int64_t align = dtype == DA_F32 ? 3 : 7;
  // a dimension of one has no stride
  const int64_t strides = (B > 1 ? sk_b | sv_b : 0) | (Hkv > 1 ? sk_h | sv_h : 0) | (N > 1 ? sk_n | sv_n : 0);
  DA_REQUIRE((strides & align) == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0,
             "%s: rows must be 16-byte aligned", who);
  Quant4Args a = {};
  a.x[0] = k; a.s_b[0] = sk_b; a.s_h[0] = sk_h; a.s_n[0] = sk_n;
  a.x[1] = v; a.s_b[1] = sv_b; a.s_h[1] = sv_h; a.s_n[1] = sv_n;
  a.codes[0] = out->k_codes; a.codes[1] = out->v_codes;
  a.scales[0] = out->k_scales; a.scales[1] = out->v_scales;
  a.counts = counts; a.ts = timestamps; a.mass = mass; a.lengths = lengths; a.index = index;
  a.o_counts = out->counts; a.o_ts = out->timestamps; a.o_mass = out->mass; a.o_lengths = out->lengths;
  a.N = N; a.M = M; a.capacity = out->capacity; a.B = (int)B; a.H = (int)Hkv; a.D = (int)D;
  const int groups = (int)((D + 31) / 32);
  const int64_t blocks = (M * 4 * groups + 256 * kQuantItems - 1) / (256 * kQuantItems);
  const dim3 grid((unsigned)blocks, (unsigned)(B * Hkv), 3);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DA_F32) launch_quantize<DA_F32>(a, groups, grid, st);
  else if (dtype == DA_F16) launch_quantize<DA_F16>(a, groups, grid, st);
  else launch_quantize<DA_BF16>(a, groups, grid, st);
  return check_launch(who);
}

extern "C" int da_kv4_dequantize(const DaKv4* kv, int64_t B, int64_t Hkv, int64_t N, int64_t D, void* k, void* v,
                                 int dtype, void* stream) {
  const char* who = "da_kv4_dequantize";
  if (int rc = check_kv4(kv, B, Hkv, D, false, who)) return rc;
  if (dtype != DA_BF16 && dtype != DA_F16 && dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: rows must be bf16, fp16 or fp32", who);
  DA_REQUIRE(k && v && (((uintptr_t)k | (uintptr_t)v) & 15) == 0, "%s: rows must be 16-byte aligned", who);
  DA_REQUIRE(N > 0 && N <= kv->capacity, "%s: needs 0 < N <= capacity", who);
  Dequant4Args a = {};
  a.codes[0] = kv->k_codes; a.codes[1] = kv->v_codes;
  a.scales[0] = kv->k_scales; a.scales[1] = kv->v_scales;
  a.x[0] = k; a.x[1] = v; a.lengths = kv->lengths; a.N = N; a.capacity = kv->capacity; a.D = (int)D;
  const int groups = (int)((D + 31) / 32);
  const int64_t blocks = (N * 4 * groups + 256 * kQuantItems - 1) / (256 * kQuantItems);
  const dim3 grid((unsigned)blocks, (unsigned)(B * Hkv), 2);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DA_F32) launch_dequantize<DA_F32>(a, groups, grid, st);
  else if (dtype == DA_F16) launch_dequantize<DA_F16>(a, groups, grid, st);
  else launch_dequantize<DA_BF16>(a, groups, grid, st);
  return check_launch(who);
}

// The choice's scratch, then the rows kept, [B, Hkv, budget].
extern "C" int64_t da_kv4_evict_workspace_size(int64_t B, int64_t Hkv, int64_t capacity, int64_t budget) {
  if (B <= 0 || Hkv <= 0 || capacity <= 0 || budget <= 0) return 0;
  if (evict_small(capacity, budget)) return 0;
  int64_t bytes;
  heavy_work(B * Hkv, capacity, nullptr, &bytes);
  return bytes + B * Hkv * budget * (int64_t)sizeof(int32_t);
}

extern "C" int da_kv4_evict(const DaKv4* kv, int64_t B, int64_t Hkv, int64_t D, int64_t budget, int64_t sinks,
                            int64_t recent, const DaKv4* out, int32_t* index, void* workspace,
                            int64_t workspace_bytes, void* stream) {
  const char* who = "da_kv4_evict";
  if (int rc = check_kv4(kv, B, Hkv, D, true, who)) return rc;
  if (int rc = check_kv4(out, B, Hkv, D, true, who)) return rc;
  if (int rc = check_budget(budget, sinks, recent, who)) return rc;
  DA_REQUIRE(budget <= out->capacity, "%s: the budget exceeds the new cache's capacity", who);
  DA_REQUIRE(kv->k_codes != out->k_codes && kv->v_codes != out->v_codes && kv->mass != out->mass &&
                 kv->counts != out->counts && kv->lengths != out->lengths,
             "%s: the rows move to other memory", who);
  const int64_t need = da_kv4_evict_workspace_size(B, Hkv, kv->capacity, budget);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %lld bytes required", who, (long long)need);
  DA_REQUIRE(((uintptr_t)workspace & 15) == 0, "%s: workspace must be 16-byte aligned", who);
  hipStream_t st = (hipStream_t)stream;
  Move4Args a = {};
  a.codes[0] = kv->k_codes; a.codes[1] = kv->v_codes;
  a.scales[0] = kv->k_scales; a.scales[1] = kv->v_scales;
  a.o_codes[0] = out->k_codes; a.o_codes[1] = out->v_codes;
  a.o_scales[0] = out->k_scales; a.o_scales[1] = out->v_scales;
  a.counts = kv->counts; a.ts = kv->timestamps; a.mass = kv->mass;
  a.o_counts = out->counts; a.o_ts = out->timestamps; a.o_mass = out->mass;
  a.capacity = kv->capacity; a.o_capacity = out->capacity; a.budget = (int)budget;
  const int groups = (int)((D + 31) / 32);
  if (evict_small(kv->capacity, budget)) {
    const HeavyArgs h = {kv->mass, kv->lengths, kv->capacity, (int)budget, (int)sinks, (int)recent, index, out->lengths};
    const dim3 heads((unsigned)(B * Hkv));
    switch (groups) {
      case 1: hipLaunchKernelGGL((evict_small_kernel<1>), heads, dim3(kHeavyThreads), 0, st, h, a); break;
      case 2: hipLaunchKernelGGL((evict_small_kernel<2>), heads, dim3(kHeavyThreads), 0, st, h, a); break;
      case 3: hipLaunchKernelGGL((evict_small_kernel<3>), heads, dim3(kHeavyThreads), 0, st, h, a); break;
      default: hipLaunchKernelGGL((evict_small_kernel<4>), heads, dim3(kHeavyThreads), 0, st, h, a); break;
    }
    return check_launch(who);
  }
  int64_t scratch;
  heavy_work(B * Hkv, kv->capacity, nullptr, &scratch);
  int32_t* rows = index ? index : (int32_t*)((char*)workspace + scratch);
  if (int rc = launch_heavy(kv->mass, kv->lengths, B * Hkv, kv->capacity, budget, sinks, recent, rows, out->lengths,
                            workspace, st, who))
    return rc;
  a.index = rows;
  const dim3 grid((unsigned)((budget * 2 * groups + 256 * kMoveItems - 1) / (256 * kMoveItems)), (unsigned)(B * Hkv), 2);
  switch (groups) {
    case 1: hipLaunchKernelGGL((move4_kernel<1>), grid, dim3(256), 0, st, a); break;
    case 2: hipLaunchKernelGGL((move4_kernel<2>), grid, dim3(256), 0, st, a); break;
    case 3: hipLaunchKernelGGL((move4_kernel<3>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((move4_kernel<4>), grid, dim3(256), 0, st, a); break;
  }
  return check_launch(who);
}

extern "C" int da_heavy_rows(const float* mass, const int32_t* lengths, int64_t B, int64_t Hkv, int64_t N,
                             int64_t budget, int64_t sinks, int64_t recent, int32_t* index, int32_t* kept,
                             void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "da_heavy_rows";
  DA_REQUIRE(mass && index && kept, "%s: null pointer", who);
  DA_REQUIRE(B > 0 && Hkv > 0 && N > 0 && N <= (1 << 26) && B * Hkv <= 65535, "%s: bad shape", who);
  if (int rc = check_budget(budget, sinks, recent, who)) return rc;
  const int64_t need = da_kv4_evict_workspace_size(B, Hkv, N, budget);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %lld bytes required", who, (long long)need);
  DA_REQUIRE(((uintptr_t)workspace & 15) == 0, "%s: workspace must be 16-byte aligned", who);
  return launch_heavy(mass, lengths, B * Hkv, N, budget, sinks, recent, index, kept, workspace, (hipStream_t)stream,
                      who);
}

template <int DT>
static void launch_update4(const Update4Args& a, bool cosine, hipStream_t st) {
  const dim3 grid((unsigned)((a.B * a.H + 3) / 4));
  if (cosine) hipLaunchKernelGGL((update4_kernel<true, DT>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((update4_kernel<false, DT>), grid, dim3(256), 0, st, a);
}

extern "C" int da_kv4_update(const void* new_k, const void* new_v, int dtype, int64_t B, int64_t Hkv, int64_t D,
                             int64_t sn_b, int64_t sn_h, void* k_exact, void* v_exact, int64_t sx_b, int64_t sx_h,
                             int64_t sx_s, const DaKv4* kv, void* k_last, int64_t exact_seq_len,
                             int64_t total_seq_len, int64_t window, float threshold, int use_cosine, void* stream) {
  const char* who = "da_kv4_update";
  DA_REQUIRE(new_k && new_v && k_exact && v_exact && k_last, "%s: null pointer", who);
  if (int rc = check_kv4(kv, B, Hkv, D, false, who)) return rc;
  if (dtype != DA_BF16 && dtype != DA_F16 && dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: rows must be bf16, fp16 or fp32", who);
  DA_REQUIRE(window > 0 && exact_seq_len >= 0 && total_seq_len >= 0, "%s: bad lengths", who);
  const uintptr_t pair_align = dtype == DA_F32 ? 7 : 3;
  DA_REQUIRE(((sn_b | sn_h | sx_b | sx_h | sx_s) & 1) == 0 &&
                 (((uintptr_t)new_k | (uintptr_t)new_v | (uintptr_t)k_exact | (uintptr_t)v_exact |
                   (uintptr_t)k_last) & pair_align) == 0,
             "%s: rows must be %d-byte aligned (even strides)", who, dtype == DA_F32 ? 8 : 4);
  Update4Args a = {};
  a.new_k = new_k; a.new_v = new_v; a.sn_b = sn_b; a.sn_h = sn_h;
  a.kx = k_exact; a.vx = v_exact; a.sx_b = sx_b; a.sx_h = sx_h; a.sx_s = sx_s;
  a.kv = *kv; a.k_last = k_last;
  a.exact_len = exact_seq_len; a.total_len = total_seq_len; a.window = window;
  a.B = (int)B; a.H = (int)Hkv; a.D = (int)D; a.thr = threshold;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DA_F32) launch_update4<DA_F32>(a, use_cosine != 0, st);
  else if (dtype == DA_F16) launch_update4<DA_F16>(a, use_cosine != 0, st);
  else launch_update4<DA_BF16>(a, use_cosine != 0, st);
  return check_launch(who);
}
