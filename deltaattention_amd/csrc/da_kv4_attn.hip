// Decode attention over key and value rows held in 4 bits (format: deltaattn_cache.h), with a
// ring of exact rows, on gfx950.
//
// For a query head: s_j = scale q . k_j + log c_j over the rows, s_j = scale q . k_j over the
// ring; out = sum_j softmax(s)_j v_j, and row j's weight, summed over the heads of its KV
// head's group, is added to its accumulated weight.
//
// The rows are what a call has to read: 34 ceil(D / 32) + 4 bytes each.  All heads of a group
// (up to 16, the columns of a 16 x 16 MFMA) share one reading of a row.  A row's values are
// E2M1 codes times a power of two, exact in bf16, and v_cvt_scalef32_pk_bf16_fp4 makes two of
// them in one instruction, so both products run on bf16 MFMA with K and V as they are; what has
// more bits is cut into bf16 parts whose sum is exact or near fp32: q into 1 (bf16), 2 (fp16)
// or 3 (fp32), the weights p into 2 (16-bit outputs) or 3.  Sums, maxima and partials are fp32.
//
// S = K Q^T, tile by tile of 16 keys: lane (r = lane % 16, t = lane / 16) of a K fragment holds
// 16 bytes of key r, which are group t of its row; MFMA m takes dims 32 t + 8 m .. + 7 of every
// lane, so four MFMAs cover 128 dims in the order that memory has them.  The accumulator of a
// lane is query head r and keys 4 t .. 4 t + 3.  O^T += V^T P^T over 32 keys: the B operand is p
// as it comes from S (slot e of lane t is key 4 t + e of the first 16, then of the second), and
// V^T comes from a bf16 copy of the tile in LDS through ds_read_b64_tr_b16 in the same order.
//
// Ring rows (bf16, fp16 or fp32, at most a few hundred) run on fp32 MFMA with values converted
// exactly, K from registers and V through LDS.
//
// The keys of a (sequence, KV head) are split over `nsplit` workgroups of four waves, tiles dealt
// out by the device's own length, so that a short cache leaves no workgroup more than a tile;
// a second launch joins the splits and adds the weights, which need the whole softmax.  A cache of
// at most 768 rows, or 1024 where the heads fill the chip, is one workgroup a head instead, which does
// all of it.
#include "da_common.hpp"
#include "../../include/deltaattn_cache.h"

namespace da {

typedef short i16x4v __attribute__((ext_vector_type(4)));

constexpr int kA4Waves = 4;                 // of a split's workgroup
constexpr int kA4Tile = 32;                 // keys a wave takes at once
constexpr int kA4VRow = 128 * 2 + 16;       // bytes of a bf16 V row in LDS, padded off the banks
constexpr int kA4Cols = 16;                 // query heads of one workgroup
constexpr float kLog2e = 1.4426950408889634f;

struct Attn4Args {
  const void* q;
  int64_t sq_b, sq_h;
  const uint8_t* kc;
  const uint8_t* ks;
  const uint8_t* vc;
  const uint8_t* vs;
  const int32_t* counts;
  const int32_t* lengths;
  int64_t capacity;
  const void* kx;
  const void* vx;
  int64_t sx_b, sx_h, sx_s;
  int exact_len;
  float scale_log2;
  void* out;
  int64_t so_b, so_h;
  float* mass;
  float* part;   // [bh][G][nsplit][128]: P.V
  float* stat;   // [bh][G][nsplit][2]: max (log2 units) and sum
  float* score;  // [bh][tile][G][32]: scores (log2 units), where the weights are wanted; score_cap rows a head
  int64_t score_cap;
  int nsplit;
  int B, Hkv, G, D;
};

constexpr int kA4Part = 128;

__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ f32x4 mfma16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

template <int SEL>
__device__ __forceinline__ uint32_t fp4_to_bf16x2(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, (bf16x2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
// eight codes (4 bytes) -> eight bf16 values
__device__ __forceinline__ u32x4 fp4_to_bf16x8(uint32_t w, float scale) {
  return u32x4{fp4_to_bf16x2<0>(w, scale), fp4_to_bf16x2<1>(w, scale), fp4_to_bf16x2<2>(w, scale),
               fp4_to_bf16x2<3>(w, scale)};
}

// max / sum over the four lanes l % 16 + 16 t, in registers
__device__ __forceinline__ float cols_max(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __builtin_fmaxf(__uint_as_float(x[0]), __uint_as_float(x[1]));
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __builtin_fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
}
__device__ __forceinline__ float cols_sum(float v) {
  const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(x[0]) + __uint_as_float(x[1]);
  const auto y = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(y[0]) + __uint_as_float(y[1]);
}

// Two fp32 values into N words of bf16 pairs, largest part first.
template <int N>
__device__ __forceinline__ void split_pair(float x0, float x1, uint32_t (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = pack_bf16x2(x0, x1);
    if (i + 1 < N) {
      x0 -= bf16_lo(w[i]);
      x1 -= bf16_hi(w[i]);
    }
  }
}

// Eight elements of a row as they are, and element e of them as fp32.
template <int DT>
struct Row8 {
  u32x4 w[DT == DA_F32 ? 2 : 1];
  __device__ __forceinline__ void clear() {
    w[0] = u32x4{0, 0, 0, 0};
    if constexpr (DT == DA_F32) w[1] = u32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    if constexpr (DT == DA_F32) {
      w[0] = *(const u32x4*)((const float*)p + at);
      w[1] = *(const u32x4*)((const float*)p + at + 4);
    } else {
      w[0] = *(const u32x4*)((const uint16_t*)p + at);
    }
  }
  __device__ __forceinline__ float get(int e) const {
    if constexpr (DT == DA_F32) return __uint_as_float(w[e >> 2][e & 3]);
    else return e & 1 ? E16<DT>::hi(w[0][e >> 1]) : E16<DT>::lo(w[0][e >> 1]);
  }
};

// Orders a wave's own LDS accesses (its tile is its own).
__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// Dim d of a query head: the weighted sum over the weights' sum, 0 where no key has a weight.
template <int DT>
__device__ __forceinline__ void store_out(const Attn4Args& a, int b, int hq, int d, float o, float L) {
  const float v = zero_bits(L) ? 0.0f : o / L;
  const int64_t at = b * a.so_b + hq * a.so_h + d;
  if constexpr (DT == DA_F32) ((float*)a.out)[at] = v;
  else ((uint16_t*)a.out)[at] = E16<DT>::bits(v);
}

// What a wave loads of 32 rows: lane (r, t) group t of rows r and 16 + r, and row lane % 32's count.
struct Tile4 {
  u32x4 kc[2], vc[2];
  uint32_t ks[2], vs[2];
  int count;
};

// One workgroup: (sequence, KV head) blockIdx.x, split blockIdx.y, heads 16 z .. of the group.
// MODE kParts: `nsplit` workgroups a head leave their partials; kScores: and the scores; kWhole: one
// workgroup of eight waves takes the head and writes the output itself; kWholeMass: and adds the weights,
// its scores in LDS.
enum Mode4 : int { kParts = 0, kScores = 1, kWhole = 2, kWholeMass = 3 };
constexpr int kWholeRows = 1024;  // most rows of a cache that kWhole and kWholeMass take (s_score holds as many)
template <int DT, int NG, int MODE>
__global__ __launch_bounds__(MODE >= kWhole ? 512 : 256, MODE >= kWhole || DT == DA_F32 ? 2 : 3) void kv4_attn_kernel(
    Attn4Args a) {
  constexpr bool WHOLE = MODE >= kWhole;
  constexpr int NW = WHOLE ? 8 : kA4Waves;
  constexpr int QP = DT == DA_BF16 ? 1 : DT == DA_F16 ? 2 : 3;
  constexpr int PP = DT == DA_F32 ? 3 : 2;
  constexpr int NJ = 2 * NG;  // output tiles of 16 dims
  constexpr int kTileBytes = kA4Tile * kA4VRow;
  constexpr int kRingRow = 128 + 4;  // floats of a ring row in LDS
  static_assert(16 * kRingRow * 4 <= kTileBytes, "16 ring rows must fit a wave's tile");
  __shared__ __attribute__((aligned(16))) char s_v[NW][kTileBytes];
  __shared__ __attribute__((aligned(16))) float s_bias[NW][kA4Tile];
  __shared__ float s_ml[NW][2][kA4Cols];
  __shared__ __attribute__((aligned(16))) float s_score[MODE == kWholeMass ? kWholeRows * kA4Cols : 4];
  __shared__ float s_weight[2][kA4Cols];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, t = lane >> 4;
  // The workgroups of a CU are a whole number of rounds apart, which without a turn of the heads
  // from split to split are splits of one head: a ragged batch's longest (16 caches of 3000 to 9000
  // rows: 33 us against 39).
  const int split = blockIdx.y, heads = gridDim.x;
  int bh = blockIdx.x + (int)((uint32_t)split * (uint32_t)heads / (uint32_t)a.nsplit);
  bh = bh >= heads ? bh - heads : bh;
  const int b = bh / a.Hkv, g = bh - b * a.Hkv;
  const int h0 = blockIdx.z * kA4Cols;
  const int cols = min(a.G - h0, kA4Cols);
  int n = a.lengths[bh];

  // ---- q in bf16 parts, the B operand: lane (head r, t), slot e of MFMA m: dim 32 t + 8 m + e
  const bool have = r < cols;
  u32x4 qf[QP][4];
  {
    const int64_t q_at = b * a.sq_b + (int64_t)(g * a.G + h0 + (have ? r : 0)) * a.sq_h;
    Row8<DT> x[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      x[m].clear();
      if (have && 32 * t + 8 * m < a.D) x[m].load(a.q, q_at + 32 * t + 8 * m);
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        uint32_t p[QP];
        split_pair<QP>(x[m].get(2 * w), x[m].get(2 * w + 1), p);
#pragma unroll
        for (int i = 0; i < QP; ++i) qf[i][m][w] = p[i];
      }
  }

  n = n < 0 ? 0 : (n > a.capacity ? (int)a.capacity : n);
  const int tiles = (n + kA4Tile - 1) / kA4Tile;
  const int rtiles = (a.exact_len + 15) / 16;
  // tiles of the rows: split s takes [s * per, (s + 1) * per); ring tiles go to the waves from
  // the last one on
  const int per = (tiles + a.nsplit - 1) / a.nsplit;
  const int t_begin = min(split * per, tiles), t_end = min(t_begin + per, tiles);
  const int nwave = a.nsplit * NW;
  const int rfirst = nwave - 1 - (split * NW + wid);
  const int64_t head_part = ((int64_t)bh * a.G + h0) * a.nsplit + split;  // of column 0; nsplit a column
  if (!WHOLE && t_begin >= t_end && nwave - 1 - (split * NW + NW - 1) >= rtiles) {  // nothing to do
    if (tid < cols) *(f32x2*)(void*)(a.stat + 2 * (head_part + (int64_t)tid * a.nsplit)) = f32x2{-INFINITY, 0.0f};
    return;
  }

  const bool grp = t < NG;
  const int tg = grp ? t : 0;
  const int64_t row0 = (int64_t)bh * a.capacity;
  const uint8_t* const kc0 = a.kc + row0 * NG * 16;
  const uint8_t* const vc0 = a.vc + row0 * NG * 16;
  const uint8_t* const ks0 = a.ks + row0 * NG;
  const uint8_t* const vs0 = a.vs + row0 * NG;
  const int32_t* const cnt0 = a.counts + row0;
  // rows past the length read the last one and carry no weight
  auto load_tile = [&](int tile, Tile4& x) {
    const int j0 = tile * kA4Tile;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const int64_t at = (int64_t)min(j0 + 16 * u + r, n - 1) * NG + tg;
      x.kc[u] = __builtin_nontemporal_load((const u32x4*)(kc0 + at * 16));
      x.vc[u] = __builtin_nontemporal_load((const u32x4*)(vc0 + at * 16));
      x.ks[u] = ks0[at];
      x.vs[u] = vs0[at];
    }
    x.count = cnt0[min(j0 + (lane & 31), n - 1)];
  };
  Tile4 cur;
  if (t_begin + wid < t_end) load_tile(t_begin + wid, cur);

  f32x4 acc[NJ];
#pragma unroll
  for (int j = 0; j < NJ; ++j) acc[j] = f32x4{0, 0, 0, 0};
  float m_run = -INFINITY, l_run = 0.0f;
  // a new maximum: what was summed shrinks by 2^(old - new).  Everything is in fp32 (and p's parts
  // keep their relative precision), so the maximum moves only where p would pass 2^16.
  auto raise = [&](float mx) {
    mx = cols_max(mx);
    if (__ballot(mx > m_run + 16.0f)) {
      const float m_new = __builtin_fmaxf(mx, m_run);
      const float f = is_neg_inf(m_run) ? 0.0f : exp2_hw(m_run - m_new);
      l_run *= f;
#pragma unroll
      for (int j = 0; j < NJ; ++j) acc[j] *= f;
      m_run = m_new;
    }
    return is_neg_inf(m_run) ? 0.0f : m_run;
  };
  char* const vt = s_v[wid];
  float* const bias = s_bias[wid];

  // ---- the ring, 16 slots at a time, in fp32: lane (r, t) loads dims 32 t + 8 m + e of slot r ----
  const int64_t x_at = b * a.sx_b + g * a.sx_h;
  for (int rt = rfirst; rt < rtiles; rt += nwave) {
    const int j0 = rt * 16;
    const bool slot = j0 + r < a.exact_len;
    const int64_t at = x_at + (int64_t)(slot ? j0 + r : 0) * a.sx_s + 32 * t;
    f32x4 s = f32x4{0, 0, 0, 0};
    Row8<DT> kx[4], vx[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      kx[m].clear();
      vx[m].clear();
      if (slot && 32 * t + 8 * m < a.D) {
        kx[m].load(a.kx, at + 8 * m);
        vx[m].load(a.vx, at + 8 * m);
      }
    }
    float* const rv = (float*)(void*)vt;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float qv = 0.0f;  // the parts' sum is q itself
#pragma unroll
        for (int i = QP - 1; i >= 0; --i) qv += (e & 1) ? bf16_hi(qf[i][m][e >> 1]) : bf16_lo(qf[i][m][e >> 1]);
        s = __builtin_amdgcn_mfma_f32_16x16x4f32(kx[m].get(e), qv, s, 0, 0, 0);
      }
      if (grp) {
        *(f32x4*)(rv + r * kRingRow + 32 * t + 8 * m) = f32x4{vx[m].get(0), vx[m].get(1), vx[m].get(2), vx[m].get(3)};
        *(f32x4*)(rv + r * kRingRow + 32 * t + 8 * m + 4) = f32x4{vx[m].get(4), vx[m].get(5), vx[m].get(6), vx[m].get(7)};
      }
    }
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = j0 + 4 * t + i < a.exact_len ? s[i] * a.scale_log2 : -INFINITY;
      mx = __builtin_fmaxf(mx, s[i]);
    }
    const float base = raise(mx);
    wave_lds_fence();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float p = exp2_hw(s[i] - base);
      l_run += p;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
        acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(rv[(4 * t + i) * kRingRow + 16 * j + r], p, acc[j], 0, 0, 0);
    }
    wave_lds_fence();
  }

  // ---- the rows, 32 at a time, the next tile's loads under this one's work ----
  // one tile's scores of all heads lie together: the heads' rows would be a power of two apart
  const int score_at = (have ? r : 0) * kA4Tile + 4 * t;
  float* const score = MODE == kScores ? a.score + (int64_t)bh * a.score_cap * a.G + h0 * kA4Tile + score_at : nullptr;
  for (int tile = t_begin + wid; tile < t_end; tile += NW) {
    const int j0 = tile * kA4Tile;
    Tile4 nxt;
    if (tile + NW < t_end) load_tile(tile + NW, nxt);
    // log2(count), or -inf for a row without weight, once a row
    if (lane < kA4Tile)
      bias[lane] = cur.count > 0 && j0 + lane < n ? __builtin_amdgcn_logf((float)cur.count) : -INFINITY;
    wave_lds_fence();
    f32x4 s[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      // a row without weight as good as zeros (its codes times 2^-127), whatever it holds: its score
      // is then finite, its weight 0
      const bool live = !is_neg_inf(bias[16 * u + r]);
      const float ksc = __uint_as_float(live ? cur.ks[u] << 23 : 0u), vsc = __uint_as_float(live ? cur.vs[u] << 23 : 0u);
      s[u] = f32x4{0, 0, 0, 0};
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        u32x4 kf = fp4_to_bf16x8(cur.kc[u][m], ksc);
        if (NG < 4 && !grp) kf = u32x4{0, 0, 0, 0};
#pragma unroll
        for (int i = QP - 1; i >= 0; --i) s[u] = mfma16(kf, qf[i][m], s[u]);
        // V to LDS as bf16
        const u32x4 v = fp4_to_bf16x8(cur.vc[u][m], vsc);
        if (grp) *(u32x4*)(vt + (16 * u + r) * kA4VRow + 64 * t + 16 * m) = v;
      }
    }
    // ---- softmax: lane (head r), keys 4 t + i of both halves ----
    float mx = -INFINITY;
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4 add = *(const f32x4*)(bias + 16 * u + 4 * t);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[u][i] = __builtin_fmaf(s[u][i], a.scale_log2, add[i]);
        mx = __builtin_fmaxf(mx, s[u][i]);
      }
    }
    if (have) {
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (MODE == kScores) *(f32x4*)(score + (int64_t)j0 * a.G + 16 * u) = s[u];
        if (MODE == kWholeMass) *(f32x4*)(s_score + j0 * cols + score_at + 16 * u) = s[u];
      }
    }
    const float base = raise(mx);
    u32x4 pf[PP];
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float p0 = exp2_hw(s[u][2 * w] - base), p1 = exp2_hw(s[u][2 * w + 1] - base);
        l_run += p0 + p1;
        uint32_t p[PP];
        split_pair<PP>(p0, p1, p);
#pragma unroll
        for (int i = 0; i < PP; ++i) pf[i][2 * u + w] = p[i];
      }
    // ---- O^T += V^T P^T ----
    wave_lds_fence();
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      // in each group of 16 lanes, lane i receives element i % 4 of the 8 bytes that lanes
      // 4 e + i / 4 address, e = 0 .. 3: dim 16 j + i of keys 4 t + e
      typedef __attribute__((address_space(3))) i16x4v lds4;
      char* const at = vt + (4 * t + (r >> 2)) * kA4VRow + 32 * j + 8 * (r & 3);
      const i16x4v v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(uint32_t)(uintptr_t)(
          const __attribute__((address_space(3))) char*)at);
      const i16x4v v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(uintptr_t)(uint32_t)(uintptr_t)(
          const __attribute__((address_space(3))) char*)(at + 16 * kA4VRow));
      const u32x2 w0 = __builtin_bit_cast(u32x2, v0), w1 = __builtin_bit_cast(u32x2, v1);
      const u32x4 vf = u32x4{w0[0], w0[1], w1[0], w1[1]};
#pragma unroll
      for (int i = PP - 1; i >= 0; --i) acc[j] = mfma16(vf, pf[i], acc[j]);
    }
    wave_lds_fence();
    cur = nxt;
  }

  // ---- join the workgroup's waves; the V tiles' LDS holds their sums ----
  l_run = cols_sum(l_run);
  if (t == 0) {
    s_ml[wid][0][r] = m_run;
    s_ml[wid][1][r] = l_run;
  }
  float* const so = (float*)(void*)vt;  // [16 heads][16 NJ + 4] of this wave
  constexpr int kRow = 16 * NJ + 4;
  static_assert(kA4Cols * kRow * 4 <= kTileBytes, "a wave's sums must fit its tile");
#pragma unroll
  for (int j = 0; j < NJ; ++j) *(f32x4*)(so + r * kRow + 16 * j + 4 * t) = acc[j];
  __syncthreads();
  for (int i = tid; i < cols * 16 * NJ; i += 64 * NW) {
    const int c = i / (16 * NJ), d = i - c * (16 * NJ);
    float M = s_ml[0][0][c];
#pragma unroll
    for (int w = 1; w < NW; ++w) M = __builtin_fmaxf(M, s_ml[w][0][c]);
    const float base = M == -INFINITY ? 0.0f : M;
    float o = 0.0f, L = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = exp2_hw(s_ml[w][0][c] - base);
      o += f * ((const float*)(const void*)s_v[w])[c * kRow + d];
      L += f * s_ml[w][1][c];
    }
    if (WHOLE) {
      if (MODE == kWholeMass && d == 0) {
        s_weight[0][c] = base;
        s_weight[1][c] = zero_bits(L) ? 0.0f : 1.0f / L;
      }
      if (d < a.D) store_out<DT>(a, b, g * a.G + h0 + c, d, o, L);
    } else {
      const int64_t to = head_part + (int64_t)c * a.nsplit;
      a.part[to * kA4Part + d] = o;
      if (d == 0) *(f32x2*)(void*)(a.stat + 2 * to) = f32x2{M, L};
    }
  }
  if (MODE == kWholeMass) {
    __syncthreads();
    for (int j = tid; j < n; j += 64 * NW) {
      const float* const at = s_score + (j & -kA4Tile) * cols + (j & (kA4Tile - 1));
      float w = 0.0f;
      for (int c = 0; c < cols; ++c) w += exp2_hw(at[c * kA4Tile] - s_weight[0][c]) * s_weight[1][c];
      a.mass[row0 + j] += w;
    }
  }
}

// Blocks [0, B Hq): one query head's splits joined, 32 lanes of four dims each, eight splits at a
// time with four in flight.  Blocks from there on add the weights: kMassKeys keys of one
// (sequence, KV head) each, after the group's maxima and sums over the splits.
constexpr int kMassKeys = 1024;
// (max, sum) of a query head over the splits, by one wave
__device__ __forceinline__ void join_stats(const float* stat, int nsplit, int lane, float& m, float& l) {
  m = -INFINITY;
  l = 0.0f;
  for (int s = lane; s < nsplit; s += 64) {
    const f32x2 v = *(const f32x2*)(const void*)(stat + 2 * s);
    const float mm = __builtin_fmaxf(m, v[0]), base = is_neg_inf(mm) ? 0.0f : mm;
    l = l * exp2_hw(m - base) + v[1] * exp2_hw(v[0] - base);
    m = mm;
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const float m2 = __shfl_xor(m, d, 64), l2 = __shfl_xor(l, d, 64);
    const float mm = __builtin_fmaxf(m, m2), base = is_neg_inf(mm) ? 0.0f : mm;
    l = l * exp2_hw(m - base) + l2 * exp2_hw(m2 - base);
    m = mm;
  }
}
template <int DT, bool MASS>
__global__ __launch_bounds__(256) void kv4_join_kernel(Attn4Args a) {
  __shared__ float s_m[64], s_l[64];
  __shared__ __attribute__((aligned(16))) f32x4 s_o[8][32];
  const int Hq = a.Hkv * a.G;
  const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
  const int heads = a.B * Hq;
  if (!MASS || (int)blockIdx.x < heads) {
    const int bhq = blockIdx.x, b = bhq / Hq, hq = bhq - b * Hq;
    const float* part = a.part + (int64_t)bhq * a.nsplit * kA4Part;
    const float* stat = a.stat + (int64_t)bhq * a.nsplit * 2;
    const int c = tid & 31, sg = tid >> 5;  // dims 4 c .. 4 c + 3, splits sg, sg + 8, ...
    const int cd = 4 * c < a.D ? 4 * c : 0;
    f32x4 v[4];
    float ms[4];
    auto load = [&](int s0) {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int s = min(s0 + 8 * u, a.nsplit - 1);
        ms[u] = s0 + 8 * u < a.nsplit ? stat[2 * s] : -INFINITY;
        v[u] = *(const f32x4*)(part + (int64_t)s * kA4Part + cd);
      }
    };
    load(sg);
    float M, L;
    join_stats(stat, a.nsplit, lane, M, L);
    const float base = is_neg_inf(M) ? 0.0f : M;
    f32x4 o = f32x4{0, 0, 0, 0};
    for (int s0 = sg; s0 < a.nsplit; s0 += 32) {
      if (s0 != sg) load(s0);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (!is_neg_inf(ms[u])) o += v[u] * exp2_hw(ms[u] - base);  // an empty split wrote no sums
    }
    s_o[sg][c] = o;
    __syncthreads();
    if (tid < a.D) {
      float w = 0.0f;
#pragma unroll
      for (int s = 0; s < 8; ++s) w += ((const float*)(const void*)s_o[s])[tid];
      store_out<DT>(a, b, hq, tid, w, L);
    }
    return;
  }
  if constexpr (MASS) {
    const int chunks = (int)((a.capacity + kMassKeys - 1) / kMassKeys);
    const int id = blockIdx.x - heads, bh = id / chunks, chunk = id - bh * chunks;
    int n = a.lengths[bh];
    n = n < 0 ? 0 : (n > a.capacity ? (int)a.capacity : n);
    const int first = chunk * kMassKeys;
    if (first >= n) return;
    for (int h = wid; h < a.G; h += 4) {
      float m, l;
      join_stats(a.stat + ((int64_t)bh * a.G + h) * a.nsplit * 2, a.nsplit, lane, m, l);
      if (lane == 0) {
        s_m[h] = is_neg_inf(m) ? 0.0f : m;
        s_l[h] = zero_bits(l) ? 0.0f : 1.0f / l;
      }
    }
    __syncthreads();
    // four keys a thread; the scores are padded to whole tiles
    const int j = first + 4 * tid;
    if (j >= n) return;
    const float* score = a.score + ((int64_t)bh * a.score_cap + (j & -kA4Tile)) * a.G + (j & (kA4Tile - 1));
    float* const mass = a.mass + (int64_t)bh * a.capacity + j;
    f32x4 w = f32x4{0, 0, 0, 0};
    for (int h = 0; h < a.G; ++h) {
      const f32x4 s = *(const f32x4*)(score + h * kA4Tile);
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] += exp2_hw(s[i] - s_m[h]) * s_l[h];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (j + i < n) mass[i] += w[i];
  }
}

// Workgroups of the attention launch: three a CU run at once (the registers of the 16-bit types' kernels:
// 124 to 171 VGPRs; fp32's 192 to 216 leave room for two, and the number was not measured for it apart),
// and no split is shorter than a tile a wave.  64 splits, or of 512 rows as many as there are up to 256, are the most
// that pay their joining (8 heads of 8297 rows: 64 10.2 us, 32 11.8, 96 12.7; one of 112207: 64 19.2,
// 128 15.1, 256 15.7; one of 1000000: 64 109, 128 61, 256 43).  A short cache is one workgroup of
// eight waves a head, without a second launch (8 heads, 500 rows: 8.1 against 9.2 us, 750: 9.7 / 9.3,
// 1000: 10.9 / 9.2; a launch is 3.4 us of the caller's time as well); 256 heads fill the chip like that
// (1000 rows: 15.4 / 20.0).
static int kv4_splits(int64_t B, int64_t Hkv, int64_t G, int64_t capacity) {
  const int64_t units = B * Hkv * ((G + kA4Cols - 1) / kA4Cols);
  if (capacity <= (units >= 256 ? kWholeRows : 768)) return 1;
  const int64_t most = (capacity + kA4Tile * kA4Waves - 1) / (kA4Tile * kA4Waves);
  int64_t want = (768 + units - 1) / units;
  const int64_t pay = capacity / 512 < 64 ? 64 : capacity / 512 > 256 ? 256 : capacity / 512;
  if (want > pay) want = pay;
  if (want > most) want = most;
  return (int)want;
}
// One launch for it all: a short cache; where weights are added, one workgroup has to see all heads of
// the group (8 heads of 60 rows with weights: 6.7 us against 10.0, 750 rows: 10.9 / 14.6; 512 heads of
// 750: 25.7 / 25.3).  768 heads and more leave one split at any capacity, which does not make the cache
// short: past kWholeRows it takes the two launches, with which it is as fast or faster too (768 heads of
// 2048 rows without weights: 50 us against 56 in one, of 4096 78 / 86, 2048 heads of 8192 339 / 365).
static bool kv4_whole(int nsplit, int64_t G, int64_t capacity, bool mass) {
  return nsplit == 1 && capacity <= kWholeRows && (!mass || G <= kA4Cols);
}
static int64_t kv4_score_cap(int64_t capacity) { return (capacity + kA4Tile - 1) / kA4Tile * kA4Tile; }

template <int DT, int NG>
static void launch_attn4_ng(const Attn4Args& a, dim3 grid, int mode, hipStream_t st) {
  if (mode == kWhole) hipLaunchKernelGGL((kv4_attn_kernel<DT, NG, kWhole>), grid, dim3(512), 0, st, a);
  else if (mode == kWholeMass) hipLaunchKernelGGL((kv4_attn_kernel<DT, NG, kWholeMass>), grid, dim3(512), 0, st, a);
  else if (mode == kScores) hipLaunchKernelGGL((kv4_attn_kernel<DT, NG, kScores>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((kv4_attn_kernel<DT, NG, kParts>), grid, dim3(256), 0, st, a);
}
template <int DT>
static int launch_attn4(const Attn4Args& a, bool mass, hipStream_t st, const char* who) {
  const dim3 grid((unsigned)(a.B * a.Hkv), (unsigned)a.nsplit, (unsigned)((a.G + kA4Cols - 1) / kA4Cols));
  const int mode = kv4_whole(a.nsplit, a.G, a.capacity, mass) ? (mass ? kWholeMass : kWhole) : mass ? kScores : kParts;
  switch ((a.D + 31) / 32) {
    case 1: launch_attn4_ng<DT, 1>(a, grid, mode, st); break;
    case 2: launch_attn4_ng<DT, 2>(a, grid, mode, st); break;
    case 3: launch_attn4_ng<DT, 3>(a, grid, mode, st); break;
    default: launch_attn4_ng<DT, 4>(a, grid, mode, st); break;
  }
  if (mode >= kWhole) return check_launch(who);
  const unsigned heads = (unsigned)(a.B * a.Hkv * a.G);
  if (mass) {
    const unsigned chunks = (unsigned)((a.capacity + kMassKeys - 1) / kMassKeys);
    hipLaunchKernelGGL((kv4_join_kernel<DT, true>), dim3(heads + (unsigned)(a.B * a.Hkv) * chunks), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL((kv4_join_kernel<DT, false>), dim3(heads), dim3(256), 0, st, a);
  }
  return check_launch(who);
}

}  // namespace da

using namespace da;

// The splits' P.V and statistics, then (accumulate) the scores.
static int64_t kv4_stat_floats(int64_t n) { return (2 * n + 3) / 4 * 4; }
extern "C" int64_t da_kv4_attention_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t capacity,
                                                   int accumulate) {
  if (B <= 0 || Hkv <= 0 || Hq <= 0 || capacity <= 0) return 0;
  const int splits = kv4_splits(B, Hkv, Hq / Hkv, capacity);
  if (kv4_whole(splits, Hq / Hkv, capacity, accumulate != 0)) return 0;
  const int64_t n = B * Hq * splits;
  const int64_t scores = accumulate ? B * Hq * kv4_score_cap(capacity) : 0;
  return (n * kA4Part + kv4_stat_floats(n) + scores) * (int64_t)sizeof(float);
}

extern "C" int da_kv4_attention(const void* q, int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t sq_b,
                                int64_t sq_h, const DaKv4* kv, const void* k_exact, const void* v_exact, int64_t sx_b,
                                int64_t sx_h, int64_t sx_s, int64_t exact_len, float scale, int accumulate, void* out,
                                int64_t so_b, int64_t so_h, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "da_kv4_attention";
  DA_REQUIRE(kv && q && out, "%s: null pointer", who);
  DA_REQUIRE(kv->k_codes && kv->k_scales && kv->v_codes && kv->v_scales && kv->counts && kv->lengths &&
                 (!accumulate || kv->mass),
             "%s: null pointer in the cache", who);
  if (dtype != DA_BF16 && dtype != DA_F16 && dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: q must be bf16, fp16 or fp32", who);
  if (D <= 0 || D > 128 || (D & 7))
    return set_error(DA_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 in [8, 128]", who);
  DA_REQUIRE(B > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0, "%s: bad head counts", who);
  if (Hq / Hkv > 64) return set_error(DA_ERR_UNSUPPORTED, "%s: GQA group above 64", who);
  DA_REQUIRE(kv->capacity > 0 && exact_len >= 0 && exact_len < (1 << 24), "%s: bad cache lengths", who);
  if (kv->capacity > (1 << 24)) return set_error(DA_ERR_UNSUPPORTED, "%s: capacity above 2^24 rows", who);
  DA_REQUIRE(exact_len == 0 || (k_exact && v_exact), "%s: null ring", who);
  const int64_t align = dtype == DA_F32 ? 3 : 7;
  // a dimension of one has no stride
  const int64_t strides = (B > 1 ? sq_b | sx_b : 0) | (Hq > 1 ? sq_h : 0) | (Hkv > 1 ? sx_h : 0) | (exact_len > 1 ? sx_s : 0);
  DA_REQUIRE((strides & align) == 0 && ((uintptr_t)q & 15) == 0 &&
                 (exact_len == 0 || (((uintptr_t)k_exact | (uintptr_t)v_exact) & 15) == 0),
             "%s: q and ring rows must be 16-byte aligned", who);
  DA_REQUIRE((((uintptr_t)kv->k_codes | (uintptr_t)kv->v_codes) & 15) == 0, "%s: codes must be 16-byte aligned", who);
  DA_REQUIRE(scale > 0.0f, "%s: scale must be positive", who);
  const int64_t need = da_kv4_attention_workspace_size(B, Hq, Hkv, kv->capacity, accumulate);
  if (need > 0 && (!workspace || workspace_bytes < need))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %lld bytes required", who, (long long)need);
  DA_REQUIRE(((uintptr_t)workspace & 15) == 0, "%s: workspace must be 16-byte aligned", who);
  Attn4Args a = {};
  a.q = q; a.sq_b = sq_b; a.sq_h = sq_h;
  a.kc = kv->k_codes; a.ks = kv->k_scales; a.vc = kv->v_codes; a.vs = kv->v_scales;
  a.counts = kv->counts; a.lengths = kv->lengths; a.capacity = kv->capacity;
  a.kx = k_exact; a.vx = v_exact; a.sx_b = sx_b; a.sx_h = sx_h; a.sx_s = sx_s; a.exact_len = (int)exact_len;
  a.scale_log2 = scale * kLog2e;
  a.out = out; a.so_b = so_b; a.so_h = so_h; a.mass = kv->mass;
  a.B = (int)B; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.D = (int)D;
  a.nsplit = kv4_splits(B, Hkv, a.G, kv->capacity);
  a.part = (float*)workspace;
  a.score_cap = kv4_score_cap(kv->capacity);
  const int64_t n = B * Hq * a.nsplit;
  a.stat = a.part + n * kA4Part;
  a.score = a.stat + kv4_stat_floats(n);
  const unsigned long long blocks = (unsigned long long)(B * Hq) + (unsigned long long)(B * Hkv) * ((kv->capacity + kMassKeys - 1) / kMassKeys);
  // a launch holds fewer than 2^32 threads
  if (B * Hkv >= (1 << 20) || blocks >= (1ull << 24)) return set_error(DA_ERR_UNSUPPORTED, "%s: too many heads and rows for one call", who);
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DA_F32) return launch_attn4<DA_F32>(a, accumulate != 0, st, who);
  if (dtype == DA_F16) return launch_attn4<DA_F16>(a, accumulate != 0, st, who);
  return launch_attn4<DA_BF16>(a, accumulate != 0, st, who);
}
