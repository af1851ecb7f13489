// The attention weight every key receives from a run of queries, on gfx950.
//
// mass_j = sum over the queries (i, h) of a KV head's group of c_j 2^(s_ij - lse_i), with
// s_ij = scale log2(e) q_i . k_j and lse_i = log2 sum_j c_j 2^(s_ij) over the keys that query
// sees.  The weights need the whole row's sum before the first of them is known, and storing
// the scores (4 bytes for 256 flops) costs more than computing them twice, so there are two
// passes over the score matrix on MFMA:
//
//   rows     S^T = K Q^T, queries as columns: running maximum and sum in the lane that owns the
//            query (16 of a tile's 32 keys a lane), no exchange until the end;
//   columns  S = Q K^T, keys as columns: sum of 2^(s - lse) over the queries, in the lane that
//            owns the key.
//
// They are one kernel with the operands swapped: a wave holds its columns' operand (64 columns of a
// 16-bit type, 32 of fp32) in registers for the whole run and the rows stream through LDS in
// double-buffered stages of 64 (fp32: 32) that the four waves of a workgroup share, worked on 32 rows
// at a time, so that each fragment read from LDS feeds two MFMAs.  Per score there is
// one fused multiply-add, one exp2 and one addition; the maximum is looked at only where a sum
// leaves fp32's comfortable range.  Queries of a group are interleaved (row = query G + head),
// so a tile's positions are close together and whole tiles are either visible or not.
//
// Both passes split their streamed axis where there are too few columns to fill the chip; the
// parts are joined by small launches in a fixed order.  Up to 128 query rows and keys a head, both
// passes are one launch of one workgroup a head.
//
// What bounds it: 8192 queries of 8 x 4 heads (305 + 333 us) keep the matrix unit busy for 40 and 36% of
// the cycles and the VALU for 62 and 53%.  Neither is full, and the sums are near all of it: at 246 to
// 254 VGPRs two waves a SIMD are what fits, and the two units take turns more than they overlap.
//
// fp32 tensors: each operand is cut into three bf16 parts, and the six products of weight
// 2^-16 and above are kept (error about 2^-24 of |q||k|, as an fp32 product's own rounding).
#include "da_common.hpp"
#include "../../include/deltaattn_cache.h"

namespace da {

constexpr int kMRow = 256;             // bytes of a row in LDS (128 16-bit dims)
constexpr float kMLog2e = 1.4426950408889634f;
constexpr float kMLarge = 1.2676506e30f;  // 2^100: a tile's sum above it moves the maximum
constexpr int kNever = 0x7fffffff;        // a time after every query's, and (negated) before every key's

struct MassArgs {
  const void* q;
  const void* k;
  int64_t sq_b, sq_h, sq_n, sk_b, sk_h, sk_n;
  const int32_t* counts;
  const int32_t* ts;
  const int32_t* lengths;
  int64_t q_start;
  float scale_log2;
  float* part;   // rows pass: [bh][R][split] (max, sum); columns pass: [split][bh][Nk] sums
  float* stats;  // [bh][R] (-max, 1 / sum); (-inf, 0) where a query sees nothing
  float* mass;
  int B, Hkv, G, gshift, Nq, Nk, D;  // gshift: log2 G, or -1
  int split, blocks;  // of the pass
};

__device__ __forceinline__ float mexp2(float x) { return __builtin_amdgcn_exp2f(x); }

// The position of query i, between the two values of kNever.
__device__ __forceinline__ int mass_pos(const MassArgs& a, int i) {
  const int64_t p = a.q_start + i;
  return p <= -kNever ? -kNever + 1 : (p >= kNever ? kNever - 1 : (int)p);
}
__device__ __forceinline__ int query_of(const MassArgs& a, int row) {
  return a.gshift >= 0 ? row >> a.gshift : row / a.G;
}

// Eight fp32 elements as NP bf16 operands of eight, largest part first.
template <int NP>
__device__ __forceinline__ void cut_chunk(f32x4 x0, f32x4 x1, u32x4 (&w)[NP]) {
  float x[8] = {x0[0], x0[1], x0[2], x0[3], x1[0], x1[1], x1[2], x1[3]};
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint16_t lo = E16<DA_BF16>::bits(x[2 * i]), hi = E16<DA_BF16>::bits(x[2 * i + 1]);
      x[2 * i] -= E16<DA_BF16>::one(lo);
      x[2 * i + 1] -= E16<DA_BF16>::one(hi);
      w[p][i] = lo | ((uint32_t)hi << 16);
    }
}

// Scheduling of a 32-row step: the product's eight fragments and 16 MFMAs among the exponentials of
// the rows before (8K prompt 697 us without, 675 with; 32K window 70 / 64).
__device__ __forceinline__ void interleave() {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);   // a read of LDS
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);   // two MFMAs
    __builtin_amdgcn_sched_group_barrier(0x402, 12, 0);  // VALU and transcendental
  }
}

// What the columns pass needs of a query: its weights are 2^(s - max) / sum.  The maximum is kept
// apart from the sum (not as one logarithm): s - max is small where the weight is large, so it
// rounds finely there.
__device__ __forceinline__ f32x2 row_stats(float M, float L) {
  return zero_bits(L) ? f32x2{-INFINITY, 0.0f} : f32x2{-M, 1.0f / L};
}

// PASS 0: rows (stream keys, columns are queries); PASS 1: columns (stream queries, columns are
// keys).  The grid runs over (sequence, KV head), then the splits, then the column blocks, the
// longest first; neighbours go to different XCDs, so one head's K and Q stay in few of their
// caches.
// KK: k steps of 16 dims a score takes (2, 4, 6 or 8: the steps are not left to a run-time bound,
// which costs a copy of the accumulators each).
template <int DT, int PASS, int KK>
__device__ __forceinline__ void mass_pass(const MassArgs& a) {
  constexpr int NP = DT == DA_F32 ? 3 : 1;
  constexpr int NW = DT == DA_F32 ? 2 : 1;    // 16-byte loads of a chunk of 8 elements
  constexpr int NCB = DT == DA_F32 ? 1 : 2;   // column blocks of 32 a wave holds
  constexpr int kTile = DT == DA_F32 ? 32 : 64;  // streamed rows a stage
  constexpr int NU = kTile / 16;              // rows a thread stages
  constexpr int MT = DT == DA_F32 ? DA_BF16 : DT;
  constexpr int kCols = 4 * NCB * 32;
  constexpr int kPart = kTile * kMRow;        // LDS bytes of one part of a stage
  __shared__ __attribute__((aligned(16))) char s_y[2][NP * kPart];
  // per row: PASS 0 log2(count); PASS 1 -max and 1 / sum
  // (three stages of them: a wave may still be at a tile's last half when others store two tiles on)
  __shared__ __attribute__((aligned(16))) float s_add[3][kTile];
  __shared__ __attribute__((aligned(16))) float s_mul[3][PASS == 1 ? kTile : 4];
  __shared__ __attribute__((aligned(16))) int s_t[3][kTile];
  __shared__ int s_flag[3], s_ext[4];
  const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cl = lane & 31, hl = lane >> 5;
  const int nbh = a.B * a.Hkv, id = blockIdx.x / nbh;
  const int bh = blockIdx.x - id * nbh, b = bh / a.Hkv, g = bh - b * a.Hkv;
  const int zb = id / a.split, part_id = id - zb * a.split;
  const int G = a.G;
  const int R = G * a.Nq;
  int n = a.lengths ? a.lengths[bh] : a.Nk;
  n = n < 0 ? 0 : (n > a.Nk ? a.Nk : n);
  const int ncol = PASS == 0 ? R : n;
  // rows pass: later queries see more keys; columns pass: earlier keys are seen by more queries
  const int block = PASS == 0 ? a.blocks - 1 - zb : zb;
  const int c0 = block * kCols;
  constexpr int es = DT == DA_F32 ? 4 : 2;
  const char* const qb = (const char*)a.q + (b * a.sq_b + (int64_t)g * G * a.sq_h) * es;
  const char* const kb = (const char*)a.k + (b * a.sk_b + g * a.sk_h) * es;
  const int32_t* const cnt = a.counts ? a.counts + (int64_t)bh * a.Nk : nullptr;
  const int32_t* const ts = a.ts ? a.ts + (int64_t)bh * a.Nk : nullptr;
  f32x2* const stats = (f32x2*)(void*)a.stats + (int64_t)bh * R;

  // ---- this workgroup's share of the streamed rows, in tiles ----
  const int c_last = min(c0 + kCols, ncol) - 1;  // below c0 where there is no column
  const int nrow = PASS == 0 ? n : R;
  int row_lo = 0, row_hi = nrow;
  if (!ts && c_last >= c0) {
    if (PASS == 0) {  // keys up to the last query's own place
      const int p = mass_pos(a, query_of(a, c_last));
      row_hi = p < row_hi ? p + 1 : row_hi;
    } else {  // from the first query that sees key c0
      const int64_t first = (int64_t)c0 - a.q_start;
      row_lo = first <= 0 ? 0 : (first >= a.Nq ? R : (int)first * G);
    }
  }
  const int tile_lo = row_lo / kTile, tile_hi = (row_hi + kTile - 1) / kTile;
  const int ntile = c_last >= c0 && tile_hi > tile_lo ? tile_hi - tile_lo : 0;
  const int per = (ntile + a.split - 1) / a.split;
  const int t_begin = tile_lo + min(part_id * per, ntile);
  const int t_end = min(t_begin + per, tile_lo + ntile);

  // ---- staging: 16 chunks of 8 elements a row, thread: rows tid / 16 + 16 u, chunk tid % 16 ----
  // Where a stage's rows are at a fixed distance from the last one's (keys; queries of a group
  // that divides a stage) the addresses are stepped, else formed again.  The waves take turns with
  // the rows' times and weights.
  const int sr = tid >> 4, sc = tid & 15;
  const bool chunk = 8 * sc < a.D;  // chunks past the head dimension stay zero
  const bool stepped = PASS == 0 || (a.gshift >= 0 && kTile >> a.gshift != 0);
  const int64_t step = (PASS == 0 ? kTile * a.sk_n : (int64_t)(kTile >> (a.gshift >= 0 ? a.gshift : 0)) * a.sq_n) * es;
  auto row_src = [&](int row) {
    if (PASS == 0) return kb + row * a.sk_n * es;
    const int i = query_of(a, row), h = row - i * G;
    return qb + (h * a.sq_h + i * a.sq_n) * es;
  };
  const char* src[NU];
#pragma unroll
  for (int u = 0; u < NU; ++u) src[u] = row_src(t_begin * kTile + sr + 16 * u) + 8 * es * sc;
  u32x4 y[NU][NW];
  float m_add = 0.0f, m_mul = 0.0f;
  int m_t = 0;
  auto load_tile = [&](int tile) {
    const int row0 = tile * kTile + sr;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
      if (!stepped) src[u] = row_src(row0 + 16 * u) + 8 * es * sc;
#pragma unroll
      for (int w = 0; w < NW; ++w) y[u][w] = u32x4{0, 0, 0, 0};
      if (chunk && row0 + 16 * u < nrow) {
#pragma unroll
        for (int w = 0; w < NW; ++w) y[u][w] = *(const u32x4*)(src[u] + 16 * w);
      }
      src[u] += step;
    }
    if (wid == (tile & 3) && lane < kTile) {
      const int row = tile * kTile + lane;
      m_add = -INFINITY;
      m_mul = 0.0f;
      m_t = -kNever;  // past the end: no weight; as a query it is masked, a key may be anything
      if (row < nrow) {
        if (PASS == 0) {
          const int c = cnt ? cnt[row] : 1;
          m_add = c <= 0 ? -INFINITY : (cnt ? __builtin_amdgcn_logf((float)c) : 0.0f);
          m_t = c <= 0 ? kNever : (ts ? ts[row] : row);  // hidden keys: masked, whatever they hold
        } else {
          const f32x2 st = stats[row];
          m_add = st[0];
          m_mul = st[1];
          // queries that see nothing: masked, whatever they hold
          m_t = is_neg_inf(m_add) ? -kNever : mass_pos(a, query_of(a, row));
        }
      }
    }
  };
  // An extreme time of the columns, to decide for whole tiles: rows pass, the earliest query (keys
  // at or before it need no mask); columns pass, the latest key.
  int ext = PASS == 0 ? mass_pos(a, query_of(a, c0)) : c_last;
  auto store_tile = [&](int st, int mt, int tile) {
    char* const at0 = s_y[st] + sr * kMRow + ((sc ^ sr) << 4);  // row % 16 is sr
    if (chunk) {
#pragma unroll
      for (int u = 0; u < NU; ++u) {
        char* const at = at0 + 16 * u * kMRow;
        if constexpr (DT == DA_F32) {
          u32x4 w[NP];
          cut_chunk<NP>(__builtin_bit_cast(f32x4, y[u][0]), __builtin_bit_cast(f32x4, y[u][1]), w);
#pragma unroll
          for (int p = 0; p < NP; ++p) *(u32x4*)(at + p * kPart) = w[p];
        } else {
          *(u32x4*)at = y[u][0];
        }
      }
    }
    if (wid == (tile & 3)) {
      // bit 0 (rows pass): a key has a weight other than 1; bit 1: a row that some column may not see
      const bool mine = lane < kTile;
      if (mine) {
        s_add[mt][lane] = m_add;
        if (PASS == 1) s_mul[mt][lane] = m_mul;
        s_t[mt][lane] = m_t;
      }
      const uint64_t odd = __ballot(mine && !zero_bits(m_add));
      // queries past the end ask for no mask, but where there is one they are behind it: a key that no
      // query sees may hold a NaN, whose product with a row of zeros is one
      const uint64_t late = __ballot(mine && (PASS == 0 ? m_t > ext : m_t < ext && tile * kTile + lane < nrow));
      if (lane == 0) s_flag[mt] = (odd ? 1 : 0) | (late ? 2 : 0);
    }
  };
  if (!chunk) {
#pragma unroll
    for (int i = 0; i < 2 * NP * NU; ++i)
      *(u32x4*)(&s_y[0][0] + (16 * i + sr) * kMRow + ((sc ^ sr) << 4)) = u32x4{0, 0, 0, 0};
  }
  if (t_begin < t_end) load_tile(t_begin);

  // ---- the columns' operand and times ----
  u32x4 x[NP][NCB][KK];
  int ct[NCB];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    const int c = c0 + (wid * NCB + cb) * 32 + cl;
    const bool have = c < ncol;
    const char* src = kb;
    ct[cb] = PASS == 0 ? kNever - 1 : -kNever + 1;
    if (have) {
      if (PASS == 0) {
        const int i = query_of(a, c), h = c - i * G;
        src = qb + (h * a.sq_h + i * a.sq_n) * es;
        ct[cb] = mass_pos(a, i);
      } else {
        src = kb + c * a.sk_n * es;
        ct[cb] = ts ? ts[c] : c;
      }
    }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const int d = 16 * kk + 8 * hl;
#pragma unroll
      for (int p = 0; p < NP; ++p) x[p][cb][kk] = u32x4{0, 0, 0, 0};
      if (have && d < a.D) {
        if constexpr (DT == DA_F32) {
          u32x4 w[NP];
          cut_chunk<NP>(*(const f32x4*)(src + 4 * d), *(const f32x4*)(src + 4 * d + 16), w);
#pragma unroll
          for (int p = 0; p < NP; ++p) x[p][cb][kk] = w[p];
        } else {
          x[0][cb][kk] = *(const u32x4*)(src + 2 * d);
        }
      }
    }
  }
  if (PASS == 1 && ts) {
    int e = -kNever + 1;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) e = max(e, ct[cb]);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) e = max(e, __shfl_xor(e, d, 64));
    if (lane == 0) s_ext[wid] = e;
    __syncthreads();
    ext = max(max(s_ext[0], s_ext[1]), max(s_ext[2], s_ext[3]));
  }

  float m_run[NCB], sum[NCB];
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    m_run[cb] = -INFINITY;
    sum[cb] = 0.0f;
  }
  const float c2 = a.scale_log2;

  // scores of 32 rows: rows half * 32 .. of stage st against the wave's columns
  auto product = [&](int st, int half, f32x16 (&s)[NCB]) {
    const char* const yb = s_y[st] + (32 * half + cl) * kMRow;
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[cb][r] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      u32x4 f[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) f[p] = *(const u32x4*)(yb + p * kPart + (((2 * kk + hl) ^ (cl & 15)) << 4));
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        if constexpr (NP == 1) {
          s[cb] = E16<MT>::mfma(f[0], x[0][cb][kk], s[cb]);
        } else {  // the smallest products first
          s[cb] = E16<MT>::mfma(f[0], x[2][cb][kk], s[cb]);
          s[cb] = E16<MT>::mfma(f[2], x[0][cb][kk], s[cb]);
          s[cb] = E16<MT>::mfma(f[1], x[1][cb][kk], s[cb]);
          s[cb] = E16<MT>::mfma(f[0], x[1][cb][kk], s[cb]);
          s[cb] = E16<MT>::mfma(f[1], x[0][cb][kk], s[cb]);
          s[cb] = E16<MT>::mfma(f[0], x[0][cb][kk], s[cb]);
        }
      }
    }
  };
  // The exponentials of 32 rows' scores into the columns' sums, `next` (the following rows' product,
  // if any) issued first: one MFMA to every few of these instructions, so that the matrix unit works
  // under them.  Register r of a block is row 8 (r / 4) + 4 hl + r % 4 of the half.
  auto reduce = [&](const f32x16 (&s)[NCB], int mt, int half, auto&& next) {
    const int flag = __builtin_amdgcn_readfirstlane(s_flag[mt]);
    const float* const add_row = s_add[mt] + 32 * half + 4 * hl;
    const float* const mul_row = s_mul[mt] + (PASS == 1 ? 32 * half + 4 * hl : 0);
    const int* const t_row = s_t[mt] + 32 * half + 4 * hl;
    float part[NCB];  // of these rows alone: long sums lose less
#pragma unroll
    for (int cb = 0; cb < NCB; ++cb) part[cb] = 0.0f;
    if (PASS == 0) {
      // the 16 scores of the lane's query in log2 units, to f
      auto each = [&](int cb, auto&& f) {
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 add = *(const f32x4*)(add_row + 8 * r4);
          const int4 t4 = *(const int4*)(t_row + 8 * r4);
          const int tt[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float v = __builtin_fmaf(s[cb][4 * r4 + i], c2, add[i]);
            f(tt[i] > ct[cb] ? -INFINITY : v);
          }
        }
      };
      float base[NCB];
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) base[cb] = is_neg_inf(m_run[cb]) ? 0.0f : m_run[cb];
      if (flag == 0) {
        next();
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
          for (int r = 0; r < 16; ++r) part[cb] += mexp2(__builtin_fmaf(s[cb][r], c2, -base[cb]));
        interleave();
      } else {
        next();
#pragma unroll
        for (int cb = 0; cb < NCB; ++cb) each(cb, [&](float v) { part[cb] += mexp2(v - base[cb]); });
      }
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) {
        if (__ballot(is_neg_inf(m_run[cb]) || part[cb] > kMLarge)) {
          float mx = m_run[cb];
          each(cb, [&](float v) { mx = __builtin_fmaxf(mx, v); });
          const float top = is_neg_inf(mx) ? 0.0f : mx;
          sum[cb] *= mexp2(m_run[cb] - top);
          part[cb] = 0.0f;
          each(cb, [&](float v) { part[cb] += mexp2(v - top); });
          m_run[cb] = mx;
        }
        sum[cb] += part[cb];
      }
    } else {
      if ((flag & 2) == 0) {
        next();
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 add = *(const f32x4*)(add_row + 8 * r4), mul = *(const f32x4*)(mul_row + 8 * r4);
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              part[cb] = __builtin_fmaf(mexp2(__builtin_fmaf(s[cb][4 * r4 + i], c2, add[i])), mul[i], part[cb]);
        }
        interleave();
      } else {
        next();
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const f32x4 add = *(const f32x4*)(add_row + 8 * r4), mul = *(const f32x4*)(mul_row + 8 * r4);
          const int4 t4 = *(const int4*)(t_row + 8 * r4);
          const int tt[4] = {t4.x, t4.y, t4.z, t4.w};
#pragma unroll
          for (int cb = 0; cb < NCB; ++cb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = mexp2(__builtin_fmaf(s[cb][4 * r4 + i], c2, add[i])) * mul[i];
              part[cb] += tt[i] < ct[cb] ? 0.0f : p;
            }
        }
      }
#pragma unroll
      for (int cb = 0; cb < NCB; ++cb) sum[cb] += part[cb];
    }
  };

  if (t_begin < t_end) store_tile(0, 0, t_begin);
  __syncthreads();
  constexpr int kHalves = kTile / 32;
  f32x16 cur[NCB], nxt[NCB];
  if (kHalves == 2 && t_begin < t_end) product(0, 0, cur);
  int mt = 0;
  for (int tile = t_begin; tile < t_end; ++tile) {
    const int st = (tile - t_begin) & 1, mn = mt == 2 ? 0 : mt + 1;
    const bool more = tile + 1 < t_end;
    if (more) load_tile(tile + 1);
    if constexpr (kHalves == 2) {
      reduce(cur, mt, 0, [&] { product(st, 1, nxt); });
      if (more) {
        store_tile(st ^ 1, mn, tile + 1);
        __syncthreads();
        reduce(nxt, mt, 1, [&] { product(st ^ 1, 0, cur); });
      } else {
        reduce(nxt, mt, 1, [] {});
      }
    } else {
      product(st, 0, cur);
      reduce(cur, mt, 0, [] {});
      if (more) store_tile(st ^ 1, mn, tile + 1);
      __syncthreads();
    }
    mt = mn;
  }

  // ---- the two halves of a column, then out ----
#pragma unroll
  for (int cb = 0; cb < NCB; ++cb) {
    const int c = c0 + (wid * NCB + cb) * 32 + cl;
    if (PASS == 0) {
      const float m2 = __shfl_xor(m_run[cb], 32, 64), l2 = __shfl_xor(sum[cb], 32, 64);
      const float M = __builtin_fmaxf(m_run[cb], m2), base = is_neg_inf(M) ? 0.0f : M;
      const float L = sum[cb] * mexp2(m_run[cb] - base) + l2 * mexp2(m2 - base);
      if (hl == 0 && c < R) {
        if (a.split == 1) {
          stats[c] = row_stats(M, L);
        } else {
          float* const p = a.part + (((int64_t)bh * R + c) * a.split + part_id) * 2;
          *(f32x2*)(void*)p = f32x2{M, L};
        }
      }
    } else {
      const float t = sum[cb] + __shfl_xor(sum[cb], 32, 64);
      if (hl == 0 && c < a.Nk) {
        float v = c < n ? t : 0.0f;
        if (cnt && c < n) v = cnt[c] > 0 ? t * (float)cnt[c] : 0.0f;
        if (a.split == 1) a.mass[(int64_t)bh * a.Nk + c] = v;
        else a.part[((int64_t)part_id * nbh + bh) * a.Nk + c] = v;
      }
    }
  }
}

template <int DT, int PASS, int KK>
__global__ __launch_bounds__(256, 2) void mass_kernel(MassArgs a) {
  mass_pass<DT, PASS, KK>(a);
}

// Both passes of a head in one launch, where neither has splits (split and blocks are 1): 16 queries
// over 64 keys, 8 groups of 4 heads, 11.1 us against 11.8, host-inclusive 13.3 / 15.7.  A pass that would
// be split is better split (64 queries over 100 keys: 18.4 against 20.0).
constexpr int kMassSmall = 128;  // query rows and keys
template <int DT, int KK>
__global__ __launch_bounds__(256, 1) void mass_small_kernel(MassArgs a) {
  mass_pass<DT, 0, KK>(a);
  __syncthreads();
  mass_pass<DT, 1, KK>(a);
}

// A query's (max, sum) parts, kJoinLanes lanes a query.
constexpr int kJoinLanes = 16;
__global__ __launch_bounds__(256) void mass_join_rows_kernel(const float* part, float* stats, int64_t rows, int split) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / kJoinLanes;
  const int l = threadIdx.x % kJoinLanes;
  const f32x2* p = (const f32x2*)(const void*)part + (i < rows ? i : rows - 1) * split;
  float M = -INFINITY, L = 0.0f;
  for (int s = l; s < split; s += kJoinLanes) {
    const f32x2 v = p[s];
    const float m = __builtin_fmaxf(M, v[0]), base = is_neg_inf(m) ? 0.0f : m;
    L = L * mexp2(M - base) + v[1] * mexp2(v[0] - base);
    M = m;
  }
#pragma unroll
  for (int d = 1; d < kJoinLanes; d <<= 1) {
    const float m2 = __shfl_xor(M, d, 64), l2 = __shfl_xor(L, d, 64);
    const float m = __builtin_fmaxf(M, m2), base = is_neg_inf(m) ? 0.0f : m;
    L = L * mexp2(M - base) + l2 * mexp2(m2 - base);
    M = m;
  }
  if (l == 0 && i < rows) ((f32x2*)(void*)stats)[i] = row_stats(M, L);
}

// The splits' column sums: 32 columns a workgroup, eight threads a column that take every eighth
// split, joined in order.
__global__ __launch_bounds__(256) void mass_join_cols_kernel(const float* part, float* mass, int64_t cols, int split) {
  __shared__ float s_v[8][32];
  const int c = threadIdx.x & 31, sg = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + c;
  float v = 0.0f;
  if (i < cols) {
#pragma unroll 4
    for (int s = sg; s < split; s += 8) v += part[(int64_t)s * cols + i];
  }
  s_v[sg][c] = v;
  __syncthreads();
  if (sg == 0 && i < cols) {
#pragma unroll
    for (int k = 1; k < 8; ++k) v += s_v[k][c];
    mass[i] = v;
  }
}

// Splits of the streamed rows.  Where pieces of 128 rows (two stages) do not fill the chip's 512
// places, a call is latency and takes them all, up to 128 (64 queries over 2048 keys: 20.5 us, with pieces
// of 256 25.6; over 32768 keys of one head 28.9, with 64 of them 34.3, with 256 28.4 and twice the
// workspace).  Else pieces of at least 256 rows, for 1024 workgroups, so that the longest end early (1024
// tokens of 8 x 4 heads 34 us, with pieces of 128 51; 8192 tokens 648, for 512 workgroups 837), up to
// 64 (1 query over 32768 keys of 8 heads: 43.7, with 128 48.9).
static int mass_split(int64_t blocks, int64_t streamed) {
  const int64_t pieces = (streamed + 127) / 128;
  if (blocks * pieces <= 512) return (int)(pieces < 128 ? pieces : 128);
  int64_t want = (1024 + blocks - 1) / blocks;
  const int64_t most = (streamed + 255) / 256;
  if (want > most) want = most;
  return (int)(want > 64 ? 64 : want);
}
struct MassPlan {
  bool small;
  int cols, split0, split1;
  int64_t blocks0, blocks1, rows, part;
};
static MassPlan mass_plan(int dtype, int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq, int64_t Nk) {
  MassPlan p;
  p.cols = dtype == DA_F32 ? 128 : 256;
  p.rows = Hq / Hkv * Nq;
  p.blocks0 = (p.rows + p.cols - 1) / p.cols;
  p.blocks1 = (Nk + p.cols - 1) / p.cols;
  p.small = p.rows <= kMassSmall && Nk <= kMassSmall;
  p.split0 = mass_split(p.blocks0 * B * Hkv, Nk);
  p.split1 = mass_split(p.blocks1 * B * Hkv, p.rows);
  const int64_t p0 = p.split0 > 1 ? B * Hkv * p.rows * p.split0 * 2 : 0;
  const int64_t p1 = p.split1 > 1 ? B * Hkv * Nk * p.split1 : 0;
  p.part = p0 > p1 ? p0 : p1;
  return p;
}

template <int DT, int PASS>
static void launch_pass(const MassArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.B * a.Hkv) * a.split * a.blocks);
  switch ((a.D + 31) / 32) {
    case 1: hipLaunchKernelGGL((mass_kernel<DT, PASS, 2>), grid, dim3(256), 0, st, a); break;
    case 2: hipLaunchKernelGGL((mass_kernel<DT, PASS, 4>), grid, dim3(256), 0, st, a); break;
    case 3: hipLaunchKernelGGL((mass_kernel<DT, PASS, 6>), grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL((mass_kernel<DT, PASS, 8>), grid, dim3(256), 0, st, a); break;
  }
}
template <int DT>
static int launch_mass(MassArgs a, const MassPlan& p, hipStream_t st, const char* who) {
  const int64_t bh = (int64_t)a.B * a.Hkv;
  if (p.small) {
    a.split = a.blocks = 1;
    switch ((a.D + 31) / 32) {
      case 1: hipLaunchKernelGGL((mass_small_kernel<DT, 2>), dim3((unsigned)bh), dim3(256), 0, st, a); break;
      case 2: hipLaunchKernelGGL((mass_small_kernel<DT, 4>), dim3((unsigned)bh), dim3(256), 0, st, a); break;
      case 3: hipLaunchKernelGGL((mass_small_kernel<DT, 6>), dim3((unsigned)bh), dim3(256), 0, st, a); break;
      default: hipLaunchKernelGGL((mass_small_kernel<DT, 8>), dim3((unsigned)bh), dim3(256), 0, st, a); break;
    }
    return check_launch(who);
  }
  a.split = p.split0;
  a.blocks = (int)p.blocks0;
  launch_pass<DT, 0>(a, st);
  if (p.split0 > 1) {
    const int64_t rows = bh * p.rows;
    hipLaunchKernelGGL(mass_join_rows_kernel, dim3((unsigned)((rows * kJoinLanes + 255) / 256)), dim3(256), 0, st,
                       a.part, a.stats, rows, p.split0);
  }
  a.split = p.split1;
  a.blocks = (int)p.blocks1;
  launch_pass<DT, 1>(a, st);
  if (p.split1 > 1) {
    const int64_t cols = bh * a.Nk;
    hipLaunchKernelGGL(mass_join_cols_kernel, dim3((unsigned)((cols + 31) / 32)), dim3(256), 0, st, a.part, a.mass,
                       cols, p.split1);
  }
  return check_launch(who);
}

}  // namespace da

using namespace da;

// The two statistics of every query row, then the splits' parts (of whichever type needs more).
extern "C" int64_t da_attention_mass_workspace_size(int64_t B, int64_t Hq, int64_t Hkv, int64_t Nq, int64_t Nk) {
  if (B <= 0 || Hkv <= 0 || Hq < Hkv || Nq <= 0 || Nk <= 0) return 0;
  const MassPlan p = mass_plan(DA_BF16, B, Hq, Hkv, Nq, Nk), p32 = mass_plan(DA_F32, B, Hq, Hkv, Nq, Nk);
  const int64_t rows = (B * Hkv * p.rows * 2 + 3) / 4 * 4;
  return (rows + (p.part > p32.part ? p.part : p32.part)) * (int64_t)sizeof(float);
}

extern "C" int da_attention_mass(const void* q, const void* k, int dtype, int64_t B, int64_t Hq, int64_t Hkv,
                                 int64_t Nq, int64_t Nk, int64_t D, int64_t sq_b, int64_t sq_h, int64_t sq_n,
                                 int64_t sk_b, int64_t sk_h, int64_t sk_n, const int32_t* counts,
                                 const int32_t* timestamps, const int32_t* lengths, int64_t q_start, float scale,
                                 float* mass, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "da_attention_mass";
  DA_REQUIRE(q && k && mass, "%s: null pointer", who);
  if (dtype != DA_BF16 && dtype != DA_F16 && dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: q and k must be bf16, fp16 or fp32", who);
  if (D <= 0 || D > 128 || (D & 7))
    return set_error(DA_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 in [8, 128]", who);
  DA_REQUIRE(B > 0 && Hq > 0 && Hkv > 0 && Hq % Hkv == 0 && Nq > 0 && Nk > 0, "%s: bad shape", who);
  if (Hq / Hkv > 64) return set_error(DA_ERR_UNSUPPORTED, "%s: GQA group above 64", who);
  if (Nk > (1 << 24) || Nq > (1 << 24) || B * Hkv > 65535)
    return set_error(DA_ERR_UNSUPPORTED, "%s: more than 2^24 keys or queries, or 65535 (sequence, head) pairs", who);
  const int64_t align = dtype == DA_F32 ? 3 : 7;
  // a dimension of one has no stride
  const int64_t strides = (B > 1 ? sq_b | sk_b : 0) | (Hq > 1 ? sq_h : 0) | (Hkv > 1 ? sk_h : 0) | (Nq > 1 ? sq_n : 0) |
                          (Nk > 1 ? sk_n : 0);
  DA_REQUIRE((strides & align) == 0 && (((uintptr_t)q | (uintptr_t)k) & 15) == 0,
             "%s: rows must be 16-byte aligned", who);
  DA_REQUIRE(scale > 0.0f, "%s: scale must be positive", who);
  DA_REQUIRE(q_start > -(1ll << 40) && q_start < (1ll << 40), "%s: q_start out of range", who);
  const int64_t need = da_attention_mass_workspace_size(B, Hq, Hkv, Nq, Nk);
  if (!workspace || workspace_bytes < need)
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %lld bytes required", who, (long long)need);
  DA_REQUIRE(((uintptr_t)workspace & 15) == 0, "%s: workspace must be 16-byte aligned", who);
  const MassPlan p = mass_plan(dtype, B, Hq, Hkv, Nq, Nk);
  // a launch holds fewer than 2^32 threads
  if (p.rows >= (1ll << 30) || B * Hkv * p.split0 * p.blocks0 >= (1ll << 24) ||
      B * Hkv * p.split1 * p.blocks1 >= (1ll << 24) || B * Hkv * p.rows >= (1ll << 28) || B * Hkv * Nk >= (1ll << 32))
    return set_error(DA_ERR_UNSUPPORTED, "%s: too many query rows or keys for one call", who);
  MassArgs a = {};
  a.q = q; a.k = k;
  a.sq_b = sq_b; a.sq_h = sq_h; a.sq_n = sq_n; a.sk_b = sk_b; a.sk_h = sk_h; a.sk_n = sk_n;
  a.counts = counts; a.ts = timestamps; a.lengths = lengths; a.q_start = q_start;
  a.scale_log2 = scale * kMLog2e;
  a.stats = (float*)workspace;
  a.part = a.stats + (B * Hkv * p.rows * 2 + 3) / 4 * 4;
  a.mass = mass;
  a.B = (int)B; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.Nq = (int)Nq; a.Nk = (int)Nk; a.D = (int)D;
  a.gshift = (a.G & (a.G - 1)) == 0 ? __builtin_ctz(a.G) : -1;
  hipStream_t st = (hipStream_t)stream;
  if (dtype == DA_F32) return launch_mass<DA_F32>(a, p, st, who);
  if (dtype == DA_F16) return launch_mass<DA_F16>(a, p, st, who);
  return launch_mass<DA_BF16>(a, p, st, who);
}
