// New tokens into a paged cache, rotated on the way (include/deltaattn_paged.h).
//
// Mathematics: dims (x, y) of a pair become (x cos - y sin, y cos + x sin) in fp32, rounded once; values
// and dims past the rotation are copied.  Bound by memory: a token is read and written once, (Hq + 2
// Hkv) rows each way, beside 4 rot bytes of cos and sin.
//
// A wave takes one token (or a share of one, where tokens are few): its lanes are the row's chunks
// times a run of heads, so a lane's cos and sin serve every head it turns.  A chunk is V elements of
// the first half and V of the second (V up to 8: 16-byte loads of a 16-bit type), or V plain ones.
#include <algorithm>

#include "da_paged.hpp"

namespace da {

struct AppendArgs {
  const char *k, *v, *q;
  char* q_out;
  int64_t sk_t, sk_h, sv_t, sv_h, sq_t, sq_h, so_t, so_h;
  const char *cos, *sin;
  int64_t rows, s_rot;
  int Hq, Hkv, D, rot;
  int per_token, parts;
  Pages pages;
  PageBatch seq;
};

// V elements of type DT at p (aligned to V elements) as fp32, and back
template <int DT, int V>
struct Chunk {
  float x[V];
  __device__ __forceinline__ void load(const char* p) {
    if constexpr (DT == DA_F32) {
      if constexpr (V == 8) {
        const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
      } else if constexpr (V == 4) {
        const f32x4 a = *(const f32x4*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = a[i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = ((const float*)p)[i];
      }
    } else if constexpr (V >= 2) {
      uint32_t w[V / 2];
      if constexpr (V == 8) {
        const u32x4 a = *(const u32x4*)p;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = a[i];
      } else if constexpr (V == 4) {
        const u32x2 a = *(const u32x2*)p;
        w[0] = a[0], w[1] = a[1];
      } else {
        w[0] = *(const uint32_t*)p;
      }
#pragma unroll
      for (int i = 0; i < V / 2; ++i) x[2 * i] = E16<DT>::lo(w[i]), x[2 * i + 1] = E16<DT>::hi(w[i]);
    } else {
      x[0] = E16<DT>::one(*(const uint16_t*)p);
    }
  }
  __device__ __forceinline__ void store(char* p) const {
    if constexpr (DT == DA_F32) {
      if constexpr (V >= 4) {
#pragma unroll
        for (int i = 0; i < V; i += 4) *(f32x4*)(p + 4 * i) = f32x4{x[i], x[i + 1], x[i + 2], x[i + 3]};
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) ((float*)p)[i] = x[i];
      }
    } else if constexpr (V == 8) {
      *(u32x4*)p = u32x4{E16<DT>::pack(x[0], x[1]), E16<DT>::pack(x[2], x[3]), E16<DT>::pack(x[4], x[5]),
                         E16<DT>::pack(x[6], x[7])};
    } else if constexpr (V == 4) {
      *(u32x2*)p = u32x2{E16<DT>::pack(x[0], x[1]), E16<DT>::pack(x[2], x[3])};
    } else if constexpr (V == 2) {
      *(uint32_t*)p = E16<DT>::pack(x[0], x[1]);
    } else {
      *(uint16_t*)p = E16<DT>::bits(x[0]);
    }
  }
};

// RT: type of cos and sin.  INTER: pairs are neighbours, a chunk holds V / 2 of them (V is 8).
template <int DT, int RT, int V, bool INTER>
__global__ __launch_bounds__(256) void append_kernel(AppendArgs a) {
  constexpr int ES = DT == DA_F32 ? 4 : 2, RS = RT == DA_F32 ? 4 : 2;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane((int)(blockIdx.x * 4 + (threadIdx.x >> 6)));
  const int t = wave / a.parts, part = wave - t * a.parts;
  if (t >= a.seq.T) return;
  const int b = sequence_of(a.seq, t, lane);
  if (b < 0) return;
  if (a.seq.cu && t >= a.seq.cu[b + 1]) return;
  // the token's place (max_seqlen does not move it), and the row of cos and sin
  const int64_t slot = a.seq.slot(b, t);
  int64_t row = a.per_token ? t : slot + (a.seq.start ? a.seq.start[b] : 0);
  row = row < 0 ? 0 : row >= a.rows ? a.rows - 1 : row;
  int page = -1;
  if (slot >= 0 && slot < a.seq.max_keys) page = a.seq.table[(int64_t)b * a.seq.table_stride + (slot >> a.pages.shift)];
  const bool kept = page >= 0 && page < a.pages.num_pages;
  const int64_t in = slot & ((1 << a.pages.shift) - 1);
  char* const kd = const_cast<char*>(a.pages.k) + ES * (page * a.pages.sk_p + in * a.pages.sk_n);
  char* const vd = const_cast<char*>(a.pages.v) + ES * (page * a.pages.sv_p + in * a.pages.sv_n);
  const char* const ks = a.k + ES * (t * a.sk_t);
  const char* const vs = a.v + ES * (t * a.sv_t);
  const char* const qs = a.q + ES * (t * a.sq_t);
  char* const qd = a.q_out + ES * (t * a.so_t);

  const int half = INTER ? 0 : a.rot / 2;
  const int pairs = half / V;                           // chunks of two halves
  const int chunks = INTER ? a.D / V : (a.D - half) / V;  // of a rotated row
  const int Hr = a.Hkv + (a.q ? a.Hq : 0);              // rotated rows: keys, then queries
  // a lane keeps its chunk and goes through the heads; the wave holds `per` heads at once
  const int per = 64 / chunks, c = lane % chunks;
  const int h0 = lane / chunks;
  float co[V], si[V];
  const int64_t rot_row = row * a.s_rot;
  if (INTER || c < pairs) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // interleaved: pair (V c + e) / 2 of the row
      const int d = INTER ? (V * c + e) >> 1 : V * c + e;
      const bool on = !INTER || 2 * d < a.rot;
      const char *pc = a.cos + RS * (rot_row + d), *ps = a.sin + RS * (rot_row + d);
      if constexpr (RT == DA_F32) {
        co[e] = on ? *(const float*)pc : 1.0f;
        si[e] = on ? *(const float*)ps : 0.0f;
      } else {
        co[e] = on ? E16<RT>::one(*(const uint16_t*)pc) : 1.0f;
        si[e] = on ? E16<RT>::one(*(const uint16_t*)ps) : 0.0f;
      }
    }
  }
  if (h0 < per) {
    for (int h = h0 + per * part; h < Hr; h += per * a.parts) {
      const bool isK = h < a.Hkv;
      if (isK && !kept) continue;
      const char* src = isK ? ks + ES * (h * a.sk_h) : qs + ES * ((h - a.Hkv) * a.sq_h);
      char* dst = isK ? kd + ES * (h * a.pages.sk_h) : qd + ES * ((h - a.Hkv) * a.so_h);
      Chunk<DT, V> x, y;
      if constexpr (INTER) {
        x.load(src + ES * V * c);
        if (V * c < a.rot) {
#pragma unroll
          for (int e = 0; e < V; e += 2) {
            const float u = x.x[e], w = x.x[e + 1];
            if (V * c + e < a.rot) {
              x.x[e] = u * co[e] - w * si[e];
              x.x[e + 1] = w * co[e] + u * si[e];
            }
          }
        }
        x.store(dst + ES * V * c);
      } else if (c < pairs) {
        x.load(src + ES * V * c);
        y.load(src + ES * (half + V * c));
        Chunk<DT, V> u, w;
#pragma unroll
        for (int e = 0; e < V; ++e) {
          u.x[e] = x.x[e] * co[e] - y.x[e] * si[e];
          w.x[e] = y.x[e] * co[e] + x.x[e] * si[e];
        }
        u.store(dst + ES * V * c);
        w.store(dst + ES * (half + V * c));
      } else {
        x.load(src + ES * (half + V * c));
        x.store(dst + ES * (half + V * c));
      }
    }
  }
  if (!kept) return;
  // values: 16-byte pieces of a row, moved as they are
  const int pieces = ES * a.D / 16;
  for (int j = lane + 64 * part; j < a.Hkv * pieces; j += 64 * a.parts) {
    const int h = j / pieces, p = j - h * pieces;
    *(u32x4*)(vd + ES * (h * a.pages.sv_h) + 16 * p) = *(const u32x4*)(vs + ES * (h * a.sv_h) + 16 * p);
  }
}

int allow_lds(const void* kernel, int bytes, bool (&done)[kMaxDevices]) {
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  const bool known = dev >= 0 && dev < kMaxDevices;
  if (e == hipSuccess && known && done[dev]) return DA_OK;
  if (e == hipSuccess) e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != hipSuccess) return set_error(DA_ERR_HIP, "hipFuncSetAttribute: %s", hipGetErrorString(e));
  if (known) done[dev] = true;
  return DA_OK;
}

int fill_pages(Pages& p, const DaPagedKV* kv, int64_t D, const char* who) {
  DA_REQUIRE(kv && kv->k && kv->v, "%s: null pages", who);
  DA_REQUIRE(kv->num_pages > 0 && kv->num_pages < (1ll << 31), "%s: no pages", who);
  DA_REQUIRE(kv->page_size >= 16 && kv->page_size < (1ll << 30) && !(kv->page_size & (kv->page_size - 1)),
             "%s: page_size must be a power of two from 16 on (got %lld)", who, (long long)kv->page_size);
  for (int64_t s : {kv->sk_p, kv->sk_h, kv->sk_n, kv->sv_p, kv->sv_h, kv->sv_n})
    DA_REQUIRE((s & 7) == 0, "%s: page strides must be multiples of 8 elements (got %lld)", who, (long long)s);
  for (int64_t s : {kv->sk_n, kv->sv_n})
    DA_REQUIRE(s >= D && s < (1ll << 23), "%s: row strides of pages must be in [head_dim, 2^23) (got %lld)", who,
               (long long)s);
  DA_REQUIRE((((uintptr_t)kv->k | (uintptr_t)kv->v) & 15) == 0, "%s: pages must be 16-byte aligned", who);
  int shift = 4;
  while ((1ll << shift) < kv->page_size) ++shift;
  p = Pages{(const char*)kv->k, (const char*)kv->v, kv->sk_p, kv->sk_h, kv->sk_n,
            kv->sv_p,           kv->sv_h,           kv->sv_n, (int)kv->num_pages, shift};
  return DA_OK;
}

int fill_batch(PageBatch& s, const DaPagedBatch* b, const Pages& p, int64_t T, const char* who) {
  DA_REQUIRE(b && b->table && b->lengths, "%s: null table or lengths", who);
  DA_REQUIRE(b->B > 0 && b->B < (1ll << 24) && b->width > 0, "%s: an empty table", who);
  DA_REQUIRE(b->table_stride >= b->width || b->B == 1, "%s: table rows overlap", who);
  DA_REQUIRE((b->width << p.shift) < (1ll << 30) && b->width < (1ll << 30), "%s: sequences of 2^30 tokens", who);
  DA_REQUIRE(b->cu ? b->max_seqlen > 0 : b->B <= T, "%s: needs max_seqlen > 0 with cu, a token for each sequence without",
             who);
  s = PageBatch{b->table, b->lengths, b->cu, b->start, b->table_stride, (int)b->B, (int)T,
                (int)(b->cu ? std::min(b->max_seqlen, T) : 1), (int)(b->width << p.shift)};
  return DA_OK;
}

template <int DT, int RT>
static int launch_append(const AppendArgs& a, bool interleaved, unsigned grid, hipStream_t st) {
  const int half = a.rot / 2;
  const dim3 g(grid), w(256);
  if (interleaved) hipLaunchKernelGGL((append_kernel<DT, RT, 8, true>), g, w, 0, st, a);
  else if (half % 8 == 0) hipLaunchKernelGGL((append_kernel<DT, RT, 8, false>), g, w, 0, st, a);
  else if (half % 4 == 0) hipLaunchKernelGGL((append_kernel<DT, RT, 4, false>), g, w, 0, st, a);
  else hipLaunchKernelGGL((append_kernel<DT, RT, 2, false>), g, w, 0, st, a);
  return check_launch("paged append");
}

}  // namespace da

using namespace da;

extern "C" int da_paged_append(const void* k, int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_t, int64_t sv_h,
                               const void* q, int64_t sq_t, int64_t sq_h, void* q_out, int64_t so_t, int64_t so_h,
                               int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, const void* cos,
                               const void* sin, int rot_dtype, int64_t rows, int64_t s_rot, int64_t rot,
                               int interleaved, int per_token, const DaPagedKV* kv, const DaPagedBatch* batch,
                               void* stream) {
  const char* who = "da_paged_append";
  if (dtype != DA_BF16 && dtype != DA_F16 && dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: tensors must be bf16, fp16 or fp32", who);
  if (D <= 0 || D > 128 || (D & 7))
    return set_error(DA_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 in [8, 128] (got %lld)", who, (long long)D);
  DA_REQUIRE(k && v && (!q || q_out), "%s: null pointer", who);
  DA_REQUIRE(T > 0 && Hkv > 0 && Hkv < (1 << 16) && (!q || (Hq > 0 && Hq < (1 << 16))), "%s: empty shape", who);
  DA_REQUIRE(T < (1ll << 26), "%s: more than 2^26 tokens", who);  // a launch has less than 2^32 threads, 64 a token
  DA_REQUIRE(rot >= 0 && rot <= D && (rot & 3) == 0, "%s: the rotated dims must be a multiple of 4 up to head_dim (got %lld)",
             who, (long long)rot);
  if (rot) {
    DA_REQUIRE(cos && sin && rows > 0, "%s: rotation needs cos and sin", who);
    DA_REQUIRE(rot_dtype == DA_F32 || rot_dtype == dtype, "%s: cos and sin must be fp32 or of the pages' type", who);
    DA_REQUIRE(s_rot >= rot / 2 || s_rot == 0 || rows == 1, "%s: rows of cos and sin overlap", who);
    DA_REQUIRE(!per_token || rows >= T, "%s: a row of cos and sin for every token is needed", who);
  }
  DA_REQUIRE((((uintptr_t)k | (uintptr_t)v | (uintptr_t)q | (uintptr_t)q_out) & 15) == 0, "%s: tensors must be 16-byte aligned",
             who);
  for (int64_t s : {sk_t, sk_h, sv_t, sv_h, q ? sq_t : 0, q ? sq_h : 0, q ? so_t : 0, q ? so_h : 0})
    DA_REQUIRE((s & 7) == 0, "%s: strides must be multiples of 8 elements (got %lld)", who, (long long)s);
  AppendArgs a = {};
  if (int rc = fill_pages(a.pages, kv, D, who)) return rc;
  if (int rc = fill_batch(a.seq, batch, a.pages, T, who)) return rc;
  a.k = (const char*)k; a.v = (const char*)v; a.q = (const char*)q; a.q_out = (char*)q_out;
  a.sk_t = sk_t; a.sk_h = sk_h; a.sv_t = sv_t; a.sv_h = sv_h;
  a.sq_t = sq_t; a.sq_h = sq_h; a.so_t = so_t; a.so_h = so_h;
  a.cos = (const char*)cos; a.sin = (const char*)sin;
  a.rows = rot ? rows : 1; a.s_rot = s_rot;
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.D = (int)D; a.rot = (int)rot;
  a.per_token = per_token ? 1 : 0;
  // up to 8 waves a token until two waves a SIMD are there
  a.parts = (int)std::max<int64_t>(1, std::min<int64_t>(8, 2048 / T));
  const int64_t waves = T * a.parts;
  const unsigned grid = (unsigned)((waves + 3) / 4);
  hipStream_t st = (hipStream_t)stream;
  const bool inter = interleaved != 0 && rot > 0;
  const bool wide = rot && rot_dtype == DA_F32;
  switch (dtype) {
    case DA_BF16: return wide ? launch_append<DA_BF16, DA_F32>(a, inter, grid, st) : launch_append<DA_BF16, DA_BF16>(a, inter, grid, st);
    case DA_F16: return wide ? launch_append<DA_F16, DA_F32>(a, inter, grid, st) : launch_append<DA_F16, DA_F16>(a, inter, grid, st);
    default: return launch_append<DA_F32, DA_F32>(a, inter, grid, st);
  }
}
