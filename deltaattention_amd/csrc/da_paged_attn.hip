// Attention of new tokens over a paged cache (include/deltaattn_paged.h).
#include <algorithm>

#include "da_paged.hpp"

namespace da {

template <int DT>
__device__ __forceinline__ float element(const char* p, int64_t i) {
  if constexpr (DT == DA_F32) return ((const float*)p)[i];
  else return E16<DT>::one(((const uint16_t*)p)[i]);
}

// One wave a (token, query head): 64 keys at a time, a lane a key for the scores and two dims a lane
// for the output.
template <int DT>
__global__ __launch_bounds__(64) void paged_simple_kernel(PagedAttnArgs a) {
  constexpr int ES = DT == DA_F32 ? 4 : 2;
  __shared__ float qs[128];
  const int lane = threadIdx.x, t = blockIdx.x, h = blockIdx.y, g = h / a.G;
  const int b = sequence_of(a.seq, t, lane);
  if (b < 0) return;
  const int n = a.seq.tokens(b), i = t - a.seq.first(b);
  if (i >= n) return;
  const char* qrow = a.q + ES * (t * a.sq_t + h * a.sq_h);
  for (int d = lane; d < a.D; d += 64) qs[d] = element<DT>(qrow, d) * a.scale_log2;
  __syncthreads();
  float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
  const int d0 = min(2 * lane, a.D - 2);
  for (int part = 0; part < 2; ++part) {
    const PageBatch& s = part ? a.seq : a.prefix;
    if (s.B == 0) continue;
    const int sb = part ? b : sequence_of(s, t, lane);
    if (sb < 0) continue;
    const int N = part ? s.keys(sb) - n + i + 1 : s.keys(sb);
    const int32_t* table = s.table + (int64_t)sb * s.table_stride;
    for (int k0 = 0; k0 < N; k0 += 64) {
      const int key = k0 + lane;
      float x = -INFINITY;
      if (key < N) {
        const int page = table[key >> a.pages.shift];
        x = 0.0f;
        if (page >= 0 && page < a.pages.num_pages) {
          const char* row = a.pages.k + ES * (page * a.pages.sk_p + g * a.pages.sk_h +
                                              (key & ((1 << a.pages.shift) - 1)) * a.pages.sk_n);
          for (int d = 0; d < a.D; ++d) x += qs[d] * element<DT>(row, d);
        }
      }
      float mt = x;
      for (int d = 1; d < 64; d <<= 1) mt = fmaxf(mt, __shfl_xor(mt, d, 64));
      const float mn = fmaxf(m, mt);
      const float alpha = m == -INFINITY ? 0.0f : exp2f(m - mn);
      const float p = mn == -INFINITY ? 0.0f : exp2f(x - mn);
      float ps = p;
      for (int d = 1; d < 64; d <<= 1) ps += __shfl_xor(ps, d, 64);
      l = l * alpha + ps;
      o0 *= alpha, o1 *= alpha;
      m = mn;
      for (int j = 0; j < min(64, N - k0); ++j) {
        const int page = table[(k0 + j) >> a.pages.shift];
        if (page < 0 || page >= a.pages.num_pages) continue;
        const char* row = a.pages.v + ES * (page * a.pages.sv_p + g * a.pages.sv_h +
                                            ((k0 + j) & ((1 << a.pages.shift) - 1)) * a.pages.sv_n);
        const float pj = __shfl(p, j, 64);
        o0 += pj * element<DT>(row, d0), o1 += pj * element<DT>(row, d0 + 1);
      }
    }
  }
  if (2 * lane >= a.D) return;
  const float inv = l > 0.0f ? 1.0f / l : 0.0f;
  char* orow = a.out + ES * (t * a.so_t + h * a.so_h);
  if constexpr (DT == DA_F32) *(f32x2*)(orow + 4 * d0) = f32x2{o0 * inv, o1 * inv};
  else *(uint32_t*)(orow + 2 * d0) = E16<DT>::pack(o0 * inv, o1 * inv);
}

// Items of up to kWholeTiles tiles are not split: one launch.
constexpr int kWholeTiles = 8;

struct PagedWs {
  int64_t slots, states, total;
};
static int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// How a call runs, by what the host knows of it.
static PagedWs plan(PagedAttnArgs& a, int dtype) {
  const int E = a.prefix.B + a.seq.B;
  const int most = std::max(a.seq.max_len, a.prefix.B ? a.prefix.max_len : 0);
  a.workers = 0;
  if (dtype == DA_F32 || (int64_t)most * a.G > kStreamRows) return PagedWs{};
  a.slot_rows = most * a.G;
  const int keys = std::max(a.seq.max_keys, a.prefix.B ? a.prefix.max_keys : 0);
  a.whole = keys <= kWholeTiles * kStreamTile;
  a.workers = a.whole ? E * a.Hkv : 2 * cu_count();
  PagedWs w;
  w.slots = a.whole ? 0 : round256(4 * (1 + (int64_t)E));
  w.states = w.slots + (a.whole ? 0 : 2 * (int64_t)a.workers * a.slot_rows * kState * 4);
  w.total = w.states + (a.prefix.B ? 2 * (int64_t)a.seq.T * a.Hq * kState * 4 : 0);
  return w;
}

static int fill_attention(PagedAttnArgs& a, int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, const DaPagedKV* kv,
                          const DaPagedBatch* batch, const DaPagedBatch* prefix, const char* who) {
  if (dtype != DA_BF16 && dtype != DA_F16 && dtype != DA_F32)
    return set_error(DA_ERR_UNSUPPORTED, "%s: tensors must be bf16, fp16 or fp32", who);
  if (D <= 0 || D > 128 || (D & 7))
    return set_error(DA_ERR_UNSUPPORTED, "%s: head_dim must be a multiple of 8 in [8, 128] (got %lld)", who, (long long)D);
  DA_REQUIRE(T > 0 && T < (1ll << 28) && Hq > 0 && Hkv > 0 && Hq < (1 << 16), "%s: empty shape", who);
  DA_REQUIRE(Hq % Hkv == 0, "%s: Hq (%lld) must be a multiple of Hkv (%lld)", who, (long long)Hq, (long long)Hkv);
  if (int rc = fill_pages(a.pages, kv, D, who)) return rc;
  if (int rc = fill_batch(a.seq, batch, a.pages, T, who)) return rc;
  if (prefix) {
    DA_REQUIRE(prefix->cu, "%s: the groups of a prefix need cu", who);
    if (int rc = fill_batch(a.prefix, prefix, a.pages, T, who)) return rc;
  }
  const int64_t keys = std::max(a.seq.max_keys, a.prefix.B ? a.prefix.max_keys : 0);
  DA_REQUIRE(((int64_t)a.seq.B + a.prefix.B) * Hkv * (keys / kStreamTile + 1) < (1ll << 31),
             "%s: tables of too many sequences, heads and pages", who);
  a.Hq = (int)Hq; a.Hkv = (int)Hkv; a.G = (int)(Hq / Hkv); a.D = (int)D;
  return DA_OK;
}

}  // namespace da

using namespace da;

extern "C" int64_t da_paged_attention_workspace_size(int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D,
                                                     const DaPagedKV* kv, const DaPagedBatch* batch,
                                                     const DaPagedBatch* prefix) {
  PagedAttnArgs a = {};
  if (fill_attention(a, dtype, T, Hq, Hkv, D, kv, batch, prefix, "da_paged_attention")) return 0;  // the call refuses it
  return plan(a, dtype).total;
}

extern "C" int da_paged_attention(const void* q, int64_t sq_t, int64_t sq_h, void* out, int64_t so_t, int64_t so_h,
                                  int dtype, int64_t T, int64_t Hq, int64_t Hkv, int64_t D, float scale,
                                  const DaPagedKV* kv, const DaPagedBatch* batch, const DaPagedBatch* prefix,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  const char* who = "da_paged_attention";
  DA_REQUIRE(q && out, "%s: null pointer", who);
  PagedAttnArgs a = {};
  if (int rc = fill_attention(a, dtype, T, Hq, Hkv, D, kv, batch, prefix, who)) return rc;
  DA_REQUIRE(scale > 0.0f, "%s: scale must be positive", who);
  DA_REQUIRE((((uintptr_t)q | (uintptr_t)out) & 15) == 0, "%s: tensors must be 16-byte aligned", who);
  for (int64_t s : {sq_t, sq_h, so_t, so_h})
    DA_REQUIRE((s & 7) == 0, "%s: strides must be multiples of 8 elements (got %lld)", who, (long long)s);
  a.q = (const char*)q; a.out = (char*)out;
  a.sq_t = sq_t; a.sq_h = sq_h; a.so_t = so_t; a.so_h = so_h;
  a.scale_log2 = scale * 1.4426950408889634f;
  const PagedWs w = plan(a, dtype);
  if (w.total > 0 && (!workspace || workspace_bytes < w.total))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %lld bytes required", who, (long long)w.total);
  DA_REQUIRE(((uintptr_t)workspace & 255) == 0, "%s: the workspace must be 256-byte aligned", who);
  char* ws = (char*)workspace;
  a.begin = (uint32_t*)ws;
  a.slots = (float*)(ws + w.slots);
  a.states = (float*)(ws + w.states);
  hipStream_t st = (hipStream_t)stream;
  if (a.workers) return launch_paged_stream(a, dtype, st);
  const dim3 grid((unsigned)T, (unsigned)Hq);
  switch (dtype) {
    case DA_BF16: hipLaunchKernelGGL(paged_simple_kernel<DA_BF16>, grid, dim3(64), 0, st, a); break;
    case DA_F16: hipLaunchKernelGGL(paged_simple_kernel<DA_F16>, grid, dim3(64), 0, st, a); break;
    default: hipLaunchKernelGGL(paged_simple_kernel<DA_F32>, grid, dim3(64), 0, st, a);
  }
  return check_launch("paged attention");
}
