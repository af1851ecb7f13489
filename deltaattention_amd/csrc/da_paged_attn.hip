// Attention of new tokens over a paged cache (include/deltaattn_paged.h): which kernel takes which
// entries, and the parts of a result joined.
//
// An entry (a sequence, or a group behind a prefix) of up to kStreamRows rows goes to the stream
// (da_paged_stream.hip); one with more rows, and all of fp32, to the row kernels (da_attn.hip's, over
// pages), whose items are blocks of rows and, where those do not fill the chip, runs of keys.
// A prefix is a list of its own, seen whole by all rows of a group at once: its keys are read once for
// the group, and each row's result is joined with that of its own sequence.
#include <algorithm>

#include "da_paged.hpp"
#include "da_tile.hpp"

namespace da {

// The parts of a row joined: a wave a (token, query head), two dims a lane.
template <int DT>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
  const int lane = threadIdx.x & 63;
  const int wid = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int t = blockIdx.x, h = blockIdx.y * 4 + wid;
  if (h >= a.Hq) return;
  const int b = sequence_of(a.seq, t, lane);
  if (b < 0) return;
  const int g = h / a.G;
  float M = -INFINITY, L = 0.0f, y0 = 0.0f, y1 = 0.0f;
  // a part's state: the running result takes it in
  auto take = [&](const float* st) {
    const f32x2 ml = *(const f32x2*)(st + 128), z = *(const f32x2*)(st + 2 * lane);
    const float mn = __builtin_fmaxf(M, ml[0]), ref = mn == -INFINITY ? 0.0f : mn;
    const float fo = exp2_fast(M - ref), fn = exp2_fast(ml[0] - ref);
    y0 = y0 * fo + z[0] * fn;
    y1 = y1 * fo + z[1] * fn;
    L = L * fo + ml[1] * fn;
    M = mn;
  };
  for (int list = a.prefix.B ? 0 : 1; list < 2; ++list) {
    const PageBatch& s = list ? a.seq : a.prefix;
    const int e = list ? b : sequence_of(s, t, lane);
    if (e < 0) continue;
    const int tokens = s.tokens(e), i = t - s.first(e);
    if (i >= tokens) {
      if (list) return;
      continue;
    }
    if (tokens * a.G > a.short_rows[list]) {  // the row kernels'
      if (!a.parts[list]) return;
      for (int p = 0; p < a.splits[list]; ++p) take(a.parts[list] + (((int64_t)p * s.T + t) * a.Hq + h) * kState);
      continue;
    }
    const int tiles = stream_tiles(a, tokens, s.keys(e), list);
    if (tiles == 0) continue;
    const uint32_t per = a.whole ? 1 : a.begin[0];
    const uint32_t U = a.whole ? 0 : a.begin[1 + (list ? a.prefix.B : 0) + e] + g * tiles;
    const uint32_t w0 = U / per, w1 = a.whole ? w0 : (U + tiles - 1) / per;
    if (w0 == w1) {
      if (a.prefix.B == 0) return;  // written where it was computed
      take(a.states + (((int64_t)list * a.seq.T + t) * a.Hq + h) * kState);
      continue;
    }
    const int r = i * a.G + h - g * a.G;
    for (uint32_t w = w0; w <= w1; ++w)
      take(a.slots + ((int64_t)(2 * w + (w == w0 && U != w0 * per ? 1 : 0)) * a.slot_rows + r) * kState);
  }
  if (2 * lane >= a.D) return;
  const float inv = L > 0.0f ? 1.0f / L : 0.0f;
  if constexpr (DT == DA_F32)
    *(f32x2*)(a.out + 4 * (t * a.so_t + h * a.so_h) + 8 * lane) = f32x2{y0 * inv, y1 * inv};
  else
    *(uint32_t*)(a.out + 2 * (t * a.so_t + h * a.so_h) + 4 * lane) = E16<DT>::pack(y0 * inv, y1 * inv);
}

// Items of up to kWholeTiles tiles are not split: one launch.
constexpr int kWholeTiles = 8;
// A part of a row kernel's item has at least so many keys.
constexpr int kPartKeys = 1024;

struct PagedPlan {
  bool stream, rows[2], wide[2], join;
  int64_t slots, states, parts[2], total;  // byte offsets in the workspace
};
static int64_t round256(int64_t x) { return (x + 255) & ~(int64_t)255; }

// How a call runs, by what the host knows of it.
static PagedPlan plan(PagedAttnArgs& a, int dtype) {
  PagedPlan p = {};
  const int E = a.prefix.B + a.seq.B;
  const PageBatch* lists[2] = {&a.prefix, &a.seq};
  int keys = 0;
  int64_t slot_rows = 0, parts = 0;
  for (int i = 0; i < 2; ++i) {
    const PageBatch& s = *lists[i];
    a.short_rows[i] = 0;
    a.splits[i] = 1;
    if (s.B == 0) continue;
    const int64_t most = (int64_t)s.max_len * a.G;
    // where every entry must have the most tokens to make up T (unless the batch is padded), the
    // row kernel takes all of a list with many rows, and no stream runs for it
    const bool even = (int64_t)s.B * s.max_len == s.T;
    if (dtype != DA_F32 && a.G <= kStreamRows && (most <= kStreamRows || !even)) {
      a.short_rows[i] = kStreamRows;
      p.stream = true;
      keys = std::max(keys, s.max_keys);
      slot_rows = std::max(slot_rows, std::min<int64_t>(most, kStreamRows));
    }
    p.rows[i] = most > a.short_rows[i];
    if (!p.rows[i]) continue;
    const RowsShape shape = paged_rows_shape(dtype, a.G);
    auto items = [&](int rows) {
      const int64_t all = (int64_t)s.B * ((s.max_len + rows - 1) / rows);
      return std::min<int64_t>(all, s.T / rows + s.B) * (a.Hq / shape.hpw);
    };
    const int64_t slots = 2 * cu_count();
    p.wide[i] = s.max_len > shape.narrow;
    const int64_t n = items(p.wide[i] ? shape.wide : shape.narrow);
    a.splits[i] = (int)std::max<int64_t>(1, std::min<int64_t>((slots + n - 1) / n, s.max_keys / kPartKeys));
    if (a.splits[i] == 1 && n < slots) p.wide[i] = false;
    if (a.splits[i] > 1 || a.prefix.B) parts |= 1 << i;
  }
  a.whole = keys <= kWholeTiles * kStreamTile;
  a.workers = a.whole ? E * a.Hkv : 2 * cu_count();
  a.slot_rows = (int)slot_rows;
  const bool cut = p.stream && !a.whole;
  p.join = a.prefix.B || cut || parts;
  const int64_t state = (int64_t)a.seq.T * a.Hq * kState * 4;
  p.slots = cut ? round256(4 * (1 + (int64_t)E)) : 0;
  p.states = p.slots + (cut ? round256(2 * (int64_t)a.workers * slot_rows * kState * 4) : 0);
  p.parts[0] = p.states + (p.stream && a.prefix.B ? 2 * round256(state) : 0);
  p.parts[1] = p.parts[0] + (parts & 1 ? round256(a.splits[0] * state) : 0);
  p.total = p.parts[1] + (parts & 2 ? round256(a.splits[1] * state) : 0);
  for (int i = 0; i < 2; ++i)
    if (!(parts >> i & 1)) p.parts[i] = -1;
  return p;
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
  const PagedPlan p = plan(a, dtype);
  if (p.total > 0 && (!workspace || workspace_bytes < p.total))
    return set_error(DA_ERR_WORKSPACE, "%s: workspace of %lld bytes required", who, (long long)p.total);
  DA_REQUIRE(((uintptr_t)workspace & 255) == 0, "%s: the workspace must be 256-byte aligned", who);
  char* ws = (char*)workspace;
  a.begin = (uint32_t*)ws;
  a.slots = (float*)(ws + p.slots);
  a.states = (float*)(ws + p.states);
  for (int i = 0; i < 2; ++i) a.parts[i] = p.parts[i] < 0 ? nullptr : (float*)(ws + p.parts[i]);
  hipStream_t st = (hipStream_t)stream;
  if (p.stream)
    if (int rc = launch_paged_stream(a, dtype, st)) return rc;
  for (int i = 0; i < 2; ++i)
    if (p.rows[i])
      if (int rc = launch_paged_rows(a, i ? a.seq : a.prefix, i == 1, p.wide[i], a.splits[i], a.parts[i], dtype, st)) return rc;
  if (!p.join) return DA_OK;
  const dim3 grid((unsigned)T, (unsigned)((Hq + 3) / 4));
  switch (dtype) {
    case DA_BF16: hipLaunchKernelGGL(paged_join_kernel<DA_BF16>, grid, dim3(256), 0, st, a); break;
    case DA_F16: hipLaunchKernelGGL(paged_join_kernel<DA_F16>, grid, dim3(256), 0, st, a); break;
    default: hipLaunchKernelGGL(paged_join_kernel<DA_F32>, grid, dim3(256), 0, st, a);
  }
  return check_launch("paged attention (join)");
}
