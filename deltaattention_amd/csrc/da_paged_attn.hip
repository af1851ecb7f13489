// Attention of new tokens over a paged cache (include/deltaattn_paged.h): which kernel takes which
// entries, and the parts of a result joined.
//
// An entry (a sequence, or a group behind a prefix) of up to kStreamRows rows goes to the stream
// (da_paged_stream.hpp); one with more rows, and all of fp32, to the row kernels (da_attn.hip's, over
// pages), whose items are blocks of rows and, where those do not fill the chip, runs of keys.
// A prefix is a list of its own, seen whole by all rows of a group at once: its keys are read once for
// the group, and each row's result is joined with that of its own sequence.
#include <algorithm>
#include <cmath>

#include "da_paged.hpp"
#include "da_tile.hpp"

namespace da {

// The parts of every row joined: a row's 128 dims over 32 lanes, eight rows of a token a workgroup; or,
// with WIDE, where rows are few, one row, whose parts eight half-waves share.
template <int DT, bool WIDE>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedAttnArgs a) {
  __shared__ float s_sum[WIDE ? 8 : 1][kState];
  const int lane = threadIdx.x & 63, t = blockIdx.x, d = 4 * (threadIdx.x & 31), half = threadIdx.x >> 5;
  const int h = WIDE ? blockIdx.y : blockIdx.y * 8 + half;
  const int entry[2] = {a.prefix.B ? sequence_of(a.prefix, t, lane) : -1, sequence_of(a.seq, t, lane)};
  if (entry[1] < 0 || h >= a.Hq) return;
  const int g = h / a.G;
  const int first = WIDE ? half : 0, by = WIDE ? 8 : 1;  // this half-wave's parts
  RowSum sum;
  for (int list = 0; list < 2; ++list) {
    const PageBatch& s = list ? a.seq : a.prefix;
    const int e = entry[list];
    if (e < 0) continue;
    const int tokens = s.tokens(e), i = t - s.first(e);
    if (i >= tokens) return;  // past max_seqlen: left as it is
    const float* state;
    int64_t step = 0;
    int n = 1;
    if (tokens * a.G > a.short_rows[list]) {  // the row kernels'
      if (!a.parts[list]) return;
      state = a.parts[list] + ((int64_t)t * a.Hq + h) * kState;
      step = (int64_t)s.T * a.Hq * kState;
      n = a.splits[list];
    } else {
      const int tiles = stream_tiles(a, tokens, s.keys(e), list);
      if (tiles == 0) continue;
      const uint32_t per = a.whole ? 1 : a.begin[0];
      const uint32_t U = a.whole ? 0 : a.begin[1 + (list ? a.prefix.B : 0) + e] + g * tiles;
      const uint32_t last = a.whole ? 0 : a.workers - 1;
      const uint32_t w0 = min(U / per, last), w1 = min((U + tiles - 1) / per, last);
      if (w0 == w1) {
        if (a.prefix.B == 0) return;  // written where it was computed
        state = a.states + (((int64_t)list * a.seq.T + t) * a.Hq + h) * kState;
      } else {
        // the first part may be its worker's last segment; the others are their workers' first
        const int r = i * a.G + h - g * a.G;
        if (first == 0) sum.take(a.slots + ((int64_t)(2 * w0 + (U != w0 * per ? 1 : 0)) * a.slot_rows + r) * kState, d);
        state = a.slots + (2 * ((int64_t)w0 + 1) * a.slot_rows + r) * kState;
        step = 2 * (int64_t)a.slot_rows * kState;
        n = w1 - w0;
      }
    }
    if (first < n) sum.take_all(state + first * step, by * step, (n - first + by - 1) / by, d);
  }
  if constexpr (WIDE) {
    *(f32x4*)(&s_sum[half][d]) = sum.y;
    if (d == 0) *(f32x2*)(&s_sum[half][128]) = f32x2{sum.M, sum.L};
    __syncthreads();
    if (half > 0) return;
    for (int i = 1; i < 8; ++i) sum.take(s_sum[i], d);
  }
  sum.template store<DT>(a, t, h, d);
}

template <int DT>
static int launch_join(const PagedAttnArgs& a, hipStream_t st) {
  const int T = a.seq.T;
  if ((int64_t)T * a.Hq <= 8 * cu_count())
    hipLaunchKernelGGL((paged_join_kernel<DT, true>), dim3((unsigned)T, (unsigned)a.Hq), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((paged_join_kernel<DT, false>), dim3((unsigned)T, (unsigned)((a.Hq + 7) / 8)), dim3(256), 0, st, a);
  return check_launch("paged attention (join)");
}

// The stream's items are not split (one launch, a workgroup an item) up to 6 tiles, and up to 16 where
// the items fill half the CUs.  One sequence of 8 heads: 400 keys 12.1 us against 11.8 split, 600 13.4 / 12.3,
// 1000 17.2 / 12.9, where a second launch costs the caller 4; 16 sequences: 600 keys 15.7 / 20.9, 2000
// 28.7 / 32.2; 64: 2000 96.5 / 98.4.
static bool stream_whole(int64_t items, int keys) {
  const int tiles = (keys + kStreamTile - 1) / kStreamTile;
  return tiles <= 6 || (tiles <= 16 && 2 * items >= cu_count());
}

// Rows of a head that a workgroup of the row kernels takes, and into how many runs it cuts the keys:
// the least of an estimate.  A run's time is its 32-key tiles times a tile's (us, measured with up to
// one workgroup a CU and with two), and 3 us to begin and end; parts cost their writing and reading,
// 3.5 TB/s, and a launch.  512 tokens of 32 heads after 5000: narrow 1 part 141 us, 4 parts 72, 8 82, wide 8 75;
// 2048 after 30011: narrow 998, wide 1204, 2 parts 903, 4 924; 512 at a sequence's start: 1 part 21, 2 31.
// `paired`: beside the stream, whose loads slow a tile and the parts' writing (1.5 TB/s).  Over 188 batches
// (16 to 300 sequences of 60 to 3000 keys behind 700 to 100000, five sets of heads) the choice costs 2%
// more than the best, 17% at most: 130 sequences of 60 keys behind 100000, 64 heads: narrow 6 parts 523 us,
// wide 24 473, wide 6 672.
static void shape_rows(PagedAttnArgs& a, int list, bool& wide, bool paired, int dtype) {
  const PageBatch& s = list ? a.seq : a.prefix;
  const RowsShape shape = paged_rows_shape(dtype);
  const double part = (double)s.T * a.Hq * kState * 8 / (paired ? 1.5e6 : 3.5e6), slots = 2.0 * cu_count();
  const int tiles = (s.max_keys + 31) / 32, dims = (a.D + 31) / 32;
  double best = 0.0;
  const int64_t most = (int64_t)s.max_len * a.G, others = s.B - 1, rest = s.T - s.max_len;
  for (int w = 0; w < (shape.wide > shape.narrow && most > shape.narrow ? 2 : 1); ++w) {
    const int rows = w ? shape.wide : shape.narrow;
    // items: those of the longest entry, and of the others if their mean is not the stream's
    const int64_t longest = (most + rows - 1) / rows;
    int64_t items = longest;
    if (others > 0 && rest * a.G > others * a.short_rows[list])
      items += std::min(others * longest, rest * a.G / rows + others);
    items *= a.Hkv;
    for (int n : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64}) {
      if (n > 1 && n > tiles) break;
      const double all = (double)items * n, rounds = all <= slots ? 1.0 : all / slots + 0.3;
      const bool two = 2 * all > slots;
      const double tile = dtype == DA_F32 ? (two ? 0.4 + 0.75 * dims : 0.25 + 0.39 * dims)
                          : paired         ? (w ? 1.2 : 0.9) * (two ? 1.5 : 1.0)
                                           : w ? (two ? 1.75 : 1.22) : (two ? 1.0 : 0.78);
      const double time = rounds * ((tiles + n - 1) / n * tile + 3.0) + (n > 1 || a.prefix.B ? n * part + (n > 1 ? 5 : 0) : 0.0);
      if ((w == 0 && n == 1) || time < best) best = time, wide = w, a.splits[list] = n;
    }
  }
}

struct PagedPlan {
  bool stream, rows[2], wide[2], join;
  int64_t records, slots, states, parts[2], total;  // byte offsets in the workspace
};
// The rows of a prefix and the stream run in one launch: both wait for memory most of the time (16 sequences
// behind 32768 tokens 43.8 us, apart 48.4).  A prompt's rows want both workgroups of a CU to themselves (512
// tokens beside 15 decoding sequences 131 us together, 117 apart).
static bool paired_rows(const PagedPlan& p, int list) { return list == 0 && p.stream; }
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
  }
  for (int i = 0; i < 2; ++i) {
    if (!p.rows[i]) continue;
    shape_rows(a, i, p.wide[i], paired_rows(p, i), dtype);
    if (a.splits[i] > 1 || a.prefix.B) parts |= 1 << i;
  }
  // a workgroup an item needs a launch of less than 2^32 threads
  a.whole = stream_whole((int64_t)E * a.Hkv, keys) && (int64_t)E * a.Hkv < (1ll << 24);
  a.workers = a.whole ? E * a.Hkv : 2 * cu_count();
  a.slot_rows = (int)slot_rows;
  const bool cut = p.stream && !a.whole;
  p.join = a.prefix.B || parts;  // else the stream joins its own parts
  const int64_t state = (int64_t)a.seq.T * a.Hq * kState * 4;
  p.records = cut ? round256(4 * (2 + (int64_t)E)) : 0;
  p.slots = p.records + (cut && !p.join ? round256(a.workers * (int64_t)sizeof(StreamRecord)) : 0);
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
  DA_REQUIRE(T * Hq < (1ll << 31), "%s: more than 2^31 rows", who);
  DA_REQUIRE(T < (1ll << 24), "%s: more than 2^24 tokens", who);  // a launch has less than 2^32 threads
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
  a.records = p.join || !p.stream || a.whole ? nullptr : (StreamRecord*)(ws + p.records);
  a.slots = (float*)(ws + p.slots);
  a.states = (float*)(ws + p.states);
  for (int i = 0; i < 2; ++i) a.parts[i] = p.parts[i] < 0 ? nullptr : (float*)(ws + p.parts[i]);
  hipStream_t st = (hipStream_t)stream;
  const bool pair = p.rows[0] && paired_rows(p, 0);
  if (p.stream && !pair)
    if (int rc = launch_paged_stream(a, dtype, st)) return rc;
  for (int i = 0; i < 2; ++i)
    if (p.rows[i])
      if (int rc = launch_paged_rows(a, i ? a.seq : a.prefix, i == 1, p.wide[i], a.splits[i], a.parts[i], pair && i == 0, dtype,
                                     st))
        return rc;
  if (a.records) return launch_paged_stream_join(a, dtype, st);
  if (!p.join) return DA_OK;
  return dtype == DA_BF16 ? launch_join<DA_BF16>(a, st) : dtype == DA_F16 ? launch_join<DA_F16>(a, st) : launch_join<DA_F32>(a, st);
}
