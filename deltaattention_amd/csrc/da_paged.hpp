// Pages and sequences of the paged cache, as the kernels see them (include/deltaattn_paged.h).
#pragma once

#include "../../include/deltaattn_paged.h"
#include "da_common.hpp"

namespace da {

struct Pages {
  const char* k;
  const char* v;
  int64_t sk_p, sk_h, sk_n;  // elements
  int64_t sv_p, sv_h, sv_n;
  int num_pages, shift;  // page size 1 << shift
};

// The sequences of a call; everything read from memory is clamped to what the tensors hold, but for the slot
// of a token, which is what lengths and cu say, in the table or not.
struct PageBatch {
  const int32_t* table;
  const int32_t* lengths;
  const int32_t* cu;
  const int32_t* start;
  int64_t table_stride;
  int B, T, max_len, max_keys;  // max_keys: width << shift
  __device__ __forceinline__ int first(int b) const {
    if (!cu) return b;
    const int s = cu[b];
    return s < 0 ? 0 : (s > T ? T : s);
  }
  // tokens that sequence b brings
  __device__ __forceinline__ int tokens(int b) const {
    if (!cu) return 1;
    const int s = first(b);
    int e = cu[b + 1];
    e = e < s ? s : (e > T ? T : e);
    return e - s > max_len ? max_len : e - s;
  }
  // tokens in its pages
  __device__ __forceinline__ int keys(int b) const {
    const int n = lengths[b];
    return n < 0 ? 0 : (n > max_keys ? max_keys : n);
  }
  // the slot of token t of sequence b: its new tokens are the last of all it has
  __device__ __forceinline__ int64_t slot(int b, int t) const {
    return (int64_t)lengths[b] + t - (cu ? (int64_t)cu[b + 1] : b + 1);
  }
  // that of its first token, within 2^30 to either side, which is farther than any key
  __device__ __forceinline__ int before(int b) const {
    const int64_t n = slot(b, first(b));
    return n < -(1 << 30) ? -(1 << 30) : n > (1 << 30) ? 1 << 30 : (int)n;
  }
};

// The sequence of token t, for a whole wave (t uniform): the last b with cu[b] <= t, -1 for a token
// before cu[0] or from cu[B] on.  Each round a wave looks at 64 places of the range that is left.  Of a cu that
// does not rise it may be another one or -1, but never one that begins after t.
__device__ __forceinline__ int sequence_of(const PageBatch& s, int t, int lane) {
  if (!s.cu) return t < s.B ? t : -1;
  int lo = 0, n = s.B + 1;  // cu[lo .. lo + n) holds the border
  while (n > 0) {
    const int step = (n + 63) >> 6;
    const int i = lo + lane * step;
    const bool before = lane * step < n && s.cu[i] <= t;
    const uint64_t all = __ballot(before);
    const int c = __popcll(all);
    if (c == 0) return -1;
    const int at = lo + (c - 1) * step;
    if (step == 1) return at < s.B && (all >> (c - 1) & 1) ? at : -1;
    n = min(step, lo + n - at);
    lo = at;
  }
  return -1;
}

// A call of paged attention.  A list is the batch's own sequences or the groups of a shared prefix;
// an item is the queries that one list entry brings to one KV head, its rows are (token, query head of
// the group) in that order.  Entries of up to kStreamRows rows are `short`: their items' keys go as one
// stream over the chip (da_paged_stream.hpp).
constexpr int kStreamRows = 32;

// An item that several workers of the stream share, kept by the one with its first part.
struct StreamRecord {
  int first, tokens, head;  // the entry's first token and its tokens, the KV head
  int slot, others;         // the first part's slot; the parts after it, each in the next worker's first slot
};

struct PagedAttnArgs {
  const char* q;
  char* out;
  int64_t sq_t, sq_h, so_t, so_h;
  int Hq, Hkv, G, D;
  float scale_log2;  // softmax scale * log2(e)
  Pages pages;
  PageBatch seq, prefix;  // prefix.B = 0: none
  int short_rows[2];  // of both lists ([0] the prefix, [1] the sequences): entries of up to so many
                      // rows are the stream's
  // stream
  int workers;       // workgroups of the stream
  int whole;         // 1: no item is split
  int slot_rows;     // rows of a slot
  uint32_t* begin;   // [2 + entries]: tiles a worker, the entries' first tiles, all tiles
  StreamRecord* records;  // [workers], where the stream's items are joined by themselves, or null
  float* slots;      // [2 workers][slot_rows][kState]: parts of items, two a worker
  float* states;     // [2 lists][T][Hq][kState], with a prefix: results of unsplit items
  // entries with more rows: their items' keys in so many parts, by list
  int splits[2];
  float* parts[2];   // [splits][T][Hq][kState], or null: the result is in out
};
// a row's result before it is joined: D sums padded to 128, the maximum (log2 units), the sum of weights
constexpr int kState = 132;
constexpr int kStreamTile = 128;  // keys

// The sequences or the prefix's groups, field by field (a reference to either would put the kernel's
// arguments into memory).
__device__ __forceinline__ PageBatch list_of(const PagedAttnArgs& a, bool own) {
  const PageBatch &x = a.seq, &y = a.prefix;
  return PageBatch{own ? x.table : y.table, own ? x.lengths : y.lengths, own ? x.cu : y.cu, own ? x.start : y.start,
                   own ? x.table_stride : y.table_stride, own ? x.B : y.B, own ? x.T : y.T, own ? x.max_len : y.max_len,
                   own ? x.max_keys : y.max_keys};
}

// tiles of an item of the stream; a sequence that sees nothing has one, which writes its zeros
__device__ __forceinline__ int stream_tiles(const PagedAttnArgs& a, int tokens, int keys, bool own) {
  if (tokens == 0 || tokens * a.G > (own ? a.short_rows[1] : a.short_rows[0])) return 0;
  const int n = (keys + kStreamTile - 1) / kStreamTile;
  return own && n == 0 ? 1 : n;
}

// Four dims d .. d + 3 of a row's sums, and the row's maximum and sum of weights, over parts.
struct RowSum {
  float M = -INFINITY, L = 0.0f;
  f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
  __device__ __forceinline__ void add(f32x2 ml, f32x4 z) {
    const float mn = __builtin_fmaxf(M, ml[0]), ref = mn == -INFINITY ? 0.0f : mn;
    const float fo = __builtin_amdgcn_exp2f(M - ref), fn = __builtin_amdgcn_exp2f(ml[0] - ref);
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = y[i] * fo + z[i] * fn;
    L = L * fo + ml[1] * fn;
    M = mn;
  }
  __device__ __forceinline__ void take(const float* state, int d) { add(*(const f32x2*)(state + 128), *(const f32x4*)(state + d)); }
  // n states `step` floats apart, four in flight
  __device__ __forceinline__ void take_all(const float* state, int64_t step, int n, int d) {
    for (int i = 0; i < n; i += 4) {
      f32x2 ml[4];
      f32x4 z[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // past the last: read again, left out
        const float* p = state + min(i + j, n - 1) * step;
        ml[j] = *(const f32x2*)(p + 128);
        z[j] = *(const f32x4*)(p + d);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i + j < n) add(ml[j], z[j]);
    }
  }
  template <int DT>
  __device__ __forceinline__ void store(const PagedAttnArgs& a, int token, int head, int d) const {
    if (d >= a.D) return;
    const float inv = L > 0.0f ? 1.0f / L : 0.0f;
    const int64_t at = token * a.so_t + head * a.so_h + d;
    if constexpr (DT == DA_F32) *(f32x4*)(a.out + 4 * at) = f32x4{y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv};
    else *(u32x2*)(a.out + 2 * at) = u32x2{E16<DT>::pack(y[0] * inv, y[1] * inv), E16<DT>::pack(y[2] * inv, y[3] * inv)};
  }
};

// Lets a kernel use more than 64 KiB of dynamic LDS on the current device (once a device).
constexpr int kMaxDevices = 64;
int allow_lds(const void* kernel, int bytes, bool (&done)[kMaxDevices]);
// Host: checks and the kernels' forms of the ABI's blocks.
int fill_pages(Pages& p, const DaPagedKV* kv, int64_t D, const char* who);
// Rows of a KV head, (token, query head of the group), that a workgroup of the row kernels takes: a
// half-size or full-size group.
struct RowsShape {
  int narrow, wide;
};
RowsShape paged_rows_shape(int dtype);
// The entries of `list` with more than short_rows rows; with_stream (not for fp32): and the stream.
int launch_paged_rows(const PagedAttnArgs& p, const PageBatch& list, bool own, bool wide, int splits, float* parts,
                      bool with_stream, int dtype, hipStream_t st);
int launch_paged_stream_join(const PagedAttnArgs& a, int dtype, hipStream_t st);
int launch_paged_stream(const PagedAttnArgs& a, int dtype, hipStream_t st);
int fill_batch(PageBatch& s, const DaPagedBatch* b, const Pages& p, int64_t T, const char* who);

}  // namespace da
