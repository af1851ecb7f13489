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

// The sequences of a call; everything read from memory is clamped to what the tensors hold.
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
};

// The sequence of token t, for a whole wave (t uniform): the last b with cu[b] <= t, -1 for a token
// before cu[0] or from cu[B] on.  Each round a wave looks at 64 places of the range that is left.
__device__ __forceinline__ int sequence_of(const PageBatch& s, int t, int lane) {
  if (!s.cu) return t < s.B ? t : -1;
  int lo = 0, n = s.B + 1;  // cu[lo .. lo + n) holds the border
  while (n > 0) {
    const int step = (n + 63) >> 6;
    const int i = lo + lane * step;
    const bool before = lane * step < n && s.cu[i] <= t;
    const int c = __popcll(__ballot(before));
    if (c == 0) return -1;
    const int at = lo + (c - 1) * step;
    if (step == 1) return at < s.B ? at : -1;
    n = min(step, lo + n - at);
    lo = at;
  }
  return -1;
}

// Host: checks and the kernels' forms of the ABI's blocks.
int fill_pages(Pages& p, const DaPagedKV* kv, int64_t D, const char* who);
int fill_batch(PageBatch& s, const DaPagedBatch* b, const Pages& p, int64_t T, const char* who);

}  // namespace da
