// The stream's kernels and their launches (da_paged_stream.hpp).
#include "da_paged_stream.hpp"

namespace da {

template <int DT, int STAGES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(3 - STAGES, 3 - STAGES)))
void paged_stream_kernel(PagedAttnArgs a) {
  stream_worker<DT, STAGES>(a, blockIdx.x);
}

// The parts of the stream's items joined, by the worker that has the first: a row's 128 dims over 32
// lanes, eight rows at a time.
template <int DT>
__global__ __launch_bounds__(256) void paged_stream_join_kernel(PagedAttnArgs a) {
  const StreamRecord rec = a.records[blockIdx.x];
  if (blockIdx.x * a.begin[0] >= a.begin[1 + a.prefix.B + a.seq.B] || rec.others == 0) return;
  const int d = 4 * (threadIdx.x & 31);
  for (int r = threadIdx.x >> 5; r < rec.tokens * a.G; r += 8) {
    RowSum sum;
    sum.take(a.slots + ((int64_t)rec.slot * a.slot_rows + r) * kState, d);
    const float* next = a.slots + (2 * ((int64_t)blockIdx.x + 1) * a.slot_rows + r) * kState;
    sum.take_all(next, 2 * (int64_t)a.slot_rows * kState, min(rec.others, a.workers - 1 - (int)blockIdx.x), d);
    sum.template store<DT>(a, rec.first + r / a.G, rec.head * a.G + r % a.G, d);
  }
}

template <int DT, int STAGES>
static int launch_stream_t(const PagedAttnArgs& a, hipStream_t st) {
  static bool done[kMaxDevices] = {};
  if (int rc = allow_lds(reinterpret_cast<const void*>(&paged_stream_kernel<DT, STAGES>), stream_lds(STAGES), done)) return rc;
  hipLaunchKernelGGL((paged_stream_kernel<DT, STAGES>), dim3((unsigned)a.workers), dim3(256), stream_lds(STAGES), st, a);
  return check_launch("paged attention (stream)");
}

int launch_paged_stream_join(const PagedAttnArgs& a, int dtype, hipStream_t st) {
  const dim3 grid((unsigned)a.workers);
  if (dtype == DA_F16) hipLaunchKernelGGL(paged_stream_join_kernel<DA_F16>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(paged_stream_join_kernel<DA_BF16>, grid, dim3(256), 0, st, a);
  return check_launch("paged attention (stream, join)");
}

int launch_paged_stream(const PagedAttnArgs& a, int dtype, hipStream_t st) {
  const bool two = a.whole && a.workers <= cu_count();
  if (dtype == DA_F16) return two ? launch_stream_t<DA_F16, 2>(a, st) : launch_stream_t<DA_F16, 1>(a, st);
  return two ? launch_stream_t<DA_BF16, 2>(a, st) : launch_stream_t<DA_BF16, 1>(a, st);
}

}  // namespace da
