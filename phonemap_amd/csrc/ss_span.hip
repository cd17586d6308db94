// ss_span.hip - attention over a sliding window with first tokens that stay
// visible, and of several sequences over a prefix they share (ss_span.h).

#include "ss_span.h"

namespace ssk {
namespace {

constexpr int kRowWaves = 4;

// one wave per row and query head
template <int HD, int KVT>
__global__ void __launch_bounds__(kRowWaves * 64) k_span_rows(const SpanArgs a, int group) {
  const int nh = a.n_kv_heads * group;
  const int64_t row = (int64_t)blockIdx.x * kRowWaves + (threadIdx.x >> 6);
  if (row >= (int64_t)a.n * nh) return;
  const int t = (int)(row / nh), h = (int)(row % nh);
  Span s[2];
  row_spans<HD, KVT>(a, t, h / group, s);
  span_row<HD, KVT>(a, a.q + (size_t)row * HD, a.out + (size_t)row * HD, s);
}

template <int HD>
hipError_t launch_hd(int group, int kv_type, const SpanArgs& a, hipStream_t s) {
  const int64_t rows = (int64_t)a.n * a.n_kv_heads * group, wgs = (rows + kRowWaves - 1) / kRowWaves;
  if (wgs > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs), block(kRowWaves * 64);
  if (kv_type)
    hipLaunchKernelGGL((k_span_rows<HD, 1>), grid, block, 0, s, a, group);
  else
    hipLaunchKernelGGL((k_span_rows<HD, 0>), grid, block, 0, s, a, group);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_span(int head_dim, int group, int kv_type, const SpanArgs& a, hipStream_t s) {
  if (head_dim == 64) return launch_hd<64>(group, kv_type, a, s);
  if (head_dim == 128) return launch_hd<128>(group, kv_type, a, s);
  if (head_dim == 256) return launch_hd<256>(group, kv_type, a, s);
  return hipErrorInvalidValue;
}

}  // namespace ssk
