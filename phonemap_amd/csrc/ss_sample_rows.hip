// ss_sample_rows.hip - the next token of every row of logits, from given random
// numbers.
//
// With x the logits of a row, M their maximum and T the temperature, entry i has
// the weight w_i = e^((x_i - M) / T) (NaN counts as -inf). What stays are the
// entries with x_i >= the k-th largest x (top-k), x_i >= the largest v at which
// the weights of the entries >= v reach top_p of all weights (top-p), and
// w_i >= min_p: three thresholds on x, so equal logits stay or go together and
// the order of the filters does not matter. The token is the first i at which
// the running sum of the weights that stay exceeds u times their sum.
//
// Weights are formed in 64 bits and summed as whole multiples of 2^-44, so no
// sum depends on the order of its terms and a draw falls to the same entry
// whatever the split: in 32 bits the running sums of a 128256-entry row are off
// by some 1e-8, and one row in a thousand would take a neighbouring entry.

#include "ss_device.h"
#include "ss_kernels.h"

namespace ssk {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr double kOne = 17592186044416.0;   // 2^44, the weight of the maximum

// unsigned key that orders like the value; NaN as -inf, -0 as 0
__device__ __forceinline__ uint32_t order(float x) {
  if (x != x) x = -INFINITY;
  const uint32_t b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// x - M, in 64 bits: 0 for the maximum (an infinite one too), -inf for NaN
__device__ __forceinline__ double gap(float x, float mx) {
  return x == mx ? 0.0 : x == x ? (double)x - (double)mx : -INFINITY;
}
__device__ __forceinline__ uint64_t weight(double g, double temperature) {
  return (uint64_t)(exp(g / temperature) * kOne + 0.5);
}
// u * total as a whole multiple, below total; u outside [0, 1) counts as the nearest end
__device__ __forceinline__ uint64_t draw_target(float u, uint64_t total) {
  if (!(u > 0.f)) return 0;
  const uint64_t t = u < 1.f ? (uint64_t)((double)u * (double)total) : total;
  return t < total ? t : total - 1;
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
// over the workgroup, in every thread
__device__ uint64_t group_sum(uint64_t v, uint64_t* red) {
  v = wave_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t t = 0;
  for (int w = 0; w < kWaves; ++w) t += red[w];
  return t;
}

// The largest key at which the sum of val(i) over the entries with that key or a
// greater one reaches target, 0 when all entries together do not; 8 bits of the
// key at a time.
template <class Val>
__device__ uint32_t key_reaching(const float* x, int V, uint64_t target, uint64_t* hist, uint64_t* carry, Val val) {
  uint32_t prefix = 0, mask = 0;
  uint64_t above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kThreads) {
      const uint32_t k = order(x[i]);
      if ((k & mask) == prefix) atomicAdd(reinterpret_cast<unsigned long long*>(&hist[(k >> shift) & 255u]), (unsigned long long)val(x[i]));
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      int b = 255;
      for (; b >= 0; --b) {
        if (above + hist[b] >= target) break;
        above += hist[b];
      }
      carry[0] = above;
      carry[1] = (uint64_t)(int64_t)b;
    }
    __syncthreads();
    above = carry[0];
    const int b = (int)(int64_t)carry[1];
    if (b < 0) return 0;
    prefix |= (uint32_t)b << shift;
    mask |= 255u << shift;
  }
  return prefix;
}

// One row by one workgroup.
__global__ void __launch_bounds__(kThreads) k_row(const SampleRowsArgs a) {
  __shared__ uint64_t red[kWaves], hist[256], carry[2];
  __shared__ uint32_t top;
  __shared__ int found;
  const int tid = threadIdx.x, V = a.V;
  const float* x = a.logits + (size_t)blockIdx.x * a.ld;
  if (tid == 0) {
    top = 0;
    found = 0x7fffffff;
  }
  __syncthreads();
  uint32_t mk = 0;
  for (int i = tid; i < V; i += kThreads) mk = max(mk, order(x[i]));
  atomicMax(&top, mk);
  __syncthreads();
  mk = top;
  const float mx = from_order(mk);
  if (mx == -INFINITY) {   // nothing to choose from
    if (tid == 0) a.out[blockIdx.x] = -1;
    return;
  }
  auto w = [&](float v) { return weight(gap(v, mx), a.temperature); };
  uint32_t least = mk;   // the least key that stays
  if (a.temperature > 0.0) {
    least = 0;
    if (a.top_k > 0 && a.top_k < V) least = key_reaching(x, V, (uint64_t)a.top_k, hist, carry, [](float) { return 1ull; });
    if (a.top_p < 1.0) {
      uint64_t s = 0;
      for (int i = tid; i < V; i += kThreads) s += w(x[i]);
      const double t = a.top_p * (double)group_sum(s, red);
      least = max(least, key_reaching(x, V, max((uint64_t)ceil(t), (uint64_t)1), hist, carry, w));
    }
  }
  auto kept = [&](float v) { return order(v) >= least && gap(v, mx) >= a.min_gap ? (a.temperature > 0.0 ? w(v) : (uint64_t)kOne) : 0ull; };
  // contiguous chunks: the thread in whose chunk the running sum passes the draw
  const int C = (V + kThreads - 1) / kThreads, i0 = min(tid * C, V), i1 = min(i0 + C, V);
  uint64_t s = 0;
  for (int i = i0; i < i1; ++i) s += kept(x[i]);
  uint64_t incl = s;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const uint64_t o = __shfl_up(incl, off, kWave);
    if ((tid & 63) >= off) incl += o;
  }
  __syncthreads();
  if ((tid & 63) == 63) red[tid >> 6] = incl;
  __syncthreads();
  uint64_t before = incl - s, total = 0;
  for (int i = 0; i < kWaves; ++i) {
    if (i < tid >> 6) before += red[i];
    total += red[i];
  }
  const uint64_t target = a.temperature > 0.0 ? draw_target(a.u[blockIdx.x], total) : 0;
  if (before <= target && target < before + s) {   // one thread
    int i = i0;
    for (uint64_t c = before + kept(x[i]); c <= target; c += kept(x[i])) ++i;
    found = i;
  }
  __syncthreads();
  if (tid == 0) a.out[blockIdx.x] = found;
}

}  // namespace

hipError_t launch_sample_rows(const SampleRowsArgs& a, hipStream_t s) {
  if (a.rows < 1 || a.V < 1 || a.V > kSampleRowsMaxV) return hipErrorInvalidValue;
  hipLaunchKernelGGL(k_row, dim3(a.rows), dim3(kThreads), 0, s, a);
  return hipGetLastError();
}

}  // namespace ssk
