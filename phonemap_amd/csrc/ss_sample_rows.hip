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
//
// The thresholds come from a histogram over bins of x / T a quarter wide, with
// the entries and the weights of each: 128 bins from the maximum's down reach
// e^-31.75, whose weight is 0 (less than half of 2^-44). The highest of the three
// thresholds lies in one bin; what lies above that bin stays, what lies below
// goes, and the bin's own entries are gathered and the threshold found among
// them. A bin with more than kList of them (equal logits), or an x / T past 2^28,
// leaves the row to `slow`, which selects by the bits of x over the whole row.
//
// Rows of up to kOneMax entries: one workgroup with the row in registers, one
// launch. Longer ones: tiles of kTile entries, a launch for their maxima and
// histograms and a launch that gathers; the row's last workgroup to finish that
// (an arrival count that the first launch clears) finds threshold and token.

#include "ss_device.h"
#include "ss_kernels.h"

namespace ssk {
namespace {

constexpr double kOne = 17592186044416.0;   // 2^44, the weight of the maximum
constexpr int kBins = 128;
constexpr int kCopies = 8;                  // of the histogram, one per lane % 8
constexpr int kList = 4096;                 // entries of the threshold's bin
constexpr int kPairs = 160;                 // up to this many are compared each with all
constexpr int kFar = 1 << 28;               // |bin| this large: not told apart

constexpr int kOneThreads = 1024, kOneEach = 32, kOneMax = kOneThreads * kOneEach;
constexpr int kTileThreads = 512, kTileEach = 16, kTile = kTileThreads * kTileEach;
constexpr int kMaxTiles = (kSampleRowsMaxV + kTile - 1) / kTile;

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
// the bin of x (4 / T: quarters of x / T), and e^(x / T - the bin's middle) times 2^44
__device__ __forceinline__ int bin_of(float x, double per) {
  const double b = x == x ? floor((double)x * per) : -INFINITY;
  return (int)fmin(fmax(b, (double)-kFar), (double)kFar);
}
__device__ __forceinline__ uint64_t bin_weight(float x, double per, int b) {
  const double r = 0.25 * ((double)x * per - ((double)b + 0.5));   // |r| <= 1/8: the ninth power is below 2e-14
  double p = 1.0 / 40320;
  p = fma(p, r, 1.0 / 5040);
  p = fma(p, r, 1.0 / 720);
  p = fma(p, r, 1.0 / 120);
  p = fma(p, r, 1.0 / 24);
  p = fma(p, r, 1.0 / 6);
  p = fma(p, r, 0.5);
  p = fma(p, r, 1.0);
  p = fma(p, r, 1.0);
  return (uint64_t)(p * kOne + 0.5);
}

__device__ __forceinline__ uint64_t wave_sum_u64(uint64_t v) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
  return v;
}
// over the workgroup of NT threads, in every thread; red: NT / 64 words
template <int NT>
__device__ uint64_t group_sum(uint64_t v, uint64_t* red) {
  v = wave_sum_u64(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) t += red[w];
  return t;
}
template <int NT>
__device__ uint32_t group_max(uint32_t v, uint64_t* red) {
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, kWave));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t t = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) t = max(t, red[w]);
  return (uint32_t)t;
}
// the sum over the threads before this one; all: over every thread
template <int NT>
__device__ uint64_t sum_before(uint64_t v, uint64_t* red, uint64_t& all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t incl = v;
#pragma unroll
  for (int off = 1; off < kWave; off <<= 1) {
    const uint64_t o = __shfl_up(incl, off, kWave);
    if (lane >= off) incl += o;
  }
  __syncthreads();
  if (lane == 63) red[wave] = incl;
  __syncthreads();
  uint64_t before = incl - v;
  all = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    if (w < wave) before += red[w];
    all += red[w];
  }
  return before;
}
__device__ __forceinline__ void add_u64(uint64_t* p, uint64_t v) {
  atomicAdd(reinterpret_cast<unsigned long long*>(p), (unsigned long long)v);
}

// Selection by the bits of the keys, 8 at a time: the largest key at which the
// sum of val(i) over the entries i < n with that key or a greater one reaches
// target, 0 when all together do not. hist: 256 words, red: NT / 64 + 2.
template <int NT, class Key, class Val>
__device__ uint32_t key_reaching(int n, uint64_t target, uint64_t* hist, uint64_t* red, Key key, Val val) {
  uint32_t prefix = 0, mask = 0;
  uint64_t above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    if (threadIdx.x < 256) hist[threadIdx.x] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += NT) {
      const uint32_t k = key(i);
      if ((k & mask) == prefix) add_u64(&hist[(k >> shift) & 255u], val(i));
    }
    __syncthreads();
    const uint64_t h = threadIdx.x < 256 ? hist[255 - threadIdx.x] : 0;   // thread 0 has the highest digit
    uint64_t all;
    const uint64_t before = above + sum_before<NT>(h, red, all);
    uint64_t* found = red + NT / 64;
    if (threadIdx.x == 0) found[0] = 256;
    __syncthreads();
    if (threadIdx.x < 256 && before < target && before + h >= target) {
      found[0] = 255 - threadIdx.x;
      found[1] = before;
    }
    __syncthreads();
    if (found[0] == 256) return 0;
    prefix |= (uint32_t)found[0] << shift;
    mask |= 255u << shift;
    above = found[1];
  }
  return prefix;
}

// What stays, and with which weight.
struct Keep {
  uint32_t least;   // the least key
  float mx;
  double temperature, min_gap;
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (order(x) < least) return 0;
    const double g = gap(x, mx);
    return g >= min_gap ? weight(g, temperature) : 0;
  }
};

// ---- a row's entries in the registers of a workgroup ---------------------------
// x[4k + j] of thread t is entry i0 + 4 (k * NT + t) + j (-inf past the row)
template <int NT, int E>
struct Chunk {
  float x[E];
  __device__ __forceinline__ static int at(int k, int j) { return 4 * (k * NT + (int)threadIdx.x) + j; }
  __device__ __forceinline__ void load(const float* row, int i0, int V) {
#pragma unroll
    for (int k = 0; k < E / 4; ++k) {
      const int i = i0 + at(k, 0);
      if (i + 4 <= V) {
        __builtin_memcpy(&x[4 * k], row + i, 16);   // (rows start on any multiple of 4 bytes)
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * k + j] = i + j < V ? row[i + j] : -INFINITY;
      }
    }
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) m = max(m, order(x[e]));
    return m;
  }
  // The entry at which the running sum of what stays passes target, given the sum
  // before these; -1: not among them. sum: of these. red: NT / 64 + 2 words.
  __device__ int pick(const Keep& keep, uint64_t before, uint64_t target, bool whole, float u, uint64_t* part, uint64_t* red) {
    constexpr int K = E / 4;
    // sums of the K rounds of 4 NT entries
    for (int k = threadIdx.x; k < K; k += NT) part[k] = 0;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < K; ++k) {
      uint64_t s = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) s += keep(x[4 * k + j]);
      s = wave_sum_u64(s);
      if ((threadIdx.x & 63) == 0 && s) add_u64(&part[k], s);
    }
    __syncthreads();
    if (whole) {   // the row is these entries: the draw goes by their sum
      uint64_t total = 0;
      for (int k = 0; k < K; ++k) total += part[k];
      target = draw_target(u, total);
    }
    int kf = -1;
    uint64_t at_k = before;
    for (int k = 0; k < K; ++k) {
      if (kf < 0 && target < at_k + part[k]) kf = k;
      if (kf < 0) at_k += part[k];
    }
    if (kf < 0) return -1;   // (uniform)
    uint64_t w[4] = {}, s = 0;
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (k == kf) {
#pragma unroll
        for (int j = 0; j < 4; ++j) s += w[j] = keep(x[4 * k + j]);
      }
    uint64_t all;
    uint64_t c = at_k + sum_before<NT>(s, red, all);
    int* found = reinterpret_cast<int*>(red + NT / 64);
    if (c <= target && target < c + s) {   // one thread
      int j = 0;
      while (c + w[j] <= target) c += w[j++];
      *found = at(kf, j);
    }
    __syncthreads();
    return *found;
  }
};

// ---- the thresholds --------------------------------------------------------------
// Where the highest of the thresholds lies, from the bins' entries and weights.
struct Edge {
  int bin;             // of the threshold (the one below all kBins: everything stays)
  uint64_t need_k;     // entries of that bin that stay by top-k (0: no limit there)
  uint64_t need_p;     // weight of that bin, as bin_weight, at which top-p cuts (0: none there)
};
struct Bins {
  uint64_t weight[kBins];   // [top - bin]
  uint32_t count[kBins];
};

// by the first wave, from bins in LDS; lane l has bins l and 64 + l
__device__ __forceinline__ Edge find_edge(const SampleRowsArgs& a, const Bins& h, int top, float mx, double per) {
  const int lane = threadIdx.x & 63;
  int kb = kBins, pb = kBins;
  uint64_t need_k = 0, need_p = 0;
  if (a.top_k) {
    uint64_t base = 0;
    for (int half = 0; half < 2 && kb == kBins; ++half) {
      const uint64_t c = h.count[64 * half + lane];
      uint64_t incl = c;
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const uint64_t o = __shfl_up(incl, off, kWave);
        if (lane >= off) incl += o;
      }
      incl += base;
      const uint64_t hit = __ballot(incl >= (uint64_t)a.top_k);
      if (hit) {
        const int l = __ffsll((unsigned long long)hit) - 1;
        kb = 64 * half + l;
        need_k = a.top_k - __shfl(incl - c, l, kWave);
      }
      base = __shfl(incl, 63, kWave);
    }
  }
  if (a.top_p < 1.0) {
    // in units of the top bin's middle
    double m[2], incl[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      m[half] = (double)h.weight[64 * half + lane] * exp(-0.25 * (64 * half + lane));
      incl[half] = m[half];
#pragma unroll
      for (int off = 1; off < kWave; off <<= 1) {
        const double o = __shfl_up(incl[half], off, kWave);
        if (lane >= off) incl[half] += o;
      }
    }
    incl[1] += __shfl(incl[0], 63, kWave);
    const double goal = a.top_p * __shfl(incl[1], 63, kWave);
    for (int half = 0; half < 2 && pb == kBins; ++half) {
      const uint64_t hit = __ballot(incl[half] >= goal);
      if (hit) {
        const int l = __ffsll((unsigned long long)hit) - 1;
        pb = 64 * half + l;
        const double above = __shfl(incl[half] - m[half], l, kWave);
        const uint64_t whole = __shfl((unsigned long long)h.weight[64 * half + lane], l, kWave);
        need_p = min((uint64_t)fmax(ceil((goal - above) * exp(0.25 * pb)), 1.0), whole);
      }
    }
  }
  int mb = kBins;
  if (a.min_gap > -INFINITY) {
    const double b = floor(((double)mx + a.min_gap) * per);
    mb = b <= (double)top - kBins ? kBins : b >= (double)top ? 0 : top - (int)b;
  }
  const int r = min(min(kb, pb), mb);
  Edge e;
  e.bin = top - r;
  e.need_k = kb == r ? need_k : 0;
  e.need_p = pb == r ? need_p : 0;
  return e;
}

// The least key that stays, among the n entries of the threshold's bin (v: their
// logits, in LDS): a thread of the workgroup for each, or selection by bits.
template <int NT>
__device__ uint32_t least_of(const Edge& e, const float* v, int n, double per, uint64_t* hist, uint64_t* red, uint32_t* least) {
  if (n <= kPairs) {
    __syncthreads();
    if (threadIdx.x == 0) *least = 0;
    __syncthreads();
    if ((int)threadIdx.x < n) {
      const float x = v[threadIdx.x];
      uint64_t ge = 0, gt = 0, wge = 0, wgt = 0;   // entries and weights at or above x, and above
      for (int j = 0; j < n; ++j) {
        const float y = v[j];
        const uint64_t w = e.need_p && y >= x ? bin_weight(y, per, e.bin) : 0;
        ge += y >= x;
        gt += y > x;
        wge += w;
        wgt += y > x ? w : 0;
      }
      uint32_t k = 0;
      if (e.need_k && gt < e.need_k && ge >= e.need_k) k = order(x);
      if (e.need_p && wgt < e.need_p && wge >= e.need_p) k = max(k, order(x));
      if (k) atomicMax(least, k);
    }
    __syncthreads();
    return *least;
  }
  uint32_t k = 0;
  if (e.need_k) k = key_reaching<NT>(n, e.need_k, hist, red, [&](int i) { return order(v[i]); }, [](int) { return 1ull; });
  if (e.need_p)
    k = max(k, key_reaching<NT>(n, e.need_p, hist, red, [&](int i) { return order(v[i]); },
                                [&](int i) { return bin_weight(v[i], per, e.bin); }));
  return k;
}

// A whole row by one workgroup without bins.
template <int NT>
__device__ int slow(const SampleRowsArgs& a, const float* x, float mx, float u, uint64_t* hist, uint64_t* red) {
  const int V = a.V, tid = threadIdx.x;
  Keep keep = {0, mx, a.temperature, -INFINITY};
  auto key = [&](int i) { return order(x[i]); };
  uint32_t least = 0;
  if (a.top_k) least = key_reaching<NT>(V, (uint64_t)a.top_k, hist, red, key, [](int) { return 1ull; });
  if (a.top_p < 1.0) {
    uint64_t s = 0;
    for (int i = tid; i < V; i += NT) s += keep(x[i]);
    const double goal = ceil(a.top_p * (double)group_sum<NT>(s, red));
    least = max(least, key_reaching<NT>(V, (uint64_t)fmax(goal, 1.0), hist, red, key, [&](int i) { return keep(x[i]); }));
  }
  keep.least = least;
  keep.min_gap = a.min_gap;
  // contiguous pieces: the thread in whose piece the running sum passes the draw
  const int C = (V + NT - 1) / NT, i0 = min(tid * C, V), i1 = min(i0 + C, V);
  uint64_t s = 0, total;
  for (int i = i0; i < i1; ++i) s += keep(x[i]);
  uint64_t c = sum_before<NT>(s, red, total);
  const uint64_t target = draw_target(u, total);
  int* found = reinterpret_cast<int*>(red + NT / 64);
  if (c <= target && target < c + s) {   // one thread
    int i = i0;
    for (c += keep(x[i]); c <= target; c += keep(x[i])) ++i;
    *found = i;
  }
  __syncthreads();
  return *found;
}

// Entries and weights per bin of a workgroup's x, in LDS; by the callers' barriers
template <int NT>
struct Histogram {
  uint64_t weight[kBins][kCopies];
  uint32_t count[kBins][kCopies];
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < kBins * kCopies; i += NT) {
      (&weight[0][0])[i] = 0;
      (&count[0][0])[i] = 0;
    }
  }
  __device__ __forceinline__ void add(float x, int top, double per, bool weights) {
    const int b = bin_of(x, per), r = top - b;
    if (r >= kBins) return;
    const int c = threadIdx.x % kCopies;
    atomicAdd(&count[r][c], 1u);
    if (weights) add_u64(&weight[r][c], bin_weight(x, per, b));
  }
  __device__ __forceinline__ void sum(int r, uint64_t& w, uint32_t& n) const {
    w = 0;
    n = 0;
#pragma unroll
    for (int c = 0; c < kCopies; ++c) {
      w += weight[r][c];
      n += count[r][c];
    }
  }
};

// ---- one workgroup per row ---------------------------------------------------------
template <int E>
__global__ void __launch_bounds__(kOneThreads) k_one(const SampleRowsArgs a) {
  constexpr int NT = kOneThreads;
  __shared__ union {
    Histogram<NT> h;
    float v[kList];
  } sh;
  __shared__ Bins bins;
  __shared__ uint64_t red[NT / 64 + 2], part[E / 4], digits[256];
  __shared__ uint32_t least;
  __shared__ int n;
  __shared__ Edge edge;
  const int tid = threadIdx.x, row = blockIdx.x;
  const float* x = a.logits + (size_t)row * a.ld;
  Chunk<NT, E> c;
  c.load(x, 0, a.V);
  const uint32_t mk = group_max<NT>(c.top(), red);
  const float mx = from_order(mk);
  if (mx == -INFINITY) {   // nothing to choose from
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (!(a.temperature > 0.0)) {
    uint32_t first = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c.x[e] == mx) first = min(first, (uint32_t)c.at(e / 4, e % 4));
    first = ~group_max<NT>(~first, red);
    if (tid == 0) a.out[row] = (int)first;
    return;
  }
  const float u = a.u[row];
  Keep keep = {0, mx, a.temperature, a.min_gap};
  if (a.top_k || a.top_p < 1.0) {
    const double per = 4.0 / a.temperature;
    const int top = bin_of(mx, per);
    sh.h.clear();
    if (tid == 0) n = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) sh.h.add(c.x[e], top, per, a.top_p < 1.0);
    __syncthreads();
    if (tid < kBins) sh.h.sum(tid, bins.weight[tid], bins.count[tid]);
    __syncthreads();
    if (tid < kWave) {
      const Edge e = find_edge(a, bins, top, mx, per);
      if (tid == 0) edge = e;
    }
    __syncthreads();
    const Edge e = edge;
    const bool far = top <= -kFar || top >= kFar;
    if (e.need_k || e.need_p || far) {
      if (far || bins.count[top - e.bin] > (uint32_t)kList) {
        const int i = slow<NT>(a, x, mx, u, digits, red);
        if (tid == 0) a.out[row] = i;
        return;
      }
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (bin_of(c.x[k], per) == e.bin) sh.v[atomicAdd(&n, 1)] = c.x[k];
      __syncthreads();
      keep.least = least_of<NT>(e, sh.v, n, per, digits, red, &least);
    }   // (else min-p alone cuts there, and the entries are asked one by one)
  }
  __syncthreads();
  const int i = c.pick(keep, 0, 0, true, u, part, red);
  if (tid == 0) a.out[row] = i;
}

// ---- many workgroups per row -------------------------------------------------------
// A row's part of the workspace
struct RowWork {
  Bins* bins;          // [tiles], each from its own maximum's bin down
  uint32_t* top;       // [tiles] the maximum's key
  int* first;          // [tiles] temperature 0: its first index
  uint64_t* kept;      // [tiles] weights that stay for certain
  uint64_t* list;      // [kList] the threshold's bin: index << 32 | x
  uint32_t* count;     // [0] entries of that list, [1] workgroups done
};
__host__ __device__ inline size_t up256(size_t n) { return (n + 255) & ~(size_t)255; }
__host__ __device__ inline RowWork row_work(void* work, int row, int tiles, size_t* bytes) {
  size_t o = 0;
  auto take = [&](size_t n) {
    const size_t at = o;
    o += up256(n);
    return at;
  };
  const size_t b = take(sizeof(Bins) * tiles), t = take(sizeof(uint32_t) * tiles), f = take(sizeof(int) * tiles),
               k = take(sizeof(uint64_t) * tiles), l = take(sizeof(uint64_t) * kList), c = take(2 * sizeof(uint32_t));
  uint8_t* p = static_cast<uint8_t*>(work) + (size_t)row * o;
  if (bytes) *bytes = o;
  return {reinterpret_cast<Bins*>(p + b),     reinterpret_cast<uint32_t*>(p + t), reinterpret_cast<int*>(p + f),
          reinterpret_cast<uint64_t*>(p + k), reinterpret_cast<uint64_t*>(p + l), reinterpret_cast<uint32_t*>(p + c)};
}
__host__ __device__ inline bool by_bins(const SampleRowsArgs& a) { return a.temperature > 0.0 && (a.top_k || a.top_p < 1.0); }

// 1. a tile's maximum and bins. Grid: tiles x rows.
__global__ void __launch_bounds__(kTileThreads) k_tiles(const SampleRowsArgs a) {
  constexpr int NT = kTileThreads;
  __shared__ Histogram<NT> h;
  __shared__ uint64_t red[NT / 64 + 2];
  const int tid = threadIdx.x, tile = blockIdx.x, row = blockIdx.y;
  const RowWork w = row_work(a.work, row, gridDim.x, nullptr);
  Chunk<NT, kTileEach> c;
  c.load(a.logits + (size_t)row * a.ld, tile * kTile, a.V);
  if (by_bins(a)) h.clear();
  const uint32_t mk = group_max<NT>(c.top(), red);
  if (tid == 0) {
    w.top[tile] = mk;
    if (tile == 0) w.count[0] = w.count[1] = 0;
  }
  const float mx = from_order(mk);
  if (!(a.temperature > 0.0)) {
    uint32_t first = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < kTileEach; ++e)
      if (c.x[e] == mx) first = min(first, (uint32_t)c.at(e / 4, e % 4));
    first = ~group_max<NT>(~first, red);
    if (tid == 0) w.first[tile] = tile * kTile + (int)first;
  }
  if (!by_bins(a) || mx == -INFINITY) return;
  const double per = 4.0 / a.temperature;
  const int top = bin_of(mx, per);
#pragma unroll
  for (int e = 0; e < kTileEach; ++e) h.add(c.x[e], top, per, a.top_p < 1.0);
  __syncthreads();
  if (tid < kBins) h.sum(tid, w.bins[tile].weight[tid], w.bins[tile].count[tid]);
}

// 2. what stays of each tile; the row's last workgroup draws. Grid: tiles x rows.
__global__ void __launch_bounds__(kTileThreads) k_draw(const SampleRowsArgs a) {
  constexpr int NT = kTileThreads, kGroups = NT / kBins;
  __shared__ union {
    Bins part[kGroups];
    struct {
      float v[kList];
      int at[kList];
    } l;
  } sh;
  __shared__ Bins bins;
  __shared__ uint64_t red[NT / 64 + 2], part[kTileEach / 4], digits[256], kept[kMaxTiles];
  __shared__ uint32_t tops[kMaxTiles], least, base;
  __shared__ Edge edge;
  __shared__ bool last;
  const int tid = threadIdx.x, tile = blockIdx.x, tiles = gridDim.x, row = blockIdx.y;
  const RowWork w = row_work(a.work, row, tiles, nullptr);
  const float* x = a.logits + (size_t)row * a.ld;
  Chunk<NT, kTileEach> c;
  c.load(x, tile * kTile, a.V);
  if (tid < tiles) tops[tid] = w.top[tid];
  __syncthreads();
  uint32_t mk = 0;
  for (int t = 0; t < tiles; ++t) mk = max(mk, tops[t]);
  const float mx = from_order(mk);
  if (mx == -INFINITY || !(a.temperature > 0.0)) {   // nothing to choose from, or the first maximum
    if (tile == 0 && tid == 0) {
      int t = 0;
      while (tops[t] != mk) ++t;
      a.out[row] = mx == -INFINITY ? -1 : w.first[t];
    }
    return;
  }
  const float u = a.u[row];
  const double per = 4.0 / a.temperature;
  const int top = bin_of(mx, per);
  Keep keep = {0, mx, a.temperature, a.min_gap};
  Edge e = {top - kBins, 0, 0};
  if (by_bins(a)) {
    const int r = tid % kBins, g = tid / kBins;
    uint64_t weight = 0;
    uint32_t count = 0;
    for (int t = g; t < tiles; t += kGroups) {
      const float m = from_order(tops[t]);
      if (m == -INFINITY) continue;
      const int at = r - (top - bin_of(m, per));
      if (at < 0) continue;
      weight += w.bins[t].weight[at];
      count += w.bins[t].count[at];
    }
    sh.part[g].weight[r] = weight;
    sh.part[g].count[r] = count;
    __syncthreads();
    if (tid < kBins) {
      uint64_t s = 0;
      uint32_t n = 0;
#pragma unroll
      for (int k = 0; k < kGroups; ++k) {
        s += sh.part[k].weight[tid];
        n += sh.part[k].count[tid];
      }
      bins.weight[tid] = s;
      bins.count[tid] = n;
    }
    __syncthreads();
    if (tid < kWave) {
      const Edge f = find_edge(a, bins, top, mx, per);
      if (tid == 0) edge = f;
    }
    __syncthreads();
    e = edge;
  }
  const bool far = by_bins(a) && (top <= -kFar || top >= kFar);
  const bool inside = e.need_k || e.need_p;   // the threshold is found among the bin's entries
  uint64_t s = 0;
  int mine = 0;
  if (!far) {
#pragma unroll
    for (int k = 0; k < kTileEach; ++k) {
      const int b = inside ? bin_of(c.x[k], per) : 0;
      if (!inside || b > e.bin) s += keep(c.x[k]);
      else if (b == e.bin) ++mine;
    }
  }
  s = group_sum<NT>(s, red);
  uint64_t all;
  int at = (int)sum_before<NT>((uint64_t)mine, red, all);
  if (tid == 0) {
    cst64(&w.kept[tile], s);
    base = all ? __hip_atomic_fetch_add(&w.count[0], (uint32_t)all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0u;
  }
  __syncthreads();
  if (mine) {
    at += (int)base;
#pragma unroll
    for (int k = 0; k < kTileEach; ++k)
      if (bin_of(c.x[k], per) == e.bin) {
        if (at < kList)
          cst64(&w.list[at], (uint64_t)(uint32_t)(tile * kTile + c.at(k / 4, k % 4)) << 32 | __float_as_uint(c.x[k]));
        ++at;
      }
  }
  vm_drain();   // what this wave published
  __syncthreads();
  if (tid == 0)
    last = __hip_atomic_fetch_add(&w.count[1], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)tiles - 1;
  __syncthreads();
  if (!last) return;

  const uint32_t n = cld(&w.count[0]);
  if (far || n > (uint32_t)kList) {
    const int i = slow<NT>(a, x, mx, u, digits, red);
    if (tid == 0) a.out[row] = i;
    return;
  }
  if (tid < tiles) kept[tid] = cld64(&w.kept[tid]);
  for (int i = tid; i < (int)n; i += NT) {
    const uint64_t y = cld64(&w.list[i]);
    sh.l.v[i] = __uint_as_float((uint32_t)y);
    sh.l.at[i] = (int)(y >> 32);
  }
  __syncthreads();
  if (inside) {
    keep.least = least_of<NT>(e, sh.l.v, (int)n, per, digits, red, &least);
    for (int i = tid; i < (int)n; i += NT)
      if (const uint64_t v = keep(sh.l.v[i])) add_u64(&kept[sh.l.at[i] / kTile], v);
    __syncthreads();
  }
  uint64_t total = 0, before = 0;
  for (int t = 0; t < tiles; ++t) total += kept[t];
  const uint64_t target = draw_target(u, total);
  int t = 0;
  while (t < tiles - 1 && target >= before + kept[t]) before += kept[t++];
  c.load(x, t * kTile, a.V);
  const int i = c.pick(keep, before, target, false, u, part, red);
  if (tid == 0) a.out[row] = t * kTile + i;
}

template <int E>
hipError_t launch_one(const SampleRowsArgs& a, hipStream_t s) {
  hipLaunchKernelGGL(k_one<E>, dim3(a.rows), dim3(kOneThreads), 0, s, a);
  return hipGetLastError();
}
int tiles_of(int V) { return V <= kOneMax ? 0 : (V + kTile - 1) / kTile; }

}  // namespace

size_t sample_rows_workspace(int rows, int V) {
  size_t bytes = 0;
  if (const int tiles = tiles_of(V)) row_work(nullptr, 0, tiles, &bytes);
  return bytes * rows;
}

hipError_t launch_sample_rows(const SampleRowsArgs& a, hipStream_t s) {
  if (a.rows < 1 || a.V < 1 || a.V > kSampleRowsMaxV) return hipErrorInvalidValue;
  if (const int tiles = tiles_of(a.V)) {
    const dim3 grid(tiles, a.rows), block(kTileThreads);
    hipLaunchKernelGGL(k_tiles, grid, block, 0, s, a);
    hipLaunchKernelGGL(k_draw, grid, block, 0, s, a);
    return hipGetLastError();
  }
  return a.V <= 4 * kOneThreads ? launch_one<4>(a, s) : a.V <= 16 * kOneThreads ? launch_one<16>(a, s) : launch_one<kOneEach>(a, s);
}

}  // namespace ssk
