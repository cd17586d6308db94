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
// Weights are formed and summed in 64 bits: in 32 the running sums of a
// 128256-entry row are off by some 1e-8, and one row in a thousand would take a
// neighbouring entry. Sums whose terms meet in no fixed order are of whole
// multiples of 2^-44, so a call gives the same tokens every time.
//
// The thresholds come from a histogram over bins of x / T a quarter wide, with
// the number of entries and the weights of each: 128 bins from the maximum's down
// reach e^-31.75, where all entries together weigh less than 2^-26. The highest
// of the three thresholds lies in one bin; what lies above that bin stays, what
// lies below goes, and the bin's own entries are gathered and the threshold found
// among them. Of a bin with more than kList of them (flat rows) one workgroup goes
// through the whole row for it. |x / T| past 2^18 leaves the row to `slow`, which
// selects by the bits of x without bins.
//
// Rows of up to kOne entries: one workgroup with the row in registers, one launch.
// Longer ones: a launch over tiles for their maxima and histograms, and one with
// some workgroups per row, each of which adds up the bins and goes through a part
// of the tiles that have entries in the threshold's bin; the last of a row to
// finish (by a count that the first launch clears) finds the threshold and draws
// within one tile. Weights are formed once, for the histogram, and again for the
// threshold's bin and the last tile.

#include <type_traits>

#include "ss_device.h"
#include "ss_kernels.h"

namespace ssk {
namespace {

constexpr double kUnit = 17592186044416.0;  // 2^44
constexpr int kBins = 128;
// Of the histogram, one per lane % 4 (64 rows of 128256, top-p: one copy 39.7 us, two
// 39.8, four 39.9, eight 40.9; of entries in few bins, top-k: 57, 44, 38, 37).
constexpr int kCopies = 4;
constexpr int kList = 8192;                 // entries of the threshold's bin
constexpr int kPairs = 256;                 // up to this many are compared each with all
constexpr float kFar = 1048576.f;           // 2^20 bins from 0: neighbours are not told apart

constexpr int kOneThreads = 512, kOne = 16 * kOneThreads;   // of 8 or 16 entries each
constexpr int kTileThreads = 512, kTileEach = 8, kTile = kTileThreads * kTileEach;
constexpr int kMaxTiles = (kSampleRowsMaxV + kTile - 1) / kTile;   // 128
constexpr int kRowThreads = 512, kRounds = 8;   // the row's workgroups go through rounds of 2048 entries, 8 at a time
constexpr int kStep = 4 * kRounds * kRowThreads;

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
// u as a fraction of 1; u outside [0, 1) counts as the nearest number inside
__device__ __forceinline__ double fraction(float u) { return u > 0.f ? fmin((double)u, 1.0 - 0x1p-53) : 0.0; }

// The row's scale of bins: 4 / T in 32 bits places x (a rounded product, still in
// the order of x), 1 / T in 64 bits weighs it.
struct Scale {
  float per;
  double inv;
  __device__ __forceinline__ float bin(float x) const { return x == x ? floorf(x * per) : -INFINITY; }
  // e^(x / T - the middle of bin b), for |x / T - that| of 1/8 and a little: the
  // eighth power's term is below 2e-12
  __device__ __forceinline__ double weight(float x, float b) const {
    const double r = fma((double)x, inv, (double)fmaf(b, -0.25f, -0.125f));
    double p = 1.0 / 5040;
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    return fma(p, r, 1.0);
  }
  // in units of 2^-44, as a whole number: the low bits of its sum with 2^52 (it is below 2)
  __device__ __forceinline__ uint64_t units(float x, float b) const {
    return (uint64_t)__double_as_longlong(fma(weight(x, b), kUnit, 0x1p52)) & 0xfffffffffffffull;
  }
};

// ---- sums over waves and workgroups ----------------------------------------------
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp64(T v) {   // 0 where no lane gives one
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xf, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(b >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
}
// sum of v (uint64_t or double) over the lanes up to this one
template <class T>
__device__ __forceinline__ T wave_upto(T v) {
  v += dpp64<0x111, 0xf>(v);   // row_shr:1
  v += dpp64<0x112, 0xf>(v);
  v += dpp64<0x114, 0xf>(v);
  v += dpp64<0x118, 0xf>(v);
  v += dpp64<0x142, 0xa>(v);   // row_bcast:15 into rows 1 and 3
  v += dpp64<0x143, 0xc>(v);   // row_bcast:31 into rows 2 and 3
  return v;
}
template <class T>
__device__ __forceinline__ T from_lane(T v, int lane) {   // lane: the same for the wave
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, lane);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(b >> 32), lane);
  return __builtin_bit_cast(T, (uint64_t)hi << 32 | lo);
}
template <class T>
__device__ __forceinline__ T wave_total(T v) {
  return from_lane(wave_upto(v), 63);
}
// over the workgroup of NT threads, in every thread, the waves in order; red: NT / 64 words
template <int NT, class T>
__device__ T group_sum(T v, T* red) {
  v = wave_total(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  T t = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) t += red[w];
  return t;
}
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t v) {
  auto up = [&](auto ctrl, auto rows) {
    v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  up(integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});
  up(integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
  up(integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
  up(integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
  up(integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});
  up(integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});
  return (uint32_t)__builtin_amdgcn_readlane((int)v, 63);
}
template <int NT>
__device__ uint32_t group_max(uint32_t v, uint64_t* red) {
  v = wave_max_u32(v);
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
  const uint64_t incl = wave_upto(v);
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

// Selection by the bits of the keys, kDigit at a time: the largest key at which
// the sum of val(x) over the entries with that key or a greater one reaches
// target, or a smaller one that parts the entries alike, 0 when all together do
// not. entries(f): f(x) of each of this thread's entries; some: one of all. one:
// what one entry's val is at most, and less than two entries' (0: not known).
// hist: 2^kDigit words, red: NT / 64 + 3.
constexpr int kDigit = 10, kDigits = 1 << kDigit;
template <int NT, class Entries, class Val>
__device__ uint32_t key_reaching(float some, uint64_t target, uint64_t one, uint64_t* hist, uint64_t* red, Entries entries,
                                 Val val) {
  constexpr int kEach = kDigits / NT;   // digits of a thread, the highest ones in thread 0
  static_assert(kEach * NT == kDigits, "whole");
  // the bits that all keys share
  const uint32_t first = order(some);
  uint32_t differ = 0;
  entries([&](float x) { differ |= order(x) ^ first; });
  for (int d = threadIdx.x; d < kDigits; d += NT) hist[d] = 0;
  int shift = (int)group_max<NT>(differ ? 32 - __clz((int)differ) : 0, red);   // as many low bits do not
  uint64_t* found = red + NT / 64;
  uint32_t mask = shift < 32 ? ~0u << shift : 0u, prefix = first & mask;
  uint64_t above = 0;
  do {
    const int bits = min(kDigit, shift);
    shift -= bits;
    const uint32_t digit = (1u << bits) - 1;
    entries([&](float x) {
      const uint32_t k = order(x);
      if ((k & mask) == prefix) add_u64(&hist[(k >> shift) & digit], val(x));
    });
    if (threadIdx.x == 0) found[0] = kDigits;
    __syncthreads();
    uint64_t h[kEach], sum = 0, all;
#pragma unroll
    for (int c = 0; c < kEach; ++c) {
      const int d = kDigits - 1 - (kEach * (int)threadIdx.x + c);
      h[c] = hist[d];
      hist[d] = 0;   // for the next digit
      sum += h[c];
    }
    uint64_t before = above + sum_before<NT>(sum, red, all);
#pragma unroll
    for (int c = 0; c < kEach; ++c) {
      if (before < target && before + h[c] >= target) {
        found[0] = kDigits - 1 - (kEach * (int)threadIdx.x + c);
        found[1] = before;
        found[2] = h[c];
      }
      before += h[c];
    }
    __syncthreads();
    if (found[0] == kDigits) return 0;
    prefix |= (uint32_t)found[0] << shift;
    mask |= digit << shift;
    above = found[1];
    const bool alone = found[2] <= one;
    __syncthreads();
    if (alone) break;   // (its key's low bits part it from nothing)
  } while (shift > 0);
  return prefix;
}

// e^(-r / 4), r < kBins, as a product of powers
__device__ __forceinline__ double fall_of(int r) {
  constexpr double kPower[7] = {0.77880078307140486825, 0.60653065971263342360, 0.36787944117144232160, 0.13533528323661269189,
                                0.01831563888873418029, 0.00033546262790251183882, 1.1253517471925911451e-7};   // e^(-2^i / 4)
  double f = 1.0;
#pragma unroll
  for (int i = 0; i < 7; ++i) f *= r >> i & 1 ? kPower[i] : 1.0;
  return f;
}

// What stays, and with which weight, in units of the middle of the maximum's bin.
struct Keep {
  Scale scale;
  const double* fall;   // fall_of(r), r < kBins
  float top;            // the maximum's bin
  float least;          // the least that stays
  __device__ __forceinline__ double operator()(float x) const {
    const float b = scale.bin(x), r = top - b;
    return r < kBins && x >= least ? scale.weight(x, b) * fall[(int)r] : 0.0;
  }
};
// the least float that stays by min-p
__device__ __forceinline__ float least_by_gap(float mx, double min_gap) {
  if (min_gap == -INFINITY) return -INFINITY;
  uint32_t k = order((float)((double)mx + min_gap));
  while (gap(from_order(k), mx) < min_gap) ++k;        // (a step at most: the sum rounds to the nearest float)
  while (gap(from_order(k - 1), mx) >= min_gap) --k;
  return from_order(k);
}

// ---- a row's entries in the registers of a workgroup ---------------------------
// x[4k + j] of thread t is entry 4 (k * NT + t) + j of those loaded (-inf past the row)
template <int NT, int E>
struct Chunk {
  static constexpr int kRounds = E / 4;
  float x[E];
  __device__ __forceinline__ static int at(int k, int j) { return 4 * (k * NT + (int)threadIdx.x) + j; }
  __device__ __forceinline__ void load(const float* row, int i0, int V) {
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      const int i = i0 + at(k, 0);
      if (i + 4 <= V) {
        __builtin_memcpy(&x[4 * k], row + i, 16);   // (rows start on any multiple of 4 bytes)
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) x[4 * k + j] = i + j < V ? row[i + j] : -INFINITY;
      }
    }
  }
  __device__ __forceinline__ uint32_t top() const {   // the maximum's key
    float m = -INFINITY;   // (fmaxf leaves a NaN aside)
#pragma unroll
    for (int e = 0; e < E; ++e) m = fmaxf(m, x[e]);
    return order(m);
  }
  // the first index of value v
  __device__ int first(float v, uint64_t* red) const {
    uint32_t i = 0xffffffffu;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (x[e] == v) i = min(i, (uint32_t)at(e / 4, e % 4));
    return (int)~group_max<NT>(~i, red);
  }
  // The first entry at which the running sum of what stays, from `before` on,
  // passes target (whole: passes target times the sum of these); where rounding
  // leaves none, the last that stays. part: kRounds * NT / 64 words, red: NT / 64 + 1.
  __device__ int pick(const Keep& keep, double before, double target, bool whole, double* part, uint64_t* red) const {
    constexpr int W = NT / 64;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    double w[E];
    uint32_t any = 0;   // 1 + the last entry with a weight
#pragma unroll
    for (int k = 0; k < kRounds; ++k) {
      double s = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[4 * k + j] = keep(x[4 * k + j]);
        s += w[4 * k + j];
        if (w[4 * k + j] > 0.0) any = at(k, j) + 1;
      }
      s = wave_upto(s);
      if (lane == 63) part[W * k + wave] = s;
    }
    any = group_max<NT>(any, red);   // (and a barrier for part)
    if (whole) {
      double total = 0.0;
      for (int p = 0; p < kRounds * W; ++p) total += part[p];
      target *= total;
    }
    int* found = reinterpret_cast<int*>(red + W);
    if (threadIdx.x == 0) *found = -1;
    __syncthreads();
    // the wave and round that the draw falls into look closer
    double c = before;
    int p = 0;
    while (p < kRounds * W && !(target < c + part[p])) c += part[p++];
    if (p < kRounds * W && wave == p % W) {
#pragma unroll
      for (int k = 0; k < kRounds; ++k)
        if (k == p / W) {
          const double s = (w[4 * k] + w[4 * k + 1]) + (w[4 * k + 2] + w[4 * k + 3]);
          const double at0 = c + (wave_upto(s) - s);
          int mine = -1, held = -1;   // the first to pass, the last that stays
#pragma unroll
          for (int j = 3; j >= 0; --j) {
            double upto = at0;
#pragma unroll
            for (int i = 0; i <= j; ++i) upto += w[4 * k + i];
            if (w[4 * k + j] > 0.0 && target < upto) mine = at(k, j);
            if (w[4 * k + j] > 0.0 && held < 0) held = at(k, j);
          }
          const uint64_t hit = __ballot(mine >= 0), some = __ballot(held >= 0);
          if (hit ? lane == __ffsll((unsigned long long)hit) - 1 : some && lane == 63 - __clzll((long long)some))
            *found = hit ? mine : held;
        }
    }
    __syncthreads();
    return *found >= 0 ? *found : (int)any - 1;
  }
};

// f(i, x[i]) of each of this thread's entries of a row, 4 of them requested at a
// time (64 hot rows of 128256 234 us, one at a time 950; eight 267, but every other
// row then takes 49 us instead of 40, for the code and registers of it)
template <int NT, class F>
__device__ __forceinline__ void over_row(const float* x, int V, F f) {
  using Round = Chunk<NT, 4>;
#pragma unroll 1
  for (int i0 = 0; i0 < V; i0 += 4 * NT) {
    Round c;
    c.load(x, i0, V);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int i = i0 + Round::at(e / 4, e % 4);
      if (i < V) f(i, c.x[e]);
    }
  }
}

// ---- the thresholds --------------------------------------------------------------
// Where the highest of the thresholds lies, from the bins' entries and weights.
struct Edge {
  int r;               // of bin top - r (kBins: everything stays)
  uint64_t need_k;     // entries of that bin that stay by top-k (0: no limit there)
  uint64_t need_p;     // weight of that bin, as Scale::weight, at which top-p cuts (0: none there)
  __device__ __forceinline__ bool inside() const { return need_k || need_p; }
};
struct Bins {
  uint64_t weight[kBins];   // [r]
  uint32_t count[kBins];
};

// by one wave, from bins in LDS; lane l has bins l and 64 + l
__device__ __forceinline__ Edge find_edge(const SampleRowsArgs& a, const Bins& h, const Keep& keep) {
  const int lane = threadIdx.x & 63;
  int kb = kBins, pb = kBins, mb = kBins;
  uint64_t need_k = 0, need_p = 0;
  if (a.top_k) {
    uint64_t base = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint64_t c = h.count[64 * half + lane], incl = base + wave_upto(c);
      const uint64_t hit = __ballot(incl >= (uint64_t)a.top_k);
      if (hit && kb == kBins) {
        const int l = __ffsll((unsigned long long)hit) - 1;
        kb = 64 * half + l;
        need_k = a.top_k - from_lane(incl - c, l);
      }
      base = from_lane(incl, 63);
    }
  }
  if (a.top_p < 1.0) {
    double m[2], incl[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      m[half] = (double)h.weight[64 * half + lane] * keep.fall[64 * half + lane];
      incl[half] = wave_upto(m[half]) + (half ? from_lane(incl[0], 63) : 0.0);
    }
    const double goal = a.top_p * from_lane(incl[1], 63);
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const uint64_t hit = __ballot(incl[half] >= goal);
      if (hit && pb == kBins) {
        const int l = __ffsll((unsigned long long)hit) - 1;
        pb = 64 * half + l;
        const double need = (goal - from_lane(incl[half] - m[half], l)) / keep.fall[pb];
        need_p = min((uint64_t)fmax(ceil(need), 1.0), h.weight[pb]);
      }
    }
  }
  if (keep.least > -INFINITY) {   // min-p's
    const float r = keep.top - keep.scale.bin(keep.least);
    mb = r < kBins ? (int)r : kBins;
  }
  const int r = min(min(kb, pb), mb);
  return {r, kb == r ? need_k : 0, pb == r ? need_p : 0};
}

// The least key that stays, among the entries of the threshold's bin
template <int NT, class Entries>
__device__ uint32_t least_among(const Edge& e, const Keep& keep, float some, uint64_t* digits, uint64_t* red, Entries entries) {
  const float bin = keep.top - (float)e.r;
  uint32_t k = 0;
  // (weights are e^-1/8 .. e^1/8 times 2^44, and a little)
  constexpr uint64_t kOneWeight = 3ull << 43;
  if (e.need_k) k = key_reaching<NT>(some, e.need_k, 1, digits, red, entries, [](float) { return 1ull; });
  if (e.need_p)
    k = max(k, key_reaching<NT>(some, e.need_p, kOneWeight, digits, red, entries,
                                [&](float x) { return keep.scale.units(x, bin); }));
  return k;
}

// The same, of the n entries of that bin (v: their
// logits, in LDS): each compared with all, by 8 threads, or selection by bits.
// digits: kDigits words.
template <int NT>
__device__ uint32_t least_of(const Edge& e, const Keep& keep, const float* v, int n, uint64_t* digits, uint64_t* red,
                             uint32_t* least) {
  const float bin = keep.top - (float)e.r;
  const int tid = threadIdx.x;
  if (n <= kPairs) {
    static_assert(kPairs <= kDigits && kPairs <= NT, "a weight per entry");
    if (tid < n) digits[tid] = e.need_p ? keep.scale.units(v[tid], bin) : 0;
    if (tid == 0) *least = 0;
    __syncthreads();
    for (int i = tid / 8; i < n; i += NT / 8) {
      const float x = v[i];
      uint32_t ge = 0, gt = 0;        // entries at or above x, and above
      uint64_t wge = 0, wgt = 0;      // and their weights
      for (int j = tid % 8; j < n; j += 8) {
        const float y = v[j];
        const uint64_t w = digits[j];
        ge += y >= x;
        gt += y > x;
        wge += y >= x ? w : 0;
        wgt += y > x ? w : 0;
      }
      uint64_t c = (uint64_t)gt << 32 | ge;
#pragma unroll
      for (int off = 1; off < 8; off <<= 1) {
        c += __shfl_xor((unsigned long long)c, off, kWave);
        wge += __shfl_xor((unsigned long long)wge, off, kWave);
        wgt += __shfl_xor((unsigned long long)wgt, off, kWave);
      }
      const bool by_k = e.need_k && (c >> 32) < e.need_k && (uint32_t)c >= e.need_k;
      const bool by_p = e.need_p && wgt < e.need_p && wge >= e.need_p;
      if (tid % 8 == 0 && (by_k || by_p)) atomicMax(least, order(x));
    }
    __syncthreads();
    return *least;
  }
  return least_among<NT>(e, keep, v[0], digits, red, [&](auto f) {
    for (int i = tid; i < n; i += NT) f(v[i]);
  });
}

// A whole row by one workgroup without bins, with weights of up to 2^44.
template <int NT>
__device__ int slow(const SampleRowsArgs& a, const float* x, float mx, float u, uint64_t* hist, uint64_t* red) {
  const int V = a.V, tid = threadIdx.x;
  auto entries = [&](auto f) { over_row<NT>(x, V, [&](int, float y) { f(y); }); };
  auto weight = [&](float y) { return (uint64_t)(exp(gap(y, mx) / a.temperature) * kUnit + 0.5); };
  uint32_t least = 0;
  if (a.top_k) least = key_reaching<NT>(mx, (uint64_t)a.top_k, 1, hist, red, entries, [](float) { return 1ull; });
  if (a.top_p < 1.0) {
    uint64_t s = 0;
    entries([&](float y) { s += weight(y); });
    const double goal = ceil(a.top_p * (double)group_sum<NT>(s, red));
    least = max(least, key_reaching<NT>(mx, (uint64_t)fmax(goal, 1.0), 0, hist, red, entries, weight));
  }
  auto kept = [&](int i) { return order(x[i]) >= least && gap(x[i], mx) >= a.min_gap ? weight(x[i]) : 0; };
  // contiguous pieces: the thread in whose piece the running sum passes the draw
  const int C = (V + NT - 1) / NT, i0 = min(tid * C, V), i1 = min(i0 + C, V);
  uint64_t s = 0, total;
  for (int i = i0; i < i1; ++i) s += kept(i);
  uint64_t c = sum_before<NT>(s, red, total);
  const uint64_t target = min((uint64_t)(fraction(u) * (double)total), total - 1);   // (the maximum stays: total > 0)
  int* found = reinterpret_cast<int*>(red + NT / 64);
  if (c <= target && target < c + s) {   // one thread
    int i = i0;
    for (c += kept(i); c <= target; c += kept(i)) ++i;
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
  __device__ __forceinline__ void add(float x, float top, const Scale& s, bool counts, bool weights) {
    const float b = s.bin(x), r = top - b;
    if (!(r < kBins)) return;
    const int c = threadIdx.x % kCopies;
    if (counts) atomicAdd(&count[(int)r][c], 1u);
    if (weights) add_u64(&weight[(int)r][c], s.units(x, b));
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

__device__ __forceinline__ Scale scale_of(const SampleRowsArgs& a) { return {(float)(4.0 / a.temperature), 1.0 / a.temperature}; }
__device__ __forceinline__ bool filtered(const SampleRowsArgs& a) { return a.top_k || a.top_p < 1.0; }
// neighbouring bins are told apart around this one
__device__ __forceinline__ bool is_near(float top) { return top > -kFar && top < kFar; }

// ---- one workgroup per row ---------------------------------------------------------
template <int E>
__global__ void __launch_bounds__(kOneThreads) k_one(const SampleRowsArgs a) {
  constexpr int NT = kOneThreads;
  using Row = Chunk<NT, E>;
  __shared__ union {
    Histogram<NT> h;
    float v[NT * E];
  } sh;
  __shared__ Bins bins;
  __shared__ double fall[kBins], part[Row::kRounds * NT / 64];
  __shared__ uint64_t red[NT / 64 + 3], digits[kDigits];
  __shared__ uint32_t least;
  __shared__ int n;
  __shared__ Edge edge;
  const int tid = threadIdx.x, row = blockIdx.x;
  const float* x = a.logits + (size_t)row * a.ld;
  Row c;
  c.load(x, 0, a.V);
  if (tid < kBins) fall[tid] = fall_of(tid);
  if (filtered(a)) sh.h.clear();
  if (tid == 0) n = 0;
  const float mx = from_order(group_max<NT>(c.top(), red));
  if (mx == -INFINITY || !(a.temperature > 0.0)) {   // nothing to choose from, or the first maximum
    const int i = mx == -INFINITY ? -1 : c.first(mx, red);
    if (tid == 0) a.out[row] = i;
    return;
  }
  const float u = a.u[row];
  const Scale scale = scale_of(a);
  Keep keep = {scale, fall, scale.bin(mx), -INFINITY};
  if (!is_near(keep.top)) {
    const int i = slow<NT>(a, x, mx, u, digits, red);
    if (tid == 0) a.out[row] = i;
    return;
  }
  keep.least = least_by_gap(mx, a.min_gap);
  if (filtered(a)) {
#pragma unroll
    for (int e = 0; e < E; ++e) sh.h.add(c.x[e], keep.top, scale, a.top_k, a.top_p < 1.0);
    __syncthreads();
    if (tid < kBins) sh.h.sum(tid, bins.weight[tid], bins.count[tid]);
    __syncthreads();
    if (tid < kWave) {
      const Edge e = find_edge(a, bins, keep);
      if (tid == 0) edge = e;
    }
    __syncthreads();
    const Edge e = edge;
    if (e.inside()) {   // (else min-p alone cuts there, and the entries are asked one by one)
#pragma unroll
      for (int k = 0; k < E; ++k)
        if (keep.top - scale.bin(c.x[k]) == (float)e.r) sh.v[atomicAdd(&n, 1)] = c.x[k];
      __syncthreads();
      keep.least = fmaxf(keep.least, from_order(least_of<NT>(e, keep, sh.v, n, digits, red, &least)));
    }
  }
  const int i = c.pick(keep, 0.0, fraction(u), true, part, red);
  if (tid == 0) a.out[row] = i;
}
// ---- many workgroups per row -------------------------------------------------------
// A row's part of the workspace
struct RowWork {
  Bins* bins;          // [tiles], each from its own maximum's bin down
  uint32_t* top;       // [tiles] the maximum's key
  int* first;          // [tiles] temperature 0: its first index
  uint64_t* list;      // [kList] the threshold's bin's entries: place << 32 | x
  uint32_t* count;     // [0] as many, [1] workgroups done
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
               l = take(sizeof(uint64_t) * kList), c = take(2 * sizeof(uint32_t));
  uint8_t* p = static_cast<uint8_t*>(work) + (size_t)row * o;
  if (bytes) *bytes = o;
  return {reinterpret_cast<Bins*>(p + b), reinterpret_cast<uint32_t*>(p + t), reinterpret_cast<int*>(p + f),
          reinterpret_cast<uint64_t*>(p + l), reinterpret_cast<uint32_t*>(p + c)};
}

// 1. a tile's maximum and bins. Grid: tiles x rows.
__global__ void __launch_bounds__(kTileThreads) k_tiles(const SampleRowsArgs a) {
  constexpr int NT = kTileThreads, E = kTileEach;
  __shared__ Histogram<NT> h;
  __shared__ uint64_t red[NT / 64 + 3];
  const int tid = threadIdx.x, tile = blockIdx.x, row = blockIdx.y;
  const RowWork w = row_work(a.work, row, gridDim.x, nullptr);
  Chunk<NT, E> c;
  c.load(a.logits + (size_t)row * a.ld, tile * kTile, a.V);
  h.clear();
  const uint32_t mk = group_max<NT>(c.top(), red);
  if (tid == 0) {
    w.top[tile] = mk;
    if (tile == 0) w.count[0] = w.count[1] = 0;
  }
  const float mx = from_order(mk);
  if (mx == -INFINITY) return;
  if (!(a.temperature > 0.0)) {
    const int i = c.first(mx, red);
    if (tid == 0) w.first[tile] = tile * kTile + i;
    return;
  }
  const Scale scale = scale_of(a);
  const float top = scale.bin(mx);
#pragma unroll
  for (int e = 0; e < E; ++e) h.add(c.x[e], top, scale, a.top_k, true);
  __syncthreads();
  if (tid < kBins) h.sum(tid, w.bins[tile].weight[tid], w.bins[tile].count[tid]);
}

// 2. threshold and token. Grid: workgroups of a row x rows.
template <int kMost>   // tiles of a wave, at most
__global__ void __launch_bounds__(kRowThreads) k_draw(const SampleRowsArgs a, int tiles) {
  constexpr int NT = kRowThreads, kWaves = NT / 64;
  using Tile = Chunk<NT, kTile / NT>;
  __shared__ float v[kList];
  __shared__ int at[kList];
  __shared__ Bins bins;
  __shared__ double fall[kBins], kept[kMaxTiles], part[Tile::kRounds * kWaves];
  __shared__ uint64_t red[kWaves + 3], digits[kDigits], edge_kept[kMaxTiles];
  __shared__ uint32_t tops[kMaxTiles], least;
  __shared__ int n;
  __shared__ uint32_t base, done;
  __shared__ bool there[kMaxTiles];   // the tile has entries in the threshold's bin
  __shared__ Edge edge;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.y;
  const int share = blockIdx.x, shares = gridDim.x;
  const RowWork w = row_work(a.work, row, tiles, nullptr);
  const float* x = a.logits + (size_t)row * a.ld;
  for (int t = tid; t < tiles; t += NT) tops[t] = w.top[t];
  if (tid < kBins) {
    fall[tid] = fall_of(tid);
    bins.weight[tid] = 0;
    bins.count[tid] = 0;
  }
  if (tid == 0) n = 0;
  __syncthreads();
  uint32_t mk = 0;
  for (int t = 0; t < tiles; ++t) mk = max(mk, tops[t]);
  const float mx = from_order(mk);
  if (mx == -INFINITY || !(a.temperature > 0.0)) {   // nothing to choose from, or the first maximum
    if (share == 0 && tid == 0) {
      int t = 0;
      while (tops[t] != mk) ++t;
      a.out[row] = mx == -INFINITY ? -1 : w.first[t];
    }
    return;
  }
  const float u = a.u[row];
  const Scale scale = scale_of(a);
  Keep keep = {scale, fall, scale.bin(mx), -INFINITY};
  if (!is_near(keep.top)) {
    if (share) return;
    const int i = slow<NT>(a, x, mx, u, digits, red);
    if (tid == 0) a.out[row] = i;
    return;
  }
  keep.least = least_by_gap(mx, a.min_gap);
  // the tiles' bins, tile t in wave t % kWaves, bins lane and 64 + lane of the row's;
  // a tile's own begin `shift` bins further down
  uint64_t weight[kMost][2];
  uint32_t count[kMost][2];
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int t = wave + k * kWaves;
    int shift = kBins;
    if (t < tiles) {
      const float m = from_order(tops[t]), d = keep.top - scale.bin(m);
      if (m > -INFINITY && d < kBins) shift = (int)d;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = lane + 64 * h - shift;
      weight[k][h] = r >= 0 ? w.bins[t].weight[r] : 0;
      count[k][h] = r >= 0 ? w.bins[t].count[r] : 0;
    }
  }
  if (filtered(a)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint64_t ws = 0;
      uint32_t cs = 0;
#pragma unroll
      for (int k = 0; k < kMost; ++k) {
        ws += weight[k][h];
        cs += count[k][h];
      }
      if (ws) add_u64(&bins.weight[lane + 64 * h], ws);
      if (cs) atomicAdd(&bins.count[lane + 64 * h], cs);
    }
  }
  __syncthreads();
  if (tid < kWave) {
    const Edge f = find_edge(a, bins, keep);
    if (tid == 0) edge = f;
  }
  __syncthreads();
  const Edge e = edge;
  // a tile's weights above the threshold's bin
#pragma unroll
  for (int k = 0; k < kMost; ++k) {
    const int t = wave + k * kWaves;
    if (t >= tiles) break;
    double s = 0.0;
    bool some = false;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = lane + 64 * h;
      if (r < e.r) s += (double)weight[k][h] * (1.0 / kUnit) * fall[r];
      some = some || (r == e.r && weight[k][h] > 0);
    }
    s = wave_upto(s);
    const bool any = __any(some);
    if (lane == 63) {
      kept[t] = s;
      edge_kept[t] = 0;
      there[t] = any;
    }
  }
  __syncthreads();
  if (e.r == kBins && share) return;
  if (e.r < kBins) {
    // that bin's entries: their places into the list, the next rounds' entries
    // requested before these are looked at
    const float bin = keep.top - (float)e.r;
    using Round = Chunk<NT, 4>;
    Round c[2][kRounds];
    auto load = [&](Round (&d)[kRounds], int i0) {
#pragma unroll
      for (int k = 0; k < kRounds; ++k) {
        const int i = i0 + 4 * k * NT;
        if (i < a.V && there[i / kTile]) d[k].load(x, i, a.V);
        else d[k].x[0] = d[k].x[1] = d[k].x[2] = d[k].x[3] = -INFINITY;
      }
    };
    auto look = [&](const Round (&d)[kRounds], int i0) {
      uint32_t hit = 0;   // bit 4k + j
#pragma unroll
      for (int k = 0; k < kRounds; ++k)
#pragma unroll
        for (int j = 0; j < 4; ++j) hit |= floorf(d[k].x[j] * scale.per) == bin ? 1u << (4 * k + j) : 0u;   // (NaN: no)
      if (!__any(hit)) return;
      const uint64_t mine = __popc(hit), upto = wave_upto(mine);
      int p = 0;
      if (lane == 63) p = atomicAdd(&n, (int)upto);   // room for the wave's
      p = __builtin_amdgcn_readlane(p, 63) + (int)(upto - mine);
      for (; hit; hit &= hit - 1, ++p) {
        const int b = __ffs(hit) - 1;
        if (p < kList) at[p] = i0 + 4 * (b / 4) * NT + Round::at(0, b % 4);
      }
    };
    const int step = kStep * shares;
    load(c[0], kStep * share);
    for (int i0 = kStep * share; i0 < a.V; i0 += 2 * step) {
      load(c[1], i0 + step);
      look(c[0], i0);
      load(c[0], i0 + 2 * step);
      look(c[1], i0 + step);
    }
    __syncthreads();
    for (int i = tid; i < min(n, kList); i += NT) v[i] = x[at[i]];
    __syncthreads();
    if (shares > 1) {   // the row's list, from its workgroups' parts
      if (tid == 0) base = n ? __hip_atomic_fetch_add(&w.count[0], (uint32_t)n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0u;
      __syncthreads();
      for (int i = tid; i < min(n, kList); i += NT)
        if (base + i < (uint32_t)kList) cst64(&w.list[base + i], (uint64_t)(uint32_t)at[i] << 32 | __float_as_uint(v[i]));
      vm_drain();   // what this wave published
      __syncthreads();
      if (tid == 0) {
        done = __hip_atomic_fetch_add(&w.count[1], 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + 1;
        if (done == (uint32_t)shares) n = (int)cld(&w.count[0]);
      }
      __syncthreads();
      if (done != (uint32_t)shares) return;
      for (int i = tid; i < min(n, kList); i += NT) {
        const uint64_t y = cld64(&w.list[i]);
        at[i] = (int)(y >> 32);
        v[i] = __uint_as_float((uint32_t)y);
      }
      __syncthreads();
    }
    if (n > kList) {   // more than the list holds: through the row again
      auto in_bin = [&](auto f) {
        over_row<NT>(x, a.V, [&](int i, float y) {
          if (floorf(y * scale.per) == bin) f(i, y);
        });
      };
      if (e.inside()) {
        auto entries = [&](auto f) { in_bin([&](int, float y) { f(y); }); };
        keep.least = fmaxf(keep.least, from_order(least_among<NT>(e, keep, v[0], digits, red, entries)));
      }
      in_bin([&](int i, float y) {
        if (y >= keep.least) add_u64(&edge_kept[i / kTile], scale.units(y, bin));
      });
    } else {
      if (e.inside())   // (else min-p alone cuts there)
        keep.least = fmaxf(keep.least, from_order(least_of<NT>(e, keep, v, n, digits, red, &least)));
      for (int i = tid; i < n; i += NT)
        if (v[i] >= keep.least) add_u64(&edge_kept[at[i] / kTile], scale.units(v[i], bin));
    }
    __syncthreads();
    for (int t = tid; t < tiles; t += NT) kept[t] += (double)edge_kept[t] * (1.0 / kUnit) * fall[e.r];
    __syncthreads();
  }
  double total = 0.0, before = 0.0;
  int held = 0;   // the last tile with a weight
  for (int t = 0; t < tiles; ++t) {
    total += kept[t];
    if (kept[t] > 0.0) held = t;
  }
  const double target = fraction(u) * total;
  int t = 0;
  while (t < held && !(target < before + kept[t])) before += kept[t++];
  Tile c;
  c.load(x, t * kTile, a.V);
  const int i = c.pick(keep, before, target, false, part, red);
  if (tid == 0) a.out[row] = t * kTile + i;
}

int tiles_of(int V) { return V <= kOne ? 0 : (V + kTile - 1) / kTile; }
// workgroups of a row in the second launch
int shares_of(int rows, int V, int n_cu) {
  const int steps = (V + kStep - 1) / kStep, room = 2 * n_cu / rows;
  return steps < 4 || room < 2 ? 1 : steps < room ? steps : room;
}

}  // namespace

size_t sample_rows_workspace(int rows, int V) {
  size_t bytes = 0;
  if (const int tiles = tiles_of(V)) row_work(nullptr, 0, tiles, &bytes);
  return bytes * rows;
}

hipError_t launch_sample_rows(const SampleRowsArgs& a, hipStream_t s) {
  if (a.rows < 1 || a.V < 1 || a.V > kSampleRowsMaxV) return hipErrorInvalidValue;
  if (const int tiles = tiles_of(a.V)) {
    hipLaunchKernelGGL(k_tiles, dim3(tiles, a.rows), dim3(kTileThreads), 0, s, a);
    const dim3 grid(shares_of(a.rows, a.V, a.n_cu), a.rows), block(kRowThreads);
    if (tiles <= 16)
      hipLaunchKernelGGL(k_draw<2>, grid, block, 0, s, a, tiles);
    else if (tiles <= 32)
      hipLaunchKernelGGL(k_draw<4>, grid, block, 0, s, a, tiles);
    else
      hipLaunchKernelGGL(k_draw<kMaxTiles * 64 / kRowThreads>, grid, block, 0, s, a, tiles);
  } else if (a.V <= 8 * kOneThreads) {
    hipLaunchKernelGGL(k_one<8>, dim3(a.rows), dim3(kOneThreads), 0, s, a);
  } else {
    hipLaunchKernelGGL(k_one<16>, dim3(a.rows), dim3(kOneThreads), 0, s, a);
  }
  return hipGetLastError();
}

}  // namespace ssk
