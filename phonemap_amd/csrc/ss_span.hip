// ss_span.hip - attention over a sliding window with first tokens that stay
// visible, and of several sequences over a prefix they share (ss_span.h), for
// few rows: a decode step.
//
// Work. A tile of query rows that share a KV head walks the blocks of 32 keys
// that some row of it sees. The blocks are dealt to `slots` workgroups and to
// the waves of each in turn, so every wave has its own softmax; a workgroup
// joins its waves through LDS, and k_span_join the slots. The sequences' rows
// over their own caches (8 rows or fewer that share K and V) and tiles of all
// sequences' rows over the prefix are workgroups of the same launch; where both
// caches are short a sequence's rows go through both in one workgroup.
//
// No LDS in the loop: K and V come from memory straight into the operands of
// v_mfma_f32_16x16x32_f16 (lane l = (n, kq) = (l % 16, l / 16) supplies
// A[n][8kq + i] and B[8kq + i][n], i = 0..7, and receives D[4kq + j][n]).
// S^T = K Q^T takes 16 keys' rows as A: lane (n, kq) loads 16 bytes of row n.
// Row 4u + j of tile t (of 2) is key 8u + 4t + j of the block, so lane (n, kq)
// receives the scores of keys 8kq .. 8kq + 7 of query row n, which are what
// O^T = V^T P^T wants of it as B. There lane (n, kq) supplies V^T[n][keys 8kq ..
// 8kq + 7]: it loads its DPL = HD / 16 dimensions DPL n .. of each of these 8
// keys (a load covers whole rows), and a v_perm per two values turns them
// round; tile j of DPL is then dimension DPL m + j. K of the next block is
// requested as soon as the current one's is used up, V during the next scores.
//
// Precision is that of the prompt rows' kernel (ss_flash.h): K and V exact, q
// and the weights as two fp16 parts, whole-number maxima in base 2, fp32 sums.
// With 8 rows or fewer (PACK) the two parts are two columns of one product, n and
// n + 8, whose results are added; more rows take two products.
//
// Reads past a span's end go through a buffer view that ends there and give 0.

#include <type_traits>

#include "ss_mfma.h"
#include "ss_span.h"

namespace ssk {
namespace {

// value of the lane 16 away (lane ^ 16) joined to this one's
__device__ __forceinline__ float max_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_8(float v) {   // row_ror:8: lane ^ 8
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), 0x128, 0xf, 0xf, true));
}
// a barrier for what is in LDS: loads from memory stay in flight
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}
// maximum over aligned groups of N lanes
template <int N>
__device__ __forceinline__ float max_lanes(float v) {
  static_assert(N == 8 || N == 16 || N == 32, "");
  v = fmaxf(v, dpp<0xb1>(v));
  v = fmaxf(v, dpp<0x4e>(v));
  v = fmaxf(v, dpp<0x141>(v));
  if constexpr (N >= 16) v = fmaxf(v, dpp<0x140>(v));
  if constexpr (N >= 32) v = max_16(v);
  return v;
}

// hi + lo = v as split8 of ss_mfma.h does, less: -1
__device__ __forceinline__ void split8(const float* v, v8h& hi, v8h& lo, float less) {
#pragma unroll
  for (int i = 0; i < 8; ++i) hi[i] = (_Float16)v[i];
  v4u h = __builtin_bit_cast(v4u, hi);
  asm("" : "+v"(h));   // (pairs, not converted a second time one by one)
  hi = __builtin_bit_cast(v8h, h);
#pragma unroll
  for (int i = 0; i < 8; ++i) lo[i] = (_Float16)__builtin_fmaf((float)hi[i], less, v[i]);
}

// f(0), .., f(N - 1), of constants
template <int N, int I = 0, class F>
__device__ __forceinline__ void each(const F& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<N, I + 1>(f);
  }
}

// The tile's rows: row r is query head g of token or sequence t, t * G + g = r0 + r < r1.
struct Rows {
  int r0, r1, kvh;
};

// One block's K and V of a wave
template <int HD, int KVT>
struct Block {
  static constexpr int kRowB = HD * (KVT == 0 ? 2 : 1);
  static constexpr int kKLoads = kRowB / 64;             // 16-byte loads of a K row's share
  static constexpr int kVWords = HD / 16 * (KVT == 0 ? 2 : 1) / 4;
  v4u k[2][kKLoads];
  uint32_t v[8][kVWords];
  float ks[KVT ? 8 : 1], vs[KVT ? 8 : 1];

  static __device__ __forceinline__ __amdgpu_buffer_rsrc_t view(const void* p, size_t from, int bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(static_cast<const uint8_t*>(p) + from), (short)0, bytes,
                                             kBufferFlags);
  }
  __device__ __forceinline__ void load_k(const Base& w, int key, int limit, int n, int kq) {
    const int live = min(limit - key, kKeys);
    const auto r = view(w.k, (size_t)key * kRowB, live * kRowB);
    const int at = (8 * (n >> 2) + (n & 3)) * kRowB + 16 * kq;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int c = 0; c < kKLoads; ++c)
        k[t][c] = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, at + 4 * t * kRowB + 64 * c, 0, 0));
    if constexpr (KVT == 1) scales(w.ks, key, live, kq, ks);
  }
  // this lane's keys 8kq + FROM .. 8kq + TO - 1, and with the first the scales of all 8
  template <int FROM, int TO>
  __device__ __forceinline__ void load_v(const Base& w, int key, int limit, int n, int kq) {
    const int live = min(limit - key, kKeys);
    const auto r = view(w.v, (size_t)key * kRowB, live * kRowB);
    const int at = 8 * kq * kRowB + 4 * kVWords * n;
#pragma unroll
    for (int i = FROM; i < TO; ++i) {
      if constexpr (kVWords == 1) {
        v[i][0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, at + i * kRowB, 0, 0);
      } else if constexpr (kVWords == 2) {
        const auto x = __builtin_amdgcn_raw_buffer_load_b64(r, at + i * kRowB, 0, 0);
        v[i][0] = x[0];
        v[i][1] = x[1];
      } else {
#pragma unroll
        for (int c = 0; c < kVWords / 4; ++c) {
          const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, at + i * kRowB + 16 * c, 0, 0));
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][4 * c + e] = x[e];
        }
      }
    }
    if constexpr (KVT == 1 && FROM == 0) scales(w.vs, key, live, kq, vs);
  }
  static __device__ __forceinline__ void scales(const float* p, int key, int live, int kq, float (&s)[KVT ? 8 : 1]) {
    const auto r = view(p, (size_t)key * 4, live * 4);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const v4u x = __builtin_bit_cast(v4u, __builtin_amdgcn_raw_buffer_load_b128(r, 32 * kq + 16 * c, 0, 0));
#pragma unroll
      for (int e = 0; e < 4; ++e) s[(4 * c + e) % (KVT ? 8 : 1)] = __uint_as_float(x[e]);
    }
  }
  // slice c (32 dimensions) of the K rows of tile t
  __device__ __forceinline__ v8h k_slice(int t, int c) const {
    if constexpr (KVT == 0) {
      return __builtin_bit_cast(v8h, k[t][c]);
    } else {
      const v4u x = k[t][c / 2];
      return __builtin_bit_cast(v8h, c % 2 ? codes8(x[2], x[3]) : codes8(x[0], x[1]));
    }
  }
  // dimension j of this lane's, keys 8kq .. 8kq + 7
  __device__ __forceinline__ v8h v_tile(int j) const {
    v4u r;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      if constexpr (KVT == 0) {
        r[p] = __builtin_amdgcn_perm(v[2 * p + 1][j / 2], v[2 * p][j / 2], j % 2 ? 0x07060302u : 0x05040100u);
      } else {   // 1024 + (code + 128) by placing the byte, less 1152
        const v2h off = {(_Float16)1152.f, (_Float16)1152.f};
        const uint32_t x = __builtin_amdgcn_perm(v[2 * p + 1][j / 4] ^ 0x80808080u, v[2 * p][j / 4] ^ 0x80808080u,
                                                 0x0c040c00u + 0x00010001u * (j % 4));
        r[p] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, x | 0x64006400u) - off);
      }
    }
    return __builtin_bit_cast(v8h, r);
  }
};
// the dimension that element i of lane kq's slice c stands for
template <int KVT>
__device__ __forceinline__ int slice_dim(int c, int kq) {
  return KVT == 0 ? 32 * c + 8 * kq : 64 * (c / 2) + 16 * kq + 8 * (c % 2);
}

__host__ __device__ constexpr int tile_rows(int rt) { return rt == 0 ? 8 : 16 * rt; }
constexpr int kW = 4, kWide = 8;   // waves of a workgroup, of k_span_each's
// and at most that many per SIMD, by their registers
__host__ __device__ constexpr int simd_waves(int hd) { return hd < 256 ? 2 : 1; }

// A workgroup's LDS: first q, its parts as rows (n and rows + n) in the order of
// the products' operand; then the waves' results.
template <int HD, int RT, int W = kW>
union Joint {
  static constexpr int kRows = tile_rows(RT);
  struct {
    _Float16 part[2 * kRows][HD + 8];
    float scale[kRows];
  } q;
  struct {
    float o[W][kRows][HD + 4];
    float m[W][kRows], l[W][kRows], e[W][kRows];
  } r;
};

// A tile of rows over the walk's blocks b with b / kW % slots == slot, by the
// workgroup's waves: the rows' outputs (part null), or the slot's share of them,
// at part[row of all rows][HD] and ml[row], to be joined. RT 0: 8 rows or fewer
// in one product; else RT tiles of 16.
template <int HD, int KVT, int RT, bool CAP, int W = kW, class Walks, class Masks>
__device__ __forceinline__ void span_tile(const SpanArgs& a, const Rows& rows, const Walks& w, int slot, int slots, float* part,
                                          float2* ml, Joint<HD, RT, W>& sh, Masks masks) {
  constexpr bool PACK = RT == 0;
  constexpr int kRows = tile_rows(RT), NT = PACK ? 1 : RT, NC = HD / 32, DPL = HD / 16;
  using Blk = Block<HD, KVT>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, kq = lane >> 4;
  const int b0 = slot * W + wave, step = slots * W;

  // the tile's q, 8 values a thread, requested ahead of the first block
  constexpr int kChunks = kRows * HD / 8, kTurns = (kChunks + W * 64 - 1) / (W * 64);
  static_assert(kChunks % 64 == 0, "whole waves");
  float qv[kTurns][8];
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int i = tid + u * W * 64, row = rows.r0 + i / (HD / 8);
    if (i < kChunks) {
      const float* qp = a.q + row_head(a, rows.kvh, min(row, rows.r1 - 1)) * HD + i % (HD / 8) * 8;
      const float4 x0 = *reinterpret_cast<const float4*>(qp), x1 = *reinterpret_cast<const float4*>(qp + 4);
      qv[u][0] = x0.x, qv[u][1] = x0.y, qv[u][2] = x0.z, qv[u][3] = x0.w;
      qv[u][4] = x1.x, qv[u][5] = x1.y, qv[u][6] = x1.z, qv[u][7] = x1.w;
    }
  }
  __builtin_amdgcn_sched_barrier(0);
  // (a wave without a block, or past its last, loads from an empty view: no
  // branch, so a wait counts the loads behind the one it is for)
  Blk blk;
  int key = 0, limit = 0;
  Base at0;   // where the block's cache lies
  auto next = [&](int b) {
    w.block(b, key, limit);
    at0 = w.base(b);
    if (b >= w.nb) key = limit = 0;
  };
  next(b0);
  blk.load_k(at0, key, limit, n, kq);
  blk.template load_v<0, 8>(at0, key, limit, n, kq);
  __builtin_amdgcn_sched_barrier(0);

  // q times the softmax's scale and log2 e, a row's largest magnitude brought to
  // [2^13, 2^14), in two parts
#pragma unroll
  for (int u = 0; u < kTurns; ++u) {
    const int i = tid + u * W * 64, r = i / (HD / 8), c = i % (HD / 8);
    if (i < kChunks) {
      const bool live = rows.r0 + r < rows.r1;
      float amax = 0.f;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        qv[u][k] = live ? qv[u][k] : 0.f;
        amax = fmaxf(amax, fabsf(qv[u][k]));
      }
      amax = max_lanes<HD / 8>(amax);
      int e = 0;
      const float c0 = CAP ? a.scale : a.scale * kLog2e;
      const float c1 = CAP ? 0.f : __builtin_fmaf(a.scale, kLog2e, -c0) + a.scale * kLog2eLow;
      frexpf(amax * c0, &e);
      const int shift = min(max(14 - e, -100), 100);
      const float s0 = ldexpf(c0, shift), s1 = ldexpf(c1, shift);
      if (c == 0) sh.q.scale[r] = ldexpf(1.0f, -shift);   // S^T holds the scores * 2^shift
      v8h hi, lo;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        float p = qv[u][k] * s0;
        asm("" : "+v"(p));   // one value for both parts
        hi[k] = (_Float16)p;
        lo[k] = (_Float16)__builtin_fmaf(qv[u][k], s1, __builtin_fmaf(qv[u][k], s0, -(float)hi[k]));
      }
      *reinterpret_cast<v8h*>(&sh.q.part[r][8 * c]) = hi;
      *reinterpret_cast<v8h*>(&sh.q.part[kRows + r][8 * c]) = lo;
    }
  }
  lds_barrier();
  // row n of each tile as B (PACK: rows 8 .. 15 are the low parts)
  v8h qh[NT][NC], ql[PACK ? 1 : NT][PACK ? 1 : NC];
  float qscale[NT];
  int row[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int r = PACK ? n & 7 : 16 * t + n;
    row[t] = rows.r0 + r;
    qscale[t] = sh.q.scale[r];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      qh[t][c] = *reinterpret_cast<const v8h*>(&sh.q.part[PACK ? n : r][slice_dim<KVT>(c, kq)]);
      if constexpr (!PACK) ql[t][c] = *reinterpret_cast<const v8h*>(&sh.q.part[kRows + r][slice_dim<KVT>(c, kq)]);
    }
  }
  lds_barrier();   // (the waves' results take q's place)

  v4f o[NT][DPL];
  float m[NT], l[NT], ex[NT];   // running maximum, this lane's share of the sum; int8: O's exponent, times 2^12
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = ex[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[t][j] = v4f{};
  }

  float less = -1.f;   // (in a register: what is left of a value is one mixed fma)
  asm("" : "+s"(less));
  // Block b. Its V is requested between its scores' products, the first one's
  // ahead of them; the next one's K behind them. (Both at once, when their
  // registers are free: 37 sequences, int8, 24.8 us instead of 24.3; 24 sequences
  // over 8000 positions 24.8 and 24.3. K between the softmax's steps too: 64 over
  // 32000 114 instead of 111.)
  auto block = [&](int b, auto first) {
    constexpr bool FIRST = decltype(first)::value;
    // the scores of keys key + 8kq + 0 .. 7
    // (the chains of products in turn: one waits for its own last)
    float sc[NT][8];
    v4f d[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t) d[t][0] = d[t][1] = v4f{};
    constexpr int kGroups = (PACK ? 1 : 2) * NC * 2;   // of NT products
    auto group = [&](auto gi) {
      constexpr int i = decltype(gi)::value, c = i / 2 % NC, u = i % 2;
      constexpr bool low = !PACK && i < NC * 2;
#pragma unroll
      for (int t = 0; t < NT; ++t)
        d[t][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(blk.k_slice(u, c), low ? ql[PACK ? 0 : t][PACK ? 0 : c] : qh[t][c],
                                                         d[t][u], 0, 0, 0);
      if constexpr (!FIRST && (i + 1) * 8 / kGroups > i * 8 / kGroups) {
        blk.template load_v<i * 8 / kGroups, (i + 1) * 8 / kGroups>(at0, key, limit, n, kq);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    each<kGroups>(group);
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sc[t][i] = PACK ? d[t][i / 4][i % 4] + swap_8(d[t][i / 4][i % 4]) : d[t][i / 4][i % 4];
        if constexpr (KVT == 1) sc[t][i] *= blk.ks[i];
      }
    const int at = key, end = limit;
    __builtin_amdgcn_sched_barrier(0);
    next(b + step);
    blk.load_k(at0, key, limit, n, kq);
    __builtin_amdgcn_sched_barrier(0);

    // the softmax of all tiles in straight code but for what happens seldom: a
    // block that some row does not see in full, a maximum that grows past the lag
    float vsc[KVT ? 8 : 1];
    if constexpr (KVT == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) vsc[i] = blk.vs[i];
    }
    if constexpr (CAP) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[t][i] = span_cap(sc[t][i] * qscale[t], a);
    }
    uint32_t hidden[NT];   // int8: bit i, this lane's key i is not seen (its V scale may be infinite)
#pragma unroll
    for (int t = 0; t < NT; ++t) hidden[t] = 0;
    if (masks.some(at, end)) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (masks.hides(at + 8 * kq + i, end, row[t])) {
            sc[t][i] = -INFINITY;
            hidden[t] |= 1u << i;
          }
    }
    float qs[NT], bmax[NT];
    bool grows = false;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      qs[t] = CAP ? kLog2e : qscale[t];
      bmax[t] = sc[t][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) bmax[t] = fmaxf(bmax[t], sc[t][i]);
      bmax[t] *= qs[t];
      grows = grows || bmax[t] > m[t] + kLag;
    }
    if (__any(grows)) {   // (the row's other lanes are asked only now)
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        bmax[t] = max_pair(max_16(bmax[t]));
        const float mn = ceilf(bmax[t] > m[t] + kLag ? fmaxf(m[t], bmax[t]) : m[t]);
        const float corr = pow2(m[t] - (mn == -INFINITY ? 0.f : mn));
        l[t] *= corr;
        if (KVT == 0 && !FIRST) {   // (nothing there yet)
#pragma unroll
          for (int j = 0; j < DPL; ++j) o[t][j] *= corr;
        }
        m[t] = mn;
      }
    }
    float pv[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // fp16: times 2^12, for the lower part's range (int8: below, by its exponent)
      const float mo = (m[t] == -INFINITY ? 0.f : m[t]) - (KVT == 0 ? kPExp : 0.f);
#pragma unroll
      for (int i = 0; i < 8; ++i) pv[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], qs[t], -mo));
      l[t] += ((pv[t][0] + pv[t][4]) + (pv[t][1] + pv[t][5])) + ((pv[t][2] + pv[t][6]) + (pv[t][3] + pv[t][7]));
    }
    if constexpr (KVT == 1) {
      float bx[NT];
      bool up = false;
      auto exponent = [](float b, float mt) { return mt + (float)max((int)(__float_as_uint(b) >> 23) - 127, -100); };
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        bx[t] = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pv[t][i] *= hidden[t] >> i & 1 ? 0.f : vsc[i];
          bx[t] = fmaxf(bx[t], pv[t][i]);
        }
        up = up || (bx[t] > 0.f && exponent(bx[t], m[t]) > ex[t] + kLagX);
      }
      if (__any(up)) {
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          bx[t] = max_pair(max_16(bx[t]));   // below 2^(e + 1)
          const float x = exponent(bx[t], m[t]);
          const float en = bx[t] > 0.f && x > ex[t] + kLagX ? x : ex[t];
          const float corr = en == ex[t] ? 1.f : pow2(ex[t] - en);
#pragma unroll
          for (int j = 0; j < DPL; ++j) o[t][j] *= corr;
          ex[t] = en;
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int to = (int)fminf(kPExp + m[t] - ex[t], 126.f);   // (past 126 with every pv 0 only)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pv[t][i] = ldexpf(pv[t][i], to);
          asm("" : "+v"(pv[t][i]));   // rounded to fp32 before it is split
        }
      }
    }
    v8h ph[NT], pl[PACK ? 1 : NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      if constexpr (PACK) {
        v8h hi, lo;
        split8(pv[t], hi, lo, less);
#pragma unroll
        for (int i = 0; i < 8; ++i) ph[t][i] = n < 8 ? hi[i] : lo[i];
      } else {
        split8(pv[t], ph[t], pl[t], less);
      }
    }
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      const v8h vt = blk.v_tile(j);
#pragma unroll
      for (int t = 0; t < NT; ++t)
        if constexpr (!PACK) o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, pl[t], o[t][j], 0, 0, 0);
#pragma unroll
      for (int t = 0; t < NT; ++t) o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, ph[t], o[t][j], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
  };
  if (b0 < w.nb) block(b0, std::true_type{});
#pragma unroll 1
  for (int b = b0 + step; b < w.nb; b += step) block(b, std::false_type{});

  // the waves' rows -> one
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] = sum_pair(sum_16(l[t])) * (KVT == 0 ? 1 / kPScale : 1.f);
    if constexpr (PACK) {
#pragma unroll
      for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[t][j][r] += swap_8(o[t][j][r]);
    }
    const int at = PACK ? n & 7 : 16 * t + n;
    if (!PACK || n < 8) {
      if (kq == 0) {
        sh.r.m[wave][at] = m[t];
        sh.r.l[wave][at] = l[t];
        sh.r.e[wave][at] = KVT == 1 ? ex[t] : m[t];
      }
      float* dst = &sh.r.o[wave][at][4 * DPL * kq];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < DPL; j += 4)
          *reinterpret_cast<float4*>(dst + DPL * r + j) = make_float4(o[t][j][r], o[t][j + 1][r], o[t][j + 2][r], o[t][j + 3][r]);
    }
  }
  __syncthreads();
  constexpr int kQuads = HD / 4;
  static_assert(kRows * kQuads % 64 == 0, "whole waves");
  for (int i = tid; i < kRows * kQuads; i += W * 64) {
    const int r = i / kQuads, c = i % kQuads, all = rows.r0 + r;
    const bool live = all < rows.r1;
    float mx = -INFINITY, lt = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) mx = fmaxf(mx, sh.r.m[k][r]);
    const float mo = mx == -INFINITY ? 0.f : mx;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      lt += sh.r.l[k][r] * pow2(sh.r.m[k][r] - mo);
      const float f = pow2(sh.r.e[k][r] - kPExp - mo);
      const float4 v = *reinterpret_cast<const float4*>(&sh.r.o[k][r][4 * c]);
      s.x += v.x * f;
      s.y += v.y * f;
      s.z += v.z * f;
      s.w += v.w * f;
    }
    const size_t head = row_head(a, rows.kvh, all);
    if (part) {
      // (a slot in which a row has no key, or -inf scores only, has the maximum
      // -inf and is not read; one with a NaN weighs in)
      if (live && c == 0) ml[head] = make_float2(lt != lt ? 0.f : mx, lt);
      if (live) reinterpret_cast<float4*>(part + head * HD)[c] = s;
    } else {
      const float f = w.nb == 0 ? 0.f : 1.f / lt;   // no position at all: 0
      s = make_float4(s.x * f, s.y * f, s.z * f, s.w * f);
      if (live) reinterpret_cast<float4*>(a.out + head * HD)[c] = s;
      mend_rows<HD, KVT>(a, live, s, head);
    }
  }
}

// Keys at or past the block's end are not there.
struct TailMask {
  __device__ __forceinline__ bool some(int key, int limit) const { return key + kKeys > limit; }
  __device__ __forceinline__ bool hides(int key, int limit, int row) const { return key >= limit; }
};
// Rows of several tokens: row r's token sees its own window alone.
struct WindowMask {
  int gs, pos0, window, sinks, t0, t1;   // the tile's first and last token
  __device__ __forceinline__ bool some(int key, int limit) const {
    return key + kKeys > limit || key + kKeys - 1 > pos0 + t0 || (key <= pos0 + t1 - window && key + kKeys > sinks);
  }
  __device__ __forceinline__ bool hides(int key, int limit, int row) const {
    const int lim = pos0 + min(row >> gs, t1);
    return key >= limit || key > lim || (key <= lim - window && key >= sinks);
  }
};

// Grid: n_kv_heads x slots x tiles of rows.
template <int HD, int KVT, int RT, bool CAP>
__global__ void __launch_bounds__(kW * 64, simd_waves(HD)) k_span_window(const SpanArgs a, int slots) {
  __shared__ Joint<HD, RT> sh;
  int i = blockIdx.x;
  const int kvh = i % a.n_kv_heads;
  i /= a.n_kv_heads;
  const int slot = i % slots, tile = i / slots, rows = a.n * a.n_kv_heads << a.gs;
  const int r0 = tile * tile_rows(RT);
  const Rows r = {r0, min(r0 + tile_rows(RT), a.n << a.gs), kvh};
  const int t0 = r.r0 >> a.gs, t1 = (r.r1 - 1) >> a.gs, end = a.pos0 + t1 + 1;   // its tokens
  Walk w;
  const size_t base = (size_t)kvh * a.max_seq * Block<HD, KVT>::kRowB;
  w.k = static_cast<const uint8_t*>(a.kc) + base;
  w.v = static_cast<const uint8_t*>(a.vc) + base;
  w.ks = a.ks;
  w.vs = a.vs;
  w.to0 = min(a.sinks, end);
  w.from1 = max(w.to0, a.pos0 + t0 + 1 - a.window);
  w.to1 = end;
  w.nb0 = blocks_of(w.to0);
  w.nb = w.nb0 + blocks_of(w.to1 - w.from1);
  float* part = slots > 1 ? slot_part<HD>(a, rows, slot) : nullptr;
  float2* ml = slot_ml<HD>(a, rows, slots, slot);
  if (a.n == 1)
    span_tile<HD, KVT, RT, CAP>(a, r, w, slot, slots, part, ml, sh, TailMask{});
  else
    span_tile<HD, KVT, RT, CAP>(a, r, w, slot, slots, part, ml, sh, WindowMask{a.gs, a.pos0, a.window, a.sinks, t0, t1});
}

// Grid: n_kv_heads x np x tiles of rows over the prefix, then n_kv_heads x no x
// sequences over their own caches; slots 0 .. np - 1 are the prefix's.
template <int HD, int KVT, int RT, bool CAP>
__global__ void __launch_bounds__(kW * 64, simd_waves(HD)) k_span_shared(const SpanArgs a, int np, int no, int tiles) {
  __shared__ union {
    Joint<HD, RT> tile;
    Joint<HD, 0> own;
  } sh;
  const int slots = np + no, rows = a.n * a.n_kv_heads << a.gs;
  int i = blockIdx.x;
  const int kvh = i % a.n_kv_heads;
  i /= a.n_kv_heads;
  Walk w;
  w.to0 = w.nb0 = w.from1 = 0;
  if (i < np * tiles) {
    const int slot = i % np, tile = i / np;
    const size_t base = (size_t)kvh * a.max_seq * Block<HD, KVT>::kRowB;
    w.k = static_cast<const uint8_t*>(a.kc) + base;
    w.v = static_cast<const uint8_t*>(a.vc) + base;
    w.ks = a.ks;
    w.vs = a.vs;
    w.to1 = a.prefix;
    w.nb = blocks_of(w.to1);
    const int r0 = tile * tile_rows(RT);
    const Rows r = {r0, min(r0 + tile_rows(RT), a.n << a.gs), kvh};
    span_tile<HD, KVT, RT, CAP>(a, r, w, slot, np, slots > 1 ? slot_part<HD>(a, rows, slot) : nullptr,
                              slot_ml<HD>(a, rows, slots, slot), sh.tile, TailMask{});
  } else {
    i -= np * tiles;
    const int slot = i % no, t = i / no;
    const size_t base = ((size_t)t * a.n_kv_heads + kvh) * a.own_max * Block<HD, KVT>::kRowB;
    w.k = static_cast<const uint8_t*>(a.ko) + base;
    w.v = static_cast<const uint8_t*>(a.vo) + base;
    w.ks = a.kos + (size_t)t * a.own_max;
    w.vs = a.vos + (size_t)t * a.own_max;
    w.to1 = own_length(a, t);
    w.nb = blocks_of(w.to1);
    const Rows r = {t << a.gs, t + 1 << a.gs, kvh};
    span_tile<HD, KVT, 0, CAP>(a, r, w, slot, no, slots > 1 ? slot_part<HD>(a, rows, np + slot) : nullptr,
                             slot_ml<HD>(a, rows, slots, np + slot), sh.own, TailMask{});
  }
}

// The prefix's blocks, then a sequence's own.
struct SharedWalk : Walk {
  Base own;
  __device__ __forceinline__ Base base(int b) const { return b < nb0 ? Base(*this) : own; }
};
// A sequence's rows over both caches in one workgroup. Grid: n_kv_heads x sequences.
template <int HD, int KVT, bool CAP>
__global__ void __launch_bounds__(kWide * 64, simd_waves(HD)) k_span_each(const SpanArgs a) {
  __shared__ Joint<HD, 0, kWide> sh;
  const int kvh = blockIdx.x % a.n_kv_heads, t = blockIdx.x / a.n_kv_heads;
  const size_t base = (size_t)kvh * a.max_seq * Block<HD, KVT>::kRowB;
  const size_t own = ((size_t)t * a.n_kv_heads + kvh) * a.own_max * Block<HD, KVT>::kRowB;
  SharedWalk w;
  w.k = static_cast<const uint8_t*>(a.kc) + base;
  w.v = static_cast<const uint8_t*>(a.vc) + base;
  w.ks = a.ks;
  w.vs = a.vs;
  w.own.k = static_cast<const uint8_t*>(a.ko) + own;
  w.own.v = static_cast<const uint8_t*>(a.vo) + own;
  w.own.ks = a.kos + (size_t)t * a.own_max;
  w.own.vs = a.vos + (size_t)t * a.own_max;
  w.to0 = a.prefix;
  w.from1 = 0;
  w.to1 = own_length(a, t);
  w.nb0 = blocks_of(w.to0);
  w.nb = w.nb0 + blocks_of(w.to1);
  const Rows r = {t << a.gs, t + 1 << a.gs, kvh};
  span_tile<HD, KVT, 0, CAP, kWide>(a, r, w, 0, 1, nullptr, nullptr, sh, TailMask{});
}

// The slots' shares -> outputs: a thread takes four outputs of a row from every
// `groups`-th slot, and the groups of a row meet in LDS.
constexpr int kJoinThreads = 256;
template <int HD, int KVT>
__global__ void __launch_bounds__(kJoinThreads) k_span_join(const SpanArgs a, int slots, int groups) {
  constexpr int kQuads = HD / 4;
  __shared__ float4 so[kJoinThreads];
  __shared__ float2 sml[kJoinThreads];
  const int tid = threadIdx.x, c = tid % kQuads, g = tid / kQuads % groups;
  const int rows = a.n * a.n_kv_heads << a.gs;
  const int64_t at = (int64_t)blockIdx.x * (kJoinThreads / kQuads / groups) + tid / kQuads / groups;
  const bool live = at < rows;
  const int row = live ? (int)at : rows - 1;
  const float2* ml = slot_ml<HD>(a, rows, slots, 0) + row;
  const float4* part = reinterpret_cast<const float4*>(a.part + (size_t)row * HD) + c;
  float mx = -INFINITY, lt = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 x, float4 v) {   // (m, l) and values held relative to m
    const float mn = fmaxf(mx, x.x), mo = mn == -INFINITY ? 0.f : mn;
    const float f0 = pow2(mx - mo), f1 = pow2(x.x - mo);
    lt = lt * f0 + x.y * f1;
    o = make_float4(o.x * f0 + v.x * f1, o.y * f0 + v.y * f1, o.z * f0 + v.z * f1, o.w * f0 + v.w * f1);
    mx = mn;
  };
  for (int s0 = g; s0 < slots; s0 += 4 * groups) {
    float2 x[4];
    float4 v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {   // (past the last: the last again, not added)
      const int s = min(s0 + k * groups, slots - 1);
      x[k] = ml[(size_t)s * rows];
      v[k] = part[(size_t)s * rows * kQuads];
    }
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (s0 + k * groups < slots) add(x[k], v[k]);
  }
  if (groups > 1) {
    so[tid] = o;
    sml[tid] = make_float2(mx, lt);
    __syncthreads();
    if (g == 0)
      for (int k = 1; k < groups; ++k) add(sml[tid + k * kQuads], so[tid + k * kQuads]);
  }
  const bool store = live && g == 0;
  bool none = false;
  if (a.own_len) none = a.prefix == 0 && own_length(a, row / (a.n_kv_heads << a.gs)) == 0;
  const float f = none ? 0.f : 1.f / lt;
  o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
  if (store) reinterpret_cast<float4*>(a.out + (size_t)row * HD)[c] = o;
  mend_rows<HD, KVT>(a, store, o, (size_t)row);
}

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a call is cut: rt (tile_rows), tiles of rows, slots of the window or the
// prefix (np) and of the own caches (no). rt -1: a window's rows for the prompt
// rows' kernel (ss_flash_span.hip).
struct Plan {
  int rt, tiles, np, no;
  bool each = false;   // k_span_each
};
int rt_of(int hd, int64_t rows) { return rows <= 8 ? 0 : rows <= 16 || hd == 256 ? 1 : 2; }
// workgroups that a device holds at once
int64_t room(int hd, int n_cu) { return (int64_t)n_cu * simd_waves(hd); }

// Blocks that a wave should walk when `rows` query rows of nb blocks are left to
// slots: a block takes a wave some 0.35 us, and a slot's share costs a row 0.26 ns
// to write and to join (head_dim 128), so nb / (4 each) slots are cheapest at each
// = sqrt(nb rows hd / 128 * 1.9e-4). In us: 1 token, 33 blocks, 32 rows 7.9 with
// one block each, 8.5 with two; 9 tokens, 131 blocks, 288 rows 17.1 and 15.6; 77
// tokens, 34 blocks, 1232 rows at head_dim 256 31.3, two 26.6, four 20.4, eight 25.6.
double blocks_each(int hd, int64_t nb, int64_t rows) { return sqrt((double)nb * (double)rows * hd / 128 * 1.9e-4); }
int slots_of(int64_t nb, double each, int64_t most) {
  if (each < 1.0) each = 1.0;
  // up to three blocks per wave a single slot does without the join (9 blocks 5.9
  // us, in three slots 7.6)
  if (nb <= 3 * kW || most <= 1) return nb > 0 ? 1 : 0;
  const int64_t want = (int64_t)ceil((double)nb / (kW * each));
  return (int)(want < 1 ? 1 : want < most ? want : most);
}

// The blocks of a window's call above which the prompt rows' kernel, whose waves
// share K and V, takes it: many per wave (512 tokens over 4096 positions, 32 heads
// on 8: 78 us, this file's 82; 100 tokens 31 and 36; 32 tokens 21 and 19; 100
// tokens over 300 positions 17 and 11).
int64_t span_blocks(int tiles, int n_kv_heads, int n_cu) {
  return tiles > 1 ? (int64_t)n_cu * 4 * 8 / ((int64_t)tiles * n_kv_heads) : INT64_MAX;
}

// first, rest: the positions of the two spans that the window's rows see between them
Plan plan_window(int hd, int group, int n_kv_heads, int n, int64_t first, int64_t rest, int n_cu) {
  const int64_t rows = (int64_t)n * group;
  Plan p = {rt_of(hd, rows), 1, 1, 0};
  const int tile = tile_rows(p.rt), tokens = tile < rows ? (tile + group - 1) / group : n;
  p.tiles = up(rows, tile);
  // a tile's tokens see as many positions less than all of them
  const int64_t nb = up(first, kKeys) + up(rest - (n - tokens) > 0 ? rest - (n - tokens) : 0, kKeys) + (p.tiles > 1);
  if (nb > span_blocks(p.tiles, n_kv_heads, n_cu)) {
    p.rt = -1;
    flash_span_shape(hd, (int)rows, n_kv_heads, up(first, kKeys) + up(rest, kKeys), n_cu, p.tiles, p.np);
    return p;
  }
  p.np = slots_of(nb, blocks_each(hd, nb, rows * n_kv_heads), room(hd, n_cu) / ((int64_t)n_kv_heads * p.tiles));
  return p;
}

// The most slots of any call with these rows, wherever it starts: with the whole
// window behind it, and, where that is for the prompt rows' kernel, with the last
// number of blocks that is not (the slots do not fall as the blocks grow, in either).
int most_window_slots(int hd, int group, int n_kv_heads, int n, int64_t first, int64_t rest, int n_cu) {
  const Plan p = plan_window(hd, group, n_kv_heads, n, first, rest, n_cu);
  if (p.rt >= 0) return p.np;
  const int64_t rows = (int64_t)n * group;
  const int tiles = up(rows, tile_rows(rt_of(hd, rows)));
  const int64_t nb = span_blocks(tiles, n_kv_heads, n_cu);
  const int np = slots_of(nb, blocks_each(hd, nb, rows * n_kv_heads), room(hd, n_cu) / ((int64_t)n_kv_heads * tiles));
  return np > p.np ? np : p.np;
}
Plan plan_shared(int hd, int group, int n_kv_heads, int n, int prefix, int own_max, int n_cu) {
  const int64_t rows = (int64_t)n * group, nbp = up(prefix, kKeys), nbo = up(own_max, kKeys);
  Plan p;
  // Short caches: a workgroup per sequence and KV head goes through both, prefix and
  // all, and nothing is joined, if that is one workgroup per compute unit at most
  // (32 heads on 8, head_dim 128, in us, and in tiles: 16 sequences, 11 blocks 6.3
  // and 10.9; 16 blocks 7.0 and 11.8; 29 blocks 11.4 and 12.1; 4 sequences, 29 blocks
  // 11.2 and 8.7; 37, 11 blocks 10.0 and 11.5; 16 with K and V per head, int8, 14
  // blocks 13.1 and 11.0. head_dim 64, 16 on 4, 26 blocks 7.1 and 9.0).
  if (hd < 256 && (nbp + nbo) * hd <= 2048 && (int64_t)n * n_kv_heads <= n_cu) return {0, 0, 1, 0, true};
  p.rt = prefix ? rt_of(hd, rows) : 0;
  p.tiles = prefix ? up(rows, tile_rows(p.rt)) : 0;
  // all workgroups at once, if that is not cheaper still with fewer slots
  const double full = (double)(nbp * p.tiles + nbo * n) * n_kv_heads / (double)(room(hd, n_cu) * kW);
  const double each = fmax(full, blocks_each(hd, nbp > nbo ? nbp : nbo, rows * n_kv_heads));
  p.np = slots_of(nbp, each, INT32_MAX);
  // More tiles than compute units: as many on each (64 sequences over 32000
  // positions, 64 tiles: four slots 110 us, three 124, five 131, seven 117, eight 118).
  const int64_t part = (int64_t)p.tiles * n_kv_heads;
  if (part * p.np > n_cu && part <= n_cu) p.np = (int)(part * p.np / n_cu * n_cu / part);
  p.no = slots_of(nbo, each, INT32_MAX);
  return p;
}
size_t slot_bytes(int slots, int head_dim, int64_t rows) {
  return slots < 2 ? 0 : (size_t)slots * rows * (head_dim + 2) * sizeof(float);
}

template <int HD, int KVT>
hipError_t launch_join(const SpanArgs& a, int slots, hipStream_t s) {
  int groups = 1;   // a power of two
  while (groups < kJoinThreads / (HD / 4) && groups * 2 < slots) groups *= 2;
  const int64_t rows = (int64_t)a.n * a.n_kv_heads << a.gs;
  const dim3 grid((unsigned)up(rows, kJoinThreads / (HD / 4) / groups));
  hipLaunchKernelGGL((k_span_join<HD, KVT>), grid, dim3(kJoinThreads), 0, s, a, slots, groups);
  return hipGetLastError();
}

template <int HD, int KVT, int RT>
hipError_t launch_rt(const SpanArgs& a, const Plan& p, hipStream_t s) {
  const dim3 block(kW * 64);
  const int64_t wgs = (int64_t)a.n_kv_heads * ((int64_t)p.np * p.tiles + (a.own_len ? (int64_t)p.no * a.n : 0));
  if (wgs > INT32_MAX) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs);
  const bool cap = a.softcap > 0.f;
  if (a.own_len && cap)
    hipLaunchKernelGGL((k_span_shared<HD, KVT, RT, true>), grid, block, 0, s, a, p.np, p.no, p.tiles);
  else if (a.own_len)
    hipLaunchKernelGGL((k_span_shared<HD, KVT, RT, false>), grid, block, 0, s, a, p.np, p.no, p.tiles);
  else if (cap)
    hipLaunchKernelGGL((k_span_window<HD, KVT, RT, true>), grid, block, 0, s, a, p.np);
  else
    hipLaunchKernelGGL((k_span_window<HD, KVT, RT, false>), grid, block, 0, s, a, p.np);
  return hipGetLastError();
}

template <int HD, int KVT>
hipError_t launch_each(const SpanArgs& a, hipStream_t s) {
  const dim3 block(kWide * 64), grid((unsigned)(a.n_kv_heads * a.n));
  if (a.softcap > 0.f)
    hipLaunchKernelGGL((k_span_each<HD, KVT, true>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((k_span_each<HD, KVT, false>), grid, block, 0, s, a);
  return hipGetLastError();
}

template <int HD, int KVT>
hipError_t launch_kv(const SpanArgs& a, const Plan& p, hipStream_t s) {
  hipError_t e = hipErrorInvalidValue;
  if constexpr (HD < 256)
    if (p.each) return launch_each<HD, KVT>(a, s);
  if (p.rt < 0) {
    e = launch_flash_span(HD, KVT, a, p.np, s);
  } else if (p.rt == 0) {
    e = launch_rt<HD, KVT, 0>(a, p, s);
  } else if (p.rt == 1) {
    e = launch_rt<HD, KVT, 1>(a, p, s);
  } else if constexpr (HD < 256) {
    e = launch_rt<HD, KVT, 2>(a, p, s);
  }
  return e != hipSuccess || p.np + p.no < 2 ? e : launch_join<HD, KVT>(a, p.np + p.no, s);
}
template <int HD>
hipError_t launch_hd(int kv_type, const SpanArgs& a, const Plan& p, hipStream_t s) {
  return kv_type ? launch_kv<HD, 1>(a, p, s) : launch_kv<HD, 0>(a, p, s);
}

}  // namespace

size_t span_window_workspace(int head_dim, int group, int n_kv_heads, int n, int window, int sinks, int n_cu) {
  return slot_bytes(most_window_slots(head_dim, group, n_kv_heads, n, sinks, (int64_t)window + n - 1, n_cu), head_dim,
                    (int64_t)n * n_kv_heads * group);
}
size_t span_shared_workspace(int head_dim, int group, int n_kv_heads, int n, int prefix, int own_max, int n_cu) {
  const Plan p = plan_shared(head_dim, group, n_kv_heads, n, prefix, own_max, n_cu);
  return slot_bytes(p.np + p.no, head_dim, (int64_t)n * n_kv_heads * group);
}

namespace {
Plan plan_call(int head_dim, const SpanArgs& a) {
  const int group = 1 << a.gs;
  if (a.own_len) return plan_shared(head_dim, group, a.n_kv_heads, a.n, a.prefix, a.own_max, a.n_cu);
  const int end = a.pos0 + a.n, first = a.sinks < end ? a.sinks : end;
  const int from = a.pos0 + 1 - a.window > first ? a.pos0 + 1 - a.window : first;
  return plan_window(head_dim, group, a.n_kv_heads, a.n, first, end - from, a.n_cu);
}
}  // namespace

size_t span_bytes(int head_dim, const SpanArgs& a) {
  const Plan p = plan_call(head_dim, a);
  return slot_bytes(p.np + p.no, head_dim, (int64_t)a.n * a.n_kv_heads << a.gs);
}

hipError_t launch_span(int head_dim, int kv_type, const SpanArgs& a, size_t ws_bytes, hipStream_t s) {
  if (((int64_t)a.n * a.n_kv_heads << a.gs) > INT32_MAX / 64 || span_bytes(head_dim, a) > ws_bytes) return hipErrorInvalidValue;
  const Plan p = plan_call(head_dim, a);
  if (head_dim == 64) return launch_hd<64>(kv_type, a, p, s);
  if (head_dim == 128) return launch_hd<128>(kv_type, a, p, s);
  if (head_dim == 256) return launch_hd<256>(kv_type, a, p, s);
  return hipErrorInvalidValue;
}

}  // namespace ssk
