// ss_span.hip - attention over a sliding window with first tokens that stay
// visible, and of several sequences over a prefix they share (ss_span.h), for
// few rows: a decode step.
//
// Work. A tile of query rows that share a KV head walks the blocks of 32 keys
// that some row of it sees. The blocks are dealt to `slots` workgroups and to
// the waves of each in turn, so every wave has its own softmax; a workgroup
// joins its waves through LDS, and k_span_join the slots. The sequences' rows
// over their own caches (8 rows or fewer that share K and V) and tiles of all
// sequences' rows over the prefix are workgroups of the same launch.
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
// round; tile j of DPL is then dimension DPL m + j. K, or V, of the next block is
// requested as soon as the current one's is used up.
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

constexpr int kKeys = 32;   // keys per block

// value of the lane 16 away (lane ^ 16) joined to this one's
__device__ __forceinline__ float max_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_16(float v) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float swap_8(float v) { return dpp<0x128>(v); }   // row_ror:8: lane ^ 8

// What a tile of rows walks: blocks of positions [0, to0), then of [from1, to1), of one KV head's K and V.
struct Walk {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
  int to0, from1, to1;
  int nb0, nb;   // blocks of the first span, of both
  __device__ __forceinline__ void block(int b, int& key, int& limit) const {
    key = b < nb0 ? kKeys * b : from1 + kKeys * (b - nb0);
    limit = b < nb0 ? to0 : to1;
  }
};

// The tile's rows: row r is query head g of token or sequence t, t * G + g = r0 + r < r1.
struct Rows {
  int r0, r1, kvh;
};
// among all rows [n][n_heads]
__device__ __forceinline__ size_t row_head(const SpanArgs& a, int kvh, int row) {
  return ((size_t)(row >> a.gs) * a.n_kv_heads + kvh << a.gs) + (row & ((1 << a.gs) - 1));
}

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
  __device__ __forceinline__ void load_k(const Walk& w, int key, int limit, int n, int kq) {
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
  __device__ __forceinline__ void load_v(const Walk& w, int key, int limit, int n, int kq) {
    const int live = min(limit - key, kKeys);
    const auto r = view(w.v, (size_t)key * kRowB, live * kRowB);
    const int at = 8 * kq * kRowB + 4 * kVWords * n;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
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
    if constexpr (KVT == 1) scales(w.vs, key, live, kq, vs);
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
// waves of a workgroup, and at most that many per SIMD by their registers
__host__ __device__ constexpr int tile_waves(int hd, int rt) { return rt == 0 && hd < 256 ? 8 : 4; }
__host__ __device__ constexpr int simd_waves(int hd) { return hd < 256 ? 2 : 1; }

template <int HD, int RT, int W>
struct Joint {   // the results of W waves
  static constexpr int kPitch = HD + 4;
  float o[W][tile_rows(RT)][kPitch];
  float m[W][tile_rows(RT)], l[W][tile_rows(RT)], e[W][tile_rows(RT)];
};

// One row in fp32 where the products could not serve it: a V that is not finite
// reaches, as 0 * inf, rows of the tile that do not see its position. Whole
// waves, rows of HD / 4 neighbouring lanes: s is this lane's share of row `head`.
template <int HD>
__device__ __forceinline__ void mend_rows(const SpanArgs& a, bool live, float4 s, size_t head) {
  const float odd = live ? (s.x - s.x) + (s.y - s.y) + (s.z - s.z) + (s.w - s.w) : 0.f;   // NaN: something is not finite
  uint64_t bad = __ballot(odd != odd);
  if (!bad) return;
  vm_drain();   // this wave's stores
  const int nh = a.n_kv_heads << a.gs;
  while (bad) {
    const int at = __ffsll((unsigned long long)bad) - 1;
    const int row = __shfl((int)head, at, kWave);
    bad &= ~(((HD / 4 < 64 ? 1ull << (HD / 4 % 64) : 0ull) - 1) << (at / (HD / 4) * (HD / 4)));
    Span sp[2];
    row_spans<HD, 0>(a, row / nh, row % nh >> a.gs, sp);
    span_row<HD, 0>(a, a.q + (size_t)row * HD, a.out + (size_t)row * HD, sp);
  }
}

// A tile of rows over the walk's blocks b with b / W % slots == slot, by W waves:
// the rows' outputs (part null), or the slot's share of them, at part[row of
// all rows][HD] and ml[row], to be joined. RT 0: 8 rows or fewer in one product;
// else RT tiles of 16.
template <int HD, int KVT, int RT, int W, class Masks>
__device__ __forceinline__ void span_tile(const SpanArgs& a, const Rows& rows, const Walk& w, int slot, int slots, float* part,
                                          float2* ml, Joint<HD, RT, W>& sh, Masks masks) {
  constexpr bool PACK = RT == 0;
  constexpr int NT = PACK ? 1 : RT, NC = HD / 32, DPL = HD / 16;
  using Blk = Block<HD, KVT>;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n = lane & 15, kq = lane >> 4;
  const int b0 = slot * W + wave, step = slots * W;

  Blk blk;
  int key = 0, limit = 0;
  if (b0 < w.nb) {
    w.block(b0, key, limit);
    blk.load_k(w, key, limit, n, kq);
    blk.load_v(w, key, limit, n, kq);
  }

  // q of row n of each tile as B: times the softmax's scale and log2 e, its
  // largest magnitude brought to [2^13, 2^14), in two parts
  v8h qh[NT][NC], ql[PACK ? 1 : NT][PACK ? 1 : NC];
  float qscale[NT];
  int row[NT];
  const bool cap = a.softcap > 0.f;
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    row[t] = rows.r0 + (PACK ? n & 7 : 16 * t + n);
    const bool live = row[t] < rows.r1;
    const int at = min(row[t], rows.r1 - 1);
    const float* qp = a.q + row_head(a, rows.kvh, at) * HD;
    float qv[NC][8], amax = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const float4 x0 = *reinterpret_cast<const float4*>(qp + slice_dim<KVT>(c, kq));
      const float4 x1 = *reinterpret_cast<const float4*>(qp + slice_dim<KVT>(c, kq) + 4);
      qv[c][0] = x0.x, qv[c][1] = x0.y, qv[c][2] = x0.z, qv[c][3] = x0.w;
      qv[c][4] = x1.x, qv[c][5] = x1.y, qv[c][6] = x1.z, qv[c][7] = x1.w;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        qv[c][i] = live ? qv[c][i] : 0.f;
        amax = fmaxf(amax, fabsf(qv[c][i]));
      }
    }
    amax = max_pair(max_16(amax));
    int e = 0;
    const float c0 = cap ? a.scale : a.scale * kLog2e;
    const float c1 = cap ? 0.f : __builtin_fmaf(a.scale, kLog2e, -c0) + a.scale * kLog2eLow;
    frexpf(amax * c0, &e);
    const int shift = min(max(14 - e, -100), 100);
    const float sh0 = ldexpf(c0, shift), sh1 = ldexpf(c1, shift);
    qscale[t] = ldexpf(1.0f, -shift);   // S^T holds the scores * 2^shift
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float p = qv[c][i] * sh0;
        asm("" : "+v"(p));   // one value for both parts
        const _Float16 hi = (_Float16)p;
        const _Float16 lo = (_Float16)__builtin_fmaf(qv[c][i], sh1, __builtin_fmaf(qv[c][i], sh0, -(float)hi));
        if constexpr (PACK) {
          qh[t][c][i] = n < 8 ? hi : lo;
        } else {
          qh[t][c][i] = hi;
          ql[t][c][i] = lo;
        }
      }
  }

  v4f o[NT][DPL];
  float m[NT], l[NT], ex[NT];   // running maximum, this lane's share of the sum; int8: O's exponent, times 2^12
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    m[t] = ex[t] = -INFINITY;
    l[t] = 0.f;
#pragma unroll
    for (int j = 0; j < DPL; ++j) o[t][j] = v4f{};
  }

#pragma unroll 1
  for (int b = b0; b < w.nb; b += step) {
    // the scores of keys key + 8kq + 0 .. 7
    float sc[NT][8];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      v4f d[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        d[u] = v4f{};
        if constexpr (!PACK) {
#pragma unroll
          for (int c = 0; c < NC; ++c) d[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(blk.k_slice(u, c), ql[t][c], d[u], 0, 0, 0);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) d[u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(blk.k_slice(u, c), qh[t][c], d[u], 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        sc[t][i] = PACK ? d[i / 4][i % 4] + swap_8(d[i / 4][i % 4]) : d[i / 4][i % 4];
        if constexpr (KVT == 1) sc[t][i] *= blk.ks[i];
      }
    }
    const int at = key, end = limit;
    __builtin_amdgcn_sched_barrier(0);
    if (b + step < w.nb) {
      w.block(b + step, key, limit);
      blk.load_k(w, key, limit, n, kq);
    }
    __builtin_amdgcn_sched_barrier(0);

    v8h ph[NT], pl[PACK ? 1 : NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      float vsc[KVT ? 8 : 1];
      if constexpr (KVT == 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) vsc[i] = blk.vs[i];
      }
      if (cap) {
#pragma unroll
        for (int i = 0; i < 8; ++i) sc[t][i] = span_cap(sc[t][i] * qscale[t], a);
      }
      masks.apply(at, end, kq, row[t], [&](int i) {
        sc[t][i] = -INFINITY;
        if constexpr (KVT == 1) vsc[i] = 0.f;
      });
      const float qs = cap ? kLog2e : qscale[t];
      float bmax = sc[t][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) bmax = fmaxf(bmax, sc[t][i]);
      bmax = max_pair(max_16(bmax)) * qs;
      if (__any(bmax > m[t] + kLag)) {
        const float mn = ceilf(fmaxf(m[t], bmax));
        const float corr = pow2(m[t] - (mn == -INFINITY ? 0.f : mn));
        l[t] *= corr;
        if constexpr (KVT == 0) {
#pragma unroll
          for (int j = 0; j < DPL; ++j) o[t][j] *= corr;
        }
        m[t] = mn;
      }
      const float mo = m[t] == -INFINITY ? 0.f : m[t];
      float pv[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) pv[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][i], qs, -mo));
      l[t] += ((pv[0] + pv[4]) + (pv[1] + pv[5])) + ((pv[2] + pv[6]) + (pv[3] + pv[7]));
      if constexpr (KVT == 1) {
        float bx = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pv[i] *= vsc[i];
          bx = fmaxf(bx, pv[i]);
        }
        bx = max_pair(max_16(bx));   // below 2^(e + 1)
        const float x = m[t] + (float)max((int)(__float_as_uint(bx) >> 23) - 127, -100);
        if (__any(bx > 0.f && x > ex[t] + kLagX)) {
          const float en = bx > 0.f ? fmaxf(ex[t], x) : ex[t];
          const float corr = en == ex[t] ? 1.f : pow2(ex[t] - en);
#pragma unroll
          for (int j = 0; j < DPL; ++j) o[t][j] *= corr;
          ex[t] = en;
        }
        const int up = (int)fminf(kPExp + m[t] - ex[t], 126.f);   // (past 126 with every pv 0 only)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pv[i] = ldexpf(pv[i], up);
          asm("" : "+v"(pv[i]));   // rounded to fp32 before it is split
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) pv[i] *= kPScale;
      }
      if constexpr (PACK) {
        v8h hi, lo;
        split8(pv, hi, lo);
#pragma unroll
        for (int i = 0; i < 8; ++i) ph[t][i] = n < 8 ? hi[i] : lo[i];
      } else {
        split8(pv, ph[t], pl[t]);
      }
    }
#pragma unroll
    for (int j = 0; j < DPL; ++j) {
      const v8h vt = blk.v_tile(j);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (!PACK) o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, pl[t], o[t][j], 0, 0, 0);
        o[t][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, ph[t], o[t][j], 0, 0, 0);
      }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (b + step < w.nb) blk.load_v(w, key, limit, n, kq);
    __builtin_amdgcn_sched_barrier(0);
  }

  // the waves' rows -> one
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    l[t] = sum_pair(sum_16(l[t]));
    if constexpr (PACK) {
#pragma unroll
      for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) o[t][j][r] += swap_8(o[t][j][r]);
    }
    const int at = PACK ? n & 7 : 16 * t + n;
    if (!PACK || n < 8) {
      if (kq == 0) {
        sh.m[wave][at] = m[t];
        sh.l[wave][at] = l[t];
        sh.e[wave][at] = KVT == 1 ? ex[t] : m[t];
      }
      float* dst = &sh.o[wave][at][4 * DPL * kq];
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int j = 0; j < DPL; j += 4)
          *reinterpret_cast<float4*>(dst + DPL * r + j) = make_float4(o[t][j][r], o[t][j + 1][r], o[t][j + 2][r], o[t][j + 3][r]);
    }
  }
  __syncthreads();
  constexpr int kQuads = HD / 4;
  static_assert(tile_rows(RT) * kQuads % (W * 64) == 0 || tile_rows(RT) * kQuads < W * 64, "whole waves");
  for (int i = tid; i < tile_rows(RT) * kQuads; i += W * 64) {
    const int r = i / kQuads, c = i % kQuads, all = rows.r0 + r;
    const bool live = all < rows.r1;
    float mx = -INFINITY, lt = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) mx = fmaxf(mx, sh.m[k][r]);
    const float mo = mx == -INFINITY ? 0.f : mx;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < W; ++k) {
      lt += sh.l[k][r] * pow2(sh.m[k][r] - mo);
      const float f = pow2(sh.e[k][r] - kPExp - mo);
      const float4 v = *reinterpret_cast<const float4*>(&sh.o[k][r][4 * c]);
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
      if constexpr (KVT == 0 && Masks::kMend) mend_rows<HD>(a, live, s, head);
    }
  }
}

// Keys at or past the block's end are not there.
struct TailMask {
  static constexpr bool kMend = false;
  template <class F>
  __device__ __forceinline__ void apply(int key, int limit, int kq, int row, F hide) const {
    if (key + kKeys > limit) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (key + 8 * kq + i >= limit) hide(i);
    }
  }
};
// Rows of several tokens: row r's token sees its own window alone.
struct WindowMask {
  static constexpr bool kMend = true;
  int gs, pos0, window, sinks, t0, t1;   // the tile's first and last token
  template <class F>
  __device__ __forceinline__ void apply(int key, int limit, int kq, int row, F hide) const {
    if (key + kKeys <= limit && key + kKeys - 1 <= pos0 + t0 && (key > pos0 + t1 - window || key + kKeys <= sinks)) return;
    const int lim = pos0 + min(row >> gs, t1), low = lim - window;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int j = key + 8 * kq + i;
      if (j >= limit || j > lim || (j <= low && j >= sinks)) hide(i);
    }
  }
};

__device__ __forceinline__ int blocks_of(int n) { return (n + kKeys - 1) / kKeys; }

// slot s of row `head` of all rows: part [slots][rows][HD], then (m, l) [slots][rows]
template <int HD>
__device__ __forceinline__ float* slot_part(const SpanArgs& a, int rows, int s) { return a.part + (size_t)s * rows * HD; }
template <int HD>
__device__ __forceinline__ float2* slot_ml(const SpanArgs& a, int rows, int slots, int s) {
  return reinterpret_cast<float2*>(a.part + (size_t)slots * rows * HD) + (size_t)s * rows;
}

// Grid: n_kv_heads x slots.
template <int HD, int KVT, int RT>
__global__ void __launch_bounds__(tile_waves(HD, RT) * 64, simd_waves(HD)) k_span_window(const SpanArgs a, int slots) {
  __shared__ Joint<HD, RT, tile_waves(HD, RT)> sh;
  const int kvh = blockIdx.x % a.n_kv_heads, slot = blockIdx.x / a.n_kv_heads;
  const int end = a.pos0 + a.n, rows = a.n * a.n_kv_heads << a.gs;
  Walk w;
  const size_t base = (size_t)kvh * a.max_seq * Block<HD, KVT>::kRowB;
  w.k = static_cast<const uint8_t*>(a.kc) + base;
  w.v = static_cast<const uint8_t*>(a.vc) + base;
  w.ks = a.ks;
  w.vs = a.vs;
  w.to0 = min(a.sinks, end);
  w.from1 = max(w.to0, a.pos0 + 1 - a.window);
  w.to1 = end;
  w.nb0 = blocks_of(w.to0);
  w.nb = w.nb0 + blocks_of(w.to1 - w.from1);
  const Rows r = {0, a.n << a.gs, kvh};
  float* part = slots > 1 ? slot_part<HD>(a, rows, slot) : nullptr;
  float2* ml = slot_ml<HD>(a, rows, slots, slot);
  if (a.n == 1)
    span_tile<HD, KVT, RT>(a, r, w, slot, slots, part, ml, sh, TailMask{});
  else
    span_tile<HD, KVT, RT>(a, r, w, slot, slots, part, ml, sh, WindowMask{a.gs, a.pos0, a.window, a.sinks, 0, a.n - 1});
}

// Grid: n_kv_heads x np x tiles of rows over the prefix, then n_kv_heads x no x
// sequences over their own caches; slots 0 .. np - 1 are the prefix's.
template <int HD, int KVT, int RT>
__global__ void __launch_bounds__(tile_waves(HD, RT) * 64, simd_waves(HD)) k_span_shared(const SpanArgs a, int np, int no, int tiles) {
  __shared__ union {
    Joint<HD, RT, tile_waves(HD, RT)> tile;
    Joint<HD, 0, tile_waves(HD, RT)> own;
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
    span_tile<HD, KVT, RT>(a, r, w, slot, np, slots > 1 ? slot_part<HD>(a, rows, slot) : nullptr,
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
    span_tile<HD, KVT, 0>(a, r, w, slot, no, slots > 1 ? slot_part<HD>(a, rows, np + slot) : nullptr,
                             slot_ml<HD>(a, rows, slots, np + slot), sh.own, TailMask{});
  }
}

// The slots' shares -> outputs; one thread per four outputs.
constexpr int kJoinThreads = 256;
template <int HD, int KVT>
__global__ void __launch_bounds__(kJoinThreads) k_span_join(const SpanArgs a, int slots) {
  constexpr int kQuads = HD / 4;
  const int rows = a.n * a.n_kv_heads << a.gs;
  const int at = (int)(((int64_t)blockIdx.x * kJoinThreads + threadIdx.x) / kQuads), c = threadIdx.x % kQuads;
  const bool live = at < rows;
  const int row = min(at, rows - 1);
  const float2* ml = slot_ml<HD>(a, rows, slots, 0) + row;
  float mx = -INFINITY;
#pragma unroll 8
  for (int s = 0; s < slots; ++s) mx = fmaxf(mx, ml[(size_t)s * rows].x);
  float lt = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = 0; s < slots; ++s) {
    const float2 x = ml[(size_t)s * rows];
    if (x.x == -INFINITY) continue;
    const float4 v = reinterpret_cast<const float4*>(slot_part<HD>(a, rows, s) + (size_t)row * HD)[c];
    const float f = pow2(x.x - mx);
    lt += x.y * f;
    o.x += v.x * f;
    o.y += v.y * f;
    o.z += v.z * f;
    o.w += v.w * f;
  }
  bool none = false;
  if (a.own_len) none = a.prefix == 0 && own_length(a, row / (a.n_kv_heads << a.gs)) == 0;
  const float f = none ? 0.f : 1.f / lt;
  o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
  if (live) reinterpret_cast<float4*>(a.out + (size_t)row * HD)[c] = o;
  if constexpr (KVT == 0)
    if (!a.own_len && a.n > 1) mend_rows<HD>(a, live, o, (size_t)row);
}

// ---- many rows: one wave per row and query head -------------------------------
constexpr int kRowWaves = 4;
template <int HD, int KVT>
__global__ void __launch_bounds__(kRowWaves * 64) k_span_rows(const SpanArgs a) {
  const int nh = a.n_kv_heads << a.gs;
  const int64_t row = (int64_t)blockIdx.x * kRowWaves + (threadIdx.x >> 6);
  if (row >= (int64_t)a.n * nh) return;
  const int t = (int)(row / nh), h = (int)(row % nh);
  Span s[2];
  row_spans<HD, KVT>(a, t, h >> a.gs, s);
  span_row<HD, KVT>(a, a.q + (size_t)row * HD, a.out + (size_t)row * HD, s);
}

int up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How a call is cut: rt (tile_rows), tiles of rows, slots of the window or the
// prefix (np) and of the own caches (no). rt -1: too many rows, k_span_rows.
struct Plan {
  int rt, tiles, np, no;
};
int rt_of(int hd, int rows) { return rows <= 8 ? 0 : rows <= 16 || hd == 256 ? 1 : 2; }

// keys: the positions that the window's rows see between them (at most)
Plan plan_window(int hd, int group, int n_kv_heads, int n, int64_t first, int64_t rest, int n_cu) {
  if ((int64_t)n * group > (hd == 256 ? 16 : 32)) return {-1, 1, 1, 0};
  Plan p;
  p.rt = rt_of(hd, n * group);
  p.tiles = 1;
  p.no = 0;
  const int64_t nb = (first + kKeys - 1) / kKeys + (rest + kKeys - 1) / kKeys;
  const int w = tile_waves(hd, p.rt), most = up(n_cu, n_kv_heads);
  const int64_t want = (nb + w - 1) / w;
  p.np = (int)(want < most ? want : most);
  return p;
}
Plan plan_shared(int hd, int group, int n_kv_heads, int n, int prefix, int own_max, int n_cu) {
  Plan p;
  const int rows = n * group;
  p.rt = prefix ? rt_of(hd, rows) : 0;
  p.tiles = prefix ? up(rows, tile_rows(p.rt)) : 0;
  const int w = tile_waves(hd, p.rt);
  const int64_t nbp = up(prefix, kKeys), nbo = up(own_max, kKeys);
  const int64_t all = (nbp * p.tiles + nbo * n) * n_kv_heads;
  const int each = up(all, (int64_t)n_cu * 8);   // blocks per wave
  p.np = up(nbp, (int64_t)w * each);
  p.no = up(nbo, (int64_t)w * each);
  return p;
}
size_t plan_bytes(const Plan& p, int head_dim, int64_t rows) {
  const int slots = p.np + p.no;
  return p.rt < 0 || slots < 2 ? 0 : (size_t)slots * rows * (head_dim + 2) * sizeof(float);
}

template <int HD, int KVT>
hipError_t launch_join(const SpanArgs& a, int slots, hipStream_t s) {
  const int64_t threads = ((int64_t)a.n * a.n_kv_heads << a.gs) * (HD / 4);
  hipLaunchKernelGGL((k_span_join<HD, KVT>), dim3((unsigned)up(threads, kJoinThreads)), dim3(kJoinThreads), 0, s, a, slots);
  return hipGetLastError();
}

template <int HD, int KVT, int RT>
hipError_t launch_rt(const SpanArgs& a, const Plan& p, hipStream_t s) {
  const dim3 block(tile_waves(HD, RT) * 64);
  const int64_t wgs = (int64_t)a.n_kv_heads * (a.own_len ? (int64_t)p.np * p.tiles + (int64_t)p.no * a.n : p.np);
  if (wgs > INT32_MAX) return hipErrorInvalidValue;
  if (a.own_len)
    hipLaunchKernelGGL((k_span_shared<HD, KVT, RT>), dim3((unsigned)wgs), block, 0, s, a, p.np, p.no, p.tiles);
  else
    hipLaunchKernelGGL((k_span_window<HD, KVT, RT>), dim3((unsigned)wgs), block, 0, s, a, p.np);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || p.np + p.no < 2 ? e : launch_join<HD, KVT>(a, p.np + p.no, s);
}

template <int HD, int KVT>
hipError_t launch_kv(const SpanArgs& a, const Plan& p, hipStream_t s) {
  if (p.rt == 0) return launch_rt<HD, KVT, 0>(a, p, s);
  if (p.rt == 1) return launch_rt<HD, KVT, 1>(a, p, s);
  if constexpr (HD < 256)
    if (p.rt == 2) return launch_rt<HD, KVT, 2>(a, p, s);
  const int64_t rows = (int64_t)a.n * a.n_kv_heads << a.gs;
  hipLaunchKernelGGL((k_span_rows<HD, KVT>), dim3((unsigned)up(rows, kRowWaves)), dim3(kRowWaves * 64), 0, s, a);
  return hipGetLastError();
}
template <int HD>
hipError_t launch_hd(int kv_type, const SpanArgs& a, const Plan& p, hipStream_t s) {
  return kv_type ? launch_kv<HD, 1>(a, p, s) : launch_kv<HD, 0>(a, p, s);
}

}  // namespace

size_t span_window_workspace(int head_dim, int group, int n_kv_heads, int n, int window, int sinks, int n_cu) {
  const Plan p = plan_window(head_dim, group, n_kv_heads, n, sinks, (int64_t)window + n - 1, n_cu);
  return plan_bytes(p, head_dim, (int64_t)n * n_kv_heads * group);
}
size_t span_shared_workspace(int head_dim, int group, int n_kv_heads, int n, int prefix, int own_max, int n_cu) {
  return plan_bytes(plan_shared(head_dim, group, n_kv_heads, n, prefix, own_max, n_cu), head_dim, (int64_t)n * n_kv_heads * group);
}

hipError_t launch_span(int head_dim, int kv_type, const SpanArgs& a, hipStream_t s) {
  const int group = 1 << a.gs;
  if ((int64_t)a.n * a.n_kv_heads * group > INT32_MAX / 64) return hipErrorInvalidValue;
  Plan p;
  if (a.own_len) {
    p = plan_shared(head_dim, group, a.n_kv_heads, a.n, a.prefix, a.own_max, a.n_cu);
  } else {
    const int end = a.pos0 + a.n, first = a.sinks < end ? a.sinks : end;
    const int from = a.pos0 + 1 - a.window > first ? a.pos0 + 1 - a.window : first;
    p = plan_window(head_dim, group, a.n_kv_heads, a.n, first, end - from, a.n_cu);
  }
  if (head_dim == 64) return launch_hd<64>(kv_type, a, p, s);
  if (head_dim == 128) return launch_hd<128>(kv_type, a, p, s);
  if (head_dim == 256) return launch_hd<256>(kv_type, a, p, s);
  return hipErrorInvalidValue;
}

}  // namespace ssk
