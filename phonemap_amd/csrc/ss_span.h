// ss_span.h - attention of rows over spans of one or two caches: what the
// kernels share, and the attention of one row by one wave.
//
// A row (a token's or a sequence's query head) sees two spans of positions:
// window, [0, min(sinks, i + 1)) and [max(that, i - window + 1), i + 1) of one
// cache (i: the row's own position); shared, the prefix's positions and the
// sequence's own. Its output is softmax(cap(q . k / sqrt(hd))) V over both, 0
// where it sees none.

#pragma once

#include <hip/hip_runtime.h>
#include <math.h>

#include "ss_device.h"
#include "ss_kernels.h"

namespace ssk {

// positions [from, to) of a cache: rows k / v of HD elements, scales ks / vs (int8)
struct Span {
  const void* k;
  const void* v;
  const float* ks;
  const float* vs;
  int from, to;
};

// own positions of sequence t, within the cache whatever the device holds
__device__ __forceinline__ int own_length(const SpanArgs& a, int t) { return min(max(a.own_len[t], 0), a.own_max); }

// The spans of row t under KV head h; KVT 0: fp16, 1: int8.
template <int HD, int KVT>
__device__ __forceinline__ void row_spans(const SpanArgs& a, int t, int h, Span (&s)[2]) {
  constexpr int kEb = KVT == 0 ? 2 : 1;
  const size_t base = (size_t)h * a.max_seq * HD * kEb;
  s[0].k = static_cast<const uint8_t*>(a.kc) + base;
  s[0].v = static_cast<const uint8_t*>(a.vc) + base;
  s[0].ks = a.ks;
  s[0].vs = a.vs;
  s[1] = s[0];
  s[0].from = 0;
  if (a.own_len) {
    const size_t own = ((size_t)t * a.n_kv_heads + h) * a.own_max * HD * kEb;
    s[0].to = a.prefix;
    s[1].k = static_cast<const uint8_t*>(a.ko) + own;
    s[1].v = static_cast<const uint8_t*>(a.vo) + own;
    if (KVT == 1) {
      s[1].ks = a.kos + (size_t)t * a.own_max;
      s[1].vs = a.vos + (size_t)t * a.own_max;
    }
    s[1].from = 0;
    s[1].to = own_length(a, t);
  } else {
    const int end = a.pos0 + t + 1;
    s[0].to = min(a.sinks, end);
    s[1].from = max(s[0].to, end - a.window);
    s[1].to = end;
  }
}

__device__ __forceinline__ float span_cap(float d, const SpanArgs& a) {
  return a.softcap > 0.f ? a.softcap * tanhf(d * a.softcap_inv) : d;
}

// One row by one wave in fp32: 64 keys at a time, one per lane, then their V
// rows, lane l taking dimensions l, l + 64, ...
template <int HD, int KVT>
__device__ __forceinline__ void span_row(const SpanArgs& a, const float* q, float* out, const Span (&sp)[2]) {
  constexpr int ND = HD / kWave;
  constexpr int kEb = KVT == 0 ? 2 : 1;
  const int lane = threadIdx.x & 63;
  float m = -INFINITY, l = 0.f, o[ND] = {};
#pragma unroll 1
  for (int part = 0; part < 2; ++part) {
    const Span s = part ? sp[1] : sp[0];
#pragma unroll 1
    for (int k0 = s.from; k0 < s.to; k0 += kWave) {
      const bool live = k0 + lane < s.to;
      float d = -INFINITY;
      if (live) {
        const uint8_t* kr = static_cast<const uint8_t*>(s.k) + (size_t)(k0 + lane) * HD * kEb;
        const float ks = KVT == 0 ? 1.f : s.ks[k0 + lane];
        d = 0.f;
#pragma unroll 1
        for (int i = 0; i < HD; i += 8) {
          float kv[8];
          if constexpr (KVT == 0) {
            const uint4 c = *reinterpret_cast<const uint4*>(kr + 2 * i);
            const uint32_t w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
            for (int k = 0; k < 8; ++k) kv[k] = h2f((uint16_t)(w[k / 2] >> (16 * (k % 2))));
          } else {
            const uint2 c = *reinterpret_cast<const uint2*>(kr + i);
#pragma unroll
            for (int k = 0; k < 8; ++k) kv[k] = (float)(int8_t)(((k < 4 ? c.x : c.y) >> (8 * (k % 4))) & 0xffu);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) d = fmaf(q[i + k], kv[k], d);
        }
        d = span_cap(d * ks * a.scale, a);
      }
      const float mn = fmaxf(m, wave_max(d));
      const float mo = mn == -INFINITY ? 0.f : mn;
      const float p = expf(d - mo), corr = expf(m - mo);
      l = l * corr + wave_sum(p);
#pragma unroll
      for (int i = 0; i < ND; ++i) o[i] *= corr;
      const float pv = KVT == 0 || !live ? p : p * s.vs[k0 + lane];
      const int nk = min(kWave, s.to - k0);
#pragma unroll 1
      for (int j = 0; j < nk; ++j) {
        const float pj = __shfl(pv, j, kWave);
        const uint8_t* vr = static_cast<const uint8_t*>(s.v) + (size_t)(k0 + j) * HD * kEb;
#pragma unroll
        for (int i = 0; i < ND; ++i) {
          const int at = lane + kWave * i;
          const float v = KVT == 0 ? h2f(reinterpret_cast<const uint16_t*>(vr)[at]) : (float)(int8_t)vr[at];
          o[i] = fmaf(pj, v, o[i]);
        }
      }
      m = mn;
    }
  }
  const bool none = sp[0].from >= sp[0].to && sp[1].from >= sp[1].to;
#pragma unroll
  for (int i = 0; i < ND; ++i) out[lane + kWave * i] = none ? 0.f : o[i] / l;
}

constexpr int kKeys = 32;   // keys per block
__device__ __forceinline__ int blocks_of(int n) { return (n + kKeys - 1) / kKeys; }

// one KV head's K and V
struct Base {
  const uint8_t* k;
  const uint8_t* v;
  const float* ks;
  const float* vs;
};
// What a tile of rows walks: blocks of positions [0, to0), then of [from1, to1).
struct Walk : Base {
  int to0, from1, to1;
  int nb0, nb;   // blocks of the first span, of both
  __device__ __forceinline__ void block(int b, int& key, int& limit) const {
    key = b < nb0 ? kKeys * b : from1 + kKeys * (b - nb0);
    limit = b < nb0 ? to0 : to1;
  }
  __device__ __forceinline__ Base base(int) const { return *this; }
};

// among all rows [n][n_heads]
__device__ __forceinline__ size_t row_head(const SpanArgs& a, int kvh, int row) {
  return ((size_t)(row >> a.gs) * a.n_kv_heads + kvh << a.gs) + (row & ((1 << a.gs) - 1));
}

// slot s of row `head` of all rows: part [slots][rows][HD], then (m, l) [slots][rows]
template <int HD>
__device__ __forceinline__ float* slot_part(const SpanArgs& a, int rows, int s) { return a.part + (size_t)s * rows * HD; }
template <int HD>
__device__ __forceinline__ float2* slot_ml(const SpanArgs& a, int rows, int slots, int s) {
  return reinterpret_cast<float2*>(a.part + (size_t)slots * rows * HD) + (size_t)s * rows;
}

// One row in fp32 where the products could not serve it: a V that is not finite
// reaches, as 0 * inf, rows of the tile that do not see its position, and meets
// two parts of a weight where it is one. Whole waves, rows of HD / 4
// neighbouring lanes: s is this lane's share of row `head`.
template <int HD, int KVT>
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
    row_spans<HD, KVT>(a, row / nh, row % nh >> a.gs, sp);
    span_row<HD, KVT>(a, a.q + (size_t)row * HD, a.out + (size_t)row * HD, sp);
  }
}

}  // namespace ssk
