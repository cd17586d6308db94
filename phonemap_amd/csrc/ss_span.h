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

}  // namespace ssk
