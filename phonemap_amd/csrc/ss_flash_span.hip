// ss_flash_span.hip - the prompt rows' attention (ss_flash.h) over a sliding
// window with first positions.

#include "ss_flash.h"

namespace ssk {
namespace {

// row tiles per workgroup: two share a workgroup's staging at head_dim 128
int row_tiles(int head_dim, int rows) { return head_dim == 128 && rows > 32 ? 2 : 1; }
int key_groups(int head_dim) { return head_dim == 256 ? 2 : 4; }

template <int HD, int RT, int KG, int DS>
hipError_t launch_shape(int kv_type, const SpanRows& a, unsigned wgs, hipStream_t s) {
  const dim3 grid(wgs), block(RT * KG * DS * 64);
  if (kv_type)
    hipLaunchKernelGGL((k_flash_rows<HD, 0, RT, KG, DS, true, false, SpanRows>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((k_flash_rows<HD, 0, RT, KG, DS, false, false, SpanRows>), grid, block, 0, s, a);
  return hipGetLastError();
}

}  // namespace

void flash_span_shape(int head_dim, int rows, int n_kv_heads, int64_t nb, int n_cu, int& tiles, int& slots) {
  const int per = 32 * row_tiles(head_dim, rows), kg = key_groups(head_dim);
  tiles = (rows + per - 1) / per;
  const int64_t steps = (nb + kg - 1) / kg, room = n_cu / ((int64_t)tiles * n_kv_heads);
  slots = (int)(room < 1 ? 1 : room < steps ? room : steps);
}

hipError_t launch_flash_span(int head_dim, int kv_type, const SpanArgs& sa, int slots, hipStream_t s) {
  SpanRows a = {};
  a.s = sa;
  a.slots = slots;
  a.q = sa.q;
  a.kc = sa.kc;
  a.vc = sa.vc;
  a.ks = sa.ks;
  a.vs = sa.vs;
  a.max_seq = sa.max_seq;
  a.n_kv_heads = sa.n_kv_heads;
  a.scale = sa.scale;
  a.softcap = sa.softcap;
  a.softcap_inv = sa.softcap_inv;
  a.out = sa.out;
  a.n_tok = sa.n;
  a.pos0 = sa.pos0;
  a.tok_q = a.tok_o = (sa.n_kv_heads << sa.gs) * head_dim;
  const int rows = sa.n << sa.gs, rt = row_tiles(head_dim, rows);
  const int64_t wgs = (int64_t)((rows + 32 * rt - 1) / (32 * rt)) * sa.n_kv_heads * slots;
  if (wgs > INT32_MAX) return hipErrorInvalidValue;
  if (head_dim == 64) return launch_shape<64, 1, 4, 1>(kv_type, a, (unsigned)wgs, s);
  if (head_dim == 256) return launch_shape<256, 1, 2, 2>(kv_type, a, (unsigned)wgs, s);
  return rt == 1 ? launch_shape<128, 1, 4, 1>(kv_type, a, (unsigned)wgs, s) : launch_shape<128, 2, 4, 1>(kv_type, a, (unsigned)wgs, s);
}

}  // namespace ssk
