// Attention of a step's packed rows over the pages of their sequences (qmm_kv_attention).
#pragma once

#include "qmm_kv_common.h"

namespace qmm {

struct KvAttn {
  KvCache c;
  KvRows r;
  const void* q;
  const uint64_t* masks;
  void* out;
  long long ldq, ldm, ldo;
  int layer, x_type, heads;
  float scale;
};

// Whether row j of a step sees the step's row i.
__device__ __forceinline__ bool kv_sees(const KvAttn& a, int row, int j, int i) {
  if (!a.masks) return i <= j;
  return i >> 6 < a.ldm && (a.masks[(long long)row * a.ldm + (i >> 6)] >> (i & 63) & 1);
}
}  // namespace qmm

// A wave a row and head, position by position with a running maximum and sum: what every
// other form of this attention has to give.
extern "C" __global__ void __launch_bounds__(256) qmm_kv_attn_rows(qmm::KvAttn a) {
  using namespace qmm;
  __shared__ int lds4[4];
  const int row = blockIdx.x;
  const int s = kv_slot_of(a.r, a.c.slots, row, lds4);
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  if (s < 0) return;
  const KvSpan sp = kv_span(a.r, s);
  const int base = a.c.length(s), j = row - sp.first, n = min(base + sp.n, a.c.capacity());
  const int dim = a.c.head_dim, R = dim / 64, G = a.heads / a.c.kv_heads;
  for (int h = blockIdx.y * 4 + wave; h < a.heads; h += 4 * gridDim.y) {
    float q[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    for (int e = 0; e < R; ++e) q[e] = load_typed(a.q, row * a.ldq + (long long)h * dim + R * lane + e, a.x_type);
    for (int t = 0; t < n; ++t) {
      if (t >= base && !kv_sees(a, row, j, t - base)) continue;
      const int p = a.c.page(s, t >> a.c.page_log);
      float d = 0.0f, v[4];
      if (p < 0) {
        d = NAN;
        for (int e = 0; e < R; ++e) v[e] = NAN;
      } else {
        const long long at = a.c.row(a.layer, p, h / G, t & ((1 << a.c.page_log) - 1)) + R * lane;
        for (int e = 0; e < R; ++e) d += q[e] * load_typed(a.c.k, at + e, a.c.dtype);
        for (int e = 0; e < R; ++e) v[e] = load_typed(a.c.v, at + e, a.c.dtype);
        d = wave_sum(d) * a.scale;
      }
      const float mx = fmaxf(m, d);
      const float x = mx == -INFINITY ? 0.0f : expf(m - mx), w = d == -INFINITY ? 0.0f : expf(d - mx);
      m = mx;
      l = l * x + w;
      for (int e = 0; e < R; ++e) o[e] = o[e] * x + w * v[e];
    }
    for (int e = 0; e < R; ++e)
      store_typed(a.out, row * a.ldo + (long long)h * dim + R * lane + e, a.x_type, l == 0.0f ? 0.0f : o[e] / l);
  }
}
