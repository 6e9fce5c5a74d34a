// The cache in pages (qmm_kv_cache): position j of slot s is row j % page of page
// table[s][j / page], a page's rows of one kv head are contiguous:
//   pool[layer][page id][kv head][row][head_dim].
// Table entries, lengths and row lists come from the caller's device memory: every index
// made of one is checked here before it is used as an address.
#pragma once

#include "qmm_common.h"

namespace qmm {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
constexpr int kTypeF32 = 0, kTypeF16 = 1, kTypeBF16 = 30;  // the C ABI's tags

struct KvCache {
  void *k, *v;
  const int32_t *table, *lens, *refs;
  int pages, dtype, layers, kv_heads, page_log, head_dim, slots, max_pages;
  __device__ __forceinline__ int esize_log() const { return dtype == kTypeF32 ? 2 : 1; }
  __device__ __forceinline__ int capacity() const { return max_pages << page_log; }  // <= 2^28
  __device__ __forceinline__ int length(int s) const { return min(max(lens[s], 0), capacity()); }
  // entry j of slot s, -1 where it names no page
  __device__ __forceinline__ int page(int s, int j) const {
    if (j < 0 || j >= max_pages) return -1;
    const int p = table[(long long)s * max_pages + j];
    return p >= 0 && p < pages ? p : -1;
  }
  // elements from the pool's start to row `r` of kv head g in page p (>= 0) of a layer
  __device__ __forceinline__ long long row(int layer, int p, int g, int r) const {
    return ((((long long)layer * pages + p) * kv_heads + g) << page_log) * head_dim + (long long)r * head_dim;
  }
};

// A step's packed rows: slot s has rows first .. first + n - 1.
struct KvRows {
  const int32_t* starts;
  int rows, max_rows;
};
struct KvSpan {
  int first, n;
};
__device__ __forceinline__ KvSpan kv_span(const KvRows& r, int s) {
  const int a = r.starts[s], b = r.starts[s + 1];
  if (a < 0 || a >= r.rows) return {0, 0};
  return {a, min(max(min(b, r.rows) - a, 0), r.max_rows)};
}
// The slot of packed row i (all threads of a workgroup of 256 call it together): as many
// slots as start at or before it, less one. -1 where it is in none.
__device__ __forceinline__ int kv_slot_of(const KvRows& r, int slots, int i, int* lds4) {
  int c = 0;
  for (int s = threadIdx.x; s < slots; s += 256) c += r.starts[s + 1] <= i ? 1 : 0;
  const int w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) c += __shfl_xor(c, o);
  if ((threadIdx.x & 63) == 0) lds4[w] = c;
  __syncthreads();
  const int s = __builtin_amdgcn_readfirstlane(lds4[0] + lds4[1] + lds4[2] + lds4[3]);
  if (s >= slots) return -1;
  const KvSpan sp = kv_span(r, s);
  return i >= sp.first && i < sp.first + sp.n ? s : -1;
}

// (both conversions and a choice: a branch between loads would have each wait for the last)
__device__ __forceinline__ float from_half(uint16_t v, int type) {
  const uint32_t h = __builtin_bit_cast(uint32_t, (float)__builtin_bit_cast(_Float16, v)), b = (uint32_t)v << 16;
  const uint32_t m = type == kTypeF16 ? ~0u : 0u;
  return __builtin_bit_cast(float, (h & m) | (b & ~m));
}
// (rounded to nearest even)
__device__ __forceinline__ uint16_t to_half(float v, int type) {
  return type == kTypeF16 ? __builtin_bit_cast(uint16_t, (_Float16)v) : __builtin_bit_cast(uint16_t, (__bf16)v);
}

// Element i of a typed array.
__device__ __forceinline__ float load_typed(const void* p, long long i, int type) {
  return type == kTypeF32 ? ((const float*)p)[i] : from_half(((const uint16_t*)p)[i], type);
}
__device__ __forceinline__ void store_typed(void* p, long long i, int type, float v) {
  if (type == kTypeF32)
    ((float*)p)[i] = v;
  else
    ((uint16_t*)p)[i] = to_half(v, type);
}
// Elements i .. i + 3; `wide`: they start on a boundary of four.
__device__ __forceinline__ void load4_typed(float (&v)[4], const void* p, long long i, int type, bool wide) {
  if (!wide) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = load_typed(p, i + e, type);
  } else if (type == kTypeF32) {
    const float4 x = *(const float4*)((const float*)p + i);
    v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
  } else {
    const uint2 x = *(const uint2*)((const uint16_t*)p + i);
    v[0] = from_half((uint16_t)x.x, type), v[1] = from_half((uint16_t)(x.x >> 16), type);
    v[2] = from_half((uint16_t)x.y, type), v[3] = from_half((uint16_t)(x.y >> 16), type);
  }
}
__device__ __forceinline__ void store4_typed(void* p, long long i, int type, bool wide, const float (&v)[4]) {
  if (!wide) {
#pragma unroll
    for (int e = 0; e < 4; ++e) store_typed(p, i + e, type, v[e]);
  } else if (type == kTypeF32) {
    *(float4*)((float*)p + i) = float4{v[0], v[1], v[2], v[3]};
  } else {
    uint2 x;
    x.x = to_half(v[0], type) | (uint32_t)to_half(v[1], type) << 16;
    x.y = to_half(v[2], type) | (uint32_t)to_half(v[3], type) << 16;
    *(uint2*)((uint16_t*)p + i) = x;
  }
}

// W values from i on, four at a time where they may be (`wide`, and W does).
template <int W>
__device__ __forceinline__ void store_values(void* p, long long i, int type, bool wide, const float (&v)[W]) {
  if (W % 4 == 0 && wide) {
#pragma unroll
    for (int e = 0; e + 3 < W; e += 4) store4_typed(p, i + e, type, true, {v[e], v[e + 1], v[e + 2], v[e + 3]});
  } else {
#pragma unroll
    for (int e = 0; e < W; ++e) store_typed(p, i + e, type, v[e]);
  }
}

}  // namespace qmm
