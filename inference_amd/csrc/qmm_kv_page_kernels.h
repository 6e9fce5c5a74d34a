// The rows of a step appended to a cache in pages, and what moves its pages: forks of
// sequences with copies of the pages that two of them would write, the accepted rows of a
// drafted tree, and the packing of the pool.
#pragma once

#include "qmm_kv_common.h"

namespace qmm {

struct KvAppend {
  KvCache c;
  KvRows r;
  const void *q, *k, *v;
  const int32_t* depths;
  const float *cos_t, *sin_t;
  void* q_out;
  long long ldq, ldk, ldv, ldqo;
  int layer, x_type, heads, positions, wide;
};

// Rounds a count up to whole pages.
__device__ __forceinline__ int kv_pages_of(int positions, int page_log) {
  return (positions + (1 << page_log) - 1) >> page_log;
}
__device__ __forceinline__ int agent_load(const int* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_store(int* p, int v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ void agent_add(int* p, int v) {
  (void)__hip_atomic_fetch_add(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// A barrier after which agent_load sees what the workgroup's agent stores and adds before it left.
__device__ __forceinline__ void agent_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();
}
}  // namespace qmm

// x cos + rotate_half(x) sin of the rows, k and v to their pages. A thread has four values
// of a head's first half and the four of the second that turn with them; head_dim / 8
// threads a head, q's heads first, then k's, then v's. Bound by the rows' bytes: 2053 rows of 32
// + 2 x 8 f32 heads of 128 into bf16 pages 19.8 us for 94 MB (17.6 at a copy's rate); one row 3.3 us, all of it latency.
extern "C" __global__ void __launch_bounds__(256) qmm_kv_append_rows(qmm::KvAppend a) {
#pragma clang fp contract(off)
  using namespace qmm;
  __shared__ int lds4[4];
  const int per = a.c.head_dim / 8, group = 256 / per;
  const int nq = a.q ? a.heads : 0, units = nq + 2 * a.c.kv_heads, blocks = (units + group - 1) / group;
  const int row = blockIdx.x / blocks, u = blockIdx.x % blocks * group + threadIdx.x / per;
  const int s = kv_slot_of(a.r, a.c.slots, row, lds4);
  if (s < 0 || u >= units) return;
  const KvSpan sp = kv_span(a.r, s);
  const int j = row - sp.first, base = a.c.length(s), half = a.c.head_dim / 2;
  const int i = 4 * (threadIdx.x % per);
  // (64 bits: a depth is the caller's)
  const long long p = (long long)base + (a.depths ? a.depths[row] : j);
  if (a.cos_t && (p < 0 || p >= a.positions)) return;
  const bool is_q = u < nq, is_v = u >= nq + a.c.kv_heads;
  const int h = is_q ? u : is_v ? u - nq - a.c.kv_heads : u - nq;
  const void* src = is_q ? a.q : is_v ? a.v : a.k;
  const long long ld = is_q ? a.ldq : is_v ? a.ldv : a.ldk;
  const long long at = row * ld + (long long)h * a.c.head_dim + i;
  float x[4], y[4];
  load4_typed(x, src, at, a.x_type, a.wide);
  load4_typed(y, src, at + half, a.x_type, a.wide);
  if (a.cos_t && !is_v) {
    float c0[4], c1[4], s0[4], s1[4];
    load4_typed(c0, a.cos_t, p * a.c.head_dim + i, kTypeF32, a.wide);
    load4_typed(c1, a.cos_t, p * a.c.head_dim + i + half, kTypeF32, a.wide);
    load4_typed(s0, a.sin_t, p * a.c.head_dim + i, kTypeF32, a.wide);
    load4_typed(s1, a.sin_t, p * a.c.head_dim + i + half, kTypeF32, a.wide);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float xe = x[e], ye = y[e];
      x[e] = xe * c0[e] + -ye * s0[e];
      y[e] = ye * c1[e] + xe * s1[e];
    }
  }
  if (is_q) {
    const long long o = row * a.ldqo + (long long)h * a.c.head_dim + i;
    store4_typed(a.q_out, o, a.x_type, a.wide, x);
    store4_typed(a.q_out, o + half, a.x_type, a.wide, y);
    return;
  }
  const int t = base + j;
  if (t >= a.c.capacity()) return;
  const int page = a.c.page(s, t >> a.c.page_log);
  if (page < 0) return;
  void* pool = is_v ? a.c.v : a.c.k;
  const long long o = a.c.row(a.layer, page, h, t & ((1 << a.c.page_log) - 1)) + i;
  store4_typed(pool, o, a.c.dtype, true, x);
  store4_typed(pool, o + half, a.c.dtype, true, y);
}

// ---------------------------------------------------------------------------
// fork
// ---------------------------------------------------------------------------
namespace qmm {

struct KvFork {
  KvCache c;
  const int32_t *parents, *keep;
  int32_t *table_out, *lens_out, *refs_out, *shortage;
  int reserve;
  // workspace
  int32_t *refs, *writers, *first;  // [pages]: counts, slots that would write the page, the lowest of them
  int32_t *free_ids;                // [pages]: free pages, the lowest first
  int32_t *table;                   // [slots][max_pages]: the old table
  int32_t *lens, *at, *parent;      // [slots]: new length, first of the slot's new pages in free_ids, parent or -1
  int32_t *copy;                    // [slots]: whether the slot's last page is copied
  int32_t *moves;                   // [1 + 3 slots]: number of copies; source, destination, rows of each
};

constexpr int kForkLists = 16384;  // entries of the lists of a small fork

// A slot's new length in positions, whole and part-filled pages of it, and those with the reserve.
struct KvGrow {
  int len, held, total;
  bool part;  // its last page is filled in part and will be written
};
__device__ __forceinline__ KvGrow kv_grow(const KvFork& f, int s) {
  const int len = agent_load(f.lens + s), lg = f.c.page_log;
  KvGrow g = {len, kv_pages_of(len, lg), 0, false};
  g.total = agent_load(f.parent + s) < 0 ? 0 : f.reserve ? kv_pages_of(len + f.reserve, lg) : g.held;
  g.part = f.reserve > 0 && (len & ((1 << lg) - 1)) != 0;
  return g;
}

// The phases, over `n` threads (t is this one) or `n` waves; a phase reads what the one
// before has written.
__device__ __forceinline__ void kv_fork_begin(const KvFork& f, long long t, long long n) {
  for (long long p = t; p < f.c.pages; p += n) {
    agent_store(f.refs + p, f.c.refs[p]);
    agent_store(f.writers + p, 0);
    agent_store(f.first + p, 0x7fffffff);
  }
  const unsigned cells = (unsigned)f.c.slots * (unsigned)f.c.max_pages;  // (2^28 at most)
  for (unsigned i = (unsigned)t; i < cells; i += (unsigned)n) {
    const int p = f.c.table[i];
    agent_store(f.table + i, p >= 0 && p < f.c.pages ? p : -1);
  }
  for (long long s = t; s < f.c.slots; s += n) {
    const int p = f.parents[s];
    const bool ok = p >= 0 && p < f.c.slots;
    int len = ok ? f.c.length(p) : 0;
    if (f.keep && f.keep[s] >= 0) len = min(len, f.keep[s]);
    agent_store(f.lens + s, len);
    agent_store(f.parent + s, ok ? p : -1);
  }
}

// The counts without the old rows and with the new ones, before any new page. A wave a slot: two adds for each entry
// (6.1 us for 128 slots of up to 94 pages, 44 for 32 of 1875).
__device__ __forceinline__ void kv_fork_count(const KvFork& f, long long w, long long waves, int lane) {
  for (long long s = w; s < f.c.slots; s += waves) {
    const long long row = s * f.c.max_pages;
    for (int j = lane; j < f.c.max_pages; j += 64) {
      const int p = agent_load(f.table + row + j);
      if (p >= 0) agent_add(f.refs + p, -1);
    }
    const int from = agent_load(f.parent + s);
    if (from < 0) continue;
    const KvGrow g = kv_grow(f, (int)s);
    for (int j = lane; j < min(g.held, f.c.max_pages); j += 64) {
      const int p = agent_load(f.table + (long long)from * f.c.max_pages + j);
      if (p < 0) continue;
      agent_add(f.refs + p, 1);
      if (g.part && j == g.held - 1) {
        agent_add(f.writers + p, 1);
        (void)__hip_atomic_fetch_min(f.first + p, (int)s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      }
    }
  }
}

// Exclusive sums of v over the 1024 threads of a workgroup, and the whole sum.
__device__ __forceinline__ int block_sums(int v, int* lds, int* total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int x = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();  // (the last call's values are read no more)
  if (lane == 63) lds[wave] = x;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int y = lds[i];
    before += i < wave ? y : 0;
    all += y;
  }
  *total = all;
  return before + x - v;
}

// One workgroup: which slots copy their last page, how many pages each takes, and which. It looks for free pages 1024 at
// a time, a dependent round each: 6.3 us for 128 slots over a thousand pages, 26 where all but 64 of 65536 are held.
__device__ __forceinline__ void kv_fork_plan(const KvFork& f, int* lds) {
  const int t = threadIdx.x, per = (f.c.slots + 1023) / 1024;
  int need = 0, over = 0, copies = 0;
  for (int i = 0; i < per; ++i) {
    const int s = t * per + i;
    if (s >= f.c.slots) break;
    const KvGrow g = kv_grow(f, s);
    int copy = -1;
    if (g.part && agent_load(f.parent + s) >= 0) {
      const int p = agent_load(f.table + (long long)agent_load(f.parent + s) * f.c.max_pages + g.held - 1);
      if (p >= 0 && !(agent_load(f.refs + p) == agent_load(f.writers + p) && agent_load(f.first + p) == s)) copy = p;
    }
    agent_store(f.copy + s, copy);
    copies += copy >= 0;
    need += (copy >= 0) + max(min(g.total, f.c.max_pages) - g.held, 0);
    over += max(g.total - f.c.max_pages, 0);
  }
  int total, none, slots_over;
  int at = block_sums(need, lds, &total);
  (void)block_sums(over, lds, &slots_over);
  int move = block_sums(copies, lds, &none);
  // the free pages, until there are enough
  int found = 0;
  for (long long p0 = 0; p0 < f.c.pages && found < total; p0 += 1024) {
    const long long p = p0 + t;
    const bool free = p < f.c.pages && agent_load(f.refs + p) == 0;
    int here;
    const int i = block_sums(free ? 1 : 0, lds, &here);
    if (free && found + i < total) agent_store(f.free_ids + found + i, (int)p);
    found += here;
  }
  const int missing = max(total - found, 0) + slots_over;
  agent_barrier();
  if (t == 0) {
    agent_store(f.shortage, missing);
    agent_store(f.moves, missing ? 0 : none);
  }
  if (missing) return;
  for (int i = 0; i < per; ++i) {
    const int s = t * per + i;
    if (s >= f.c.slots) break;
    const KvGrow g = kv_grow(f, s);
    const int p = agent_load(f.copy + s);
    agent_store(f.at + s, at);
    if (p >= 0) {
      agent_add(f.refs + p, -1);
      agent_store(f.moves + 1 + 3 * move, p);
      agent_store(f.moves + 2 + 3 * move, agent_load(f.free_ids + at));
      agent_store(f.moves + 3 + 3 * move, g.len & ((1 << f.c.page_log) - 1));
      ++move;
    }
    at += (p >= 0) + max(g.total - g.held, 0);
  }
  for (int i = t; i < total; i += 1024) agent_store(f.refs + agent_load(f.free_ids + i), 1);
}

__device__ __forceinline__ void kv_fork_commit(const KvFork& f, long long t, long long n) {
  const bool ok = agent_load(f.shortage) == 0;
  // (refs_out and table_out may be the cache's own: without room they get back what they held)
  for (long long p = t; p < f.c.pages; p += n) f.refs_out[p] = ok ? agent_load(f.refs + p) : f.c.refs[p];
  const int lane = (int)(t & 63);
  for (long long s = t >> 6; s < f.c.slots; s += n >> 6) {  // a wave a row
    const long long row = s * f.c.max_pages;
    if (!ok) {
      for (int j = lane; j < f.c.max_pages; j += 64) f.table_out[row + j] = f.c.table[row + j];
      if (lane == 0) f.lens_out[s] = f.c.lens[s];
      continue;
    }
    const int from = agent_load(f.parent + s), at = agent_load(f.at + s), copy = agent_load(f.copy + s) >= 0;
    const KvGrow g = kv_grow(f, (int)s);
    for (int j = lane; j < f.c.max_pages; j += 64) {
      int p = -1;
      if (from >= 0 && j < g.held && !(copy && j == g.held - 1))
        p = agent_load(f.table + (long long)from * f.c.max_pages + j);
      else if (j < g.total && (copy || j >= g.held))  // (a copied last page is the first of the slot's new ones)
        p = agent_load(f.free_ids + at + copy + j - g.held);
      f.table_out[row + j] = p;
    }
    if (lane == 0) f.lens_out[s] = g.len;
  }
}
// The listed pages' first rows (a whole page: rows = page size) to other pages, in every layer
// and of every kv head. Sources and destinations are disjoint. A workgroup takes a head's rows
// of a page, side and layer at a time. Bound by the bytes: 512 of 2048 pages of 32 KB moved in 8
// layers 113 us for 537 MB there and back (16 KB at a time over the heads, four loads a thread
// in flight: 2% more, and for half-filled pages of 64 rows 41 us against 29).
__device__ __forceinline__ void kv_copy_pages(const KvCache& c, const int* moves, long long first, long long step) {
  const long long items = (long long)moves[0] * c.layers * 2 * c.kv_heads;
  for (long long i = first; i < items; i += step) {
    const int g = (int)(i % c.kv_heads), side = (int)(i / c.kv_heads % 2);
    const int layer = (int)(i / (2 * c.kv_heads) % c.layers);
    const int* m = moves + 1 + 3 * (i / (2LL * c.kv_heads * c.layers));
    char* pool = (char*)(side ? c.v : c.k);
    const u32x4* src = (const u32x4*)(pool + (c.row(layer, m[0], g, 0) << c.esize_log()));
    u32x4* dst = (u32x4*)(pool + (c.row(layer, m[1], g, 0) << c.esize_log()));
    const int n = (m[2] * c.head_dim << c.esize_log()) / 16;
    for (int x = threadIdx.x; x < n; x += 256) dst[x] = src[x];
  }
}
}  // namespace qmm

extern "C" __global__ void __launch_bounds__(256) qmm_kv_copy_pages(qmm::KvCache c, const int* moves) {
  qmm::kv_copy_pages(c, moves, blockIdx.x, gridDim.x);
}
extern "C" __global__ void __launch_bounds__(256) qmm_kv_fork_begin(qmm::KvFork f) {
  qmm::kv_fork_begin(f, blockIdx.x * 256LL + threadIdx.x, gridDim.x * 256LL);
}
extern "C" __global__ void __launch_bounds__(256) qmm_kv_fork_count(qmm::KvFork f) {
  qmm::kv_fork_count(f, blockIdx.x * 4LL + (threadIdx.x >> 6), gridDim.x * 4LL, threadIdx.x & 63);
}
extern "C" __global__ void __launch_bounds__(1024) qmm_kv_fork_plan(qmm::KvFork f) {
  __shared__ int lds[16];
  qmm::kv_fork_plan(f, lds);
}
// The lists by the first `lists` workgroups and the copies by the others, neither of which reads
// what the other writes (128 slots of four prompts in 8 layers 52.0 us, in two launches 55.2).
extern "C" __global__ void __launch_bounds__(256) qmm_kv_fork_commit(qmm::KvFork f, int lists) {
  if (blockIdx.x < (unsigned)lists)
    qmm::kv_fork_commit(f, blockIdx.x * 256LL + threadIdx.x, lists * 256LL);
  else
    qmm::kv_copy_pages(f.c, f.moves, blockIdx.x - lists, gridDim.x - lists);
}

// All phases of a small fork in one workgroup, its lists in LDS: launches and round trips to
// memory cost more than the work (with the copies, 4 slots of 64 pages 11.0 us against 15.4 in
// four launches, 32 of 256 13.6 against 19.3; with the lists in memory 13.4 and 20.8).
extern "C" __global__ void __launch_bounds__(1024) qmm_kv_fork_small(qmm::KvFork f) {
  using namespace qmm;
  __shared__ int lds[16];
  __shared__ int32_t lists[kForkLists];
  int32_t* at = lists;
  auto take = [&](int n) {
    int32_t* p = at;
    at += n;
    return p;
  };
  f.refs = take(f.c.pages), f.writers = take(f.c.pages), f.first = take(f.c.pages), f.free_ids = take(f.c.pages);
  f.lens = take(f.c.slots), f.at = take(f.c.slots), f.parent = take(f.c.slots), f.copy = take(f.c.slots);
  f.table = take(f.c.slots * f.c.max_pages);
  const int t = threadIdx.x;
  kv_fork_begin(f, t, 1024);
  agent_barrier();
  kv_fork_count(f, t >> 6, 16, t & 63);
  agent_barrier();
  kv_fork_plan(f, lds);
  agent_barrier();
  kv_fork_commit(f, t, 1024);
}

// ---------------------------------------------------------------------------
// accept
// ---------------------------------------------------------------------------
namespace qmm {
struct KvAccept {
  KvCache c;
  const int32_t *path, *counts;
  int32_t* lens_out;
  long long ld_path;
  int max_path;
};

// Entries d0 .. d0 + 63 of a slot's path, one a lane of a wave: how many of them hold (each above
// the one before, `last` before the first; its position and its place in pages of the slot), and
// this lane's.
struct KvStep {
  int from, src, dst;  // the entry; the pages of its position and of its place
};
__device__ __forceinline__ int kv_path(const KvAccept& a, int s, int base, int d0, int n, int& last, KvStep& e) {
  const int lane = threadIdx.x & 63, d = d0 + lane;
  e.from = d < n ? a.path[s * a.ld_path + d] : -1;
  int before = __shfl_up(e.from, 1);
  if (lane == 0) before = last;
  bool ok = d < n && e.from > before && e.from < a.c.capacity() - base;
  if (ok) {
    e.src = a.c.page(s, (base + e.from) >> a.c.page_log);
    e.dst = a.c.page(s, (base + d) >> a.c.page_log);
    ok = e.src >= 0 && e.dst >= 0;
  }
  last = __builtin_amdgcn_readlane(e.from, 63);
  const uint64_t bad = ~__ballot(ok);
  return bad ? __builtin_ctzll(bad) : 64;
}
}  // namespace qmm

// Position base + path[d] to base + d, a thread a 16-byte column of a layer's, side's and
// head's rows. path[d] >= d and rises, so that no entry is on a row that an earlier one's goes
// to: eight are read and then written. The lengths here too, unless another workgroup may yet
// read them (lens_out null). 16 trees with 8 rows accepted each in 32 layers of 8 bf16 heads of 128:
// 5.4 us for 14.7 MB, of which the launch, the lists' round trips and one of the rows' are most.
extern "C" __global__ void __launch_bounds__(256) qmm_kv_accept_rows(qmm::KvAccept a) {
  using namespace qmm;
  __shared__ long long from[64], to[64];
  __shared__ int held;
  const KvCache& c = a.c;
  const int s = blockIdx.y, base = c.length(s), n = min(a.counts[s], a.max_path), t = threadIdx.x;
  const int per = (c.head_dim << c.esize_log()) / 16, low = (1 << c.page_log) - 1;
  const unsigned i = blockIdx.x * 256 + t;
  const bool on = i < 2u * c.layers * c.kv_heads * per;
  const int x = (int)(i % per), g = (int)(i / per % c.kv_heads), side = (int)(i / per / c.kv_heads % 2);
  const int layer = on ? (int)(i / per / c.kv_heads / 2) : 0;
  u32x4* pool = (u32x4*)((char*)(side ? c.v : c.k) + (c.row(layer, 0, g, 0) << c.esize_log())) + x;
  int last = -1, done = 0;
  for (int d0 = 0; d0 < n; d0 += 64) {
    if (t < 64) {
      KvStep e;
      const int k = kv_path(a, s, base, d0, n, last, e);
      if (t < k) {  // (in 16-byte units from the head's rows in page 0)
        from[t] = c.row(0, e.src, 0, (base + e.from) & low) / c.head_dim * per;
        to[t] = c.row(0, e.dst, 0, (base + d0 + t) & low) / c.head_dim * per;
      }
      if (t == 0) held = k;
    }
    __syncthreads();
    const int k = held;
    if (on)
      for (int d = 0; d < k; d += 8) {
        u32x4 v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = pool[from[min(d + e, k - 1)]];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (d + e < k && from[d + e] != to[d + e]) pool[to[d + e]] = v[e];
      }
    done += k;
    if (k < 64) break;
    __syncthreads();
  }
  if (a.lens_out && blockIdx.x == 0 && t == 0) a.lens_out[s] = base + done;
}

// The lengths alone, a wave a slot.
extern "C" __global__ void __launch_bounds__(256) qmm_kv_accept_lens(qmm::KvAccept a) {
  using namespace qmm;
  const int s = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (s >= a.c.slots) return;
  const int base = a.c.length(s);
  int d = 0;
  if (a.path) {
    const int n = min(a.counts[s], a.max_path);
    for (int last = -1; d < n;) {
      KvStep e;
      const int k = kv_path(a, s, base, d, n, last, e);
      d += k;
      if (k < 64) break;
    }
  } else {  // page by page
    const int n = min(max(a.counts[s], 0), a.c.capacity() - base);
    while (d < n && a.c.page(s, (base + d) >> a.c.page_log) >= 0)
      d = min(((((base + d) >> a.c.page_log) + 1) << a.c.page_log) - base, n);
  }
  if ((threadIdx.x & 63) == 0) a.lens_out[s] = base + d;
}

// ---------------------------------------------------------------------------
// compact
// ---------------------------------------------------------------------------
namespace qmm {
struct KvCompact {
  KvCache c;
  int32_t *table_out, *refs_out, *used;
  // workspace
  int32_t *map, *refs;  // [pages]: where a page goes, the new counts
  int32_t* moves;       // [1 + 3 pages / 2], as a fork's
};
}  // namespace qmm

// One workgroup: the pages in use, then the i-th of those behind their number to the i-th
// free one below it, 1024 pages a round: 8.4 us for 2048 pages, 145 for 65536.
extern "C" __global__ void __launch_bounds__(1024) qmm_kv_compact_plan(qmm::KvCompact k) {
  using namespace qmm;
  __shared__ int lds[16];
  const int t = threadIdx.x, pages = k.c.pages;
  int mine = 0, used;
  for (int p = t; p < pages; p += 1024) mine += k.c.refs[p] != 0;
  (void)block_sums(mine, lds, &used);
  int src = 0, dst = 0;
  for (int p0 = 0; p0 < pages; p0 += 1024) {
    const int p = p0 + t;
    const int refs = p < pages ? k.c.refs[p] : 0;
    const bool from = p < pages && refs != 0 && p >= used, to = p < used && refs == 0;
    int ns, nd;
    const int i = block_sums(from, lds, &ns), j = block_sums(to, lds, &nd);
    if (from) agent_store(k.moves + 1 + 3 * (src + i), p);
    if (to) agent_store(k.moves + 2 + 3 * (dst + j), p);
    if (p < pages) {
      agent_store(k.map + p, p);
      agent_store(k.refs + p, p < used ? refs : 0);
    }
    src += ns;
    dst += nd;
  }
  agent_barrier();
  if (t == 0) {
    agent_store(k.moves, src);
    k.used[0] = used;
  }
  for (int i = t; i < src; i += 1024) {
    const int a = agent_load(k.moves + 1 + 3 * i), b = agent_load(k.moves + 2 + 3 * i);
    agent_store(k.moves + 3 + 3 * i, 1 << k.c.page_log);
    agent_store(k.map + a, b);
    agent_store(k.refs + b, k.c.refs[a]);
  }
}

// The lists and the copies, as a fork's.
extern "C" __global__ void __launch_bounds__(256) qmm_kv_compact_commit(qmm::KvCompact k, int lists) {
  using namespace qmm;
  if (blockIdx.x >= (unsigned)lists) {
    kv_copy_pages(k.c, k.moves, blockIdx.x - lists, gridDim.x - lists);
    return;
  }
  const long long n = lists * 256LL, t = blockIdx.x * 256LL + threadIdx.x;
  for (long long p = t; p < k.c.pages; p += n) k.refs_out[p] = k.refs[p];
  const long long cells = (long long)k.c.slots * k.c.max_pages;
  for (long long i = t; i < cells; i += n) {
    const int p = k.c.table[i];
    k.table_out[i] = p >= 0 && p < k.c.pages ? k.map[p] : p;
  }
}
