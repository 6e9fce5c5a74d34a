// Host side of the cache in pages and of the beam search's selection (included by
// qmm_host.cpp after its helpers). Kernels: qmm_kv_*_kernels.h, qmm_beam_kernels.h.
#pragma once

namespace {

bool kv_type(int dtype) { return dtype == QMM_F32 || dtype == QMM_F16 || dtype == QMM_BF16; }
size_t kv_esize(int dtype) { return dtype == QMM_F32 ? 4 : 2; }
size_t kv_align(size_t v) { return (v + 255) & ~(size_t)255; }

// The kernels' by-value arguments (qmm::KvCache, KvRows, ...).
struct KvCache {
  void *k, *v;
  const int32_t *table, *lens, *refs;
  int pages, dtype, layers, kv_heads, page_log, head_dim, slots, max_pages;
};
struct KvRows {
  const int32_t* starts;
  int rows, max_rows;
};

int kv_shape(const qmm_kv_cache* c) {
  if (!c) return fail(QMM_ERR_INVALID, "null cache");
  if (!kv_type(c->dtype)) return fail(QMM_ERR_INVALID, "cache type %d (QMM_F32, QMM_F16 or QMM_BF16)", c->dtype);
  if (c->head_dim != 64 && c->head_dim != 128 && c->head_dim != 256)
    return fail(QMM_ERR_INVALID, "head_dim %d (64, 128 or 256)", c->head_dim);
  if (c->page_size < 16 || c->page_size > 1024 || (c->page_size & (c->page_size - 1)))
    return fail(QMM_ERR_INVALID, "page size %d (a power of two, 16 .. 1024)", c->page_size);
  if (c->layers < 1 || c->layers > 1024 || c->kv_heads < 1 || c->kv_heads > 256)
    return fail(QMM_ERR_INVALID, "%d layers of %d kv heads (1 .. 1024, 1 .. 256)", c->layers, c->kv_heads);
  if (c->pages < 1 || c->pages > (1LL << 24)) return fail(QMM_ERR_INVALID, "%lld pages (1 .. 2^24)", (long long)c->pages);
  if (c->slots < 1 || c->slots > 4096 || c->max_pages < 1 || c->max_pages > (1 << 20) ||
      (int64_t)c->max_pages * c->page_size > (1LL << 28) || (int64_t)c->slots * c->max_pages > (1LL << 28))
    return fail(QMM_ERR_INVALID, "table of %d slots x %d pages: slots <= 4096, max_pages <= 2^20, max_pages * page_size "
                "and slots * max_pages <= 2^28", c->slots, c->max_pages);
  return QMM_OK;
}

int kv_cache(const qmm_kv_cache* c, KvCache* out) {
  QMM_TRY(kv_shape(c));
  if (!c->k || !c->v || !c->table || !c->lens || !c->refs) return fail(QMM_ERR_INVALID, "null pointer in the cache");
  if ((uintptr_t)c->k % 16 || (uintptr_t)c->v % 16) return fail(QMM_ERR_INVALID, "cache pools must be 16-byte aligned");
  *out = {c->k, c->v, c->table, c->lens, c->refs, (int)c->pages, c->dtype, c->layers, c->kv_heads,
          __builtin_ctz((unsigned)c->page_size), c->head_dim, c->slots, c->max_pages};
  return QMM_OK;
}

int kv_layer(const qmm_kv_cache* c, int layer) {
  if (layer < 0 || layer >= c->layers) return fail(QMM_ERR_INVALID, "layer %d of %d", layer, c->layers);
  return QMM_OK;
}

// A workspace of `need` bytes, laid out in parts of 256 bytes.
int kv_workspace(const void* ws, size_t bytes, size_t need) {
  if (need == 0) return QMM_OK;
  if (!ws || bytes < need) return fail(QMM_ERR_INVALID, "workspace of %zu B < %zu B needed", ws ? bytes : 0, need);
  if ((uintptr_t)ws % 16) return fail(QMM_ERR_INVALID, "workspaces must be 16-byte aligned");
  return QMM_OK;
}

template <typename T>
T* kv_take(uint8_t*& p, size_t n) {
  T* at = (T*)p;
  p += kv_align(n * sizeof(T));
  return at;
}

int kv_launch(Device* d, const char* name, unsigned gx, unsigned gy, unsigned block, hipStream_t s, void** args) {
  hipFunction_t f;
  QMM_TRY(kernel(d, name, &f));
  QMM_HIP(hipModuleLaunchKernel(f, gx, gy, 1, block, 1, 1, 0, s, args, nullptr));
  return QMM_OK;
}

int kv_check_rows(int64_t rows) {
  if (rows < 0 || rows > (1LL << 20)) return fail(QMM_ERR_INVALID, "%lld rows (0 .. 2^20)", (long long)rows);
  return QMM_OK;
}

// Rows of `n` values apart by ld; `what` names them.
int kv_stride(int64_t rows, int64_t ld, int64_t n, const char* what) {
  if (ld > (1LL << 40) || (rows > 1 && ld < n)) return fail(QMM_ERR_INVALID, "%s: row stride %lld of rows of %lld", what, (long long)ld, (long long)n);
  return QMM_OK;
}

// Whether `rows` rows of na and nb bytes, apart by lda and ldb, share a byte (rows of one stride may lie between each
// other; of two strides they are taken to where their ranges meet).
bool kv_meet(const void* a, int64_t lda, int64_t na, const void* b, int64_t ldb, int64_t nb, int64_t rows) {
  const uintptr_t a0 = (uintptr_t)a, b0 = (uintptr_t)b;
  const uintptr_t a1 = a0 + (uintptr_t)((rows - 1) * lda + na), b1 = b0 + (uintptr_t)((rows - 1) * ldb + nb);
  if (a1 <= b0 || b1 <= a0) return false;
  if (rows == 1 || lda != ldb) return true;
  const uintptr_t off = (b0 - a0) % (uintptr_t)lda, ld = (uintptr_t)lda;  // of b's row in one of a's strides
  return b0 >= a0 ? off < (uintptr_t)na || off + (uintptr_t)nb > ld
                  : kv_meet(b, ldb, nb, a, lda, na, rows);
}

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

struct KvAttn {
  KvCache c;
  KvRows r;
  const void* q;
  const uint64_t* masks;
  void* out;
  float *part, *state;
  long long ldq, ldm, ldo;
  int layer, x_type, heads, wide, out_wide, splits, chunk;
  int tiles, group_rows, join_lanes;
  float scale;
};

// Bytes that a call reads or writes (p null: none).
struct KvBytes {
  const void* p;
  size_t n;
};
bool kv_meet(const KvBytes& a, const KvBytes& b) {
  return a.p && b.p && (uintptr_t)a.p < (uintptr_t)b.p + b.n && (uintptr_t)b.p < (uintptr_t)a.p + a.n;
}
// A call's outputs lie apart from each other and from its inputs; output i may be input i itself.
int kv_apart(std::initializer_list<KvBytes> outs, std::initializer_list<KvBytes> ins, const char* rule) {
  for (const KvBytes* a = outs.begin(); a != outs.end(); ++a) {
    for (const KvBytes* b = a + 1; b != outs.end(); ++b)
      if (kv_meet(*a, *b)) return fail(QMM_ERR_INVALID, "%s", rule);
    for (const KvBytes* b = ins.begin(); b != ins.end(); ++b)
      if (kv_meet(*a, *b) && !(a - outs.begin() == b - ins.begin() && a->p == b->p)) return fail(QMM_ERR_INVALID, "%s", rule);
  }
  return QMM_OK;
}

// How an attention's rows and positions are split. form 0, 1: one tile of 16 or 32 columns (rows
// x heads of a kv head) a slot, 2: groups of four tiles of 32. `splits` chunks of a slot's
// positions at most, of `chunk` (a multiple of 128) or more.
struct KvSplit {
  int form, tiles, group_rows, splits, chunk;
  size_t parts;  // bytes of the partial outputs, a multiple of 256
  size_t bytes;
};
KvSplit kv_split(const qmm_kv_cache* c, int64_t rows, int max_rows, int64_t max_len, int heads) {
  KvSplit p;
  const int64_t G = heads / c->kv_heads, per = 32 / G, most_rows = std::min<int64_t>(max_rows, std::max<int64_t>(rows, 1));
  p.form = most_rows * G <= 16 ? 0 : most_rows <= per ? 1 : 2;
  p.group_rows = (int)(p.form == 0 ? 16 / G : p.form == 1 ? per : 4 * per);
  p.tiles = (int)ceil_div(most_rows, p.group_rows);
  const int64_t most = std::min<int64_t>(max_len, (int64_t)c->max_pages * c->page_size);
  const int64_t units = (int64_t)c->slots * c->kv_heads * p.tiles;
  // Few columns: a chunk's record is small, so many short chunks even out sequences of different lengths (24 of up to
  // 8000 positions: 86.7 us with 10 chunks, 89.5 with 4), but not so short that the chip is full of their beginnings
  // (64 of up to 1000: 28 us whole, 34 in two; one of 30000: 28 us with chunks of 256, 34 of 128). More columns: a
  // chunk writes and reads 0.5 KB a column (8 trees of up to 26 nodes over up to 4000 positions: 50 us with 12 chunks
  // of at least 384, 58 with 32), unless CUs would be idle (one tree over 3000 positions: 33 us with 8, 27 with 24).
  auto splits = [&](int64_t wgs, int64_t least) { return std::max<int64_t>(1, std::min<int64_t>(wgs / units, ceil_div(most, least))); };
  p.splits = (int)(p.form == 0 ? splits(units < 64 ? 1024 : 2048, 128 * ceil_div(units, 64))
                               : std::max(splits(768, 384), splits(256, 128)));
  p.chunk = (int)ceil_div(ceil_div(most, p.splits), 128) * 128;
  const size_t records = p.splits > 1 ? (size_t)rows * heads * p.splits : 0;
  p.parts = kv_align(records * c->head_dim * 4);
  p.bytes = p.parts + kv_align(records * 8);
  return p;
}

// List entries up to which one workgroup does a fork (qmm::kForkLists).
constexpr int64_t kKvForkSmall = 16384;
struct KvFork {
  KvCache c;
  const int32_t *parents, *keep;
  int32_t *table_out, *lens_out, *refs_out, *shortage;
  int reserve;
  int32_t *refs, *writers, *first, *free_ids, *table, *lens, *at, *parent, *copy, *moves;
};

struct KvAccept {
  KvCache c;
  const int32_t *path, *counts;
  int32_t* lens_out;
  long long ld_path;
  int max_path;
};

struct KvCompact {
  KvCache c;
  int32_t *table_out, *refs_out, *used;
  int32_t *map, *refs, *moves;
};

// Workgroups for up to `most` page copies: as many as fill the chip (how many copies there are is known on the device
// alone).
unsigned kv_copy_grid(const Device* d, const KvCache& c, int64_t most) {
  return (unsigned)std::min<int64_t>(most * c.layers * 2 * c.kv_heads, 8LL * d->num_cu);
}

// Workgroups of 256 for n elements, at most a few a CU.
unsigned kv_grid(const Device* d, int64_t n) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(n, 256), 4LL * d->num_cu)); }

struct BeamArgs {
  const void* logits;
  long long ld;
  const float* scores;
  const int32_t* finished;
  int32_t *tokens, *parents, *out_finished;
  float* out_scores;
  double* sums;
  float* maxima;
  uint64_t* lists;
  int type, beams, vocab, count, eos, slices, wide;
};
constexpr int64_t kBeamSlice = 4096, kBeamMaxVocab = 1 << 20;
constexpr int kBeamMax = 64, kBeamMaxCount = 128;

}  // namespace

extern "C" {

int qmm_kv_append(const qmm_kv_cache* cache, int layer, const void* q, const void* k, const void* v, int x_dtype,
                  int64_t rows, int64_t ldq, int64_t ldk, int64_t ldv, const int32_t* starts, const int32_t* depths,
                  const float* cos_t, const float* sin_t, int64_t positions, void* q_out, int64_t ldqo, int heads,
                  void* stream) {
  KvAppend a = {};
  QMM_TRY(kv_cache(cache, &a.c));
  QMM_TRY(kv_layer(cache, layer));
  QMM_TRY(kv_check_rows(rows));
  if (rows && (!k || !v || !starts || (!cos_t != !sin_t) || (q && !q_out))) return fail(QMM_ERR_INVALID, "null pointer");
  if (!kv_type(x_dtype)) return fail(QMM_ERR_INVALID, "row type %d (QMM_F32, QMM_F16 or QMM_BF16)", x_dtype);
  if (q && (heads < 1 || heads > 8192)) return fail(QMM_ERR_INVALID, "%d heads (1 .. 8192)", heads);
  if (cos_t && (positions < 1 || positions > (1LL << 30))) return fail(QMM_ERR_INVALID, "tables of %lld positions", (long long)positions);
  const int64_t dim = cache->head_dim, width = cache->kv_heads * dim;
  QMM_TRY(kv_stride(rows, ldk, width, "k"));
  QMM_TRY(kv_stride(rows, ldv, width, "v"));
  if (q) {
    QMM_TRY(kv_stride(rows, ldq, heads * dim, "q"));
    QMM_TRY(kv_stride(rows, ldqo, heads * dim, "q_out"));
  }
  if (rows == 0) return QMM_OK;
  if (q) {
    const int64_t e = (int64_t)kv_esize(x_dtype), out = heads * dim * e;
    if ((!(q == q_out && (ldq == ldqo || rows == 1)) && kv_meet(q, ldq * e, out, q_out, ldqo * e, out, rows)) ||
        kv_meet(k, ldk * e, width * e, q_out, ldqo * e, out, rows) || kv_meet(v, ldv * e, width * e, q_out, ldqo * e, out, rows))
      return fail(QMM_ERR_INVALID, "q_out overlaps the rows (it may be q itself)");
  }
  Device* d;
  QMM_TRY(current_device(&d));
  const size_t four = 4 * kv_esize(x_dtype);
  auto even = [&](const void* p, int64_t ld) { return !p || ((uintptr_t)p % four == 0 && ld % 4 == 0); };
  a.r = {starts, (int)rows, (int)rows};
  a.q = q, a.k = k, a.v = v, a.depths = depths, a.cos_t = cos_t, a.sin_t = sin_t, a.q_out = q_out;
  a.ldq = ldq, a.ldk = ldk, a.ldv = ldv, a.ldqo = ldqo;
  a.layer = layer, a.x_type = x_dtype, a.heads = q ? heads : 0, a.positions = (int)positions;
  a.wide = even(q, ldq) && even(k, ldk) && even(v, ldv) && even(q ? q_out : nullptr, ldqo) &&
           (uintptr_t)cos_t % 16 == 0 && (uintptr_t)sin_t % 16 == 0;
  const int group = 256 / (cache->head_dim / 8);
  const int64_t blocks = ceil_div(a.heads + 2 * cache->kv_heads, group);
  if (rows * blocks >= (1LL << 24)) return fail(QMM_ERR_INVALID, "%lld rows of %d heads are too many", (long long)rows, a.heads);
  void* args[] = {&a};
  return kv_launch(d, "qmm_kv_append_rows", (unsigned)(rows * blocks), 1, 256, (hipStream_t)stream, args);
}

static int kv_check_attention(const qmm_kv_cache* cache, int64_t rows, int max_rows, int64_t max_len, int heads) {
  QMM_TRY(kv_shape(cache));
  QMM_TRY(kv_check_rows(rows));
  if (heads < 1 || heads % cache->kv_heads || heads / cache->kv_heads > 32)
    return fail(QMM_ERR_INVALID, "%d heads over %d kv heads (a multiple, up to 32 times)", heads, cache->kv_heads);
  if (max_rows < 1) return fail(QMM_ERR_INVALID, "max_rows %d", max_rows);
  if (max_len < 1) return fail(QMM_ERR_INVALID, "max_len %lld", (long long)max_len);
  return QMM_OK;
}

size_t qmm_kv_attention_workspace_size(const qmm_kv_cache* cache, int64_t rows, int max_rows, int64_t max_len,
                                       int heads) {
  if (kv_check_attention(cache, rows, max_rows, max_len, heads) != QMM_OK) return 0;
  return kv_split(cache, rows, max_rows, max_len, heads).bytes;
}

int qmm_kv_attention(const qmm_kv_cache* cache, int layer, const void* q, int x_dtype, int64_t rows, int64_t ldq,
                     const int32_t* starts, const uint64_t* masks, int64_t ldm, int max_rows, int64_t max_len,
                     int heads, float scale, void* out, int64_t ldo, void* ws, size_t ws_bytes, void* stream) {
  QMM_TRY(kv_check_attention(cache, rows, max_rows, max_len, heads));
  KvAttn a = {};
  QMM_TRY(kv_cache(cache, &a.c));
  QMM_TRY(kv_layer(cache, layer));
  if (rows && (!q || !starts || !out)) return fail(QMM_ERR_INVALID, "null pointer");
  if (!std::isfinite(scale)) return fail(QMM_ERR_INVALID, "scale %g", scale);
  if (!kv_type(x_dtype)) return fail(QMM_ERR_INVALID, "row type %d (QMM_F32, QMM_F16 or QMM_BF16)", x_dtype);
  if (masks && (ldm < 1 || ldm > (1 << 20) || max_rows > 64 * ldm))
    return fail(QMM_ERR_INVALID, "masks of %lld words for %d rows a slot", (long long)ldm, max_rows);
  QMM_TRY(kv_stride(rows, ldq, (int64_t)heads * cache->head_dim, "q"));
  QMM_TRY(kv_stride(rows, ldo, (int64_t)heads * cache->head_dim, "out"));
  const int64_t esize = (int64_t)kv_esize(x_dtype), row_bytes = heads * cache->head_dim * esize;
  if (rows && !(q == out && (ldq == ldo || rows == 1)) && kv_meet(q, ldq * esize, row_bytes, out, ldo * esize, row_bytes, rows))
    return fail(QMM_ERR_INVALID, "out overlaps q (it may be q itself)");
  QMM_TRY(kv_workspace(ws, ws_bytes, qmm_kv_attention_workspace_size(cache, rows, max_rows, max_len, heads)));
  if (rows == 0) return QMM_OK;
  Device* d;
  QMM_TRY(current_device(&d));
  const KvSplit p = kv_split(cache, rows, max_rows, max_len, heads);
  const int64_t units = (int64_t)cache->slots * p.splits * cache->kv_heads;
  if ((units + 7) / 8 * 8 * p.tiles >= (1LL << 24)) return fail(QMM_ERR_INVALID, "%d slots of up to %d rows are too many at once", cache->slots, max_rows);
  const size_t four = 4 * kv_esize(x_dtype);
  a.r = {starts, (int)rows, max_rows};
  a.q = q, a.masks = masks, a.out = out, a.ldq = ldq, a.ldm = ldm, a.ldo = ldo;
  a.part = (float*)ws, a.state = ws ? (float*)((uint8_t*)ws + p.parts) : nullptr;
  a.layer = layer, a.x_type = x_dtype, a.heads = heads, a.scale = scale;
  a.wide = (uintptr_t)q % four == 0 && ldq % 4 == 0;
  a.out_wide = (uintptr_t)out % four == 0 && ldo % 4 == 0;
  a.splits = p.splits, a.chunk = p.chunk, a.tiles = p.tiles, a.group_rows = p.group_rows;
  // (a thread has four chunks' loads in flight)
  a.join_lanes = 1;
  while (4 * a.join_lanes < p.splits && a.join_lanes < 1024 / cache->head_dim) a.join_lanes *= 2;
  // parts that hold the bits of q (24, 11, 8) in the cache's type, and of the weights
  int qp = 1, pp = 1;
  if (cache->dtype == QMM_BF16) {
    qp = x_dtype == QMM_F32 ? 3 : x_dtype == QMM_F16 ? 2 : 1;
    pp = x_dtype == QMM_F32 ? 3 : 2;
  } else if (cache->dtype == QMM_F16) {
    qp = x_dtype == QMM_F32 ? 2 : 1;
    pp = 2;
  }
  char name[64];
  const char* const forms[] = {"n16", "n32", "wide"};
  snprintf(name, sizeof(name), "qmm_kv_attn_%s_d%d_%s_q%d_p%d", mx_type_name(cache->dtype), cache->head_dim, forms[p.form], qp, pp);
  const unsigned threads = cache->dtype == QMM_F32 && cache->head_dim == 256 && p.form != 2 ? 128 : 256;
  const hipStream_t s = (hipStream_t)stream;
  void* args[] = {&a};
  QMM_TRY(kv_launch(d, name, (unsigned)((units + 7) / 8 * 8 * p.tiles), 1, threads, s, args));
  if (p.splits == 1) return QMM_OK;
  return kv_launch(d, "qmm_kv_attn_join", (unsigned)rows, ceil_div(heads, 1024 / (cache->head_dim * a.join_lanes)), 256, s, args);
}

size_t qmm_kv_fork_workspace_size(const qmm_kv_cache* cache) {
  if (kv_shape(cache) != QMM_OK) return 0;
  const size_t pages = (size_t)cache->pages, slots = (size_t)cache->slots, cells = slots * (size_t)cache->max_pages;
  return 4 * kv_align(4 * pages) + kv_align(4 * cells) + 4 * kv_align(4 * slots) + kv_align(4 * (1 + 3 * slots));
}

int qmm_kv_fork(const qmm_kv_cache* cache, const int32_t* parents, const int32_t* keep, int reserve,
                int32_t* table_out, int32_t* lens_out, int32_t* refs_out, int32_t* shortage, void* ws,
                size_t ws_bytes, void* stream) {
  KvFork f = {};
  QMM_TRY(kv_cache(cache, &f.c));
  if (!parents || !table_out || !lens_out || !refs_out || !shortage) return fail(QMM_ERR_INVALID, "null pointer");
  if (reserve < 0 || reserve > cache->max_pages * cache->page_size)
    return fail(QMM_ERR_INVALID, "reserve of %d positions (0 .. max_pages * page_size)", reserve);
  const size_t need = qmm_kv_fork_workspace_size(cache), pages = (size_t)cache->pages, slots = (size_t)cache->slots;
  const int64_t cells = (int64_t)cache->slots * cache->max_pages;
  QMM_TRY(kv_workspace(ws, ws_bytes, need));
  // (parents and keep are read before any list is written, but beside the workspace)
  const char* const rule = "fork: the new lists may be the cache's own, and overlap them, each other, shortage and the workspace in no other way";
  QMM_TRY(kv_apart({{table_out, 4 * (size_t)cells}, {lens_out, 4 * slots}, {refs_out, 4 * pages}, {shortage, 4}, {ws, need}},
                   {{cache->table, 4 * (size_t)cells}, {cache->lens, 4 * slots}, {cache->refs, 4 * pages}}, rule));
  QMM_TRY(kv_apart({{ws, need}}, {{nullptr, 0}, {parents, 4 * slots}, {keep, 4 * slots}}, "fork: the workspace overlaps parents or keep"));
  Device* d;
  QMM_TRY(current_device(&d));
  uint8_t* p = (uint8_t*)ws;
  f.parents = parents, f.keep = keep, f.reserve = reserve;
  f.table_out = table_out, f.lens_out = lens_out, f.refs_out = refs_out, f.shortage = shortage;
  f.refs = kv_take<int32_t>(p, pages), f.writers = kv_take<int32_t>(p, pages), f.first = kv_take<int32_t>(p, pages);
  f.free_ids = kv_take<int32_t>(p, pages), f.table = kv_take<int32_t>(p, (size_t)cells);
  f.lens = kv_take<int32_t>(p, slots), f.at = kv_take<int32_t>(p, slots), f.parent = kv_take<int32_t>(p, slots);
  f.copy = kv_take<int32_t>(p, slots), f.moves = kv_take<int32_t>(p, 1 + 3 * slots);
  const hipStream_t s = (hipStream_t)stream;
  void* args[] = {&f};
  const int64_t n = std::max<int64_t>(cells, cache->pages);
  if (cells + 4 * (cache->pages + cache->slots) <= kKvForkSmall) {
    QMM_TRY(kv_launch(d, "qmm_kv_fork_small", 1, 1, 1024, s, args));
    if (reserve == 0) return QMM_OK;  // nothing is about to be written: no copies
    void* copy[] = {&f.c, &f.moves};
    return kv_launch(d, "qmm_kv_copy_pages", kv_copy_grid(d, f.c, cache->slots), 1, 256, s, copy);
  } else {
    QMM_TRY(kv_launch(d, "qmm_kv_fork_begin", kv_grid(d, n), 1, 256, s, args));
    QMM_TRY(kv_launch(d, "qmm_kv_fork_count", kv_grid(d, 64LL * cache->slots), 1, 256, s, args));
    QMM_TRY(kv_launch(d, "qmm_kv_fork_plan", 1, 1, 1024, s, args));
    int lists = (int)kv_grid(d, n);
    void* last[] = {&f, &lists};
    return kv_launch(d, "qmm_kv_fork_commit", lists + (reserve ? kv_copy_grid(d, f.c, cache->slots) : 0), 1, 256, s, last);
  }
}

int qmm_kv_accept(const qmm_kv_cache* cache, const int32_t* path, int64_t ld_path, const int32_t* counts,
                  int32_t* lens_out, void* stream) {
  KvAccept a = {};
  QMM_TRY(kv_cache(cache, &a.c));
  if (!counts || !lens_out) return fail(QMM_ERR_INVALID, "null pointer");
  const uintptr_t out = (uintptr_t)lens_out, lens = 4 * (uintptr_t)cache->slots;
  auto meets = [&](const void* p, uintptr_t n) { return p && out < (uintptr_t)p + n && (uintptr_t)p < out + lens; };
  if (path && (ld_path < 1 || ld_path > (1 << 20))) return fail(QMM_ERR_INVALID, "paths of %lld entries (1 .. 2^20)", (long long)ld_path);
  if ((lens_out != cache->lens && meets(cache->lens, lens)) || (lens_out != counts && meets(counts, lens)) ||
      meets(path, lens * (uintptr_t)ld_path) || meets(cache->table, lens * (uintptr_t)cache->max_pages) ||
      meets(cache->refs, 4 * (uintptr_t)cache->pages))
    return fail(QMM_ERR_INVALID, "lens_out overlaps the lengths, the counts (it may be either itself), the paths or the pages' lists");
  Device* d;
  QMM_TRY(current_device(&d));
  a.path = path, a.counts = counts, a.lens_out = lens_out, a.ld_path = ld_path, a.max_path = (int)ld_path;
  const hipStream_t s = (hipStream_t)stream;
  void* args[] = {&a};
  if (path) {
    // (lengths that stand where they or the counts are read from change behind the last read, in a launch of their own)
    const bool own = lens_out == cache->lens || lens_out == counts;
    if (own) a.lens_out = nullptr;
    const int64_t columns = 2LL * cache->layers * cache->kv_heads * ((int64_t)cache->head_dim * kv_esize(cache->dtype) / 16);
    QMM_TRY(kv_launch(d, "qmm_kv_accept_rows", ceil_div(columns, 256), (unsigned)cache->slots, 256, s, args));
    if (!own) return QMM_OK;
    a.lens_out = lens_out;
  }
  return kv_launch(d, "qmm_kv_accept_lens", ceil_div(cache->slots, 4), 1, 256, s, args);
}

size_t qmm_kv_compact_workspace_size(const qmm_kv_cache* cache) {
  if (kv_shape(cache) != QMM_OK) return 0;
  const size_t pages = (size_t)cache->pages;
  return 2 * kv_align(4 * pages) + kv_align(4 * (1 + 3 * (pages / 2 + 1)));
}

int qmm_kv_compact(const qmm_kv_cache* cache, int32_t* table_out, int32_t* refs_out, int32_t* used, void* ws,
                   size_t ws_bytes, void* stream) {
  KvCompact k = {};
  QMM_TRY(kv_cache(cache, &k.c));
  if (!table_out || !refs_out || !used) return fail(QMM_ERR_INVALID, "null pointer");
  const size_t need = qmm_kv_compact_workspace_size(cache), pages = (size_t)cache->pages, slots = (size_t)cache->slots;
  const size_t cells = slots * (size_t)cache->max_pages;
  QMM_TRY(kv_workspace(ws, ws_bytes, need));
  QMM_TRY(kv_apart({{table_out, 4 * cells}, {refs_out, 4 * pages}, {used, 4}, {ws, need}},
                   {{cache->table, 4 * cells}, {cache->refs, 4 * pages}, {nullptr, 0}, {nullptr, 0}, {cache->lens, 4 * slots}},
                   "compact: the new lists may be the cache's own, and overlap them, each other, used and the workspace in no other way"));
  Device* d;
  QMM_TRY(current_device(&d));
  uint8_t* p = (uint8_t*)ws;
  k.table_out = table_out, k.refs_out = refs_out, k.used = used;
  k.map = kv_take<int32_t>(p, pages), k.refs = kv_take<int32_t>(p, pages), k.moves = kv_take<int32_t>(p, 1 + 3 * (pages / 2 + 1));
  const hipStream_t s = (hipStream_t)stream;
  void* args[] = {&k};
  QMM_TRY(kv_launch(d, "qmm_kv_compact_plan", 1, 1, 1024, s, args));
  int lists = (int)kv_grid(d, std::max<int64_t>((int64_t)cache->slots * cache->max_pages, cache->pages));
  void* last[] = {&k, &lists};
  return kv_launch(d, "qmm_kv_compact_commit", lists + kv_copy_grid(d, k.c, cache->pages / 2 + 1), 1, 256, s, last);
}

static int beam_shape(int64_t batch, int beams, int64_t vocab, int count) {
  if (batch < 1 || batch > 65535 || beams < 1 || beams > kBeamMax || vocab < 1 || vocab > kBeamMaxVocab || count < 1 ||
      count > kBeamMaxCount || batch * beams > 65535)
    return fail(QMM_ERR_INVALID, "beam search of %lld x %d beams over %lld tokens, %d continuations (up to 65535 beams in "
                "all, %d a search, 2^20 tokens, %d continuations)", (long long)batch, beams, (long long)vocab, count, kBeamMax, kBeamMaxCount);
  return QMM_OK;
}

size_t qmm_beam_select_workspace_size(int64_t batch, int beams, int64_t vocab, int count) {
  if (beam_shape(batch, beams, vocab, count) != QMM_OK) return 0;
  const size_t lists = (size_t)(batch * beams) * ceil_div(vocab, kBeamSlice);
  return kv_align(8 * lists) + kv_align(4 * lists) + kv_align(8 * lists * (size_t)count);
}

int qmm_beam_select(const void* logits, int dtype, int64_t ld, int64_t batch, int beams, int64_t vocab,
                    const float* scores, const int32_t* finished, int eos, int count, int32_t* tokens,
                    int32_t* parents, float* out_scores, int32_t* out_finished, void* ws, size_t ws_bytes,
                    void* stream) {
  QMM_TRY(beam_shape(batch, beams, vocab, count));
  if (!logits || !scores || !tokens || !parents || !out_scores) return fail(QMM_ERR_INVALID, "null pointer");
  if (!kv_type(dtype)) return fail(QMM_ERR_INVALID, "logits of type %d (QMM_F32, QMM_F16 or QMM_BF16)", dtype);
  if (eos < -1 || eos >= vocab) return fail(QMM_ERR_INVALID, "end token %d of %lld tokens (-1: none)", eos, (long long)vocab);
  if (finished && eos < 0) return fail(QMM_ERR_INVALID, "finished beams need an end token");
  QMM_TRY(kv_stride(batch * beams, ld, vocab, "logits"));
  const size_t need = qmm_beam_select_workspace_size(batch, beams, vocab, count);
  QMM_TRY(kv_workspace(ws, ws_bytes, need));
  const size_t rows = (size_t)(batch * beams), slices = ceil_div(vocab, kBeamSlice), out = 4 * (size_t)batch * (size_t)count;
  // (a search's workgroup reads its own beams' scores and ends before it writes: in place where it writes as many)
  const bool place = count == beams;
  const KvBytes in_scores = {scores, 4 * rows}, in_ends = {finished, 4 * rows}, none = {nullptr, 0};
  const KvBytes in_logits = {logits, (((rows - 1) * (size_t)(rows > 1 ? ld : 0)) + (size_t)vocab) * kv_esize(dtype)};
  const char* const rule = "beam selection: results overlap each other, the workspace or what is read (scores and ends may change in place "
                           "where count is beams)";
  QMM_TRY(kv_apart({{out_scores, out}, {out_finished, out}, {tokens, out}, {parents, out}, {ws, need}},
                   {place ? in_scores : none, place ? in_ends : none, none, none, none, in_logits, place ? none : in_scores,
                    place ? none : in_ends}, rule));
  Device* d;
  QMM_TRY(current_device(&d));
  uint8_t* p = (uint8_t*)ws;
  BeamArgs a = {};
  a.logits = logits, a.ld = ld, a.scores = scores, a.finished = finished;
  a.tokens = tokens, a.parents = parents, a.out_finished = out_finished, a.out_scores = out_scores;
  a.sums = kv_take<double>(p, rows * slices), a.maxima = kv_take<float>(p, rows * slices);
  a.lists = kv_take<uint64_t>(p, rows * slices * (size_t)count);
  a.type = dtype, a.beams = beams, a.vocab = (int)vocab, a.count = count, a.eos = eos, a.slices = (int)slices;
  a.wide = (uintptr_t)logits % 16 == 0 && ld * (int64_t)kv_esize(dtype) % 16 == 0;
  const hipStream_t s = (hipStream_t)stream;
  void* args[] = {&a};
  QMM_TRY(kv_launch(d, dtype == QMM_F32 ? "qmm_beam_slices_f32" : dtype == QMM_F16 ? "qmm_beam_slices_f16" : "qmm_beam_slices_bf16", (unsigned)slices, (unsigned)rows, 256, s, args));
  return kv_launch(d, "qmm_beam_merge", (unsigned)batch, 1, 256, s, args);
}

int qmm_reorder_rows(const void* src, int64_t src_rows, int64_t ld_src, void* dst, int64_t ld_dst,
                     int64_t row_bytes, const int32_t* index, int64_t rows, void* stream) {
  if (!src || !dst || !index) return fail(QMM_ERR_INVALID, "null pointer");
  if (src_rows < 0 || rows < 0 || rows > (1LL << 20) || src_rows > INT32_MAX || row_bytes < 0 || row_bytes > (1LL << 40) ||
      ld_src > (1LL << 40) || ld_dst > (1LL << 40) || (src_rows > 1 && ld_src > (1LL << 62) / src_rows) || (src_rows > 1 && ld_src < row_bytes) || (rows > 1 && ld_dst < row_bytes))
    return fail(QMM_ERR_INVALID, "reorder of %lld rows of %lld bytes out of %lld", (long long)rows, (long long)row_bytes, (long long)src_rows);
  if (rows == 0 || src_rows == 0 || row_bytes == 0) return QMM_OK;
  const uintptr_t s0 = (uintptr_t)src, d0 = (uintptr_t)dst;
  if (s0 < d0 + (uintptr_t)((rows - 1) * ld_dst + row_bytes) && d0 < s0 + (uintptr_t)((src_rows - 1) * ld_src + row_bytes))
    return fail(QMM_ERR_INVALID, "reorder: the rows overlap their source");
  Device* d;
  QMM_TRY(current_device(&d));
  long long sr = src_rows, ls = ld_src, ldd = ld_dst, rb = row_bytes;
  const uintptr_t bits = s0 | d0 | (uintptr_t)ld_src | (uintptr_t)ld_dst | (uintptr_t)row_bytes;
  int unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
  void* args[] = {&src, &sr, &ls, &dst, &ldd, &rb, &index, &unit};
  return kv_launch(d, "qmm_beam_reorder", (unsigned)rows, std::min(ceil_div(row_bytes / unit, 256), 64u), 256, (hipStream_t)stream, args);
}

}  // extern "C"
