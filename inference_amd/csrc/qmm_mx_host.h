// Host side of the microscaled types and of the scored routing (included by
// qmm_host.cpp after its helpers and qmm_qtensor). Formats and kernels:
// qmm_mx_common.h, qmm_mx_quant_kernels.h, qmm_mx_gemm_kernels.h, qmm_route_kernels.h.
#pragma once

namespace {

// qmm_mx_common.h's layout constants.
constexpr int64_t kMxTile = 32, kMxChunk = 256, kMxUnit = 4352, kMxXUnit = 12544;

bool is_mx(int dtype) { return dtype == QMM_MXFP4; }

int64_t mx_chunks(int64_t k) { return (k + kMxChunk - 1) / kMxChunk; }
size_t mx_weight_bytes(int64_t n, int64_t k) {
  return (size_t)((n + kMxTile - 1) / kMxTile) * (size_t)mx_chunks(k) * (size_t)kMxUnit;
}

size_t mx_align(size_t v) { return (v + 255) & ~(size_t)255; }

// Bytes of the digit planes of m rows of k values.
size_t mx_planes(int64_t m, int64_t k) {
  return (size_t)((m + kMxTile - 1) / kMxTile) * (size_t)mx_chunks(k) * (size_t)kMxXUnit;
}

const char* mx_type_name(int dtype) {
  return dtype == QMM_F32 ? "f32" : dtype == QMM_F16 ? "f16" : dtype == QMM_BF16 ? "bf16" : nullptr;
}
size_t mx_type_size(int dtype) { return dtype == QMM_F32 ? 4 : 2; }

// One workgroup a 32 x 256 unit of the weight.
int mx_units(int64_t n, int64_t k, unsigned* grid) {
  const int64_t u = (n + kMxTile - 1) / kMxTile * mx_chunks(k);
  if (u > (1LL << 31) - 1) return fail(QMM_ERR_INVALID, "MXFP4 tensor too large");
  *grid = (unsigned)u;
  return QMM_OK;
}

int mx_ggml(Device* d, const char* name, const void* src, int64_t n, int64_t k, void* dst, hipStream_t s) {
  unsigned grid = 0;
  QMM_TRY(mx_units(n, k, &grid));
  int nn = (int)n, kk = (int)k, kc = (int)mx_chunks(k);
  void* args[] = {&src, &nn, &kk, &dst, &kc};
  return launch(d, name, grid, 256, 0, s, args);
}

int mx_quantize_w(Device* d, const void* w, int w_dtype, int64_t n, int64_t k, void* out, hipStream_t s) {
  char name[40];
  snprintf(name, sizeof(name), "qmm_mx_quantize_w_%s", mx_type_name(w_dtype));
  // four values a thread and load
  if ((uintptr_t)w % (4 * mx_type_size(w_dtype))) return fail(QMM_ERR_INVALID, "MXFP4 quantize: the weight must start on a boundary of four values");
  return mx_ggml(d, name, w, n, k, out, s);
}

int mx_dequantize(Device* d, const void* w, int64_t n, int64_t k, void* dst, int out_dtype, hipStream_t s) {
  char name[40];
  snprintf(name, sizeof(name), "qmm_mx_dequantize_%s", mx_type_name(out_dtype));
  if ((uintptr_t)dst % (4 * mx_type_size(out_dtype))) return fail(QMM_ERR_INVALID, "MXFP4 dequantize: the output must start on a boundary of four values");
  return mx_ggml(d, name, w, n, k, dst, s);
}

// Whether rows of a typed matrix all start on a boundary of four values.
int mx_wide(const void* x, int dtype, int64_t ldx) {
  const int64_t four = 4 * (int64_t)mx_type_size(dtype);
  return (uintptr_t)x % four == 0 && ldx % 4 == 0;
}

// Whether rows of a typed output all start on 16-byte boundaries.
int mx_wide16(const void* y, int dtype, int64_t ldy) {
  return (uintptr_t)y % 16 == 0 && ldy * (int64_t)mx_type_size(dtype) % 16 == 0;
}

// Activation limits: a workgroup's rows are reached by 32-bit offsets (128 rows, five
// 32-row tiles of the planes where routed rows do not start on one: 514 MB of 2^21
// columns), and a grid has fewer than 2^31 units.
int mx_check_rows(int64_t m, int64_t k) {
  if (m > (1LL << 21) || k > (1LL << 21) || (m + kMxTile - 1) / kMxTile * mx_chunks(k) > (1LL << 30))
    return fail(QMM_ERR_INVALID, "activation of %lld x %lld is too large", (long long)m, (long long)k);
  return QMM_OK;
}

// A workspace of `need` bytes (0: none); its parts are read 16 bytes at a time.
int mx_check_ws(const void* ws, size_t bytes, size_t need) {
  if (need == 0) return QMM_OK;
  if (!ws || bytes < need) return fail(QMM_ERR_INVALID, "workspace of %zu B < %zu B needed", ws ? bytes : 0, need);
  if ((uintptr_t)ws % 16) return fail(QMM_ERR_INVALID, "workspaces must be 16-byte aligned");
  return QMM_OK;
}

int mx_here(const qmm_qtensor* w) {
  int dev = 0;
  QMM_HIP(hipGetDevice(&dev));
  if (dev != w->device) return fail(QMM_ERR_INVALID, "tensor lives on device %d, current device is %d", w->device, dev);
  return QMM_OK;
}

unsigned mx_plane_units(int64_t m, int64_t k) { return (unsigned)((m + kMxTile - 1) / kMxTile * mx_chunks(k)); }

// Planes of m rows: row i is row src[i] of x, or row i (src null).
int mx_quantize_x(Device* d, const void* x, int x_dtype, int64_t m, int64_t k, int64_t ldx, const int32_t* src,
                  uint8_t* planes, hipStream_t s) {
  char name[40];
  snprintf(name, sizeof(name), "qmm_mx_quantize_x_%s", mx_type_name(x_dtype));
  long long ld = ldx;
  int mm = (int)m, kk = (int)k, kc = (int)mx_chunks(k), wide = mx_wide(x, x_dtype, ldx);
  void* args[] = {&x, &ld, &mm, &kk, &kc, &wide, &src, &planes};
  return launch(d, name, mx_plane_units(m, k), 256, 0, s, args);
}

// The kernels' by-value argument (qmm::MxOut).
struct MxOut {
  const void* w;
  void* y;
  const void* bias;
  int y_type, bias_type, accumulate, wide;
};

// The product's tiles (kernels qmm_mx_gemm_<name>): rows, columns, threads, and the time
// of one on a CU at k = 4096, measured with every CU busy (us; two of the first run side
// by side, so it counts once for each).
struct MxTileCfg {
  const char* name;
  int rows, cols, threads;
  double us;
};
constexpr MxTileCfg kMxTiles[] = {{"128x256", 128, 256, 256, 41.0}, {"128x128", 128, 128, 256, 24.0}, {"64x128k4", 64, 128, 512, 13.4}};

// The tile with the least rounds x time: the wide ones do more per byte, the narrow one
// (which splits K over its waves) fills the chip with few rows or columns (333 x 4096 x
// 4096: 41.6, 27.7 and 14.2 us; 512 x 14336 x 4096: 48.9, 47.0 and 54.2).
const MxTileCfg& mx_tile_for(const Device* d, int64_t row_tiles64, int64_t row_tiles128, int64_t n) {
  const MxTileCfg* best = nullptr;
  double least = 0.0;
  for (const MxTileCfg& c : kMxTiles) {
    const int64_t tiles = (c.rows == 64 ? row_tiles64 : row_tiles128) * ((n + c.cols - 1) / c.cols);
    const double us = (double)((tiles + d->num_cu - 1) / d->num_cu) * c.us;
    if (!best || us < least) {
      best = &c;
      least = us;
    }
  }
  return *best;
}

// Unquantized rows of a product (qmm::MxRaw).
struct MxRaw {
  const void* x;
  long long ldx;
  const int32_t* src;
  int type, wide;
};

// Rows of the narrow kernels: of a tile, of unquantized rows.
constexpr int64_t kMxGemvRows = 16, kMxRawRows = 2;

// Dense rows that the narrow kernels take: one tile, or tiles of rows by 64 columns that
// are two a CU at most (128 rows x 4096 x 4096: 13.6 us against 17.8 by the wide ones, 32 x
// 4096 x 14336 22.4 against 40.1, 32 x 14336 x 4096 17.6 against 19.1; at 3.5 a CU, 64 x
// 14336 x 4096, 22.8 against 21.6).
bool mx_gemv_rows(const Device* d, int64_t m, int64_t n) {
  return m <= kMxGemvRows || ceil_div(m, kMxGemvRows) * (int64_t)ceil_div(n, 64) <= 2 * (int64_t)d->num_cu;
}
// Routed rows: one tile an expert or less (gate and up, and down: 512 rows over 64 experts
// of 2048 x 1408 43 and 23 us against 54 and 37, 1024 rows 48 and 30 against 56 and 38;
// 128 rows over 8 experts of 4096 x 14336 125 and 60 against 123 and 50).
bool mx_gemv_experts(int64_t pairs, int64_t active) { return pairs <= kMxGemvRows * active; }

// The narrow kernels' launch over `row_tiles` tiles of rows: a workgroup takes a group of
// `tiles` 16-column tiles (raw rows, which every workgroup quantizes for itself: as many
// groups as any other but one, 16 waves a CU in all). Four waves split K where that fills
// the chip with 16 waves a CU, else 8 or 16, at a chunk of 256 columns each at least; a
// wave has two chunks in flight (of one tile) where it has two.
struct MxGemv {
  int waves, tiles, depth;
  unsigned grid;
};
MxGemv mx_gemv_plan(const Device* d, int64_t n, int64_t k, int64_t row_tiles, int tiles, bool raw) {
  const int64_t kc = mx_chunks(k), fill = (int64_t)d->num_cu * 16, groups = ceil_div(n, 16 * tiles);
  MxGemv p;
  p.tiles = tiles;
  p.waves = 4;
  while (p.waves < 16 && p.waves < kc && groups * row_tiles * p.waves < fill) p.waves *= 2;
  p.depth = tiles == 1 && kc > p.waves ? 2 : 1;
  p.grid = (unsigned)groups;
  if (raw) {
    const int64_t want = std::max<int64_t>(fill / p.waves / row_tiles, 1), per = (groups + want - 1) / want;
    p.grid = (unsigned)((groups + per - 1) / per);
  }
  return p;
}
// Planes: four tiles a group, since every group reads the rows' digits (16 rows x 65536 x
// 4096: 32.3 us against 44.3; 24 tokens' down products over 64 experts of 2048 x 1408 18.5
// against 25.3), unless that leaves half of the chip idle with 16 waves a group (16 x 4096 x
// 4096: 10.3 us against 9.5).
MxGemv mx_planes_plan(const Device* d, int64_t n, int64_t k, int64_t row_tiles) {
  const bool wide = ceil_div(n, 64) * row_tiles * 32 >= (int64_t)d->num_cu * 16;
  return mx_gemv_plan(d, n, k, row_tiles, wide ? 4 : 1, false);
}
const char* mx_raw_name(const MxRaw* raw) { return !raw ? "" : raw->type == QMM_F32 ? "_raw32" : "_raw16"; }

// LDS of unquantized rows' digits, and the widest rows that take that way.
unsigned mx_raw_lds(int64_t k) { return (unsigned)(mx_chunks(k) * 1024); }
constexpr int64_t kMxRawCols = 16384;
bool mx_raw_fits(int64_t m, int64_t k) { return m <= kMxRawRows && k <= kMxRawCols; }

// y = x . W^T over m dense rows: of digit planes, or (up to two rows) of raw ones.
int mx_product(Device* d, const qmm_qtensor* w, const uint8_t* planes, const MxRaw* raw, int64_t m, MxOut o, int64_t ldy,
               hipStream_t s) {
  o.w = w->data;
  o.wide = mx_wide16(o.y, o.y_type, ldy);
  int mm = (int)m, n = (int)w->n, k = (int)w->k, ld = (int)ldy;
  hipFunction_t f;
  char name[40];
  if (mx_gemv_rows(d, m, n)) {
    MxRaw r = raw ? *raw : MxRaw();
    const MxGemv p = raw ? mx_gemv_plan(d, n, k, 1, 1, true) : mx_planes_plan(d, n, k, ceil_div(m, kMxGemvRows));
    snprintf(name, sizeof(name), "qmm_mx_gemv%s_w%d_n%d_u%d", mx_raw_name(raw), p.waves, p.tiles, p.depth);
    void* args[] = {&o, &mm, &n, &k, &planes, &r, &ld};
    QMM_TRY(kernel(d, name, &f));
    QMM_HIP(hipModuleLaunchKernel(f, p.grid, ceil_div(m, kMxGemvRows), 1, 64 * p.waves, 1, 1, raw ? mx_raw_lds(k) : 0, s, args, nullptr));
    return QMM_OK;
  }
  int kc = (int)mx_chunks(k);
  void* args[] = {&o, &mm, &n, &kc, &planes, &ld};
  const MxTileCfg& c = mx_tile_for(d, ceil_div(m, 64), ceil_div(m, 128), n);
  snprintf(name, sizeof(name), "qmm_mx_gemm_%s", c.name);
  QMM_TRY(kernel(d, name, &f));
  QMM_HIP(hipModuleLaunchKernel(f, ceil_div(n, c.cols), ceil_div(m, c.rows), 1, c.threads, 1, 1, 0, s, args, nullptr));
  return QMM_OK;
}

// The same of expert-ordered rows: expert e's are rows offsets[e] + i of the planes and
// of the output. One or two weights.
int mx_expert_product(Device* d, const qmm_qtensor* const* w, int count, int experts, const uint8_t* planes,
                      int64_t pairs, const int32_t* counts, const int32_t* offsets,
                      float* const* y, hipStream_t s) {
  MxOut o[2] = {};
  for (int j = 0; j < 2; ++j) {
    const int i = j < count ? j : 0;
    o[j].w = w[i]->data;
    o[j].y = y[i];
    o[j].wide = mx_wide16(y[i], QMM_F32, w[0]->n / experts);
  }
  int E = experts, P = (int)pairs, n = (int)(w[0]->n / experts), k = (int)w[0]->k, kc = (int)mx_chunks(k), ld = n;
  hipFunction_t f;
  const int64_t active = std::min<int64_t>(experts, pairs);
  char name[40];
  if (mx_gemv_experts(pairs, active)) {
    const int64_t tiles = pairs / kMxGemvRows + active;
    if (tiles > 65535) return fail(QMM_ERR_INVALID, "too many routed rows");
    const MxGemv p = mx_planes_plan(d, n, k, active * count);
    snprintf(name, sizeof(name), "qmm_mx_expert_gemv_w%d_n%d_u%d", p.waves, p.tiles, p.depth);
    void* args[] = {&o[0], &o[1], &E, &P, &n, &k, &counts, &offsets, &planes, &ld};
    QMM_TRY(kernel(d, name, &f));
    QMM_HIP(hipModuleLaunchKernel(f, p.grid, (unsigned)tiles, (unsigned)count, 64 * p.waves, 1, 1, 0, s, args, nullptr));
    return QMM_OK;
  }
  void* args[] = {&o[0], &o[1], &E, &P, &n, &kc, &counts, &offsets, &planes, &ld};
  // (the tiles that there will be, each expert's last one half full)
  const MxTileCfg& c = mx_tile_for(d, pairs / 64 + (active + 1) / 2, pairs / 128 + (active + 1) / 2, (int64_t)n * count);
  const int64_t tiles = pairs / c.rows + active;
  if (tiles > 65535) return fail(QMM_ERR_INVALID, "too many routed rows");
  snprintf(name, sizeof(name), "qmm_mx_expert_gemm_%s", c.name);
  QMM_TRY(kernel(d, name, &f));
  QMM_HIP(hipModuleLaunchKernel(f, ceil_div(n, c.cols), (unsigned)tiles, (unsigned)count, c.threads, 1, 1, 0, s, args, nullptr));
  return QMM_OK;
}

// silu(gate) * up of m rows as the digit planes of the down product's rows: dense rows
// (experts 0) or routed ones, of planes or (up to kMxRawRows an expert) raw.
int mx_glu(Device* d, const qmm_qtensor* gate, const qmm_qtensor* up, int experts, const uint8_t* planes,
           const MxRaw* raw, int64_t m, const int32_t* counts, const int32_t* offsets, uint8_t* out,
           hipStream_t s) {
  const int64_t F = gate->n / std::max(experts, 1), active = std::min<int64_t>(experts, m);
  MxOut o = {};
  o.w = gate->data;
  o.y = out;
  const void* uw = up->data;
  int E = experts, P = (int)m, n = (int)F, k = (int)gate->k, kc = (int)mx_chunks(k);
  hipFunction_t f;
  char name[40];
  const bool gemv = experts ? mx_gemv_experts(m, active) : mx_gemv_rows(d, m, 2 * F);
  const int64_t bm = gemv ? (raw ? kMxRawRows : kMxGemvRows) : 128;
  const int64_t tiles = experts ? m / bm + active : ceil_div(m, bm);
  if (tiles > 65535) return fail(QMM_ERR_INVALID, "too many rows");
  if (gemv) {
    MxRaw r = raw ? *raw : MxRaw();
    const MxGemv p = mx_gemv_plan(d, n, k, experts ? active : ceil_div(m, bm), 2, raw);
    snprintf(name, sizeof(name), "qmm_mx_glu_gemv%s_w%d", mx_raw_name(raw), p.waves);
    void* args[] = {&o, &uw, &E, &P, &n, &k, &counts, &offsets, &planes, &r};
    QMM_TRY(kernel(d, name, &f));
    QMM_HIP(hipModuleLaunchKernel(f, p.grid, (unsigned)tiles, 1, 64 * p.waves, 1, 1, raw ? mx_raw_lds(k) : 0, s, args,
                                  nullptr));
    return QMM_OK;
  }
  if (!experts) {
    void* args[] = {&o, &uw, &P, &n, &kc, &planes};
    QMM_TRY(kernel(d, "qmm_mx_glu_128x128", &f));
    QMM_HIP(hipModuleLaunchKernel(f, ceil_div(n, 128), (unsigned)tiles, 1, 256, 1, 1, 0, s, args, nullptr));
    return QMM_OK;
  }
  void* args[] = {&o, &uw, &E, &P, &n, &kc, &counts, &offsets, &planes};
  QMM_TRY(kernel(d, "qmm_mx_expert_glu_128x128", &f));
  QMM_HIP(hipModuleLaunchKernel(f, ceil_div(n, 128), (unsigned)tiles, 1, 256, 1, 1, 0, s, args, nullptr));
  return QMM_OK;
}

// How a call routes its tokens.
struct Routing {
  bool scored = false;  // qmm_moe_route_scored's rules; else qmm_moe_route_ex's
  int score = 0, groups = 1, topk_groups = 1, group_top = 1;
  const float* bias = nullptr;
  int renormalize = 1;
  float scale = 1.0f;
};

struct RouteArgs {  // the kernels' by-value argument (qmm::RouteArgs)
  int T, E, k, sigmoid, groups, topk_groups, group_top, renorm;
  float scale;
};

constexpr int kRouteMaxTokens = 65536, kRouteMaxExperts = 1024, kRouteMaxTopk = 32, kRouteSmall = 16;

int check_routing(int64_t tokens, int experts, int topk, const Routing& r) {
  if (tokens < 1 || tokens > kRouteMaxTokens || experts < 1 || experts > kRouteMaxExperts || topk < 1 ||
      topk > kRouteMaxTopk || topk > experts)
    return fail(QMM_ERR_INVALID, "routing limits: 1 <= tokens <= %d, 1 <= experts <= %d, 1 <= topk <= min(%d, experts)",
                kRouteMaxTokens, kRouteMaxExperts, kRouteMaxTopk);
  if (r.score != QMM_SCORE_SOFTMAX && r.score != QMM_SCORE_SIGMOID)
    return fail(QMM_ERR_INVALID, "routing score %d (softmax = 0, sigmoid = 1)", r.score);
  if (r.groups < 1 || r.groups > 64 || experts % r.groups || r.topk_groups < 1 || r.topk_groups > r.groups)
    return fail(QMM_ERR_INVALID, "routing groups: 1 <= topk_groups <= groups <= 64, experts %% groups == 0");
  if (r.group_top < 1 || r.group_top > 2 || r.group_top > experts / r.groups)
    return fail(QMM_ERR_INVALID, "a group's score is the sum of its 1 or 2 best experts (group_top %d, groups of %d)",
                r.group_top, experts / r.groups);
  if (topk > r.topk_groups * (experts / r.groups))
    return fail(QMM_ERR_INVALID, "topk %d experts out of %d groups of %d", topk, r.topk_groups, experts / r.groups);
  if (!(r.scale == r.scale)) return fail(QMM_ERR_INVALID, "routed scaling factor is NaN");
  return QMM_OK;
}

// Registers of 64 experts that a wave holds.
int route_regs(int experts) { return experts <= 64 ? 1 : experts <= 128 ? 2 : experts <= 256 ? 4 : 16; }
// One launch on one CU (16 tokens of up to 64 experts, 8 of 128, 4 of 256), or the
// selections on all and then the lists: 16 tokens of 64 experts 7.9 us against 7.5, 8 of
// 128 7.6 against 8.8, 16 of 128 10.1 against 8.8, 4 of 256 9.0 against 10.5, 16 of 256
// 12.9 against 10.5.
bool route_is_small(int64_t tokens, int experts) {
  return experts <= 256 && tokens * route_regs(experts) <= kRouteSmall;
}

size_t route_scratch(int64_t tokens, int experts, int topk) {
  if (route_is_small(tokens, experts)) return 0;
  return mx_align((size_t)tokens * topk * 2) + mx_align((size_t)tokens * topk * 4);
}

int route_scored(Device* d, const float* logits, int64_t tokens, int experts, int topk, const Routing& r,
                 int32_t* counts, int32_t* offsets, int32_t* pair_token, float* pair_weight, int32_t* token_pairs,
                 uint8_t* ws, hipStream_t s) {
  RouteArgs a = {(int)tokens, experts, topk, r.score == QMM_SCORE_SIGMOID, r.groups, r.topk_groups, r.group_top,
                 r.renormalize ? 1 : 0, r.scale};
  const float* bias = r.bias;
  const int R = route_regs(experts);
  char name[32];
  // a wave a token; one workgroup also makes the lists
  if (route_is_small(tokens, experts)) {
    snprintf(name, sizeof(name), "qmm_route_small_r%d", R);
    void* args[] = {&logits, &bias, &a, &counts, &offsets, &pair_token, &pair_weight, &token_pairs};
    return launch(d, name, 1, 1024, 0, s, args);
  }
  void* ids = ws;
  void* wts = ws + mx_align((size_t)tokens * topk * 2);
  snprintf(name, sizeof(name), "qmm_route_tokens_r%d", R);
  void* a1[] = {&logits, &bias, &a, &ids, &wts};
  QMM_TRY(launch(d, name, ceil_div(tokens, 4), 256, 0, s, a1));
  void* a2[] = {&a, &ids, &wts, &counts, &offsets, &pair_token, &pair_weight, &token_pairs};
  return launch(d, "qmm_route_lists", experts, 1024, 0, s, a2);
}

}  // namespace
