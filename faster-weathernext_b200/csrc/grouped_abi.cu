// C ABI of the products grouped by expert (include/fwn_attn.h): argument checks, plans, tensor maps and launches.
#include <algorithm>
#include <cstring>

#include "abi.cuh"
#include "grouped.cuh"
#include "rms.cuh"

using namespace fwn;

namespace {

int64_t round_up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
size_t take(size_t& at, int64_t bytes) {  // the next `bytes` of a workspace
  const size_t here = at;
  at += static_cast<size_t>(round_up(bytes, 256));
  return here;
}

fwn_status check_grouped(const fwn_grouped_desc* d) {
  if (!d) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "desc is null");
  if (d->m < 0 || d->n <= 0 || d->k <= 0 || d->groups <= 0)
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bad shape m=%lld n=%d k=%d groups=%d", static_cast<long long>(d->m), d->n, d->k, d->groups);
  if (d->groups > kGroupsMax) return abi_fail(FWN_ERR_UNSUPPORTED, "groups=%d exceeds %d", d->groups, kGroupsMax);
  if (d->m > INT32_MAX - 1024) return abi_fail(FWN_ERR_UNSUPPORTED, "m=%lld too large", static_cast<long long>(d->m));
  if (d->n > (1 << 20) || d->k > (1 << 20)) return abi_fail(FWN_ERR_UNSUPPORTED, "n=%d or k=%d exceeds 2^20", d->n, d->k);
  if (!abi_float(d->out_dtype) || !abi_float(d->bias_dtype) || !abi_float(d->x_dtype))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "out, bias and dy are bf16 or float32");
  if (d->act != FWN_ACT_NONE && d->act != FWN_ACT_GELU_TANH && d->act != FWN_ACT_SWISH)
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "unknown activation %d", d->act);
  if (d->flags & ~FWN_LINEAR_B_N_CONTIGUOUS) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "unknown flags %d", d->flags);
  const bool b_mn = d->flags & FWN_LINEAR_B_N_CONTIGUOUS;
  const int64_t inner = b_mn ? d->n : d->k, outer = b_mn ? d->k : d->n;
  if ((d->m > 1 && d->lda < d->k) || (outer > 1 && d->ldb < inner) ||
      (d->groups > 1 && d->b_stride < inner))
    return abi_fail(FWN_ERR_INVALID_ARGUMENT, "a stride is below what it strides over");
  return FWN_OK;
}

bool tma_rows(const void* p, int64_t es, int64_t outer, int64_t ld) { return abi_aligned(p, 16) && (outer <= 1 || ld * es % 16 == 0); }
fwn_status check_operands(const fwn_grouped_desc& d, const void* a, const void* b) {
  const int64_t outer = d.flags & FWN_LINEAR_B_N_CONTIGUOUS ? d.k : d.n;
  if (!tma_rows(a, 2, d.m, d.lda) || !tma_rows(b, 2, outer, d.ldb) || (d.groups > 1 && d.b_stride % 8 != 0))
    return abi_fail(FWN_ERR_UNSUPPORTED, "rows of a and b start and stride by multiples of 16 bytes (fwn_linear_pack lays out others)");
  return FWN_OK;
}

fwn_status rows_map(CUtensorMap* map, const void* p, int32_t dtype, int64_t cols, int64_t rows, int64_t ld, int box_bytes, int box_rows) {
  const int64_t dims[2] = {cols, rows}, strides[1] = {rows > 1 ? ld : round_up(cols, 16 / abi_size(dtype))};
  return abi_map(map, p, dtype, 2, dims, strides, box_bytes, box_rows);
}
// Weights [groups, outer, inner].
fwn_status weight_map(CUtensorMap* map, const void* p, int64_t inner, int64_t outer, int64_t ld, int64_t groups, int64_t stride, int box_rows) {
  const int64_t row = outer > 1 ? ld : round_up(inner, 8), dims[3] = {inner, outer, groups},
                strides[2] = {row, groups > 1 ? stride : outer * row};
  return abi_map(map, p, FWN_DTYPE_BF16, 3, dims, strides, 128, box_rows);
}

int64_t tiles_most(int64_t m, int groups, int64_t unit) { return m / unit + std::min<int64_t>(m, groups); }

// The same choice between the forms of the 256 x 256 tile as the projections' (sixteen epilogue warps and four stages, or
// eight and five), by the length of k and what the epilogue does.
int pair_form(int64_t kb, int32_t act, bool pre, bool direct) {
  const bool many = pre || direct ? kb >= 20 : act != FWN_ACT_NONE ? kb >= 10 : true;
  return many ? kTile256Long : kTile256;
}
constexpr int kStageCost[kLinearTiles] = {55, 47, 31, 28}, kEpilogueCost[kLinearTiles] = {150, 200, 120, 100};  // 0.01 us

// The tile of a product of rows: the projections' time model (a stage of k, an epilogue that overlaps the next tile), with
// half a tile more for each expert that can have rows: their last tiles are on average half empty.
int plan_rows(int64_t m, int64_t n, int64_t k, int groups, int32_t act, bool pre, bool direct, int sms) {
  const int64_t kb = (k + 63) / 64, hit = std::min<int64_t>(groups, m);
  const int form = pair_form(kb, act, pre, direct);
  int best_tile = kTile64;
  int64_t best = INT64_MAX;
  for (int t = 0; t < kLinearTiles; ++t) {
    if (linear_pair(t) && t != form) continue;
    const int64_t tm = linear_tile_m(t), tn = linear_tile_n(t), slots = linear_pair(t) ? sms / 2 : sms;
    const int64_t tiles = std::max(hit, (2 * m + hit * tm) / (2 * tm)) * ((n + tn - 1) / tn);
    const int64_t waves = (tiles + slots - 1) / slots;
    const int64_t cost = waves * std::max<int64_t>(kb * kStageCost[t], kEpilogueCost[t]) + kEpilogueCost[t];
    if (cost < best) {
      best = cost;
      best_tile = t;
    }
  }
  return best_tile;
}

// The weights' gradient: out [rows, cols] of each expert, its rows summed over whole (run 0) or in equal runs of at most
// `run` stages, which balance experts of different sizes and fill the SMs where experts and tiles are few, at the cost of a
// float32 part for each run, written and added through L2. The sizes are on the device: the choice goes by their mean, and
// experts at once lose where one is far above it, whose tiles run on as many SMs as they are (81,924 x 512 x 2,048: even experts
// 8 in runs 133 + 17 us, 64 at once 137; half of the rows one expert's: 153 + 14 and 271; nine tenths: 132 + 19 and 378).
struct WeightPlan {
  int tile, run;     // run: stages of 64 rows at most; 0: an expert's rows at once
  int64_t most;      // runs (or experts)
};
constexpr int64_t kMaxStages = 1 << 20;  // of a run: a tile's epilogue waits for it, within the limit of its waits
WeightPlan plan_weights(int64_t m, int64_t rows, int64_t cols, int groups, int sms) {
  WeightPlan pl{};
  const int64_t hit = std::min<int64_t>(groups, m), all = (m + 63) / 64 + hit / 2;
  int64_t best = INT64_MAX;
  for (int t = kTile256Long; t < kLinearTiles; ++t) {
    const int64_t slots = linear_pair(t) ? sms / 2 : sms;
    const int64_t tiles = ((rows + linear_tile_m(t) - 1) / linear_tile_m(t)) * ((cols + linear_tile_n(t) - 1) / linear_tile_n(t));
    // Whole: the walk deals experts' tiles of uneven length round: one tile more than the mean.
    if ((m + 63) / 64 <= kMaxStages) {
      const int64_t mean = std::max<int64_t>(1, all / hit);
      const int64_t cost = (tiles * groups * std::max<int64_t>(mean * kStageCost[t], kEpilogueCost[t])) / slots + 2 * mean * kStageCost[t] + kEpilogueCost[t];
      if (cost < best) {
        best = cost;
        pl = {t, 0, groups};
      }
    }
    for (int64_t want = 1; want <= 256; want += want < 16 ? 1 : want / 8) {
      const int64_t run = (all + want - 1) / want;
      if (run > kMaxStages || (run < 4 && want > 1)) continue;
      const int64_t runs = all / run + hit / 2 + 1;
      const int64_t waves = (runs * tiles + slots - 1) / slots;
      const int64_t cost = waves * std::max<int64_t>(run * kStageCost[t], kEpilogueCost[t]) + kEpilogueCost[t] + 430 +
                           static_cast<int64_t>(8.0 * runs * rows * cols / 2.5e4);
      if (cost < best) {
        best = cost;
        pl = {t, static_cast<int>(run), tiles_most(m, groups, run * 64)};
      }
    }
  }
  return pl;
}

fwn_status check_items(int64_t items) {
  if (items > INT32_MAX - 1024) return abi_fail(FWN_ERR_UNSUPPORTED, "too many tiles (%lld)", static_cast<long long>(items));
  return FWN_OK;
}

struct ForwardPlan {
  bool rows;                 // few rows
  int tile;
  size_t offsets, first, maps, bytes;
};
ForwardPlan plan_forward(const fwn_grouped_desc& d, bool out_tma, int sms) {
  ForwardPlan pl{};
  pl.rows = d.m <= kLinearRowsMax && !(d.flags & FWN_LINEAR_B_N_CONTIGUOUS);
  if (pl.rows) return pl;
  pl.tile = plan_rows(d.m, d.n, d.k, d.groups, d.act, false, !out_tma, sms);
  pl.maps = take(pl.bytes, 2ll * d.groups * sizeof(CUtensorMap));
  pl.offsets = take(pl.bytes, 4ll * (d.groups + 1));
  pl.first = take(pl.bytes, 4ll * (d.groups + 1));
  return pl;
}

struct BackwardPlan {
  bool cast;                 // d_pre is written (an activation, or dy is not bf16 rows that TMA can address)
  int64_t ldp;               // its row stride
  int pre_tile, a_tile;
  WeightPlan w;
  bool turned;               // d_b is [k, n] of each expert
  int64_t w_rows, w_cols;
  size_t d_pre, maps, offsets, first[kGroupFirsts], part_sum, part_w, bytes;
};
BackwardPlan plan_backward(const fwn_grouped_desc& d, const void* dy, int sms) {
  BackwardPlan pl{};
  const bool act = d.act != FWN_ACT_NONE;
  pl.cast = act || d.x_dtype != FWN_DTYPE_BF16 || !tma_rows(dy, 2, d.m, d.ldx);
  pl.ldp = pl.cast ? round_up(d.n, 8) : d.ldx;
  pl.pre_tile = plan_rows(d.m, d.n, d.k, d.groups, d.act, true, false, sms);
  pl.a_tile = plan_rows(d.m, d.k, d.n, d.groups, FWN_ACT_NONE, false, d.k % 8 != 0, sms);
  pl.turned = d.flags & FWN_LINEAR_B_N_CONTIGUOUS;
  pl.w_rows = pl.turned ? d.k : d.n;
  pl.w_cols = pl.turned ? d.n : d.k;
  pl.w = plan_weights(d.m, pl.w_rows, pl.w_cols, d.groups, sms);
  if (pl.cast) pl.d_pre = take(pl.bytes, d.m * pl.ldp * 2);
  pl.maps = take(pl.bytes, static_cast<int64_t>(kGroupMaps) * d.groups * sizeof(CUtensorMap));
  pl.offsets = take(pl.bytes, 4ll * (d.groups + 1));
  for (auto& f : pl.first) f = take(pl.bytes, 4ll * (d.groups + 1));
  // The sums' parts and, after them on the stream, the weights' share a place.
  const int64_t unit = act ? linear_tile_m(pl.pre_tile) : kCastRows, per = act ? unit / 32 : 1;
  const int64_t sums = tiles_most(d.m, d.groups, unit) * per * d.n * 4;
  const int64_t parts = pl.w.run > 0 ? pl.w.most * pl.w_rows * round_up(pl.w_cols, 4) * 4 : 0;
  pl.part_sum = pl.part_w = take(pl.bytes, std::max(sums, parts));
  return pl;
}

LinearParams params_of(const fwn_grouped_desc& d) {
  LinearParams p{};
  p.m = d.m;
  p.n = d.n;
  p.k = d.k;
  p.act = d.act == FWN_ACT_GELU_TANH ? 1 : d.act == FWN_ACT_SWISH ? 2 : 0;
  p.bias_bf16 = d.bias_dtype == FWN_DTYPE_BF16;
  p.x_f32 = d.x_dtype == FWN_DTYPE_F32;
  p.out_f32 = d.out_dtype == FWN_DTYPE_F32;
  p.splits = 1;
  p.k_blocks = (d.k + 63) / 64;
  p.chunk = p.k_blocks;
  return p;
}

}  // namespace

extern "C" {

fwn_status fwn_linear_grouped_workspace_size(const fwn_grouped_desc* desc, size_t* bytes) {
  if (!bytes) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bytes is null");
  if (fwn_status s = check_grouped(desc); s != FWN_OK) return s;
  *bytes = desc->m == 0 ? 0 : plan_forward(*desc, true, abi_sms()).bytes;
  return abi_ok();
}

fwn_status fwn_linear_grouped(const fwn_grouped_desc* desc, const void* a, const void* b, const void* bias,
                              const int32_t* offsets, void* out, void* workspace, size_t workspace_bytes, void* stream) {
  fwn_status s = check_grouped(desc);
  if (s != FWN_OK) return s;
  const fwn_grouped_desc& d = *desc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (d.m == 0) return abi_ok();
  if (!a || !b || !offsets || !out) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  const int64_t es = abi_size(d.out_dtype);
  if ((s = abi_elements({{a, 2}, {b, 2}, {bias, abi_size(d.bias_dtype)}, {offsets, 4}, {out, es}})) != FWN_OK) return s;
  const int sms = abi_sms();
  const bool out_tma = tma_rows(out, es, d.m, d.n);
  const ForwardPlan pl = plan_forward(d, out_tma, sms);
  LinearParams p = params_of(d);
  p.bias = bias;
  p.out = out;
  p.ldo = d.n;
  p.b_mn = d.flags & FWN_LINEAR_B_N_CONTIGUOUS;
  cudaError_t e;
  if (pl.rows) {
    const bool wide = d.k % 8 == 0 && tma_rows(a, 2, d.m, d.lda) && tma_rows(b, 2, d.n, d.ldb) && (d.groups == 1 || d.b_stride % 8 == 0);
    if ((e = launch_grouped_rows(a, d.lda, b, d.ldb, d.b_stride, wide, offsets, d.groups, p, st)) != cudaSuccess)
      return abi_cuda_fail(e, "grouped rows");
    return abi_ok();
  }
  if ((s = check_operands(d, a, b)) != FWN_OK) return s;
  if (!workspace || workspace_bytes < pl.bytes || !abi_aligned(workspace, 256))
    return abi_fail(FWN_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) needed", pl.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int tm = linear_tile_m(pl.tile), tn = linear_tile_n(pl.tile);
  p.n_tiles = (d.n + tn - 1) / tn;
  if (p.out_f32) p.chunk = kLinearChunk;
  p.out_direct = !out_tma;
  const int64_t items = tiles_most(d.m, d.groups, tm) * p.n_tiles;
  if ((s = check_items(items)) != FWN_OK) return s;
  GroupMaps maps;
  CUtensorMap tb;
  const int cols = linear_chunk_cols(pl.tile, p.out_f32);
  if ((s = rows_map(&maps.map[0], a, FWN_DTYPE_BF16, d.k, d.m, d.lda, 128, 128)) != FWN_OK) return s;
  maps.map[1] = maps.map[0];
  if (!p.out_direct && (s = rows_map(&maps.map[1], out, d.out_dtype, d.n, d.m, d.n, cols * static_cast<int>(es), 32)) != FWN_OK) return s;
  s = p.b_mn ? weight_map(&tb, b, d.n, d.k, d.ldb, d.groups, d.b_stride, 64)
             : weight_map(&tb, b, d.k, d.n, d.ldb, d.groups, d.b_stride, linear_box_n(pl.tile));
  if (s != FWN_OK) return s;
  GroupSetup g{};
  g.given = offsets;
  g.groups = d.groups;
  g.m = d.m;
  g.offsets = reinterpret_cast<int32_t*>(ws + pl.offsets);
  g.first[0] = reinterpret_cast<int32_t*>(ws + pl.first);
  g.unit[0] = tm;
  g.maps = reinterpret_cast<CUtensorMap*>(ws + pl.maps);
  g.n_maps = p.out_direct ? 1 : 2;
  g.clear = out;
  g.clear_row = d.n * es;
  if ((e = launch_group_setup(g, maps, st)) != cudaSuccess) return abi_cuda_fail(e, "experts' maps");
  GroupParams gp{};
  gp.offsets = g.offsets;
  gp.first = g.first[0];
  gp.map_a = g.maps;
  gp.map_o = g.maps + d.groups;
  gp.groups = d.groups;
  if ((e = launch_grouped_forward(pl.tile, tb, p, gp, items, sms, st)) != cudaSuccess) return abi_cuda_fail(e, "grouped product");
  return abi_ok();
}

fwn_status fwn_linear_grouped_bwd_workspace_size(const fwn_grouped_desc* desc, const void* dy, size_t* bytes) {
  if (!bytes) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "bytes is null");
  if (fwn_status s = check_grouped(desc); s != FWN_OK) return s;
  *bytes = desc->m == 0 ? 0 : plan_backward(*desc, dy, abi_sms()).bytes;
  return abi_ok();
}

fwn_status fwn_linear_grouped_bwd(const fwn_grouped_desc* desc, const void* a, const void* b, const void* bias,
                                  const int32_t* offsets, const void* dy, void* d_a, void* d_b, void* d_bias, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  fwn_status s = check_grouped(desc);
  if (s != FWN_OK) return s;
  const fwn_grouped_desc& d = *desc;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t bs = abi_size(d.bias_dtype), xs = abi_size(d.x_dtype);
  if (d_bias && !bias) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "d_bias needs the bias");
  if ((s = abi_elements({{a, 2}, {b, 2}, {d_a, 2}, {d_b, 2}, {dy, xs}, {bias, bs}, {d_bias, bs}, {offsets, 4}})) != FWN_OK) return s;
  cudaError_t e = cudaSuccess;
  if (d.m == 0) {
    if (d_b) e = cudaMemsetAsync(d_b, 0, static_cast<size_t>(d.groups) * d.n * d.k * 2, st);
    if (e == cudaSuccess && d_bias) e = cudaMemsetAsync(d_bias, 0, static_cast<size_t>(d.groups) * d.n * bs, st);
    if (e != cudaSuccess) return abi_cuda_fail(e, "clear the gradients");
    return abi_ok();
  }
  if (!a || !b || !dy || !offsets) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "null pointer");
  if (d.m > 1 && d.ldx < d.n) return abi_fail(FWN_ERR_INVALID_ARGUMENT, "ldx is below n");
  if ((s = check_operands(d, a, b)) != FWN_OK) return s;
  const int sms = abi_sms();
  const BackwardPlan pl = plan_backward(d, dy, sms);
  if (!workspace || workspace_bytes < pl.bytes || !abi_aligned(workspace, 256))
    return abi_fail(FWN_ERR_WORKSPACE, "workspace of %zu bytes (256-byte aligned) needed", pl.bytes);
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const bool act = d.act != FWN_ACT_NONE, b_mn = d.flags & FWN_LINEAR_B_N_CONTIGUOUS;
  const void* d_pre = pl.cast ? ws + pl.d_pre : dy;

  // Maps: 0 a, 1 dy, 2 d_pre (stored) for the gradient of the pre-activation; 3 d_pre, 4 d_a; 5 d_pre, 6 a summed over rows.
  GroupMaps maps;
  const bool x_tma = tma_rows(dy, xs, d.m, d.ldx), da_tma = tma_rows(d_a, 2, d.m, d.k);
  const int pre_cols = linear_chunk_cols(pl.pre_tile, d.x_dtype == FWN_DTYPE_F32), a_cols = linear_chunk_cols(pl.a_tile, false);
  if ((s = rows_map(&maps.map[0], a, FWN_DTYPE_BF16, d.k, d.m, d.lda, 128, 128)) != FWN_OK) return s;
  for (int i = 1; i < kGroupMaps; ++i) maps.map[i] = maps.map[0];
  if (act) {
    if (x_tma && (s = rows_map(&maps.map[1], dy, d.x_dtype, d.n, d.m, d.ldx, pre_cols * static_cast<int>(xs), 32)) != FWN_OK) return s;
    if ((s = rows_map(&maps.map[2], d_pre, FWN_DTYPE_BF16, d.n, d.m, pl.ldp, pre_cols * 2, 32)) != FWN_OK) return s;
  }
  if (d_a) {
    if ((s = rows_map(&maps.map[3], d_pre, FWN_DTYPE_BF16, d.n, d.m, pl.ldp, 128, 128)) != FWN_OK) return s;
    if (da_tma && (s = rows_map(&maps.map[4], d_a, FWN_DTYPE_BF16, d.k, d.m, d.k, a_cols * 2, 32)) != FWN_OK) return s;
  }
  if (d_b) {
    if ((s = rows_map(&maps.map[5], d_pre, FWN_DTYPE_BF16, d.n, d.m, pl.ldp, 128, 64)) != FWN_OK) return s;
    if ((s = rows_map(&maps.map[6], a, FWN_DTYPE_BF16, d.k, d.m, d.lda, 128, 64)) != FWN_OK) return s;
  }
  GroupSetup g{};
  g.given = offsets;
  g.groups = d.groups;
  g.m = d.m;
  g.offsets = reinterpret_cast<int32_t*>(ws + pl.offsets);
  for (int i = 0; i < kGroupFirsts; ++i) g.first[i] = reinterpret_cast<int32_t*>(ws + pl.first[i]);
  g.unit[0] = act ? linear_tile_m(pl.pre_tile) : kCastRows;
  g.unit[1] = linear_tile_m(pl.a_tile);
  g.unit[2] = pl.w.run * 64;
  g.maps = reinterpret_cast<CUtensorMap*>(ws + pl.maps);
  g.n_maps = kGroupMaps;
  g.clear = d_a;
  g.clear_row = 2ll * d.k;
  if ((e = launch_group_setup(g, maps, st)) != cudaSuccess) return abi_cuda_fail(e, "experts' maps");
  auto map_of = [&](int i) { return g.maps + static_cast<int64_t>(i) * d.groups; };
  GroupParams gp{};
  gp.offsets = g.offsets;
  gp.groups = d.groups;

  float* part_sum = d_bias ? reinterpret_cast<float*>(ws + pl.part_sum) : nullptr;
  gp.first = g.first[0];
  if (act) {
    LinearParams p = params_of(d);
    p.bias = bias;
    p.x = dy;
    p.ldx = d.ldx;
    p.x_direct = !x_tma;
    p.out = ws + pl.d_pre;
    p.ldo = pl.ldp;
    p.out_f32 = false;
    p.pre_grad = true;
    p.b_mn = b_mn;
    p.colsum = part_sum;
    p.n_tiles = (d.n + linear_tile_n(pl.pre_tile) - 1) / linear_tile_n(pl.pre_tile);
    if (d_bias && !p.bias_bf16) p.chunk = kLinearChunk;
    const int64_t items = tiles_most(d.m, d.groups, g.unit[0]) * p.n_tiles;
    if ((s = check_items(items)) != FWN_OK) return s;
    CUtensorMap tb;
    s = b_mn ? weight_map(&tb, b, d.n, d.k, d.ldb, d.groups, d.b_stride, 64)
             : weight_map(&tb, b, d.k, d.n, d.ldb, d.groups, d.b_stride, linear_box_n(pl.pre_tile));
    if (s != FWN_OK) return s;
    gp.map_a = map_of(0);
    gp.map_x = map_of(1);
    gp.map_o = map_of(2);
    if ((e = launch_grouped_pre_grad(pl.pre_tile, tb, p, gp, items, sms, st)) != cudaSuccess) return abi_cuda_fail(e, "grouped act'");
  } else if (pl.cast || d_bias) {
    const bool wide = d.n % 8 == 0 && x_tma;
    if ((e = launch_grouped_cast(dy, d.x_dtype == FWN_DTYPE_F32, d.ldx, d.n, pl.cast ? ws + pl.d_pre : nullptr, pl.ldp, part_sum, gp,
                                 tiles_most(d.m, d.groups, kCastRows), wide, st)) != cudaSuccess)
      return abi_cuda_fail(e, "grouped cast");
  }
  if (d_bias && (e = launch_grouped_column_sum(part_sum, gp.first, d.groups, tiles_most(d.m, d.groups, g.unit[0]),
                                               act ? g.unit[0] / 32 : 1, d.n, d_bias, d.bias_dtype == FWN_DTYPE_BF16, st)) != cudaSuccess)
    return abi_cuda_fail(e, "grouped column sums");

  if (d_a) {
    LinearParams p = params_of(d);
    p.act = 0;
    p.n = d.k;
    p.k = d.n;
    p.out = d_a;
    p.ldo = d.k;
    p.out_f32 = false;
    p.out_direct = !da_tma;
    p.b_mn = !b_mn;
    p.k_blocks = p.chunk = (d.n + 63) / 64;
    p.n_tiles = (d.k + linear_tile_n(pl.a_tile) - 1) / linear_tile_n(pl.a_tile);
    const int64_t items = tiles_most(d.m, d.groups, g.unit[1]) * p.n_tiles;
    if ((s = check_items(items)) != FWN_OK) return s;
    CUtensorMap tb;
    s = p.b_mn ? weight_map(&tb, b, d.k, d.n, d.ldb, d.groups, d.b_stride, 64)
               : weight_map(&tb, b, d.n, d.k, d.ldb, d.groups, d.b_stride, linear_box_n(pl.a_tile));
    if (s != FWN_OK) return s;
    gp.first = g.first[1];
    gp.map_a = map_of(3);
    gp.map_o = map_of(4);
    if ((e = launch_grouped_forward(pl.a_tile, tb, p, gp, items, sms, st)) != cudaSuccess) return abi_cuda_fail(e, "grouped d_a");
  }

  if (d_b) {
    const bool runs = pl.w.run > 0;
    const int64_t ldp = round_up(pl.w_cols, 4);
    LinearParams p = params_of(d);
    p.act = 0;
    p.m = pl.w_rows;
    p.n = static_cast<int>(pl.w_cols);
    p.a_mn = p.b_mn = true;
    p.out = runs ? static_cast<void*>(ws + pl.part_w) : d_b;
    p.ldo = runs ? ldp : pl.w_cols;
    p.out_f32 = runs;
    p.out_direct = !runs && !(tma_rows(d_b, 2, 2, pl.w_cols));
    p.m_tiles = static_cast<int>((pl.w_rows + linear_tile_m(pl.w.tile) - 1) / linear_tile_m(pl.w.tile));
    p.n_tiles = static_cast<int>((pl.w_cols + linear_tile_n(pl.w.tile) - 1) / linear_tile_n(pl.w.tile));
    const int64_t items = pl.w.most * p.m_tiles * p.n_tiles;
    if ((s = check_items(items)) != FWN_OK) return s;
    CUtensorMap to = maps.map[0];
    if (!p.out_direct) {
      const int64_t es = runs ? 4 : 2, dims[3] = {pl.w_cols, pl.w_rows, pl.w.most}, strides[2] = {p.ldo, pl.w_rows * p.ldo};
      s = abi_map(&to, p.out, runs ? FWN_DTYPE_F32 : FWN_DTYPE_BF16, 3, dims, strides,
                  linear_chunk_cols(pl.w.tile, runs) * static_cast<int>(es), 32);
      if (s != FWN_OK) return s;
    }
    gp.first = g.first[2];
    gp.map_a = map_of(pl.turned ? 6 : 5);
    gp.map_b = map_of(pl.turned ? 5 : 6);
    gp.by_run = runs;
    if ((e = launch_grouped_weights(pl.w.tile, to, p, gp, items, sms, st)) != cudaSuccess) return abi_cuda_fail(e, "grouped d_b");
    if (runs && (e = launch_grouped_run_sum(reinterpret_cast<float*>(ws + pl.part_w), gp.first, d.groups, pl.w_rows,
                                            static_cast<int>(pl.w_cols), ldp, d_b, st)) != cudaSuccess)
      return abi_cuda_fail(e, "grouped run sums");
  }
  return abi_ok();
}

}  // extern "C"
