// fa2_latent.hip - C ABI and launch logic of latent attention and of attention for
// trees of drafts (declared in include/fa2_latent.h).
#include "fa2_latent.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "fa2_host.h"
#include "fa2_kernel_rows.h"
#include "fa2_kernel_rows16.h"
#include "fa2_latent_append.h"

namespace fa2 {
namespace {

constexpr int64_t kLim = INT32_MAX / 2;  // 32-bit counters inside the kernels
// Workgroups of 256 threads in a grid row: its threads are counted in 32 bits.
constexpr int64_t kMaxGrid = (int64_t(1) << 24) - 1;

int launched() { return hipGetLastError() == hipSuccess ? FA2_OK : FA2_ERR_HIP; }

bool latent_dims_ok(int64_t latent, int64_t rope) {
  return (latent == 256 || latent == 512) && rope == kLaRope;
}

bool half_type(int32_t dtype) { return dtype == FA2_DTYPE_F16 || dtype == FA2_DTYPE_BF16; }

// ---- the writer ----------------------------------------------------------------

// Rows of a workgroup.
int64_t append_rows(int64_t latent) { return kLaThreads / 64 * (latent == 512 ? 1 : 2); }

int validate_append(const fa2_latent_append_params* p) {
  if (!p) return FA2_ERR_NULL_POINTER;
  if (!half_type(p->dtype)) return FA2_ERR_BAD_DTYPE;
  if (p->weight_dtype != p->dtype && p->weight_dtype != FA2_DTYPE_F32) return FA2_ERR_BAD_DTYPE;
  if (!latent_dims_ok(p->latent_dim, p->rope_dim)) return FA2_ERR_HEAD_DIM;
  if (p->batch < 0 || p->num_rows < 0 || p->page_size <= 0 || p->num_pages < 0 ||
      p->table_width < 0 || p->table_stride < 0 || p->positions < 0 || p->rope_stride < 0 ||
      p->x_ts < 0 || !(p->eps >= 0.f))
    return FA2_ERR_BAD_SHAPE;
  if (p->batch > kLim || p->num_rows > kLim || p->page_size > kLim || p->num_pages > kLim ||
      p->table_width > kLim || p->positions > kLim)
    return FA2_ERR_TOO_LARGE;
  if (cdiv(p->num_rows, append_rows(p->latent_dim)) > kMaxGrid) return FA2_ERR_TOO_LARGE;
  if (!stride_ok(p->x_ts, 2) || p->rope_stride % 4) return FA2_ERR_ALIGNMENT;
  return FA2_OK;
}

template <int DT>
void launch_append(int64_t latent, const LatentAppendArgs& a, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(cdiv(a.num_rows, append_rows(latent)))), block(kLaThreads);
  if (latent == 512)
    hipLaunchKernelGGL((fa2_latent_append_kernel<DT, 512>), grid, block, 0, st, a);
  else
    hipLaunchKernelGGL((fa2_latent_append_kernel<DT, 256>), grid, block, 0, st, a);
}

// ---- decode with many rows per key ------------------------------------------------

static_assert(kMaskTree == FA2_MASK_TREE && kRbMaxTree == FA2_TREE_MAX,
              "the kernels' mask words hold what the calls take");

// What the two decode calls share.
struct RowsCall {
  bool latent;
  int layout;
  int32_t dtype, mask;
  int64_t batch, q_heads, kv_heads, q_len, dv;
  int64_t kv_len;  // dense: keys; ragged: total rows
  int64_t page_size, num_pages, table_width;
};

struct RowsPlan {
  int64_t rows;  // of a unit: heads of a kv head times tokens
  int rg;        // 32-row groups of a q-block; 0: units of up to 16 rows
  int64_t part_rows, streams, segs, whole;
  bool cut;      // units may be cut: the merge is launched
  size_t off_ml, off_o, total;
};

// The balanced walk's costs, in tiles of 64 keys (fa2_decode_walk.h): units of up to kRbShort
// tiles stay whole, as do all of them if that costs the longest workgroup no more than kRbWhole
// (half of it where no workgroup would be idle): a cut unit's partials are 2 to 8 times those of
// the other decode kernels.
// (4 x 900 keys of 16 heads: 17.2 us; segments of at least 1 tile 18.2, of 4 20.9; kRbWhole 32:
// 30.0, as units stay whole on 4 workgroups.)
constexpr int64_t kRbMinTiles = 2;
constexpr int64_t kRbWhole = 16, kRbShort = 4;

int rows_plan(const RowsCall& c, RowsPlan* pl) {
  pl->rows = c.q_heads / c.kv_heads * c.q_len;
  if (pl->rows > kLim) return FA2_ERR_TOO_LARGE;
  const int64_t cus = cu_count_current_device();
  // The smallest q-block that holds the rows (4 x 900 keys of 16 heads: 17.4 us with up to 16
  // rows, 26 with 32; 128-row blocks read K and V least often beyond that).
  const int64_t least = c.dv == 64 ? 2 : 1;  // (a wave has 32 dims at least)
  pl->rg = static_cast<int>(pl->rows <= kR16Rows ? 0
                            : pl->rows <= 32     ? least
                            : pl->rows <= 64     ? 2
                                                 : 4);
  const int64_t block_rows = pl->rg ? 32 * pl->rg : kR16Rows;
  const int64_t nqb = cdiv(pl->rows, block_rows);
  // workgroups per CU (RowsTile::kOcc)
  const bool two = pl->rg > 0 && (c.latent ? c.dv == 256 && pl->rg < 4 : c.dv < 256);
  const int64_t wgs = two ? 2 * cus : cus;
  pl->part_rows = std::min<int64_t>(pl->rows, block_rows);
  pl->streams = c.kv_heads * nqb;
  // tiles of the call at most (lengths are on the device)
  const int64_t keys = c.layout == FA2_LAYOUT_PAGED ? c.table_width * c.page_size : c.kv_len;
  const int64_t tiles = std::max<int64_t>(cdiv(keys, kBN), 1);
  const int64_t total = c.layout == FA2_LAYOUT_RAGGED ? tiles + c.batch : tiles * c.batch;
  if (total >= (int64_t(1) << 30)) return FA2_ERR_TOO_LARGE;
  pl->segs = std::min(std::max<int64_t>(1, wgs / pl->streams), cdiv(total, kRbMinTiles));
  const int64_t grid = pl->streams * pl->segs;
  // (one segment per stream cuts no unit, and neither do short ones)
  pl->cut = pl->segs > 1 && tiles > kRbShort;
  const int64_t slots = pl->cut ? 2 * grid : 0;
  if (pl->streams * c.batch > kMaxGrid || grid > kMaxGrid) return FA2_ERR_TOO_LARGE;
  const int64_t idle = std::max<int64_t>(0, grid - pl->streams * c.batch);
  pl->whole = std::max(kRbWhole / 2, kRbWhole * idle / grid);
  size_t off = static_cast<size_t>(pl->streams * c.batch) * sizeof(int2);
  off = (off + 255) & ~size_t(255);
  pl->off_ml = off;
  off += static_cast<size_t>(slots * pl->part_rows) * 2 * sizeof(float);
  off = (off + 255) & ~size_t(255);
  pl->off_o = off;
  off += static_cast<size_t>(slots * pl->part_rows * c.dv) * sizeof(float);
  pl->total = off;
  return FA2_OK;
}

// Strides and pointers are the caller's; ra.a.k .. v and the tables are set.
int rows_fill(const RowsCall& c, const RowsPlan& pl, float scale, void* workspace, RowsArgs* ra) {
  KArgs& a = ra->a;
  a.batch = static_cast<int32_t>(c.batch);
  a.hq = static_cast<int32_t>(c.q_heads);
  a.hkv = static_cast<int32_t>(c.kv_heads);
  a.q_len = static_cast<int32_t>(pl.rows);
  a.kv_len = static_cast<int32_t>(c.layout == FA2_LAYOUT_PAGED ? c.table_width * c.page_size
                                                               : c.kv_len);
  a.page_size = static_cast<int32_t>(c.page_size);
  a.mask = c.mask;
  a.scale_log2 = scale * 1.4426950408889634f;
  char* ws = static_cast<char*>(workspace);
  ra->info = reinterpret_cast<int2*>(ws);
  a.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
  a.part_o = reinterpret_cast<float*>(ws + pl.off_o);
  a.part_rows = static_cast<int32_t>(pl.part_rows);
  a.block_rows = pl.rg ? 32 * pl.rg : kR16Rows;
  a.walk_streams = static_cast<int32_t>(pl.streams);
  a.walk_segs = static_cast<int32_t>(pl.segs);
  a.walk_min = kRbMinTiles;
  a.walk_whole = static_cast<int32_t>(pl.whole);
  a.walk_short = kRbShort;
  a.walk_rounds = static_cast<int32_t>(cdiv(c.batch, pl.segs));
  a.pack_m = static_cast<int32_t>(c.q_len);
  ra->num_pages = static_cast<int32_t>(c.num_pages);
  // n / page_size for n < 2^30 as (2 n * page_mul) >> 32 >> page_sh, with page_sh =
  // floor(log2 page_size) and page_mul = ceil(2^(31 + page_sh) / page_size): page_mul
  // is off by less than 1, the quotient by less than n / 2^(31 + page_sh), which is
  // under 1 / page_size since 2^page_sh > page_size / 2
  const int64_t page = std::max<int64_t>(c.page_size, 1);
  int sh = 0;
  while ((int64_t(2) << sh) <= page) ++sh;
  ra->page_sh = static_cast<uint32_t>(sh);
  ra->page_mul = static_cast<uint32_t>(cdiv(int64_t(1) << (31 + sh), page));
  return FA2_OK;
}

template <int DT, int DK, int DV, bool LAT, int MODE>
void launch_rows(const RowsArgs& ra, const RowsPlan& pl, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(pl.streams * pl.segs)), block(kRbThreads);
  constexpr int least = DV > 64 ? 1 : 2;
  if (pl.rg == 0)
    hipLaunchKernelGGL((fa2_decode_rows16_kernel<DT, DK, DV, LAT, MODE>), grid,
                       dim3(Rows16Tile<DK, DV, LAT>::kThreads), 0, st, ra);
  else if (pl.rg == 4 && pl.streams > ra.a.hkv)
    hipLaunchKernelGGL((fa2_decode_rows_kernel<DT, DK, DV, LAT, 4, MODE, false>), grid, block, 0,
                       st, ra);
  else if (pl.rg == 4)
    hipLaunchKernelGGL((fa2_decode_rows_kernel<DT, DK, DV, LAT, 4, MODE, true>), grid, block, 0, st,
                       ra);
  else if (pl.rg > least)
    hipLaunchKernelGGL((fa2_decode_rows_kernel<DT, DK, DV, LAT, 2, MODE, true>), grid, block, 0, st,
                       ra);
  else
    hipLaunchKernelGGL((fa2_decode_rows_kernel<DT, DK, DV, LAT, least, MODE, true>), grid, block, 0,
                       st, ra);
  if (pl.cut)
    hipLaunchKernelGGL((fa2_rows_merge_kernel<DT, DV>),
                       dim3(static_cast<uint32_t>(pl.streams * ra.a.batch),
                            static_cast<uint32_t>(cdiv(pl.part_rows, kMergeRows<DV>))),
                       dim3(256), 0, st, ra);
}

template <int DT, int MODE>
void launch_tree_dim(int64_t d, const RowsArgs& ra, const RowsPlan& pl, hipStream_t st) {
  if (d == 64) launch_rows<DT, 64, 64, false, MODE>(ra, pl, st);
  else if (d == 128) launch_rows<DT, 128, 128, false, MODE>(ra, pl, st);
  else launch_rows<DT, 256, 256, false, MODE>(ra, pl, st);
}

template <int DT>
void launch_tree(int layout, int64_t d, const RowsArgs& ra, const RowsPlan& pl, hipStream_t st) {
  if (layout == FA2_LAYOUT_DENSE) launch_tree_dim<DT, FA2_LAYOUT_DENSE>(d, ra, pl, st);
  else if (layout == FA2_LAYOUT_RAGGED) launch_tree_dim<DT, FA2_LAYOUT_RAGGED>(d, ra, pl, st);
  else launch_tree_dim<DT, FA2_LAYOUT_PAGED>(d, ra, pl, st);
}

template <int DT>
void launch_latent(int64_t latent, const RowsArgs& ra, const RowsPlan& pl, hipStream_t st) {
  if (latent == 512) launch_rows<DT, 576, 512, true, FA2_LAYOUT_PAGED>(ra, pl, st);
  else launch_rows<DT, 320, 256, true, FA2_LAYOUT_PAGED>(ra, pl, st);
}

bool scale_ok(float s) { return s > 0.f && std::isfinite(s); }

// Sizes that both decode calls check.
int validate_rows_sizes(const RowsCall& c) {
  if (!half_type(c.dtype)) return FA2_ERR_BAD_DTYPE;
  if (c.batch < 0 || c.q_heads <= 0 || c.kv_heads <= 0 || c.q_len < 0 || c.kv_len < 0 ||
      c.q_heads % c.kv_heads)
    return FA2_ERR_BAD_SHAPE;
  if (c.mask == FA2_MASK_TREE && c.q_len > FA2_TREE_MAX) return FA2_ERR_BAD_SHAPE;
  if (c.layout == FA2_LAYOUT_PAGED &&
      (c.page_size <= 0 || c.num_pages < 0 || c.table_width < 0))
    return FA2_ERR_PAGED_ARGS;
  if (c.batch > 64 * kWalkMaxPer || c.q_heads > 65536 || c.q_len > kLim || c.kv_len > kLim)
    return FA2_ERR_TOO_LARGE;
  if (c.layout == FA2_LAYOUT_PAGED) {
    // keys of a table row in 30 bits
    if (c.page_size > kLim || c.num_pages > kLim || c.table_width > kLim ||
        (c.table_width > 0 && c.page_size > kLim / c.table_width))
      return FA2_ERR_TOO_LARGE;
  }
  return FA2_OK;
}

RowsCall call_of(const fa2_latent_decode_params& p) {
  return {true,   FA2_LAYOUT_PAGED, p.dtype,      p.mask, p.batch,     p.q_heads,   1,
          p.q_len, p.latent_dim, 0, p.page_size, p.num_pages, p.table_width};
}

int validate_latent(const fa2_latent_decode_params* p) {
  if (!p) return FA2_ERR_NULL_POINTER;
  if (!half_type(p->dtype)) return FA2_ERR_BAD_DTYPE;
  if (p->mask != FA2_MASK_NONE && p->mask != FA2_MASK_CAUSAL_BOTTOM_RIGHT &&
      p->mask != FA2_MASK_TREE)
    return FA2_ERR_BAD_MASK;
  if (!latent_dims_ok(p->latent_dim, p->rope_dim)) return FA2_ERR_HEAD_DIM;
  if (p->table_stride < 0) return FA2_ERR_PAGED_ARGS;
  const int s = validate_rows_sizes(call_of(*p));
  if (s != FA2_OK) return s;
  const int64_t strides[] = {p->q_sb, p->q_sh, p->q_ss, p->o_sb, p->o_sh, p->o_ss};
  for (int64_t x : strides)
    if (!stride_ok(x, 2)) return FA2_ERR_ALIGNMENT;
  if (p->q_len > 0 && p->q_heads > 1 && p->o_sh != p->q_len * p->o_ss) return FA2_ERR_Q_LAYOUT;
  return FA2_OK;
}

RowsCall call_of(const fa2_tree_decode_params& p) {
  const bool paged = p.layout == FA2_LAYOUT_PAGED;
  return {false,   p.layout,   p.dtype,    FA2_MASK_TREE, p.batch, p.q_heads, p.kv_heads,
          p.q_len, p.head_dim, p.kv_len,
          paged ? p.page_size : 1, paged && p.page_size > 0 ? p.kv_len / p.page_size : 0,
          paged ? p.table_width : 0};
}

int validate_tree(const fa2_tree_decode_params* p) {
  if (!p) return FA2_ERR_NULL_POINTER;
  if (p->layout < FA2_LAYOUT_DENSE || p->layout > FA2_LAYOUT_PAGED) return FA2_ERR_BAD_LAYOUT;
  if (!half_type(p->dtype)) return FA2_ERR_BAD_DTYPE;
  if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256) return FA2_ERR_HEAD_DIM;
  if (p->layout == FA2_LAYOUT_PAGED && (p->k_table_stride < 0 || p->v_table_stride < 0))
    return FA2_ERR_PAGED_ARGS;
  const int s = validate_rows_sizes(call_of(*p));
  if (s != FA2_OK) return s;
  const int64_t strides[] = {p->q_sb, p->q_sh, p->q_ss, p->k_sb, p->k_sh, p->k_ss,
                             p->v_sb, p->v_sh, p->v_ss, p->o_sb, p->o_sh, p->o_ss};
  for (int64_t x : strides)
    if (!stride_ok(x, 2)) return FA2_ERR_ALIGNMENT;
  // eight rows are addressed by 32-bit offsets from the first
  const int64_t row_lim = int64_t(1) << 25;
  for (int64_t x : {p->k_ss, p->v_ss})
    if (x < 0 || x * 2 > row_lim) return FA2_ERR_TOO_LARGE;
  if (p->q_len > 0 && p->q_heads / p->kv_heads > 1 && p->o_sh != p->q_len * p->o_ss)
    return FA2_ERR_Q_LAYOUT;
  return FA2_OK;
}

template <typename P>
int rows_workspace(const P* p, int valid, size_t* bytes) {
  if (!bytes) return FA2_ERR_NULL_POINTER;
  if (valid != FA2_OK) return valid;
  *bytes = 0;
  if (p->batch == 0 || p->q_len == 0) return FA2_OK;
  RowsPlan pl{};
  const int s = rows_plan(call_of(*p), &pl);
  if (s == FA2_OK) *bytes = pl.total;
  return s;
}

// The plan, the workspace's checks and the common arguments.
template <typename P>
int rows_begin(const P* p, RowsPlan* pl, RowsArgs* ra) {
  if (!scale_ok(p->softmax_scale)) return FA2_ERR_BAD_SHAPE;
  const RowsCall c = call_of(*p);
  if (c.mask == FA2_MASK_TREE && !p->tree) return FA2_ERR_NULL_POINTER;
  int s = rows_plan(c, pl);
  if (s != FA2_OK) return s;
  if (!p->workspace || p->workspace_bytes < pl->total) return FA2_ERR_WORKSPACE;
  if (!aligned16(p->workspace)) return FA2_ERR_ALIGNMENT;
  KArgs& a = ra->a;
  a.q = p->q;
  a.o = p->o;
  a.q_sb = p->q_sb; a.q_sh = p->q_sh; a.q_ss = p->q_ss;
  a.o_sb = p->o_sb; a.o_sh = p->o_sh;
  a.o_ss = p->q_len > 1 ? p->o_ss : p->o_sh;  // rows of a unit: its heads
  ra->tree = p->tree;
  ra->tree_sb = p->tree_sb;
  ra->tree_sr = p->tree_sr;
  return rows_fill(c, *pl, p->softmax_scale, p->workspace, ra);
}

// ---- the expanded form -------------------------------------------------------------

constexpr size_t kClaimAt = 128;  // of the claim counters, in the 256 bytes of the counts

struct PrefillPlan {
  bool pair;  // the two-head kernel over pairs of q-blocks; else the one-head kernel
  int64_t work_ub, npairs, grid, wgs;  // items, times heads, unit slots, workgroups
  int splits;
  bool plan, inline_plan;  // ragged: the plan kernel's list, or each workgroup's own
  size_t off_work, off_count, off_ml, off_o, total;
};

int validate_prefill(const fa2_latent_prefill_params* p) {
  if (!p) return FA2_ERR_NULL_POINTER;
  if (p->layout != FA2_LAYOUT_DENSE && p->layout != FA2_LAYOUT_RAGGED) return FA2_ERR_BAD_LAYOUT;
  if (!half_type(p->dtype)) return FA2_ERR_BAD_DTYPE;
  if (p->mask < FA2_MASK_NONE || p->mask > FA2_MASK_CAUSAL_BOTTOM_RIGHT) return FA2_ERR_BAD_MASK;
  if ((p->head_dim != 64 && p->head_dim != 128) || p->rope_dim != kLaRope)
    return FA2_ERR_HEAD_DIM;
  if (p->batch < 0 || p->heads <= 0 || p->q_len < 0 || p->kv_len < 0) return FA2_ERR_BAD_SHAPE;
  if (p->layout == FA2_LAYOUT_RAGGED && (!p->q_indptr || !p->kv_indptr)) return FA2_ERR_RAGGED_ARGS;
  const int64_t strides[] = {p->q_sb, p->q_sh, p->q_ss, p->k_sb, p->k_sh, p->k_ss, p->v_sb,
                             p->v_sh, p->v_ss, p->o_sb, p->o_sh, p->o_ss, p->kr_sb, p->kr_ss};
  for (int64_t x : strides)
    if (!stride_ok(x, 2)) return FA2_ERR_ALIGNMENT;
  if (p->batch > kLim || p->heads > 65536 || p->q_len > kLim || p->kv_len > kLim)
    return FA2_ERR_TOO_LARGE;
  // a tile's (or q-block's) rows are addressed by 32-bit offsets from its first row
  const int64_t row_lim = int64_t(1) << 25;
  for (int64_t x : {p->q_ss, p->k_ss, p->v_ss, p->o_ss, p->kr_ss})
    if (x < 0 || x * 2 > row_lim) return FA2_ERR_TOO_LARGE;
  return FA2_OK;
}

int prefill_plan(const fa2_latent_prefill_params* p, PrefillPlan* pl) {
  const bool ragged = p->layout == FA2_LAYOUT_RAGGED;
  const int64_t nqb = cdiv(p->q_len, kBM), cus = cu_count_current_device();
  // items of `rows` rows (ragged: one more for each sequence at most)
  auto items = [&](int64_t rows) {
    return (ragged ? cdiv(p->q_len, rows) + p->batch : cdiv(p->q_len, rows) * p->batch);
  };
  if (items(kBM) * p->heads > kMaxGrid - kXcds) return FA2_ERR_TOO_LARGE;
  // Pairs of q-blocks on one workgroup per CU where sequences have four q-blocks on average
  // (a lone block leaves half of the workgroup without rows) and the pairs fill the CUs: 825 to
  // 855 TFLOP/s on 16 prompts of 128-4096.  Else one q-block per workgroup, two workgroups per
  // CU, the keys split over idle ones: one prompt of 333, 16 heads 15.1 us (pairs 19); in one
  // run, 8 chunks of 100-512 rows over up to 4000 more, 16 heads, 118 (pairs 143), of 384-512 over
  // none 28 (33), over up to 1000 58 (62), over up to 4000 141 (151).  Ragged pairs read the shared
  // part's prefix sum anew for each tile and wait for all loads there, which dense ones and one
  // q-block do not: 16 prompts of 2048 take 852 ragged and 835 dense.
  const bool many = ragged ? p->q_len >= 4 * kBM * p->batch : nqb >= 4;
  pl->pair = many && cus >= kXcds && items(2 * kBM) * p->heads >= cus;
  pl->work_ub = items(pl->pair ? 2 * kBM : kBM);
  pl->npairs = pl->work_ub * p->heads;
  pl->grid = cdiv(pl->npairs, kXcds) * kXcds;
  // Splits of the keys where the units leave CUs idle, kMinSplitTiles tiles each at least
  // (ragged: the plan kernel lowers the count to what the longest sequence takes).
  int64_t keys = p->kv_len;
  if (p->mask == FA2_MASK_CAUSAL_TOP_LEFT) keys = std::min(keys, p->q_len);
  const int64_t slots = cus * (pl->pair ? 1 : 2);
  int64_t s = std::min(cdiv(slots, std::max<int64_t>(pl->npairs, 1)),
                       cdiv(keys, kBN) / kMinSplitTiles);
  s = pl->pair ? 1 : std::max<int64_t>(1, std::min<int64_t>(s, FA2_MAX_SPLITS));
  pl->splits = static_cast<int>(s);
  pl->wgs = pl->pair ? std::min(pl->grid, cus) : pl->grid;
  pl->inline_plan =
      ragged && !pl->pair && s == 1 && p->batch <= kInlinePlanMaxBatch && pl->grid <= slots;
  pl->plan = ragged && !pl->inline_plan;
  size_t off = 0;
  pl->off_work = off;
  if (pl->plan) off += static_cast<size_t>(pl->work_ub) * sizeof(int2);
  off = (off + 255) & ~size_t(255);
  pl->off_count = off;  // the item count, the split count, the claim counters at kClaimAt
  if (pl->plan) off += 256;
  const size_t parts = s > 1 ? static_cast<size_t>(s * pl->grid) : 0;
  pl->off_ml = off;
  off += parts * kBM * 2 * sizeof(float);
  off = (off + 255) & ~size_t(255);
  pl->off_o = off;
  off += parts * kBM * p->head_dim * sizeof(float);
  pl->total = off;
  return FA2_OK;
}

template <int DT, int D, int MODE>
void launch_prefill_typed(const KArgs& a, const PrefillPlan& pl, hipStream_t st) {
  if constexpr (MODE == FA2_LAYOUT_RAGGED) {
    if (pl.plan)
      hipLaunchKernelGGL((fa2_plan_kernel<MODE>), dim3(1), dim3(kPlanThreads), 0, st, a,
                         const_cast<int2*>(a.work), const_cast<int32_t*>(a.work_count));
  }
  if (!pl.pair) {
    hipLaunchKernelGGL((fa2_fwd_lds_kernel<DT, D, MODE, true, false, false, kLaRope>),
                       dim3(static_cast<uint32_t>(pl.wgs), pl.splits), dim3(kThreads), 0, st, a);
    if (pl.splits > 1)
      hipLaunchKernelGGL((fa2_combine_kernel<DT, D, MODE>),
                         dim3(static_cast<uint32_t>(pl.grid), kBM / kCombineRows<D>),
                         dim3(kThreads), 0, st, a);
    return;
  }
  // (ragged units are claimed: KArgs::claim)
  hipLaunchKernelGGL((fa2_fwd_pp_kernel<DT, D, MODE, true, MODE == FA2_LAYOUT_RAGGED, false, false,
                                        false, kLaRope>),
                     dim3(static_cast<uint32_t>(pl.wgs)), dim3(kPPThreads), 0, st, a);
}

template <int DT>
void launch_prefill(const fa2_latent_prefill_params* p, const KArgs& a, const PrefillPlan& pl,
                    hipStream_t st) {
  if (p->layout == FA2_LAYOUT_DENSE) {
    if (p->head_dim == 64) launch_prefill_typed<DT, 64, FA2_LAYOUT_DENSE>(a, pl, st);
    else launch_prefill_typed<DT, 128, FA2_LAYOUT_DENSE>(a, pl, st);
  } else {
    if (p->head_dim == 64) launch_prefill_typed<DT, 64, FA2_LAYOUT_RAGGED>(a, pl, st);
    else launch_prefill_typed<DT, 128, FA2_LAYOUT_RAGGED>(a, pl, st);
  }
}

}  // namespace
}  // namespace fa2

using namespace fa2;

extern "C" size_t fa2_latent_params_size(int which) {
  switch (which) {
    case 0: return sizeof(fa2_latent_append_params);
    case 1: return sizeof(fa2_latent_decode_params);
    case 2: return sizeof(fa2_tree_decode_params);
    case 3: return sizeof(fa2_latent_prefill_params);
    default: return 0;
  }
}

extern "C" int fa2_latent_append(const fa2_latent_append_params* p, void* stream) {
  const int s = validate_append(p);
  if (s != FA2_OK) return s;
  if (p->batch == 0 || p->num_rows == 0) return FA2_OK;
  if (!p->x || !p->cache || !p->weight || !p->indptr || (p->positions && !p->rope) ||
      (p->table_width && !p->block_table))
    return FA2_ERR_NULL_POINTER;
  const void* ptrs[] = {p->x, p->rows_out, p->cache, p->weight, p->rope};
  for (const void* x : ptrs)
    if (!aligned16(x)) return FA2_ERR_ALIGNMENT;
  LatentAppendArgs a{};
  a.x = static_cast<const char*>(p->x);
  a.out = static_cast<char*>(p->rows_out);
  a.cache = static_cast<char*>(p->cache);
  a.w = static_cast<const char*>(p->weight);
  a.rope = p->rope;
  a.indptr = p->indptr;
  a.start = p->start_pos;
  a.table = p->block_table;
  a.x_ts = p->x_ts * 2;
  a.rope_stride = p->rope_stride;
  a.table_stride = p->table_stride;
  a.batch = static_cast<int32_t>(p->batch);
  a.num_rows = static_cast<int32_t>(p->num_rows);
  a.page_size = static_cast<int32_t>(p->page_size);
  a.num_pages = static_cast<int32_t>(p->num_pages);
  a.table_width = static_cast<int32_t>(p->table_width);
  a.positions = static_cast<int32_t>(p->positions);
  a.inter = p->interleaved ? 1 : 0;
  a.w32 = p->weight_dtype == FA2_DTYPE_F32 ? 1 : 0;
  a.eps = p->eps;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == FA2_DTYPE_F16) launch_append<FA2_DTYPE_F16>(p->latent_dim, a, st);
  else launch_append<FA2_DTYPE_BF16>(p->latent_dim, a, st);
  return launched();
}

extern "C" int fa2_latent_decode_workspace_size(const fa2_latent_decode_params* p, size_t* bytes) {
  return rows_workspace(p, validate_latent(p), bytes);
}

extern "C" int fa2_latent_decode(const fa2_latent_decode_params* p, void* stream) {
  int s = validate_latent(p);
  if (s != FA2_OK) return s;
  if (p->batch == 0 || p->q_len == 0) return FA2_OK;
  if (!p->q || !p->o || !p->cache) return FA2_ERR_NULL_POINTER;
  if (!p->kv_lens || p->num_pages == 0 || (p->table_width > 0 && !p->block_table))
    return FA2_ERR_PAGED_ARGS;
  if (!aligned16(p->q) || !aligned16(p->o) || !aligned16(p->cache)) return FA2_ERR_ALIGNMENT;
  RowsPlan pl{};
  RowsArgs ra{};
  s = rows_begin(p, &pl, &ra);
  if (s != FA2_OK) return s;
  KArgs& a = ra.a;
  a.k = a.v = p->cache;
  a.kv_indptr = p->kv_lens;
  a.k_table = a.v_table = p->block_table;
  a.k_table_stride = a.v_table_stride = p->table_stride;
  a.k_ss = a.v_ss = p->latent_dim + p->rope_dim;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == FA2_DTYPE_F16) launch_latent<FA2_DTYPE_F16>(p->latent_dim, ra, pl, st);
  else launch_latent<FA2_DTYPE_BF16>(p->latent_dim, ra, pl, st);
  return launched();
}

extern "C" int fa2_tree_decode_workspace_size(const fa2_tree_decode_params* p, size_t* bytes) {
  return rows_workspace(p, validate_tree(p), bytes);
}

extern "C" int fa2_tree_decode(const fa2_tree_decode_params* p, void* stream) {
  int s = validate_tree(p);
  if (s != FA2_OK) return s;
  if (p->batch == 0 || p->q_len == 0) return FA2_OK;
  if (!p->q || !p->o || (p->kv_len && (!p->k || !p->v))) return FA2_ERR_NULL_POINTER;
  if (p->layout == FA2_LAYOUT_RAGGED && !p->kv_indptr) return FA2_ERR_RAGGED_ARGS;
  if (p->layout == FA2_LAYOUT_PAGED &&
      (!p->kv_indptr || p->kv_len < p->page_size ||
       (p->table_width > 0 && (!p->k_block_table || !p->v_block_table))))
    return FA2_ERR_PAGED_ARGS;
  const void* ptrs[] = {p->q, p->o, p->k, p->v};
  for (const void* x : ptrs)
    if (!aligned16(x)) return FA2_ERR_ALIGNMENT;
  RowsPlan pl{};
  RowsArgs ra{};
  s = rows_begin(p, &pl, &ra);
  if (s != FA2_OK) return s;
  KArgs& a = ra.a;
  a.k = p->k;
  a.v = p->v;
  a.kv_indptr = p->kv_indptr;
  a.k_table = p->k_block_table;
  a.v_table = p->v_block_table;
  a.k_sb = p->k_sb; a.k_sh = p->k_sh; a.k_ss = p->k_ss;
  a.v_sb = p->v_sb; a.v_sh = p->v_sh; a.v_ss = p->v_ss;
  a.k_table_stride = p->k_table_stride;
  a.v_table_stride = p->v_table_stride;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == FA2_DTYPE_F16) launch_tree<FA2_DTYPE_F16>(p->layout, p->head_dim, ra, pl, st);
  else launch_tree<FA2_DTYPE_BF16>(p->layout, p->head_dim, ra, pl, st);
  return launched();
}

extern "C" int fa2_latent_prefill_workspace_size(const fa2_latent_prefill_params* p,
                                                 size_t* bytes) {
  if (!bytes) return FA2_ERR_NULL_POINTER;
  int s = validate_prefill(p);
  if (s != FA2_OK) return s;
  *bytes = 0;
  if (p->batch == 0 || p->q_len == 0) return FA2_OK;
  PrefillPlan pl{};
  s = prefill_plan(p, &pl);
  if (s == FA2_OK) *bytes = pl.total;
  return s;
}

extern "C" int fa2_latent_prefill(const fa2_latent_prefill_params* p, void* stream) {
  int s = validate_prefill(p);
  if (s != FA2_OK) return s;
  if (p->batch == 0 || p->q_len == 0) return FA2_OK;
  if (!p->q || !p->o || (p->kv_len && (!p->k || !p->kr || !p->v))) return FA2_ERR_NULL_POINTER;
  if (!scale_ok(p->softmax_scale)) return FA2_ERR_BAD_SHAPE;
  const void* ptrs[] = {p->q, p->o, p->k, p->kr, p->v};
  for (const void* x : ptrs)
    if (!aligned16(x)) return FA2_ERR_ALIGNMENT;
  PrefillPlan pl{};
  s = prefill_plan(p, &pl);
  if (s != FA2_OK) return s;
  if (pl.total && (!p->workspace || p->workspace_bytes < pl.total)) return FA2_ERR_WORKSPACE;
  if (!aligned16(p->workspace)) return FA2_ERR_ALIGNMENT;
  KArgs a{};
  a.q = p->q;
  a.k = p->k;
  a.v = p->v;
  a.o = p->o;
  a.kr = p->kr;
  a.q_indptr = p->q_indptr;
  a.kv_indptr = p->kv_indptr;
  a.q_sb = p->q_sb; a.q_sh = p->q_sh; a.q_ss = p->q_ss;
  a.k_sb = p->k_sb; a.k_sh = p->k_sh; a.k_ss = p->k_ss;
  a.v_sb = p->v_sb; a.v_sh = p->v_sh; a.v_ss = p->v_ss;
  a.o_sb = p->o_sb; a.o_sh = p->o_sh; a.o_ss = p->o_ss;
  a.kr_sb = p->kr_sb; a.kr_ss = p->kr_ss;
  a.batch = static_cast<int32_t>(p->batch);
  a.hq = a.hkv = static_cast<int32_t>(p->heads);
  a.q_len = static_cast<int32_t>(p->q_len);
  a.kv_len = static_cast<int32_t>(p->kv_len);
  a.page_size = 1;
  a.page_shift = 0;
  a.nqb = static_cast<int32_t>(cdiv(p->q_len, pl.pair ? 2 * kBM : kBM));
  a.qpair = pl.pair ? 1 : 0;
  a.block_rows = kBM;
  a.work_ub = static_cast<int32_t>(pl.work_ub);
  a.npairs = static_cast<int32_t>(pl.npairs);
  a.mask = p->mask;
  a.num_splits = pl.splits;
  a.part_slots = static_cast<int32_t>(pl.grid);
  a.part_rows = kBM;
  a.units = static_cast<int32_t>(pl.grid);
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  a.dv = static_cast<int32_t>(p->head_dim);
  char* ws = static_cast<char*>(p->workspace);
  if (pl.plan) {
    int32_t* count = reinterpret_cast<int32_t*>(ws + pl.off_count);
    a.work = reinterpret_cast<const int2*>(ws + pl.off_work);
    a.work_count = count;
    if (pl.splits > 1) a.split_count = count + 1;
    // Units are claimed per XCD, so that its workgroups run the q-blocks of one or two
    // sequences at a time and share their K/V in its L2, as in fa2_fwd.
    if (pl.pair) a.claim = count + kClaimAt / sizeof(int32_t);
  }
  if (pl.splits > 1) {
    a.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
    a.part_o = reinterpret_cast<float*>(ws + pl.off_o);
  }
  a.inline_plan = pl.inline_plan ? 1 : 0;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == FA2_DTYPE_F16) launch_prefill<FA2_DTYPE_F16>(p, a, pl, st);
  else launch_prefill<FA2_DTYPE_BF16>(p, a, pl, st);
  return launched();
}
