// fa2_ops.hip - C ABI and launch logic of the operators around the attention
// (declared in include/fa2_ops.h).
#include "fa2_ops.h"

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "fa2_host.h"
#include "fa2_fp4_rows.h"
#include "fa2_kernel_decode_fp4.h"
#include "fa2_norm_rope.h"

namespace fa2 {
namespace {

constexpr int64_t kLim = INT32_MAX / 2;  // 32-bit counters inside the kernels

int launched() { return hipGetLastError() == hipSuccess ? FA2_OK : FA2_ERR_HIP; }

int log2_exact(int64_t n) {  // -1: not a power of two
  for (int s = 0; s < 31; ++s)
    if ((int64_t(1) << s) == n) return s;
  return -1;
}

// ---- norms and rotation ------------------------------------------------------

int validate_norm_rope(const fa2_norm_rope_params* p) {
  if (!p) return FA2_ERR_NULL_POINTER;
  if (p->dtype < FA2_DTYPE_F16 || p->dtype > FA2_DTYPE_F32) return FA2_ERR_BAD_DTYPE;
  if (p->weight_dtype != p->dtype && p->weight_dtype != FA2_DTYPE_F32) return FA2_ERR_BAD_DTYPE;
  const int64_t d = p->head_dim;
  if (d != 16 && d != 32 && d != 64 && d != 128 && d != 256) return FA2_ERR_HEAD_DIM;
  if (p->tokens < 0 || p->q_heads < 0 || p->kv_heads < 0 || p->positions < 0 ||
      p->rotary_dim < 0 || p->rotary_dim > d || p->rotary_dim % 16 || p->rope_stride < 0 ||
      !(p->eps >= 0.f))
    return FA2_ERR_BAD_SHAPE;
  if (p->tokens > 0 && (p->q_rows <= 0 || p->k_rows <= 0)) return FA2_ERR_BAD_SHAPE;
  if (p->tokens > kLim || p->q_heads > 65536 || p->kv_heads > 65536 || p->positions > kLim ||
      p->q_rows > kLim || p->k_rows > kLim)
    return FA2_ERR_TOO_LARGE;
  const int eb = elt_bytes(p->dtype);
  const int64_t strides[] = {p->q_sb,  p->q_sh,  p->q_ss,  p->k_sb,  p->k_sh,  p->k_ss,
                             p->qo_sb, p->qo_sh, p->qo_ss, p->ko_sb, p->ko_sh, p->ko_ss};
  for (int64_t s : strides)
    if (!stride_ok(s, eb)) return FA2_ERR_ALIGNMENT;
  if (p->rope_stride % 4) return FA2_ERR_ALIGNMENT;
  return FA2_OK;
}

template <int DT, int D>
void launch_norm_rope(const NormRopeArgs& a, int u, uint32_t grid, hipStream_t st) {
  const dim3 g(grid), block(kNrThreads);
  // Stores past the caches where there are many rows of 16 bits and the lanes' chunks are
  // runs of memory; two chunks side by side per lane (neighbouring pairs, dims that are
  // not rotated) are half lines there.  Past / through the caches, us, 40 heads of D128: 2048
  // tokens 9.3 / 11.8, 8192 34.0 / 35.3, with the 4-bit append after it 45.5 / 46.0, but
  // with attention over sequences of 1024 after it 133.8 / 129.9; 8192 in neighbouring
  // pairs 46.7 / 38.1, half of the dims rotated 40.8 / 37.7, fp32 59.4 / 57.3.
  if (u != 4)
    hipLaunchKernelGGL((fa2_norm_rope_kernel<DT, D, 1, false>), g, block, 0, st, a);
  else if (DT != FA2_DTYPE_F32 && a.rot == D && !a.inter)
    hipLaunchKernelGGL((fa2_norm_rope_kernel<DT, D, 4, DT != FA2_DTYPE_F32>), g, block, 0, st, a);
  else
    hipLaunchKernelGGL((fa2_norm_rope_kernel<DT, D, 4, false>), g, block, 0, st, a);
}

template <int DT>
void launch_norm_rope_dim(int64_t d, const NormRopeArgs& a, int u, uint32_t grid, hipStream_t st) {
  switch (d) {
    case 16: return launch_norm_rope<DT, 16>(a, u, grid, st);
    case 32: return launch_norm_rope<DT, 32>(a, u, grid, st);
    case 64: return launch_norm_rope<DT, 64>(a, u, grid, st);
    case 128: return launch_norm_rope<DT, 128>(a, u, grid, st);
    default: return launch_norm_rope<DT, 256>(a, u, grid, st);
  }
}

// ---- the 4-bit cache -----------------------------------------------------------

bool fp4_dim_ok(int64_t d) { return d == 64 || d == 128 || d == 256; }

int validate_rows(const fa2_fp4_rows_params* p) {
  if (!p) return FA2_ERR_NULL_POINTER;
  if (p->dtype < FA2_DTYPE_F16 || p->dtype > FA2_DTYPE_F32) return FA2_ERR_BAD_DTYPE;
  if (!fp4_dim_ok(p->head_dim)) return FA2_ERR_HEAD_DIM;
  if (p->batch < 0 || p->kv_heads <= 0 || p->num_rows < 0 || p->page_size <= 0 ||
      p->num_pages < 0 || p->table_width < 0 || p->k_table_stride < 0 || p->v_table_stride < 0)
    return FA2_ERR_BAD_SHAPE;
  if (p->batch > kLim || p->num_rows > kLim || p->page_size > kLim || p->num_pages > kLim ||
      p->table_width > kLim || p->kv_heads > kLim / (p->head_dim / 2) ||
      p->page_size > kLim / (p->kv_heads * (p->head_dim / 2)))  // (a page's bytes: 31 bits)
    return FA2_ERR_TOO_LARGE;
  const int eb = elt_bytes(p->dtype);
  const int64_t strides[] = {p->k_ts, p->k_hs, p->v_ts, p->v_hs};
  for (int64_t s : strides)
    if (!stride_ok(s, eb)) return FA2_ERR_ALIGNMENT;
  return FA2_OK;
}

int fp4_rows(const fa2_fp4_rows_params* p, void* stream, bool append) {
  int s = validate_rows(p);
  if (s != FA2_OK) return s;
  if (p->batch == 0 || p->num_rows == 0) return FA2_OK;
  const bool has_v = p->v || p->v_codes || p->v_scales || p->v_block_table;
  const bool tables = p->table_width > 0;  // (tables without columns may be null)
  if (!p->k || !p->k_codes || !p->k_scales || !p->indptr || (tables && !p->k_block_table) ||
      (has_v && (!p->v || !p->v_codes || !p->v_scales || (tables && !p->v_block_table))))
    return FA2_ERR_NULL_POINTER;
  if (!aligned16(p->k) || !aligned16(p->k_codes) ||
      (has_v && (!aligned16(p->v) || !aligned16(p->v_codes))))
    return FA2_ERR_ALIGNMENT;
  const int64_t eb = elt_bytes(p->dtype);
  Fp4RowsArgs a{};
  a.x[0] = static_cast<char*>(p->k);
  a.x[1] = static_cast<char*>(p->v);
  a.codes[0] = p->k_codes;
  a.codes[1] = p->v_codes;
  a.scales[0] = p->k_scales;
  a.scales[1] = p->v_scales;
  a.table[0] = p->k_block_table;
  a.table[1] = p->v_block_table;
  a.table_stride[0] = p->k_table_stride;
  a.table_stride[1] = p->v_table_stride;
  a.ts[0] = p->k_ts * eb;
  a.hs[0] = p->k_hs * eb;
  a.ts[1] = p->v_ts * eb;
  a.hs[1] = p->v_hs * eb;
  a.indptr = p->indptr;
  a.start = p->start_pos;
  a.batch = static_cast<int32_t>(p->batch);
  a.heads = static_cast<int32_t>(p->kv_heads);
  a.words = static_cast<int32_t>(p->kv_heads * (p->head_dim / 8));
  a.word_shift = log2_exact(p->head_dim / 8);
  a.num_rows = static_cast<int32_t>(p->num_rows);
  a.page_size = static_cast<int32_t>(p->page_size);
  a.page_shift = log2_exact(p->page_size);
  a.num_pages = static_cast<int32_t>(p->num_pages);
  a.table_width = static_cast<int32_t>(p->table_width);
  a.has_v = has_v ? 1 : 0;
  a.rows_at_once = std::max(kF4Threads / a.words, 1);
  a.block_rows = 4 * a.rows_at_once;
  const dim3 grid(static_cast<uint32_t>(cdiv(p->num_rows, a.block_rows)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Gathered rows of more than 256 MB, which pass the caches: fewer writers at once write in
  // longer runs.  8 heads of D128 bf16, us at 8 / 6 / 5 / 4 / 3 waves per SIMD: 156 k rows (638
  // MB) 152 / 145 / 139.5 / 145 / 168, 400 k 407 / 391 / 364 / 375 / 446; 32 heads, 72 k rows 280 /
  // 276 / 273 / 266 / 263; fp32 156 k rows 289 / - / 285 / 275 / 280; 17 k bf16 (71 MB) 17.4 at any.
  const bool large =
      p->num_rows > (int64_t(1) << 28) / (p->kv_heads * p->head_dim * eb * (has_v ? 2 : 1));
  auto go = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    if (append)
      hipLaunchKernelGGL((fa2_fp4_append_kernel<DT>), grid, dim3(kF4Threads), 0, st, a);
    else if (large)
      hipLaunchKernelGGL((fa2_fp4_gather_kernel<DT, 5>), grid, dim3(kF4Threads), 0, st, a);
    else
      hipLaunchKernelGGL((fa2_fp4_gather_kernel<DT, 8>), grid, dim3(kF4Threads), 0, st, a);
  };
  if (p->dtype == FA2_DTYPE_F16) go(std::integral_constant<int, FA2_DTYPE_F16>{});
  else if (p->dtype == FA2_DTYPE_BF16) go(std::integral_constant<int, FA2_DTYPE_BF16>{});
  else go(std::integral_constant<int, FA2_DTYPE_F32>{});
  return launched();
}

// The balanced walk's costs, in KV tiles of 64 keys (fa2_decode_walk.h).  A segment of
// cut units has kD4MinTiles at least (2 instead of 4: 1 x 2500 keys 14.4 / 12.4 us, 4 x 2500
// the same); the grid has a workgroup per kD4GridTiles at most (2 or 4: the same).
// Units stay whole where that costs at most kD4Whole tiles, in proportion to the CUs
// that whole units leave idle and half of it at least, or they have kD4Short at most.
// Whole / cut, us, 8 kv heads of D128.  Whole by the rule: 1 x 1023 keys 9.9 / 11.3, 4 x 1023
// 10.5 / 12.0, 8 x 700 9.1 / 11.4, 16 x 500-1000 10.2 / 12.5, 16 x 1500 12.7 / 14.2, 32 x
// 1000-2000 15.9 / 16.5, and at its border 8 x 1500 12.5 / 11.7 to 12.5.  Cut: 8 x 1900 14.2 /
// 13.1, 4 x 2500 16.9 / 14.2, 8 x 2500 17.1 / 14.0; but 24 x 1500-2500, whose 192 units nearly
// fill the CUs, 17.3 / 22.1: the rule holds no cost of cutting unequal units.
constexpr int64_t kD4MinTiles = 4;
constexpr int64_t kD4GridTiles = 2;
constexpr int64_t kD4Whole = 24, kD4Short = 12;
constexpr int64_t kD4Wide = 24;  // (fp4_plan)

struct Fp4Plan {
  int64_t rows;        // of a unit: Hq / Hkv * q_len
  int rb;              // 16-row blocks of a q-block
  int64_t part_rows;
  int64_t streams, segs, whole;
  size_t off_ml, off_o, total;
};

int validate_fp4_decode(const fa2_fp4_decode_params* p) {
  if (!p) return FA2_ERR_NULL_POINTER;
  if (p->dtype != FA2_DTYPE_F16 && p->dtype != FA2_DTYPE_BF16) return FA2_ERR_BAD_DTYPE;
  if (p->mask != FA2_MASK_NONE && p->mask != FA2_MASK_CAUSAL_BOTTOM_RIGHT) return FA2_ERR_BAD_MASK;
  if (!fp4_dim_ok(p->head_dim)) return FA2_ERR_HEAD_DIM;
  if (p->batch < 0 || p->q_heads <= 0 || p->kv_heads <= 0 || p->q_len < 0 ||
      p->q_heads % p->kv_heads)
    return FA2_ERR_BAD_SHAPE;
  if (p->page_size <= 0 || p->num_pages < 0 || p->table_width < 0 || p->k_table_stride < 0 ||
      p->v_table_stride < 0)
    return FA2_ERR_PAGED_ARGS;
  if (p->batch > 64 * kWalkMaxPer || p->q_heads > 65536 || p->q_len > kLim ||
      p->page_size > kLim || p->num_pages > kLim || p->table_width > kLim)
    return FA2_ERR_TOO_LARGE;
  // a page's bytes and the keys of a table row in 31 bits
  if (p->page_size > kLim / (p->kv_heads * (p->head_dim / 2)) ||
      (p->table_width > 0 && p->page_size > kLim / p->table_width))
    return FA2_ERR_TOO_LARGE;
  const int64_t strides[] = {p->q_sb, p->q_sh, p->q_ss, p->o_sb, p->o_sh, p->o_ss};
  for (int64_t s : strides)
    if (!stride_ok(s, 2)) return FA2_ERR_ALIGNMENT;
  if (p->q_heads / p->kv_heads > 1 &&
      (p->q_sh != p->q_len * p->q_ss || p->o_sh != p->q_len * p->o_ss))
    return FA2_ERR_Q_LAYOUT;
  return FA2_OK;
}

int fp4_plan(const fa2_fp4_decode_params* p, Fp4Plan* pl) {
  pl->rows = p->q_heads / p->kv_heads * p->q_len;
  if (pl->rows > kLim) return FA2_ERR_TOO_LARGE;
  const int64_t wgs = cu_count_current_device();
  const int64_t tiles = std::max<int64_t>(cdiv(p->table_width * p->page_size, kBN), 1);
  const int64_t total = tiles * p->batch;  // (at most: lengths are on the device)
  if (total >= (int64_t(1) << 30)) return FA2_ERR_TOO_LARGE;
  // More than 16 rows: q-blocks of 32 share K and V, q-blocks of 16 have less to add up
  // (D = 256 has no registers for 32).  16 where every unit of them still has a workgroup
  // and the tables hold kD4Wide tiles per workgroup at most.  20 rows of D128, q-blocks
  // of 16 / 32, us: 8 kv heads, 4 x 1000 keys 10.6 / 14.6, 16 x 2048 (256 units, 16 tiles) 15.7
  // / 19.6, 16 x 8192 (64 tiles) 47 / 39.7, 32 x 1000-3000 (512 units) 37.9 / 35.0; 4 kv heads,
  // 33 x 100-2000 (264 units, 17 tiles) 23.6 / 18.6.
  const bool wide = p->head_dim <= 128 && pl->rows > 16 &&
                    (p->batch * p->kv_heads * cdiv(pl->rows, 16) > wgs ||
                     total * p->kv_heads > kD4Wide * wgs);
  pl->rb = wide ? 2 : 1;
  const int64_t nqb = cdiv(pl->rows, 16 * pl->rb);
  pl->part_rows = std::min<int64_t>(pl->rows, 16 * pl->rb);
  pl->streams = p->kv_heads * nqb;
  pl->segs = std::min(std::max<int64_t>(1, wgs / pl->streams), cdiv(total, kD4GridTiles));
  const int64_t part_bytes = 2 * pl->streams * pl->segs * pl->part_rows * p->head_dim * 4;
  if (part_bytes >= (int64_t(1) << 31) || pl->streams * p->batch > kLim)
    return FA2_ERR_TOO_LARGE;
  const int64_t grid = pl->streams * pl->segs;
  const int64_t idle = std::max<int64_t>(0, grid - pl->streams * p->batch);
  pl->whole = std::max(kD4Whole / 2, kD4Whole * idle / grid);
  const size_t slots = static_cast<size_t>(2 * grid);
  size_t off = static_cast<size_t>(pl->streams * p->batch) * sizeof(uint64_t);
  off = (off + 255) & ~size_t(255);
  pl->off_ml = off;
  off += slots * pl->part_rows * 2 * sizeof(float);
  off = (off + 255) & ~size_t(255);
  pl->off_o = off;
  off += slots * pl->part_rows * p->head_dim * sizeof(float);
  pl->total = off;
  return FA2_OK;
}

bool fp4_empty(const fa2_fp4_decode_params* p) { return p->batch == 0 || p->q_len == 0; }

template <int DT, int D, bool BLOCKS>
void launch_fp4_decode(const Fp4Args& a, int rb, uint32_t grid, hipStream_t st) {
  const dim3 block(kD4Threads);
  if constexpr (D <= 128) {
    if (rb == 2) {
      hipLaunchKernelGGL((fa2_decode_fp4_kernel<DT, D, 2, BLOCKS>), dim3(grid), block, 0, st, a);
      return;
    }
  }
  hipLaunchKernelGGL((fa2_decode_fp4_kernel<DT, D, 1, BLOCKS>), dim3(grid), block, 0, st, a);
}

template <int DT, int D>
void launch_fp4_decode_pages(const Fp4Args& a, int rb, uint32_t grid, hipStream_t st) {
  if (a.a.page_size % 16 == 0)
    launch_fp4_decode<DT, D, true>(a, rb, grid, st);
  else
    launch_fp4_decode<DT, D, false>(a, rb, grid, st);
}

template <int DT>
void launch_fp4_decode_dim(int64_t d, const Fp4Args& a, int rb, uint32_t grid, hipStream_t st) {
  if (d == 64) launch_fp4_decode_pages<DT, 64>(a, rb, grid, st);
  else if (d == 128) launch_fp4_decode_pages<DT, 128>(a, rb, grid, st);
  else launch_fp4_decode_pages<DT, 256>(a, rb, grid, st);
}

}  // namespace
}  // namespace fa2

using namespace fa2;

extern "C" size_t fa2_ops_params_size(int which) {
  switch (which) {
    case 0: return sizeof(fa2_norm_rope_params);
    case 1: return sizeof(fa2_fp4_rows_params);
    case 2: return sizeof(fa2_fp4_decode_params);
    default: return 0;
  }
}

extern "C" int fa2_norm_rope(const fa2_norm_rope_params* p, void* stream) {
  int s = validate_norm_rope(p);
  if (s != FA2_OK) return s;
  if (p->tokens == 0 || p->q_heads + p->kv_heads == 0) return FA2_OK;
  if ((p->q_heads && (!p->q || !p->q_out || !p->q_weight)) ||
      (p->kv_heads && (!p->k || !p->k_out || !p->k_weight)) || !p->position ||
      (p->rotary_dim && p->positions && !p->rope))
    return FA2_ERR_NULL_POINTER;
  const void* ptrs[] = {p->q, p->k, p->q_out, p->k_out, p->q_weight, p->k_weight, p->rope};
  for (const void* x : ptrs)
    if (!aligned16(x)) return FA2_ERR_ALIGNMENT;
  const int eb = elt_bytes(p->dtype);
  const int64_t lanes = p->head_dim * eb / 32;
  // Four heads of a token per lane group (their loads in flight together, the
  // table's row and the weights read once) where that still gives every CU a
  // wave for each of its four SIMDs, else one.
  const int64_t u = p->tokens * (cdiv(p->q_heads, 4) + cdiv(p->kv_heads, 4)) * lanes >=
                            int64_t(cu_count_current_device()) * 4 * 64
                        ? 4
                        : 1;
  NormRopeArgs a{};
  a.x[0] = static_cast<const char*>(p->q);
  a.x[1] = static_cast<const char*>(p->k);
  a.y[0] = static_cast<char*>(p->q_out);
  a.y[1] = static_cast<char*>(p->k_out);
  a.w[0] = static_cast<const char*>(p->q_weight);
  a.w[1] = static_cast<const char*>(p->k_weight);
  a.rope = p->rope;
  a.pos = p->position;
  a.sb[0] = p->q_sb * eb; a.sh[0] = p->q_sh * eb; a.ss[0] = p->q_ss * eb;
  a.sb[1] = p->k_sb * eb; a.sh[1] = p->k_sh * eb; a.ss[1] = p->k_ss * eb;
  a.ob[0] = p->qo_sb * eb; a.oh[0] = p->qo_sh * eb; a.os[0] = p->qo_ss * eb;
  a.ob[1] = p->ko_sb * eb; a.oh[1] = p->ko_sh * eb; a.os[1] = p->ko_ss * eb;
  a.rope_stride = p->rope_stride;
  a.heads[0] = static_cast<int32_t>(p->q_heads);
  a.heads[1] = static_cast<int32_t>(p->kv_heads);
  a.rows[0] = static_cast<int32_t>(p->q_rows);
  a.rows[1] = static_cast<int32_t>(p->k_rows);
  a.blocks[0] = static_cast<int32_t>(cdiv(p->q_heads, u));
  a.blocks[1] = static_cast<int32_t>(cdiv(p->kv_heads, u));
  const int64_t units = p->tokens * (a.blocks[0] + a.blocks[1]);
  if (units * lanes > kLim) return FA2_ERR_TOO_LARGE;
  a.units = static_cast<int32_t>(units);
  a.positions = static_cast<int32_t>(p->positions);
  a.rot = static_cast<int32_t>(p->rotary_dim);
  a.inter = p->interleaved ? 1 : 0;
  a.pos64 = p->position_64 ? 1 : 0;
  a.w32 = p->weight_dtype == FA2_DTYPE_F32 ? 1 : 0;
  a.eps = p->eps;
  const uint32_t grid = static_cast<uint32_t>(cdiv(units * lanes, kNrThreads));
  hipStream_t st = static_cast<hipStream_t>(stream);
  switch (p->dtype) {
    case FA2_DTYPE_F16:
      launch_norm_rope_dim<FA2_DTYPE_F16>(p->head_dim, a, static_cast<int>(u), grid, st);
      break;
    case FA2_DTYPE_BF16:
      launch_norm_rope_dim<FA2_DTYPE_BF16>(p->head_dim, a, static_cast<int>(u), grid, st);
      break;
    default:
      launch_norm_rope_dim<FA2_DTYPE_F32>(p->head_dim, a, static_cast<int>(u), grid, st);
  }
  return launched();
}

extern "C" int fa2_fp4_append(const fa2_fp4_rows_params* p, void* stream) {
  return fp4_rows(p, stream, true);
}

extern "C" int fa2_fp4_gather(const fa2_fp4_rows_params* p, void* stream) {
  return fp4_rows(p, stream, false);
}

extern "C" int fa2_fp4_decode_workspace_size(const fa2_fp4_decode_params* p, size_t* bytes) {
  if (!bytes) return FA2_ERR_NULL_POINTER;
  int s = validate_fp4_decode(p);
  if (s != FA2_OK) return s;
  *bytes = 0;
  if (fp4_empty(p)) return FA2_OK;
  Fp4Plan pl{};
  s = fp4_plan(p, &pl);
  if (s == FA2_OK) *bytes = pl.total;
  return s;
}

extern "C" int fa2_fp4_decode(const fa2_fp4_decode_params* p, void* stream) {
  int s = validate_fp4_decode(p);
  if (s != FA2_OK) return s;
  if (fp4_empty(p)) return FA2_OK;
  if (!p->q || !p->o || !p->k_codes || !p->k_scales || !p->v_codes || !p->v_scales)
    return FA2_ERR_NULL_POINTER;
  if (!p->kv_lens || p->num_pages == 0 ||
      (p->table_width > 0 && (!p->k_block_table || !p->v_block_table)))
    return FA2_ERR_PAGED_ARGS;
  // (the kernel's running maximum is that of q . k, the scores' only for scales above 0)
  if (!(p->softmax_scale > 0.f && std::isfinite(p->softmax_scale))) return FA2_ERR_BAD_SHAPE;
  const void* ptrs[] = {p->q, p->o, p->k_codes, p->v_codes};
  for (const void* x : ptrs)
    if (!aligned16(x)) return FA2_ERR_ALIGNMENT;
  for (const uint8_t* x : {p->k_scales, p->v_scales})  // (read in words)
    if (reinterpret_cast<uintptr_t>(x) % 4) return FA2_ERR_ALIGNMENT;
  Fp4Plan pl{};
  s = fp4_plan(p, &pl);
  if (s != FA2_OK) return s;
  if (!p->workspace || p->workspace_bytes < pl.total) return FA2_ERR_WORKSPACE;
  if (!aligned16(p->workspace)) return FA2_ERR_ALIGNMENT;

  Fp4Args fa{};
  KArgs& a = fa.a;
  a.q = p->q;
  a.k = p->k_codes;
  a.v = p->v_codes;
  a.o = p->o;
  a.kv_indptr = p->kv_lens;
  a.k_table = p->k_block_table;
  a.v_table = p->v_block_table;
  a.q_sb = p->q_sb; a.q_sh = p->q_sh; a.q_ss = p->q_ss;
  a.o_sb = p->o_sb; a.o_sh = p->o_sh; a.o_ss = p->o_ss;
  a.k_table_stride = p->k_table_stride;
  a.v_table_stride = p->v_table_stride;
  a.batch = static_cast<int32_t>(p->batch);
  a.hq = static_cast<int32_t>(p->q_heads);
  a.hkv = static_cast<int32_t>(p->kv_heads);
  a.q_len = static_cast<int32_t>(pl.rows);
  a.kv_len = static_cast<int32_t>(p->table_width * p->page_size);
  a.page_size = static_cast<int32_t>(p->page_size);
  a.mask = p->mask;
  a.num_splits = 1;
  a.scale_log2 = p->softmax_scale * 1.4426950408889634f;
  char* ws = static_cast<char*>(p->workspace);
  a.merge_ctr = reinterpret_cast<uint64_t*>(ws);
  try {
    a.merge_tag = next_merge_tag();
  } catch (...) {  // (no random device: no tag, no call)
    return FA2_ERR_HIP;
  }
  a.part_ml = reinterpret_cast<float*>(ws + pl.off_ml);
  a.part_o = reinterpret_cast<float*>(ws + pl.off_o);
  a.part_rows = static_cast<int32_t>(pl.part_rows);
  a.walk_streams = static_cast<int32_t>(pl.streams);
  a.walk_segs = static_cast<int32_t>(pl.segs);
  a.walk_min = kD4MinTiles;
  a.walk_whole = static_cast<int32_t>(pl.whole);
  a.walk_short = kD4Short;
  const int64_t grid = pl.streams * pl.segs;
  a.walk_dj = static_cast<int32_t>(pl.segs);
  a.walk_ds = 0;
  a.walk_rounds = static_cast<int32_t>(cdiv(pl.streams * p->batch, grid));
  a.pack_m = static_cast<int32_t>(p->q_len);
  a.dv = static_cast<int32_t>(p->head_dim);
  fa.ks = p->k_scales;
  fa.vs = p->v_scales;
  fa.num_pages = static_cast<int32_t>(p->num_pages);
  fa.table_width = static_cast<int32_t>(p->table_width);
  const int64_t d = p->head_dim;
  fa.head_codes = static_cast<uint32_t>(p->page_size * (d / 2));
  fa.head_scales = static_cast<uint32_t>(p->page_size * (d / 32));
  fa.page_codes = static_cast<uint32_t>(p->kv_heads * p->page_size * (d / 2));
  fa.page_scales = static_cast<uint32_t>(p->kv_heads * p->page_size * (d / 32));
  // n / page_size for n < 2^30 as (2 n * page_mul) >> 32 >> page_sh, with page_sh =
  // floor(log2 page_size) and page_mul = ceil(2^(31 + page_sh) / page_size): page_mul
  // is off by less than 1, the quotient by less than n / 2^(31 + page_sh), which is
  // under 1 / page_size since 2^page_sh > page_size / 2
  int sh = 0;
  while ((int64_t(2) << sh) <= p->page_size) ++sh;
  fa.page_sh = static_cast<uint32_t>(sh);
  fa.page_mul = static_cast<uint32_t>(cdiv(int64_t(1) << (31 + sh), p->page_size));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (p->dtype == FA2_DTYPE_F16)
    launch_fp4_decode_dim<FA2_DTYPE_F16>(d, fa, pl.rb, static_cast<uint32_t>(grid), st);
  else
    launch_fp4_decode_dim<FA2_DTYPE_BF16>(d, fa, pl.rb, static_cast<uint32_t>(grid), st);
  return launched();
}
