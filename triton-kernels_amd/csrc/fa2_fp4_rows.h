// fa2_fp4_rows.h - rows into and out of a paged cache held in 4 bits
// (include/fa2_ops.h): quantise and write, read and expand.
//
// Row t of a ragged [T, H, D] tensor is row j = t - indptr[b] of its sequence b, at
// logical position n = start[b] + j: row n % P of page table[b][n / P].  The 32
// values of a block share the power of two 2^e that keeps the largest, a,
// within the code range after rounding (a / 2^e < 7, code 6 at most):
//   e = floor(log2 a) - 2, one more where a >= 1.75 * 2^floor(log2 a),
// kept in a range where every value of the cache is exact in the row's type.
// v_cvt_scalef32_pk_fp4_f32 rounds x / 2^e to the nearest code, ties to even,
// and saturates at 6.  A block that holds an infinity or NaN is NaN (scale 255).
//
// Both are copies bound by HBM: rows are touched once in 16 or 32 bits and once
// in 4.25.  A thread takes 8 values (a code word), four neighbouring lanes a block:
// its maximum is two quad exchanges.  Rows are located as in fa2_kv_append.h:
// indptr and the starts in LDS, one lane per row; a thread takes a column of its own of
// four rows, which the writer loads before their places are known (64 rows 5.25 -> 4.95
// us; 10.7 k rows the same).  The cache's side goes in whole blocks: lane i of a quad
// moves the four words of the block in row i, and a 4 x 4 transpose within the quad
// (DPP) turns them from or into a word of each row.  (A word and a scale byte per
// lane and row takes three memory instructions for each KB of rows, not 1.5.)
// Measured on MI355X, 8 heads of D128 bf16: 156 k rows gathered in 139.6 us (5.8 TB/s; a copy
// of 1 GiB 5.05), calls back to back; by kernel traces, 10.7 k rows appended in 14.8 and
// gathered in 12.1 (3.8 and 4.6 TB/s: one latency after another, all workgroups at once),
// 64 rows in 5.0 and 4.8.  fp32: 156 k rows gathered in 285 (5.1 TB/s), 10.7 k appended in 22.
// At 8 waves per SIMD, where 156 k rows take 152 us, a word at a time took 178 and
// workgroups of 8 / 12 / 16 rows per thread 154 / 162 / 163.
// Gathered rows of 16 bits are stored non-temporally (156 k rows 157.5 -> 139.6 us; with
// attention of 16 queries per sequence after it 372 -> 375, which would rather find them
// in the caches: 17 k rows 53.5 -> 54.5, 2 k rows and 64 queries 30.4 -> 33.3), fp32 rows
// through the caches (156 k rows 558 -> 285).
#pragma once

#include "fa2_values.h"

namespace fa2 {

constexpr int kF4Rows = 128;     // rows per workgroup at most
constexpr int kF4Indptr = 512;   // sequences whose indptr fits LDS
constexpr int kF4Threads = 256;

struct Fp4RowsArgs {
  char* x[2];        // rows of K and V (append: read; gather: written)
  uint8_t* codes[2];
  uint8_t* scales[2];
  const int32_t* table[2];
  int64_t table_stride[2];
  int64_t ts[2], hs[2];  // byte strides (row, head) of x
  const int32_t* indptr;
  const int32_t* start;  // may be null: every sequence starts at 0
  int32_t batch, heads, words, num_rows, page_size, page_shift, num_pages, table_width;
  int32_t block_rows;    // rows per workgroup: 4 * rows_at_once, <= kF4Rows
  int32_t rows_at_once;  // rows that the workgroup's threads cover, one word each
  int32_t word_shift;    // log2 of the code words of a head
  int32_t has_v;
};

// Lane i of a quad gives w[j] to lane j, as its w[i].
__device__ __forceinline__ void quad_transpose(uint32_t (&w)[4]) {
  const int lane = threadIdx.x;
  auto swap = [](uint32_t& keep_a, uint32_t& keep_b, bool high, auto ctrl) {
    // low lanes send b and receive it from the high lanes' a
    const uint32_t send = high ? keep_a : keep_b;
    const uint32_t got = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
        0, static_cast<int>(send), decltype(ctrl)::value, 0xF, 0xF, true));
    if (high)
      keep_a = got;
    else
      keep_b = got;
  };
  using Xor1 = std::integral_constant<int, 0xB1>;
  using Xor2 = std::integral_constant<int, 0x4E>;
  swap(w[0], w[1], lane & 1, Xor1{});
  swap(w[2], w[3], lane & 1, Xor1{});
  swap(w[0], w[2], lane & 2, Xor2{});
  swap(w[1], w[3], lane & 2, Xor2{});
}
// The value of lane J of the quad.
template <int J>
__device__ __forceinline__ uint32_t quad_lane(uint32_t x) {
  return static_cast<uint32_t>(
      __builtin_amdgcn_update_dpp(0, static_cast<int>(x), J * 0x55, 0xF, 0xF, true));
}

// Offset of each of the workgroup's rows in the codes, head 0, in LDS; -1: no such
// row, -2: the row has no page.  `meanwhile` runs while the prefix sums are on their way.
template <typename F>
__device__ __forceinline__ void fp4_locate(const Fp4RowsArgs& a, int r0, int64_t (*at)[kF4Rows],
                                           int (*sh)[kF4Indptr + 1], F meanwhile) {
  const int tid = threadIdx.x;
  const bool staged = a.batch <= kF4Indptr;
  auto start_of = [&](int b) { return a.start && b < a.batch ? a.start[b] : 0; };
  int ip0 = 0, st0 = 0;
  if (staged && tid <= a.batch) {
    ip0 = a.indptr[tid];
    st0 = start_of(tid);
  }
  meanwhile();
  if (staged) {
    if (tid <= a.batch) {
      sh[0][tid] = ip0;
      sh[1][tid] = st0;
    }
    for (int i = tid + kF4Threads; i <= a.batch; i += kF4Threads) {
      sh[0][i] = a.indptr[i];
      sh[1][i] = start_of(i);
    }
    __syncthreads();
  }
  const int* ip = staged ? sh[0] : a.indptr;
  if (tid < a.block_rows) {
    const int t = r0 + tid;
    int64_t pos[2] = {-1, -1};
    if (t < a.num_rows) {
      int lo = 0, hi = a.batch - 1;  // the last b with indptr[b] <= t
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (ip[mid] <= t) lo = mid;
        else hi = mid - 1;
      }
      const int j = t - ip[lo];
      if (j >= 0 && t < ip[lo + 1]) {
        const int64_t n = (staged ? sh[1][lo] : start_of(lo)) + static_cast<int64_t>(j);
        const int64_t lp = a.page_shift >= 0 ? n >> a.page_shift : n / a.page_size;
        const bool in = n >= 0 && lp < a.table_width;
        const int64_t off = n - lp * a.page_size;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          pos[v] = -2;
          if (!in || (v && !a.has_v)) continue;
          const int64_t pg = a.table[v][lo * a.table_stride[v] + lp];
          if (pg >= 0 && pg < a.num_pages)
            pos[v] = (pg * a.page_size * a.heads + off) << (a.word_shift + 2);
        }
      }
    }
    at[0][tid] = pos[0];
    at[1][tid] = pos[1];
  }
  __syncthreads();
}

// E8M0 byte of a block whose largest magnitude has the fp32 bits `bits`
template <int DT>
__device__ __forceinline__ uint32_t fp4_scale(uint32_t bits) {
  constexpr int lo = DT == FA2_DTYPE_F16 ? 127 - 23 : 127 - 100;
  constexpr int hi = DT == FA2_DTYPE_F16 ? 127 + 13 : 127 + 125;
  const int ex = static_cast<int>(bits >> 23);
  if (ex == 255) return 255;
  const int e = ex - 2 + ((bits & 0x7FFFFFu) >= 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(min(max(e, lo), hi));
}

// This thread's words: column `col` of rows `first`, first + step, ...; columns
// cols ... further where a row has more words than the workgroup threads.
struct Fp4Share {
  int first, step, col;
  uint32_t code;  // its block's offset in a row's codes
};
__device__ __forceinline__ Fp4Share fp4_share(const Fp4RowsArgs& a, int col0) {
  Fp4Share s;
  const int tid = threadIdx.x;
  s.first = a.rows_at_once > 1 ? tid / a.words : 0;
  s.col = tid - s.first * a.words + col0;
  s.step = a.rows_at_once;
  if (s.first >= a.rows_at_once || s.col >= a.words) s.first = kF4Rows;  // none
  const int h = s.col >> a.word_shift;
  s.code = static_cast<uint32_t>(h * a.page_size << (a.word_shift + 2)) +
           (s.col & ((1 << a.word_shift) - 4)) * 4;
  return s;
}

template <int DT>
__global__ __launch_bounds__(kF4Threads) void fa2_fp4_append_kernel(Fp4RowsArgs a) {
  constexpr int kW = DT == FA2_DTYPE_F32 ? 2 : 1;  // 16-byte loads of 8 values
  __shared__ int64_t at[2][kF4Rows];
  __shared__ int sh[2][kF4Indptr + 1];
  const int r0 = blockIdx.x * a.block_rows;
  const int rows = min(a.block_rows, a.num_rows - r0);
  u32x4 in[4][2][kW];
  Fp4Share s;
  auto load = [&](int col0) {  // this thread's word of four rows of K and V
    s = fp4_share(a, col0);
    const int h = s.col >> a.word_shift, w = s.col & ((1 << a.word_shift) - 1);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = u * s.step + s.first;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const char* src =
            a.x[v] + static_cast<int64_t>(r0 + r) * a.ts[v] + h * a.hs[v] + w * (16 * kW);
#pragma unroll
        for (int i = 0; i < kW; ++i) in[u][v][i] = (u32x4){0u, 0u, 0u, 0u};
        if (r < rows && (v == 0 || a.has_v))
#pragma unroll
          for (int i = 0; i < kW; ++i)
            in[u][v][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src) + i);
      }
    }
  };
  // (the rows are read whether they have a place or not: their loads need not wait for it)
  fp4_locate(a, r0, at, sh, [&] { load(0); });
  for (int col0 = 0;;) {
    // (all threads go round together: the lanes of a quad exchange values)
    const int own = (threadIdx.x & 3) * s.step + s.first;  // the row this lane writes
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      uint32_t code[4], scale = 0;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float x[8];
#pragma unroll
        for (int i = 0; i < kW; ++i) unpack16<DT>(in[u][v][i], x + 8 / kW * i);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          top = max(top, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
        top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
                           0, static_cast<int>(top), 0xB1, 0xF, 0xF, true)));
        top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(
                           0, static_cast<int>(top), 0x4E, 0xF, 0xF, true)));
        const uint32_t sb = fp4_scale<DT>(top);
        const float f = __builtin_bit_cast(float, sb << 23);
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], f, 3);
        code[u] = sb == 255 ? 0 : c;
        scale = (threadIdx.x & 3) == u ? sb : scale;
      }
      quad_transpose(code);
      const int64_t p = own < rows ? at[v][own] : -1;
      if (p >= 0) {
        const int64_t c = p + s.code;
        *reinterpret_cast<u32x4*>(a.codes[v] + c) = (u32x4){code[0], code[1], code[2], code[3]};
        a.scales[v][c >> 4] = static_cast<uint8_t>(scale);
      }
    }
    col0 += kF4Threads;
    if (col0 >= a.words) break;
    load(col0);
  }
}

// The 8 values of a code word in DT at 2^(sb - 127)
template <int DT>
__device__ __forceinline__ void fp4_expand8(uint32_t w, uint32_t sb, u32x4* r) {
  if constexpr (DT != FA2_DTYPE_F32) {
    r[0] = fp4_values<DT == FA2_DTYPE_BF16>(w, sb);
  } else {
    const float f = __builtin_bit_cast(float, sb << 23);
    const f32x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 0);
    const f32x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 1);
    const f32x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 2);
    const f32x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 3);
    r[0] = __builtin_bit_cast(u32x4, (f32x4){x0[0], x0[1], x1[0], x1[1]});
    r[1] = __builtin_bit_cast(u32x4, (f32x4){x2[0], x2[1], x3[0], x3[1]});
  }
}

// WAVES: at most so many waves per SIMD (fa2_ops.hip has the rule and what it measured).
template <int DT, int WAVES>
__global__ __launch_bounds__(kF4Threads) __attribute__((amdgpu_waves_per_eu(1, WAVES))) void
fa2_fp4_gather_kernel(Fp4RowsArgs a) {
  constexpr int kW = DT == FA2_DTYPE_F32 ? 2 : 1;
  __shared__ int64_t at[2][kF4Rows];
  __shared__ int sh[2][kF4Indptr + 1];
  const int r0 = blockIdx.x * a.block_rows;
  fp4_locate(a, r0, at, sh, [] {});
  const int rows = min(a.block_rows, a.num_rows - r0);
  for (int col0 = 0; col0 < a.words; col0 += kF4Threads) {
    const Fp4Share s = fp4_share(a, col0);
    const int h = s.col >> a.word_shift, w = s.col & ((1 << a.word_shift) - 1);
    char* dst[2];
#pragma unroll
    for (int v = 0; v < 2; ++v)
      dst[v] = a.x[v] + static_cast<int64_t>(r0 + s.first) * a.ts[v] + h * a.hs[v] + w * (16 * kW);
    const int own = (threadIdx.x & 3) * s.step + s.first;  // the row this lane reads
    uint32_t code[2][4], scale[2];
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      const int64_t p = own < rows ? at[v][own] : -1;
      u32x4 x = (u32x4){0u, 0u, 0u, 0u};  // (no page: zeros)
      scale[v] = 127;
      if (p >= 0) {
        const int64_t c = p + s.code;
        x = *reinterpret_cast<const u32x4*>(a.codes[v] + c);
        scale[v] = a.scales[v][c >> 4];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) code[v][i] = x[i];
    }
#pragma unroll
    for (int v = 0; v < 2; ++v) {
      quad_transpose(code[v]);
      const uint32_t sb[4] = {quad_lane<0>(scale[v]), quad_lane<1>(scale[v]),
                              quad_lane<2>(scale[v]), quad_lane<3>(scale[v])};
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int r = u * s.step + s.first;
        u32x4 x[kW];
        fp4_expand8<DT>(code[v][u], sb[u], x);
        if (r < rows && at[v][r] != -1 && (v == 0 || a.has_v))
#pragma unroll
          for (int i = 0; i < kW; ++i)
          {
            // fp32: a lane's 32 bytes leave as two stores, which past the caches would
            // be half lines each
            u32x4* d = reinterpret_cast<u32x4*>(dst[v]) + i;
            if constexpr (kW == 1)
              __builtin_nontemporal_store(x[i], d);
            else
              *d = x[i];
          }
        dst[v] += s.step * a.ts[v];
      }
    }
  }
}

}  // namespace fa2
