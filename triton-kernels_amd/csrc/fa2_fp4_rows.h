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
// indptr in LDS, one lane per row, then all lanes copy.
#pragma once

#include "fa2_device.h"

namespace fa2 {

constexpr int kF4Rows = 64;      // rows per workgroup at most
constexpr int kF4Indptr = 512;   // sequences whose indptr fits LDS
constexpr int kF4Threads = 256;
constexpr int kF4Pieces = 512;   // code words of K (and of V) per workgroup

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
  int32_t block_rows;    // rows per workgroup, <= kF4Rows
  int32_t word_shift;    // log2 of the code words of a head
  int32_t has_v;
};

// Cache row of each of the workgroup's rows in LDS: page * P * H + place in the
// page (the head adds head * P); -1: no such row, -2: the row has no page.
__device__ __forceinline__ void fp4_locate(const Fp4RowsArgs& a, int r0, int64_t (*at)[kF4Rows],
                                           int* ip_sh) {
  const int tid = threadIdx.x;
  const bool staged = a.batch <= kF4Indptr;
  if (staged) {
    for (int i = tid; i <= a.batch; i += kF4Threads) ip_sh[i] = a.indptr[i];
    __syncthreads();
  }
  const int* ip = staged ? ip_sh : a.indptr;
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
        const int64_t n = (a.start ? a.start[lo] : 0) + static_cast<int64_t>(j);
        const int64_t lp = a.page_shift >= 0 ? n >> a.page_shift : n / a.page_size;
        const bool in = n >= 0 && lp < a.table_width;
        const int64_t off = n - lp * a.page_size;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          pos[v] = -2;
          if (!in || (v && !a.has_v)) continue;
          const int64_t pg = a.table[v][lo * a.table_stride[v] + lp];
          if (pg >= 0 && pg < a.num_pages) pos[v] = pg * a.page_size * a.heads + off;
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

template <int DT>
__device__ __forceinline__ void fp4_unpack8(const u32x4* r, float* x) {
  if constexpr (DT == FA2_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint32_t w = r[i / 4][i % 4];
      x[i] = __builtin_bit_cast(float, w);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t w = r[0][i];
      if constexpr (DT == FA2_DTYPE_BF16) {
        x[2 * i] = __builtin_bit_cast(float, w << 16);
        x[2 * i + 1] = __builtin_bit_cast(float, w & 0xFFFF0000u);
      } else {
        const f32x2 f = __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
        x[2 * i] = f[0];
        x[2 * i + 1] = f[1];
      }
    }
  }
}

template <int DT>
__global__ __launch_bounds__(kF4Threads) void fa2_fp4_append_kernel(Fp4RowsArgs a) {
  constexpr int kW = DT == FA2_DTYPE_F32 ? 2 : 1;  // 16-byte loads of 8 values
  __shared__ int64_t at[2][kF4Rows];
  __shared__ int ip_sh[kF4Indptr + 1];
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * a.block_rows;
  fp4_locate(a, r0, at, ip_sh);
  const int rows = min(a.block_rows, a.num_rows - r0);
  const int total = rows * a.words;
  constexpr int kUnroll = kF4Pieces / kF4Threads;
  for (int base = 0; base < total; base += kF4Threads * kUnroll) {
    u32x4 in[kUnroll][2][kW];
    int64_t to[kUnroll][2];  // code word's index
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int idx = base + u * kF4Threads + tid;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        to[u][v] = -1;
#pragma unroll
        for (int i = 0; i < kW; ++i) in[u][v][i] = (u32x4){0u, 0u, 0u, 0u};
      }
      if (idx < total) {
        const int r = idx / a.words;
        const int c = idx - r * a.words;
        const int h = c >> a.word_shift;
        const int w = c & ((1 << a.word_shift) - 1);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int64_t p = at[v][r];
          if (p < 0) continue;
          const char* s = a.x[v] + static_cast<int64_t>(r0 + r) * a.ts[v] + h * a.hs[v] +
                          w * (16 * kW);
#pragma unroll
          for (int i = 0; i < kW; ++i)
            in[u][v][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(s) + i);
          to[u][v] = ((p + static_cast<int64_t>(h) * a.page_size) << a.word_shift) + w;
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        float x[8];
        fp4_unpack8<DT>(in[u][v], x);
        // (the lanes of a block take part together: `words` is a multiple of 4)
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          top = max(top, __builtin_bit_cast(uint32_t, x[i]) & 0x7FFFFFFFu);
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 1)));
        top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 2)));
        const uint32_t sb = fp4_scale<DT>(top);
        const float f = __builtin_bit_cast(float, sb << 23);
        uint32_t code = 0;
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[0], x[1], f, 0);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[2], x[3], f, 1);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[4], x[5], f, 2);
        code = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(code, x[6], x[7], f, 3);
        if (sb == 255) code = 0;
        if (to[u][v] >= 0) {
          reinterpret_cast<uint32_t*>(a.codes[v])[to[u][v]] = code;
          if ((to[u][v] & 3) == 0) a.scales[v][to[u][v] >> 2] = static_cast<uint8_t>(sb);
        }
      }
    }
  }
}

// The 8 values of a code word in DT at 2^(sb - 127)
template <int DT>
__device__ __forceinline__ void fp4_expand8(uint32_t w, uint32_t sb, u32x4* r) {
  const float f = __builtin_bit_cast(float, sb << 23);
  if constexpr (DT == FA2_DTYPE_BF16) {
    r[0] = (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3))};
  } else if constexpr (DT == FA2_DTYPE_F16) {
    r[0] = (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 3))};
  } else {
    const f32x2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 0);
    const f32x2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 1);
    const f32x2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 2);
    const f32x2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, f, 3);
    r[0] = __builtin_bit_cast(u32x4, (f32x4){x0[0], x0[1], x1[0], x1[1]});
    r[1] = __builtin_bit_cast(u32x4, (f32x4){x2[0], x2[1], x3[0], x3[1]});
  }
}

template <int DT>
__global__ __launch_bounds__(kF4Threads) void fa2_fp4_gather_kernel(Fp4RowsArgs a) {
  constexpr int kW = DT == FA2_DTYPE_F32 ? 2 : 1;
  __shared__ int64_t at[2][kF4Rows];
  __shared__ int ip_sh[kF4Indptr + 1];
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * a.block_rows;
  fp4_locate(a, r0, at, ip_sh);
  const int rows = min(a.block_rows, a.num_rows - r0);
  const int total = rows * a.words;
  constexpr int kUnroll = kF4Pieces / kF4Threads;
  for (int base = 0; base < total; base += kF4Threads * kUnroll) {
    uint32_t code[kUnroll][2], sb[kUnroll][2];
    char* to[kUnroll][2];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int idx = base + u * kF4Threads + tid;
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        to[u][v] = nullptr;
        code[u][v] = 0;
        sb[u][v] = 127;
      }
      if (idx < total) {
        const int r = idx / a.words;
        const int c = idx - r * a.words;
        const int h = c >> a.word_shift;
        const int w = c & ((1 << a.word_shift) - 1);
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const int64_t p = at[v][r];
          if (p == -1 || (v && !a.has_v)) continue;
          to[u][v] = a.x[v] + static_cast<int64_t>(r0 + r) * a.ts[v] + h * a.hs[v] + w * (16 * kW);
          if (p < 0) continue;  // no page: zeros
          const int64_t i = ((p + static_cast<int64_t>(h) * a.page_size) << a.word_shift) + w;
          code[u][v] = reinterpret_cast<const uint32_t*>(a.codes[v])[i];
          sb[u][v] = a.scales[v][i >> 2];
        }
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u)
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        if (!to[u][v]) continue;
        u32x4 r[kW];
        fp4_expand8<DT>(code[u][v], sb[u][v], r);
#pragma unroll
        for (int i = 0; i < kW; ++i) reinterpret_cast<u32x4*>(to[u][v])[i] = r[i];
      }
  }
}

}  // namespace fa2
