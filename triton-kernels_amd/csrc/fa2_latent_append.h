// fa2_latent_append.h - new rows of a latent cache: the norm of the latent, the
// rotation of the shared key part, and the copy into the pages (include/fa2_latent.h).
//
//   (c, r) -> (c * rsqrt(mean(c^2) + eps) * weight, r rotated to the row's position)
//
// A copy bound by HBM for many rows and by latency for few.  latent / 8 lanes take a
// row, 16 bytes of the latent each; the first 8 of them also 16 bytes of the rotated
// part, whose pairs (i, i + 32) lie four lanes apart.  The row is loaded first; its
// sequence is found meanwhile by a 64-way search of the prefix sums (one load for
// up to 64 sequences, two up to 4096), then start, table entry and position's angles
// follow one another.  The sum of squares, the norm and the rotation are fp32; each value is
// rounded once, to the row's type.
//
// Measured on MI355X: 64 rows 3.5 us (a launch 2, the rest that chain of loads; 4.0 with the
// host's call), 10754 rows of 16 sequences, rows returned as well, 11.4 (37 MB, 3.3 TB/s; a
// copy of 1 GiB reaches 5.1).
#pragma once

#include "fa2_values.h"

namespace fa2 {

constexpr int kLaThreads = 256;
constexpr int kLaRope = 64;

struct LatentAppendArgs {
  const char* x;
  char* out;    // may be null
  char* cache;
  const char* w;
  const float* rope;
  const int32_t* indptr;
  const int32_t* start;  // may be null
  const int32_t* table;
  int64_t x_ts, rope_stride, table_stride;  // bytes, elements, elements
  int32_t batch, num_rows, page_size, num_pages, table_width, positions;
  int32_t inter, w32;
  float eps;
};

// The sequence b of row t (uniform over the wave): how many of indptr[1 ..] are at
// most t; a.batch past the last.
__device__ __forceinline__ int latent_sequence(const LatentAppendArgs& a, int t) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = a.batch;
  while (n > 64) {
    const int step = (n + 63) >> 6;
    const int e = a.indptr[lo + min((lane + 1) * step, n)];
    const int c = __popcll(__ballot(e <= t));  // (c * step >= n: all of them)
    const int at = min(c * step, n);
    lo += at;
    n = min(step, n - at);
  }
  const int e = lane < n ? a.indptr[lo + 1 + lane] : INT32_MAX;
  return lo + __popcll(__ballot(e <= t));
}

template <int DT, int R>
__global__ __launch_bounds__(kLaThreads) void fa2_latent_append_kernel(LatentAppendArgs a) {
  constexpr int kLanes = R / 8;          // of a row
  constexpr int kRows = 64 / kLanes;     // rows of a wave
  constexpr int kWidth = (R + kLaRope) * 2;
  const int lane = threadIdx.x & 63;
  const int li = lane % kLanes;
  const int t0 = (blockIdx.x * (kLaThreads / 64) + (threadIdx.x >> 6)) * kRows;
  const int t = t0 + lane / kLanes;
  const bool in = t < a.num_rows;
  const bool tail = li < 8;

  const char* src = a.x + (in ? t : 0) * a.x_ts;
  const u32x4 xc = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + li * 16));
  const u32x4 xr = __builtin_nontemporal_load(
      reinterpret_cast<const u32x4*>(src + R * 2 + (li & 7) * 16));
  float w[8];
  if (a.w32) {
    unpack16<FA2_DTYPE_F32>(*reinterpret_cast<const u32x4*>(a.w + li * 32), w);
    unpack16<FA2_DTYPE_F32>(*reinterpret_cast<const u32x4*>(a.w + li * 32 + 16), w + 4);
  } else {
    unpack16<DT>(*reinterpret_cast<const u32x4*>(a.w + li * 16), w);
  }

  int b = latent_sequence(a, t0);
  if constexpr (kRows == 2) {
    const int b1 = latent_sequence(a, t0 + 1);
    b = lane / kLanes ? b1 : b;
  }
  bool held = in && b < a.batch;
  const int first = held ? a.indptr[b] : 0;
  const int64_t n = held ? (a.start ? a.start[b] : 0) + static_cast<int64_t>(t - first) : 0;
  held = held && t >= first;  // (before the first sequence: no row)
  const bool known = n >= 0 && n < a.positions;
  int64_t at = -1;
  if (held && n >= 0) {
    const int64_t lp = n / a.page_size;
    if (lp < a.table_width) {
      const int64_t pg = a.table[b * a.table_stride + lp];
      if (pg >= 0 && pg < a.num_pages) at = pg * a.page_size + (n - lp * a.page_size);
    }
  }

  // the latent's norm
  float c[8];
  unpack16<DT>(xc, c);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(c[i], c[i], ss);
#pragma unroll
  for (int d = 1; d < kLanes; d <<= 1) ss += __shfl_xor(ss, d);
  float r = 1.f / __builtin_sqrtf(ss * (1.f / R) + a.eps);
  if (!known) r = __builtin_nanf("");
#pragma unroll
  for (int i = 0; i < 8; ++i) c[i] = c[i] * r * w[i];

  // the rotation: lanes 0 .. 7 hold 8 values each (the others repeat them)
  float x[8], z[8];
  unpack16<DT>(xr, x);
  const int k = li & 7;
  const float* row = a.rope + (known ? n : 0) * a.rope_stride;
  const float bad = known ? 0.f : __builtin_nanf("");
  if (a.inter) {  // pairs 4 k ..+3
    f32x4 cs = (f32x4){bad, bad, bad, bad}, sn = cs;
    if (known) {
      cs = *reinterpret_cast<const f32x4*>(row + 4 * k);
      sn = *reinterpret_cast<const f32x4*>(row + kLaRope / 2 + 4 * k);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      z[2 * i] = x[2 * i] * cs[i] - x[2 * i + 1] * sn[i];
      z[2 * i + 1] = x[2 * i + 1] * cs[i] + x[2 * i] * sn[i];
    }
  } else {  // pairs 8 (k % 4) ..+7, first members in lanes 0 .. 3
    const float sign = k < 4 ? -1.f : 1.f;
    f32x4 cs[2], sn[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      cs[h] = sn[h] = (f32x4){bad, bad, bad, bad};
      if (known) {
        cs[h] = *reinterpret_cast<const f32x4*>(row + 8 * (k & 3) + 4 * h);
        sn[h] = *reinterpret_cast<const f32x4*>(row + kLaRope / 2 + 8 * (k & 3) + 4 * h);
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float other = __shfl_xor(x[i], 4);
      z[i] = x[i] * cs[i >> 2][i & 3] + sign * other * sn[i >> 2][i & 3];
    }
  }

  const u32x4 yc = pack16<DT>(c), yr = pack16<DT>(z);
  if (held && at >= 0) {
    char* dst = a.cache + at * kWidth;
    *reinterpret_cast<u32x4*>(dst + li * 16) = yc;
    if (tail) *reinterpret_cast<u32x4*>(dst + R * 2 + k * 16) = yr;
  }
  if (held && a.out) {
    char* dst = a.out + static_cast<int64_t>(t) * kWidth;
    *reinterpret_cast<u32x4*>(dst + li * 16) = yc;
    if (tail) *reinterpret_cast<u32x4*>(dst + R * 2 + k * 16) = yr;
  }
}

}  // namespace fa2
