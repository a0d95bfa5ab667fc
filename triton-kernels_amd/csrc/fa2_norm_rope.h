// fa2_norm_rope.h - RMS norm of each query and key head and the rotation of its
// position, in one pass (include/fa2_ops.h).
//
//   y = x * rsqrt(mean(x^2) + eps) * w;  the first R dims in pairs (a, b):
//   (a cos - b sin, b cos + a sin), cos and sin from row `position` of a table.
//
// Bound by HBM: each value is read once and written once.  A row (one head of
// one token) is held by D / (2 E) lanes (E values = 16 bytes), 2 E values each:
// lane i takes the chunks that are rotated with each other, i and i + R / (2 E) of
// the first R dims (pairs i, i + R/2) or 2 i and 2 i + 1 (neighbouring pairs), the
// lanes behind them two chunks of the dims that are only normalised.  So the
// rotation needs no exchange between lanes, and either order of pairs takes
// the same E cosines and sines.  A lane group takes U heads of a token: their
// loads are in flight together, the table's row and the weights are read once.
// Measured on MI355X, 32 + 8 heads of D128 bf16, us: 64 tokens 4.0 and 512 5.7 (kernel
// traces; the calls are bound by the host), 2048 9.3 (4.6 TB/s), 8192 34.0 (5.05 TB/s; a
// copy of 1 GiB 5.05), calls back to back; fp32 8192 57.3 (5.9 TB/s).
#pragma once

#include "fa2_values.h"

namespace fa2 {

constexpr int kNrThreads = 256;

struct NormRopeArgs {
  const char* x[2];  // q, k
  char* y[2];
  const char* w[2];
  const float* rope;
  const void* pos;  // int32, or int64 where pos64
  int64_t sb[2], sh[2], ss[2];  // byte strides of x: (batch, head, row)
  int64_t ob[2], oh[2], os[2];  // ... and of y
  int64_t rope_stride;          // elements
  int32_t heads[2], rows[2];    // token t is row t % rows of batch t / rows
  int32_t blocks[2];            // lane groups per token
  int32_t units, positions, rot, inter;
  int32_t w32;  // fp32 weights
  int32_t pos64;
  float eps;
};

// PAST: stores past the caches, all dims rotated in pairs (i, i + D / 2) (fa2_ops.hip has the
// rule and what it measured).
template <int DT, int D, int U, bool PAST>
__global__ __launch_bounds__(kNrThreads) void fa2_norm_rope_kernel(NormRopeArgs a) {
  constexpr int E = DT == FA2_DTYPE_F32 ? 4 : 8;
  constexpr int kLanes = D / (2 * E);  // of a row
  const int gid = (blockIdx.x * kNrThreads + threadIdx.x) / kLanes;
  const int lane = threadIdx.x % kLanes;
  if (gid >= a.units) return;  // (whole lane groups)
  const int per = a.blocks[0] + a.blocks[1];
  const int t = gid / per;
  int hb = gid - t * per;
  const int which = hb >= a.blocks[0] ? 1 : 0;
  if (which) hb -= a.blocks[0];
  const int h0 = hb * U;
  const int heads = a.heads[which];
  const int b = t / a.rows[which];
  const int m = t - b * a.rows[which];
  const char* x = a.x[which] + b * a.sb[which] + m * a.ss[which] + h0 * a.sh[which];
  char* y = a.y[which] + b * a.ob[which] + m * a.os[which] + h0 * a.oh[which];

  // this lane's chunks, and its first pair
  const int nrot = a.rot / (2 * E);
  const bool rotated = PAST || lane < nrot, inter = !PAST && a.inter;
  const int c0 = rotated && !inter ? lane : 2 * lane;
  const int c1 = rotated && !inter ? lane + nrot : 2 * lane + 1;

  u32x4 in[U][2];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (h0 + u >= heads) break;
    const char* r = x + u * a.sh[which];
    in[u][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(r + c0 * 16));
    in[u][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(r + c1 * 16));
  }
  const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.pos)[t]
                              : static_cast<const int32_t*>(a.pos)[t];
  float c[E], s[E], w[2 * E];
#pragma unroll
  for (int i = 0; i < E; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  const bool bad = pos < 0 || pos >= a.positions;  // no such row: NaN
  if (rotated && !bad) {
    const float* row = a.rope + pos * a.rope_stride + lane * E;
    const float* row2 = row + a.rot / 2;
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const f32x4 cc = *reinterpret_cast<const f32x4*>(row + i);
      const f32x4 sn = *reinterpret_cast<const f32x4*>(row2 + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        c[i + j] = cc[j];
        s[i + j] = sn[j];
      }
    }
  }
  const char* wp = a.w[which];
  if (DT == FA2_DTYPE_F32 || a.w32) {
#pragma unroll
    for (int i = 0; i < E; i += 4) {
      const f32x4 w0 = *reinterpret_cast<const f32x4*>(wp + (c0 * E + i) * 4);
      const f32x4 w1 = *reinterpret_cast<const f32x4*>(wp + (c1 * E + i) * 4);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        w[i + j] = w0[j];
        w[E + i + j] = w1[j];
      }
    }
  } else {
    unpack16<DT>(*reinterpret_cast<const u32x4*>(wp + c0 * 16), w);
    unpack16<DT>(*reinterpret_cast<const u32x4*>(wp + c1 * 16), w + E);
  }

#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (h0 + u >= heads) break;
    float v[2 * E];
    unpack16<DT>(in[u][0], v);
    unpack16<DT>(in[u][1], v + E);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 2 * E; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
#pragma unroll
    for (int d = 1; d < kLanes; d <<= 1) ss += __shfl_xor(ss, d);
    float r = 1.f / __builtin_sqrtf(ss * (1.f / D) + a.eps);
    if (bad) r = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 2 * E; ++i) v[i] = v[i] * r * w[i];
    // pairs (i, E + i), or neighbours, of the lane's 2 E values
    float z[2 * E];
    if (!rotated) {  // (a rotation by cos 1, sin 0 would spread infinities and NaN)
#pragma unroll
      for (int i = 0; i < 2 * E; ++i) z[i] = v[i];
    } else if (inter) {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        z[2 * i] = v[2 * i] * c[i] - v[2 * i + 1] * s[i];
        z[2 * i + 1] = v[2 * i + 1] * c[i] + v[2 * i] * s[i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < E; ++i) {
        z[i] = v[i] * c[i] - v[E + i] * s[i];
        z[E + i] = v[E + i] * c[i] + v[i] * s[i];
      }
    }
    char* o = y + u * a.oh[which];
    u32x4* o0 = reinterpret_cast<u32x4*>(o + c0 * 16);
    u32x4* o1 = reinterpret_cast<u32x4*>(o + c1 * 16);
    if constexpr (PAST) {
      __builtin_nontemporal_store(pack16<DT>(z), o0);
      __builtin_nontemporal_store(pack16<DT>(z + E), o1);
    } else {
      *o0 = pack16<DT>(z);
      *o1 = pack16<DT>(z + E);
    }
  }
}

}  // namespace fa2
