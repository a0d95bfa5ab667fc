// fa2_latent_prefill.h - the expanded form of latent attention (include/fa2_latent.h).
//
// The two-head kernel (fa2_kernel_pp.h) with its q-blocks in pairs runs it: S gets the
// MFMAs of the shared part's 64 dims, whose tiles have LDS slots of their own (K and V are
// read per head, the shared rows once per head too, from L2).  This file has the
// merge of its splits.
#pragma once

#include "fa2_kernel_pp.h"

namespace fa2 {

// Rows of q-block blockIdx.x % 2 of pair unit blockIdx.x / 2 (combine_row).
template <int DT, int D, int MODE>
__global__ __launch_bounds__(kThreads) void fa2_latent_combine_kernel(KArgs a) {
  const int S = launch_splits(a);
  if (S <= 1) return;  // the forward kernel wrote the output
  const Work w = decode_work<MODE>(a, blockIdx.x >> 1, 2);
  if (!w.valid) return;
  constexpr int kTPR = D / 4;
  const int grp = blockIdx.x & 1;
  const int r = blockIdx.y * kCombineRows<D> + threadIdx.x / kTPR;
  const int col = (threadIdx.x % kTPR) * 4;
  const int qrow = (2 * w.qblk + grp) * kBM + r;
  if (qrow >= w.Lq) return;
  combine_row<DT, D>(a, 2 * w.pair + grp, r, col, S,
                     w.o_base + static_cast<int64_t>(qrow) * a.o_ss + col);
}

}  // namespace fa2
