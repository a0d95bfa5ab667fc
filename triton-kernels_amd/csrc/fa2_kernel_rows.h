// fa2_kernel_rows.h - decode attention with many query rows per K/V row: the
// absorbed form of latent attention (every head reads the same cached row) and
// trees of drafts over 16-bit K/V caches.
//
//   s_rn = scale q_r . k_n (n visible to r),  p_rn = exp(s_rn - m_r),
//   o_r = sum_n p_rn v_n / sum_n p_rn
//
// The rows of a unit (sequence, kv head) are its heads times its tokens: up to 128 in
// latent attention's decode step, 8 to 16 times the decode kernels'.  Latent attention:
// k_n is the whole cached row (DK = latent + 64), v_n its first DV = latent values, so a
// row is read once for both products, from one LDS tile.  Per key the kernel reads
// 2 DK (+ 2 DV) bytes and does 2 (DK + DV) FLOP a row: 16 rows of a latent are bound by
// HBM, 128 rows (242 FLOP a byte) by neither alone, so loads and MFMAs have to overlap.
//   * Workgroup = 4 waves.  RG row groups of 32 rows: a wave takes one of them and all
//     DV dims (RG = 4), half (2) or a quarter (1) of them, S computed by each.  Up to 16
//     rows: fa2_kernel_rows16.h.
//   * S^T = K Q^T and O^T += V^T P^T by v_mfma_f32_32x32x16, so that a lane holds one
//     row's scores: the softmax needs one cross-lane step, and P^T is the second
//     product's operand as it lies in the registers.  V^T by ds_read_b64_tr_b16.
//   * Tiles of 32 or 64 keys go straight to LDS (global_load_lds), 3 to 6 slots a
//     workgroup, in groups of 8 rows whose base is a scalar: a page of 8 rows or more costs
//     one block-table entry of LDS and no vector address.  The loads of a tile stand between
//     the MFMAs of S.
//   * fp32 scores, maxima, sums and O; the weights are rounded once, to the tensors' type,
//     for the second product, and summed as rounded.  The maximum is raised when a score
//     passes it by 2^8 only, so fp16 weights, lifted by 2^7, end at 2^15.
//   * Workgroups share the tiles evenly (fa2_decode_walk.h, rows_locate); a unit cut by
//     segments leaves fp32 partials, which a second launch merges in piece order
//     (fa2_rows_merge_kernel): no atomics, the same bits every time.
//
// Measured on MI355X, us per call: 64 latents of 512-8192 keys, 128 heads 128 to 131 (605
// TFLOP/s, 2.6 TB/s; MFMAs busy for 29 % of the cycles, as S, softmax and PV of a tile follow one
// another on one wave per SIMD; the kernel alone takes 116 in the first calls of a loop and 131
// after 50), 17 trees of 7 drafts over latents of 256 values 48, 64 trees of 16 drafts Hq32/Hkv8
// D128 207 (4.7 TB/s), 16 trees of 61 drafts 114 to 118 (610 TFLOP/s, MFMAs busy for 31 %).
#pragma once

#include "fa2_decode_walk.h"
#include "fa2_kernel_pp.h"

namespace fa2 {

constexpr int kRbWaves = 4;
constexpr int kRbThreads = 64 * kRbWaves;
constexpr int kRbTable = 2048;  // block-table entries in LDS (K and V share them)
constexpr int kRbMaxTree = 64;  // drafts of a tree: bits of a mask word

// Mask of a call beyond enum fa2_mask: the drafts that each draft sees.
constexpr int kMaskTree = 3;

// A second piece of a workgroup costs about as much as this many tiles of kBN keys (1 to 6
// measure the same; with 0, 17 trees of 7 drafts take 59 us instead of 53 in the same run, 16
// latents of 16000-32768 keys 91 instead of 88).
constexpr int kRbSwitch = 2;

struct RowsArgs {
  KArgs a;  // q rows: token m of head h at h * q_sh + m * q_ss; o rows: o_ss apart
  int2* info;  // of each unit: its pieces and the part slot of the first (rows_info)
  const uint8_t* tree;  // bool [batch, pack_m, pack_m]
  int64_t tree_sb, tree_sr;
  int32_t num_pages;
  uint32_t page_mul, page_sh;  // n / page_size = umulhi(2 n, page_mul) >> page_sh, n < 2^30
};

// Rows of DK values in LDS: 16-byte chunks, chunk c of row r at c ^ swz(r) (in groups
// of 8 chunks, or of 16 where a row is a multiple of 256 bytes).  Bits of r run
// backwards through the swizzle, so that both reads hit distinct banks: 16 rows at one
// chunk (K, one row per lane) and 4 rows at 4 neighbouring chunks (V, transposed).
template <int DK>
struct RowsGeo {
  static constexpr int kNC = DK / 8;  // chunks of a row
  static constexpr int kRowBytes = DK * 2;
  static constexpr bool kWide = kNC % 16 == 0;
  static constexpr int kGI = kNC / 8;  // 1 KB loads of 8 rows
  static_assert(kNC % 8 == 0, "rows of whole swizzle groups");
  static constexpr int kG = kWide ? 8 : 4;  // 32-byte steps of a swizzle group
  __device__ __forceinline__ static uint32_t swz(int r) {
    return kWide ? ((r & 1) << 3) | ((r & 2) << 1) | ((r & 4) >> 1) | ((r & 8) >> 3)
                 : ((r & 2) << 1) | ((r & 4) >> 1) | ((r & 8) >> 3);
  }
};

// Tile shape: workgroups per CU, keys of a tile and LDS slots.  Two workgroups where their
// tiles fit the CU's 160 KB and the registers 256 a lane: one's softmax runs under the other's
// MFMAs.
template <int DK, int DV, bool LAT, int RG>
struct RowsTile {
  using G = RowsGeo<DK>;
  static constexpr int kRow = G::kRowBytes + (LAT ? 0 : DV * 2);
  static constexpr int kOcc = kRow > 640 || (LAT && RG == 4) ? 1 : 2;
  static constexpr int kBudget = kOcc == 2 ? 70000 : 150000;
  static constexpr int kKeys = kRow * 64 * 4 <= kBudget ? 64 : 32;
  static constexpr int kSlot = kRow * kKeys;
  static constexpr int kSlots = kBudget / kSlot < 6 ? kBudget / kSlot : 6;
  static_assert(kSlots >= 3, "tiles in flight");
};

struct RowsPiece {
  int b, kvh, qblk, Lk;
  int t0, T;     // first tile of kBN keys and their count
  int np, mine;  // pieces of the unit, this one's index
  int us, W, unit;
};

// A workgroup's segment and, for batches of up to 64, every length in the lanes of each
// wave (which then locates the segment by itself: one load, no barrier, no load per piece).
struct RowsWalk {
  DecSegment sg;
  int lens;
  bool in_lanes;
  bool aligned;  // units start at segments: they take whole segments of the stream
};

// walk_locate's rule; sh: LDS.  Every thread of the workgroup.
template <int LM>
__device__ __forceinline__ RowsWalk rows_locate(const KArgs& a, int k, DecSegment* sh) {
  RowsWalk w;
  const int lane = threadIdx.x & 63;
  w.in_lanes = a.batch <= 64;
  w.aligned = false;
  w.lens = 0;
  if (!w.in_lanes) {
    if (threadIdx.x < 64) walk_locate<LM>(a, k, sh);
    __syncthreads();
    auto rd = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    w.sg = DecSegment{rd(sh->j), rd(sh->us), rd(sh->s0), rd(sh->s1), rd(sh->C)};
    return w;
  }
  if (lane < a.batch) w.lens = walk_len<LM>(a, lane);
  const int W = lane < a.batch ? walk_weight(w.lens) : 0;
  int incl = W, longest = W;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {  // (lanes past the batch count nothing)
    if (d >= a.batch) break;
    const int y = __shfl_up(incl, d);
    if (lane >= d) incl += y;
    longest = max(longest, __shfl_xor(longest, d));
  }
  longest = __builtin_amdgcn_readfirstlane(longest);
  int total = __builtin_amdgcn_readlane(incl, a.batch - 1);
  int C = max((total + a.walk_segs - 1) / a.walk_segs, a.walk_min);
  if (longest <= a.walk_short || walk_keep_whole(a, longest, C, a.walk_whole)) {
    w.sg = DecSegment{k, 0, 0, 0, 0};
    return w;
  }
  // Units that start at segments: sum ceil(W / A) <= total / A + batch segments, so A = total /
  // (segs - batch) will do; no workgroup has two pieces then, which is worth kRbSwitch tiles.
  int room = W;
  if (a.walk_segs > a.batch) {
    const int free = a.walk_segs - a.batch;
    const int A = max((total + free - 1) / free, a.walk_min);
    if (A <= C + kRbSwitch) {
      w.aligned = true;
      C = A;
      room = (W + A - 1) / A * A;
      incl = room;
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        if (d >= a.batch) break;
        const int y = __shfl_up(incl, d);
        if (lane >= d) incl += y;
      }
      total = __builtin_amdgcn_readlane(incl, a.batch - 1);
    }
  }
  const int s0 = min(k * C, total);
  if (s0 >= total) {
    w.sg = DecSegment{a.batch, total, total, total, C};
    return w;
  }
  const int j = __builtin_ctzll(__ballot(incl > s0));  // the first whose end is past s0
  w.sg = DecSegment{j, __builtin_amdgcn_readlane(incl - room, j), s0, min(s0 + C, total), C};
  return w;
}

// The piece of sequence j's unit (starting at us in its stream) in the segment; false past
// the segment's end.
template <int LM>
__device__ __forceinline__ bool rows_piece(const KArgs& a, const RowsWalk& w, int stream,
                                           int seg_k, int j, int us, RowsPiece& p) {
  const DecSegment& sg = w.sg;
  const bool whole = sg.C == 0;
  if (j >= a.batch || (!whole && us >= sg.s1)) return false;
  p.b = j;
  p.kvh = stream % a.hkv;
  p.qblk = stream / a.hkv;
  p.Lk = w.in_lanes ? __builtin_amdgcn_readlane(w.lens, j)
                    : __builtin_amdgcn_readfirstlane(walk_len<LM>(a, j));
  const int n = (p.Lk + kBN - 1) / kBN;
  p.us = us;
  p.W = n > 1 ? n : 1;
  p.unit = j * a.walk_streams + stream;
  if (whole) {
    p.t0 = 0;
    p.T = n;
    p.np = 1;
    p.mine = 0;
    return true;
  }
  const int b = max(us, sg.s0), e = min(us + p.W, sg.s1);
  p.t0 = b - us;
  p.T = n > 0 ? e - b : 0;
  const int kf = us / sg.C;
  p.np = (us + p.W - 1) / sg.C - kf + 1;
  p.mine = seg_k - kf;
  if (w.aligned) p.W = p.np * sg.C;  // (the room that it takes)
  return true;
}

// What the merge of a unit has to know, by its first piece.
__device__ __forceinline__ void rows_info(const RowsArgs& ra, const DecSegment& sg, int stream,
                                          const RowsPiece& p) {
  if (p.mine != 0) return;
  const int slot =
      p.np > 1 ? static_cast<int>(walk_slot(ra.a, sg.C, p.us, stream, 0)) : 0;
  ra.info[p.unit] = make_int2(p.np, slot);
}

// The merge of cut units, launched behind the kernels that cut them: workgroup (x, y) takes
// rows y * kMergeRows .. of unit x, a thread 4 columns of a row over all pieces, in order, up
// to 8 of them in flight.  (One workgroup per unit that merges in the first kernel, as the
// 16-bit decode kernels do, takes a memory round trip for every 64 KB of partials, 32 to 256 KB
// a piece of a latent: with blocks of 32 rows 4 x 900 keys of 16 heads took 36 us, with this
// launch 26.  Pieces of a few KB were not measured.)
template <int DV>
constexpr int kMergeRows = DV >= 1024 ? 1 : 1024 / DV;  // rows of 256 threads

template <int DT, int DV>
__global__ __launch_bounds__(256) void fa2_rows_merge_kernel(RowsArgs ra) {
  constexpr bool BF = Elt<DT>::kBF;
  const KArgs& a = ra.a;
  const int unit = blockIdx.x;
  const int2 info = ra.info[unit];
  if (info.x <= 1) return;  // the unit was whole
  const int b = unit / a.walk_streams, stream = unit - b * a.walk_streams;
  const int kvh = stream % a.hkv, q0 = stream / a.hkv * a.block_rows;
  const int r = blockIdx.y * kMergeRows<DV> + threadIdx.x / (DV / 4);
  const int col = (threadIdx.x % (DV / 4)) * 4;
  if (r >= a.part_rows || q0 + r >= a.q_len) return;
  auto row_of = [&](int s) -> int64_t {  // walk_slot
    const int slot = s == 0 ? info.y : ((info.y >> 1) + s * a.walk_streams) * 2;
    return static_cast<int64_t>(slot) * a.part_rows + r;
  };
  float m = -INFINITY, l = 0.f;
  f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
  auto add = [&](auto nc, int s0) {  // pieces s0 ..+N - 1
    constexpr int N = decltype(nc)::value;
    f32x2 ml[N];
    f32x4 x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int64_t at = row_of(s0 + j);
      ml[j] = *reinterpret_cast<const f32x2*>(a.part_ml + at * 2);
      x[j] = *reinterpret_cast<const f32x4*>(a.part_o + at * DV + col);
    }
    float mn = m;
#pragma unroll
    for (int j = 0; j < N; ++j) mn = fmaxf(mn, ml[j][0]);
    const float mu = mn == -INFINITY ? 0.f : mn;
    const float al = fast_exp2(m - mu);
    l *= al;
    acc *= al;
    m = mn;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float w = fast_exp2(ml[j][0] - mu);
      l += w * ml[j][1];
      acc += w * x[j];
    }
  };
  const int n = __builtin_amdgcn_readfirstlane(info.x);
  int s0 = 0;
  for (; s0 + 8 <= n; s0 += 8) add(std::integral_constant<int, 8>{}, s0);
  if (n & 4) add(std::integral_constant<int, 4>{}, s0), s0 += 4;
  if (n & 2) add(std::integral_constant<int, 2>{}, s0), s0 += 2;
  if (n & 1) add(std::integral_constant<int, 1>{}, s0);
  const float inv = 1.f / l;  // 0/0 -> NaN for a row with no key
  *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.o) + b * a.o_sb +
                            static_cast<int64_t>(kvh) * (a.hq / a.hkv) * a.o_sh +
                            static_cast<int64_t>(q0 + r) * a.o_ss + col) =
      (u32x2){pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv)};
}

// Element offsets of a piece's K and V row 0 (paged: of its kv head).
template <int MODE>
__device__ __forceinline__ void rows_bases(const KArgs& a, const RowsPiece& p, int64_t& kbase,
                                           int64_t& vbase) {
  kbase = p.kvh * a.k_sh;
  vbase = p.kvh * a.v_sh;
  if constexpr (MODE == FA2_LAYOUT_DENSE) {
    kbase += p.b * a.k_sb;
    vbase += p.b * a.v_sb;
  } else if constexpr (MODE == FA2_LAYOUT_RAGGED) {
    const int64_t ks = a.kv_indptr[p.b];
    kbase += ks * a.k_ss;
    vbase += ks * a.v_ss;
  }
}

// Block-table entries page0 .. page0 + last of sequence b, clamped into the pool, on their
// way to LDS: this thread's first ones in registers, the rest behind them.  (V's lie behind
// K's.  What is loaded between load and store does not delay the entries.)
template <bool LAT, int NT>
struct RowsTable {
  int k, v;
  __device__ __forceinline__ void load(const RowsArgs& ra, int b, int page0, int last) {
    const KArgs& a = ra.a;
    const int i = page0 + min(static_cast<int>(threadIdx.x), last);
    k = a.k_table[b * a.k_table_stride + i];
    if constexpr (!LAT) v = a.v_table[b * a.v_table_stride + i];
  }
  __device__ __forceinline__ void store(const RowsArgs& ra, int b, int page0, int last,
                                        int* tab) const {
    const KArgs& a = ra.a;
    auto in = [&](int e) { return min(max(e, 0), ra.num_pages - 1); };
    const int tid = threadIdx.x;
    if (tid <= last) {
      tab[tid] = in(k);
      if constexpr (!LAT) tab[kRbTable / 2 + tid] = in(v);
    }
    for (int i = tid + NT; i <= last; i += NT) {
      tab[i] = in(a.k_table[b * a.k_table_stride + page0 + i]);
      if constexpr (!LAT) tab[kRbTable / 2 + i] = in(a.v_table[b * a.v_table_stride + page0 + i]);
    }
  }
};

// What a tile's places behind the last key take for V.  Their weights are zero; the last row
// itself, repeated there, would turn its infinite values into NaN (0 * inf) for the rows that
// see it.  (A latent's row needs none of this: an infinite value in it is NaN in the result
// wherever a row sees it, by a score that is not finite and 0 * inf.)
static __device__ const u32x4 kNoValue = {0, 0, 0, 0};

// x, whose uses are not computed ahead of this place (registers of the tile loop).
__device__ __forceinline__ int here(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// The mask rows of sequence b's tree as words in LDS, a row per wave and step.  The loads of up
// to 16 rows are in flight at once.  (A round trip for each, of 61: 6 us a piece.)
template <int NW>
struct RowsTree {
  static constexpr int kMax = kRbMaxTree / NW;
  uint8_t x[kMax];
  // f(step, row) over the wave's rows; the last rows repeat
  template <typename F>
  __device__ __forceinline__ void each(const KArgs& a, int wave, F&& f) {
    static_for<kMax / 4>([&](auto g) {
      if (wave + decltype(g)::value * 4 * NW < a.pack_m) {
        static_for<4>([&](auto j) {
          constexpr int s = decltype(g)::value * 4 + decltype(j)::value;
          f(std::integral_constant<int, s>{}, min(wave + s * NW, a.pack_m - 1));
        });
      }
    });
  }
  __device__ __forceinline__ void load(const RowsArgs& ra, int b, int wave, int lane) {
    const uint8_t* t = ra.tree + b * ra.tree_sb + min(lane, ra.a.pack_m - 1);
    each(ra.a, wave, [&](auto s, int row) { x[decltype(s)::value] = t[row * ra.tree_sr]; });
  }
  // one row after the other, where the registers do not allow more
  __device__ __forceinline__ static void fill(const RowsArgs& ra, int b, int wave, int lane,
                                              uint64_t* sh) {
    for (int i = wave; i < ra.a.pack_m; i += NW) {
      const uint8_t sees =
          lane < ra.a.pack_m ? ra.tree[b * ra.tree_sb + i * ra.tree_sr + lane] : uint8_t(0);
      const uint64_t word = __ballot(sees != 0);
      if (lane == 0) sh[i] = word;
    }
  }
  __device__ __forceinline__ void store(const KArgs& a, int wave, int lane, uint64_t* sh) {
    each(a, wave, [&](auto s, int row) {
      const uint64_t word = __ballot(lane < a.pack_m && x[decltype(s)::value] != 0);
      if (lane == 0) sh[row] = word;
    });
  }
};

// Bit x: key n + x is seen by draft m; off: keys before the drafts (below zero where there
// are fewer keys than drafts), word: the drafts that m sees (kMaskTree).
__device__ __forceinline__ uint32_t rows_sees(const KArgs& a, int n, int Lk, int off, int m,
                                              uint64_t word) {
  if (a.mask == kMaskTree) {
    const int x = n - off;  // the first key's place among the drafts
    return x >= 64   ? 0u
           : x >= 0  ? static_cast<uint32_t>(word >> x)
           : x > -32 ? (static_cast<uint32_t>(word << -x) | ((1u << -x) - 1u))
                     : ~0u;
  }
  const int c = (a.mask == FA2_MASK_NONE ? Lk : min(off + m + 1, Lk)) - n;
  return c >= 32 ? ~0u : c <= 0 ? 0u : (1u << c) - 1u;
}

// Wait until at most n tiles of IPT loads each are in flight (n <= MAXN, uniform).
template <int IPT, int MAXN>
__device__ __forceinline__ void rows_wait(int n) {
  static_assert(MAXN * IPT <= 63 && MAXN <= 4, "vmcnt field");
  if (MAXN >= 4 && n >= 4) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MAXN >= 4 ? 4 * IPT : 0) : "memory");
  else if (MAXN >= 3 && n >= 3) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MAXN >= 3 ? 3 * IPT : 0) : "memory");
  else if (MAXN >= 2 && n >= 2) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MAXN >= 2 ? 2 * IPT : 0) : "memory");
  else if (n >= 1) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(IPT) : "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// A wave-uniform address in scalar registers.
__device__ __forceinline__ uint64_t scalar_addr(const char* p) {
  const uint64_t at = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<int>(at));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<int>(at >> 32));
  return (static_cast<uint64_t>(hi) << 32) | lo;
}

// 16 bytes per lane to LDS from a scalar base and a 32-bit offset per lane (wait states
// as dma_buffer_x4).
template <bool NT = false>
__device__ __forceinline__ void rows_dma(uint64_t base, uint32_t off, uint32_t lds_addr) {
  if constexpr (NT)
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(off), "s"(base),
                   "{m0}"(__builtin_amdgcn_readfirstlane(static_cast<int>(lds_addr))));
  else
    asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1"
                 :
                 : "v"(off), "s"(base),
                   "{m0}"(__builtin_amdgcn_readfirstlane(static_cast<int>(lds_addr))));
}

// MFMAs of the kernels with O^T of 256 dims or more a wave: O^T in AGPRs (mma32_acc), S in VGPRs
// (mma32_vgpr), as the compiler left to itself moves O^T to and fro for every tile (17 trees of
// 7 drafts, 256 dims: 59 us, so 53 in the same run) and spills Q (512 dims: 1739 us in the first
// version, so 130).  Two wait states stand between a VALU write of an operand and its MFMA; who
// reads the result waits 24 (mma32_wait; the longest MFMA asks for 20).
template <bool BF>
__device__ __forceinline__ void mma32_acc(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (BF)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
  else
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
template <bool BF>
__device__ __forceinline__ void mma32_vgpr(f32x16& c, u32x4 a, u32x4 b) {
  if constexpr (BF)
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
  else
    asm volatile("s_nop 1\n\tv_mfma_f32_32x32x16_f16 %0, %1, %2, %0" : "+v"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mma32_wait(f32x16& c) {
  asm volatile("s_nop 15\n\ts_nop 7" : "+v"(c));
}
// c lies in AGPRs here: what scales or stores it takes its elements apart behind this, so that
// the loops carry it whole.
__device__ __forceinline__ void in_acc(f32x16& c) { asm volatile("" : "+a"(c)); }

// NT: loads past the caches, where no other q-block reads the same K and V (64 trees of 16
// drafts 205 us, without it 227; of 61 drafts, two q-blocks, it cost 4 %).
template <int DT, int DK, int DV, bool LAT, int RG, int MODE, bool NT>
__global__ __launch_bounds__(kRbThreads, (RowsTile<DK, DV, LAT, RG>::kOcc)) void
fa2_decode_rows_kernel(RowsArgs ra) {
  static_assert(DT != FA2_DTYPE_F32, "16-bit rows");
  static_assert(RG == 1 || RG == 2 || RG == 4, "row groups");
  constexpr bool BF = Elt<DT>::kBF;
  constexpr bool kPaged = MODE == FA2_LAYOUT_PAGED;
  constexpr int LM = kPaged ? kModePagedCapped : MODE;
  using GK = RowsGeo<DK>;
  using GV = RowsGeo<LAT ? DK : DV>;
  using TL = RowsTile<DK, DV, LAT, RG>;
  constexpr int TK = TL::kKeys, NS = TL::kSlots, SB = TK / 32;
  constexpr int DC = DK / 16;               // k-steps of S
  constexpr int DG = kRbWaves / RG;         // waves that share a row group's dims
  constexpr int DBW = DV / 32 / DG;         // 32-dim blocks of a wave's O^T
  static_assert(DBW >= 1, "dims of a wave");
  static_assert(DBW < 8 || SB == 1, "mma32_wait");
  constexpr bool kAcc = DBW >= 8;           // O^T lies in the AGPRs
  constexpr int GPW = TK / 32;              // 8-row groups a wave loads per tile
  constexpr int IPT = GPW * (GK::kGI + (LAT ? 0 : GV::kGI));
  constexpr int kVOff = LAT ? 0 : TK * GK::kRowBytes;  // V rows in a slot
  constexpr int kTab = LAT ? kRbTable : kRbTable / 2;
  // fp16 weights are scaled by 2^7 (at most 2^15 with the lazy maximum): small ones keep
  // their bits in fp16's range
  constexpr float kLift = BF ? 0.f : 7.f;

  __shared__ __attribute__((aligned(1024))) char tiles[NS * TL::kSlot];
  __shared__ int tab[kPaged ? kRbTable : 1];
  __shared__ uint64_t tree_sh[kRbMaxTree];
  __shared__ DecSegment seg_sh;

  const KArgs& a = ra.a;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31;
  const int hi = lane >> 5;
  const int rg = wave / DG;
  const int dg = wave % DG;
  const int d0 = dg * DBW;
  const int stream = static_cast<int>(blockIdx.x) % a.walk_streams;
  const int seg_k = static_cast<int>(blockIdx.x) / a.walk_streams;

  const RowsWalk walk = rows_locate<LM>(a, seg_k, &seg_sh);
  const DecSegment& sg = walk.sg;
  auto page_of = [&](int n) -> int {
    return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(n), ra.page_mul) >> ra.page_sh);
  };

  // ---- LDS addresses ---------------------------------------------------------
  const uint32_t tiles0 = lds_addr_of(tiles);
  // K row l32 of a 32-key block, chunk 2 cc + hi
  const uint32_t koff = l32 * GK::kRowBytes + ((hi ^ GK::swz(l32)) * 16);
  // V: lane i of 16-lane group g reads row 16 c + 8 rr + 4 (g / 2) + i / 4, dims
  // 32 d + 16 (g % 2) + 4 (i % 4); see RowsGeo for the place of a chunk
  constexpr int KM = GV::kG / 2;  // 32-dim blocks of a swizzle group
  uint32_t voff;
  {
    const int g = lane >> 4, i = lane & 15;
    const int r = 4 * (g >> 1) + (i >> 2);
    const uint32_t c = 4 * (d0 & (KM - 1)) + 2 * (g & 1) + ((i & 3) >> 1);
    voff = kVOff + r * GV::kRowBytes + ((c ^ GV::swz(r)) * 16) + (i & 1) * 8 +
           (d0 / KM) * KM * 64;
  }
  // loads: byte offset of this lane's chunk within the 8 rows of a group, whose rows
  // are 8 (wave & 1) ..+7 in the swizzle
  const uint32_t ksb = static_cast<uint32_t>(a.k_ss * 2), vsb = static_cast<uint32_t>(a.v_ss * 2);
  auto lane_row = [&](auto geo, int i, int ln) -> int { return (i * 64 + ln) / decltype(geo)::kNC; };
  auto lane_chunk = [&](auto geo, int i, int ln) -> uint32_t {
    using G = decltype(geo);
    return static_cast<uint32_t>((i * 64 + ln) % G::kNC) ^
           G::swz(8 * (wave & 1) + (i * 64 + ln) / G::kNC);
  };
  uint32_t kl[GK::kGI], vl[LAT ? 1 : GV::kGI];
#pragma unroll
  for (int i = 0; i < GK::kGI; ++i) kl[i] = lane_row(GK{}, i, lane) * ksb + lane_chunk(GK{}, i, lane) * 16;
  if constexpr (!LAT) {
#pragma unroll
    for (int i = 0; i < GV::kGI; ++i) vl[i] = lane_row(GV{}, i, lane) * vsb + lane_chunk(GV{}, i, lane) * 16;
  }
  const bool even_pages = !kPaged || a.page_size % 8 == 0;

  RowsPiece p;
  if (!rows_piece<LM>(a, walk, stream, seg_k, sg.j, sg.us, p)) return;
  for (;;) {
    // ---- the piece's rows, mask and first block-table entries -----------------
    const int q0 = p.qblk * (32 * RG);
    const int row = q0 + rg * 32 + l32;
    const int m = row % a.pack_m;  // draft
    const int nrows = min(a.q_len - q0, 32 * RG);
    int64_t kbase, vbase;
    rows_bases<MODE>(a, p, kbase, vbase);
    const char* kptr = static_cast<const char*>(a.k) + kbase * 2;
    const char* vptr = static_cast<const char*>(a.v) + vbase * 2;

    f32x16 o[DBW];
#pragma unroll
    for (int d = 0; d < DBW; ++d) {
      o[d] = (f32x16){};
      if constexpr (kAcc) in_acc(o[d]);
    }
    float m_run = -INFINITY, l_run = 0.f;
    const int off = p.Lk - a.pack_m;  // keys that every row sees
    const int full = a.mask == FA2_MASK_NONE ? p.Lk : min(off + (a.mask == kMaskTree ? 0 : 1), p.Lk);
    const int kend = min((p.t0 + p.T) * kBN, p.Lk);
    uint64_t word = 0;

    // ---- windows: keys whose block-table entries lie in LDS --------------------
    int ka = p.t0 * kBN, kb, page0;
    RowsTable<LAT, kRbThreads> entries;
    auto window = [&]() {
      kb = kend;
      page0 = 0;
      if constexpr (kPaged) {
        page0 = page_of(ka);
        const int64_t lim = (static_cast<int64_t>(page0) + kTab) * a.page_size;
        if (lim < kend) kb = ka + max((static_cast<int>(lim) - ka) / kBN * kBN, kBN);
        if (ka < kend) entries.load(ra, p.b, page0, page_of(kb - 1) - page0);
      }
    };
    RowsTree<kRbWaves> sees;
    if (a.mask == kMaskTree) {
      if constexpr (LAT) sees.fill(ra, p.b, wave, lane, tree_sh);
      else sees.load(ra, p.b, wave, lane);
    }
    window();
    u32x4 qf[DC];
    {
      const int qr = min(row, a.q_len - 1);  // (rows past the last repeat it: not stored)
      const int h = p.kvh * (a.hq / a.hkv) + qr / a.pack_m;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + p.b * a.q_sb + h * a.q_sh +
                            (qr % a.pack_m) * a.q_ss + hi * 8;
#pragma unroll
      for (int c = 0; c < DC; ++c) qf[c] = *reinterpret_cast<const u32x4*>(src + c * 16);
    }
    if constexpr (!LAT)
      if (a.mask == kMaskTree) sees.store(a, wave, lane, tree_sh);
    for (; ka < kend; ka = kb, window()) {
      if constexpr (kPaged) entries.store(ra, p.b, page0, page_of(kb - 1) - page0, tab);
      __syncthreads();  // the table and the mask are in LDS, the slots are free
      if (a.mask == kMaskTree) word = tree_sh[m];
      // Q is there before the first tile goes out: a later wait of the compiler's would drain
      // the tiles in flight
      __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)

      const int T = (kb - ka + TK - 1) / TK;
      // A tile goes out 8 rows at a time, each group of one page: its block-table entries are
      // read from LDS a tile ahead (fetch), its bases are scalars (aim), and its loads stand
      // between the MFMAs of S (send).
      auto whole = [&](int t) { return even_pages && ka + (t + 1) * TK <= kb; };
      int ek[GPW] = {}, ev[GPW] = {};
      auto fetch = [&](int t) {
        if constexpr (kPaged) {
#pragma unroll
          for (int g = 0; g < GPW; ++g) {
            const int at = page_of(min(ka + t * TK + 8 * (wave + 4 * g), kb - 1)) - page0;
            ek[g] = tab[at];
            if constexpr (!LAT) ev[g] = tab[kTab + at];
          }
        }
      };
      uint64_t sk[GPW], sv[GPW];
      auto aim = [&](int t) {
#pragma unroll
        for (int g = 0; g < GPW; ++g) {
          const int n = ka + t * TK + 8 * (wave + 4 * g);
          int64_t rk = n, rv = n;
          if constexpr (kPaged) {
            const int in = n - page_of(n) * a.page_size;
            rk = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(ek[g])) * a.page_size + in;
            if constexpr (!LAT)
              rv = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(ev[g])) * a.page_size + in;
          }
          sk[g] = scalar_addr(kptr + rk * (a.k_ss * 2));
          if constexpr (!LAT) sv[g] = scalar_addr(vptr + rv * (a.v_ss * 2));
        }
      };
      auto send = [&](auto jc, uint32_t slot) {
        constexpr int j = decltype(jc)::value, kPer = IPT / GPW;
        constexpr int g = j / kPer, r = j % kPer;
        constexpr bool V = r >= GK::kGI;
        constexpr int i = V ? r - GK::kGI : r;
        const uint32_t grp = wave + 4 * g;
        if constexpr (V)
          rows_dma<NT>(sv[g], vl[LAT ? 0 : i], slot + kVOff + grp * 8 * GV::kRowBytes + i * 1024);
        else
          rows_dma<NT>(sk[g], kl[i], slot + grp * 8 * GK::kRowBytes + i * 1024);
      };
      // The rest: a row per lane; places past the window hold its last K row (masked) and
      // zeros of V (kNoValue).
      auto send_rows = [&](auto is_v, int n, uint32_t dst) {
        constexpr bool V = decltype(is_v)::value;
        using G = std::conditional_t<V, GV, GK>;
        const char* base = V ? vptr : kptr;
        const int64_t ss = V ? a.v_ss : a.k_ss;
        const int* tb = tab + (V ? kTab : 0);
        const int ln = here(lane);
#pragma unroll
        for (int i = 0; i < G::kGI; ++i) {
          const int at = n + lane_row(G{}, i, ln), nr = min(at, kb - 1);
          int64_t r = nr;
          if constexpr (kPaged) {
            const int pg = page_of(nr);
            r = static_cast<int64_t>(tb[pg - page0]) * a.page_size + (nr - pg * a.page_size);
          }
          const char* src = base + r * ss * 2 + lane_chunk(G{}, i, ln) * 16;
          if (V && at >= kb) src = reinterpret_cast<const char*>(&kNoValue);
          dma_global_x4<NT>(src, dst + i * 1024);
        }
      };
      auto send_part = [&](int t) {
        const uint32_t slot = tiles0 + (t % NS) * TL::kSlot;
#pragma unroll
        for (int g = 0; g < GPW; ++g) {
          const int grp = wave + 4 * g, n = ka + t * TK + 8 * grp;
          send_rows(std::integral_constant<bool, false>{}, n, slot + grp * 8 * GK::kRowBytes);
          if constexpr (!LAT)
            send_rows(std::integral_constant<bool, true>{}, n,
                      slot + kVOff + grp * 8 * GV::kRowBytes);
        }
      };
      for (int t = 0; t < NS - 1 && t < T; ++t) {
        if (whole(t)) {
          fetch(t);
          aim(t);
          static_for<IPT>([&](auto jc) { send(jc, tiles0 + t * TL::kSlot); });
        } else {
          send_part(t);
        }
      }
      if (NS - 1 < T) fetch(NS - 1);
      for (int t = 0; t < T; ++t) {
        rows_wait<IPT, NS - 2>(T - 1 - t);
        pp_barrier();  // tile t is there, and slot t - 1 has been read
        const int tn = t + NS - 1;
        const bool ahead = tn < T && whole(tn);
        if (ahead) {
          aim(tn);
          fetch(tn + 1);
        } else if (tn < T) {
          send_part(tn);
        }
        const uint32_t next = tiles0 + (tn % NS) * TL::kSlot;
        const uint32_t slot = tiles0 + (t % NS) * TL::kSlot;
        const int n0 = ka + t * TK;

        // ---- S^T = K Q^T -------------------------------------------------------
        f32x16 s[SB];
#pragma unroll
        for (int sb = 0; sb < SB; ++sb) s[sb] = (f32x16){};
        auto scores = [&](auto dma) {
          constexpr bool kDma = decltype(dma)::value;
          constexpr int kN = DC * SB, kAhead = 6 < kN ? 6 : kN;
          auto frag = [&](auto kc) -> u32x4 {
            constexpr int cc = decltype(kc)::value / SB, sb = decltype(kc)::value % SB;
            return *(const lds_u32x4_t*)(lds_ptr(slot + (koff ^ (32u * (cc % GK::kG)))) +
                                         sb * 32 * GK::kRowBytes + (cc / GK::kG) * GK::kG * 32);
          };
          f32x16 s2 = (f32x16){};  // odd k-steps of a single block: two chains of MFMAs
          __builtin_amdgcn_sched_barrier(0);
          u32x4 fr[kN];
          static_for<kAhead>([&](auto kc) { fr[decltype(kc)::value] = frag(kc); });
          static_for<kN>([&](auto kc) {
            constexpr int k = decltype(kc)::value, cc = k / SB, sb = k % SB;
            if constexpr (kAcc)
              mma32_vgpr<BF>(s[sb], fr[k], qf[cc]);
            else if constexpr (SB == 1 && (cc & 1))
              s2 = mma32<BF>(fr[k], qf[cc], s2);
            else
              s[sb] = mma32<BF>(fr[k], qf[cc], s[sb]);
            if constexpr (k + kAhead < kN)
              fr[k + kAhead] = frag(std::integral_constant<int, k + kAhead>{});
            if constexpr (kDma) {  // loads [k IPT / kN, (k + 1) IPT / kN)
              constexpr int j0 = k * IPT / kN, j1 = (k + 1) * IPT / kN;
              static_for<j1 - j0>([&](auto x) {
                send(std::integral_constant<int, j0 + decltype(x)::value>{}, next);
              });
            }
            if constexpr (kAcc) __builtin_amdgcn_sched_barrier(0);
          });
          if constexpr (!kAcc) {
            __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
            for (int k = 0; k < kN - kAhead; ++k) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
          if constexpr (kAcc) mma32_wait(s[0]);
          else if constexpr (SB == 1) s[0] += s2;
        };
        if (ahead) scores(std::integral_constant<bool, true>{});
        else scores(std::integral_constant<bool, false>{});

        // ---- mask: key n0 + 32 sb + 8 (i / 4) + 4 hi + i % 4 of element i --------
        if (n0 + TK > full) {
#pragma unroll
          for (int sb = 0; sb < SB; ++sb) {
            const uint32_t sees =
                rows_sees(a, n0 + 32 * sb, p.Lk, off, m, word) >> (4 * hi);
#pragma unroll
            for (int i = 0; i < 16; ++i)
              if (!(sees & (1u << ((i >> 2) * 8 + (i & 3))))) s[sb][i] = -INFINITY;
          }
        }

        // ---- softmax -------------------------------------------------------------
        float mx = -INFINITY;
#pragma unroll
        for (int sb = 0; sb < SB; ++sb)
#pragma unroll
          for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[sb][i]);
        mx = max_xor32_valu(mx);
        const float mt = mx * a.scale_log2;
        const bool need = mt > m_run + kRescaleThreshold;
        if (__any(need)) {
          const float alpha = fast_exp2(need ? m_run - mt : 0.f);
          m_run = need ? mt : m_run;
          l_run *= alpha;
          if (n0 > p.t0 * kBN) {  // (nothing yet before the piece's first tile)
#pragma unroll
            for (int d = 0; d < DBW; ++d) {
              if constexpr (kAcc) in_acc(o[d]);
              o[d] *= alpha;
              if constexpr (kAcc) {
                in_acc(o[d]);
                __builtin_amdgcn_sched_barrier(0);
              }
            }
          }
        }
        const float m_use = (m_run == -INFINITY ? 0.f : m_run) - kLift;
        u32x4 pf[2 * SB];
#pragma unroll
        for (int sb = 0; sb < SB; ++sb) {
          float e[16];
#pragma unroll
          for (int i = 0; i < 16; ++i)
            e[i] = fast_exp2(__builtin_fmaf(s[sb][i], a.scale_log2, -m_use));
#pragma unroll
          for (int h = 0; h < 2; ++h)
            pf[sb * 2 + h] = (u32x4){pack2<BF>(e[h * 8 + 0], e[h * 8 + 1]),
                                     pack2<BF>(e[h * 8 + 2], e[h * 8 + 3]),
                                     pack2<BF>(e[h * 8 + 4], e[h * 8 + 5]),
                                     pack2<BF>(e[h * 8 + 6], e[h * 8 + 7])};
        }
        // (the sum of the rounded weights, those that the product with V applies)
#pragma unroll
        for (int c = 0; c < 2 * SB; ++c)
#pragma unroll
          for (int j = 0; j < 4; ++j) l_run = dot2_ones<BF>(pf[c][j], l_run);

        // ---- O^T += V^T P^T --------------------------------------------------------
        {
          constexpr int kN = 2 * SB * DBW, kAhead = 4 < kN ? 4 : kN;
          auto frag = [&](auto kc) -> u32x4 {
            constexpr int c = decltype(kc)::value / DBW, d = decltype(kc)::value % DBW;
            constexpr int kImm = 16 * c * GV::kRowBytes + (d / KM) * KM * 64;
            const u32x2 lo = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(
                           lds_ptr(slot + (voff ^ (64u * (d % KM)))) + kImm)));
            const u32x2 up = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)(
                           lds_ptr(slot + (voff ^ (64u * (d % KM)) ^ 16u)) + kImm +
                           8 * GV::kRowBytes)));
            return (u32x4){lo[0], lo[1], up[0], up[1]};
          };
          __builtin_amdgcn_sched_barrier(0);
          u32x4 fr[kN];
          static_for<kAhead>([&](auto kc) { fr[decltype(kc)::value] = frag(kc); });
          static_for<kN>([&](auto kc) {
            constexpr int k = decltype(kc)::value, c = k / DBW, d = k % DBW;
            if constexpr (kAcc) mma32_acc<BF>(o[d], fr[k], pf[c]);
            else o[d] = mma32<BF>(fr[k], pf[c], o[d]);
            if constexpr (k + kAhead < kN)
              fr[k + kAhead] = frag(std::integral_constant<int, k + kAhead>{});
            if constexpr (kAcc) __builtin_amdgcn_sched_barrier(0);
          });
          if constexpr (!kAcc) {
            __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);
#pragma unroll
            for (int k = 0; k < kN - kAhead; ++k) {
              __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
              __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if constexpr (kAcc) asm volatile("s_nop 15\n\ts_nop 7" ::: "memory");  // the last MFMAs
      __syncthreads();  // the window's table and slots have been read
    }

    // ---- the piece's end ---------------------------------------------------------
    const float l_tot = sum_xor32(l_run);
    const int le = here(lane), hi = le >> 5;
    const int r = rg * 32 + (le & 31);
    const int64_t obase = p.b * a.o_sb + p.kvh * (a.hq / a.hkv) * a.o_sh;
    if (p.np == 1) {
      if (r < nrows) {
        const float inv = 1.f / l_tot;  // 0/0 -> NaN for a row with no key
        uint16_t* dst = static_cast<uint16_t*>(a.o) + obase +
                        static_cast<int64_t>(q0 + r) * a.o_ss + d0 * 32 + hi * 4;
#pragma unroll
        for (int d = 0; d < DBW; ++d) {
          if constexpr (kAcc) in_acc(o[d]);
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<u32x2*>(dst + d * 32 + g * 8) =
                (u32x2){pack2<BF>(o[d][g * 4 + 0] * inv, o[d][g * 4 + 1] * inv),
                        pack2<BF>(o[d][g * 4 + 2] * inv, o[d][g * 4 + 3] * inv)};
          if constexpr (kAcc) __builtin_amdgcn_sched_barrier(0);
        }
      }
    } else {
      const int64_t slot = walk_slot(a, sg.C, p.us, stream, p.mine);
      if (r < nrows) {
        float* ml = a.part_ml + (slot * a.part_rows + r) * 2;
        float* po = a.part_o + (slot * a.part_rows + r) * DV + d0 * 32 + hi * 4;
        if (dg == 0 && hi == 0) *reinterpret_cast<f32x2*>(ml) = (f32x2){m_run, l_tot};
#pragma unroll
        for (int d = 0; d < DBW; ++d) {
          if constexpr (kAcc) in_acc(o[d]);
#pragma unroll
          for (int g = 0; g < 4; ++g)
            *reinterpret_cast<f32x4*>(po + d * 32 + g * 8) =
                (f32x4){o[d][g * 4 + 0], o[d][g * 4 + 1], o[d][g * 4 + 2], o[d][g * 4 + 3]};
          if constexpr (kAcc) __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    if (tid == 0) rows_info(ra, sg, stream, p);
    if (!rows_piece<LM>(a, walk, stream, seg_k, walk_next(a, sg, p.b), p.us + p.W, p)) return;
    __syncthreads();  // the mask is free
  }
}

}  // namespace fa2
