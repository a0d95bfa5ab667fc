// fa2_kernel_decode_fp4.h - decode and speculative decode attention over a
// paged cache held in 4 bits (include/fa2_ops.h), fp16/bf16 queries.
//
//   s_ij = q_i . k_j,  o_i = sum_j exp((s_ij - m_i) / sqrt(D)) v_j / sum_j exp(...)
//
// A value of the cache is e2m1 * 2^(scale - 127), exact in the queries' type
// (the append keeps it in range), and v_cvt_scalef32_pk_{f16,bf16}_fp4 makes two
// of them per instruction at full rate, scale included: the kernel computes what
// the 16-bit decode kernel computes on the cache's values.
//   * Workgroup = 8 waves, one per CU, over an equal share of the call's KV
//     tiles (fa2_decode_walk.h; kernel comment below).  A wave walks tiles of 32
//     keys, tile i of the workgroup's range to wave i % 8, and keeps its own (m, l,
//     O); they are added up in LDS at a piece's end.
//   * A page's rows of a kv head are contiguous.  Direct-to-LDS loads of whole
//     rows bring a tile per wave, across the ends of the pieces; its codes are
//     read into registers at once (they are few) and the next tile is on its way
//     while it is computed.  (Tiles in flight in registers instead need the loop
//     once per tile: 50 KB of code.  More tiles in flight in LDS gained nothing in long
//     calls of an earlier form of this kernel: 49.3 / 47.1 / 46.4 us at 3 / 2 / 1 for 16 x
//     16000-32768 keys of 4 heads of D128; short calls were not measured.)
//   * S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32, up to 16 RB rows
//     of the unit as columns.  A lane expands D / 4 dims of a key of K, in the
//     layout of the MFMA's A operand (lane: row l % 16, dims D / 4 * (l / 16)
//     ..; the queries take the dims of a k-step in the same order).  Of V it
//     expands D / 16 dims of the 8 keys that its P^T fragment has, and pairs them
//     by key with v_perm: block i of O^T is dim i of every 16 lanes.  (V back
//     through LDS in 16 bits, for transpose reads, took two thirds of the LDS
//     time, and that 75 % of a tile's.)
//   * P goes to the MFMA as the sum of two 16-bit values, high and low part, which costs
//     1 to 3.5 % of a long call, 6 % with 20 rows.  bf16: 16 bits of a weight, off by 2^-18 of it, so that 0.22 % of
//     the outputs of 64 sequences of 512-8192 keys round the other way than the exact
//     ones (0.04 % with exact weights); a third part, which makes them exact, takes
//     64.1 us for 60.9 there, 22.2 for 20.7 with 20 rows.  fp16: 22 bits, and weights from
//     2^11 down (kLift), so that one of 2^-25 of a wave's largest still has 11 and none is
//     off by more than 2^-36 of that (from 1 down, 2^-20 is off by up to 3 %).
//   * Running maxima and sums in fp32, raised only when a score passes the
//     maximum by 2^8 (bf16, as in the 16-bit kernels) or 2^4.
// Measured on MI355X, us per call, calls back to back (and the cache's bytes per s; under
// the profiler the kernel alone takes 3 to 12 % more than such a call): 64 sequences of
// 512-8192 keys, 32 / 8 heads of D128, 61 (5.1 TB/s), of D64 52 (3.1), of D256 109 (5.8);
// 16 of 16000-32768, 32 / 4 heads, 43 (4.8); 16 of 8200 with 8 drafts, 8 / 8 heads of D64, 25
// (2.9); 33 of 100-4096 with 5 drafts, 16 / 4 heads, 21 (1.6); 4 of 1023, 10.5.  The 16-bit
// decode reads 6.1 TB/s.  The long calls are bound by the loop's instructions as much as
// by memory (6 to 8 % less with every page in L2, both under the profiler); the short
// ones by what a workgroup does once: 3 us until its first tile is there, about 2 us
// per change of units, 4 us to count and merge cut units.
#pragma once

#include "fa2_decode_walk.h"
#include "fa2_kernel_lds.h"
#include "fa2_values.h"

namespace fa2 {

constexpr int kD4Waves = 8;
constexpr int kD4Threads = 64 * kD4Waves;
constexpr int kD4Tile = 32;    // keys of a wave's tile

typedef __attribute__((address_space(3))) f32x4 lds_f32x4_t;
typedef __attribute__((address_space(3))) f32x2 lds_f32x2_t;
typedef __attribute__((address_space(3))) u32x2 lds_u32x2_t;
typedef __attribute__((address_space(3))) uint32_t lds_u32_t;
typedef __attribute__((address_space(3))) uint16_t lds_u16_t;
typedef __attribute__((address_space(3))) uint8_t lds_u8_t;

struct Fp4Args {
  KArgs a;  // a.k, a.v: the codes; a.kv_len: keys a row of the tables can hold
  const uint8_t* ks;  // scales
  const uint8_t* vs;
  int32_t num_pages, table_width;
  uint32_t page_codes, page_scales;  // bytes of a page, and of its rows of one head
  uint32_t head_codes, head_scales;
  uint32_t page_mul, page_sh;  // n / page_size = (2 n * page_mul) >> 32 >> page_sh
};

template <bool BF>
__device__ __forceinline__ f32x4 mma16x32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (BF)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Values 2 B and 2 B + 1 of a code word, at the scale with the float's bits `f`.
template <bool BF, int B>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, uint32_t f) {
  if constexpr (BF)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(
                                            w, __builtin_bit_cast(float, f), B));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(
                                            w, __builtin_bit_cast(float, f), B));
}

// fp32 of the low / high half of a packed pair
template <bool BF>
__device__ __forceinline__ f32x2 unpack2(uint32_t w) {
  if constexpr (BF)
    return (f32x2){__builtin_bit_cast(float, w << 16),
                   __builtin_bit_cast(float, w & 0xFFFF0000u)};
  else
    return __builtin_convertvector(__builtin_bit_cast(f16x2, w), f32x2);
}

// Direct-to-LDS loads, lane i to lds + 16 i (or 4 i), from per-lane addresses; wait
// states as dma_buffer_x4.
__device__ __forceinline__ void fp4_dma16(const void* p, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %0, off nt"
               :
               : "v"(p), "{m0}"(__builtin_amdgcn_readfirstlane(static_cast<int>(lds))));
}
// From a uniform base and a 32-bit offset per lane (readlane, then the load).
__device__ __forceinline__ void fp4_dma16_base(uint64_t base, uint32_t off, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dwordx4 %0, %1 nt"
               :
               : "v"(off), "s"(base),
                 "{m0}"(__builtin_amdgcn_readfirstlane(static_cast<int>(lds))));
}
__device__ __forceinline__ void fp4_dma4(const void* p, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off"
               :
               : "v"(p), "{m0}"(__builtin_amdgcn_readfirstlane(static_cast<int>(lds))));
}

__device__ __forceinline__ void fp4_dma2(const void* p, uint32_t lds) {  // into a word each
  asm volatile("s_nop 0\n\tglobal_load_lds_ushort %0, off"
               :
               : "v"(p), "{m0}"(__builtin_amdgcn_readfirstlane(static_cast<int>(lds))));
}

// Geometry at head dim D.
template <int D>
struct Fp4Geo {
  static constexpr int kRow = D / 2;                  // bytes of a row of codes
  static constexpr int kNC = kRow / 16;               // its 16-byte chunks
  static constexpr int kCode = kD4Tile * kRow;        // a tile's codes of K (or V)
  static constexpr int kLoads = kCode / 1024;         // ... and their loads
  static constexpr int kScale = D == 256 ? 256 : 128; // LDS bytes of its scales
  static constexpr int kScaleRow = D == 256 ? 8 : 4;
  static constexpr int kScaleLoads = D == 256 ? 2 : 1;  // (K and V in one up to 128)
  static constexpr int kTile = 2 * kCode + 2 * kScale;
  static constexpr int kNI = D / 16;                  // dims of V of a lane, blocks of O^T
  static constexpr int kPD = 64;                      // dims merged at a time
  static constexpr int kPH = D / kPD;                 // phases
  static constexpr int kRP = 16 / kNI;                // accumulator rows of a lane per phase
  static constexpr int kPitch = (kPD + 4) * 4;        // merge rows
  static constexpr int kStage = 16 * kPitch;          // a wave's merge area: a phase of 16 rows
  static constexpr int kTable = 256;                  // block-table entries of a window
  // chunk c of row r lies at chunk c ^ ksw(r): 8 lanes reading a chunk of 8 rows
  // hit distinct banks
  static __device__ __forceinline__ int ksw(int r) {
    return D == 64 ? (r >> 3) & 1 : D == 128 ? (r >> 2) & 3 : (r >> 1) & 7;
  }
  // Row p of a block of V in LDS is key vkey(p) of it: the four lane groups read
  // keys four apart, and so four rows side by side.
  static __device__ __forceinline__ int vkey(int p) { return (p & 16) + ((p & 15) >> 2) + 4 * (p & 3); }
  // The dim of O that value sd of merge phase h is.  (Value r of block i in lane group
  // g is dim D / 4 * g + kNI * r + i; a phase takes kRP rows of each.)
  static __device__ __forceinline__ int dim(int h, int sd) {
    return (sd >> 4) * (D / 4) + 16 * h + (sd & 15);
  }
};

// x of the lane and of lane ^ 16 (or ^ 32), in the same order in both.
template <int X>
__device__ __forceinline__ f32x2 lane_pair(float x) {
  const int w = __builtin_bit_cast(int, x);
  u32x2 y;
  if constexpr (X == 16)
    y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(w, w, false, false));
  else
    y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(w, w, false, false));
  return __builtin_bit_cast(f32x2, y);
}
template <bool MAX>
__device__ __forceinline__ float over_groups(float x) {  // the four lanes l % 16
  const f32x2 y = lane_pair<16>(x);
  const f32x2 z = lane_pair<32>(MAX ? fmaxf(y[0], y[1]) : y[0] + y[1]);
  return MAX ? fmaxf(z[0], z[1]) : z[0] + z[1];
}

// Sum (or maximum, of numbers >= 0) over the lanes up to each, on the VALU.
template <bool MAX>
__device__ __forceinline__ int wave_scan(int x) {
  auto join = [](int a, int b) { return MAX ? max(a, b) : a + b; };
  x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, false));  // row_shr 1, 2, 4, 8
  x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, false));
  x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, false));
  x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, false));
  x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false));  // row_bcast 15, 31
  x = join(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false));
  return x;
}

// The walk here, for batches of up to 64 sequences (their lengths are in the lanes; longer
// batches take the walk as it is):
//   * Units start at segments where that makes segments at most kAlign tiles longer:
//     then a workgroup has one piece.
//   * Otherwise a unit takes kGap tiles of room in its stream besides its own, what a
//     change of units costs, so that workgroups with several have fewer tiles.
// Neither / the second alone / both, us: 33 x 100-4096 keys with 5 drafts of 16 / 4 heads
// 32.6 / 24.8 / 20.8; 16 x 4096-8192 of 32 / 2 heads 21.4 / 19.9 / 16.0; 16 x 8200 with 8
// drafts of 8 / 8 heads of D64 28.8 / 25.6 / 25.3.  (kAlign, kGap) of (8, 5), (8, 3), (8, 6), (4,
// 5), (16, 8), (24, 4) take 16.0, 16.0, 16.0, 16.6, 16.8, 17.1 for the second, which has 16 rows;
// for the first, which has 32, (12, 8), (8, 6), (16, 8), (8, 3), (24, 4), (4, 5) take 20.8, 21.7,
// 21.7, 21.8, 23.5, 27.5.
//
// BLOCKS: pages of whole blocks of 16 rows, whose addresses are found once per block
// instead of once per row: 64 x 512-8192 keys in pages of 16 take 61.5 us, 66.5 without.
template <int DT, int D, int RB, bool BLOCKS>
__global__ __launch_bounds__(kD4Threads, 2) void fa2_decode_fp4_kernel(
    Fp4Args fa) {
  using G = Fp4Geo<D>;
  constexpr bool BF = Elt<DT>::kBF;
  constexpr int MODE = kModePagedCapped;
  constexpr int DJ = D / 32;        // S k-steps = code words of a lane
  constexpr int kStep = kD4Tile * kD4Waves;
  constexpr int kSub = D == 256 ? 2 : 1;  // scales of a lane's dims
  static_assert(kD4Waves * G::kStage >= kMergePieceBytes<kD4Threads>, "merge area");
  // fp16 weights are at most 2^kRaise * 2^kLift = 2^15
  constexpr float kRaise = BF ? kRescaleThreshold : 4.f, kLift = BF ? 0.f : 11.f;
  constexpr int kAlign = RB == 1 ? 8 : 12, kGap = RB == 1 ? 5 : 8;  // tiles

  __shared__ __attribute__((aligned(1024))) char tiles[kD4Waves * G::kTile];
  __shared__ __attribute__((aligned(128))) char stage[2 * kD4Waves * G::kStage];
  __shared__ __attribute__((aligned(8))) float mrg_ml[kD4Waves][16][2];
  __shared__ int tab[3][2][G::kTable];
  __shared__ DecSegment seg_sh[kD4Waves];
  __shared__ int merge_flag[2];

  const KArgs& a = fa.a;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const bool causal = a.mask != FA2_MASK_NONE;
  const int stream = static_cast<int>(blockIdx.x) % a.walk_streams;
  const int seg_k = static_cast<int>(blockIdx.x) / a.walk_streams;

  // This workgroup's units: all of one kv head and q-block.
  const int kvh = stream % a.hkv, qblk = stream / a.hkv;
  const int head0 = kvh * (a.hq / a.hkv);
  const int q0 = qblk * (16 * RB), rows = min(a.q_len - q0, 16 * RB);

  // The segment, found by each wave for itself (no barrier).  A batch of up to 64
  // keeps its lengths in the lanes (walk_locate's rule, on one length per lane).
  const bool in_lanes = a.batch <= 64;
  const int lens = in_lanes && lane < a.batch ? walk_len<MODE>(a, lane) : 0;
  DecSegment sg;
  int room = 0;  // in_lanes: what the lane's unit takes of its stream (0: no unit)
  int gap = 0;   // ... and of that, ahead of its tiles
  if (in_lanes) {
    const int W = lane < a.batch ? walk_weight(lens) : 0;
    int total = __builtin_amdgcn_readlane(wave_scan<false>(W), 63);
    const int longest = __builtin_amdgcn_readlane(wave_scan<true>(W), 63);
    int C = max((total + a.walk_segs - 1) / a.walk_segs, a.walk_min);
    sg = DecSegment{seg_k, 0, 0, 0, 0};
    if (longest > a.walk_short && !walk_keep_whole(a, longest, C, a.walk_whole)) {
      int incl = 0;
      bool fit = false;
      if (a.batch <= a.walk_segs) {
        for (int c = C; c <= C + kAlign && !fit; c += kAlign / 2) {
          // n = ceil(W / c): a first guess off by one at most, put right
          const float inv = __builtin_amdgcn_rcpf(static_cast<float>(c));
          int n = static_cast<int>(static_cast<float>(W) * inv);
          n += n * c < W;
          n -= (n - 1) * c >= W && n > 0;
          incl = wave_scan<false>(n);
          fit = __builtin_amdgcn_readlane(incl, 63) <= a.walk_segs;
          if (fit) {
            C = c;
            incl *= c;
            room = n * c;
          }
        }
      }
      if (!fit) {
        gap = kGap;
        room = W ? W + kGap : 0;
        incl = wave_scan<false>(room);
        total = __builtin_amdgcn_readlane(incl, 63);
        C = max((total + a.walk_segs - 1) / a.walk_segs, a.walk_min);
      }
      total = __builtin_amdgcn_readlane(incl, 63);
      const int s0 = min(seg_k * C, total);
      const uint64_t at = __ballot(incl - room <= s0 && s0 < incl);
      sg = DecSegment{a.batch, total, total, total, C};
      if (at) {
        const int j = __builtin_ctzll(at);
        sg = DecSegment{j, __builtin_amdgcn_readlane(incl - room, j) + gap, s0,
                        min(s0 + C, total), C};
      }
    }
  } else {
    walk_locate<MODE>(a, seg_k, &seg_sh[wave]);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    sg.j = __builtin_amdgcn_readfirstlane(seg_sh[wave].j);
    sg.us = __builtin_amdgcn_readfirstlane(seg_sh[wave].us);
    sg.s0 = __builtin_amdgcn_readfirstlane(seg_sh[wave].s0);
    sg.s1 = __builtin_amdgcn_readfirstlane(seg_sh[wave].s1);
    sg.C = __builtin_amdgcn_readfirstlane(seg_sh[wave].C);
  }

  // A piece (DecPiece without what is the same for all of the workgroup's), and a
  // window of it: keys [ka, kb), all of it unless its block-table entries exceed
  // the LDS table.
  struct Window {
    // sequence, its tiles' start in the stream and number, its room, its length
    int b, us, W, room, Lk;
    int np, mine;       // pieces of the unit, this one's index
    int ka, kb, kend;   // kend: the piece's end
    int page0;          // first logical page
  };
  // The piece of sequence j's unit, from us in the stream (as walk_piece).
  auto piece_at = [&](Window& v, int j, int us) -> bool {
    const bool whole = sg.C == 0;
    if (j >= a.batch || (!whole && us >= sg.s1)) return false;
    v.b = j;
    v.us = us;
    v.Lk = in_lanes ? __builtin_amdgcn_readlane(lens, j) : walk_len<MODE>(a, j);
    v.W = walk_weight(v.Lk);
    v.room = in_lanes ? __builtin_amdgcn_readlane(room, j) : v.W;
    v.np = 1;
    v.mine = 0;
    v.ka = 0;
    v.kend = v.Lk;
    if (!whole) {
      // (segment k starts at k C: only its ends can lie in other segments' units)
      const int kf = us >= sg.s0 ? seg_k : us / sg.C;
      const int kl = us + v.W <= sg.s1 ? seg_k : (us + v.W - 1) / sg.C;
      v.np = kl - kf + 1;
      v.mine = seg_k - kf;
      v.ka = max(sg.s0 - us, 0) * kBN;
      v.kend = min(min(us + v.W, sg.s1) - us, (v.Lk + kBN - 1) / kBN) * kBN;
      v.kend = min(v.kend, v.Lk);
    }
    return true;
  };
  // n / page_size for n < 2^30 (fa2_fp4_decode)
  auto page_of = [&](int n) {
    return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(n), fa.page_mul) >> fa.page_sh);
  };
  auto window_at = [&](Window& v, int ka) {
    v.ka = ka;
    v.kb = v.kend;
    v.page0 = page_of(ka);
    const int64_t lim = (static_cast<int64_t>(v.page0) + G::kTable) * a.page_size;
    if (lim < v.kend) {  // whole tiles, so that every window starts at one
      const int n = (static_cast<int>(lim) - ka) / kD4Tile * kD4Tile;
      v.kb = ka + max(n, kD4Tile);
    }
  };
  auto first_window = [&](Window& v, int j, int us) -> bool {
    if (!piece_at(v, j, us)) return false;
    window_at(v, v.ka);
    return true;
  };
  auto next_window = [&](const Window& c, Window& v) -> bool {
    if (c.kb < c.kend) {
      v = c;
      window_at(v, c.kb);
      return true;
    }
    return first_window(v, walk_next(a, sg, c.b), c.us + c.room);
  };
  // Entries of a window's pages, clamped into the pool: one per thread, K's by the
  // first half of the workgroup; loaded, then put into LDS.
  static_assert(2 * G::kTable <= kD4Threads, "one entry per thread");
  const int half = wave / (kD4Waves / 2), slot_t = tid % (kD4Threads / 2);
  auto fetch_entry = [&](const Window& v) -> int {
    if (v.ka >= v.kb || slot_t > page_of(v.kb - 1) - v.page0) return 0;
    const int col = min(v.page0 + slot_t, fa.table_width - 1);
    return half ? a.v_table[v.b * a.v_table_stride + col]
                : a.k_table[v.b * a.k_table_stride + col];
  };
  auto put_entry = [&](int e, int buf) {
    if (slot_t < G::kTable) tab[buf][half][slot_t] = min(max(e, 0), fa.num_pages - 1);
  };

  // Block-table entries are in LDS for this window (tab[buf]) and the next one, and on
  // their way for the one after.
  Window cur, nxt, nn;
  bool has_next = false, has_nn = false;
  if (!first_window(cur, sg.j, sg.us)) return;
  const int entry0 = fetch_entry(cur);
  int buf = 0;
  auto buf_after = [&](int n) { return buf + n >= 3 ? buf + n - 3 : buf + n; };

  // ---- loads ---------------------------------------------------------------
  const uint8_t* kc = static_cast<const uint8_t*>(a.k);
  const uint8_t* vc = static_cast<const uint8_t*>(a.v);
  const uint32_t hc = kvh * fa.head_codes, hs = kvh * fa.head_scales;
  const uint32_t src = lds_addr_of(tiles) + wave * G::kTile;  // this wave's tile
  // Page and row in it of key nk of a window.
  auto place = [&](int nk, int page0, int tb, int which, uint32_t& off) {
    const int lp = page_of(nk);
    off = nk - lp * a.page_size;
    return static_cast<uint32_t>(tab[tb][which][lp - page0]);
  };
  auto codes_at = [&](int v, uint32_t pg, uint32_t off) {
    return (v ? vc : kc) + (uint64_t(pg) * fa.page_codes + (hc + off));
  };
  auto scales_at = [&](int v, uint32_t pg, uint32_t off) {
    return (v ? fa.vs : fa.ks) + (uint64_t(pg) * fa.page_scales + (hs + off));
  };
  auto load_scales = [&](const uint8_t* p, uint32_t lds) {
    if constexpr (D == 64)
      fp4_dma2(p, lds);
    else
      fp4_dma4(p, lds);
  };
  // The tile at key n < kb of a window, whole rows; a lane's scales are a word: of a
  // key (of half of it at D = 256), lanes below 32 K's, the others V's up to D =
  // 128.  issue_rows: any page size, an address per lane and load; keys past the
  // window are its last one (their weights are zero).
  auto issue_rows = [&](int kb, int page0, int tb, int n) {
    uint32_t off;
#pragma unroll
    for (int v = 0; v < 2; ++v)
#pragma unroll
      for (int i = 0; i < G::kLoads; ++i) {
        const int r = (i * 64 + lane) / G::kNC;
        const uint32_t pg = place(min(n + (v ? G::vkey(r) : r), kb - 1), page0, tb, v, off);
        const int c = (lane % G::kNC) ^ (v ? 0 : G::ksw(r));
        fp4_dma16(codes_at(v, pg, off * G::kRow + c * 16), src + v * G::kCode + i * 1024);
      }
#pragma unroll
    for (int i = 0; i < G::kScaleLoads; ++i) {
      const int v = D == 256 ? i : lane >> 5;
      const int r = D == 256 ? lane >> 1 : lane & 31;
      const uint32_t pg = place(min(n + r, kb - 1), page0, tb, v, off);
      load_scales(scales_at(v, pg, off * (D / 32) + (D == 256 ? 4 * (lane & 1) : 0)),
                  src + 2 * G::kCode + i * 256);
    }
  };
  // issue_blocks: page_size a multiple of 16.  The 16 keys of a block are one run
  // of memory: 16 lanes look up a block each (K's two, V's two), and a load takes
  // its base from theirs.  (Blocks past the window are its last one, rows past
  // it in a block what its page holds.)
  // this lane's place in load i of a block (of both, at D = 64) of K or V
  auto run = [&](int v, int i) -> uint32_t {
    const int r = i * (64 / G::kNC) + lane / G::kNC;
    return (v ? G::vkey(r) : r) * G::kRow + ((lane % G::kNC) ^ (v ? 0 : G::ksw(r))) * 16;
  };
  uint32_t run_k[G::kLoads > 1 ? G::kLoads / 2 : 1], run_v[G::kLoads > 1 ? G::kLoads / 2 : 1];
#pragma unroll
  for (int i = 0; i < (G::kLoads > 1 ? G::kLoads / 2 : 1); ++i) {
    run_k[i] = run(0, i);
    run_v[i] = run(1, i);
  }
  auto issue_blocks = [&](int kb, int page0, int tb, int n) {
    const int top = (kb - 1) & ~15;  // (a window starts at a multiple of 32)
    uint32_t off;
    const uint32_t pg = place(min(n + 16 * (g & 1), top), page0, tb, g >> 1, off);
    if constexpr (D == 64) {  // a load takes both blocks
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        uint32_t o2;
        const uint32_t p2 = place(min(n + 16 * (lane >> 5), top), page0, tb, v, o2);
        fp4_dma16(codes_at(v, p2, (o2 - 16 * (lane >> 5)) * G::kRow + (v ? run_v[0] : run_k[0])),
                  src + v * G::kCode);
      }
    } else {
      const uint64_t at = reinterpret_cast<uint64_t>(codes_at(g >> 1, pg, off * G::kRow));
      const int lo = static_cast<int>(at), hi = static_cast<int>(at >> 32);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        const uint64_t base =
            (static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readlane(hi, 16 * b)))
             << 32) |
            static_cast<uint32_t>(__builtin_amdgcn_readlane(lo, 16 * b));
#pragma unroll
        for (int i = 0; i < G::kLoads / 2; ++i)
          fp4_dma16_base(base, b < 2 ? run_k[i] : run_v[i],
                         src + b * (G::kCode / 2) + i * 1024);
      }
    }
    if constexpr (D == 256) {
#pragma unroll
      for (int v = 0; v < 2; ++v) {
        const int x = lane >> 5;
        const uint32_t p2 = place(min(n + 16 * x, top), page0, tb, v, off);
        load_scales(scales_at(v, p2, off * (D / 32) + 4 * (lane & 31)),
                    src + 2 * G::kCode + v * 256);
      }
    } else {
      load_scales(scales_at(g >> 1, pg, (off + l16) * (D / 32)), src + 2 * G::kCode);
    }
  };
  // The next tile of this wave, in this window or the next one, where there is one.
  int ic = 0, jn = 0;  // its key in either
  bool fly = false;    // whether a tile is on its way
  auto issue_next = [&]() {
    const bool here = ic < cur.kb;
    fly = here || (has_next && jn < nxt.kb);
    if (__builtin_expect(fly, 1)) {
      const int n = here ? ic : jn, kb = here ? cur.kb : nxt.kb;
      const int p0 = here ? cur.page0 : nxt.page0, tb = here ? buf : buf_after(1);
      ic += here ? kStep : 0;
      jn += here ? 0 : kStep;
      if constexpr (BLOCKS)
        issue_blocks(kb, p0, tb, n);
      else
        issue_rows(kb, p0, tb, n);
    }
  };

  // ---- state ---------------------------------------------------------------
  u32x4 q[RB][DJ];
  float m[RB], l[RB];
  f32x4 o[RB][G::kNI];
  uint32_t nans[RB];  // NaN blocks of V that a row sees, by the lane's scales
  // Q^T (B operand): lane row l16, the dims of its group in k-step order
  auto fetch_q = [&](const Window& v, u32x4 (&x)[RB][DJ]) {
    const int64_t base = v.b * a.q_sb + head0 * a.q_sh + q0 * a.q_ss;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int r = 16 * rb + l16;
#pragma unroll
      for (int j = 0; j < DJ; ++j) {
        x[rb][j] = (u32x4){0u, 0u, 0u, 0u};
        if (r < rows)
          x[rb][j] = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(a.q) + base +
                                                     r * a.q_ss + g * (D / 4) + 8 * j);
      }
    }
  };
  auto reset = [&]() {
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = -INFINITY;
      l[rb] = 0.f;
      nans[rb] = 0;
#pragma unroll
      for (int i = 0; i < G::kNI; ++i) o[rb][i] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
  };
  // A wait that the compiler sees: with a value of its own in flight at the head of
  // the tile loop, the first use there would wait for the tiles loaded after it.
  auto settle = [] { __builtin_amdgcn_s_waitcnt(0x0F70); };  // vmcnt(0)

  // places in a tile: this lane's dims of V (rows from there: kRow apart by 4), its
  // scales (of 4 keys, one word each) and the byte in them
  const uint32_t vat = G::kCode + g * G::kRow + l16 * (D / 32);
  const uint32_t vsat = 2 * G::kCode + G::kScale + 4 * g * G::kScaleRow +
                        (D == 256 ? 4 * (l16 >> 3) : 0);
  const uint32_t vbyte = D == 64 ? l16 >> 3 : D == 128 ? l16 >> 2 : (l16 >> 1) & 3;
  const uint32_t vrot = (8 * vbyte + 9) & 31;  // ... turned to a float's exponent

  // This wave's tile, at key n0; kb: the window's end, full: no key
  // below it is hidden from any row, last: the last key that the lane's rows see.
  auto compute = [&](int n0, int kb, int full, const int (&last)[RB]) {
    const bool edge = n0 + kD4Tile > full;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    constexpr int kVW = D == 256 ? 2 : 1;  // words of V of a lane and key
    uint32_t kw[2][DJ], ks[2], vw[8][kVW], vs[8];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = 16 * x + l16;
      const uint32_t row = src + r * G::kRow;
      if constexpr (D == 64) {
        const u32x2 y =
            *(const lds_u32x2_t*)lds_ptr(row + ((g >> 1) ^ G::ksw(r)) * 16 + (g & 1) * 8);
        kw[x][0] = y[0];
        kw[x][1] = y[1];
      } else {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
          const u32x4 y =
              *(const lds_u32x4_t*)lds_ptr(row + ((g * (D / 128) + i) ^ G::ksw(r)) * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) kw[x][4 * i + j] = y[j];
        }
      }
      const uint32_t at = src + 2 * G::kCode + r * G::kScaleRow + g * (D / 4) / 32;
      if constexpr (D == 256)
        ks[x] = *(const lds_u16_t*)lds_ptr(at);
      else
        ks[x] = *(const lds_u8_t*)lds_ptr(at);
      // V: keys 16 x + 4 g ..+3, as the P^T fragment has them
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t va = src + vat + (16 * x + 4 * k) * G::kRow;
        if constexpr (D == 64) {
          vw[4 * x + k][0] = *(const lds_u16_t*)lds_ptr(va);
        } else if constexpr (D == 128) {
          vw[4 * x + k][0] = *(const lds_u32_t*)lds_ptr(va);
        } else {
          const u32x2 y = *(const lds_u32x2_t*)lds_ptr(va);
          vw[4 * x + k][0] = y[0];
          vw[4 * x + k][1] = y[1];
        }
      }
      const uint32_t sa = src + vsat + 16 * x * G::kScaleRow;
      if constexpr (D == 256) {
#pragma unroll
        for (int k = 0; k < 4; ++k) vs[4 * x + k] = *(const lds_u32_t*)lds_ptr(sa + 8 * k);
      } else {
        const u32x4 y = *(const lds_u32x4_t*)lds_ptr(sa);
#pragma unroll
        for (int k = 0; k < 4; ++k) vs[4 * x + k] = y[k];
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the tile is read
    issue_next();

    f32x4 s[RB][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) s[rb][x] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < DJ; ++j) {
        const uint32_t sb = D == 256 ? (j < DJ / 2 ? ks[x] & 255u : ks[x] >> 8) : ks[x];
        const u32x4 kf = fp4_values<BF>(kw[x][j], sb);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb][x] = mma16x32<BF>(kf, q[rb][j], s[rb][x]);
      }
    }
    // scales of V as floats: the byte in the place of the exponent
#pragma unroll
    for (int k = 0; k < 8; ++k)
      vs[k] = __builtin_amdgcn_alignbit(vs[k], vs[k], vrot) & 0x7F800000u;
    // Keys past the end hold anything: zeros.  A block of V that is NaN must
    // not reach the rows that do not see its key (0 * NaN): where drafts may be
    // hidden, zeros, and NaN at the end (nans).
    if (__builtin_expect(edge, 0)) {
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int key = n0 + 16 * (k >> 2) + (k & 3);  // of lane group 0
        const bool in = key + 4 * g < kb;
        const bool bad = in && causal && vs[k] == 0x7F800000u;
        const uint64_t at = __ballot(bad);
        if (at) {
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int gk = 0; gk < 4; ++gk)
#pragma unroll
              for (int u = 0; u < kSub; ++u) {
                // a lane that has the scale of this lane's dims of O
                const int of = D == 64 ? 8 * (g >> 1) : D == 128 ? 4 * g : 4 * g + 2 * u;
                if (key + 4 * gk <= last[rb])
                  nans[rb] |= static_cast<uint32_t>((at >> (16 * gk + of)) & 1) << u;
              }
        }
        if (bad || !in) {
          vs[k] = 0x3F800000u;
#pragma unroll
          for (int j = 0; j < kVW; ++j) vw[k][j] = 0u;
        }
      }
    }
    u32x4 ph[RB], pl[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      if (__builtin_expect(edge, 0)) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int key = n0 + 16 * x + 4 * g + r;
            s[rb][x][r] = key <= last[rb] ? s[rb][x][r] : -INFINITY;
          }
      }
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[rb][x][r]);
      if (__builtin_expect(__any((mx - m[rb]) * a.scale_log2 > kRaise), 0)) {
        mx = over_groups<true>(mx);
        const float mn = fmaxf(m[rb], mx);
        const float alpha = fast_exp2((m[rb] - (mn == -INFINITY ? 0.f : mn)) * a.scale_log2);
        m[rb] = mn;
        l[rb] *= alpha;
#pragma unroll
        for (int i = 0; i < G::kNI; ++i) o[rb][i] *= alpha;
      }
      // (the difference is taken before the scale: no score is too large for it)
      const float mu = m[rb] == -INFINITY ? 0.f : m[rb];
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        float e[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float y = s[rb][x][r] - mu;
          e[r] = fast_exp2(BF ? y * a.scale_log2 : __builtin_fmaf(y, a.scale_log2, kLift));
          l[rb] += e[r];
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t hw = pack2<BF>(e[2 * r], e[2 * r + 1]);
          const f32x2 h = unpack2<BF>(hw);
          const uint32_t lw = pack2<BF>(e[2 * r] - h[0], e[2 * r + 1] - h[1]);
          ph[rb][2 * x + r] = hw;
          pl[rb][2 * x + r] = lw;
        }
      }
    }
    // O^T: dims 2 t and 2 t + 1 of each lane's, 8 keys each
    auto pair_step = [&](auto tc) {
      constexpr int t = decltype(tc)::value;
      uint32_t c[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) c[k] = fp4_pair<BF, t & 3>(vw[k][t >> 2], vs[k]);
      u32x4 va, vb;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        va[k] = __builtin_amdgcn_perm(c[2 * k + 1], c[2 * k], 0x05040100u);
        vb[k] = __builtin_amdgcn_perm(c[2 * k + 1], c[2 * k], 0x07060302u);
      }
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        o[rb][2 * t] = mma16x32<BF>(va, pl[rb], o[rb][2 * t]);
        o[rb][2 * t + 1] = mma16x32<BF>(vb, pl[rb], o[rb][2 * t + 1]);
        o[rb][2 * t] = mma16x32<BF>(va, ph[rb], o[rb][2 * t]);
        o[rb][2 * t + 1] = mma16x32<BF>(vb, ph[rb], o[rb][2 * t + 1]);
      }
    };
    pair_step(std::integral_constant<int, 0>{});
    pair_step(std::integral_constant<int, 1>{});
    if constexpr (D >= 128) {
      pair_step(std::integral_constant<int, 2>{});
      pair_step(std::integral_constant<int, 3>{});
    }
    if constexpr (D == 256) {
      pair_step(std::integral_constant<int, 4>{});
      pair_step(std::integral_constant<int, 5>{});
      pair_step(std::integral_constant<int, 6>{});
      pair_step(std::integral_constant<int, 7>{});
    }
  };

  constexpr bool kAhead = D <= 128;  // the next piece's Q is loaded ahead
  u32x4 qn[RB][kAhead ? DJ : 1];
  fetch_q(cur, q);
  has_next = next_window(cur, nxt);  // (while the first entries are on their way)
  const int entry1 = has_next ? fetch_entry(nxt) : 0;
  if constexpr (kAhead)
    if (has_next) fetch_q(nxt, qn);
  reset();
  put_entry(entry0, 0);
  put_entry(entry1, 1);
  __syncthreads();  // the tables are in LDS

  // ---- pieces' ends ----------------------------------------------------------
  // The waves' states meet in LDS: wave x's row r, kPD dims, at area + x * ws + r *
  // kPitch, its maximum (log2 units) and sum in mrg_ml; added up in wave
  // order and written, to the output or to the piece's part slot.
  auto put_state = [&](auto rbc, auto hc_, uint32_t at) {  // phase h of this lane's row
    constexpr int rb = decltype(rbc)::value, h = decltype(hc_)::value;
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      f32x4 y;
#pragma unroll
      for (int u = 0; u < 4; ++u) y[u] = o[rb][(e + u) % G::kNI][h * G::kRP + (e + u) / G::kNI];
      *(lds_f32x4_t*)lds_ptr(at + 64 * g + 4 * e) = y;
    }
  };
  auto put_stats = [&](auto rbc) {
    constexpr int rb = decltype(rbc)::value;
    if (__any(nans[rb])) {
      const float nan = __builtin_nanf("");
#pragma unroll
      for (int i = 0; i < G::kNI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)  // (two scales at D = 256: dims 64 g + 16 r + i)
          if ((nans[rb] >> (D == 256 ? r >> 1 : 0)) & 1) o[rb][i][r] = nan;
    }
    l[rb] = over_groups<false>(l[rb]);
    if (g == 0) {
      mrg_ml[wave][l16][0] = m[rb] * a.scale_log2;  // (-inf stays -inf)
      mrg_ml[wave][l16][1] = l[rb];
    }
  };
  struct Cut {  // a piece of a cut unit (np 0: none)
    int b, np, us, mine;
  };
  // 16 rows from 16 rb on of the piece cur, n of them, phases H and H + 1, one in each area
  const uint32_t area0 = lds_addr_of(stage), area1 = area0 + kD4Waves * G::kStage;
  constexpr int kTwo = G::kPH > 1 ? 2 : 1;
  bool dirty = false;  // the areas may still be read
  auto add_up = [&](int r0, int n, int h0) {
    const int sd = (tid % 16) * 4;  // 16 threads a row and phase, four dims each
    const int it = tid / 16, hh = it % kTwo, lr = it / kTwo;
    if (lr >= n) return;
    const uint32_t at = (hh ? area1 : area0) + lr * G::kPitch + sd * 4;
    f32x2 ml[kD4Waves];
#pragma unroll
    for (int w = 0; w < kD4Waves; ++w) ml[w] = *reinterpret_cast<const f32x2*>(mrg_ml[w][lr]);
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < kD4Waves; ++w) mt = fmaxf(mt, ml[w][0]);
    const float mu = mt == -INFINITY ? 0.f : mt;
    float lt = 0.f;
    f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kD4Waves; ++w) {
      const float f = fast_exp2(ml[w][0] - mu);
      lt += f * ml[w][1];
      acc += f * *(const lds_f32x4_t*)lds_ptr(at + w * G::kStage);
    }
    const int r = r0 + lr;
    const int dim = G::dim(h0 + hh, sd);
    if (cur.np == 1) {
      // (0/0 -> NaN for a row with no key, as in 16 bits; otherwise lt >= 1)
      const float inv = __builtin_amdgcn_rcpf(lt);
      *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.o) + cur.b * a.o_sb + head0 * a.o_sh +
                                (q0 + r) * a.o_ss + dim) =
          (u32x2){pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv)};
    } else {
      // the slot of this workgroup's piece (walk_slot, without its division)
      const int64_t slot = (static_cast<int64_t>(seg_k) * a.walk_streams + stream) * 2 +
                           (cur.mine == 0 && cur.us != sg.s0);
      const uint32_t pr = static_cast<uint32_t>(a.part_rows);
      __builtin_amdgcn_raw_buffer_store_b128(
          __builtin_bit_cast(u32x4, acc),
          make_rsrc_uniform(a.part_o + slot * pr * D, pr * D * 4), (r * D + dim) * 4, 0, kCpolSc1);
      if (h0 + hh == 0 && sd == 0)
        __builtin_amdgcn_raw_buffer_store_b64(
            (u32x2){__builtin_bit_cast(uint32_t, mt), __builtin_bit_cast(uint32_t, lt)},
            make_rsrc_uniform(a.part_ml + slot * pr * 2, pr * 8), r * 8, 0, kCpolSc1);
    }
  };
  static_assert(kD4Threads / 16 >= 16 * kTwo, "one pass");
  auto merge16 = [&](auto rbc) {
    constexpr int rb = decltype(rbc)::value;
    if (16 * rb >= rows) return;
    const int n = min(rows - 16 * rb, 16);
    auto phases = [&](auto h) {
      constexpr int H = decltype(h)::value;
      if (dirty) __syncthreads();
      if constexpr (H == 0) put_stats(rbc);
      if (l16 < n) {
        const uint32_t at = wave * G::kStage + l16 * G::kPitch;
        put_state(rbc, h, area0 + at);
        if constexpr (G::kPH > 1) put_state(rbc, std::integral_constant<int, H + 1>{}, area1 + at);
      }
      __syncthreads();
      add_up(16 * rb, n, H);
      dirty = true;
    };
    phases(std::integral_constant<int, 0>{});
    if constexpr (G::kPH > 2) phases(std::integral_constant<int, 2>{});
  };
  // Cut units are counted when the workgroup is done: it has two at most, one
  // from each end of its segment.
  Cut cut[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};

  // This wave's first tile of a window: the tiles of consecutive windows go
  // round the waves without a gap, so that none gets more than its share.
  int turn = wave;
  auto turn_after = [&](const Window& v) {
    return (turn - (v.kb - v.ka + kD4Tile - 1) / kD4Tile) & (kD4Waves - 1);
  };
  ic = cur.ka + turn * kD4Tile;
  if (has_next) jn = nxt.ka + turn_after(cur) * kD4Tile;
  issue_next();
  has_nn = has_next && next_window(nxt, nn);  // (while the first tile is on its way)
  int entry = has_nn ? fetch_entry(nn) : 0;
  settle();

  for (;;) {
    const int off = cur.Lk - a.pack_m;
    int last[RB];  // last visible key of this lane's rows
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      last[rb] = causal ? min(cur.kb - 1, off + diag_row(a, q0 + 16 * rb + l16)) : cur.kb - 1;
    const int full = causal ? min(cur.kb, off + 1) : cur.kb;
    for (int n0 = cur.ka + turn * kD4Tile; n0 < cur.kb; n0 += kStep) {
      // The two waves of a SIMD (i and i + 4) take turns in going first: left to
      // itself, the older one finishes its share early and the other is alone.  Without /
      // with, us, runs in turn within 0.1 of each other: 64 x 512-8192 keys 62.25 / 61.2, 33 x
      // 100-4096 with 5 drafts 21.06 / 20.76, 16 x 2000-8192 of D256 26.65 / 26.32, 16 x 8200 with
      // drafts 26.69 / 26.40, 4 x 1023 10.6 / 10.5, 16 x 16000-32768 44.5 both; 4 x 300-600, 8.1 /
      // 8.3.
      if (((n0 / kStep) ^ (wave >> 2)) & 1)
        __builtin_amdgcn_s_setprio(1);
      else
        __builtin_amdgcn_s_setprio(0);
      compute(n0, cur.kb, full, last);
    }
    turn = turn_after(cur);

    const bool piece_end = cur.kb >= cur.kend;
    if (piece_end) {
      if (cur.np > 1) {
        cut[1] = cut[0];
        cut[0] = Cut{cur.b, cur.np, cur.us, cur.mine};
      }
      merge16(std::integral_constant<int, 0>{});
      if constexpr (RB > 1) merge16(std::integral_constant<int, 1>{});
    }
    if (!has_next) break;
    if (piece_end) {
      if constexpr (kAhead) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int j = 0; j < DJ; ++j) q[rb][j] = qn[rb][j];
      } else {
        fetch_q(nxt, q);
      }
      reset();
    }
    cur = nxt;
    nxt = nn;
    has_next = has_nn;
    buf = buf_after(1);
    ic = jn;
    if (has_next) {
      jn = nxt.ka + turn_after(cur) * kD4Tile;
      // (its place was the table of the window before the one that ended, which no
      // wave reads since the last barrier)
      put_entry(entry, buf_after(1));
      __syncthreads();
      dirty = false;
      has_nn = next_window(nxt, nn);
      entry = has_nn ? fetch_entry(nn) : 0;
      if constexpr (kAhead)
        if (nxt.b != cur.b) fetch_q(nxt, qn);
    }
    if constexpr (!kAhead) settle();
    if (!fly) issue_next();  // (this wave had no tile in the window before)
  }
  // the words that count the cut units, read ahead of the count
  uint64_t word = 0;
  if ((tid == 0 && cut[0].np) || (tid == 64 && cut[1].np))
    word = merge_word(a, cut[tid ? 1 : 0].b * a.walk_streams + stream);
  if (cut[0].np == 0) return;
  merge_publish();
  __syncthreads();
  // one wave counts each; the last of a unit's pieces merges them
  if (tid == 0)
    merge_flag[0] = merge_arrive(a, cut[0].b * a.walk_streams + stream, cut[0].np, word);
  if (tid == 64 && cut[1].np)
    merge_flag[1] = merge_arrive(a, cut[1].b * a.walk_streams + stream, cut[1].np, word);
  __syncthreads();
#pragma unroll 1
  for (int i = 0; i < 2; ++i) {
    const Cut c = i ? cut[1] : cut[0];
    if (c.np == 0 || *static_cast<volatile int*>(&merge_flag[i]) == 0) continue;
    if (i) __syncthreads();
    merge_pieces<DT, D, kD4Threads, 16 * RB>(
        a, [&](int s) { return walk_slot(a, sg.C, c.us, stream, s); }, c.np, rows,
        c.b * a.o_sb + head0 * a.o_sh, q0, stage);
  }
}

}  // namespace fa2
