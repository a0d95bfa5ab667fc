// fa2_kernel_rows16.h - the decode calls of fa2_kernel_rows.h for units of up to 16 rows
// (16 heads of a latent, a tree of a few drafts): every wave streams tiles of its own.
//
// With 16 rows a K/V byte meets 16 to 30 FLOP: HBM bounds long caches and latency short ones,
// so what counts is that each CU has enough bytes in flight.  One workgroup per CU; tile i of
// its keys goes to wave i % NW, which has one slot of LDS, fills it by itself and keeps its own
// (m, l, O): no barrier stands in the tile loop.  K(t + 1) goes out once S(t) has read K(t),
// V(t + 1) once the second product has read V(t); a latent's row is both, so its next tile goes
// out behind the second product.  v_mfma_f32_16x16x32, rows as columns; at the end of a piece the
// waves' states meet in LDS, in wave order.  Loads are non-temporal (rows are read once).
//
// Measured on MI355X: 16 latents of 16000-32768 keys, 16 heads, 83 us per call (5.3 TB/s; a
// copy reaches 5.1, a plain read 6.9; equal shares end up to 10 % apart), 4 of 700-1100 keys
// 17.4 (the 32-row kernel 26): 1.0 us to locate the segment, 1.4 and 2.2 for block table and Q,
// 4 for the states, 3.9 for the merge.
#pragma once

#include "fa2_kernel_decode_wave.h"
#include "fa2_kernel_rows.h"

namespace fa2 {

constexpr int kR16Rows = 16;

// Waves of a workgroup (one per CU) and keys of a wave's tile.
template <int DK, int DV, bool LAT>
struct Rows16Tile {
  static constexpr int kRow = DK * 2 + (LAT ? 0 : DV * 2);
  static constexpr int kKeys = kRow <= 256 ? 64 : 32;
  static constexpr int kSlot = kRow * kKeys;
  static constexpr int kWaves = kSlot <= 16384 ? 8 : 4;
  static constexpr int kThreads = 64 * kWaves;
};

template <int DT, int DK, int DV, bool LAT, int MODE>
__global__ __launch_bounds__((Rows16Tile<DK, DV, LAT>::kThreads), 1) void
fa2_decode_rows16_kernel(RowsArgs ra) {
  static_assert(DT != FA2_DTYPE_F32, "16-bit rows");
  constexpr bool BF = Elt<DT>::kBF;
  constexpr bool kPaged = MODE == FA2_LAYOUT_PAGED;
  constexpr int LM = kPaged ? kModePagedCapped : MODE;
  using GK = RowsGeo<DK>;
  using GV = RowsGeo<LAT ? DK : DV>;
  using TL = Rows16Tile<DK, DV, LAT>;
  constexpr int NW = TL::kWaves, NT = TL::kThreads, TK = TL::kKeys;
  constexpr int KB = TK / 16;  // 16-key blocks of a tile
  constexpr int KK = TK / 32;  // 32-key PV steps
  constexpr int DJ = DK / 32;  // S k-steps
  constexpr int DB = DV / 16;  // 16-dim blocks of O^T
  constexpr int kKOps = TK / 8 * GK::kGI;  // loads of a tile's K
  constexpr int kVOps = LAT ? 0 : TK / 8 * GV::kGI;
  static_assert(kKOps + kVOps <= 63, "vmcnt field");
  constexpr int kVOff = LAT ? 0 : TK * GK::kRowBytes;
  constexpr int kTab = LAT ? kRbTable : kRbTable / 2;
  constexpr int kPitch = (DV + 4) * 4;  // merge rows
  constexpr float kLift = BF ? 0.f : 7.f;  // as fa2_decode_rows_kernel
  constexpr int R = kR16Rows;

  __shared__ __attribute__((aligned(1024))) char tiles[NW * TL::kSlot];
  __shared__ float mrg_ml[NW][R][2], sum_ml[R][2];
  __shared__ int tab[kPaged ? kRbTable : 1];
  __shared__ uint64_t tree_sh[R];
  __shared__ DecSegment seg_sh;
  static_assert(NW * R * kPitch <= NW * TL::kSlot, "merge in the tile slots");

  const KArgs& a = ra.a;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const int stream = static_cast<int>(blockIdx.x) % a.walk_streams;
  const int seg_k = static_cast<int>(blockIdx.x) / a.walk_streams;

  const RowsWalk walk = rows_locate<LM>(a, seg_k, &seg_sh);
  const DecSegment& sg = walk.sg;
  auto page_of = [&](int n) -> int {
    return static_cast<int>(__umulhi(2u * static_cast<uint32_t>(n), ra.page_mul) >> ra.page_sh);
  };

  // ---- LDS addresses (RowsGeo) -------------------------------------------------
  const uint32_t tiles0 = lds_addr_of(tiles);
  const uint32_t slot = tiles0 + wave * TL::kSlot;
  // K row 16 kb + l16, chunk 4 j + g
  const uint32_t koff = slot + l16 * GK::kRowBytes + ((g ^ GK::swz(l16)) * 16);
  // V rows 4 g + l16 / 4 (and 16 further), dims 16 d + 4 (l16 % 4)
  const int vr = 4 * g + (l16 >> 2);
  const uint32_t voff = slot + kVOff + vr * GV::kRowBytes +
                        ((((l16 & 3) >> 1) ^ GV::swz(vr)) * 16) + (l16 & 1) * 8;
  const uint32_t ksb = static_cast<uint32_t>(a.k_ss * 2), vsb = static_cast<uint32_t>(a.v_ss * 2);
  auto lane_row = [&](auto geo, int i) -> int { return (i * 64 + lane) / decltype(geo)::kNC; };
  auto lane_chunk = [&](auto geo, int i, int grp) -> uint32_t {
    using G = decltype(geo);
    return static_cast<uint32_t>((i * 64 + lane) % G::kNC) ^
           G::swz(8 * (grp & 1) + (i * 64 + lane) / G::kNC);
  };
  // (rows 8 further flip the lowest bit of the chunk)
  uint32_t kl[GK::kGI], vl[LAT ? 1 : GV::kGI];
#pragma unroll
  for (int i = 0; i < GK::kGI; ++i) kl[i] = lane_row(GK{}, i) * ksb + lane_chunk(GK{}, i, 0) * 16;
  if constexpr (!LAT) {
#pragma unroll
    for (int i = 0; i < GV::kGI; ++i)
      vl[i] = lane_row(GV{}, i) * vsb + lane_chunk(GV{}, i, 0) * 16;
  }
  // (the flip as an exclusive or needs row strides of 32 bytes)
  const bool even = (!kPaged || a.page_size % 8 == 0) && ksb % 32 == 0 && vsb % 32 == 0;

  RowsPiece p;
  if (!rows_piece<LM>(a, walk, stream, seg_k, sg.j, sg.us, p)) return;
  for (;;) {
    const int m = l16 % a.pack_m;  // draft
    const int rows = a.q_len;
    int64_t kbase, vbase;
    rows_bases<MODE>(a, p, kbase, vbase);
    const char* kptr = static_cast<const char*>(a.k) + kbase * 2;
    const char* vptr = static_cast<const char*>(a.v) + vbase * 2;

    f32x4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    float m_run = -INFINITY, l_run = 0.f;
    const int off = p.Lk - a.pack_m;  // keys that every row sees
    const int full =
        a.mask == FA2_MASK_NONE ? p.Lk : min(off + (a.mask == kMaskTree ? 0 : 1), p.Lk);
    const int kend = min((p.t0 + p.T) * kBN, p.Lk);
    uint64_t word = 0;

    int ka = p.t0 * kBN, kb, page0;
    RowsTable<LAT, NT> entries;
    auto window = [&]() {  // keys whose block-table entries lie in LDS
      kb = kend;
      page0 = 0;
      if constexpr (kPaged) {
        page0 = page_of(ka);
        const int64_t lim = (static_cast<int64_t>(page0) + kTab) * a.page_size;
        if (lim < kend) kb = ka + max((static_cast<int>(lim) - ka) / kBN * kBN, kBN);
        if (ka < kend) entries.load(ra, p.b, page0, page_of(kb - 1) - page0);
      }
    };
    RowsTree<NW> sees;
    if (a.mask == kMaskTree) {
      if constexpr (LAT) sees.fill(ra, p.b, wave, lane, tree_sh);
      else sees.load(ra, p.b, wave, lane);
    }
    window();
    u32x4 qf[DJ];
    {
      const int qr = min(l16, rows - 1);  // (rows past the last repeat it: not stored)
      const int h = p.kvh * (a.hq / a.hkv) + qr / a.pack_m;
      const uint16_t* src = static_cast<const uint16_t*>(a.q) + p.b * a.q_sb + h * a.q_sh +
                            (qr % a.pack_m) * a.q_ss + g * 8;
#pragma unroll
      for (int j = 0; j < DJ; ++j) qf[j] = *reinterpret_cast<const u32x4*>(src + j * 32);
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

      auto issue = [&](auto is_v, int n0) {
        constexpr bool V = decltype(is_v)::value;
        using G = std::conditional_t<V, GV, GK>;
        const char* base = V ? vptr : kptr;
        const int64_t ss = V ? a.v_ss : a.k_ss;
        const int* tb = tab + (V ? kTab : 0);
        const uint32_t dst = slot + (V ? kVOff : 0);
        if (even && n0 + TK <= kb) {  // groups of 8 rows, each of one page
#pragma unroll
          for (int grp = 0; grp < TK / 8; ++grp) {
            const int n = n0 + 8 * grp;
            int64_t r = n;
            if constexpr (kPaged) {
              const int pg = page_of(n);
              r = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(tb[pg - page0])) * a.page_size +
                  (n - pg * a.page_size);
            }
            const uint64_t sbase = scalar_addr(base + r * (ss * 2));
#pragma unroll
            for (int i = 0; i < G::kGI; ++i)
              rows_dma<true>(sbase, (V ? vl[LAT ? 0 : i] : kl[V ? 0 : i]) ^ (16u * (grp & 1)),
                             dst + (grp * G::kGI + i) * 1024);
          }
          return;
        }
        // a row per lane; places past the window hold its last K row (masked) and zeros of V
        // (kNoValue)
        for (int grp = 0; grp < TK / 8; ++grp) {
#pragma unroll
          for (int i = 0; i < G::kGI; ++i) {
            const int at = n0 + 8 * grp + lane_row(G{}, i), nr = min(at, kb - 1);
            int64_t r = nr;
            if constexpr (kPaged) {
              const int pg = page_of(nr);
              r = static_cast<int64_t>(tb[pg - page0]) * a.page_size + (nr - pg * a.page_size);
            }
            const char* src = base + r * ss * 2 + lane_chunk(G{}, i, grp) * 16;
            if (V && at >= kb) src = reinterpret_cast<const char*>(&kNoValue);
            dma_global_x4<true>(src, dst + (grp * G::kGI + i) * 1024);
          }
        }
      };
      using IsK = std::integral_constant<bool, false>;
      using IsV = std::integral_constant<bool, true>;
      constexpr int kStep = TK * NW;
      int n0 = ka + wave * TK;
      if (n0 < kb) {
        issue(IsK{}, n0);
        if constexpr (!LAT) issue(IsV{}, n0);
      }
      for (; n0 < kb; n0 += kStep) {
        const bool more = n0 + kStep < kb;
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kVOps) : "memory");  // K(t)
        // ---- S^T = K Q^T: lane: row l16, keys 16 kb + 4 g + r ---------------------
        f32x4 s[KB];
#pragma unroll
        for (int x = 0; x < KB; ++x) s[x] = (f32x4){0.f, 0.f, 0.f, 0.f};
        {
          constexpr int kN = DJ * KB, kAhead = 8 < kN ? 8 : kN;
          auto frag = [&](auto kc) -> u32x4 {
            constexpr int j = decltype(kc)::value / KB, x = decltype(kc)::value % KB;
            constexpr int kM = GK::kG / 2;  // k-steps of a swizzle group
            return *(const lds_u32x4_t*)(lds_ptr(koff ^ (64u * (j % kM))) +
                                         x * 16 * GK::kRowBytes + (j / kM) * kM * 64);
          };
          __builtin_amdgcn_sched_barrier(0);
          u32x4 fr[kN];
          static_for<kAhead>([&](auto kc) { fr[decltype(kc)::value] = frag(kc); });
          static_for<kN>([&](auto kc) {
            constexpr int k = decltype(kc)::value, j = k / KB, x = k % KB;
            s[x] = mma16<BF>(fr[k], qf[j], s[x]);
            if constexpr (k + kAhead < kN)
              fr[k + kAhead] = frag(std::integral_constant<int, k + kAhead>{});
          });
          __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
          for (int k = 0; k < kN - kAhead; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          }
          __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        if constexpr (!LAT) {  // the reads of K(t) are complete: its slot takes K(t + 1)
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          if (more) issue(IsK{}, n0 + kStep);
        }
        if (n0 + TK > full) {
#pragma unroll
          for (int x = 0; x < KB; x += 2) {
            const uint32_t sees =
                rows_sees(a, n0 + 16 * x, p.Lk, off, m, word) >> (4 * g);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (!(sees & (1u << ((i >> 2) * 16 + (i & 3))))) s[x + (i >> 2)][i & 3] = -INFINITY;
          }
        }
        // ---- softmax ---------------------------------------------------------------
        float mx = -INFINITY;
#pragma unroll
        for (int x = 0; x < KB; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[x][r]);
        mx *= a.scale_log2;
        if (__any(mx > m_run + kRescaleThreshold)) {
          mx = fmaxf(mx, __shfl_xor(mx, 16));
          mx = fmaxf(mx, __shfl_xor(mx, 32));
          const float mn = fmaxf(m_run, mx);
          const float alpha = fast_exp2(m_run - (mn == -INFINITY ? 0.f : mn));
          m_run = mn;
          l_run *= alpha;
          if (n0 >= p.t0 * kBN + kStep) {  // (nothing yet before the wave's first tile)
#pragma unroll
            for (int d = 0; d < DB; ++d) o[d] *= alpha;
          }
        }
        const float mu = (m_run == -INFINITY ? 0.f : m_run) - kLift;
        u32x4 pf[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
          float e[8];
#pragma unroll
          for (int r = 0; r < 8; ++r)
            e[r] = fast_exp2(__builtin_fmaf(s[2 * kk + (r >> 2)][r & 3], a.scale_log2, -mu));
          pf[kk] = (u32x4){pack2<BF>(e[0], e[1]), pack2<BF>(e[2], e[3]), pack2<BF>(e[4], e[5]),
                           pack2<BF>(e[6], e[7])};
#pragma unroll
          for (int x = 0; x < 4; ++x) l_run = dot2_ones<BF>(pf[kk][x], l_run);
        }
        // ---- O^T += V^T P^T -----------------------------------------------------------
        if constexpr (!LAT) {
          if (more)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kKOps) : "memory");  // V(t)
          else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        {
          constexpr int kN = KK * DB, kAhead = 6 < kN ? 6 : kN;
          constexpr int kM = GV::kG;  // 16-dim blocks of a swizzle group
          auto frag = [&](auto kc) -> u32x4 {
            constexpr int kk = decltype(kc)::value / DB, d = decltype(kc)::value % DB;
            lds_char_t* va = lds_ptr(voff ^ (32u * (d % kM))) + kk * 32 * GV::kRowBytes +
                             (d / kM) * kM * 32;
            const u32x2 lo = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)va));
            const u32x2 up = __builtin_bit_cast(
                u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                           (lds_v4i16_t*)(va + 16 * GV::kRowBytes)));
            return (u32x4){lo[0], lo[1], up[0], up[1]};
          };
          __builtin_amdgcn_sched_barrier(0);
          u32x4 fr[kN];
          static_for<kAhead>([&](auto kc) { fr[decltype(kc)::value] = frag(kc); });
          static_for<kN>([&](auto kc) {
            constexpr int k = decltype(kc)::value, kk = k / DB, d = k % DB;
            o[d] = mma16<BF>(fr[k], pf[kk], o[d]);
            if constexpr (k + kAhead < kN)
              fr[k + kAhead] = frag(std::integral_constant<int, k + kAhead>{});
          });
          __builtin_amdgcn_sched_group_barrier(0x100, 2 * kAhead, 0);
#pragma unroll
          for (int k = 0; k < kN - kAhead; ++k) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          }
          __builtin_amdgcn_sched_group_barrier(0x008, kAhead, 0);
          __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (more) {
          if constexpr (LAT) issue(IsK{}, n0 + kStep);
          else issue(IsV{}, n0 + kStep);
        }
      }
      __syncthreads();  // the window's table and slots have been read
    }

    // ---- the piece's end: the waves' states meet in LDS, in wave order -----------------
    l_run += __shfl_xor(l_run, 16);
    l_run += __shfl_xor(l_run, 32);
    if (g == 0) {
      mrg_ml[wave][l16][0] = m_run;
      mrg_ml[wave][l16][1] = l_run;
    }
    __syncthreads();
    float mg = -INFINITY;
#pragma unroll
    for (int x = 0; x < NW; ++x) mg = fmaxf(mg, mrg_ml[x][l16][0]);
    const float mu = mg == -INFINITY ? 0.f : mg;
    const float f = fast_exp2(m_run - mu);
    if (l16 < rows) {
      const uint32_t po = tiles0 + (wave * R + l16) * kPitch + 16 * g;
#pragma unroll
      for (int d = 0; d < DB; ++d) *(lds_f32x4_t*)(lds_ptr(po) + 64 * d) = o[d] * f;
    }
    if (wave == 0 && g == 0) {
      float lt = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) lt += mrg_ml[x][l16][1] * fast_exp2(mrg_ml[x][l16][0] - mu);
      sum_ml[l16][0] = mg;
      sum_ml[l16][1] = lt;
    }
    __syncthreads();
    const int64_t obase = p.b * a.o_sb + p.kvh * (a.hq / a.hkv) * a.o_sh;
    const int64_t part = p.np == 1 ? 0 : walk_slot(a, sg.C, p.us, stream, p.mine);
    constexpr int kTPR = DV / 4, kRP = NT / kTPR;  // threads of a row, rows at once
    const int col = (tid % kTPR) * 4;
#pragma unroll
    for (int r0 = 0; r0 < R; r0 += kRP) {
      const int r = r0 + tid / kTPR;
      if (r >= rows) break;
      f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < NW; ++x)
        acc += *(const lds_f32x4_t*)(lds_ptr(tiles0 + (x * R + r) * kPitch + col * 4));
      if (p.np == 1) {  // 0/0 -> NaN for a row with no key
        const float inv = 1.f / sum_ml[r][1];
        *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.o) + obase +
                                  static_cast<int64_t>(r) * a.o_ss + col) =
            (u32x2){pack2<BF>(acc[0] * inv, acc[1] * inv), pack2<BF>(acc[2] * inv, acc[3] * inv)};
      } else {
        const int64_t at = part * a.part_rows + r;
        if (col == 0)
          *reinterpret_cast<f32x2*>(a.part_ml + at * 2) = (f32x2){sum_ml[r][0], sum_ml[r][1]};
        *reinterpret_cast<f32x4*>(a.part_o + at * DV + col) = acc;
      }
    }
    if (tid == 0) rows_info(ra, sg, stream, p);
    if (!rows_piece<LM>(a, walk, stream, seg_k, walk_next(a, sg, p.b), p.us + p.W, p)) return;
    __syncthreads();  // the merge area and the mask are free
  }
}

}  // namespace fa2
