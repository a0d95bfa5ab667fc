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
//     tiles (fa2_decode_walk.h).  A wave walks tiles of 32 keys, tile i of
//     the workgroup's range to wave i % 8, and keeps its own (m, l, O).
//   * A page's rows of a kv head are contiguous: the 16 rows of a block are one
//     run of 8 D bytes, which the 64 lanes load straight in the layout of the
//     MFMA's A operand (lane: row l % 16, D / 4 dims from D / 4 * (l / 16); the
//     queries take the dims of a k-step in the same order).  kRing tiles per
//     wave are in flight in registers, across the ends of the pieces.
//   * S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32, up to 16 RB rows
//     of the unit as columns.  V goes through LDS in 16 bits, as its rows
//     come in and in columns as PV takes them (transpose reads).
//   * P goes to the MFMA as the sum of two 16-bit values, high and low part, so
//     that the weights carry 16 to 22 bits: the MFMAs have the time (a CU's
//     share of the HBM rate is one tile of 4.3 KB in 440 cycles, of which 24
//     MFMAs on four SIMDs take 100), and the output is then off by its own
//     rounding alone.
//   * Running maxima and sums in fp32, raised only when a score passes the
//     maximum by 2^8, as in the 16-bit kernels.
#pragma once

#include "fa2_decode_walk.h"
#include "fa2_kernel_lds.h"

namespace fa2 {

constexpr int kD4Waves = 8;
constexpr int kD4Threads = 64 * kD4Waves;
constexpr int kD4Tile = 32;    // keys of a wave's tile
constexpr int kD4Table = 512;  // block-table entries of a window (K and V each)

typedef __attribute__((address_space(3))) f32x4 lds_f32x4_t;

struct Fp4Args {
  KArgs a;  // a.k, a.v: the codes; a.kv_len: keys a row of the tables can hold
  const uint8_t* ks;  // scales
  const uint8_t* vs;
  int32_t num_pages, table_width;
  uint32_t page_codes, page_scales;  // bytes of a page, and of its rows of one head
  uint32_t head_codes, head_scales;
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

// The 8 values of a code word at the scale with E8M0 byte `sb` (255: NaN).
template <bool BF>
__device__ __forceinline__ u32x4 fp4_values(uint32_t w, uint32_t sb) {
  const float f = __builtin_bit_cast(float, sb << 23);
  if constexpr (BF)
    return (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, f, 3))};
  else
    return (u32x4){
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, f, 3))};
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

// A block of 16 keys' codes in one lane: D / 32 words, and its scale byte(s).
template <int D>
struct Fp4Block {
  uint32_t w[D / 32];
  uint32_t s;
};

template <int D>
__device__ __forceinline__ void fp4_load(Fp4Block<D>& b, const uint8_t* codes,
                                         const uint8_t* scales, uint64_t coff, uint64_t soff,
                                         uint32_t cl, uint32_t sl) {
  const uint8_t* c = codes + coff;
  const uint8_t* s = scales + soff;
  if constexpr (D == 64) {
    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(c + cl));
    b.w[0] = x[0];
    b.w[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < D / 128; ++i) {
      const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(c + cl) + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) b.w[4 * i + j] = x[j];
    }
  }
  if constexpr (D == 256)
    b.s = *reinterpret_cast<const uint16_t*>(s + sl);
  else
    b.s = s[sl];
}

// EVEN: page_size is a multiple of 16, so the 16 keys of a block lie in one
// page: its place is computed on the scalar unit.
template <int DT, int D, int RB, int RING, bool EVEN>
__global__ __launch_bounds__(kD4Threads, 1) void fa2_decode_fp4_kernel(Fp4Args fa) {
  constexpr bool BF = Elt<DT>::kBF;
  constexpr int MODE = kModePagedCapped;
  constexpr int DJ = D / 32;        // S k-steps = code words of a lane = V chunks of a lane
  constexpr int DB = D / 16;        // 16-dim blocks of O^T
  constexpr int kRow = D * 2;       // bytes of a V row in LDS
  constexpr int kVBytes = kD4Tile * kRow;
  constexpr int kPitch = (D + 4) * 4;  // merge rows
  constexpr int kMrg = kD4Waves * 16 * kPitch;
  constexpr int kLds0 = kD4Waves * kVBytes > kMrg ? kD4Waves * kVBytes : kMrg;
  constexpr int kLds =
      kLds0 > kMergePieceBytes<kD4Threads> ? kLds0 : kMergePieceBytes<kD4Threads>;
  constexpr int kStep = kD4Tile * kD4Waves;

  __shared__ __attribute__((aligned(1024))) char lds[kLds];
  __shared__ float mrg_ml[kD4Waves][16][2];
  __shared__ int tab[2][2][kD4Table];
  __shared__ DecSegment seg_sh;
  __shared__ int merge_flag;

  const KArgs& a = fa.a;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15;
  const int g = lane >> 4;
  const bool causal = a.mask != FA2_MASK_NONE;
  const int stream = static_cast<int>(blockIdx.x) % a.walk_streams;
  const int seg_k = static_cast<int>(blockIdx.x) / a.walk_streams;

  if (wave == 0) walk_locate<MODE>(a, seg_k, &seg_sh);
  __syncthreads();
  DecSegment sg;
  sg.j = __builtin_amdgcn_readfirstlane(seg_sh.j);
  sg.us = __builtin_amdgcn_readfirstlane(seg_sh.us);
  sg.s0 = __builtin_amdgcn_readfirstlane(seg_sh.s0);
  sg.s1 = __builtin_amdgcn_readfirstlane(seg_sh.s1);
  sg.C = __builtin_amdgcn_readfirstlane(seg_sh.C);

  // A window: keys [ka, kb) of a piece, all of it unless its block-table
  // entries exceed the LDS table.
  struct Window {
    DecPiece p;
    int ka, kb, kend;  // kend: the piece's end
    int page0;         // first logical page
  };
  auto page_of = [&](int n) { return a.page_shift >= 0 ? n >> a.page_shift : n / a.page_size; };
  auto window_at = [&](Window& v, int ka) {
    v.ka = ka;
    v.kb = v.kend;
    v.page0 = page_of(ka);
    const int64_t lim = (static_cast<int64_t>(v.page0) + kD4Table) * a.page_size;
    if (lim < v.kend) {  // whole tiles, so that every window starts at one
      const int n = (static_cast<int>(lim) - ka) / kD4Tile * kD4Tile;
      v.kb = ka + max(n, kD4Tile);
    }
  };
  auto first_window = [&](Window& v, int j, int us) -> bool {
    if (!walk_piece<MODE>(a, sg, stream, seg_k, j, us, v.p)) return false;
    v.kend = min((v.p.t0 + v.p.T) * kBN, v.p.w.Lk);
    window_at(v, v.p.t0 * kBN);
    return true;
  };
  auto next_window = [&](const Window& c, Window& v) -> bool {
    if (c.kb < c.kend) {
      v = c;
      window_at(v, c.kb);
      return true;
    }
    return first_window(v, walk_next(a, sg, c.p.w.b), c.p.us + c.p.W);
  };
  // entries of the window's pages, clamped into the pool
  auto load_table = [&](const Window& v, int buf) {
    if (v.ka >= v.kb) return;
    const int last = page_of(v.kb - 1);
    for (int i = tid; i <= last - v.page0; i += kD4Threads) {
      const int col = min(v.page0 + i, fa.table_width - 1);
      const int pk = a.k_table[v.p.w.b * a.k_table_stride + col];
      const int pv = a.v_table[v.p.w.b * a.v_table_stride + col];
      tab[buf][0][i] = min(max(pk, 0), fa.num_pages - 1);
      tab[buf][1][i] = min(max(pv, 0), fa.num_pages - 1);
    }
  };

  Window cur, nxt;
  if (!first_window(cur, sg.j, sg.us)) return;
  bool has_next = next_window(cur, nxt);
  load_table(cur, 0);
  if (has_next) load_table(nxt, 1);
  int buf = 0;

  // ---- loads ---------------------------------------------------------------
  struct Tile {
    Fp4Block<D> k[2], v[2];
  };
  Tile ring[RING];
  const uint8_t* kc = static_cast<const uint8_t*>(a.k);
  const uint8_t* vc = static_cast<const uint8_t*>(a.v);
  const uint32_t gdim = g * (D / 8);         // this lane's bytes of a row ...
  const uint32_t gscale = (g * (D / 4)) / 32;  // ... and first scale
  const uint32_t cl = l16 * (D / 2) + gdim;
  const uint32_t sl = l16 * (D / 32) + gscale;
  const uint32_t hc = (stream % a.hkv) * fa.head_codes, hs = (stream % a.hkv) * fa.head_scales;
  struct Source {  // the window that loads are for
    int ka, kb, page0, tb;
  };
  auto source = [](const Window& v, int tb) { return Source{v.ka, v.kb, v.page0, tb}; };
  // The tile of v at key n.  Keys past the window are its last block's or
  // last key's (their weights are zero); a window without keys reads page 0.
  auto issue = [&](Tile& t, const Source& v, int n) {
    const int top = max(v.kb - 1, v.ka);
    const int tb = v.tb;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if constexpr (EVEN) {
        // (16-aligned: ka is a multiple of 32, and so is every tile's start)
        const int nb = min(n + 16 * x, v.ka + ((top - v.ka) & ~15));
        const int lp = page_of(nb);
        const uint32_t off = nb - lp * a.page_size;
        const int slot = v.ka < v.kb ? lp - v.page0 : 0;
        const uint32_t pk = __builtin_amdgcn_readfirstlane(v.ka < v.kb ? tab[tb][0][slot] : 0);
        const uint32_t pv = __builtin_amdgcn_readfirstlane(v.ka < v.kb ? tab[tb][1][slot] : 0);
        const uint32_t oc = hc + off * (D / 2), os = hs + off * (D / 32);
        fp4_load<D>(t.k[x], kc, fa.ks, uint64_t(pk) * fa.page_codes + oc,
                    uint64_t(pk) * fa.page_scales + os, cl, sl);
        fp4_load<D>(t.v[x], vc, fa.vs, uint64_t(pv) * fa.page_codes + oc,
                    uint64_t(pv) * fa.page_scales + os, cl, sl);
      } else {
        const int nk = min(n + 16 * x + l16, top);
        const int lp = page_of(nk);
        const uint32_t off = nk - lp * a.page_size;
        const int slot = v.ka < v.kb ? lp - v.page0 : 0;
        const uint32_t pk = v.ka < v.kb ? tab[tb][0][slot] : 0;
        const uint32_t pv = v.ka < v.kb ? tab[tb][1][slot] : 0;
        const uint32_t oc = hc + off * (D / 2) + gdim, os = hs + off * (D / 32) + gscale;
        fp4_load<D>(t.k[x], kc, fa.ks, uint64_t(pk) * fa.page_codes + oc,
                    uint64_t(pk) * fa.page_scales + os, 0, 0);
        fp4_load<D>(t.v[x], vc, fa.vs, uint64_t(pv) * fa.page_codes + oc,
                    uint64_t(pv) * fa.page_scales + os, 0, 0);
      }
    }
  };

  // ---- state ---------------------------------------------------------------
  u32x4 q[RB][DJ];
  float m[RB], l[RB];
  f32x4 o[RB][DB];
  int q0 = 0, rows = 0;
  // Q^T (B operand): lane row l16, the dims of its group in k-step order
  auto load_q = [&](const Window& v) {
    q0 = v.p.w.qblk * (16 * RB);
    rows = min(v.p.w.Lq - q0, 16 * RB);
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int r = 16 * rb + l16;
#pragma unroll
      for (int j = 0; j < DJ; ++j) {
        q[rb][j] = (u32x4){0u, 0u, 0u, 0u};
        if (r < rows)
          q[rb][j] = *reinterpret_cast<const u32x4*>(
              static_cast<const uint16_t*>(a.q) + v.p.w.q_base +
              static_cast<int64_t>(q0 + r) * a.q_ss + g * (D / 4) + 8 * j);
      }
      m[rb] = -INFINITY;
      l[rb] = 0.f;
#pragma unroll
      for (int d = 0; d < DB; ++d) o[rb][d] = (f32x4){0.f, 0.f, 0.f, 0.f};
    }
  };

  // V in LDS: row r, 32-byte chunk pair p at p ^ vsw(r), so that the 8 rows that 32
  // lanes of a transpose read hit distinct banks
  auto vsw = [](int r) { return D >= 128 ? r & 7 : (r >> 1) & 3; };
  const uint32_t vbuf = lds_addr_of(lds) + wave * kVBytes;
  const int vr = 4 * g + (l16 >> 2);
  const uint32_t voff = vr * kRow + vsw(vr) * 32 + (l16 & 3) * 8;

  auto compute = [&](const Tile& t, int n0, int kb, int full, const int (&last)[RB]) {
    const bool edge = n0 + kD4Tile > full;
    f32x4 s[RB][2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) s[rb][x] = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < DJ; ++j) {
        const uint32_t sb = D == 256 ? (j < DJ / 2 ? t.k[x].s & 255u : t.k[x].s >> 8) : t.k[x].s;
        const u32x4 kf = fp4_values<BF>(t.k[x].w[j], sb);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) s[rb][x] = mma16x32<BF>(kf, q[rb][j], s[rb][x]);
      }
    }
    u32x4 ph[RB], pl[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      if (edge) {
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            s[rb][x][r] = n0 + 16 * x + 4 * g + r <= last[rb] ? s[rb][x][r] : -INFINITY;
      }
      float mx = -INFINITY;
#pragma unroll
      for (int x = 0; x < 2; ++x)
#pragma unroll
        for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[rb][x][r]);
      if (__any((mx - m[rb]) * a.scale_log2 > kRescaleThreshold)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mn = fmaxf(m[rb], mx);
        const float alpha = fast_exp2((m[rb] - (mn == -INFINITY ? 0.f : mn)) * a.scale_log2);
        m[rb] = mn;
        l[rb] *= alpha;
#pragma unroll
        for (int d = 0; d < DB; ++d) o[rb][d] *= alpha;
      }
      // (the difference is taken before the scale: no score is too large for it)
      const float mu = m[rb] == -INFINITY ? 0.f : m[rb];
      float e[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        e[r] = fast_exp2((s[rb][r >> 2][r & 3] - mu) * a.scale_log2);
        l[rb] += e[r];
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        ph[rb][r] = pack2<BF>(e[2 * r], e[2 * r + 1]);
        const uint32_t hw = ph[rb][r];
        const f32x2 h = unpack2<BF>(hw);
        pl[rb][r] = pack2<BF>(e[2 * r] - h[0], e[2 * r + 1] - h[1]);
      }
    }
    // V: 16 bits, to LDS.  Keys past the end hold anything: zeros instead.  A
    // block that is NaN must not reach the rows that do not see its key (0 *
    // NaN): where drafts may be hidden, zeros, and NaN afterwards (nan_keys).
    constexpr int kSub = D == 256 ? 2 : 1;  // scales of a lane
    uint64_t nan_at[2][kSub] = {};
    bool nan_keys = false;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int r = 16 * x + l16;
      uint32_t vw[DJ], vs = t.v[x].s;
#pragma unroll
      for (int j = 0; j < DJ; ++j) vw[j] = t.v[x].w[j];
      if (edge) {
        const bool in = n0 + r < kb;
        bool drop[kSub];
#pragma unroll
        for (int u = 0; u < kSub; ++u) {
          const bool bad = in && causal && ((vs >> (8 * u)) & 255u) == 255u;
          nan_at[x][u] = __ballot(bad);
          nan_keys = nan_keys || nan_at[x][u] != 0;
          drop[u] = bad || !in;
          if (drop[u]) vs = (vs & ~(255u << (8 * u))) | (127u << (8 * u));
        }
#pragma unroll
        for (int j = 0; j < DJ; ++j)
          if (drop[j * kSub / DJ]) vw[j] = 0u;
      }
#pragma unroll
      for (int j = 0; j < DJ; ++j) {
        const uint32_t sb = D == 256 ? (j < DJ / 2 ? vs & 255u : vs >> 8) : vs;
        const int c = g * DJ + j;
        *(lds_u32x4_t*)lds_ptr(vbuf + r * kRow + (((c >> 1) ^ vsw(r)) * 32) + (c & 1) * 16) =
            fp4_values<BF>(vw[j], sb);
      }
    }
    asm volatile("" ::: "memory");  // (a wave's LDS operations are performed in order)
    constexpr int kH = DB / 2;  // half of the V^T fragments are read before their MFMAs
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      u32x4 vf[kH];
#pragma unroll
      for (int d = 0; d < kH; ++d) {
        const uint32_t va = vbuf + (voff ^ (32u * (h * kH + d)));
        const u32x2 lo = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)lds_ptr(va)));
        const u32x2 hi = __builtin_bit_cast(
            u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4i16_t*)lds_ptr(va + 16 * kRow)));
        vf[d] = (u32x4){lo[0], lo[1], hi[0], hi[1]};
      }
#pragma unroll
      for (int d = 0; d < kH; ++d)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
          o[rb][h * kH + d] = mma16x32<BF>(vf[d], pl[rb], o[rb][h * kH + d]);
          o[rb][h * kH + d] = mma16x32<BF>(vf[d], ph[rb], o[rb][h * kH + d]);
        }
    }
    asm volatile("" ::: "memory");
    if (nan_keys) {
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll 1
          for (int k = 0; k < 16; ++k) {
            if (n0 + 16 * x + k > last[rb]) break;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
              // the lane group and scale that hold dims 16 d ..+15
              const int gg = d * 4 / DB, u = kSub == 1 ? 0 : (d / 2) & 1;
              if ((nan_at[x][u] >> (16 * gg + k)) & 1) {
                const float nan = __builtin_nanf("");
                o[rb][d] = (f32x4){nan, nan, nan, nan};
              }
            }
          }
    }
  };

  load_q(cur);
  __syncthreads();  // the tables are in LDS
  // This wave's first tile of a window: the tiles of consecutive windows go
  // round the waves without a gap, so that none gets more than its share.
  int turn = wave;
#pragma unroll
  for (int i = 0; i < RING; ++i) issue(ring[i], source(cur, 0), cur.ka + turn * kD4Tile + i * kStep);

  for (;;) {
    const Work& w = cur.p.w;
    int last[RB];  // last visible key of this lane's rows
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
      last[rb] = causal ? min(cur.kb - 1, w.off + diag_row(a, q0 + 16 * rb + l16)) : cur.kb - 1;
    // no key below this one is hidden from any row
    const int full = causal ? min(cur.kb, w.off + 1) : cur.kb;
    const int turn_next = (turn - (cur.kb - cur.ka + kD4Tile - 1) / kD4Tile) & (kD4Waves - 1);

    // Rounds of RING tiles; a round's slots are loaded again with the next
    // round's tiles, or the next window's first ones, as they are used.
    for (int n0 = cur.ka + turn * kD4Tile;;) {
      const bool more = n0 + RING * kStep < cur.kb;
      const bool here = more || !has_next;
      const int nx = here ? n0 + RING * kStep : nxt.ka + turn_next * kD4Tile;
      const Source src = here ? source(cur, buf) : source(nxt, buf ^ 1);
#pragma unroll
      for (int i = 0; i < RING; ++i) {
        if (n0 + i * kStep < cur.kb) compute(ring[i], n0 + i * kStep, cur.kb, full, last);
        issue(ring[i], src, nx + i * kStep);
      }
      if (!more) break;
      n0 += RING * kStep;
    }
    turn = turn_next;

    if (cur.kb >= cur.kend) {
      // ---- the piece's end: merge the waves' states, 16 rows at a time --------
      const DecPiece& p = cur.p;
      const int64_t slot = p.np == 1 ? 0 : walk_slot(a, sg.C, p.us, stream, p.mine);
      const uint32_t pr = static_cast<uint32_t>(a.part_rows);
      const __amdgpu_buffer_rsrc_t rm = make_rsrc_uniform(a.part_ml + slot * pr * 2, pr * 8);
      const __amdgpu_buffer_rsrc_t ro = make_rsrc_uniform(a.part_o + slot * pr * D, pr * D * 4);
      const uint32_t area = lds_addr_of(lds);
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        if (16 * rb >= rows) break;
        float lw = l[rb];
        lw += __shfl_xor(lw, 16);
        lw += __shfl_xor(lw, 32);
        const float mw = m[rb] * a.scale_log2;  // (-inf stays -inf)
        if (rb > 0) __syncthreads();  // the rows before are read
        if (g == 0) {
          mrg_ml[wave][l16][0] = mw;
          mrg_ml[wave][l16][1] = lw;
        }
        __syncthreads();
        float mg = -INFINITY;
#pragma unroll
        for (int x = 0; x < kD4Waves; ++x) mg = fmaxf(mg, mrg_ml[x][l16][0]);
        const float f = fast_exp2(mw - (mg == -INFINITY ? 0.f : mg));
        const uint32_t po = area + (wave * 16 + l16) * kPitch + 16 * g;
#pragma unroll
        for (int d = 0; d < DB; ++d) *(lds_f32x4_t*)lds_ptr(po + 64 * d) = o[rb][d] * f;
        __syncthreads();
        constexpr int kTPR = D / 4;
        constexpr int kRP = kD4Threads / kTPR;
        const int col = (tid % kTPR) * 4;
        for (int lr = tid / kTPR; lr < 16; lr += kRP) {
          const int r = 16 * rb + lr;
          if (r >= rows) continue;
          float mt = -INFINITY;
#pragma unroll
          for (int x = 0; x < kD4Waves; ++x) mt = fmaxf(mt, mrg_ml[x][lr][0]);
          const float mu = mt == -INFINITY ? 0.f : mt;
          float lt = 0.f;
          f32x4 acc = (f32x4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int x = 0; x < kD4Waves; ++x) {
            lt += mrg_ml[x][lr][1] * fast_exp2(mrg_ml[x][lr][0] - mu);
            acc += *(const lds_f32x4_t*)lds_ptr(area + (x * 16 + lr) * kPitch + col * 4);
          }
          if (p.np == 1) {  // 0/0 -> NaN for a row with no key, as the 16-bit kernels
            const float inv = 1.f / lt;
            *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.o) + w.o_base +
                                      static_cast<int64_t>(q0 + r) * a.o_ss + col) =
                (u32x2){pack2<BF>(acc[0] * inv, acc[1] * inv),
                        pack2<BF>(acc[2] * inv, acc[3] * inv)};
          } else {
            if (col == 0)
              __builtin_amdgcn_raw_buffer_store_b64(
                  (u32x2){__builtin_bit_cast(uint32_t, mt), __builtin_bit_cast(uint32_t, lt)}, rm,
                  r * 8, 0, kCpolSc1);
            __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, acc), ro,
                                                   (r * D + col) * 4, 0, kCpolSc1);
          }
        }
      }
      __syncthreads();  // (also where the unit has no rows in this block)
      if (p.np > 1) {
        merge_publish();
        __syncthreads();
        if (merge_count(a, p.unit, p.np, &merge_flag))
          merge_pieces<DT, D, kD4Threads, 16 * RB>(
              a, [&](int s) { return walk_slot(a, sg.C, p.us, stream, s); }, p.np, rows, w.o_base,
              q0, lds);
      }
      if (has_next) load_q(nxt);
    }
    if (!has_next) return;
    __syncthreads();  // the finished window's table and the merge area are free
    cur = nxt;
    buf ^= 1;
    has_next = next_window(cur, nxt);
    if (has_next) load_table(nxt, buf ^ 1);
    __syncthreads();  // the table (read at this window's end) is in LDS
  }
}

}  // namespace fa2
