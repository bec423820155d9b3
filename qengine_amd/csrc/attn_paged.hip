// Gated flash-decoding over a paged KV cache for a batch of sequences, 1..8 rows each, optionally
// with a sliding window and first tokens that stay visible (include/qe_paged.h).
//
// The arithmetic of a tile is the contiguous decode's (attn_decode.hip, attn_tile.hpp): four waves
// of 32-position tiles, S^T = K Q^T and O^T += V^T P^T on MFMA, K one tile ahead through LDS DMA, V in
// registers. What differs:
//  * A tile is two halves of 16 positions with a buffer resource each, whose base comes from the page
//    table; a lane holds the page of one of the wave's next 64 tiles and readlane hands it out, so the
//    loop waits for no table entry. Pages are powers of two >= 16, so no half crosses a page.
//  * The grid is a list of (sequence, slice, KV head) items that every workgroup derives from pos: a wave
//    scan over the sequences' slice counts. Work goes by the lengths at hand, not by the longest possible.
//  * Slices start at multiples of their size and tiles go to waves by their place in the slice, both
//    counted from position 0. So the rows of a call share a slice whatever their windows, a tile that a
//    row does not attend is an exact no-op for it, and a row's bits depend on no other row or sequence.
//  * Masked tiles (a row's end, the edges of a window, unmapped pages): scores outside are -inf, V rows
//    that no row attends are zeroed, and where a V row that only some rows attend is not finite the
//    product is formed row by row (0 * inf would reach the others).
//  * The output is rounded once: bf16(O / L * sigmoid(gate)) in fp32 (the contiguous decode keeps the
//    rounding points of the reference, which has no paged cache).
#include <algorithm>

#include "attn_split.hpp"
#include "attn_tile.hpp"
#include "qe_paged.h"

namespace qe {
namespace paged {

constexpr int WAVES = 4;
constexpr int MAX_ROWS = 8;
constexpr int MAX_COLS = 32;  // query columns of a workgroup: two MFMA tiles

struct Call {
  int B, R, Hq, Hkv, grp, N, M, lp;  // lp: log2 of the page size
  int cap;                           // positions a table row can hold
  int NS, mins;                      // slots of a row's partials; least slice
  NsDiv nd;
  int window, sinks;
  int rc, hc, hch;                   // rows and heads of a column chunk, head chunks
  uint32_t hkv_m;                    // floor(2^32 / Hkv), or 2^32 - 1
  long ldt, ldp, ldo;
  float scale_log2, v_scale;
};

// ceil(x / d), floor(x / d) for 0 <= x < 2^24, 0 < d: the quotient, correctly rounded to 24 bits, is below
// the next whole number where the exact one is (it is by at least 1 / d > x / d * 2^-24).
__device__ __forceinline__ int div_floor(int x, int d) { return (int)((float)x / (float)d); }
__device__ __forceinline__ int div_ceil(int x, int d) { return div_floor(x + d - 1, d); }

// Slices of the row at position p: size ch, slice i is [i ch, (i + 1) ch). Those of a row without a gap
// between its first tokens and its window are 0 .. cnt - 1; with one, 0 .. nsk - 1 (the first tokens)
// and wlo .. (the window).
struct RowSlices {
  int L, lo;  // attended: [0, min(sinks, L)) and [lo, L)
  int ch, nsk, wlo, cnt;
  bool gap;
};
__device__ __forceinline__ int count_to(const RowSlices& s, int L) {  // slices up to position L
  const int nch = div_ceil(L, s.ch);
  return s.gap ? s.nsk + (s.lo < L ? max(nch - s.wlo, 0) : 0) : nch;
}
__device__ __forceinline__ RowSlices row_slices(const Call& a, int p) {
  RowSlices s;
  s.L = min(p + 1, a.cap);
  s.lo = a.window ? max(p + 1 - a.window, 0) : 0;
  s.gap = s.lo > a.sinks;
  const int V = a.window ? min(s.L, a.sinks + a.window) : s.L;
  s.ch = max(a.mins, split_size(V, a.nd));
  s.nsk = s.gap ? div_ceil(a.sinks, s.ch) : 0;
  s.wlo = s.gap ? max(div_floor(min(s.lo, a.cap), s.ch), s.nsk) : 0;
  s.cnt = count_to(s, s.L);
  return s;
}
// slot of slice i in the row's partials (-1: the row attends nothing there)
__device__ __forceinline__ int slot_of(const RowSlices& s, int i) {
  if (i < s.nsk) return i;
  const int k = i - s.wlo + s.nsk;
  return i >= s.wlo && k < s.cnt ? k : -1;
}

// The slices of a sequence's rows [tc, tc + rn): rows [0, tB) have one size, rows [tB, rn) the next (the
// size is a step function of the length with steps of 32 NS positions or more, and rn <= 8). pos >= 0.
struct SeqItems {
  int tB, nA, nB;
};
__device__ __forceinline__ SeqItems seq_items(const Call& a, int p0, int rn) {
  const RowSlices f = row_slices(a, p0);
  SeqItems q{rn, 0, 0};
  const RowSlices l = row_slices(a, p0 + rn - 1);
  if (f.ch == l.ch) {
    q.nA = count_to(f, l.L);
  } else {
    int t = 1;
    while (row_slices(a, p0 + t).ch == f.ch) ++t;
    q.tB = t;
    q.nA = count_to(f, min(p0 + t, a.cap));
    q.nB = count_to(row_slices(a, p0 + t), l.L);
  }
  return q;
}
// pos as the kernels use it: far past any table it stops growing (no overflow, attends the same)
__device__ __forceinline__ int pos_of(const int* pos, int b) { return min(pos[b], 1 << 30); }

// Inclusive sum over the wave's 64 lanes.
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // row_bcast:15 into rows 1, 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // row_bcast:31 into rows 2, 3
  return v;
}

// One item: rows [r0, r1) of the chunk, slice [beg, end) of sequence b.
struct Item {
  int b, p0;  // position of the chunk's first row
  int r0, r1, slice, beg, end;
};

// The x-th item of the call's chunk of rows [tc, tc + rn); false past the last one. Uniform.
__device__ __forceinline__ bool find_item(const Call& a, const int* pos, int tc, int rn, int x, int lane,
                                          Item& it) {
  const int K = (a.B + WAVE - 1) / WAVE;  // sequences per lane, consecutive
  int mine = 0, p = -1;
  for (int i = 0; i < K; ++i) {
    const int b = lane * K + i;
    p = b < a.B ? pos_of(pos, b) : -1;
    if (p >= 0) {
      const SeqItems q = seq_items(a, p + tc, rn);
      mine += q.nA + q.nB;
    }
  }
  const int upto = wave_scan(mine);
  const int at = __popcll(__ballot(upto <= x));  // the lane whose sequences hold item x
  if (at >= WAVE) return false;
  x -= __builtin_amdgcn_readlane(upto - mine, at);
  SeqItems q;
  for (int i = 0;; ++i) {
    if (i >= K) return false;  // (pos changed meanwhile)
    it.b = at * K + i;
    p = K == 1 ? __builtin_amdgcn_readlane(p, at) : __builtin_amdgcn_readfirstlane(pos_of(pos, it.b));
    if (p >= 0) {
      q = seq_items(a, p + tc, rn);
      q.nA = __builtin_amdgcn_readfirstlane(q.nA);
      q.nB = __builtin_amdgcn_readfirstlane(q.nB);
      if (x < q.nA + q.nB) break;
      x -= q.nA + q.nB;
    }
  }
  it.p0 = p + tc;
  const bool second = x >= q.nA;
  it.r0 = second ? q.tB : 0;
  it.r1 = second ? rn : q.tB;
  const int k = second ? x - q.nA : x;
  const RowSlices s = row_slices(a, it.p0 + it.r0);
  it.slice = __builtin_amdgcn_readfirstlane(k < s.nsk ? k : k - s.nsk + s.wlo);
  const int ch = __builtin_amdgcn_readfirstlane(s.ch);
  it.beg = it.slice * ch;
  it.end = min(it.beg + ch, min(it.p0 + it.r1, a.cap));
  return true;
}

// ---- a tile of the paged cache: two halves of 16 positions, a resource each
struct Halves {
  __amdgpu_buffer_rsrc_t h[2];
};
template <bool KV8>
struct Tile {
  u32x4_t v[8][2];
};
template <>
struct Tile<true> {
  u32x2_t v[8][2];
};

template <bool KV8>
__device__ __forceinline__ void issue_k(uint32_t ks_s, const Halves& r, uint32_t kl) {
  asm volatile("" : "+v"(kl));  // offsets formed at each issue, not kept across the loop
  if constexpr (KV8) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      buffer_load16_to_lds_at(r.h[j >> 2], (kl ^ (64u * (j & 3))) + 1024u * (j & 3), ks_s + 1024u * j);
  } else {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      buffer_load16_to_lds_at(r.h[j >> 3], (kl ^ (32u * (j & 7))) + 1024u * (j & 7), ks_s + 1024u * j);
  }
}
template <bool KV8>
__device__ __forceinline__ void issue_v(Tile<KV8>& t, const Halves& r, uint32_t vl) {
  asm volatile("" : "+v"(vl));
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if constexpr (KV8)
        t.v[e][h] = buffer_load8_stream(r.h[e >> 2], vl + 256u * (e & 3) + 128u * h);
      else
        t.v[e][h] = buffer_load16_stream(r.h[e >> 2], vl + 512u * (e & 3) + 256u * h);
    }
}
__device__ __forceinline__ u32x4_t v_bf16(u32x4_t v) { return v; }
__device__ __forceinline__ u32x4_t v_bf16(u32x2_t v) { return fp8x8_to_bf16x8(v); }
// nonzero where one of the packed values (two bf16, four E4M3FN codes) is infinite or NaN: a carry into the
// sign bit from the exponent (the code) plus one
template <bool KV8>
__device__ __forceinline__ uint32_t not_finite(uint32_t x) {
  return KV8 ? ((x & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u : ((x & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}

// What the masks of an item's tiles need: per column the attended [0, min(sinks, L)) and [lo, L), for
// the item the same of its rows together.
template <int NT>
struct Masks {
  int L[NT], lo[NT], row[NT];  // columns of other rows: L = 0
  int sinks, Lmin, Lmax, lo_min, lo_max;
  bool rows;  // more than one
};

// The masks of a tile: scores outside are -inf, V rows that no row attends are 0. True where a V row that
// some of the rows attend is not finite. bad: halves without a page.
template <int NT, bool KV8>
__device__ __forceinline__ bool mask_tile(Tile<KV8>& b, f32x4_t (&sacc)[NT][2], int p0, int bad,
                                          const Masks<NT>& mk, int g4) {
  uint32_t odd = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int p = p0 + 16 * (e >> 2) + 4 * g4 + (e & 3);
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const bool in = p < mk.L[ct] && (p < mk.sinks || p >= mk.lo[ct]) && !(bad >> (e >> 2) & 1);
      sacc[ct][e >> 2][e & 3] = in ? sacc[ct][e >> 2][e & 3] : -INFINITY;
    }
    const bool any = p < mk.Lmax && (p < mk.sinks || p >= mk.lo_min);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < (KV8 ? 2 : 4); ++i) {
        b.v[e][h][i] = any ? b.v[e][h][i] : 0u;
        odd |= not_finite<KV8>(b.v[e][h][i]);
      }
    }
  }
  return mk.rows && __any(odd);
}

// A masked tile with V values that are not finite, and rows that do not all attend them: 0 * inf in O^T +=
// V^T P^T would reach the rows that do not. The columns that attend such a value get it here, by an MFMA that
// counts +inf, -inf and NaN (weights 1, 64, 4096; a tile has 32 positions), and its place in V becomes 0.
template <int NT, bool KV8>
__device__ __forceinline__ void take_odd(Tile<KV8>& b, const f32x4_t (&sacc)[NT][2],
                                         f32x4_t (&acc)[NT][16]) {
  u32x4_t in[NT];  // 1 where the column attends the position
#pragma unroll
  for (int ct = 0; ct < NT; ++ct)
#pragma unroll
    for (int d = 0; d < 4; ++d)
      in[ct][d] = (sacc[ct][d >> 1][2 * (d & 1)] != -INFINITY ? 0x3f80u : 0u) |
                  (sacc[ct][d >> 1][2 * (d & 1) + 1] != -INFINITY ? 0x3f800000u : 0u);
  const auto kind = [](uint32_t h) __attribute__((always_inline)) {  // a bf16 in the upper half
    const uint32_t m = h & 0x7fff0000u;
    return m < 0x7f800000u ? 0u : m > 0x7f800000u ? 0x4580u : h >> 31 ? 0x4280u : 0x3f80u;
  };
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u32x4_t a;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t x = v_bf16(b.v[2 * d][hh])[i >> 1], y = v_bf16(b.v[2 * d + 1][hh])[i >> 1];
        a[d] = kind(i & 1 ? x & 0xffff0000u : x << 16) | kind(i & 1 ? y & 0xffff0000u : y << 16) << 16;
      }
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const f32x4_t n = mfma16x16x32(as_bf16x8(a), as_bf16x8(in[ct]), f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int z = (int)n[k];
          float v = z & 63 ? INFINITY : 0.f;
          if (z & 0xfc0) v -= INFINITY;  // (inf - inf: NaN)
          if (z >= 4096) v = __builtin_nanf("");
          acc[ct][8 * hh + i][k] += v;
        }
      }
    }
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < (KV8 ? 2 : 4); ++i) {
        // the sign bits not_finite() sets, widened over their values
        const uint32_t o = not_finite<KV8>(b.v[e][h][i]);
        b.v[e][h][i] &= ~(KV8 ? (o >> 7) * 0xffu : (o >> 15) * 0xffffu);
      }
}

// part_o [rows][Hq][NS][256] (unnormalised O), part_ml [rows][Hq][NS][2] = (max in log2 units, sum).
template <int NT, bool KV8>
__global__ void __launch_bounds__(WAVES * WAVE) __attribute__((amdgpu_waves_per_eu(NT == 1 && KV8 ? 2 : 1, 2)))
attn_paged_partials_kernel(const __bf16* __restrict__ q, const char* __restrict__ kp,
                           const char* __restrict__ vp, const int* __restrict__ table,
                           const int* __restrict__ pos, float* __restrict__ part_o,
                           float* __restrict__ part_ml, Call a) {
  constexpr int LROW = KV8 ? 8 : 9;              // log2 of a cache row's bytes
  constexpr int SLOT = TILE << LROW;             // LDS bytes of a K tile
  constexpr int WAREA = 2 * SLOT;                // a wave's two K slots
  constexpr int MERGE = 16 * WAVE * 16;          // a wave's accumulators of one column tile
  static_assert(WAREA >= MERGE, "the merge reuses the K slots");
  __shared__ __attribute__((aligned(256))) char lds[WAVES * WAREA];
  __shared__ float s_m[WAVES][16 * NT], s_l[WAVES][16 * NT];
  const int lane = threadIdx.x & (WAVE - 1);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int c = lane & 15, g4 = lane >> 4;
  const int tc = blockIdx.y / a.hch * a.rc, hc = (blockIdx.y % a.hch) * a.hc;
  const int rn = min(a.rc, a.R - tc), hn = min(a.hc, a.grp - hc), ncols = rn * hn;
  const uint32_t ks_s = lds_byte_uniform(lds + w * WAREA);
  uint32_t kl, vl;
  if constexpr (KV8) {
    const TileLanes8 tl(lane);
    kl = tl.kl, vl = tl.vl;
  } else {
    const TileLanes tl(lane);
    kl = tl.kl, vl = tl.vl;
  }

  bool again = false;
  for (int x = blockIdx.x;; x += gridDim.x) {
    int item = (int)__umulhi((uint32_t)x, a.hkv_m);
    if (x - item * a.Hkv >= a.Hkv) ++item;
    const int g = x - item * a.Hkv;
    Item it;
    if (!find_item(a, pos, tc, rn, item, lane, it)) return;

    // Q^T as the MFMA B operand: column ct*16+c is (row t, head g*grp + hc + j), col = t*hn + j
    bf16x8_t qb[NT][8];
    Masks<NT> mk;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const int col = ct * 16 + c, t = col / hn, j = col - t * hn;
      const bool mine = col < ncols && t >= it.r0 && t < it.r1;
      mk.row[ct] = mine ? t : -1;
      mk.L[ct] = mine ? min(it.p0 + t + 1, a.cap) : 0;
      mk.lo[ct] = a.window ? it.p0 + t + 1 - a.window : 0;
      if (col < ncols) {
        const u32x4_t* src = reinterpret_cast<const u32x4_t*>(
            q + ((size_t)(it.b * a.R + tc + t) * a.Hq + g * a.grp + hc + j) * HD);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qb[ct][ks] = as_bf16x8(src[4 * ks + g4]);
      } else {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qb[ct][ks] = as_bf16x8(u32x4_t{0u, 0u, 0u, 0u});
      }
    }
    mk.rows = it.r1 - it.r0 > 1;
    mk.Lmin = min(it.p0 + it.r0 + 1, a.cap), mk.Lmax = min(it.p0 + it.r1, a.cap);
    mk.lo_min = a.window ? it.p0 + it.r0 + 1 - a.window : 0;
    mk.lo_max = a.window ? it.p0 + it.r1 - a.window : 0;
    mk.sinks = a.window ? a.sinks : 0;

    // The wave's tiles: j = beg / 32 + w, + 4, ..., without those wholly between the first tokens and the
    // windows. Lane i holds the pages of the halves of tile jb + 4 i.
    const int* trow = table + (size_t)it.b * a.ldt;
    const int jlo = max(mk.lo_min, 0) / TILE, jend = (it.end + TILE - 1) / TILE;
    const auto skip = [&](int j) __attribute__((always_inline)) {
      return j < jlo && j * TILE >= mk.sinks ? j + (jlo - j + WAVES - 1) / WAVES * WAVES : j;
    };
    int j = skip(it.beg / TILE + w);
    int jb = 0, pgA = 0, pgB = 0;
    const auto pages_from = [&](int j0) __attribute__((always_inline)) {
      jb = j0;
      const int p = (j0 + WAVES * lane) * TILE;
      const int ia = p >> a.lp, ib = (p + 16) >> a.lp;
      pgA = ia < a.M ? trow[ia] : -1;
      pgB = ib < a.M ? trow[ib] : -1;
    };
    // resources of tile j's halves in both pools; rows at or past the slice's end read 0
    const auto halves = [&](int j, Halves& kh, Halves& vh) __attribute__((always_inline)) {
      const int at = (j - jb) / WAVES, p = j * TILE;
      int bad = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pg = __builtin_amdgcn_readlane(h ? pgB : pgA, at);
        const bool ok = (unsigned)pg < (unsigned)a.N;
        bad |= ok ? 0 : 1 << h;
        const int ph = p + 16 * h, left = ok ? min(max(it.end - ph, 0), 16) : 0;
        const size_t off = (((size_t)(ok ? pg : 0) * a.Hkv + g) << (a.lp + LROW)) +
                           ((size_t)(ph & ((1 << a.lp) - 1)) << LROW);
        kh.h[h] = make_rsrc_uniform(kp + off, (uint32_t)left << LROW);
        vh.h[h] = make_rsrc_uniform(vp + off, (uint32_t)left << LROW);
      }
      return bad;
    };

    float m[NT], l[NT];
    f32x4_t acc[NT][16];  // [8hh + i]: O^T dims 128hh + 32g4 + 8ii + i (tile::pv_half)
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      m[ct] = -INFINITY;
      l[ct] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[ct][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    if (again) lds_barrier();  // the previous item's merge has read every wave's slots
    again = true;

    Tile<KV8> buf;
    const auto compute = [&](uint32_t slot, int j, int bad) __attribute__((always_inline)) {
      const u32x4_t* kt =
          (const u32x4_t*)((__attribute__((address_space(3))) const u32x4_t*)(uintptr_t)slot);
      wave_lds_fence();
      f32x4_t sacc[NT][2];
      if constexpr (KV8)
        qk_tile8<NT>(kt, qb, c, g4, sacc);
      else
        tile::qk_tile<NT, NT == 1, NT == 2 ? 2 : 0>(kt, qb, c, g4, sacc);
      wave_lds_fence();
      const int p = j * TILE;
      if (p + TILE > mk.Lmin || bad || (p < mk.lo_max && p + TILE > mk.sinks)) {
        if (mask_tile<NT, KV8>(buf, sacc, p, bad, mk, g4)) take_odd<NT, KV8>(buf, sacc, acc);
      }
      u32x4_t pb_hi[NT], pb_lo[NT];
      const int none[NT] = {};
      tile::softmax_tile<NT, false, true>(sacc, p, none, a.scale_log2, g4, m, l, acc, pb_hi, pb_lo);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        u32x4_t vr[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) vr[e] = v_bf16(buf.v[e][hh]);
        tile::pv_half<NT, true>(vr, hh, pb_hi, pb_lo, acc);
      }
    };
    if (j < jend) {
      pages_from(j);
      uint32_t cur = ks_s, nxt = ks_s + SLOT;
      Halves kh, vh;
      int bad = halves(j, kh, vh);
      issue_k<KV8>(cur, kh, kl);
      __builtin_amdgcn_sched_barrier(0);
      issue_v<KV8>(buf, vh, vl);
      for (;;) {
        const int jn = skip(j + WAVES);
        const bool more = jn < jend;  // uniform
        int bad_n = 0;
        if (more) {
          if (jn - jb >= WAVES * WAVE) pages_from(jn);
          bad_n = halves(jn, kh, vh);
        }
        vmcnt_wait<16>();  // this tile's K: its V (16 loads) may remain
        __builtin_amdgcn_sched_barrier(0);
        if (more) issue_k<KV8>(nxt, kh, kl);
        __builtin_amdgcn_sched_barrier(0);
        compute(cur, j, bad);
        __builtin_amdgcn_sched_barrier(0);
        if (!more) break;
        issue_v<KV8>(buf, vh, vl);
        j = jn, bad = bad_n;
        const uint32_t t = cur;
        cur = nxt, nxt = t;
      }
    }

    // ---- merge the waves in order 0..3 and write the slice's partial
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      l[ct] = group4_sum(l[ct]);
      if (g4 == 0) {
        s_m[w][ct * 16 + c] = m[ct];
        s_l[w][ct * 16 + c] = l[ct];
      }
    }
    const auto s_acc = [&](int v, int i) __attribute__((always_inline)) -> f32x4_t& {
      return reinterpret_cast<f32x4_t*>(lds + v * WAREA)[i * WAVE + lane];
    };
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const int t = mk.row[ct];
      if (ct > 0) lds_barrier();  // the previous column tile's reads are done
      if (t >= 0) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s_acc(w, i) = acc[ct][i];
      }
      lds_barrier();
      const int sl = t < 0 ? -1 : slot_of(row_slices(a, it.p0 + t), it.slice);
      if (sl >= 0 && sl < a.NS) {
        const int col = ct * 16 + c;
        float M = -INFINITY, wsc[WAVES], L = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; ++v) M = fmaxf(M, s_m[v][col]);
#pragma unroll
        for (int v = 0; v < WAVES; ++v) {
          const float mv = s_m[v][col];
          wsc[v] = mv == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv - M);
          L += s_l[v][col] * wsc[v];
        }
        const int head = g * a.grp + hc + (col - t * hn);
        const size_t at = ((size_t)(it.b * a.R + tc + t) * a.Hq + head) * a.NS + sl;
        if (w == 0 && g4 == 0) {
          part_ml[2 * at] = M;
          part_ml[2 * at + 1] = L;
        }
        const int h = w >> 1, i0 = 4 * (w & 1);
        f32x4_t mo[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int v = 0; v < WAVES; ++v) sum += s_acc(v, 8 * h + i0 + k) * wsc[v];
          mo[k] = sum;
        }
        float* dst = part_o + at * HD + 128 * h + 32 * g4 + i0;
#pragma unroll
        for (int ii = 0; ii < 4; ++ii)
          reinterpret_cast<f32x4_t*>(dst + 8 * ii)[0] =
              f32x4_t{mo[0][ii], mo[1][ii], mo[2][ii], mo[3][ii]};
      }
    }
  }
}

// Merge of a row's slices and the gate: one wave per (head, row, 16 dims), lane = (slot group g of 16,
// 4 dims). A group takes slots s0 + 16 i + g; the groups meet in a fixed tree.
constexpr int CDIMS = 16;
__device__ __forceinline__ float group16_sum(float v) {
  v = xor16_pair(xor32_pair(v, true), true);
  v = v + dpp<0x128>(v);
  return v + dpp<0x1B>(dpp<0x141>(v));
}
__device__ __forceinline__ float group16_max(float v) {
  v = fmaxf(v, dpp<0x128>(v));
  v = fmaxf(v, dpp<0x1B>(dpp<0x141>(v)));
  return xor32_pair(xor16_pair(v, false), false);
}
__global__ void __launch_bounds__(WAVES * WAVE)
attn_paged_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                          const int* __restrict__ pos, const __bf16* __restrict__ qg,
                          __bf16* __restrict__ out, Call a) {
  constexpr int G = 16, U = 4;
  const int lane = threadIdx.x & (WAVE - 1), w = threadIdx.x / WAVE, cd = lane & 3, g = lane >> 2;
  const int h = blockIdx.x, row = blockIdx.y, dim = (blockIdx.z * WAVES + w) * CDIMS + 4 * cd;
  const int b = row / a.R, t = row - b * a.R;
  const int p0 = pos_of(pos, b);
  if (p0 < 0) return;
  const __bf16* gp = qg + (size_t)row * a.ldp + (size_t)h * 2 * HD + HD + dim;
  float gate[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) gate[i] = bf16_to_f32(gp[i]);
  const int cnt = min(row_slices(a, p0 + t).cnt, a.NS);
  const size_t base = ((size_t)row * a.Hq + h) * a.NS;
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f, M = -INFINITY;
  for (int s0 = 0; s0 < cnt; s0 += G * U) {
    f32x4_t po[U];
    float2 ml[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int s = s0 + G * i + g;
      po[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
      ml[i] = make_float2(-INFINITY, 0.f);
      if (s < cnt) {
        po[i] = *reinterpret_cast<const f32x4_t*>(part_o + (base + s) * HD + dim);
        ml[i] = *reinterpret_cast<const float2*>(part_ml + 2 * (base + s));
      }
    }
    const float bm = group16_max(fmaxf(M, fmaxf(fmaxf(ml[0].x, ml[2].x), fmaxf(ml[1].x, ml[3].x))));
    if (bm != M) {
      const float r = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - bm);
      O *= r;
      L *= r;
      M = bm;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const bool use = ml[i].x != -INFINITY;
      const float f = use ? __builtin_amdgcn_exp2f(ml[i].x - M) : 0.f;
      const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
      L += (use ? ml[i].y : 0.f) * f;
      O += (use ? po[i] : zero) * f;
    }
  }
  L = group16_sum(L);
#pragma unroll
  for (int i = 0; i < 4; ++i) O[i] = group16_sum(O[i]);
  if (g == 0) {
    __bf16* op = out + (size_t)row * a.ldo + (size_t)h * HD + dim;
#pragma unroll
    for (int i = 0; i < 4; ++i)  // a row that attends nothing: 0
      op[i] = f32_to_bf16(L == 0.f ? 0.f : (O[i] / L) * a.v_scale * sigmoid_f32(gate[i]));
  }
}

// Least slice of a call: see launch().
static int least_slice(int B, int Hkv) {
  const long units = (long)B * Hkv;
  return units <= 8 ? 32 : units <= 32 ? 128 : 512;
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <bool KV8>
static hipError_t launch(const void* q, const void* kp, const void* vp, const int* table, long ldt,
                         const int* pos, const void* qg, long ldp, float* part_o, float* part_ml,
                         void* out, long ldo, int B, int R, int Hq, int Hkv, int N, int P, int M, int NS,
                         int window, int sinks, float scale, float v_scale, hipStream_t stream) {
  if (B < 1 || B > QE_PAGED_MAX_SEQS || R < 1 || R > MAX_ROWS || Hq < 1 || Hkv < 1 || Hq % Hkv != 0 ||
      N < 1 || P < 16 || P > 32768 || (P & (P - 1)) || M < 1 || (long)M * P > SPLIT_L_MAX - 64 || NS < 1 ||
      window < 0 || window >= SPLIT_L_MAX || (window > 0 && NS < 4) || sinks < 0 || ldt < M ||
      ldp < (long)Hq * 2 * HD || ldo < (long)Hq * HD || !(scale > 0.f) || !(scale <= 3.4e38f) || !q || !kp ||
      !vp || !table || !pos || !qg || !part_o || !part_ml || !out || !aligned16(q) || !aligned16(kp) ||
      !aligned16(vp) || !aligned16(part_o) || (reinterpret_cast<uintptr_t>(part_ml) & 7) ||
      Hkv > 65535 || (long)B * Hkv * NS > 0x3fffffffL)
    return hipErrorInvalidValue;
  Call a{};
  a.B = B, a.R = R, a.Hq = Hq, a.Hkv = Hkv, a.grp = Hq / Hkv, a.N = N, a.M = M;
  a.lp = __builtin_ctz((unsigned)P);
  a.cap = M * P;
  a.NS = NS, a.mins = least_slice(B, Hkv);
  a.window = window, a.sinks = window ? std::min(sinks, a.cap) : 0;
  a.nd = ns_div(window ? NS - 3 : NS);
  a.hch = (a.grp + MAX_COLS - 1) / MAX_COLS;
  a.hc = (a.grp + a.hch - 1) / a.hch;
  const int most = a.hch > 1 ? 1 : std::min(R, MAX_COLS / a.grp), rch = (R + most - 1) / most;
  a.rc = (R + rch - 1) / rch;
  a.hkv_m = Hkv == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / (unsigned)Hkv);
  a.ldt = ldt, a.ldp = ldp, a.ldo = ldo;
  a.scale_log2 = scale * 1.4426950408889634f, a.v_scale = v_scale;
  const long slices = window ? NS : std::min<long>(NS, (a.cap + a.mins - 1) / a.mins);
  const unsigned items = (unsigned)std::min<long>((long)B * slices * Hkv, 4l * compute_units());
  const dim3 grid(items, rch * a.hch), block(WAVES * WAVE);
  const auto* Q = static_cast<const __bf16*>(q);
  const auto *K = static_cast<const char*>(kp), *V = static_cast<const char*>(vp);
  if (a.rc * a.hc <= 16)
    attn_paged_partials_kernel<1, KV8><<<grid, block, 0, stream>>>(Q, K, V, table, pos, part_o, part_ml, a);
  else
    attn_paged_partials_kernel<2, KV8><<<grid, block, 0, stream>>>(Q, K, V, table, pos, part_o, part_ml, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  attn_paged_combine_kernel<<<dim3(Hq, B * R, HD / CDIMS / WAVES), block, 0, stream>>>(
      part_o, part_ml, pos, static_cast<const __bf16*>(qg), static_cast<__bf16*>(out), a);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace qe

using namespace qe;

extern "C" hipError_t qe_attn_decode_paged(const void* q, const void* kp, const void* vp,
                                           const int* table, long ldt, const int* pos, const void* qg,
                                           long ldp, float* part_o, float* part_ml, void* out, long ldo,
                                           int B, int R, int Hq, int Hkv, int N, int P, int M, int NS,
                                           int window, int sinks, float scale, hipStream_t stream) {
  return paged::launch<false>(q, kp, vp, table, ldt, pos, qg, ldp, part_o, part_ml, out, ldo, B, R, Hq,
                              Hkv, N, P, M, NS, window, sinks, scale, 1.f, stream);
}

extern "C" hipError_t qe_attn_decode_paged_fp8(const void* q, const void* kp, const void* vp,
                                               const int* table, long ldt, const int* pos,
                                               const void* qg, long ldp, float* part_o, float* part_ml,
                                               void* out, long ldo, int B, int R, int Hq, int Hkv, int N,
                                               int P, int M, int NS, int window, int sinks, float scale,
                                               float k_scale, float v_scale, hipStream_t stream) {
  if (!kv_scale_ok(k_scale) || !kv_scale_ok(v_scale)) return hipErrorInvalidValue;
  return paged::launch<true>(q, kp, vp, table, ldt, pos, qg, ldp, part_o, part_ml, out, ldo, B, R, Hq,
                             Hkv, N, P, M, NS, window, sinks, scale * k_scale, v_scale, stream);
}
