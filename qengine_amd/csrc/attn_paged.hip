// Gated flash-decoding over a paged KV cache for a batch of sequences, 1..8 rows each, optionally
// with a sliding window and first tokens that stay visible (include/qe_paged.h).
//
// The arithmetic of a tile is the contiguous decode's (attn_decode.hip, attn_tile.hpp): tiles of 32
// positions a wave, S^T = K Q^T and O^T += V^T P^T on MFMA, K one tile ahead through LDS DMA, V in
// registers. It streams the cache: 6 flops a byte at 6 heads a group, so HBM bounds it (64 sequences of up to
// 8,000 positions, 24 / 4 heads, bf16: 718 MB in 128 us, 5.6 TB/s with both launches; one of
// 131,000, fp8: 268 MB in 49 us), and short calls its two launches (one sequence of 1,000: 9.2 us). What differs:
//  * A tile's buffer resources have their base from the page table, read a tile ahead. Pages are powers of two;
//    with pages of 16 positions a tile is two halves with a resource each.
//  * In a batch every wave is a worker of its own: persistent waves take equal parts of the call's work, which
//    each derives from pos (a wave scan over the sequences' tiles), and write a slice's partial without meeting
//    the others. With four waves a slice and a merge per slice instead, the waves wait for one another and items
//    are four times as coarse (7 sequences of up to 24,011 positions 43.9 us against 39.0; 64 of up to 8,000
//    132.6 / 129.4; 32 with a window of 4,096 100.3 / 103.2).
//  * The parts go by the lengths at hand; the least slice and the form of the call by what the tables can hold
//    (plan()), so that short sequences in wide tables are cut coarsely (2 of 1,000, 24 / 4 heads, tables of 1,024 /
//    8,192 / 131,072 positions: 9.7 / 12.4 / 17.0 us).
//  * Above 32 query columns (rows times heads a group) the rows are cut into chunks, each a pass over the cache
//    (16 sequences of 4,000, 24 / 4 heads, bf16, 5 / 6 rows: 61.5 / 91.4 us).
//  * Slices start at multiples of their size and tiles go to waves by their place in the slice, both
//    counted from position 0. So the rows of a call share a slice whatever their windows, a tile that a
//    row does not attend is an exact no-op for it, and a row's bits depend on no other row or sequence.
//  * Masked tiles (a row's end, the edges of a window, unmapped pages): scores outside are -inf, V rows
//    that no row attends are zeroed, and a V value that only some rows attend and that is not finite is
//    taken apart (take_odd; 0 * inf would reach the others). What an attended value of that kind makes of
//    the output is decided by the merge (odd_values).
//  * The output is rounded once: bf16(O / L * sigmoid(gate)) in fp32 (the contiguous decode keeps the
//    rounding points of the reference, which has no paged cache).
#include <algorithm>
#include <type_traits>

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
  int NS, mins, most;                // slots of a row's partials; least slice; slices that a row can have
  NsDiv nd;
  int window, sinks;
  int rc, hc, hch;                   // rows and heads of a column chunk, head chunks
  int parts;                         // waves, or (few items) workgroups, of a KV head
  uint32_t hkv_m;                    // floor(2^32 / Hkv), or 2^32 - 1
  long ldt, ldp, ldo;
  size_t rh;                         // rows times heads
  float scale_log2, v_scale;
};

// floor(x / d), ceil(x / d) for 0 <= x < 2^24, d >= 32: the estimate is off by less than one (the reciprocal
// and the product by 2^-22 of x / d < 2^19), then corrected.
__device__ __forceinline__ int div_floor(int x, int d) {
  int q = (int)((float)x * __builtin_amdgcn_rcpf((float)d));
  const int r = x - q * d;
  q += r >= d;
  return q - (r < 0);
}
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
// split_size, above 128 positions (a tile for every wave) in multiples of 128
__device__ __forceinline__ int slice_size(const Call& a, int L) {
  constexpr int ALL = WAVES * TILE;
  const int ch = split_size(L, a.nd);
  return max(a.mins, ch <= ALL ? ch : (ch + ALL - 1) / ALL * ALL);
}
__device__ __forceinline__ RowSlices row_slices(const Call& a, int p) {
  RowSlices s;
  s.L = min(p + 1, a.cap);
  s.lo = s.nsk = s.wlo = 0, s.gap = false;
  if (a.window) {
    s.lo = max(p + 1 - a.window, 0);
    s.gap = s.lo > a.sinks;
    s.ch = slice_size(a, min(s.L, a.sinks + a.window));
    if (s.gap) {
      s.nsk = div_ceil(a.sinks, s.ch);
      s.wlo = max(div_floor(min(s.lo, a.cap), s.ch), s.nsk);
    }
  } else {
    s.ch = slice_size(a, s.L);
  }
  s.cnt = count_to(s, s.L);
  return s;
}
// slot of slice i in the row's partials (-1: the row attends nothing there)
__device__ __forceinline__ int slot_of(const RowSlices& s, int i) {
  if (i < s.nsk) return i;
  const int k = i - s.wlo + s.nsk;
  return i >= s.wlo && k < s.cnt ? k : -1;
}

// The items of a sequence's rows at positions p0 .. p0 + rn - 1 (p0 >= 0): the slices of rows [0, tB), which
// have one size, then those of rows [tB, rn), which have the next (the size is a step function of the length
// with steps of 32 NS positions or more, and rn <= 8).
struct SeqItems {
  RowSlices f;  // of the first row
  int tB, nA, n;
};
__device__ __forceinline__ SeqItems seq_items(const Call& a, int p0, int rn) {
  SeqItems q;
  q.f = row_slices(a, p0);
  q.tB = rn, q.nA = q.n = q.f.cnt;
  if (rn > 1) {
    const RowSlices l = row_slices(a, p0 + rn - 1);
    if (q.f.ch == l.ch) {
      q.nA = q.n = count_to(q.f, l.L);
    } else {
      int t = 1;
      while (row_slices(a, p0 + t).ch == q.f.ch) ++t;
      q.tB = t;
      q.nA = count_to(q.f, min(p0 + t, a.cap));
      q.n = q.nA + count_to(row_slices(a, p0 + t), l.L);
    }
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

// One item: rows [r0, r1) of the chunk (whose first row is at position p0), slice [beg, end) of sequence b.
struct Item {
  int b, p0, r0, r1, slice, beg, end;
};

__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Where a workgroup is in a sequence's items (SeqItems, in scalar registers).
struct Cursor {
  Item it;
  int k, nA, n, tB;      // the item's number
  int ch, nsk, wlo, lo;  // the first row's slices
  int at, len, hi;       // (parts of a line, below)
};
__device__ __forceinline__ void place_item(const Call& a, int rn, Cursor& c) {
  int k = c.k, nsk = c.nsk, wlo = c.wlo, ch = c.ch;
  c.it.r0 = 0, c.it.r1 = c.tB;
  if (k >= c.nA) {
    const RowSlices s = row_slices(a, c.it.p0 + c.tB);
    k -= c.nA, nsk = uni(s.nsk), wlo = uni(s.wlo), ch = uni(s.ch);
    c.it.r0 = c.tB, c.it.r1 = rn;
  }
  c.it.slice = k < nsk ? k : k - nsk + wlo;
  c.it.beg = c.it.slice * ch;
  c.it.end = min(c.it.beg + ch, min(c.it.p0 + c.it.r1, a.cap));
}

// The items of a batch: a sequence's lie along a line, one after another, each as long as its tiles plus
// OVER, and the sequences follow one another. Wave i of a KV head takes the items that begin in the i-th
// of equal parts of the line. Places count from the part's begin.
constexpr int OVER = 2;  // what an item costs beside its tiles, in tiles

// A sequence's length on the line: a little more than its tiles, and OVER for each item.
__device__ __forceinline__ int line_of(const Call& a, const SeqItems& q, int p0, int rn) {
  const int last = min(p0 + rn, a.cap);
  const int tiles = q.f.gap ? max(last - q.f.lo, 0) / TILE + a.sinks / TILE + 2 : (last + TILE - 1) / TILE;
  return q.n * OVER + tiles;
}
__device__ __forceinline__ int place_of(const Call& a, const Cursor& c) {
  const int tiles = c.k < c.nsk || c.nsk + c.wlo == 0
                        ? c.k * c.ch / TILE
                        : a.sinks / TILE + 1 + max((c.wlo + c.k - c.nsk) * c.ch - c.lo, 0) / TILE;
  return c.at + min(c.k * OVER + tiles, c.len - 1);
}

// The call's sequences as a wave holds them: up to 64, one a lane, with their items. Beyond that a lane has several
// consecutive ones and only their length on the line; an item's sequence is then looked up again.
struct Lanes {
  int K;                 // sequences a lane
  int p, n, nA, tB, ch, nsk, wlo, lo, len;  // (one a lane) of its sequence; p < 0: idle
  int upto;              // place on the line where the lane's sequences end
};
__device__ __forceinline__ void lane_seq(const Call& a, Lanes& l, int p, int rn) {
  const SeqItems q = seq_items(a, p, rn);
  l.n = q.n, l.nA = q.nA, l.tB = q.tB;
  l.ch = q.f.ch, l.nsk = q.f.nsk, l.wlo = q.f.wlo, l.lo = q.f.lo;
  l.len = line_of(a, q, p, rn);
}
__device__ __forceinline__ Lanes lanes_of(const Call& a, const int* pos, int tc, int rn, int lane) {
  Lanes l{};
  l.K = (a.B + WAVE - 1) / WAVE;
  l.p = -1;
  int mine = 0;
  for (int s = 0; s < l.K; ++s) {
    const int b = lane * l.K + s;
    l.p = b < a.B ? pos_of(pos, b) : -1;
    l.n = l.len = 0;
    if (l.p >= 0) lane_seq(a, l, l.p += tc, rn);
    mine += l.len;
  }
  l.upto = wave_scan(mine);
  return l;
}
// Opens sequence b at its item 0; false if it is idle.
__device__ __forceinline__ bool open_sequence(const Call& a, const Lanes& l, const int* pos, int tc, int rn, int b,
                                              Cursor& c) {
  const auto at = [&](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, b); };
  c.it.b = b, c.k = 0;
  if (l.K == 1) {
    c.it.p0 = at(l.p), c.n = at(l.n), c.nA = at(l.nA), c.tB = at(l.tB);
    c.ch = at(l.ch), c.nsk = at(l.nsk), c.wlo = at(l.wlo), c.lo = at(l.lo), c.len = at(l.len);
    return c.it.p0 >= 0;
  }
  const int p = uni(pos_of(pos, b));
  if (p < 0) {
    c.n = c.len = 0;
    return false;
  }
  Lanes one{};
  lane_seq(a, one, p + tc, rn);
  c.it.p0 = p + tc, c.n = uni(one.n), c.nA = uni(one.nA), c.tB = uni(one.tB);
  c.ch = uni(one.ch), c.nsk = uni(one.nsk), c.wlo = uni(one.wlo), c.lo = uni(one.lo), c.len = uni(one.len);
  return true;
}
// The cursor's item, if it begins in the part. At the end of a sequence: the next one's first.
__device__ __forceinline__ bool take_item(const Call& a, const Lanes& l, const int* pos, int tc, int rn,
                                          Cursor& c) {
  while (c.k >= c.n) {
    c.at += c.len;
    const int b = c.it.b + 1;
    if (b >= a.B) return false;
    open_sequence(a, l, pos, tc, rn, b, c);  // (an idle one has no items)
  }
  if (place_of(a, c) >= c.hi) return false;
  place_item(a, rn, c);
  return true;
}
// The first item of part i of `parts`.
__device__ __forceinline__ bool first_item(const Call& a, const Lanes& l, const int* pos, int tc, int rn, int i,
                                           int parts, Cursor& c) {
  const int total = __builtin_amdgcn_readlane(l.upto, WAVE - 1);
  const int part = uni((int)(((unsigned)total + parts - 1) / (unsigned)parts)), lo = i * part;
  c.hi = min(part, total - lo);
  const int at = __popcll(__ballot(l.upto <= lo));  // the lane whose sequences hold the part's begin
  if (lo >= total || at >= WAVE) return false;
  c.at = (at > 0 ? __builtin_amdgcn_readlane(l.upto, at - 1) : 0) - lo;
  for (int s = 0;; ++s) {
    const int b = at * l.K + s;
    if (s >= l.K || b >= a.B) return false;  // (pos changed meanwhile)
    if (open_sequence(a, l, pos, tc, rn, b, c) && c.at + c.len > 0) break;
    c.at += c.len;
  }
  // the first item from the part's begin on: an estimate, then steps
  c.k = min(max(-c.at, 0) / (c.ch / TILE + OVER), c.n);
  while (c.k > 0 && (c.k >= c.n || place_of(a, c) >= 0)) --c.k;
  while (c.k < c.n && place_of(a, c) < 0) ++c.k;
  return take_item(a, l, pos, tc, rn, c);
}

// ---- a tile of the paged cache: one buffer resource, or with pages of 16 positions (P16) one for each half
struct Rsrc {
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

template <bool KV8, bool P16>
__device__ __forceinline__ void issue_k(uint32_t ks_s, const Rsrc& r, uint32_t kl) {
  asm volatile("" : "+v"(kl));  // offsets formed at each issue, not kept across the loop
  constexpr int N = KV8 ? 8 : 16, HALF = P16 ? N / 2 : N, SWZ = KV8 ? 64 : 32, CYC = KV8 ? 4 : 8;
#pragma unroll
  for (int j = 0; j < N; ++j)
    buffer_load16_to_lds_at(r.h[j / HALF], (kl ^ (SWZ * (j % CYC))) + 1024u * (j % HALF), ks_s + 1024u * j);
}
template <bool KV8, bool P16>
__device__ __forceinline__ void issue_v(Tile<KV8>& t, const Rsrc& r, uint32_t vl) {
  asm volatile("" : "+v"(vl));
  constexpr uint32_t ROW = KV8 ? 256 : 512;
#pragma unroll
  for (int e = 0; e < 8; ++e)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t off = vl + ROW * (e & 3) + ROW / 2 * h + (P16 ? 0 : 16 * ROW * (e >> 2));
      if constexpr (KV8)
        t.v[e][h] = buffer_load8_stream(r.h[P16 ? e >> 2 : 0], off);
      else
        t.v[e][h] = buffer_load16_stream(r.h[P16 ? e >> 2 : 0], off);
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
  int L[NT], lo[NT];  // columns of other rows: L = 0
  int sinks, Lmin, Lmax, lo_min, lo_max;
  bool rows;  // more than one
};

// The masks of a tile: scores outside are -inf, V rows that no row attends are 0. True where a V row that
// some of the rows attend is not finite. bad: halves without a page. in: bit e where the column attends.
template <int NT, bool KV8>
__device__ __forceinline__ bool mask_tile(Tile<KV8>& b, f32x4_t (&sacc)[NT][2], int p0, int bad,
                                          const Masks<NT>& mk, int g4, uint32_t (&in)[NT]) {
  uint32_t odd = 0;
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) in[ct] = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int p = p0 + 16 * (e >> 2) + 4 * g4 + (e & 3);
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const bool on = p < mk.L[ct] && (p < mk.sinks || p >= mk.lo[ct]) && !(bad >> (e >> 2) & 1);
      sacc[ct][e >> 2][e & 3] = on ? sacc[ct][e >> 2][e & 3] : -INFINITY;
      in[ct] |= on ? 1u << e : 0u;
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
// V^T P^T would reach the rows that do not. The columns that attend such a value get a NaN here, as an unmasked
// tile's product gives them, by an MFMA that counts these values, and its place in V becomes 0.
template <int NT, bool KV8>
__device__ __forceinline__ void take_odd(Tile<KV8>& b, uint32_t (&bits)[NT], f32x4_t (&acc)[NT][16]) {
  u32x4_t in[NT];  // 1 where the column attends the position
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    asm volatile("" : "+v"(bits[ct]));  // (as bits: kept as comparisons they would cost scalar registers)
#pragma unroll
    for (int d = 0; d < 4; ++d)
      in[ct][d] = (bits[ct] >> (2 * d) & 1 ? 0x3f80u : 0u) | (bits[ct] >> (2 * d + 1) & 1 ? 0x3f800000u : 0u);
  }
  const auto odd = [](uint32_t h) __attribute__((always_inline)) {  // a bf16 in the upper half
    return (h & 0x7fff0000u) < 0x7f800000u ? 0u : 0x3f80u;
  };
#pragma unroll
  for (int hh = 0; hh < 2; ++hh)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u32x4_t a;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        const uint32_t x = v_bf16(b.v[2 * d][hh])[i >> 1], y = v_bf16(b.v[2 * d + 1][hh])[i >> 1];
        a[d] = odd(i & 1 ? x : x << 16) | odd(i & 1 ? y : y << 16) << 16;
      }
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const f32x4_t n = mfma16x16x32(as_bf16x8(a), as_bf16x8(in[ct]), f32x4_t{0.f, 0.f, 0.f, 0.f});
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[ct][8 * hh + i][k] = n[k] > 0.f ? __builtin_nanf("") : acc[ct][8 * hh + i][k];
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

// Place of a partial's dims in its 256 floats: [half][ii][i / 4][g4][i % 4] for dim 128 half + 32 g4 + 8 ii + i, so
// that a store of the accumulators' lanes (c, g4) writes 64 bytes on end, not 16 in each of four lines.
__device__ __forceinline__ int dim_of(int at) {  // of the first of 4 floats
  return (at & 128) + 32 * (at >> 2 & 3) + 8 * (at >> 5 & 3) + 4 * (at >> 4 & 1);
}

// part_o [NS][rows][Hq][256] (unnormalised O, dim_of), part_ml [NS][rows][Hq][2] = (max in log2 units, sum).
// BATCH: persistent waves that take a part of the call's items each. While a wave computes the last tile of an
// item, K of its first tile of the next one is on its way, and V while it stores the partial, so that the
// memory latency of an item's begin is paid once. Otherwise (few items) four waves are a workgroup and an
// item is (slice, KV head; sequence), without the search for it.
template <int NT, bool KV8, bool P16, bool BATCH>
__global__ void __launch_bounds__(WAVES * WAVE) __attribute__((amdgpu_waves_per_eu(NT == 1 && KV8 ? 2 : 1, 2)))
attn_paged_partials_kernel(const __bf16* __restrict__ q, const char* __restrict__ kp,
                           const char* __restrict__ vp, const int* __restrict__ table,
                           const int* __restrict__ pos, float* __restrict__ part_o,
                           float* __restrict__ part_ml, Call a) {
  constexpr int WPI = BATCH ? 1 : WAVES;         // waves of an item
  constexpr int LROW = KV8 ? 8 : 9;              // log2 of a cache row's bytes
  constexpr int SLOT = TILE << LROW;             // LDS bytes of a K tile
  // The merge of four waves takes rounds of MACC accumulators of one column tile per wave, through the K slot that
  // the wave's last tile left. An fp8 slot holds half of them; with two column tiles, where registers allow one
  // workgroup per CU, there is room for buffers of their own.
  constexpr bool OWN = KV8 && NT == 2 && !BATCH;
  constexpr int HALVES = KV8 && !OWN ? 2 : 1, MACC = 16 / HALVES;
  static_assert(BATCH || OWN || MACC * WAVE * 16 == SLOT, "a round of the merge fills a K slot");
  __shared__ __attribute__((aligned(256))) char lds[WAVES * (2 * SLOT + (OWN ? MACC * WAVE * 16 : 0))];
  __shared__ __attribute__((aligned(16))) float s_ml[16 * NT][2][WAVES];  // (m, l) of a column's waves
  __shared__ __attribute__((aligned(16))) uint32_t s_slot[WAVES];
  const int lane = threadIdx.x & (WAVE - 1);
  const int w = uni(threadIdx.x / WAVE);
  const int c = lane & 15, g4 = lane >> 4;
  const int tc = blockIdx.y / a.hch * a.rc, hc = (blockIdx.y % a.hch) * a.hc;
  const int rn = min(a.rc, a.R - tc), hn = min(a.hc, a.grp - hc), ncols = rn * hn;
  int i = (int)__umulhi(blockIdx.x, a.hkv_m);
  if ((int)blockIdx.x - i * a.Hkv >= a.Hkv) ++i;
  const int g = blockIdx.x - i * a.Hkv;
  uint32_t cur = lds_byte_uniform(lds + w * 2 * SLOT), nxt = cur + SLOT;
  uint32_t kl, vl;
  if constexpr (KV8) {
    const TileLanes8 tl(lane);
    kl = tl.kl, vl = tl.vl;
  } else {
    const TileLanes tl(lane);
    kl = tl.kl, vl = tl.vl;
  }
  Cursor cu;
  Lanes lanes{};
  if constexpr (BATCH) {
    lanes = lanes_of(a, pos, tc, rn, lane);
    if (!first_item(a, lanes, pos, tc, rn, i * WAVES + w, a.parts, cu)) return;
  } else {
    const int p = pos_of(pos, blockIdx.z);
    if (p < 0) return;
    const int far = min(p + tc + rn, a.cap), ch = slice_size(a, far);
    if (!a.window && ch == slice_size(a, min(p + tc + 1, a.cap))) {  // slice i, if it is there (cu.n: no further one)
      if (i * ch >= far) return;
      cu.k = cu.n = 0;
      cu.it = Item{(int)blockIdx.z, p + tc, 0, rn, i, i * ch, min(i * ch + ch, far)};
    } else {
      const SeqItems q = seq_items(a, p + tc, rn);
      cu.it.b = blockIdx.z, cu.it.p0 = p + tc;
      cu.nA = uni(q.nA), cu.n = uni(q.n), cu.tB = uni(q.tB);
      cu.ch = uni(q.f.ch), cu.nsk = uni(q.f.nsk), cu.wlo = uni(q.f.wlo);
      if (i >= cu.n) return;
      cu.k = i;
      place_item(a, rn, cu);
    }
  }
  Item it = cu.it;

  // Column ct*16+c is (row t, head g*grp + hc + j), col = t*hn + j; t = -1: padding
  int trow[NT];
#pragma unroll
  for (int ct = 0; ct < NT; ++ct) {
    const int col = ct * 16 + c;
    trow[ct] = col < ncols ? col / hn : -1;
  }
  const int sinks = a.window ? a.sinks : 0;

  // A wave's tiles of an item: j = beg / 32 + w, + 4, ..., without those wholly between the first tokens and
  // the windows: the current one and the one after it, with the pages of their halves. Pages are read by scalar
  // loads a tile ahead, where no LDS read is in flight (the two share a counter and return in no order).
  struct Tiles {
    int j, jn, jend, jlo;
    int pg[2], pgn[2];
  };
  const auto skip = [&](int j, int jlo) __attribute__((always_inline)) {
    return j < jlo && j * TILE >= sinks ? j + (jlo - j + WPI - 1) / WPI * WPI : j;
  };
  const auto pages_of = [&](int (&pg)[2], int b, int j) __attribute__((always_inline)) {
    const int* row = table + (size_t)b * a.ldt;
    const int at = j * TILE >> a.lp;
    pg[0] = row[min(at, a.M - 1)];
    if constexpr (P16) pg[1] = at + 1 < a.M ? row[min(at + 1, a.M - 1)] : -1;
  };
  const auto tiles_of = [&](const Item& it) __attribute__((always_inline)) {
    Tiles t;
    t.jlo = a.window ? max(it.p0 + it.r0 + 1 - a.window, 0) / TILE : 0;
    t.jend = (it.end + TILE - 1) / TILE;
    t.j = skip(it.beg / TILE + (BATCH ? 0 : w), t.jlo);
    t.jn = skip(t.j + WPI, t.jlo);
    pages_of(t.pg, it.b, t.j);
    pages_of(t.pgn, it.b, t.jn);
    return t;
  };
  // resources of a tile in both pools; rows at or past the slice's end, or without a page, read 0. Returns the
  // halves without a page.
  const auto resources = [&](int j, int pgA, int pgB, int end, Rsrc& kr, Rsrc& vr)
      __attribute__((always_inline)) {
    constexpr int H = P16 ? 2 : 1, ROWS = TILE / H;
    int bad = 0;
#pragma unroll
    for (int h = 0; h < H; ++h) {
      const int pg = h ? pgB : pgA, ph = j * TILE + 16 * h;
      const bool ok = (unsigned)pg < (unsigned)a.N;
      bad |= ok ? 0 : P16 ? 1 << h : 3;
      const int left = ok ? min(max(end - ph, 0), ROWS) : 0;
      const size_t off = (((size_t)(ok ? pg : 0) * a.Hkv + g) << (a.lp + LROW)) +
                         ((size_t)(ph & ((1 << a.lp) - 1)) << LROW);
      kr.h[h] = make_rsrc_uniform(kp + off, (uint32_t)left << LROW);
      vr.h[h] = make_rsrc_uniform(vp + off, (uint32_t)left << LROW);
    }
    return bad;
  };
  bf16x8_t qb[NT][8];  // Q^T as the MFMA B operand
  const auto load_q = [&](int b) __attribute__((always_inline)) {
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const int t = trow[ct], j = ct * 16 + c - t * hn;
      if (t >= 0) {
        const u32x4_t* src = reinterpret_cast<const u32x4_t*>(
            q + ((size_t)(b * a.R + tc + t) * a.Hq + g * a.grp + hc + j) * HD);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qb[ct][ks] = as_bf16x8(src[4 * ks + g4]);
      } else {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qb[ct][ks] = as_bf16x8(u32x4_t{0u, 0u, 0u, 0u});
      }
    }
  };

  Tile<KV8> buf;
  Rsrc kr, vr;
  int bad = 0;
  Tiles ti;
  bool on;  // the wave has a tile of the item, and it is on its way
  const auto begin = [&]() __attribute__((always_inline)) {
    ti = tiles_of(it);
    on = ti.j < ti.jend;
    if (BATCH || on) {
      bad = resources(ti.j, ti.pg[0], ti.pg[1], on ? it.end : 0, kr, vr);
      issue_k<KV8, P16>(cur, kr, kl);
      __builtin_amdgcn_sched_barrier(0);
      issue_v<KV8, P16>(buf, vr, vl);
    }
  };
  bool merged = false;  // since the last barrier
  load_q(it.b);  // ahead of the tiles' loads: a wait for it is none for them
  __builtin_amdgcn_sched_barrier(0);
  if constexpr (BATCH) begin();

  for (;;) {
    // the next item, and this wave's first tiles in it
    bool more_items = false;
    Item it2 = it;
    Tiles t2{};
    if constexpr (BATCH) {
      ++cu.k;
      more_items = take_item(a, lanes, pos, tc, rn, cu);
      it2 = cu.it;
      if (more_items) t2 = tiles_of(it2);
    } else {
      if (merged) lds_barrier();  // every wave has read the merge's slots
      begin();
    }
    const bool on2 = t2.j < t2.jend;

    Masks<NT> mk;
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      const int t = trow[ct];
      const bool mine = t >= it.r0 && t < it.r1;
      mk.L[ct] = mine ? min(it.p0 + t + 1, a.cap) : 0;
      mk.lo[ct] = a.window ? it.p0 + t + 1 - a.window : 0;
    }
    mk.rows = it.r1 - it.r0 > 1;
    mk.Lmin = min(it.p0 + it.r0 + 1, a.cap), mk.Lmax = min(it.p0 + it.r1, a.cap);
    mk.lo_min = a.window ? it.p0 + it.r0 + 1 - a.window : 0;
    mk.lo_max = a.window ? it.p0 + it.r1 - a.window : 0;
    mk.sinks = sinks;

    float m[NT], l[NT];
    f32x4_t acc[NT][16];  // [8hh + i]: O^T dims 128hh + 32g4 + 8ii + i (tile::pv_half)
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) {
      m[ct] = -INFINITY;
      l[ct] = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[ct][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
    const auto compute = [&](bool last) __attribute__((always_inline)) {
      const u32x4_t* kt =
          (const u32x4_t*)((__attribute__((address_space(3))) const u32x4_t*)(uintptr_t)cur);
      wave_lds_fence();
      f32x4_t sacc[NT][2];
      if constexpr (KV8)
        qk_tile8<NT>(kt, qb, c, g4, sacc);
      else
        tile::qk_tile<NT, NT == 1, NT == 2 ? 2 : 0>(kt, qb, c, g4, sacc);
      wave_lds_fence();
      const int p = ti.j * TILE;
      if (!last) {
        ti.j = ti.jn;
        ti.jn = skip(ti.jn + WPI, ti.jlo);
        pages_of(ti.pgn, it.b, ti.jn);
      }
      if (p + TILE > mk.Lmin || bad || (p < mk.lo_max && p + TILE > mk.sinks)) {
        uint32_t in[NT];
        if (mask_tile<NT, KV8>(buf, sacc, p, bad, mk, g4, in)) take_odd<NT, KV8>(buf, in, acc);
      }
      u32x4_t pb_hi[NT], pb_lo[NT];
      const int none[NT] = {};
      tile::softmax_tile<NT, false, true>(sacc, p, none, a.scale_log2, g4, m, l, acc, pb_hi, pb_lo);
#pragma unroll
      for (int hh = 0; hh < 2; ++hh) {
        u32x4_t rows[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) rows[e] = v_bf16(buf.v[e][hh]);
        tile::pv_half<NT, true>(rows, hh, pb_hi, pb_lo, acc);
      }
    };
    // K of a tile has landed when at most 16 loads are under way: its V was issued after it. The compiler's
    // waits for V count on the K loads behind it, so a loop issues both in every step (of a wave that has no
    // further tile, with empty resources) or is left before its last tile.
    if constexpr (BATCH) {
      for (;;) {
        // the tile after this one: of this item, or the first of the next
        const bool last = !on || ti.jn >= ti.jend;
        int jn = ti.jn, end = it.end, pg[2] = {ti.pgn[0], ti.pgn[1]};
        if (last) jn = t2.j, end = on2 ? it2.end : 0, pg[0] = t2.pg[0], pg[1] = t2.pg[1];
        const int bad_n = resources(jn, pg[0], pg[1], end, kr, vr);
        vmcnt_wait<16>();
        __builtin_amdgcn_sched_barrier(0);
        issue_k<KV8, P16>(nxt, kr, kl);
        __builtin_amdgcn_sched_barrier(0);
        if (on) compute(last);
        __builtin_amdgcn_sched_barrier(0);
        if (last && more_items && it2.b != it.b) {
          load_q(it2.b);
          // waited for here, not by every tile of the loop
#pragma unroll
          for (int ct = 0; ct < NT; ++ct)
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) asm volatile("" : "+v"(qb[ct][ks]));
        }
        __builtin_amdgcn_sched_barrier(0);
        issue_v<KV8, P16>(buf, vr, vl);
        bad = bad_n;
        if (last) break;
        const uint32_t t = cur;
        cur = nxt, nxt = t;
      }
    } else if (on) {
      while (ti.jn < ti.jend) {
        const int bad_n = resources(ti.jn, ti.pgn[0], ti.pgn[1], it.end, kr, vr);
        vmcnt_wait<16>();
        __builtin_amdgcn_sched_barrier(0);
        issue_k<KV8, P16>(nxt, kr, kl);
        __builtin_amdgcn_sched_barrier(0);
        compute(false);
        __builtin_amdgcn_sched_barrier(0);
        issue_v<KV8, P16>(buf, vr, vl);
        bad = bad_n;
        const uint32_t t = cur;
        cur = nxt, nxt = t;
      }
      vmcnt_wait<16>();
      compute(true);
    }

    // ---- the slice's partial
    // a row's slot; without a window slice i's is i
    const auto slot = [&](int ct) __attribute__((always_inline)) {
      const int t = trow[ct];
      int sl = -1;
      if (t >= it.r0 && t < it.r1)
        sl = !a.window ? (it.beg < mk.L[ct] ? it.slice : -1) : slot_of(row_slices(a, it.p0 + t), it.slice);
      return sl < a.NS ? sl : -1;
    };
    const auto place = [&](int ct, int sl) __attribute__((always_inline)) {
      const int t = trow[ct], head = g * a.grp + hc + (ct * 16 + c - t * hn);
      return (size_t)sl * a.rh + (size_t)(it.b * a.R + tc + t) * a.Hq + head;
    };
#pragma unroll
    for (int ct = 0; ct < NT; ++ct) l[ct] = group4_sum(l[ct]);
    merged = !BATCH && it.end - it.beg > TILE;
    if (!merged) {
      // a wave's item; or one tile, where the other waves hold m = -inf, l = 0, O = 0: wave 0's are the partial
      if (BATCH || w == 0) {
#pragma unroll
        for (int ct = 0; ct < NT; ++ct) {
          const int sl = slot(ct);
          if (sl < 0) continue;
          const size_t at = place(ct, sl);
          if (g4 == 0) *reinterpret_cast<float2*>(part_ml + 2 * at) = make_float2(m[ct], l[ct]);
          float* dst = part_o + at * HD + 4 * g4;
#pragma unroll
          for (int hh = 0; hh < 2; ++hh)
#pragma unroll
            for (int ii = 0; ii < 4; ++ii)
#pragma unroll
              for (int i = 0; i < 8; i += 4)
                *reinterpret_cast<f32x4_t*>(dst + 128 * hh + 32 * ii + 4 * i) =
                    f32x4_t{acc[ct][8 * hh + i][ii], acc[ct][8 * hh + i + 1][ii], acc[ct][8 * hh + i + 2][ii],
                            acc[ct][8 * hh + i + 3][ii]};
        }
      }
    } else if constexpr (!BATCH) {
      // the waves' merge, in order 0..3
      const uint32_t park = OWN ? lds_byte_uniform(lds + WAVES * 2 * SLOT + w * (MACC * WAVE * 16)) : cur;
#pragma unroll
      for (int ct = 0; ct < NT; ++ct)
        if (g4 == 0) s_ml[ct * 16 + c][0][w] = m[ct], s_ml[ct * 16 + c][1][w] = l[ct];
      if (lane == 0) s_slot[w] = park;
      const auto s_acc = [&](uint32_t at, int i) __attribute__((always_inline)) {
        return (__attribute__((address_space(3))) f32x4_t*)(uintptr_t)(at + i * (WAVE * 16));
      };
#pragma unroll
      for (int ct = 0; ct < NT; ++ct) {
        const int sl = slot(ct);
#pragma unroll
        for (int hf = 0; hf < HALVES; ++hf) {
          if (ct > 0 || hf > 0) lds_barrier();  // the previous round's reads are done
          if (trow[ct] >= it.r0 && trow[ct] < it.r1) {
#pragma unroll
            for (int i = 0; i < MACC; ++i) *s_acc(park + lane * 16, i) = acc[ct][MACC * hf + i];
          }
          lds_barrier();
          if (sl >= 0) {
            // this thread's accumulators: the i-th of each half (128 dims), i0 .. i0 + PER
            constexpr int PER = MACC / WAVES;
            const int h = HALVES == 2 ? hf : w >> 1, i0 = HALVES == 2 ? PER * w : PER * (w & 1);
            const int k0 = HALVES == 2 ? i0 : 8 * h + i0;
            const u32x4_t from = *reinterpret_cast<const u32x4_t*>(s_slot) + (uint32_t)((k0 * WAVE + lane) * 16);
            const f32x4_t mv = *reinterpret_cast<const f32x4_t*>(s_ml[ct * 16 + c][0]);
            const f32x4_t lv = *reinterpret_cast<const f32x4_t*>(s_ml[ct * 16 + c][1]);
            f32x4_t x[WAVES][PER];
#pragma unroll
            for (int v = 0; v < WAVES; ++v)
#pragma unroll
              for (int k = 0; k < PER; ++k) x[v][k] = *s_acc(from[v], k);
            __builtin_amdgcn_sched_barrier(0);  // all on their way at once (read one by one: 1.2 us of 2 per merge)
            const float M = fmaxf(fmaxf(mv[0], mv[1]), fmaxf(mv[2], mv[3]));
            float wsc[WAVES], L = 0.f;
#pragma unroll
            for (int v = 0; v < WAVES; ++v) {
              wsc[v] = mv[v] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mv[v] - M);
              L = __builtin_fmaf(lv[v], wsc[v], L);
            }
            const size_t at = place(ct, sl);
            if (w == 0 && g4 == 0 && hf == 0)
              *reinterpret_cast<float2*>(part_ml + 2 * at) = make_float2(M, L);
            f32x4_t mo[PER];
#pragma unroll
            for (int k = 0; k < PER; ++k) {
              f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
              for (int v = 0; v < WAVES; ++v)
#pragma unroll
                for (int ii = 0; ii < 4; ++ii) sum[ii] = __builtin_fmaf(x[v][k][ii], wsc[v], sum[ii]);
              mo[k] = sum;
            }
            float* dst = part_o + at * HD + 128 * h + 16 * (i0 >> 2) + 4 * g4 + (i0 & 3);
#pragma unroll
            for (int ii = 0; ii < 4; ++ii) {
              if constexpr (PER == 4)
                *reinterpret_cast<f32x4_t*>(dst + 32 * ii) = f32x4_t{mo[0][ii], mo[1][ii], mo[2][ii], mo[3][ii]};
              else
                *reinterpret_cast<float2*>(dst + 32 * ii) = make_float2(mo[0][ii], mo[1][ii]);
            }
          }
        }
      }
    }
    if constexpr (BATCH) {
      if (!more_items) {
        vmcnt_wait<0>();  // no LDS DMA may still target this workgroup's LDS
        return;
      }
      if (on2) {
        const uint32_t t = cur;
        cur = nxt, nxt = t;
      }
      it = it2, ti = t2, on = on2;
    } else {
      cu.k += a.parts;  // (more items than slots: rows with two slice sizes)
      if (cu.k >= cu.n) return;
      place_item(a, rn, cu);
      it = cu.it;
    }
  }
}

// Merge of a row's slices and the gate. A wave takes 256 / G dims of a (head, row): G groups of lanes, lane =
// (group, 4 dims); a group takes slots s0 + G i + group, and the groups meet in a fixed tree. The first AHEAD * G
// slots are loaded before the position arrives (clamped to the slots a row can have; those that do not count are
// selected away): a memory round trip less for rows of no more slices.
template <int G>
__device__ __forceinline__ float groups(float v, bool sum) {
  const auto op = [&](float x, float y) __attribute__((always_inline)) { return sum ? x + y : fmaxf(x, y); };
  if constexpr (G > 1) {
    v = xor32_pair(v, sum);
    v = xor16_pair(v, sum);
  }
  if constexpr (G == 16) {
    v = op(v, dpp<0x128>(v));               // lane ^ 8
    v = op(v, dpp<0x1B>(dpp<0x141>(v)));    // lane ^ 4
  }
  return v;
}

// The positions that the row at position p attends where they have a page: [0, first) and [lo, L).
struct Reach {
  int first, lo, L;
};
__device__ __forceinline__ Reach reach_of(const Call& a, int p) {
  Reach r;
  r.L = min(p + 1, a.cap);
  r.first = a.window ? min(a.sinks, r.L) : 0;
  r.lo = max(a.window ? max(p + 1 - a.window, 0) : 0, r.first);
  return r;
}
// Which V values that are not finite the row attends in the lane's 4 dims: per dim 3 bits, +inf, -inf, NaN. The groups
// take positions in turn, U at a time each, until what is sought (the same in every group) is NaN. bf16 pools.
template <int G>
__device__ __forceinline__ uint32_t odd_values(const Call& a, const __bf16* vp, const int* row, const Reach& r, int kvh,
                                               int dim, int g, const bool (&sought)[4]) {
  constexpr int U = 4;
  uint32_t seen = 0;
  const auto look = [&](int from, int to) __attribute__((always_inline)) {
    for (int j0 = from + g; __any(j0 < to); j0 += G * U) {
      int page[U];
#pragma unroll
      for (int u = 0; u < U; ++u) page[u] = j0 + G * u < to ? row[(j0 + G * u) >> a.lp] : -1;
      u32x2_t v[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const size_t at = (((size_t)page[u] * a.Hkv + kvh) << a.lp) + ((j0 + G * u) & ((1 << a.lp) - 1));
        v[u] = u32x2_t{0u, 0u};
        if ((unsigned)page[u] < (unsigned)a.N) v[u] = *reinterpret_cast<const u32x2_t*>(vp + at * HD + dim);
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t x = v[u][i >> 1] >> (16 * (i & 1)) & 0xffffu, m = x & 0x7fffu;
          seen |= (m < 0x7f80u ? 0u : m > 0x7f80u ? 4u : x >> 15 ? 2u : 1u) << (3 * i);
        }
#pragma unroll
      for (int o = WAVE / G; o < WAVE; o <<= 1) seen |= __shfl_xor((int)seen, o);
      bool open = false;
#pragma unroll
      for (int i = 0; i < 4; ++i) open |= sought[i] && (seen >> (3 * i) & 7) < 3;  // (3: both infinities; 4: a NaN)
      if (!__any(open)) return;
    }
  };
  look(0, r.first);
  look(r.lo, r.L);
  return seen;
}
// Whether the row attends any position.
__device__ __forceinline__ bool attends_any(const Call& a, const int* row, const Reach& r, int lane) {
  bool any = false;
  const auto look = [&](int from, int to) __attribute__((always_inline)) {
    if (from >= to) return;
    for (int j = (from >> a.lp) + lane; j <= (to - 1) >> a.lp; j += WAVE) any |= (unsigned)row[j] < (unsigned)a.N;
  };
  look(0, r.first);
  look(r.lo, r.L);
  return __any(any);
}

template <int G, int AHEAD>
__global__ void __launch_bounds__(WAVES * WAVE)
attn_paged_combine_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml,
                          const int* __restrict__ pos, const __bf16* __restrict__ qg,
                          __bf16* __restrict__ out, const __bf16* __restrict__ vp, const int* __restrict__ table,
                          Call a) {
  constexpr int LD = WAVE / G;  // lanes of a group
  const int lane = threadIdx.x & (WAVE - 1), w = uni(threadIdx.x / WAVE), g = lane / LD;
  // waves: (row, head, chunk of dims), the chunk fastest
  const int id = blockIdx.x * WAVES + w, at = (id % G) * (4 * LD) + 4 * (lane % LD);
  const int dim = dim_of(at);
  const int rh = id / G, row = (int)((unsigned)rh / (unsigned)a.Hq), h = rh - row * a.Hq;
  if (row >= a.B * a.R) return;
  const int b = row / a.R, t = row - b * a.R;
  const size_t base = (size_t)row * a.Hq + h;
  f32x4_t O = {0.f, 0.f, 0.f, 0.f};
  float L = 0.f, M = -INFINITY;
  const auto load = [&](auto n, int s0, int most, auto& po, auto& ml) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < decltype(n)::value; ++i) {
      const int s = min(s0 + G * i + g, most - 1);
      po[i] = *reinterpret_cast<const f32x4_t*>(part_o + ((size_t)s * a.rh + base) * HD + at);
      ml[i] = *reinterpret_cast<const float2*>(part_ml + 2 * ((size_t)s * a.rh + base));
    }
  };
  const auto add = [&](auto n, int s0, int cnt, const auto& po, const auto& ml) __attribute__((always_inline)) {
    constexpr int U = decltype(n)::value;
    float mv[U], bm = M;
#pragma unroll
    for (int i = 0; i < U; ++i) {
      mv[i] = s0 + G * i + g < cnt ? ml[i].x : -INFINITY;
      bm = fmaxf(bm, mv[i]);
    }
    bm = groups<G>(bm, false);
    if (bm != M) {
      const float r = M == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(M - bm);
      O *= r;
      L *= r;
      M = bm;
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
      // A slot without a finite maximum holds zeros, or NaN from a NaN among the scores, which stays one
      const bool use = s0 + G * i + g < cnt;
      const float f = mv[i] != -INFINITY ? __builtin_amdgcn_exp2f(mv[i] - M) : 1.f;
      const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
      L += (use ? ml[i].y : 0.f) * f;
      O += (use ? po[i] : zero) * f;
    }
  };
  using First = std::integral_constant<int, AHEAD>;
  using More = std::integral_constant<int, 4>;
  const __bf16* gp = qg + (size_t)row * a.ldp + (size_t)h * 2 * HD + HD + dim;
  float gate[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) gate[i] = bf16_to_f32(gp[i]);
  const int p0 = pos_of(pos, b);
  f32x4_t po[AHEAD];
  float2 ml[AHEAD];
  load(First{}, 0, a.most, po, ml);
  __builtin_amdgcn_sched_barrier(0);
  // (An idle row stores nothing. It does not leave here: the loads would move behind the wait for its position.)
  const int p = p0 < 0 ? 0 : p0 + t;
  const int cnt = min(row_slices(a, p).cnt, a.NS);
#pragma unroll
  for (int i = 0; i < 4; ++i) gate[i] = sigmoid_f32(gate[i]);
  add(First{}, 0, cnt, po, ml);
  for (int s0 = G * AHEAD; s0 < cnt; s0 += G * 4) {
    f32x4_t po[4];
    float2 ml[4];
    load(More{}, s0, cnt, po, ml);
    add(More{}, s0, cnt, po, ml);
  }
  L = groups<G>(L, true);
#pragma unroll
  for (int i = 0; i < 4; ++i) O[i] = groups<G>(O[i], true);
  // A V value that is not finite leaves its dim of O not finite, but not with its sign (a weight's two terms and
  // weights of 0 make NaN of infinities): what the row attends decides. (vp: bf16 pools; E4M3FN has only NaN.)
  bool odd[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) odd[i] = !(fabsf(O[i]) < INFINITY);
  if (__builtin_expect(vp && p0 >= 0 && L < INFINITY && __any(odd[0] || odd[1] || odd[2] || odd[3]), 0)) {
    const uint32_t seen = odd_values<G>(a, vp, table + (size_t)b * a.ldt, reach_of(a, p), h / a.grp, dim, g, odd);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t s = odd[i] ? seen >> (3 * i) & 7 : 0;
      if (s) O[i] = s == 1 ? INFINITY : s == 2 ? -INFINITY : __builtin_nanf("");
    }
  }
  // No weight at all: the row attends nothing, or every score is -inf, which has no softmax.
  if (__builtin_expect(L == 0.f && p0 >= 0 && attends_any(a, table + (size_t)b * a.ldt, reach_of(a, p), lane), 0))
    L = __builtin_nanf("");
  if (g == 0 && p0 >= 0) {
    __bf16* op = out + (size_t)row * a.ldo + (size_t)h * HD + dim;
#pragma unroll
    for (int i = 0; i < 4; ++i)  // a row that attends nothing: 0
      op[i] = f32_to_bf16(L == 0.f ? 0.f : (O[i] / L) * a.v_scale * gate[i]);
  }
}

// How a call is cut, from its sizes alone (not from R: a row's bits are the same in calls of one row).
struct Plan {
  int mins, slices;  // least slice; slices that a row can have at most
  bool batch;
};
static Plan plan(int B, int Hkv, int cap, int NS, int window, int sinks) {
  const auto slices = [&](int ch) {
    const long dense = ((long)cap + ch - 1) / ch;
    const long seen = ((long)sinks + ch - 1) / ch + ((long)window + ch - 2) / ch + 1;
    return (int)std::min<long>(NS, window ? std::min(dense, seen) : dense);
  };
  const int cus = compute_units();
  // A workgroup an item, slices of 32, where all run at once.
  Plan p{TILE, slices(TILE), false};
  if ((long)B * Hkv * p.slices <= cus) return p;
  const long span = window ? std::min<long>(cap, (long)window + sinks) : cap;
  const long pairs = (long)B * Hkv, work = pairs * span;
  const auto least = [&](long share, int most) {
    return (int)std::min<long>(most, std::max<long>(128, (share + 127) / 128 * 128));
  };
  // Slices of a CU's share, up to two a CU: as a batch they would leave most waves without work (us, so / as a batch;
  // 24 / 4 heads, bf16 if not said): 3 with a window of 500, 32 / 8 heads 11.6 / 13.5, 4 of 16,384, 16 / 2 heads, fp8
  // 18.7 / 24, 27 of 350, fp8 13.7 / 16.3, 16 of up to 6,000, 4 rows, 16 / 2 heads, fp8 25.0 / 25.9.
  p.mins = least(work / cus, 512);
  p.slices = slices(p.mins);
  if (pairs * p.slices <= 2 * cus) return p;
  // Few long sequences, where NS makes the slices longer than a batch's: a wave alone would take as long as the
  // call (5 of up to 96,486, fp8 60.8 / 82; 3 of up to 117,989 92.9 / 108).
  if (span >= 512L * NS && pairs * NS <= 8 * cus) {
    p.mins = 256;
    p.slices = slices(p.mins);
    return p;
  }
  // A batch, slices of about half of a wave's share of the positions that the tables hold: short ones cost
  // partials (written, read again) and an item's begin each, long ones balance. us at 128 / 256 / 384 / 512 / 768
  // (* as below): 7 of up to 24,011 46 / 42 / 45 / 39* / 45, 64 of up to 8,000 148 / 138 / 133 / 129* / 131, 32 with a
  // window of 4,096 115 / 111 / 103* / 113 / 103, 43 of 3 rows with one of 654, fp8 41* / 45 / - / 56.
  p.mins = least(work * 3 / 5 / cus / WAVES, 512);
  p.slices = slices(p.mins);
  p.batch = true;
  return p;
}

// plan() as the tests ask for it: the least slice, the slices that a row can have at most, whether it is a batch.
void decode_form(int B, int Hkv, int cap, int NS, int window, int sinks, int (&form)[3]) {
  const Plan p = plan(B, Hkv, cap, NS, window, sinks);
  form[0] = p.mins, form[1] = p.slices, form[2] = p.batch;
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
  a.NS = NS;
  a.window = window, a.sinks = window ? std::min(sinks, a.cap) : 0;
  a.nd = ns_div(window ? NS - 3 : NS);
  const Plan pl = plan(B, Hkv, a.cap, NS, window, a.sinks);
  a.mins = pl.mins, a.most = pl.slices;
  a.hch = (a.grp + MAX_COLS - 1) / MAX_COLS;
  a.hc = (a.grp + a.hch - 1) / a.hch;
  const int most = a.hch > 1 ? 1 : std::min(R, MAX_COLS / a.grp), rch = (R + most - 1) / most;
  a.rc = (R + rch - 1) / rch;
  a.hkv_m = Hkv == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / (unsigned)Hkv);
  a.ldt = ldt, a.ldp = ldp, a.ldo = ldo;
  a.rh = (size_t)B * R * Hq;
  a.scale_log2 = scale * 1.4426950408889634f, a.v_scale = v_scale;
  // as many workgroups as run at once: 128 KB of LDS each, or 64 KB and 256 registers
  const int NT = a.rc * a.hc <= 16 ? 1 : 2, at_once = compute_units() * (KV8 && NT == 1 ? 2 : 1);
  const bool batch = pl.batch;
  const int groups = batch ? std::max(1, at_once / Hkv) : pl.slices;
  a.parts = batch ? groups * WAVES : groups;
  const dim3 grid((unsigned)(groups * Hkv), rch * a.hch, batch ? 1 : B), block(WAVES * WAVE);
  const auto* Q = static_cast<const __bf16*>(q);
  const auto *K = static_cast<const char*>(kp), *V = static_cast<const char*>(vp);
  const auto go = [&](auto nt, auto p16, auto bt) {
    attn_paged_partials_kernel<decltype(nt)::value, KV8, decltype(p16)::value, decltype(bt)::value>
        <<<grid, block, 0, stream>>>(Q, K, V, table, pos, part_o, part_ml, a);
  };
  const auto by_batch = [&](auto nt, auto p16) {
    batch ? go(nt, p16, std::true_type{}) : go(nt, p16, std::false_type{});
  };
  const auto by_page = [&](auto nt) {
    P == 16 ? by_batch(nt, std::true_type{}) : by_batch(nt, std::false_type{});
  };
  NT == 1 ? by_page(std::integral_constant<int, 1>{}) : by_page(std::integral_constant<int, 2>{});
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const long heads = (long)B * R * Hq;
  const auto merge = [&](auto G, auto ahead) {
    constexpr int g = decltype(G)::value;
    attn_paged_combine_kernel<g, decltype(ahead)::value>
        <<<dim3((unsigned)((heads * g + WAVES - 1) / WAVES)), block, 0, stream>>>(
            part_o, part_ml, pos, static_cast<const __bf16*>(qg), static_cast<__bf16*>(out),
            KV8 ? nullptr : static_cast<const __bf16*>(vp), table, a);
  };
  // (Not by R: the forms add in different orders.) Many slots of few heads: 16 dims a wave and 64 slots ahead (one
  // row of 24 heads, 32 / 64 slots: 10.4 / 51.2 us a call in a graph against 10.6 / 52.8 with 64 dims and 8 slots). Few
  // slots, or many heads: all dims a wave and 4 slots (192 rows of 32 heads, one slot: 42.4 against 50.7; 66 of 16, 8
  // slots: 61.9 / 62.3; 64 of 24, up to 16 slots: 127.7 / 128.6; but 7 of 24, 47 slots: 44.7 / 40.4).
  const long row = (long)B * Hq;
  if (a.most > 8 && row <= 64)
    merge(std::integral_constant<int, 16>{}, std::integral_constant<int, 4>{});
  else if (a.most <= 4 || (a.most <= 16 && row >= 256))
    merge(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
  else
    merge(std::integral_constant<int, 4>{}, std::integral_constant<int, 2>{});
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
