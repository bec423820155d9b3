// The product of 8-bit rows and a 4-bit weight (microscaled formats) on gfx950's scaled matrix instructions: codes
// and scales go into them as they lie in memory, no value is converted. The kernel for up to 16 rows (and small
// products of more), and the choice between it and those of mx_gemm_block.hip and mx_gemm_tile.hip.
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "mx_common.hpp"
#include "mx_form.hpp"
#include "mx_gemm.hpp"

namespace qe {
namespace mx {

// ------------------------------------------------------------------------------ up to 16 rows
// Streams the weight: bound by memory. A workgroup takes MT tiles of 16 weight rows; its waves, as many as K has
// groups of 512 values, or a whole fraction of that (at most 16), share K by groups and their sums are added in order.
// A wave loads a whole group (MT 4 KB of codes) before it multiplies, so that a CU has up to 128 KB on the way. A
// column of the product is one row of x, which no other column touches, and the split goes by K alone: a row's bits
// do not depend on the others. 1 x 14336 x 5120 8.6 us (39 MB, 4.5 TB/s; a copy reaches 4.9), 1 x 34816 x 5120
// 18.6 us, 5 x 5120 x 17408 12.2 us (160 workgroups; 47 MB).
constexpr int ROW_WAVES = 16;

template <int MT, bool ONE>
__global__ void __launch_bounds__(ROW_WAVES * WAVE, 4)
gemm_mx4_rows_kernel(const Product c, int per) {
  __shared__ f32x4_t part[ROW_WAVES][MT][WAVE];
  const int n = c.n, N = c.N, K = c.K;
  const Layout L(N, K);
  const int lane = threadIdx.x & (WAVE - 1), r = lane & 15, g = lane >> 4, Kb = K / BLOCK;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE), waves = blockDim.x / WAVE;
  const int rt = blockIdx.x * MT, col = blockIdx.y * 16;
  const int beg = w * per, end = min(beg + per, L.KS);
  const bool live = col + r < n;
  const int rows = min(16, n - col);
  const uint32_t tiles = (uint32_t)min(MT, L.RT - rt);
  // what lies past the row's end, rows past n and weight rows past N read as zeros: they lie outside the buffers
  const __amdgpu_buffer_rsrc_t wr = make_rsrc_uniform(c.wq + (size_t)rt * L.KT * 1024, tiles * L.KT * 1024u);
  const __amdgpu_buffer_rsrc_t ar = make_rsrc_uniform(c.wscale + (size_t)rt * L.KS * 256, tiles * L.KS * 256u);
  const __amdgpu_buffer_rsrc_t xr =
      make_rsrc_uniform(c.xq + (size_t)col * c.ldx, (uint32_t)((size_t)(rows - 1) * c.ldx + K));
  const uint32_t off = live ? 0u : 0x80000000u;
  const uint32_t xo = (uint32_t)(r * c.ldx) + 16 * g;
  const uint8_t* sr = c.xs + (size_t)(col + min(r, rows - 1)) * c.lds;
  f32x4_t acc[MT];
  u32x4_t a[MT][4], b[4][2], sb;
  uint32_t sa[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto load = [&](int J) {
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int m = 0; m < MT; ++m)
        a[m][t] = buffer_load16_stream(
            wr, (uint32_t)((m * L.KT + J * 4 + t) * 1024 + lane * 16) | (J * 4 + t < L.KT ? 0u : 0x80000000u));
#pragma unroll
    for (int m = 0; m < MT; ++m)
      sa[m] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(ar, (m * L.KS + J) * 256 + lane * 4, 0, 0);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = J * 512 + t * 128 + h * 64;
        b[t][h] = buffer_load16(xr, (xo + k) | off | (k + 16 * g < K ? 0u : 0x80000000u));
      }
    // the group's 16 scales of a row; the last group's come from the row's end, shifted down below
    if (!ONE || Kb >= 16) {
      __builtin_memcpy(&sb, sr + min(J * 16, Kb - 16), 16);
    } else {
      sb = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t v = sr[min(e, Kb - 1)];
        sb[e / 4] |= (e < Kb ? v : 0u) << (8 * (e & 3));
      }
    }
  };
  auto multiply = [&](int J) {
    const int cut = J * 16 - (Kb - 16);  // bytes
    if ((!ONE || Kb >= 16) && cut > 0) {
      uint64_t lo = (uint64_t)sb[1] << 32 | sb[0], hi = (uint64_t)sb[3] << 32 | sb[2];
      if (cut >= 8) lo = hi, hi = 0;
      const int bits = (cut & 7) * 8;
      lo = lo >> bits | (bits ? hi << (64 - bits) : 0);
      hi >>= bits;
      sb = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
#define QE_TILE(T)                                                                  \
  _Pragma("unroll") for (int m = 0; m < MT; ++m) acc[m] =                           \
      mfma16<T>(a[m][T], b[T][0], b[T][1], acc[m], sa[m], sb[T] >> (8 * g));
    QE_TILE(0) QE_TILE(1) QE_TILE(2) QE_TILE(3)
#undef QE_TILE
  };
  // the other waves' loads are in flight while one multiplies
  if constexpr (ONE) {
    load(beg);
    multiply(beg);
  } else {
    for (int J = beg; J < end; ++J) {
      load(J);
      multiply(J);
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    asm volatile("" : "+v"(acc[m]));  // the products stay out of branches in which lanes are off
    part[w][m][lane] = acc[m];
  }
  __syncthreads();
  for (int m = w; m < MT; m += waves) {
    f32x4_t t = part[0][m][lane];
    for (int p = 1; p < waves; ++p) t += part[p][m][lane];
    const int j = (rt + m) * 16 + 4 * g;
    if (live && j < N) store4(c.out + (size_t)(col + r) * c.ldo + j, N - j, t);
  }
}

// Tiles of a workgroup: two, so that a row of x is read half as often, while that leaves as many workgroups as 5/8 of
// the CUs; four where x has more rows than the loads of two hide. us of 1 / 2 / 4 on N weight rows:
//   K = 5120   N 4096            5120              8192              12288             14336
//    1 row     4.5 / 5.1 / 6.7   5.8 / 5.4 / 6.9   6.8 / 6.1 / 7.5   10.3 / 9.6 / 8.9  11.7 / 10.1 / 9.4
//    16 rows   6.2 / 6.8 / 8.5   9.2 / 7.0 / 8.6   9.6 / 7.6 / 9.1   12.7 / 12 / 9.8   18.7 / 12.8 / 10.4
//   K = 17408
//    5 rows    11.7 / 13.1 / 21  16.3 / 14.2 / 22  18.0 / 15.9 / 26  25.8 / 26.8 / 30  30.2 / 28.2 / 33
//    16 rows   14.8 / 17.7 / 26  24.7 / 18.0 / 26  26.5 / 20.8 / 29  37.2 / 34.4 / 33  46.3 / 37.1 / 35
// The rule is on the wrong side between one and 5/4 workgroups a CU (N = 4608: 1 row 5.8 / 5.3, 16 rows 9.2 / 7.0), for
// 16 rows between 8192 and 12288 (10240: 11.8 / 9.2), and on the longest sums and widest weights, where four tiles hold
// more than the registers (14 of them spilled; 16 x 17408 x 17408 48.8 / 56.5).
static hipError_t gemm_rows(const Product& c, hipStream_t stream) {
  const Layout L(c.N, c.K);
  const int per = (L.KS + ROW_WAVES - 1) / ROW_WAVES, waves = (L.KS + per - 1) / per, xt = (c.n + 15) / 16;
  const long units = (long)L.RT * xt, cus = compute_units();
  const int mt = c.n > 8 && units >= 3 * cus ? 4 : 4 * units >= 5 * cus ? 2 : 1;
  const dim3 grid((L.RT + mt - 1) / mt, xt), block(waves * WAVE);
#define QE_RUN(...) __VA_ARGS__<<<grid, block, 0, stream>>>(c, per)
  if (per == 1) {
    if (mt == 1) QE_RUN(gemm_mx4_rows_kernel<1, true>);
    else if (mt == 2) QE_RUN(gemm_mx4_rows_kernel<2, true>);
    else QE_RUN(gemm_mx4_rows_kernel<4, true>);
  } else {
    if (mt == 1) QE_RUN(gemm_mx4_rows_kernel<1, false>);
    else if (mt == 2) QE_RUN(gemm_mx4_rows_kernel<2, false>);
    else QE_RUN(gemm_mx4_rows_kernel<4, false>);
  }
#undef QE_RUN
  return hipGetLastError();
}

// ------------------------------------------------------------------------------ which kernel
// Up to 16 rows always go to the streaming kernel, or a row's bits would depend on the others. More rows do where the
// work is small and K short (us, it / the best of the others: 32 x 1000 x 1000 3.9 / 5.6, 102 x 171 x 2176 4.6 / 6.8;
// past the rule 25 x 13906 x 128 4.8 / 5.4, 55 x 15157 x 352 8.2 / 6.9, 17 x 5120 x 6144 9.6 / 7.8).
//
// Between the others decides what each would take, in us: what a call costs at once; the steps of 128 of K of the
// workgroups that take turns on a CU (a little longer while every CU has one), but no less than reading the weight at
// 7 TB/s, longer by what the last turn leaves idle (32 x 34816 x 5120: 32.8 on 272 tiles of 32 x 128, 24.2 on 136 of
// 64 x 256); a workgroup's start and end; and outputs (MB; a split writes and reads fp32 as well). The constants are
// least squares over 120 calls from 17 x 80 x 64 to 2048 x 34816 x 5120, of block kernels that have become 15 to 20 %
// faster since (300 x 5120 x 6144 is priced 18.0 us and takes 14.5). On 128 calls of today's, 17 to 2048 rows, the
// choice is 1.8 % behind the best kernel and split on average, 22 % at most (26 x 16937 x 4704: 18.2, 14.9 on 32 x 128
// alone). us, tiles of 256 x 256 / 256 x 160 / 128 x 256 / 64 x 256 / 64 x 128 / 32 x 128 / 32 x 64:
//   2048 x 34816 x 5120  281 / 295 / 326 / 425 / 491 / - / 1128
//   2048 x 5120 x 6144   60 / 51 / 68 / 75 / 83 / 125 / 197
//   1024 x 5120 x 5120   46 / 33 / 29 / 39 / 37 / - / 80
//   64 x 34816 x 5120    46 / 38 / 36 / 30 / 35 / 41 / 47 (272 tiles of 64 x 128 on 256 CUs, 136 of 64 x 256)
//   300 x 5120 x 6144    53 / 38 / 31 / 20 / 15.6 / 21 / 27
//   687 x 1326 x 5056    - / - / - / - / 15.8 / 12.6 / -
//   77 x 5001 x 6176     56 / 38 / 34 / 25 / 19 / 14.3 / 11.4
// Splits: 128 x 5120 x 17408 on 64 x 128, 48 us in one part, 31 in 2, 34 in 4; 40 x 100 x 17408 on 32 x 64, 16 in
// one, 9 in 4.
struct Cost {
  int rows, cols;  // of a tile
  double call, step, full, group, split, out;
};
constexpr int TILES = (int)TileKind::COUNT, KINDS = TILES + (int)BlockKind::COUNT;
static const Cost costs[KINDS] = {{256, 256, 11.7, 0.91, 0.17, 0.0, 0.0, 0.22},  // in TileKind's order
                                  {128, 256, 7.4, 0.53, 0.18, 0.0, 0.0, 0.26},
                                  {256, 160, 8.1, 0.63, 0.19, 0.0, 0.0, 0.28},
                                  {64, 128, 3.0, 0.25, 0.03, 1.2, 2.6, 0.32},  // in BlockKind's
                                  {64, 256, 4.0, 0.33, 0.12, 1.8, 2.2, 0.38},
                                  {32, 128, 2.7, 0.34, 0.03, 2.6, 2.6, 0.20},
                                  {32, 64, 2.4, 0.50, 0.00, 2.5, 2.6, 0.11}};

constexpr int ROWS = -1;
struct Choice {
  int kind;  // ROWS, or an index into costs
  int splits;
  double us;
};

static long tiles(const Cost& c, int n, int N) {
  return (long)((n + c.rows - 1) / c.rows) * ((N + c.cols - 1) / c.cols);
}

static double estimate(int kind, int splits, int n, int N, int K, long cus) {
  const Cost& c = costs[kind];
  const double turns = (double)tiles(c, n, N) * splits / cus, mb = 2e-6 * n * N;
  const int steps =
      kind < TILES ? std::max((K + 127) / 128, 2) : block_parts((BlockKind)(kind - TILES), K, splits).part;
  const double work = std::ceil(turns) * steps * (c.step + c.full * std::min(turns, 1.));
  const double weight = N * (K * 17. / 32 / 7e6) * std::max(std::ceil(turns) / turns, 1.);
  return c.call + std::max(work, weight) + turns * c.group +
         (splits > 1 ? c.split + c.out * mb * (2 * splits + 1) : c.out * mb);
}

static size_t split_bytes(int n, int N, int splits) {
  return splits > 1 ? (size_t)splits * n * ((N + 15) / 16 * 16) * 4 : 0;
}

static Choice choose(int n, int N, int K, size_t ws_bytes, long cus) {
  const Layout L(N, K);
  if (n <= 16 || (L.KS <= ROW_WAVES && (long)((n + 15) / 16) * L.RT * L.KS <= 2000)) return {ROWS, 1, 4.};
  Choice best = {ROWS, 1, 1e30};
  for (int kind = 0; kind < KINDS; ++kind)
    for (int splits = 1; splits <= (kind < TILES ? 1 : 8); splits *= 2) {
      if (splits > 1 && (block_parts((BlockKind)(kind - TILES), K, splits).splits != splits ||
                         split_bytes(n, N, splits) > ws_bytes))
        continue;
      const double us = estimate(kind, splits, n, N, K, cus);
      if (us < best.us) best = {kind, splits, us};
    }
  return best;
}

// A call, or two: the weight rows whose tiles give every CU the same number, and the others by what suits them (two
// launches: by 3 % at least). 2048 x 34816 x 5120 is 1088 tiles of 256 x 256, 4.25 a CU: 281 us, with the last 2048
// weight rows in 256 blocks of 64 x 256 275 us (both in turn on one card, 40 calls in a row; one call by itself 279 and
// 260); 1024 x 34816 x 5120 165 and 140 us.
struct Plan {
  Choice first, rest;
  int cut;  // weight rows of the first; N if that is all
};

static Plan plan(int n, int N, int K, size_t ws_bytes) {
  const long cus = compute_units();
  Plan best = {choose(n, N, K, ws_bytes, cus), {}, N};
  if (best.first.kind == ROWS) return best;
  double least = 0.97 * best.first.us;
  for (int kind = 0; kind < KINDS; ++kind) {
    const long all = tiles(costs[kind], n, N), xtiles = (n + costs[kind].rows - 1) / costs[kind].rows;
    const long cut = all / cus * cus / xtiles * costs[kind].cols;  // a multiple of 32
    if (cut <= 0 || cut >= N) continue;
    const double us = estimate(kind, 1, n, (int)cut, K, cus);
    if (us >= least) continue;
    const Choice rest = choose(n, N - (int)cut, K, ws_bytes, cus);
    if (us + rest.us < least) least = us + rest.us, best = {{kind, 1, us}, rest, (int)cut};
  }
  return best;
}

}  // namespace mx
}  // namespace qe

using namespace qe;
using namespace qe::mx;

extern "C" size_t qe_gemm_mx4_ws_size(int n, int N, int K) {
  if (!dims_ok(n, 1) || !dims_ok(N, K)) return 0;
  K = (K + BLOCK - 1) / BLOCK * BLOCK;  // of the rows
  const Plan p = plan(n, N, K, SIZE_MAX);
  return p.cut < N ? split_bytes(n, N - p.cut, p.rest.splits) : split_bytes(n, N, p.first.splits);
}

static hipError_t run(const Choice& c, const Product& p, hipStream_t stream) {
  if (c.kind == ROWS) return gemm_rows(p, stream);
  if (c.kind < TILES) return gemm_tiles((TileKind)c.kind, p, stream);
  return gemm_blocks((BlockKind)(c.kind - TILES), c.splits, p, stream);
}

static bool product_ok(const GemmArgs& a) {
  return a.wq && a.xq && a.xs && a.out && dims_ok(a.n, a.K) && dims_ok(a.N, a.K) && a.K % BLOCK == 0 &&
         ld_ok(a.ldx, a.K) && a.ldx % 16 == 0 && ld_ok(a.lds, a.K / BLOCK) && ld_ok(a.ldo, a.N) &&
         aligned(a.wq, 16) && aligned(a.xq, 16) && aligned(a.out, 2) && aligned(a.ws, 16);
}

static Product product(const GemmArgs& a) {
  return {static_cast<const uint8_t*>(a.wq),
          static_cast<const uint8_t*>(a.wq) + Layout(a.N, a.K).scales(),
          static_cast<const uint8_t*>(a.xq),
          static_cast<const uint8_t*>(a.xs),
          static_cast<__bf16*>(a.out),
          static_cast<float*>(a.ws),
          a.ldx, a.lds, a.ldo, a.n, a.N, a.K};
}

extern "C" hipError_t qe_gemm_mx4(const void* wq, const void* xq, long ldx, const void* xs, long lds, void* out,
                                  long ldo, int n, int N, int K, void* ws, size_t ws_bytes, hipStream_t stream) {
  const GemmArgs a = {wq, xq, ldx, xs, lds, out, ldo, n, N, K, ws, ws ? ws_bytes : 0};
  if (!product_ok(a)) return hipErrorInvalidValue;
  const Layout L(N, K);
  Product p = product(a);
  const Plan how = plan(n, N, K, a.ws_bytes);
  p.N = how.cut;
  const hipError_t e = run(how.first, p, stream);
  if (e != hipSuccess || how.cut == N) return e;
  p.wq += (size_t)(how.cut / 16) * L.KT * 1024;
  p.wscale += (size_t)(how.cut / 16) * L.KS * 256;
  p.out += how.cut;
  p.N = N - how.cut;
  return run(how.rest, p, stream);
}

// ------------------------------------------------------------------------------ for the tests
namespace qe {
namespace mx {

Form gemm_form(int n, int N, int K, size_t ws_bytes) {
  const Plan p = plan(n, N, K, ws_bytes);
  return {p.first.kind, p.first.splits, p.cut, p.rest.kind, p.rest.splits};
}

bool gemm_form_ok(int kernel, int splits, int n, int N, int K, size_t ws_bytes) {
  if (kernel < ROWS || kernel >= KINDS) return false;
  if (kernel < TILES) return splits == 1 && (kernel != ROWS || (n + 15) / 16 <= 65535);  // a grid's second axis
  return splits >= 1 && block_parts((BlockKind)(kernel - TILES), K, splits).splits == splits &&
         split_bytes(n, N, splits) <= ws_bytes;
}

hipError_t gemm_as(int kernel, int splits, const GemmArgs& a, hipStream_t stream) {
  if (!product_ok(a) || !gemm_form_ok(kernel, splits, a.n, a.N, a.K, a.ws ? a.ws_bytes : 0))
    return hipErrorInvalidValue;
  return run({kernel, splits, 0.}, product(a), stream);
}

}  // namespace mx
}  // namespace qe
