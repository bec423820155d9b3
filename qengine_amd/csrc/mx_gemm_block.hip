// The product of 8-bit rows and a 4-bit weight for tens to hundreds of rows: small tiles, K shared by groups of waves
// and, where there are few tiles, by workgroups.
//
// Bound by a step's chain on a CU, no single part of it: a tile of 64 x 128 takes 0.2 us a step, of which 256 cycles
// are products, 48 KB are read from LDS and 16 KB loaded. 320 x 5120 x 6144, 15.7 us: 12.6 without the products, 14.6
// without the LDS reads, 12.1 without the loads, 11.4 with products and barriers alone; 13.9 and 14.7 with all of x
// or of the weight from the L2. Deeper stages, one barrier for two steps, the weight straight into registers and
// wider waves gave nothing or less. 300 x 5120 x 6144 14.7 us (200 tiles of 64 x 128); 77 x 5001 x 6176 10.6 us (237
// of 32 x 64, four parts of K side by side, 13 steps); 64 x 34816 x 5120 28.8 us (256 of 64 x 128, and
// 64 of 32 x 64 for the weight rows past them; 29.0 on 136 of 64 x 256), bound by memory.
#include <limits.h>

#include <algorithm>

#include "mx_common.hpp"
#include "mx_gemm.hpp"

namespace qe {
namespace mx {

// 8 waves, WX by WW by WK: WK groups of waves, each with a part of K of its own, multiply a tile of WX TX 32 rows by
// WW TW 32 weight rows. A stage holds 128 values of each part.
template <int WX, int WW, int WK, int TX, int TW, int STAGES>
struct Block {
  static constexpr int WAVES = WX * WW * WK, ROWS = WX * TX * 32, COLS = WW * TW * 32;
  static constexpr int XB = ROWS * 128, PART = XB + COLS * 64, STAGE = WK * PART, ST = STAGES;
  static constexpr int XL = WK * ROWS / 8 / WAVES, WL = WK * COLS / 16 / WAVES, LOADS = XL + WL;  // a wave's loads
  static_assert(WAVES == 8 && XL * WAVES * 8 == WK * ROWS && WL * WAVES * 16 == WK * COLS, "whole loads");
  static constexpr int Q = TX * TW * 4;  // 16-byte pieces of a lane's sums
  static constexpr int SUM = WK > 1 ? WAVES * Q * 1024 : 0;
  static constexpr int LDS = std::max(ST * STAGE, SUM);
  static constexpr int PER_CU = 2 * LDS <= 163840 ? 2 : 1;
};

struct BlockCall : Product {
  int xtiles, wtiles;
  int part;  // 128-value tiles of a part of K
};

template <int WX, int WW, int WK, int TX, int TW, int STAGES, bool ONCE,
          class T = Block<WX, WW, WK, TX, TW, STAGES>>
__global__ void __launch_bounds__(T::WAVES * WAVE, 2 * T::PER_CU)
gemm_mx4_block_kernel(const BlockCall c) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[T::LDS];
  const Layout L(c.N, c.K);
  const int lane = threadIdx.x & (WAVE - 1), r = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int wx = w % WX, ww = w / WX % WW, wk = w / (WX * WW);
  // workgroups go to the 8 XCDs in turn: each gets neighbouring tiles, the row tiles of a weight tile first, so that
  // the weight is read by one L2
  const int tiles = c.xtiles * c.wtiles, q8 = tiles / 8, r8 = tiles % 8, xcd = blockIdx.x % 8;
  const int tile = xcd * q8 + min(xcd, r8) + (int)blockIdx.x / 8;
  const int x0 = tile % c.xtiles * T::ROWS, c0 = tile / c.xtiles * T::COLS, rt0 = c0 / 16;
  const int KT = L.KT, Kb = c.K / BLOCK;
  const int k0 = (blockIdx.y * WK + wk) * c.part;  // this wave's first tile of K

  // loads: as in the kernel for many rows, pieces of x (8 rows of 128 bytes, slot s of row i holds chunk s ^ (i / 2 %
  // 8)) and of the weight (a 16-row tile's 1 KB) of every part
  const __amdgpu_buffer_rsrc_t xr =
      make_rsrc_uniform(c.xq + (size_t)x0 * c.ldx, (uint32_t)((size_t)(min(T::ROWS, c.n - x0) - 1) * c.ldx + c.K));
  const __amdgpu_buffer_rsrc_t wr = make_rsrc_uniform(c.wq + (size_t)rt0 * KT * 1024,
                                                      (uint32_t)min(T::COLS / 16, L.RT - rt0) * KT * 1024u);
  uint32_t xo[T::XL], xl[T::XL], wo[T::WL], wl[T::WL];
  int xk[T::XL], wkt[T::WL];  // byte in the row, tile of K
#pragma unroll
  for (int i = 0; i < T::XL; ++i) {
    const int id = w + i * T::WAVES, part = id / (T::ROWS / 8), p = id % (T::ROWS / 8);
    const int chunk16 = ((lane & 7) ^ ((p & 1) * 4 + (lane >> 4))) * 16;
    xk[i] = (int)(blockIdx.y * WK + part) * c.part * 128 + chunk16;
    xo[i] = (uint32_t)((p * 8 + (lane >> 3)) * c.ldx);
    xl[i] = lds_byte_uniform(smem) + part * T::PART + p * 1024;
  }
#pragma unroll
  for (int i = 0; i < T::WL; ++i) {
    const int id = w + i * T::WAVES, part = id / (T::COLS / 16), p = id % (T::COLS / 16);
    wkt[i] = (int)(blockIdx.y * WK + part) * c.part;
    wo[i] = (uint32_t)p * KT * 1024u + lane * 16;
    wl[i] = lds_byte_uniform(smem) + part * T::PART + T::XB + p * 1024;
  }
  auto fetch = [&](int s, int stage) {
#pragma unroll
    for (int i = 0; i < T::XL; ++i) {
      const int k = xk[i] + s * 128;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (__attribute__((address_space(3))) void*)(uintptr_t)(xl[i] + stage * T::STAGE), 16,
          (int)((xo[i] + k) | (k >= c.K ? 0x80000000u : 0u)), 0, 0, 0);  // past the row: zeros
    }
#pragma unroll
    for (int i = 0; i < T::WL; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr, (__attribute__((address_space(3))) void*)(uintptr_t)(wl[i] + stage * T::STAGE), 16,
          (int)(wo[i] + min(wkt[i] + s, KT - 1) * 1024), 0, 0, ONCE ? CPOL_NT : 0);
  };

  // Scales of four steps. Of x, 16 bytes of lane r's row, the last ones shifted down from the row's end: no byte past
  // the row is read, and blocks past K get code 0. Of the weight, dwords of four tiles each: a part begins within one.
  constexpr int SCALES = 2 * TW + TX;  // loads of scales()
  const bool small = Kb < 16;
  const int last16 = small ? 0 : Kb - 16;
  const __amdgpu_buffer_rsrc_t sr = make_rsrc_uniform(c.wscale + (size_t)rt0 * L.KS * 256,
                                                      (uint32_t)min(T::COLS / 16, L.RT - rt0) * L.KS * 256u);
  const uint32_t so = (uint32_t)(ww * TW * 2 + (r >> 4)) * L.KS * 256u + ((r & 15) + 16 * g) * 4;
  const uint8_t *xp[TX], *xp16[TX];
#pragma unroll
  for (int i = 0; i < TX; ++i) {
    xp[i] = c.xs + (size_t)min(x0 + (wx * TX + i) * 32 + r, c.n - 1) * c.lds;
    xp16[i] = small ? c.wq : xp[i];  // of no account where rows have fewer than 16 blocks
  }
  uint32_t sw[TW][2], sw0[TW][2], sw1[TW][2], sw2[TW][2];  // four steps' bytes; dwords at hand, the next, loaded
  u32x4_t sx[TX], sx2[TX];
  auto weight_scales = [&](int J) {
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sw2[j][h] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(
            sr, (int)(so + j * 2 * L.KS * 256 + min(J, L.KS - 1) * 256 + h * 128), 0, 0);
  };
  auto scales = [&](int k) {  // of tiles k .. k + 3
    weight_scales(k / 4 + 1);
#pragma unroll
    for (int i = 0; i < TX; ++i) __builtin_memcpy(&sx2[i], xp16[i] + min(k * 4, last16), 16);
  };
  auto take = [&](int k) {
    const int cut = min(k * 4 - last16, 16);  // bytes
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sw0[j][h] = sw1[j][h];
        sw1[j][h] = sw2[j][h];
        sw[j][h] = __builtin_amdgcn_alignbyte(sw1[j][h], sw0[j][h], k & 3);
      }
    if (!small && cut > 0) {
#pragma unroll
      for (int i = 0; i < TX; ++i) {
        uint64_t lo = (uint64_t)sx2[i][1] << 32 | sx2[i][0], hi = (uint64_t)sx2[i][3] << 32 | sx2[i][2];
        if (cut >= 8) lo = hi, hi = 0;
        if (cut >= 16) lo = 0;
        const int bits = (cut & 7) * 8;
        lo = lo >> bits | (bits ? hi << (64 - bits) : 0);
        hi >>= bits;
        sx2[i] = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
    }
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sx[i][e] = sx2[i][e] >> (8 * g);
  };

  f32x16_t acc[TX][TW];
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
  const int slot = r / 2 & 7;
  const uint8_t* xf = smem + wk * T::PART + (wx * TX * 32 + r) * 128;
  const uint8_t* wf = smem + wk * T::PART + T::XB + (ww * TW * 2 + (r >> 4)) * 1024 + ((r & 15) + 16 * g) * 16;

  weight_scales(k0 / 4);
#pragma unroll
  for (int j = 0; j < TW; ++j)
#pragma unroll
    for (int h = 0; h < 2; ++h) sw1[j][h] = sw2[j][h];
  scales(k0);
  if (small) {
#pragma unroll
    for (int i = 0; i < TX; ++i) {
      sx2[i] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t v = xp[i][min(k0 * 4 + e, Kb - 1)];
        sx2[i][e / 4] |= (k0 * 4 + e < Kb ? v : 0u) << (8 * (e & 3));
      }
    }
  }
#pragma unroll
  for (int s = 0; s < T::ST; ++s) {
    __builtin_amdgcn_sched_barrier(0);  // in this order: the waits below count them
    fetch(s, s);
  }
  __builtin_amdgcn_sched_barrier(0);
  take(k0);
  u32x4_t a[2][2][TW], b[2][2][TX][2];
  auto read = [&](int stage, int to) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int j = 0; j < TW; ++j)
        a[to][h][j] = *reinterpret_cast<const u32x4_t*>(wf + stage * T::STAGE + j * 2048 + h * 512);
#pragma unroll
      for (int i = 0; i < TX; ++i)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          b[to][h][i][e] = *reinterpret_cast<const u32x4_t*>(xf + stage * T::STAGE + i * 4096 +
                                                             (((4 * h + 2 * e + g) ^ slot) << 4));
    }
  };
  vmcnt_wait<(T::ST - 1) * T::LOADS>();
  lds_barrier();
  read(0, 0);
  int stage = 0;
  // A step, whose operands are in registers: the next step's are read behind the barrier (that stage has landed: only
  // the ST - 2 steps after it are out, and scales loaded since), the loads of the step ST ahead take the place of
  // this one, which every wave has read ahead of the barrier. Reads and loads are issued between the step's products,
  // or the matrix cores would wait until they all are (64 x 256 tiles, 300 x 5120 x 6144: 21.5 -> 19.5 us).
#define QE_STEP(S, MORE)                                                                                      \
  {                                                                                                           \
    vmcnt_wait<(T::ST - 2) * T::LOADS + (MORE && S >= 1 && S <= T::ST - 2 ? SCALES : 0)>();                   \
    lds_barrier();                                                                                            \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    _Pragma("unroll") for (int i = 0; i < TX; ++i) _Pragma("unroll") for (int j = 0; j < TW; ++j) acc[i][j] = \
        mfma32<S, 0>(a[S & 1][0][j], b[S & 1][0][i][0], b[S & 1][0][i][1], acc[i][j], sw[j][0], sx[i][S]);    \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    const int next = stage + 1 < T::ST ? stage + 1 : 0;                                                       \
    read(next, 1 - (S & 1));                                                                                  \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    if (MORE && S == 0) scales(k0 + s0 + 4);                                                                  \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    fetch(s0 + S + T::ST, stage);                                                                             \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    _Pragma("unroll") for (int i = 0; i < TX; ++i) _Pragma("unroll") for (int j = 0; j < TW; ++j) acc[i][j] = \
        mfma32<S, 2>(a[S & 1][1][j], b[S & 1][1][i][0], b[S & 1][1][i][1], acc[i][j], sw[j][1], sx[i][S]);    \
    _Pragma("unroll") for (int i = 0; i < TX; ++i) _Pragma("unroll") for (int j = 0; j < TW; ++j)             \
        asm volatile("" : "+v"(acc[i][j]));                                                                   \
    __builtin_amdgcn_sched_barrier(0);                                                                        \
    stage = next;                                                                                             \
  }
  int s0 = 0;
  for (; s0 + 4 <= c.part; s0 += 4) {
    QE_STEP(0, 1) QE_STEP(1, 1) QE_STEP(2, 1) QE_STEP(3, 1)
    take(k0 + s0 + 4);
  }
  if (s0 < c.part) {  // the last one to three; no scales behind them
    QE_STEP(0, 0)
    if (s0 + 1 < c.part) { QE_STEP(1, 0) }
    if (s0 + 2 < c.part) { QE_STEP(2, 0) }
  }
#undef QE_STEP
  vmcnt_wait<0>();

  // piece q of tile (i, j): four neighbouring outputs of row r, at 8 (q % 4) + 4 g of the tile's 32
  auto give = [&](int row, int col, f32x4_t t) {
    if (row >= c.n) return;
    if (c.ws) {
      if (col < 16 * L.RT)
        *reinterpret_cast<f32x4_t*>(c.ws + ((size_t)blockIdx.y * c.n + row) * (16 * (size_t)L.RT) + col) = t;
    } else {
      store4(c.out + (size_t)row * c.ldo + col, c.N - col, t);
    }
  };
  if constexpr (WK == 1) {
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int j = 0; j < TW; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          give(x0 + (wx * TX + i) * 32 + r, c0 + (ww * TW + j) * 32 + 8 * e + 4 * g,
               f32x4_t{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]});
  } else {
    __syncthreads();  // every wave has read its last stage
    f32x4_t* sum = reinterpret_cast<f32x4_t*>(smem);
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int j = 0; j < TW; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          sum[(w * T::Q + (i * TW + j) * 4 + e) * WAVE + lane] =
              f32x4_t{acc[i][j][4 * e], acc[i][j][4 * e + 1], acc[i][j][4 * e + 2], acc[i][j][4 * e + 3]};
    __syncthreads();
    for (int id = w; id < WX * WW * T::Q; id += T::WAVES) {
      const int v = id / T::Q, q = id % T::Q;  // a wave of the first group, its piece
      f32x4_t t = sum[id * WAVE + lane];
#pragma unroll
      for (int k = 1; k < WK; ++k) t += sum[(k * WX * WW * T::Q + id) * WAVE + lane];
      give(x0 + (v % WX * TX + q / 4 / TW) * 32 + r, c0 + (v / WX * TW + q / 4 % TW) * 32 + q % 4 * 8 + 4 * g, t);
    }
  }
}

// The splits' partial sums, in order.
__global__ void __launch_bounds__(256)
mx4_sum_kernel(const float* ws, __bf16* out, long ldo, int n, int N, int width, int splits) {
  const int row = blockIdx.x, col = (blockIdx.y * 256 + threadIdx.x) * 4;
  if (col >= N) return;
  const f32x4_t* p = reinterpret_cast<const f32x4_t*>(ws + (size_t)row * width + col);
  f32x4_t t = *p;
  for (int s = 1; s < splits; ++s) t += p[(size_t)s * n * width / 4];
  store4(out + (size_t)row * ldo + col, N - col, t);
}

static Parts parts(int wk, int K, int splits) {
  const int KT = (K + 127) / 128, part = (KT + wk * splits - 1) / (wk * splits);
  return {part, (KT + wk * part - 1) / (wk * part)};
}

template <int WX, int WW, int WK, int TX, int TW, int STAGES>
static hipError_t run(const Product& p, int splits, hipStream_t stream) {
  using T = Block<WX, WW, WK, TX, TW, STAGES>;
  const long xt = (p.n + T::ROWS - 1) / T::ROWS, wt = (p.N + T::COLS - 1) / T::COLS;
  if (xt * wt > UINT_MAX / (T::WAVES * WAVE)) return hipErrorInvalidValue;  // the grid's threads
  const Parts k = parts(WK, p.K, splits);
  BlockCall c = {p, (int)xt, (int)wt, k.part};
  if (k.splits == 1) c.ws = nullptr;
  const dim3 grid(xt * wt, k.splits), block(T::WAVES * WAVE);
  // A weight that is read once, and so large that no cache will hold it until the next call, passes the caches'
  // favour: 64 x 34816 x 5120 (95 MB) on 64 x 256 31.6 -> 29.0 us (smaller ones may still be there: 32 x 14336 x
  // 5120, 41 MB, 9.6 us, 12.4 past them; from memory 13.1 and 12.5).
  if constexpr (T::ROWS == 64) {
    if (xt == 1 && Layout(p.N, p.K).scales() >= 64u << 20) {
      gemm_mx4_block_kernel<WX, WW, WK, TX, TW, STAGES, true><<<grid, block, 0, stream>>>(c);
    } else {
      gemm_mx4_block_kernel<WX, WW, WK, TX, TW, STAGES, false><<<grid, block, 0, stream>>>(c);
    }
  } else {
    gemm_mx4_block_kernel<WX, WW, WK, TX, TW, STAGES, false><<<grid, block, 0, stream>>>(c);
  }
  if (k.splits > 1)
    mx4_sum_kernel<<<dim3(p.n, (p.N + 1023) / 1024), dim3(256), 0, stream>>>(p.ws, p.out, p.ldo, p.n, p.N,
                                                                            (p.N + 15) / 16 * 16, k.splits);
  return hipGetLastError();
}

Parts block_parts(BlockKind kind, int K, int splits) {
  return parts(kind == BlockKind::X32_W64_K4 ? 4 : kind == BlockKind::X32_W128_K2 ? 2 : 1, K, splits);
}

hipError_t gemm_blocks(BlockKind kind, int splits, const Product& p, hipStream_t stream) {
  switch (kind) {
    case BlockKind::X64_W128: return run<2, 4, 1, 1, 1, 4>(p, splits, stream);
    case BlockKind::X64_W256: return run<2, 4, 1, 1, 2, 4>(p, splits, stream);
    case BlockKind::X32_W128_K2: return run<1, 4, 2, 1, 1, 4>(p, splits, stream);
    case BlockKind::X32_W64_K4: return run<1, 2, 4, 1, 1, 3>(p, splits, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mx
}  // namespace qe
