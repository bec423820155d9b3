// The product of 8-bit rows and a 4-bit weight for many rows: tiles of WX x TX x 32 rows by WW x TW x 32 weight rows.
#include "mx_common.hpp"
#include "mx_gemm.hpp"

namespace qe {
namespace mx {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));

template <int SA, int SB>
__device__ __forceinline__ f32x16_t mfma32(u32x4_t a, u32x4_t b0, u32x4_t b1, f32x16_t d, uint32_t sa, uint32_t sb) {
  const i32x8_t A = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t B = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(A, B, d, 4, 0, SA, (int)sa, SB, (int)sb);
}

// A stage holds 64 values along K of a tile's rows and weight rows.
template <int WX, int WW, int TX, int TW>
struct Tile {
  static constexpr int WAVES = WX * WW, ROWS = WX * TX * 32, COLS = WW * TW * 32;
  static constexpr int XB = ROWS * 64, STAGE = XB + COLS * 32;  // bytes: x, then the weight
  static constexpr int STAGES = 6;
  static constexpr int DX = (ROWS / 16 + WAVES - 1) / WAVES, DW = (COLS / 32 + WAVES - 1) / WAVES;  // a wave's loads
  static constexpr int PITCH = TW * 64 + 16;  // of a row in the epilogue, bytes
  static constexpr int LDS = STAGES * STAGE > WAVES * 32 * PITCH ? STAGES * STAGE : WAVES * 32 * PITCH;
};

template <int WX, int WW, int TX, int TW>
__global__ void __launch_bounds__(WX * WW * WAVE, (WX * WW + 3) / 4)
gemm_mx4_tile_kernel(const uint8_t* wq, const uint8_t* xq, long ldx, const uint8_t* xs, long lds, __bf16* out,
                     long ldo, int n, int N, int K, int xtiles, int tiles, bool vec) {
  using T = Tile<WX, WW, TX, TW>;
  __shared__ __attribute__((aligned(1024))) uint8_t smem[T::LDS];
  const Layout L(N, K);
  const int lane = threadIdx.x & (WAVE - 1), r = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int wx = w % WX, ww = w / WX;
  // workgroups go to the 8 XCDs in turn: each gets neighbouring tiles, the row tiles of a weight tile first
  const int q8 = tiles / 8, r8 = tiles % 8, xcd = blockIdx.x % 8, at = blockIdx.x / 8;
  const int tile = xcd * q8 + min(xcd, r8) + at;
  const int x0 = (tile % xtiles) * T::ROWS, c0 = (tile / xtiles) * T::COLS, rt0 = c0 / 16;
  const int KT = L.KT, Kb = K / BLOCK;

  // x: 16 rows of 64 bytes a load; slot c of row i holds chunk c ^ (i / 4 % 4). The weight: half of two 16-row
  // tiles' 1 KB a load. Rows and chunks past the matrix are zeros.
  const __amdgpu_buffer_rsrc_t xr =
      make_rsrc_uniform(xq + (size_t)x0 * ldx, (uint32_t)((size_t)(min(T::ROWS, n - x0) - 1) * ldx + K));
  const __amdgpu_buffer_rsrc_t wr = make_rsrc_uniform(wq + (size_t)rt0 * KT * 1024,
                                                      (uint32_t)min(T::COLS / 16, L.RT - rt0) * KT * 1024u);
  const int chunk16 = ((lane & 3) ^ (lane >> 4)) * 16;
  uint32_t xo[T::DX], wo[T::DW], xl[T::DX], wl[T::DW];
#pragma unroll
  for (int i = 0; i < T::DX; ++i) {
    const int id = min(w + i * T::WAVES, T::ROWS / 16 - 1);
    xo[i] = (uint32_t)((id * 16 + (lane >> 2)) * ldx + chunk16);
    xl[i] = lds_byte_uniform(smem) + id * 1024;
  }
#pragma unroll
  for (int i = 0; i < T::DW; ++i) {
    const int id = min(w + i * T::WAVES, T::COLS / 32 - 1);
    wo[i] = (uint32_t)(id * 2 + (lane >> 5)) * KT * 1024u + (lane & 31) * 16;
    wl[i] = lds_byte_uniform(smem) + T::XB + id * 1024;
  }
  constexpr int LOADS = T::DX + T::DW;
  auto fetch = [&](int t, int slot) {  // this wave's loads of stage t
    const uint32_t past = t * 64 + chunk16 >= K ? 0x80000000u : 0u;  // outside the buffer
#pragma unroll
    for (int i = 0; i < T::DX; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (__attribute__((address_space(3))) void*)(uintptr_t)(xl[i] + slot * T::STAGE), 16,
          (int)((xo[i] + t * 64) | past), 0, 0, 0);
#pragma unroll
    for (int i = 0; i < T::DW; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr, (__attribute__((address_space(3))) void*)(uintptr_t)(wl[i] + slot * T::STAGE), 16,
          (int)(wo[i] + min(t, 2 * KT - 1) * 512), 0, 0, 0);
  };

  // Scales of four steps: of x, 16 bytes of lane r's row; of the weight, a dword for blocks g and 2 + g of a tile. The
  // last ones of x come from the row's end, shifted down: no byte past the row is read, and blocks past K
  // get code 0.
  const __amdgpu_buffer_rsrc_t sr = make_rsrc_uniform(wq + L.scales() + (size_t)rt0 * L.KS * 256,
                                                      (uint32_t)min(T::COLS / 16, L.RT - rt0) * L.KS * 256u);
  const uint32_t so = (uint32_t)(ww * TW * 2 + (r >> 4)) * L.KS * 256u + ((r & 15) + 16 * g) * 4;
  const uint8_t* xp[TX];
#pragma unroll
  for (int i = 0; i < TX; ++i) xp[i] = xs + (size_t)min(x0 + (wx * TX + i) * 32 + r, n - 1) * lds;
  uint32_t sw[TW][2], sw2[TW][2];
  u32x4_t sx[TX], sx2[TX];
  constexpr int SCALES = 2 * TW + TX;  // loads of scales()
  auto scales = [&](int J) {  // from K's end on anything: never used
    const bool more = J < L.KS && Kb >= 16;
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sw2[j][h] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(
            sr, (int)(so + j * 2 * L.KS * 256 + min(J, L.KS - 1) * 256 + h * 128), 0, 0);
#pragma unroll
    for (int i = 0; i < TX; ++i) __builtin_memcpy(&sx2[i], more ? xp[i] + min(J * 16, Kb - 16) : wq, 16);
  };
  auto take = [&](int J) {  // the loaded ones become those of steps 4 J ..
    const int cut = Kb >= 16 ? min(max(J * 16 - (Kb - 16), 0), 16) : 0;  // bytes
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) sw[j][h] = sw2[j][h];
#pragma unroll
    for (int i = 0; i < TX; ++i) {
      uint64_t lo = (uint64_t)sx2[i][1] << 32 | sx2[i][0], hi = (uint64_t)sx2[i][3] << 32 | sx2[i][2];
      if (cut >= 8) lo = hi, hi = 0;
      const int bits = (cut & 7) * 8;
      lo = lo >> bits | (bits ? hi << (64 - bits) : 0);
      hi >>= bits;
      // lanes 32 .. 63 hold blocks 1 and 3 of a step where the others hold 0 and 2
      sx[i] = u32x4_t{(uint32_t)lo >> (8 * g), (uint32_t)(lo >> 32) >> (8 * g), (uint32_t)hi >> (8 * g),
                      (uint32_t)(hi >> 32) >> (8 * g)};
    }
  };

  f32x16_t acc[TX][TW];
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;

  const uint8_t* xf = smem + (wx * TX * 32 + r) * 64;
  const uint8_t* wf = smem + T::XB + (ww * TW * 2 + (r >> 4)) * 512 + ((r & 15) + 16 * g) * 16;
  const int at0 = (g ^ (r / 4 & 3)) << 4, at1 = ((2 + g) ^ (r / 4 & 3)) << 4;
  u32x4_t a[TW], b[TX][2];
  auto read = [&](int slot) {
#pragma unroll
    for (int j = 0; j < TW; ++j) a[j] = *reinterpret_cast<const u32x4_t*>(wf + slot * T::STAGE + j * 1024);
#pragma unroll
    for (int i = 0; i < TX; ++i) {
      b[i][0] = *reinterpret_cast<const u32x4_t*>(xf + slot * T::STAGE + i * 2048 + at0);
      b[i][1] = *reinterpret_cast<const u32x4_t*>(xf + slot * T::STAGE + i * 2048 + at1);
    }
  };

  if (Kb >= 16) {
    scales(0);
  } else {  // one group of four steps: its scales a byte at a time
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sw2[j][h] =
            (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(sr, (int)(so + j * 2 * L.KS * 256 + h * 128), 0, 0);
#pragma unroll
    for (int i = 0; i < TX; ++i) {
      sx2[i] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t v = xp[i][min(e, Kb - 1)];
        sx2[i][e / 4] |= (e < Kb ? v : 0u) << (8 * (e & 3));
      }
    }
  }
#pragma unroll
  for (int t = 0; t < T::STAGES - 1; ++t) fetch(t, t);
  vmcnt_wait<(T::STAGES - 2) * LOADS>();
  lds_barrier();
  // Two halves of the workgroup, a wave of each on every SIMD, take turns: between two barriers one half reads its
  // operands of a stage and issues loads, the other multiplies, so the matrix cores always have a wave that does
  // nothing else. The first half reads stage t in turn 2 t, the second in turn 2 t + 1; stage t + 5 goes into
  // the place of stage t - 1, which both have read by then, and stage t + 1 has landed for every wave before
  // turn 2 t + 2: only the four after it are out (and, from the third stage of eight, the next scales).
  const bool second = w >= T::WAVES / 2;
  int slot = 0;
  if (second) lds_barrier();
#define QE_HALF(S, H)                                                                                       \
  {                                                                                                         \
    constexpr int OUT = (T::STAGES - 2) * LOADS + (2 * S + H >= 2 && 2 * S + H <= 5 ? SCALES : 0);          \
    read(slot);                                                                                             \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    if (S == 1 && H == 0) scales(kt / 4 + 1);                                                               \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    fetch(2 * (kt + S) + H + T::STAGES - 1, slot >= 1 ? slot - 1 : T::STAGES - 1);                          \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    vmcnt_wait<OUT>();                                                                                      \
    lds_barrier();                                                                                          \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    __builtin_amdgcn_s_setprio(1);                                                                          \
    _Pragma("unroll") for (int i = 0; i < TX; ++i) _Pragma("unroll") for (int j = 0; j < TW; ++j)           \
        acc[i][j] = mfma32<S, 2 * H>(a[j], b[i][0], b[i][1], acc[i][j], sw[j][H], sx[i][S]);                \
    __builtin_amdgcn_s_setprio(0);                                                                          \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    lds_barrier();                                                                                          \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    slot = slot + 1 < T::STAGES ? slot + 1 : 0;                                                             \
  }
#define QE_STEP(S) QE_HALF(S, 0) QE_HALF(S, 1)
  int kt = 0;
  for (; kt + 4 <= KT; kt += 4) {
    take(kt / 4);
    QE_STEP(0) QE_STEP(1) QE_STEP(2) QE_STEP(3)
  }
  if (kt < KT) {  // the last one to three steps: a loop with exits between would wait for all loads at each of them
    take(kt / 4);
    QE_STEP(0)
    if (kt + 1 < KT) { QE_STEP(1) }
    if (kt + 2 < KT) { QE_STEP(2) }
  }
#undef QE_STEP
#undef QE_HALF
  if (!second) lds_barrier();

  // out: a wave's 32 rows at a time through LDS, so that a row's neighbouring values leave in 16-byte stores
#pragma unroll
  for (int i = 0; i < TX; ++i)
#pragma unroll
    for (int j = 0; j < TW; ++j) asm volatile("" : "+v"(acc[i][j]));  // products stay out of branches
  vmcnt_wait<0>();  // the last loads into LDS
  __syncthreads();
  uint8_t* mine = smem + w * 32 * T::PITCH;
#pragma unroll
  for (int i = 0; i < TX; ++i) {
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const u32x2_t v = {pack_bf16x2(acc[i][j][4 * e], acc[i][j][4 * e + 1]),
                           pack_bf16x2(acc[i][j][4 * e + 2], acc[i][j][4 * e + 3])};
        *reinterpret_cast<u32x2_t*>(mine + r * T::PITCH + j * 64 + e * 16 + g * 8) = v;
      }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int t = 0; t < TW * 2; ++t) {
      const int p = lane + t * WAVE;  // piece of 8 values
      const int row = x0 + (wx * TX + i) * 32 + p / (TW * 4), j = c0 + ww * TW * 32 + p % (TW * 4) * 8;
      const u32x4_t v = *reinterpret_cast<const u32x4_t*>(mine + p / (TW * 4) * T::PITCH + p % (TW * 4) * 16);
      if (row < n) {
        __bf16* o = out + (size_t)row * ldo + j;
        if (vec && j + 8 <= N)
          *reinterpret_cast<u32x4_t*>(o) = v;
        else
          for (int e = 0; e < 8; ++e)
            if (j + e < N) reinterpret_cast<uint16_t*>(o)[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

template <int WX, int WW, int TX, int TW>
static hipError_t run(const uint8_t* wq, const uint8_t* xq, long ldx, const uint8_t* xs, long lds, __bf16* out,
                      long ldo, int n, int N, int K, hipStream_t stream) {
  using T = Tile<WX, WW, TX, TW>;
  const int xt = (n + T::ROWS - 1) / T::ROWS, tiles = xt * ((N + T::COLS - 1) / T::COLS);
  const auto kernel = gemm_mx4_tile_kernel<WX, WW, TX, TW>;
  kernel<<<dim3(tiles), dim3(T::WAVES * WAVE), 0, stream>>>(wq, xq, ldx, xs, lds, out, ldo, n, N, K, xt, tiles,
                                                                 ldo % 8 == 0 && aligned(out, 16));
  return hipGetLastError();
}

hipError_t gemm_tiles(const uint8_t* wq, const uint8_t* xq, long ldx, const uint8_t* xs, long lds, __bf16* out,
                      long ldo, int n, int N, int K, hipStream_t stream) {
  return run<4, 2, 2, 4>(wq, xq, ldx, xs, lds, out, ldo, n, N, K, stream);
}

}  // namespace mx
}  // namespace qe
