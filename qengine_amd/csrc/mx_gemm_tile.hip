// The product of 8-bit rows and a 4-bit weight for many rows: tiles of WX x TX x 32 rows by WW x TW x 32 weight rows.
//
// Bound by the matrix cores at the clock that the card's power allows: 2048 x 32768 x 5120 is four tiles of 256 x 256
// a CU, 250 us, 2,750 TFLOP/s (a library's product of two 8-bit matrices: 2,700), the cores busy 70 % of the time at
// 1.9 GHz; on zeros, at full clock, it takes 209 us. 64 KB of LDS reads a step against 2,048 cycles of products: a
// wave's 64 x 128 outputs take 128 of its registers, and larger ones do not fit.
#include <limits.h>

#include <algorithm>

#include "mx_common.hpp"
#include "mx_gemm.hpp"

namespace qe {
namespace mx {

template <int WX, int WW, int TX, int TW>
struct Tile {
  static constexpr int WAVES = WX * WW, ROWS = WX * TX * 32, COLS = WW * TW * 32;
  static constexpr int XB = ROWS * 128, STAGE = XB + COLS * 64;  // bytes of a stage: x, then the weight
  static constexpr int DX = (ROWS / 8 + WAVES - 1) / WAVES, DW = (COLS / 16 + WAVES - 1) / WAVES;  // a wave's loads
  static_assert(WAVES % 2 == 0, "a wave's loads of x are of one parity");
  static constexpr int PER_CU = 3 * STAGE <= 81920 && TX * TW <= 2 ? 2 : 1;  // workgroups
  // on the way out a wave turns 32 rows of OUT values at a time around in its share of a stage
  static constexpr int OUT = STAGE / WAVES >= 32 * 144 && TW % 2 == 0 ? 64 : 32;
  static constexpr int PITCH = OUT * 2 + (STAGE / WAVES >= 32 * (OUT * 2 + 16) ? 16 : 0);  // bytes
  static_assert(STAGE / WAVES >= 32 * PITCH, "its share holds them");
};

struct Call : Product {
  int xtiles, tiles;
};

template <int WX, int WW, int TX, int TW, class T = Tile<WX, WW, TX, TW>>
__global__ void __launch_bounds__(T::WAVES * WAVE, T::WAVES / 4 * T::PER_CU)
gemm_mx4_tile_kernel(const Call c) {
  __shared__ __attribute__((aligned(1024))) uint8_t smem[3 * T::STAGE];
  const Layout L(c.N, c.K);
  const int lane = threadIdx.x & (WAVE - 1), r = lane & 31, g = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int wx = w % WX, ww = w / WX;
  const int KT = L.KT, Kb = c.K / BLOCK;
  const int steps = max(KT, 2);  // of a tile: the loads run two steps ahead, into the next tile

  // Workgroups go to the 8 XCDs in turn; each XCD gets neighbouring tiles, the row tiles of a weight tile first, and
  // its workgroups take them in turn.
  const int q8 = c.tiles / 8, r8 = c.tiles % 8, xcd = blockIdx.x % 8;
  const int stride = ((int)gridDim.x - xcd + 7) / 8;
  const int begin = xcd * q8 + min(xcd, r8), end = begin + q8 + (xcd < r8 ? 1 : 0);

  // x: 8 rows of 128 bytes a load; slot s of row i holds chunk s ^ (i / 2 % 8), so that 16 rows' reads of a chunk meet
  // no bank twice and the row's 128 bytes are one request. The weight: a 16-row tile's 1 KB a load. Rows and
  // chunks past the matrix are zeros: they lie outside the buffers.
  const int chunk16 = ((lane & 7) ^ ((min(w, T::ROWS / 8 - 1) & 1) * 4 + (lane >> 4))) * 16;
  uint32_t xo[T::DX], wo[T::DW], xl[T::DX], wl[T::DW];
#pragma unroll
  for (int i = 0; i < T::DX; ++i) {
    const int id = min(w + i * T::WAVES, T::ROWS / 8 - 1);
    xo[i] = (uint32_t)((id * 8 + (lane >> 3)) * c.ldx + chunk16);
    xl[i] = lds_byte_uniform(smem) + id * 1024;
  }
#pragma unroll
  for (int i = 0; i < T::DW; ++i) {
    const int id = min(w + i * T::WAVES, T::COLS / 16 - 1);
    wo[i] = (uint32_t)id * KT * 1024u + lane * 16;
    wl[i] = lds_byte_uniform(smem) + T::XB + id * 1024;
  }
  struct Place {
    int x0, c0;       // first row, first weight row
    uint64_t xb, wb, sb;  // addresses of their codes, and of the weight's scales
    uint32_t xn, wn, sn;  // bytes from there on (0: no tile)
  };
  auto place = [&](int tile) {
    Place p = {0, 0, (uint64_t)c.xq, (uint64_t)c.wq, (uint64_t)c.wscale, 0u, 0u, 0u};
    if (tile < end) {
      p.x0 = tile % c.xtiles * T::ROWS;
      p.c0 = tile / c.xtiles * T::COLS;
      p.xb += (uint64_t)p.x0 * c.ldx;
      p.wb += (uint64_t)(p.c0 / 16) * KT * 1024u;
      p.xn = (uint32_t)((min(T::ROWS, c.n - p.x0) - 1) * c.ldx + c.K);
      p.wn = (uint32_t)min(T::COLS / 16, L.RT - p.c0 / 16) * KT * 1024u;
      p.sb += (uint64_t)(p.c0 / 16) * L.KS * 256u;
      p.sn = (uint32_t)min(T::COLS / 16, L.RT - p.c0 / 16) * L.KS * 256u;
    }
    return p;
  };
  int tile = begin + (int)blockIdx.x / 8;
  Place cur = place(tile), next = place(tile + stride);

  constexpr int LOADS = T::DX + T::DW;
  Place from = cur;  // where the loads are: two steps ahead of the products
  int at = -1;       // their step
  auto fetch = [&](int stage, int i) {  // load i of this wave
    if (i < T::DX) {
      const uint32_t past = at * 128 + chunk16 >= c.K ? 0x80000000u : 0u;
      const __amdgpu_buffer_rsrc_t xr = make_rsrc_uniform((const void*)from.xb, from.xn);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          xr, (__attribute__((address_space(3))) void*)(uintptr_t)(xl[i] + stage * T::STAGE), 16,
          (int)((xo[i] + at * 128) | past), 0, 0, 0);
    } else {
      const __amdgpu_buffer_rsrc_t wr = make_rsrc_uniform((const void*)from.wb, from.wn);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          wr, (__attribute__((address_space(3))) void*)(uintptr_t)(wl[i - T::DX] + stage * T::STAGE), 16,
          (int)(wo[i - T::DX] + min(at, KT - 1) * 1024), 0, 0, 0);
    }
  };
  auto advance = [&]() {  // ahead of a step's loads
    ++at;
    asm volatile("" : "+s"(at));  // or the compiler works out all of the loop's wraps in its first turn
    const bool wrap = at == steps;
    at = wrap ? 0 : at;
    from.xb = wrap ? next.xb : from.xb;
    from.wb = wrap ? next.wb : from.wb;
    from.xn = wrap ? next.xn : from.xn;
    from.wn = wrap ? next.wn : from.wn;
  };

  // Scales of four steps: of x, 16 bytes of lane r's row; of the weight, a dword for blocks g and 2 + g of a tile. The
  // last ones of x come from the row's end, shifted down: no byte past the row is read, and blocks past K
  // get code 0. Rows of fewer than 16 blocks are read a byte at a time, as a tile begins.
  const uint32_t so = (uint32_t)(ww * TW * 2 + (r >> 4)) * L.KS * 256u + ((r & 15) + 16 * g) * 4;
  uint32_t sw[TW][2], sw2[TW][2];
  u32x4_t sx[TX], sx2[TX];
  constexpr int SCALES = 2 * TW + TX;  // loads of scales()
  auto row_of = [&](int x0, int i) { return (size_t)min(x0 + (wx * TX + i) * 32 + r, c.n - 1); };
  // (with fewer than 16 blocks a row, what is loaded ahead is never used: from a place of no account)
  const bool small = Kb < 16;
  const int last16 = small ? 0 : Kb - 16;
  int group = -1;  // of four steps, the loaded one
  uint64_t sb = cur.sb;
  uint32_t sn = cur.sn;
  const uint8_t *xp[TX], *xp2[TX];  // lane r's rows of this tile, of the next
  auto rows_of = [&](const Place& p, const uint8_t* (&to)[TX]) {
#pragma unroll
    for (int i = 0; i < TX; ++i) to[i] = small ? c.wq : c.xs + row_of(p.x0, i) * c.lds;
  };
  auto scales = [&]() {  // the next group's, past the tile's end those of the next tile's first
    ++group;
    asm volatile("" : "+s"(group));
    const bool wrap = group * 4 >= steps;
    group = wrap ? 0 : group;
    sb = wrap ? next.sb : sb;
    sn = wrap ? next.sn : sn;
    const __amdgpu_buffer_rsrc_t sr = make_rsrc_uniform((const void*)(sb + group * 256), sn - group * 256u);
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        sw2[j][h] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(sr, (int)(so + j * 2 * L.KS * 256 + h * 128), 0, 0);
#pragma unroll
    for (int i = 0; i < TX; ++i) {
      xp[i] = wrap ? xp2[i] : xp[i];
      __builtin_memcpy(&sx2[i], xp[i] + min(group * 16, last16), 16);
    }
  };
  auto small_scales = [&](int x0) {
    int last = Kb - 1;
    asm volatile("" : "+s"(last));  // sixteen addresses stay out of the registers of the loop
#pragma unroll
    for (int i = 0; i < TX; ++i) {
      const uint8_t* p = c.xs + row_of(x0, i) * c.lds;
      sx2[i] = u32x4_t{0u, 0u, 0u, 0u};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t v = p[min(e, last)];
        sx2[i][e / 4] |= (e <= last ? v : 0u) << (8 * (e & 3));
      }
    }
  };
  auto take = [&](int J, const Place& p) {  // the loaded ones become those of steps 4 J ..
    if (small) small_scales(p.x0);
    const int cut = J * 16 - last16;  // bytes
#pragma unroll
    for (int j = 0; j < TW; ++j)
#pragma unroll
      for (int h = 0; h < 2; ++h) sw[j][h] = sw2[j][h];
    if (!small && cut > 0) {
#pragma unroll
      for (int i = 0; i < TX; ++i) {
        uint64_t lo = (uint64_t)sx2[i][1] << 32 | sx2[i][0], hi = (uint64_t)sx2[i][3] << 32 | sx2[i][2];
        if (cut >= 8) lo = hi, hi = 0;
        const int bits = (cut & 7) * 8;
        lo = lo >> bits | (bits ? hi << (64 - bits) : 0);
        hi >>= bits;
        sx2[i] = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
      }
    }
    // lanes 32 .. 63 hold blocks 1 and 3 of a step where the others hold 0 and 2
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sx[i][e] = sx2[i][e] >> (8 * g);
  };

  const bool lines = ((uintptr_t)c.out & 127) == 0 && (c.ldo & 63) == 0;
  f32x16_t acc[TX][TW];
  // where this lane reads, in the stage of the step at hand
  const int slot = r / 2 & 7;
  uint32_t wa = T::XB + (ww * TW * 2 + (r >> 4)) * 1024 + ((r & 15) + 16 * g) * 16, xa[2][2];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 2; ++e) xa[h][e] = (wx * TX * 32 + r) * 128 + (((4 * h + 2 * e + g) ^ slot) << 4);
  u32x4_t a[TW], b[TX][2];
  auto read = [&](int h) {
#pragma unroll
    for (int j = 0; j < TW; ++j) a[j] = *reinterpret_cast<const u32x4_t*>(smem + wa + j * 2048 + h * 512);
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) b[i][e] = *reinterpret_cast<const u32x4_t*>(smem + xa[h][e] + i * 4096);
  };
  int stage = 0;
  auto turn_stage = [&]() {
    const uint32_t by = stage == 2 ? (uint32_t)(-2 * T::STAGE) : (uint32_t)T::STAGE;
    stage = stage == 2 ? 0 : stage + 1;
    wa += by;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) xa[h][e] += by;
  };

  rows_of(cur, xp);
  rows_of(next, xp2);
  scales();
  advance();
#pragma unroll
  for (int i = 0; i < LOADS; ++i) fetch(0, i);
  advance();
#pragma unroll
  for (int i = 0; i < LOADS; ++i) fetch(1, i);
  take(0, cur);
  vmcnt_wait<LOADS>();
  lds_barrier();
  // Two halves of the workgroup, a wave of each on every SIMD, take turns: between two barriers one half reads its
  // operands of half a step (64 values) and issues loads, the other multiplies, so the matrix cores always have a
  // wave that does nothing else. The first half of the workgroup reads half step t in turn 2 t, the second in
  // turn 2 t + 1. Step k's two turns of each load step k + 2 into the place of step k - 1, which both have read
  // by then; step k + 1 has landed for every wave before its first turn: only step k + 2 is out (and, in
  // the first step of four, the next scales). The empty asm keeps the products where they are: the compiler takes
  // them for movable arithmetic, and would put them behind the next branch.
  const bool second = w >= T::WAVES / 2;
  if (second) lds_barrier();
#define QE_HALF(S, H)                                                                                       \
  {                                                                                                         \
    read(H);                                                                                                \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    if (H == 1) vmcnt_wait<LOADS / 2 + (S == 0 ? SCALES : 0)>();                                            \
    lds_barrier();                                                                                          \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    __builtin_amdgcn_s_setprio(1);                                                                          \
    const int free = stage >= 1 ? stage - 1 : 2;                                                            \
    if (H == 0) advance();                                                                                  \
    if (S == 0 && H == 0) scales();                                                                         \
    _Pragma("unroll") for (int t = H * (LOADS / 2); t < (H ? LOADS : LOADS / 2); ++t) fetch(free, t);       \
    if (H == 1) turn_stage();                                                                               \
    _Pragma("unroll") for (int i = 0; i < TX; ++i) _Pragma("unroll") for (int j = 0; j < TW; ++j)           \
        acc[i][j] = mfma32<S, 2 * H>(a[j], b[i][0], b[i][1], acc[i][j], sw[j][H], sx[i][S]);                \
    _Pragma("unroll") for (int q = 0; q < TX * TW; ++q) {                                                   \
      __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x6, 8, 0);                                                      \
      __builtin_amdgcn_sched_group_barrier(0x10, 2, 0);                                                     \
    }                                                                                                       \
    __builtin_amdgcn_s_setprio(0);                                                                          \
    _Pragma("unroll") for (int i = 0; i < TX; ++i) _Pragma("unroll") for (int j = 0; j < TW; ++j)           \
        asm volatile("" : "+v"(acc[i][j]));                                                                 \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
    lds_barrier();                                                                                          \
    __builtin_amdgcn_sched_barrier(0);                                                                      \
  }
#define QE_STEP(S) QE_HALF(S, 0) QE_HALF(S, 1)
  for (; tile < end; tile += stride) {
#pragma unroll
    for (int i = 0; i < TX; ++i)
#pragma unroll
      for (int j = 0; j < TW; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
    int kt = 0;
    for (; kt + 4 <= steps; kt += 4) {
      QE_STEP(0) QE_STEP(1) QE_STEP(2) QE_STEP(3)
      if (kt + 4 < steps) take(kt / 4 + 1, cur); else take(0, next);
    }
    if (kt < steps) {  // the last one to three: a loop with exits between would wait for all loads at each of them
      QE_STEP(0)
      if (kt + 1 < steps) { QE_STEP(1) }
      if (kt + 2 < steps) { QE_STEP(2) }
      take(0, next);
    }
    // Out, past the caches' favour where rows start on whole lines: a turn's outputs are as much as the L2s hold, and
    // the operands stay in them (2048 x 5120 x 6144 50 us against 54, 2048 x 34816 x 5120 the same; rows that start
    // within a line: 1736 x 22508 x 512 81 us against 40). That while the next tile's first two steps load. The place
    // of the last step is free: this half's turn begins when the other half has read it too, and loads go there only
    // behind the barrier below.
    uint8_t* mine = smem + (stage >= 1 ? stage - 1 : 2) * T::STAGE + w * (T::STAGE / T::WAVES);
#pragma unroll
    for (int i = 0; i < TX; ++i) {
#pragma unroll
      for (int part = 0; part < TW * 32 / T::OUT; ++part) {
#pragma unroll
        for (int jj = 0; jj < T::OUT / 32; ++jj)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const f32x16_t& d = acc[i][part * (T::OUT / 32) + jj];
            *reinterpret_cast<u32x2_t*>(mine + r * T::PITCH + jj * 64 + e * 16 + g * 8) =
                u32x2_t{pack_bf16x2(d[4 * e], d[4 * e + 1]), pack_bf16x2(d[4 * e + 2], d[4 * e + 3])};
          }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        constexpr int PER = T::OUT / 8;  // pieces of 8 values a row
#pragma unroll
        for (int t = 0; t < PER / 2; ++t) {
          const int pr = (lane + t * WAVE) / PER, pc = lane % PER;
          const int row = cur.x0 + (wx * TX + i) * 32 + pr, col = cur.c0 + ww * TW * 32 + part * T::OUT + pc * 8;
          const u32x4_t v = *reinterpret_cast<const u32x4_t*>(mine + pr * T::PITCH + pc * 16);
          __bf16* o = c.out + (size_t)min(row, c.n - 1) * c.ldo + col;
          if (row < c.n) {
            if (col + 8 <= c.N && lines)
              __builtin_nontemporal_store(v, reinterpret_cast<u32x4_t*>(o));
            else if (col + 8 <= c.N)
              __builtin_memcpy(o, &v, 16);  // at any address
            else
              for (int e = 0; e < 8; ++e)
                if (col + e < c.N) reinterpret_cast<uint16_t*>(o)[e] = (uint16_t)(v[e / 2] >> (16 * (e & 1)));
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
    lds_barrier();
    cur = next;
    next = place(tile + 2 * stride);
    rows_of(next, xp2);
  }
#undef QE_STEP
#undef QE_HALF
  if (!second) lds_barrier();
  vmcnt_wait<0>();  // loads into LDS that nothing reads
}

template <int WX, int WW, int TX, int TW>
static hipError_t run(const Product& p, hipStream_t stream) {
  using T = Tile<WX, WW, TX, TW>;
  const long xt = (p.n + T::ROWS - 1) / T::ROWS, tiles = xt * ((p.N + T::COLS - 1) / T::COLS);
  if (tiles > INT_MAX / 2) return hipErrorInvalidValue;  // more outputs than there is memory
  const Call c = {p, (int)xt, (int)tiles};
  gemm_mx4_tile_kernel<WX, WW, TX, TW>
      <<<dim3(std::min((int)tiles, compute_units() * T::PER_CU)), dim3(T::WAVES * WAVE), 0, stream>>>(c);
  return hipGetLastError();
}

hipError_t gemm_tiles(TileKind kind, const Product& p, hipStream_t stream) {
  switch (kind) {
    case TileKind::X256_W256: return run<4, 2, 2, 4>(p, stream);
    case TileKind::X128_W256: return run<4, 2, 1, 4>(p, stream);
    case TileKind::X256_W160: return run<8, 1, 1, 5>(p, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace mx
}  // namespace qe
