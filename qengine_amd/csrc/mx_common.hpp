// Microscaled formats on gfx950: the layout of a 4-bit weight, and the scale of a block of 32 values.
#pragma once
#include "qe_device.hpp"
#include "qe_mx.h"

namespace qe {
namespace mx {

constexpr int BLOCK = 32;  // values under one scale

// An [N][K] weight in memory: tiles of 16 rows by 128 values, row tile by row tile, a tile's 1 KB in lane order of
// the 16x16x128 matrix instruction (lane r + 16 g: the 32 codes of row r, block g, 16 bytes, the lower half of
// a byte first); then the scales, 256 bytes for four tiles along K: lane r + 16 g holds the four scale codes
// of row r, block g of the tiles in order, which is the instruction's scale register, its byte picked by op_sel.
// A wave reads both as they lie, 16 and 4 bytes a lane. Rows and blocks past the matrix are zero codes under
// scale code 0.
struct Layout {
  int RT, KT, KS;  // row tiles, tiles along K, groups of four of them
  __host__ __device__ Layout(int N, int K) : RT((N + 15) / 16), KT((K + 127) / 128), KS((KT + 3) / 4) {}
  __host__ __device__ size_t scales() const { return (size_t)RT * KT * 1024; }  // where the scales begin
  __host__ __device__ size_t bytes() const { return scales() + (size_t)RT * KS * 256; }
};

__host__ inline bool dims_ok(int rows, int width) {
  return rows >= 1 && rows <= QE_MX_MAX_ROWS && width >= 1 && width <= QE_MX_MAX_WIDTH;
}
__host__ inline bool ld_ok(long ld, long width) { return ld >= width && ld < (1L << 23); }
__host__ inline bool aligned(const void* p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }

// Scale codes of a block whose largest magnitude has the fp32 bits `top` (sign off): the smallest exponent at which
// it does not round past the largest code, 255 for an infinity or NaN. A mantissa from 1.75 on (E2M1: 7 = 1.75 *
// 2^2 would round to 8), or above 1.8125 (E4M3: 464 = 1.8125 * 2^8 is the last that rounds to 448), carries
// into the exponent.
__device__ __forceinline__ int scale4(uint32_t top) {
  return top >= 0x7f800000u ? 255 : max((int)((top + 0x200000u) >> 23) - 2, 0);
}
__device__ __forceinline__ int scale8(uint32_t top) {
  return top >= 0x7f800000u ? 255 : max((int)((top + 0x17ffffu) >> 23) - 8, 0);
}
// 2^-e of scale code c (c <= 253, as above for finite blocks): exact, and normal for every such code.
__device__ __forceinline__ float inverse(int c) { return __uint_as_float((uint32_t)(254 - c) << 23); }
// 2^e of scale code c: subnormal for 0, NaN for 255.
__device__ __forceinline__ float value(int c) {
  return __uint_as_float(c == 0 ? 0x00400000u : c == 255 ? 0x7fc00000u : (uint32_t)c << 23);
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The largest of four neighbouring lanes (4i .. 4i + 3).
__device__ __forceinline__ uint32_t quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, false));  // lane ^ 1
  return max(v, (uint32_t)__builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, false));  // lane ^ 2
}

// Eight values over 2^e as E4M3 codes (|v| / 2^e <= 464, so none becomes NaN), or eight NaN codes under scale 255.
__device__ __forceinline__ u32x2_t codes8(const float (&v)[8], int c) {
  if (c == 255) return u32x2_t{0x7f7f7f7fu, 0x7f7f7f7fu};
  const float f = inverse(c);
  int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0] * f, v[1] * f, 0, false);
  a = __builtin_amdgcn_cvt_pk_fp8_f32(v[2] * f, v[3] * f, a, true);
  int b = __builtin_amdgcn_cvt_pk_fp8_f32(v[4] * f, v[5] * f, 0, false);
  b = __builtin_amdgcn_cvt_pk_fp8_f32(v[6] * f, v[7] * f, b, true);
  return u32x2_t{(uint32_t)a, (uint32_t)b};
}

}  // namespace mx
}  // namespace qe
