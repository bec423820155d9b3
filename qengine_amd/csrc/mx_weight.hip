// Weights in microscaled 4-bit floating point (E2M1 codes, a scale for 32 values): from bf16, and back.
//
// A lane owns a block: it reads 64 bytes of its row, so no lane needs another's values, and its 16 bytes of codes
// are where the tile's layout has them; a wave covers 16 rows by 512 values and writes 4 KB of codes and 256
// bytes of scales, both contiguous. Bound by memory.
#include "mx_common.hpp"

namespace qe {
namespace mx {

// 32 values of row `row` from k on (16-byte pieces where VEC), zeros from K on, as eight pieces of four dwords.
template <bool VEC>
__device__ __forceinline__ void load_block(const __bf16* __restrict__ row, int k, int K, u32x4_t (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = u32x4_t{0u, 0u, 0u, 0u};
    if constexpr (VEC) {
      if (k + 8 * i < K) v[i] = *reinterpret_cast<const u32x4_t*>(row + k + 8 * i);
    } else {
      const uint16_t* p = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + 8 * i + j < K) v[i][j / 2] |= (uint32_t)p[k + 8 * i + j] << (16 * (j & 1));
    }
  }
}

template <bool VEC>
__global__ void __launch_bounds__(256)
mx4_quant_kernel(const __bf16* __restrict__ w, long ldw, uint8_t* __restrict__ wq, int N, int K) {
  const Layout L(N, K);
  const int lane = threadIdx.x & (WAVE - 1), r = lane & 15, g = lane >> 4;
  const int J = blockIdx.y * 4 + threadIdx.x / WAVE, rt = blockIdx.x;
  if (J >= L.KS) return;
  const int row = rt * 16 + r;
  const __bf16* src = w + (size_t)min(row, N - 1) * ldw;
  uint32_t scales = 0;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int kt = J * 4 + t;
    if (kt >= L.KT) break;
    u32x4_t v[4];
    load_block<VEC>(src, kt * 128 + g * BLOCK, row < N ? K : 0, v);
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        top = max(top, max(v[i][j] << 16 & 0x7fffffffu, v[i][j] & 0x7fff0000u));
    const int c = scale4(top);
    u32x4_t codes = {0u, 0u, 0u, 0u};
    if (c != 255) {
      const float f = inverse(c);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t d = 0;
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][0]) * f, hi_bf16(v[i][0]) * f, 1.0f, 0);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][1]) * f, hi_bf16(v[i][1]) * f, 1.0f, 1);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][2]) * f, hi_bf16(v[i][2]) * f, 1.0f, 2);
        d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][3]) * f, hi_bf16(v[i][3]) * f, 1.0f, 3);
        codes[i] = d;
      }
    }
    scales |= (uint32_t)c << (8 * t);
    reinterpret_cast<u32x4_t*>(wq + ((size_t)rt * L.KT + kt) * 1024)[lane] = codes;
  }
  reinterpret_cast<uint32_t*>(wq + L.scales() + ((size_t)rt * L.KS + J) * 256)[lane] = scales;
}

template <bool VEC>
__global__ void __launch_bounds__(256)
mx4_dequant_kernel(const uint8_t* __restrict__ wq, __bf16* __restrict__ out, long ldo, int N, int K) {
  const Layout L(N, K);
  const int lane = threadIdx.x & (WAVE - 1), r = lane & 15, g = lane >> 4;
  const int J = blockIdx.y * 4 + threadIdx.x / WAVE, rt = blockIdx.x;
  const int row = rt * 16 + r;
  if (J >= L.KS || row >= N) return;
  const uint32_t scales = reinterpret_cast<const uint32_t*>(wq + L.scales() + ((size_t)rt * L.KS + J) * 256)[lane];
  __bf16* dst = out + (size_t)row * ldo;
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int kt = J * 4 + t, k = kt * 128 + g * BLOCK;
    if (k >= K) break;
    const u32x4_t codes = reinterpret_cast<const u32x4_t*>(wq + ((size_t)rt * L.KT + kt) * 1024)[lane];
    const float f = value((int)(scales >> (8 * t) & 255u));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // exact in fp32, and a bf16 value: a subnormal scale too
      const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 0);
      const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 1);
      const auto d = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 2);
      const auto e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(codes[i], 1.0f, 3);
      const u32x4_t v = {pack_bf16x2(a[0] * f, a[1] * f), pack_bf16x2(b[0] * f, b[1] * f),
                         pack_bf16x2(d[0] * f, d[1] * f), pack_bf16x2(e[0] * f, e[1] * f)};
      if constexpr (VEC) {
        if (k + 8 * i < K) *reinterpret_cast<u32x4_t*>(dst + k + 8 * i) = v;
      } else {
        uint16_t* p = reinterpret_cast<uint16_t*>(dst);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (k + 8 * i + j < K) p[k + 8 * i + j] = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
      }
    }
  }
}

}  // namespace mx
}  // namespace qe

using namespace qe;
using namespace qe::mx;

extern "C" size_t qe_mx4_bytes(int N, int K) { return dims_ok(N, K) ? Layout(N, K).bytes() : 0; }

// Whole 16-byte pieces: the width and the row stride are multiples of 8 values, the base is aligned.
static bool pieces(const void* p, long ld, int K) { return K % 8 == 0 && ld % 8 == 0 && aligned(p, 16); }

extern "C" hipError_t qe_mx4_quant(const void* w, long ldw, void* wq, int N, int K, hipStream_t stream) {
  if (!w || !wq || !dims_ok(N, K) || !ld_ok(ldw, K) || !aligned(wq, 16) || !aligned(w, 2))
    return hipErrorInvalidValue;
  const Layout L(N, K);
  const dim3 grid(L.RT, (L.KS + 3) / 4);
  const auto* W = static_cast<const __bf16*>(w);
  auto* Q = static_cast<uint8_t*>(wq);
  if (pieces(w, ldw, K))
    mx4_quant_kernel<true><<<grid, dim3(256), 0, stream>>>(W, ldw, Q, N, K);
  else
    mx4_quant_kernel<false><<<grid, dim3(256), 0, stream>>>(W, ldw, Q, N, K);
  return hipGetLastError();
}

extern "C" hipError_t qe_mx4_dequant(const void* wq, void* out, long ldo, int N, int K, hipStream_t stream) {
  if (!wq || !out || !dims_ok(N, K) || !ld_ok(ldo, K) || !aligned(wq, 16) || !aligned(out, 2))
    return hipErrorInvalidValue;
  const Layout L(N, K);
  const dim3 grid(L.RT, (L.KS + 3) / 4);
  const auto* Q = static_cast<const uint8_t*>(wq);
  auto* O = static_cast<__bf16*>(out);
  if (pieces(out, ldo, K))
    mx4_dequant_kernel<true><<<grid, dim3(256), 0, stream>>>(Q, O, ldo, N, K);
  else
    mx4_dequant_kernel<false><<<grid, dim3(256), 0, stream>>>(Q, O, ldo, N, K);
  return hipGetLastError();
}
