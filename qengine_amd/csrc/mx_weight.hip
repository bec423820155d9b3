// Weights in microscaled 4-bit floating point (E2M1 codes, a scale for 32 values): from bf16, and back.
//
// Both are bound by memory: 2 + 17/32 bytes a value. A workgroup owns 16 rows by 512 values: 4 KB of codes and 256
// bytes of scales, both contiguous. In bf16 a lane holds 8 neighbouring values, a quad a block, and 16 lanes a row's
// 256 bytes, so that one instruction covers 4 rows by two whole lines; in codes a lane has 16 bytes, a block of one
// row. A quad turns one into the other: lane q's dword of row 4 i + l is dword q of lane i, a 4 x 4 transposition.
// 34816 x 5120, four weights in turn: 81 us there, 79 us back (5.6 and 5.7 TB/s; a large copy reaches 4.8, but reads
// as much as it writes), 173 us as a pair, where each begins behind the other's stores. With a block of 64 bytes a
// lane, whose instructions touch 64 lines each, 130 us one way.
#include <limits.h>

#include <type_traits>

#include "mx_common.hpp"

namespace qe {
namespace mx {

// Lane q of a quad gives d[i] to lane i, as that lane's d[q].
__device__ __forceinline__ u32x4_t quad_transpose(u32x4_t d, int q) {
  auto swap = [](uint32_t v, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)v, decltype(ctrl)::value, 0xF, 0xF, false);
  };
  constexpr std::integral_constant<int, 0xB1> one{};  // lane ^ 1
  constexpr std::integral_constant<int, 0x4E> two{};  // lane ^ 2
  const bool o = q & 1, h = q & 2;
  const uint32_t a = swap(o ? d[0] : d[1], one), b = swap(o ? d[2] : d[3], one);
  const uint32_t e0 = o ? a : d[0], e1 = o ? d[1] : a, e2 = o ? b : d[2], e3 = o ? d[3] : b;
  const uint32_t c = swap(h ? e0 : e2, two), f = swap(h ? e1 : e3, two);
  return h ? u32x4_t{c, f, e2, e3} : u32x4_t{e0, e1, c, f};
}

// A workgroup has 16 rows by 512 values, a wave 128 of them.
struct Place {
  int rt, J, t, q, g, l;  // 16 rows, 512 values, tile of 128; quarter of a block, block, row of four
  __device__ __forceinline__ Place(const Layout& L) {
    rt = blockIdx.x / L.KS;
    J = blockIdx.x % L.KS;
    t = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    q = threadIdx.x & 3;
    g = threadIdx.x >> 2 & 3;
    l = threadIdx.x >> 4 & 3;
  }
  __device__ __forceinline__ int code_lane() const { return 4 * q + l + 16 * g; }
};

__global__ void __launch_bounds__(256)
mx4_quant_kernel(const __bf16* __restrict__ w, long ldw, uint8_t* __restrict__ wq, int N, int K) {
  __shared__ uint32_t scales[WAVE];  // a lane's four, by bytes
  const Layout L(N, K);
  const Place p(L);
  const int kt = p.J * 4 + p.t, k = kt * 128 + p.g * BLOCK + 8 * p.q;
  u32x4_t v[4];  // of row 4 i + l
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = p.rt * 16 + 4 * i + p.l;
    const __bf16* src = w + (size_t)row * ldw + k;
    v[i] = u32x4_t{0u, 0u, 0u, 0u};
    if (row < N && k + 8 <= K)
      __builtin_memcpy(&v[i], src, 16);  // at any address
    else if (row < N)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) v[i][j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(src)[j] << (16 * (j & 1));
  }
  u32x4_t codes;
  uint32_t mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) top = max(top, max(v[i][j] << 16 & 0x7fffffffu, v[i][j] & 0x7fff0000u));
    const int c = scale4(quad_max(top));
    const float f = inverse(min(c, 253));
    uint32_t d = 0;
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][0]) * f, hi_bf16(v[i][0]) * f, 1.0f, 0);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][1]) * f, hi_bf16(v[i][1]) * f, 1.0f, 1);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][2]) * f, hi_bf16(v[i][2]) * f, 1.0f, 2);
    d = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(d, lo_bf16(v[i][3]) * f, hi_bf16(v[i][3]) * f, 1.0f, 3);
    codes[i] = c == 255 ? 0u : d;
    mine = p.q == i ? (uint32_t)c : mine;
  }
  if (kt < L.KT)
    reinterpret_cast<u32x4_t*>(wq + ((size_t)p.rt * L.KT + kt) * 1024)[p.code_lane()] = quad_transpose(codes, p.q);
  reinterpret_cast<uint8_t*>(scales + p.code_lane())[p.t] = kt < L.KT ? (uint8_t)mine : 0;
  __syncthreads();
  if (p.t == 0)
    reinterpret_cast<uint32_t*>(wq + L.scales() + ((size_t)p.rt * L.KS + p.J) * 256)[threadIdx.x] =
        scales[threadIdx.x];
}

__global__ void __launch_bounds__(256)
mx4_dequant_kernel(const uint8_t* __restrict__ wq, __bf16* __restrict__ out, long ldo, int N, int K) {
  const Layout L(N, K);
  const Place p(L);
  const int kt = p.J * 4 + p.t, k = kt * 128 + p.g * BLOCK + 8 * p.q;
  if (kt >= L.KT) return;
  const int scale = wq[L.scales() + ((size_t)p.rt * L.KS + p.J) * 256 + p.code_lane() * 4 + p.t];
  const u32x4_t d =
      quad_transpose(reinterpret_cast<const u32x4_t*>(wq + ((size_t)p.rt * L.KT + kt) * 1024)[p.code_lane()], p.q);
  auto give = [&](int i, int c) {  // c: the scale of row 4 i + l
    const float f = value(c);
    // exact in fp32, and a bf16 value: a subnormal scale too
    const auto a = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 0);
    const auto b = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 1);
    const auto e = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 2);
    const auto h = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(d[i], 1.0f, 3);
    const u32x4_t v = {pack_bf16x2(a[0] * f, a[1] * f), pack_bf16x2(b[0] * f, b[1] * f),
                       pack_bf16x2(e[0] * f, e[1] * f), pack_bf16x2(h[0] * f, h[1] * f)};
    const int row = p.rt * 16 + 4 * i + p.l;
    __bf16* dst = out + (size_t)row * ldo + k;
    if (row < N && k + 8 <= K)
      __builtin_memcpy(dst, &v, 16);  // at any address
    else if (row < N)
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (k + j < K) reinterpret_cast<uint16_t*>(dst)[j] = (uint16_t)(v[j / 2] >> (16 * (j & 1)));
  };
  // lane i of a quad has the scale of row 4 i + l
  give(0, __builtin_amdgcn_mov_dpp(scale, 0x00, 0xF, 0xF, false));
  give(1, __builtin_amdgcn_mov_dpp(scale, 0x55, 0xF, 0xF, false));
  give(2, __builtin_amdgcn_mov_dpp(scale, 0xAA, 0xF, 0xF, false));
  give(3, __builtin_amdgcn_mov_dpp(scale, 0xFF, 0xF, 0xF, false));
}

}  // namespace mx
}  // namespace qe

using namespace qe;
using namespace qe::mx;

extern "C" size_t qe_mx4_bytes(int N, int K) { return dims_ok(N, K) ? Layout(N, K).bytes() : 0; }

// Workgroups; 0 if more than a grid holds.
static uint32_t groups(const Layout& L) {
  const size_t g = (size_t)L.RT * L.KS;
  return g <= UINT_MAX / 256 ? (uint32_t)g : 0;
}

extern "C" hipError_t qe_mx4_quant(const void* w, long ldw, void* wq, int N, int K, hipStream_t stream) {
  if (!w || !wq || !dims_ok(N, K) || !ld_ok(ldw, K) || !aligned(wq, 16) || !aligned(w, 2) || !groups(Layout(N, K)))
    return hipErrorInvalidValue;
  mx4_quant_kernel<<<dim3(groups(Layout(N, K))), dim3(256), 0, stream>>>(static_cast<const __bf16*>(w), ldw,
                                                                         static_cast<uint8_t*>(wq), N, K);
  return hipGetLastError();
}

extern "C" hipError_t qe_mx4_dequant(const void* wq, void* out, long ldo, int N, int K, hipStream_t stream) {
  if (!wq || !out || !dims_ok(N, K) || !ld_ok(ldo, K) || !aligned(wq, 16) || !aligned(out, 2) ||
      !groups(Layout(N, K)))
    return hipErrorInvalidValue;
  mx4_dequant_kernel<<<dim3(groups(Layout(N, K))), dim3(256), 0, stream>>>(static_cast<const uint8_t*>(wq),
                                                                           static_cast<__bf16*>(out), ldo, N, K);
  return hipGetLastError();
}
