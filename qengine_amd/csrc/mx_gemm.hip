// The product of 8-bit rows and a 4-bit weight (microscaled formats) on gfx950's scaled matrix instructions: codes
// and scales go into them as they lie in memory, no value is converted.
#include "mx_common.hpp"
#include "mx_gemm.hpp"

namespace qe {
namespace mx {

typedef int i32x8_t __attribute__((ext_vector_type(8)));

// D (16 x 16) += A (16 weight rows x 128) * B (128 x 16 rows), A E2M1 and B E4M3 codes. Lane r + 16 g: A's row r,
// block g (16 bytes); B's row r at 16 g .. 16 g + 15 and 64 + 16 g .. 64 + 16 g + 15; the scales of A's and of B's row r,
// block g (byte T of `sa`, byte 0 of `sb`). It gets D's rows 4 g .. 4 g + 3 of column r.
template <int T>
__device__ __forceinline__ f32x4_t mfma_mx(u32x4_t a, u32x4_t b0, u32x4_t b1, f32x4_t d, uint32_t sa, uint32_t sb) {
  const i32x8_t A = {(int)a[0], (int)a[1], (int)a[2], (int)a[3], 0, 0, 0, 0};
  const i32x8_t B = {(int)b0[0], (int)b0[1], (int)b0[2], (int)b0[3], (int)b1[0], (int)b1[1], (int)b1[2], (int)b1[3]};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(A, B, d, 4, 0, T, (int)sa, 0, (int)sb);
}

constexpr int WAVES = 8;

template <int NT>
__global__ void __launch_bounds__(WAVES * WAVE)
gemm_mx4_kernel(const uint8_t* __restrict__ wq, const uint8_t* __restrict__ xq, long ldx,
                const uint8_t* __restrict__ xs, long lds, __bf16* __restrict__ out, long ldo, int n, int N, int K) {
  __shared__ f32x4_t part[WAVES][NT][WAVE];
  const Layout L(N, K);
  const int lane = threadIdx.x & (WAVE - 1), r = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
  const int rt = blockIdx.x, col = blockIdx.y * 16 * NT;
  f32x4_t acc[NT];
  const uint8_t *xr[NT], *sr[NT];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    acc[i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    const size_t row = min(col + 16 * i + r, n - 1);
    xr[i] = xq + row * ldx;
    sr[i] = xs + row * lds;
  }
  for (int J = w; J < L.KS; J += WAVES) {
    const uint32_t sa = reinterpret_cast<const uint32_t*>(wq + L.scales() + ((size_t)rt * L.KS + J) * 256)[lane];
#define QE_STEP(T)                                                                                               \
  if (J * 4 + T < L.KT) {                                                                                        \
    const int kt = J * 4 + T, k = kt * 128 + 16 * g;                                                             \
    const u32x4_t a = reinterpret_cast<const u32x4_t*>(wq + ((size_t)rt * L.KT + kt) * 1024)[lane];              \
    _Pragma("unroll") for (int i = 0; i < NT; ++i) {                                                             \
      u32x4_t b0 = {0u, 0u, 0u, 0u}, b1 = {0u, 0u, 0u, 0u};                                                      \
      uint32_t sb = 0;                                                                                           \
      if (k < K) b0 = *reinterpret_cast<const u32x4_t*>(xr[i] + k);                                              \
      if (k + 64 < K) b1 = *reinterpret_cast<const u32x4_t*>(xr[i] + k + 64);                                    \
      if (kt * 4 + g < K / BLOCK) sb = sr[i][kt * 4 + g];                                                        \
      acc[i] = mfma_mx<T>(a, b0, b1, acc[i], sa, sb);                                                            \
    }                                                                                                            \
  }
    QE_STEP(0) QE_STEP(1) QE_STEP(2) QE_STEP(3)
#undef QE_STEP
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    asm volatile("" : "+v"(acc[i]));  // the products stay out of the stores' branches, where lanes are off
    part[w][i][lane] = acc[i];
  }
  __syncthreads();
  for (int i = w; i < NT; i += WAVES) {
    f32x4_t t = part[0][i][lane];
    for (int p = 1; p < WAVES; ++p) t += part[p][i][lane];
    const int row = col + 16 * i + r, j = rt * 16 + 4 * g;
    if (row < n)
      for (int e = 0; e < 4; ++e)
        if (j + e < N) out[(size_t)row * ldo + j + e] = f32_to_bf16(t[e]);
  }
}

}  // namespace mx
}  // namespace qe

using namespace qe;
using namespace qe::mx;

extern "C" size_t qe_gemm_mx4_ws_size(int, int, int) { return 0; }

extern "C" hipError_t qe_gemm_mx4(const void* wq, const void* xq, long ldx, const void* xs, long lds, void* out,
                                  long ldo, int n, int N, int K, void* ws, size_t, hipStream_t stream) {
  if (!wq || !xq || !xs || !out || !dims_ok(n, K) || !dims_ok(N, K) || K % BLOCK || !ld_ok(ldx, K) || ldx % 16 ||
      !ld_ok(lds, K / BLOCK) || !ld_ok(ldo, N) || !aligned(wq, 16) || !aligned(xq, 16) || !aligned(out, 2) || !aligned(ws, 16))
    return hipErrorInvalidValue;
  const int RT = Layout(N, K).RT;
  const auto *W = static_cast<const uint8_t*>(wq), *X = static_cast<const uint8_t*>(xq),
             *S = static_cast<const uint8_t*>(xs);
  auto* O = static_cast<__bf16*>(out);
  if (n <= 16)
    gemm_mx4_kernel<1><<<dim3(RT), dim3(WAVES * WAVE), 0, stream>>>(W, X, ldx, S, lds, O, ldo, n, N, K);
  else if (n > 128)
    return gemm_tiles(W, X, ldx, S, lds, O, ldo, n, N, K, stream);
  else
    gemm_mx4_kernel<4><<<dim3(RT, (n + 63) / 64), dim3(WAVES * WAVE), 0, stream>>>(W, X, ldx, S, lds, O, ldo, n, N, K);
  return hipGetLastError();
}
