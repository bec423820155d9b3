// Rows in microscaled 8-bit floating point (E4M3 codes, a scale for 32 values): of a norm with the residual's
// addition, of SwiGLU, or of plain bf16 rows. The value is rounded once, from fp32 to its code.
//
// A lane has 8 values (a 16-byte read at any address, an 8-byte write), so a block is four neighbouring lanes and its
// largest magnitude two lane moves. Bound by memory, one row by the launch: SwiGLU of 2048 x 17408 36 us (4.9 TB/s, a
// large copy's rate), the norm of 2048 x 5120 14 us from the caches, 19 us from memory; of one row 2.7 us in a graph.
// Odd widths cost 5 to 15 % more (value by value it was 2 to 3 times: 2048 x 5001 norm 52 us, 21.5 us so). The norm's
// arithmetic is fp32, as in the framework's other norms: a value that lies within a few 2^-24 of the border between
// two codes may get the other one (about 15 of 10.5 million). In 64 bits it would not, at 3.0 us for one row and 20.5
// us for 2048.
#include <algorithm>

#include "mx_common.hpp"

namespace qe {
namespace mx {

__device__ __forceinline__ void unpack8(u32x4_t x, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = lo_bf16(x[i]);
    v[2 * i + 1] = hi_bf16(x[i]);
  }
}

// Values 8 c .. 8 c + 7 of a row of K, zeros from K on: the last ones come from the row's end, shifted down (TINY, K
// < 8: value by value; a choice at run time would cost one row's norm 0.15 us of 2.7).
template <bool TINY>
__device__ __forceinline__ void load8(const __bf16* row, int c, int K, float (&v)[8]) {
  u32x4_t x = {0u, 0u, 0u, 0u};
  if constexpr (!TINY) {
    __builtin_memcpy(&x, row + min(8 * c, K - 8), 16);
    const int cut = min(8 * c - (K - 8), 8);
    if (cut > 0) {
      uint64_t lo = (uint64_t)x[1] << 32 | x[0], hi = (uint64_t)x[3] << 32 | x[2];
      if (cut >= 4) lo = hi, hi = 0;
      if (cut >= 8) lo = 0;
      const int bits = (cut & 3) * 16;
      lo = lo >> bits | (bits ? hi << (64 - bits) : 0);
      hi >>= bits;
      x = u32x4_t{(uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32)};
    }
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (8 * c + j < K) x[j / 2] |= (uint32_t)reinterpret_cast<const uint16_t*>(row)[8 * c + j] << (16 * (j & 1));
  }
  unpack8(x, v);
}

// Eight values of this lane, a quarter of a block whose other quarters its three neighbours hold: codes and scale to
// row `q`, `s` at 8-value piece c (c < the padded width / 8; the caller's lanes of a block agree on that).
__device__ __forceinline__ void store8(const float (&v)[8], uint8_t* q, uint8_t* s, int c, bool live) {
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, magnitude(v[i]));
  const int code = scale8(quad_max(top));
  if (!live) return;
  reinterpret_cast<u32x2_t*>(q)[c] = codes8(v, code);
  if ((c & 3) == 0) s[c >> 2] = (uint8_t)code;
}

// silu(g) * u, g >= FAR. exp and the reciprocal are the instructions' (1 ulp each, 2^-23); the exponential's argument
// is off by 2^-24 (its rounding) and 2^-26 (the constant's) of itself. In all (0.61 |g| + 4) 2^-23 of the value, 2^-17
// at the most, far below the code's 2^-4.
constexpr float FAR = -64.f;
__device__ __forceinline__ float swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g)) * u;
}
// The same below FAR, where 1 + e^-g is e^-g in fp32 and leaves its range from g = -88 on, while g e^g u need not: e^g
// as a fraction in [1/2, 1) and an exponent that u takes first. Below 2^-300 no u has a code.
__device__ __forceinline__ float swiglu_far(float g, float u) {
  const float x = fmaxf(1.44269504f * g, -300.f), e = floorf(x) + 1.f;
  return g * ldexpf(__builtin_amdgcn_exp2f(x - e) * u, (int)e);
}

// ------------------------------------------------------------------------------ SwiGLU, plain rows
template <bool GLU, bool TINY>
__global__ void __launch_bounds__(256)
act_mx8_kernel(const __bf16* __restrict__ x, long ldx, uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ s,
               long lds, int K) {
  const size_t r = blockIdx.x;
  const __bf16* xr = x + r * ldx;
  const int c = blockIdx.y * blockDim.x + threadIdx.x;
  float v[8];
  load8<TINY>(xr, c, K, v);
  if constexpr (GLU) {
    float u[8];
    load8<TINY>(xr + K, c, K, u);
    float g[8], least = v[0];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      g[i] = v[i];
      least = fminf(least, g[i]);
      v[i] = swiglu(g[i], u[i]);
    }
    if (least < FAR) {  // hardly ever
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = g[i] < FAR ? swiglu_far(g[i], u[i]) : v[i];
    }
  }
  store8(v, q + r * ldq, s + r * lds, c, c < (K + BLOCK - 1) / BLOCK * 4);
}

// ------------------------------------------------------------------------------ RMSNorm1p
constexpr int NORM_THREADS = 1024;  // most of a workgroup

// Sum over the workgroup: wave butterflies, then the wave partials in order.
__device__ __forceinline__ float sum_rows(float v, float* red) {
  const int nw = blockDim.x / WAVE;
  v = wave_sum_fast(v);
  if ((threadIdx.x & (WAVE - 1)) == 0) red[threadIdx.x / WAVE] = v;
  __syncthreads();
  float t = red[0];
  for (int i = 1; i < nw; ++i) t += red[i];
  return t;
}

// Piece c of a row, with delta added; the sum, rounded, is written and taken on with.
template <bool TINY>
__device__ __forceinline__ void load_sum(const __bf16* x, const __bf16* delta, __bf16* sum, int c, int K,
                                         float (&v)[8]) {
  load8<TINY>(x, c, K, v);
  if (!delta) return;
  float d[8];
  load8<TINY>(delta, c, K, d);
  u32x4_t o;
#pragma unroll
  for (int j = 0; j < 4; ++j) o[j] = pack_bf16x2(v[2 * j] + d[2 * j], v[2 * j + 1] + d[2 * j + 1]);
  unpack8(o, v);
  if (8 * c + 8 <= K) {
    __builtin_memcpy(sum + 8 * c, &o, 16);
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (8 * c + j < K) reinterpret_cast<uint16_t*>(sum)[8 * c + j] = (uint16_t)(o[j / 2] >> (16 * (j & 1)));
  }
}

template <bool TINY>
__device__ __forceinline__ void weigh8(const __bf16* w, int c, int K, float inv, float (&v)[8]) {
  float g[8];
  load8<TINY>(w, c, K, g);
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = (v[j] * inv) * (1.0f + g[j]);
}

__device__ __forceinline__ float squares(const float (&v)[8]) {
  float t = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) t += v[j] * v[j];
  return t;
}

// A workgroup a row, C pieces of 8 values a thread, all in registers: piece c of thread t is t + c * threads.
template <int C, bool TINY>
__global__ void __launch_bounds__(NORM_THREADS)
norm_mx8_kernel(const __bf16* x, long ldx, const __bf16* delta, long ldd, const __bf16* __restrict__ w, __bf16* sum,
                long ldsum, uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ s, long lds, int K, float eps) {
  __shared__ float red[NORM_THREADS / WAVE];
  const size_t r = blockIdx.x;
  float v[C][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    load_sum<TINY>(x + r * ldx, delta ? delta + r * ldd : nullptr, sum + r * ldsum, threadIdx.x + i * blockDim.x, K,
                   v[i]);
    ss += squares(v[i]);
  }
  const float inv = 1.0f / sqrtf(sum_rows(ss, red) / (float)K + eps);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    weigh8<TINY>(w, c, K, inv, v[i]);
    store8(v[i], q + r * ldq, s + r * lds, c, c < (K + BLOCK - 1) / BLOCK * 4);
  }
}

// Rows that registers do not hold: two passes (the second reads what this thread read or wrote, so no other thread's
// write is involved).
__global__ void __launch_bounds__(NORM_THREADS)
norm_mx8_wide_kernel(const __bf16* x, long ldx, const __bf16* delta, long ldd, const __bf16* __restrict__ w,
                     __bf16* sum, long ldsum, uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ s, long lds,
                     int K, float eps) {
  __shared__ float red[NORM_THREADS / WAVE];
  const size_t r = blockIdx.x;
  const int pieces = (K + BLOCK - 1) / BLOCK * 4;
  float v[8];
  float ss = 0.f;
  for (int c = threadIdx.x; c < pieces; c += blockDim.x) {
    load_sum<false>(x + r * ldx, delta ? delta + r * ldd : nullptr, sum + r * ldsum, c, K, v);
    ss += squares(v);
  }
  const float inv = 1.0f / sqrtf(sum_rows(ss, red) / (float)K + eps);
  const __bf16* from = delta ? sum + r * ldsum : x + r * ldx;
  for (int c = threadIdx.x; c < pieces; c += blockDim.x) {  // whole blocks enter: a multiple of four lanes
    load8<false>(from, c, K, v);
    weigh8<false>(w, c, K, inv, v);
    store8(v, q + r * ldq, s + r * lds, c, true);
  }
}

}  // namespace mx
}  // namespace qe

using namespace qe;
using namespace qe::mx;

constexpr int LAUNCH_ROWS = 1 << 21;  // a grid has fewer than 2^32 threads

static bool rows_ok(const void* q, long ldq, const void* s, long lds, int n, int K) {
  const long blocks = (K + BLOCK - 1) / BLOCK;
  return q && s && dims_ok(n, K) && ld_ok(ldq, blocks * BLOCK) && ldq % 16 == 0 && aligned(q, 16) &&
         ld_ok(lds, blocks);
}

template <bool GLU>
static hipError_t act(const void* x, long ldx, void* q, long ldq, void* s, long lds, int n, int K,
                      hipStream_t stream) {
  if (!x || !rows_ok(q, ldq, s, lds, n, K) || !ld_ok(ldx, GLU ? 2L * K : K) || !aligned(x, 2))
    return hipErrorInvalidValue;
  const auto* X = static_cast<const __bf16*>(x);
  auto *Q = static_cast<uint8_t*>(q), *S = static_cast<uint8_t*>(s);
  const int pieces = (K + BLOCK - 1) / BLOCK * 4;
  const int threads = std::min((pieces + WAVE - 1) / WAVE * WAVE, 256);
  for (int r = 0; r < n; r += LAUNCH_ROWS) {
    const dim3 grid(std::min(n - r, LAUNCH_ROWS), (pieces + threads - 1) / threads);
    if (K >= 8)
      act_mx8_kernel<GLU, false><<<grid, dim3(threads), 0, stream>>>(X + r * ldx, ldx, Q + r * ldq, ldq, S + r * lds,
                                                                     lds, K);
    else
      act_mx8_kernel<GLU, true><<<grid, dim3(threads), 0, stream>>>(X + r * ldx, ldx, Q + r * ldq, ldq, S + r * lds,
                                                                    lds, K);
  }
  return hipGetLastError();
}

extern "C" hipError_t qe_quant_mx8(const void* x, long ldx, void* q, long ldq, void* s, long lds, int n, int K,
                                   hipStream_t stream) {
  return act<false>(x, ldx, q, ldq, s, lds, n, K, stream);
}

extern "C" hipError_t qe_swiglu_mx8(const void* gu, long ldg, void* q, long ldq, void* s, long lds, int n, int K,
                                    hipStream_t stream) {
  return act<true>(gu, ldg, q, ldq, s, lds, n, K, stream);
}

extern "C" hipError_t qe_rmsnorm1p_mx8(const void* x, long ldx, const void* delta, long ldd, const void* w,
                                       void* sum, long ldsum, void* q, long ldq, void* s, long lds, int n, int K,
                                       float eps, hipStream_t stream) {
  if (!x || !w || !rows_ok(q, ldq, s, lds, n, K) || !ld_ok(ldx, K) || !aligned(x, 2) || !aligned(w, 2) ||
      (delta != nullptr) != (sum != nullptr) ||
      (delta && (!ld_ok(ldd, K) || !ld_ok(ldsum, K) || !aligned(delta, 2) || !aligned(sum, 2))))
    return hipErrorInvalidValue;
  const auto *X = static_cast<const __bf16*>(x), *D = static_cast<const __bf16*>(delta),
             *W = static_cast<const __bf16*>(w);
  auto* Sum = static_cast<__bf16*>(sum);
  auto *Q = static_cast<uint8_t*>(q), *S = static_cast<uint8_t*>(s);
  const int pieces = (K + BLOCK - 1) / BLOCK * 4;
  const int C = pieces <= NORM_THREADS ? 1 : pieces <= 2 * NORM_THREADS ? 2 : 4;
  const int threads = std::min(((pieces + C - 1) / C + WAVE - 1) / WAVE * WAVE, NORM_THREADS);
  for (int r = 0; r < n; r += LAUNCH_ROWS) {
    const __bf16* d = D ? D + r * ldd : nullptr;
    __bf16* to = Sum ? Sum + r * ldsum : nullptr;
#define QE_NORM(...)                                                                                              \
  __VA_ARGS__<<<dim3(std::min(n - r, LAUNCH_ROWS)), dim3(threads), 0, stream>>>(X + r * ldx, ldx, d, ldd, W, to,  \
                                                                                ldsum, Q + r * ldq, ldq,          \
                                                                                S + r * lds, lds, K, eps)
    if (K < 8) QE_NORM(norm_mx8_kernel<1, true>);
    else if (C == 1) QE_NORM(norm_mx8_kernel<1, false>);
    else if (C == 2) QE_NORM(norm_mx8_kernel<2, false>);
    else if (pieces <= 4 * NORM_THREADS) QE_NORM(norm_mx8_kernel<4, false>);
    else QE_NORM(norm_mx8_wide_kernel);
  }
#undef QE_NORM
  return hipGetLastError();
}
