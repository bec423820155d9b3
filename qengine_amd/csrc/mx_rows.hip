// Rows in microscaled 8-bit floating point (E4M3 codes, a scale for 32 values): of a norm with the residual's
// addition, of SwiGLU, or of plain bf16 rows. The value is rounded once, from fp32 to its code.
//
// Vector forms give a lane 8 values (a 16-byte read, an 8-byte write), so a block is four neighbouring lanes and its
// largest magnitude two lane moves; scalar forms, for widths or strides that are no multiple of 8, give a lane
// one value and a block half a wave. Bound by memory, one row by the launch: SwiGLU of 2048 x 17408 36 us (4.9 TB/s, a
// large copy's rate), the norm of 2048 x 5120 14 us from the caches, 19 us from memory; of one row 2.7 us in a graph.
// The norm's arithmetic is fp32, as in the framework's other norms: a value that lies within a few 2^-24 of the border
// between two codes may get the other one (about 15 of 10.5 million). In 64 bits it would not, at 3.0 us for
// one row and 20.5 us for 2048.
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

// One value a lane, a block 32 lanes.
__device__ __forceinline__ void store1(float v, uint8_t* q, uint8_t* s, int k, bool live) {
  uint32_t top = magnitude(v);
#pragma unroll
  for (int o = 1; o < BLOCK; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
  const int code = scale8(top);
  if (!live) return;
  q[k] = code == 255 ? 0x7f : (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v * inverse(code), 0.f, 0, false) & 0xff);
  if ((k & 31) == 0) s[k >> 5] = (uint8_t)code;
}

// silu(g) * u: exp and the reciprocal are the instructions' (1 ulp each), about 2^-22 relative in all, far below
// the code's 2^-4.
__device__ __forceinline__ float swiglu(float g, float u) {
  return g * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * g)) * u;
}

// ------------------------------------------------------------------------------ SwiGLU, plain rows
template <bool GLU, bool VEC>
__global__ void __launch_bounds__(256)
act_mx8_kernel(const __bf16* __restrict__ x, long ldx, uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ s,
               long lds, int K) {
  const size_t r = blockIdx.x;
  const __bf16* xr = x + r * ldx;
  uint8_t *qr = q + r * ldq, *sr = s + r * lds;
  const int c = blockIdx.y * 256 + threadIdx.x, Kp = (K + BLOCK - 1) / BLOCK * BLOCK;
  if constexpr (VEC) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (c < K / 8) {
      unpack8(reinterpret_cast<const u32x4_t*>(xr)[c], v);
      if constexpr (GLU) {
        float u[8];
        unpack8(reinterpret_cast<const u32x4_t*>(xr + K)[c], u);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = swiglu(v[i], u[i]);
      }
    }
    store8(v, qr, sr, c, c < Kp / 8);
  } else {
    float v = 0.f;
    if (c < K) {
      v = bf16_to_f32(xr[c]);
      if constexpr (GLU) v = swiglu(v, bf16_to_f32(xr[K + c]));
    }
    store1(v, qr, sr, c, c < Kp);
  }
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

// A workgroup a row, C pieces of 8 values a thread, all in registers: piece c of thread t is t + c * threads.
template <int C>
__global__ void __launch_bounds__(NORM_THREADS)
norm_mx8_vec_kernel(const __bf16* __restrict__ x, long ldx, const __bf16* __restrict__ delta, long ldd,
                    const __bf16* __restrict__ w, __bf16* __restrict__ sum, long ldsum, uint8_t* __restrict__ q,
                    long ldq, uint8_t* __restrict__ s, long lds, int K, float eps) {
  __shared__ float red[NORM_THREADS / WAVE];
  const size_t r = blockIdx.x;
  const int K8 = K / 8, P8 = (K + BLOCK - 1) / BLOCK * 4;
  float v[C][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    if (c < K8) {
      unpack8(reinterpret_cast<const u32x4_t*>(x + r * ldx)[c], v[i]);
      if (delta) {
        float d[8];
        unpack8(reinterpret_cast<const u32x4_t*>(delta + r * ldd)[c], d);
        u32x4_t o;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          o[j] = pack_bf16x2(v[i][2 * j] + d[2 * j], v[i][2 * j + 1] + d[2 * j + 1]);
          v[i][2 * j] = lo_bf16(o[j]);
          v[i][2 * j + 1] = hi_bf16(o[j]);
        }
        reinterpret_cast<u32x4_t*>(sum + r * ldsum)[c] = o;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss += v[i][j] * v[i][j];
  }
  const float inv = 1.0f / sqrtf(sum_rows(ss, red) / (float)K + eps);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = threadIdx.x + i * blockDim.x;
    if (c < K8) {
      float g[8];
      unpack8(reinterpret_cast<const u32x4_t*>(w)[c], g);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (v[i][j] * inv) * (1.0f + g[j]);
    }
    store8(v[i], q + r * ldq, s + r * lds, c, c < P8);
  }
}

// Any width, stride and alignment: strided values, two passes over the row (the second reads what this thread read or
// wrote, so no other thread's write is involved).
__global__ void __launch_bounds__(NORM_THREADS)
norm_mx8_kernel(const __bf16* x, long ldx, const __bf16* delta, long ldd, const __bf16* __restrict__ w, __bf16* sum,
                long ldsum, uint8_t* __restrict__ q, long ldq, uint8_t* __restrict__ s, long lds, int K, float eps) {
  __shared__ float red[NORM_THREADS / WAVE];
  const size_t r = blockIdx.x;
  const int Kp = (K + BLOCK - 1) / BLOCK * BLOCK;
  float ss = 0.f;
  for (int c = threadIdx.x; c < K; c += blockDim.x) {
    float v = bf16_to_f32(x[r * ldx + c]);
    if (delta) {
      const __bf16 b = f32_to_bf16(v + bf16_to_f32(delta[r * ldd + c]));
      sum[r * ldsum + c] = b;
      v = bf16_to_f32(b);
    }
    ss += v * v;
  }
  const float inv = 1.0f / sqrtf(sum_rows(ss, red) / (float)K + eps);
  const __bf16* from = delta ? sum + r * ldsum : x + r * ldx;
  // whole waves enter: a block's lanes meet in store1
  for (int c = threadIdx.x; c - (int)(threadIdx.x & (WAVE - 1)) < Kp; c += blockDim.x) {
    const float v = c < K ? (bf16_to_f32(from[c]) * inv) * (1.0f + bf16_to_f32(w[c])) : 0.f;
    store1(v, q + r * ldq, s + r * lds, c, c < Kp);
  }
}

}  // namespace mx
}  // namespace qe

using namespace qe;
using namespace qe::mx;

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
  const int Kp = (K + BLOCK - 1) / BLOCK * BLOCK;
  if (K % 8 == 0 && ldx % 8 == 0 && aligned(x, 16))
    act_mx8_kernel<GLU, true><<<dim3(n, (Kp / 8 + 255) / 256), dim3(256), 0, stream>>>(X, ldx, Q, ldq, S, lds, K);
  else
    act_mx8_kernel<GLU, false><<<dim3(n, (Kp + 255) / 256), dim3(256), 0, stream>>>(X, ldx, Q, ldq, S, lds, K);
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
  const int P8 = (K + BLOCK - 1) / BLOCK * 4;
  const bool vec = K % 8 == 0 && ldx % 8 == 0 && aligned(x, 16) && aligned(w, 16) && P8 <= 4 * NORM_THREADS &&
                   (!delta || (ldd % 8 == 0 && ldsum % 8 == 0 && aligned(delta, 16) && aligned(sum, 16)));
#define QE_NORM(...) \
  __VA_ARGS__<<<dim3(n), dim3(threads), 0, stream>>>(X, ldx, D, ldd, W, Sum, ldsum, Q, ldq, S, lds, K, eps)
  if (vec) {
    const int C = P8 <= NORM_THREADS ? 1 : P8 <= 2 * NORM_THREADS ? 2 : 4;
    const int threads = ((P8 + C - 1) / C + WAVE - 1) / WAVE * WAVE;
    if (C == 1) QE_NORM(norm_mx8_vec_kernel<1>);
    else if (C == 2) QE_NORM(norm_mx8_vec_kernel<2>);
    else QE_NORM(norm_mx8_vec_kernel<4>);
  } else {
    const int threads = K >= NORM_THREADS ? NORM_THREADS : (K + WAVE - 1) / WAVE * WAVE;
    QE_NORM(norm_mx8_kernel);
  }
#undef QE_NORM
  return hipGetLastError();
}
