// q/k RMSNorm1p + partial rotate-half RoPE of the new rows of a batch, k and v written to the pages of a
// paged KV cache (include/qe_paged.h). fp32 throughout, the angle in fp64, one rounding at the end.
//
// A half-wave holds one head of one row (lane L: dims 8L .. 8L+7, 16-byte accesses), a workgroup eight heads
// of a row. The cos / sin of the row's rd/2 frequencies, its most expensive step, are computed once per
// workgroup into LDS, one frequency per thread, while the head's row is on its way; the rotate-half partner
// goes through the half-wave's own LDS row. A call is a chain of latencies (position, page, row, sincos),
// not bytes: one row, 24 / 4 heads, 4.0 us in a graph, 2.7 of them the kernel; four rows of each of 64 sequences
// into fp8 pages (7.9 MB) 5.5 us.
#include "qe_device.hpp"
#include "qe_paged.h"

namespace qe {
namespace paged {

struct PrepCall {
  int R, Hq, Hkv, N, M, lp, rd, wpr;  // wpr: workgroups per row
  long ldp, ldt;
  float eps, k_inv, v_inv;
};

constexpr int HW = 32;       // lanes of a head
constexpr int UPW = HD / HW; // heads of a workgroup

// 8 consecutive values of a row; VEC: 16-byte aligned
template <bool VEC>
__device__ __forceinline__ u32x4_t load8(const __bf16* p) {
  if constexpr (VEC) return *reinterpret_cast<const u32x4_t*>(p);
  const uint16_t* s = reinterpret_cast<const uint16_t*>(p);
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (uint32_t)s[2 * i] | (uint32_t)s[2 * i + 1] << 16;
  return r;
}

template <bool FP8, bool VEC>
__global__ void __launch_bounds__(HD)
attn_prep_paged_kernel(const __bf16* __restrict__ qg, const __bf16* __restrict__ k,
                       const __bf16* __restrict__ v, const __bf16* __restrict__ qnw,
                       const __bf16* __restrict__ knw, const float* __restrict__ inv_freq,
                       const int* __restrict__ pos, __bf16* __restrict__ q_out, char* __restrict__ kp,
                       char* __restrict__ vp, const int* __restrict__ table, PrepCall a) {
  __shared__ __attribute__((aligned(16))) float xn_all[UPW][HD];
  __shared__ __attribute__((aligned(16))) float2 cst[HD / 2];
  const int tid = threadIdx.x, hw = tid / HW, L = tid & (HW - 1);
  const int row = blockIdx.x / a.wpr, b = row / a.R, t = row - b * a.R;
  const int p0 = pos[b];
  const int nh = a.Hq + a.Hkv, hb_raw = (blockIdx.x - row * a.wpr) * UPW + hw, hb = min(hb_raw, nh - 1);
  const bool is_q = hb < a.Hq;
  const int h = is_q ? hb : hb - a.Hq;
  const size_t at = (size_t)row * a.ldp;
  const u32x4_t xr = load8<VEC>(is_q ? qg + at + (size_t)h * 2 * HD + 8 * L : k + at + (size_t)h * HD + 8 * L);
  const u32x4_t vr = is_q ? u32x4_t{0u, 0u, 0u, 0u} : load8<VEC>(v + at + (size_t)h * HD + 8 * L);
  const u32x4_t wr = load8<VEC>((is_q ? qnw : knw) + 8 * L);
  const int half = a.rd >> 1;
  const float fr = tid < half ? inv_freq[tid] : 0.f;
  if (p0 < 0) return;  // an idle sequence (uniform)
  const long long p = (long long)p0 + t;
  int page = -1;
  if (!is_q && p >> a.lp < a.M) page = table[(size_t)b * a.ldt + (size_t)(p >> a.lp)];
  if (tid < half) {
    double sn, cs;
    sincos((double)p * (double)fr, &sn, &cs);
    cst[tid] = make_float2((float)cs, (float)sn);
  }
  float x[8], y[8];
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = lo_bf16(xr[i]);
    x[2 * i + 1] = hi_bf16(xr[i]);
    s += x[2 * i] * x[2 * i] + x[2 * i + 1] * x[2 * i + 1];
  }
  s = s + dpp<0xB1>(s);                // lane ^ 1
  s = s + dpp<0x4E>(s);                // lane ^ 2
  s = s + dpp<0x1B>(dpp<0x141>(s));    // lane ^ 4
  s = s + dpp<0x128>(s);               // lane ^ 8
  s = xor16_pair(s, true);
  const float inv = 1.0f / sqrtf(s / (float)HD + a.eps);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = x[2 * i] * inv * (1.0f + lo_bf16(wr[i]));
    x[2 * i + 1] = x[2 * i + 1] * inv * (1.0f + hi_bf16(wr[i]));
  }
  float* xn = xn_all[hw];
  *reinterpret_cast<f32x4_t*>(&xn[8 * L]) = f32x4_t{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f32x4_t*>(&xn[8 * L + 4]) = f32x4_t{x[4], x[5], x[6], x[7]};
  lds_barrier();  // the table; the half-wave's row
  if (hb_raw >= nh) return;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int c = 8 * L + i;
    y[i] = x[i];
    if (c < a.rd) {
      const bool lo = c < half;
      const float2 e = cst[lo ? c : c - half];
      const float rot = lo ? -xn[c + half] : xn[c - half];
      y[i] = x[i] * e.x + rot * e.y;
    }
  }
  u32x4_t yo;
#pragma unroll
  for (int i = 0; i < 4; ++i) yo[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
  if (is_q) {
    __bf16* o = q_out + ((size_t)row * a.Hq + h) * HD + 8 * L;
    if constexpr (VEC) {
      *reinterpret_cast<u32x4_t*>(o) = yo;
    } else {
      uint16_t* s = reinterpret_cast<uint16_t*>(o);
#pragma unroll
      for (int i = 0; i < 4; ++i) s[2 * i] = (uint16_t)yo[i], s[2 * i + 1] = (uint16_t)(yo[i] >> 16);
    }
  } else if ((unsigned)page < (unsigned)a.N) {
    const size_t dst = ((((size_t)page * a.Hkv + h) << a.lp) + (size_t)(p & ((1ll << a.lp) - 1))) * HD + 8 * L;
    if constexpr (FP8) {
      uint32_t kw[2] = {0u, 0u}, vw[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float vf = i & 1 ? hi_bf16(vr[i >> 1]) : lo_bf16(vr[i >> 1]);
        kw[i >> 2] |= (uint32_t)f32_to_fp8(y[i] * a.k_inv) << (8 * (i & 3));
        vw[i >> 2] |= (uint32_t)f32_to_fp8(vf * a.v_inv) << (8 * (i & 3));
      }
      *reinterpret_cast<uint2*>(kp + dst) = make_uint2(kw[0], kw[1]);
      *reinterpret_cast<uint2*>(vp + dst) = make_uint2(vw[0], vw[1]);
    } else {
      *reinterpret_cast<u32x4_t*>(kp + 2 * dst) = yo;
      *reinterpret_cast<u32x4_t*>(vp + 2 * dst) = vr;
    }
  }
}

template <bool FP8>
static hipError_t launch_prep(const void* qg, const void* k, const void* v, long ldp, const void* qnw,
                              const void* knw, const float* inv_freq, const int* pos, void* q_out,
                              void* kp, void* vp, const int* table, long ldt, int B, int R, int Hq,
                              int Hkv, int N, int P, int M, int rd, float eps, float k_inv, float v_inv,
                              hipStream_t stream) {
  const auto a16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  if (B < 1 || B > QE_PAGED_MAX_SEQS || R < 1 || (long)B * R > 65535 || Hq < 1 || Hkv < 1 || N < 1 ||
      P < 16 || P > 32768 || (P & (P - 1)) || M < 1 || (long)M * P > (1 << 23) - 64 || rd < 0 || rd > HD ||
      (rd & 1) || ldt < M || ldp < 1 || (long)Hq + Hkv > 16384 || !qg || !k || !v || !qnw || !knw ||
      !inv_freq || !pos || !q_out || !kp || !vp || !table || !a16(kp) || !a16(vp))
    return hipErrorInvalidValue;
  PrepCall a{};
  a.R = R, a.Hq = Hq, a.Hkv = Hkv, a.N = N, a.M = M, a.lp = __builtin_ctz((unsigned)P), a.rd = rd;
  a.wpr = (Hq + Hkv + UPW - 1) / UPW;
  a.ldp = ldp, a.ldt = ldt, a.eps = eps, a.k_inv = k_inv, a.v_inv = v_inv;
  const bool vec = a16(qg) && a16(k) && a16(v) && a16(qnw) && a16(knw) && a16(q_out) && ldp % 8 == 0;
  auto kern = vec ? attn_prep_paged_kernel<FP8, true> : attn_prep_paged_kernel<FP8, false>;
  kern<<<dim3((unsigned)(B * R * a.wpr)), dim3(HD), 0, stream>>>(
      static_cast<const __bf16*>(qg), static_cast<const __bf16*>(k), static_cast<const __bf16*>(v),
      static_cast<const __bf16*>(qnw), static_cast<const __bf16*>(knw), inv_freq, pos,
      static_cast<__bf16*>(q_out), static_cast<char*>(kp), static_cast<char*>(vp), table, a);
  return hipGetLastError();
}

}  // namespace paged
}  // namespace qe

using namespace qe;

extern "C" hipError_t qe_attn_prep_paged(const void* qg, const void* k, const void* v, long ldp,
                                         const void* qnw, const void* knw, const float* inv_freq,
                                         const int* pos, void* q_out, void* kp, void* vp,
                                         const int* table, long ldt, int B, int R, int Hq, int Hkv,
                                         int N, int P, int M, int rd, float eps, hipStream_t stream) {
  return paged::launch_prep<false>(qg, k, v, ldp, qnw, knw, inv_freq, pos, q_out, kp, vp, table, ldt, B, R,
                                   Hq, Hkv, N, P, M, rd, eps, 1.f, 1.f, stream);
}

extern "C" hipError_t qe_attn_prep_paged_fp8(const void* qg, const void* k, const void* v, long ldp,
                                             const void* qnw, const void* knw, const float* inv_freq,
                                             const int* pos, void* q_out, void* kp, void* vp,
                                             const int* table, long ldt, int B, int R, int Hq, int Hkv,
                                             int N, int P, int M, int rd, float eps, float k_scale,
                                             float v_scale, hipStream_t stream) {
  if (!kv_scale_ok(k_scale) || !kv_scale_ok(v_scale)) return hipErrorInvalidValue;
  return paged::launch_prep<true>(qg, k, v, ldp, qnw, knw, inv_freq, pos, q_out, kp, vp, table, ldt, B, R,
                                  Hq, Hkv, N, P, M, rd, eps, 1.f / k_scale, 1.f / v_scale, stream);
}
