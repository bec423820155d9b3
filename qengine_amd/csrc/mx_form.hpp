// How a product of 8-bit rows and a 4-bit weight is run (host only): which kernels its choice takes, and a call of a
// given one, so that tests reach each of them at any size, whatever the choice's constants say.
#pragma once
#include <stddef.h>
#include <hip/hip_runtime_api.h>

namespace qe {
namespace mx {

// The arguments of qe_gemm_mx4.
struct GemmArgs {
  const void *wq, *xq;
  long ldx;
  const void* xs;
  long lds;
  void* out;
  long ldo;
  int n, N, K;
  void* ws;
  size_t ws_bytes;
};

// Kernels: -1 streams the weight (up to 16 rows always); 0 .. 2 the tiles of 256 x 256, 128 x 256 and 256 x 160; 3 ..
// 6 those of 64 x 128, 64 x 256, 32 x 128 (K in two) and 32 x 64 (K in four), which may split K further.
// `cut` weight rows go to the first, the others (none if cut is N) to the second.
struct Form {
  int kernel, splits, cut, rest_kernel, rest_splits;
};
Form gemm_form(int n, int N, int K, size_t ws_bytes);

// Whether a kernel takes a call in so many splits with so large a workspace, and that call (tests only).
bool gemm_form_ok(int kernel, int splits, int n, int N, int K, size_t ws_bytes);
hipError_t gemm_as(int kernel, int splits, const GemmArgs& a, hipStream_t stream);

}  // namespace mx
}  // namespace qe
