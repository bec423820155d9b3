// The parts of the product of 8-bit rows and a 4-bit weight.
#pragma once
#include "qe_device.hpp"

namespace qe {
namespace mx {

// Many rows, in tiles (mx_gemm_tile.hip).
hipError_t gemm_tiles(const uint8_t* wq, const uint8_t* xq, long ldx, const uint8_t* xs, long lds, __bf16* out,
                      long ldo, int n, int N, int K, hipStream_t stream);

}  // namespace mx
}  // namespace qe
