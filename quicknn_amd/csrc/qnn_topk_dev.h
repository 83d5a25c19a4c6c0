// qnn_topk_dev.h -- what token sampling (qnn_decode.hip), beam selection
// (qnn_beam.hip) and paged attention share: the bits of a score whose order as
// unsigned words is the scores' order, and a wave's largest word.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace qnn {
namespace dev {

// (-0 as +0.)
__device__ __forceinline__ uint32_t order_bits(float s) {
  const uint32_t u = __float_as_uint(s == 0.0f ? 0.0f : s);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// Wave-wide maximum of an unsigned word (all 64 lanes active), uniform
// result: row_shr 1, 2, 4, 8 leave each row's maximum in its lane 15,
// row_bcast 15 and 31 carry it to lane 63.  Lanes without a source read 0,
// the identity of the maximum.
__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x111, 0xf, 0xf, true)));  // row_shr:1
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x112, 0xf, 0xf, true)));  // row_shr:2
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x114, 0xf, 0xf, true)));  // row_shr:4
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x118, 0xf, 0xf, true)));  // row_shr:8
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x142, 0xa, 0xf, false)));  // row_bcast:15
  x = max(x, uint32_t(__builtin_amdgcn_update_dpp(0, int(x), 0x143, 0xc, 0xf, false)));  // row_bcast:31
  return uint32_t(__builtin_amdgcn_readlane(int(x), 63));
}

}  // namespace dev
}  // namespace qnn
