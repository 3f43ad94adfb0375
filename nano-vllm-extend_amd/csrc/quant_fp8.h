// Values to e4m3 in groups of 128 (gdn::fp8_scale), 8 per lane: what the quantizer and the
// 8-bit GEMM's own quantizing launch share.
#pragma once

#include "gdn_common.h"

namespace {

// The 8 values of a lane, as fp32.
template <bool kF32>
__device__ __forceinline__ void load8(const void* p, int64_t at, float (&v)[8]) {
  if constexpr (kF32) {
    const float4 a = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    const float4 b = *reinterpret_cast<const float4*>(static_cast<const float*>(p) + at + 4);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 a = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p) + at);
    const uint16_t* s = reinterpret_cast<const uint16_t*>(&a);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = gdn::bf2f(s[i]);
  }
}

__device__ __forceinline__ float max8(const float (&v)[8]) {
  float m = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
  return m;
}

__device__ __forceinline__ uint2 pack8(const float (&v)[8], float inv) {
  return make_uint2(gdn::f2fp8x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                    gdn::f2fp8x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}

// Group `grp` (row grp / G, columns 128 (grp % G) ..) by 16 neighbouring lanes, 8 values
// each.
template <bool kF32>
__device__ __forceinline__ void quant_group(const void* __restrict__ x, int64_t sx, uint8_t* __restrict__ y, int64_t sy,
                                            float* __restrict__ scale, int64_t ss_row, int64_t ss_grp, int64_t M,
                                            int G, int64_t grp, int lane) {
  const int64_t row = grp / G;
  const int g = static_cast<int>(grp - row * G);
  if (row >= M) return;
  const int c = g * gdn::kFp8Group + lane * 8;
  float v[8];
  load8<kF32>(x, row * sx + c, v);
  float m = max8(v);
#pragma unroll
  for (int d = 8; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  const float s = gdn::fp8_scale(m);
  *reinterpret_cast<uint2*>(y + row * sy + c) = pack8(v, 1.0f / s);
  if (lane == 0) scale[row * ss_row + g * ss_grp] = s;
}

}  // namespace
