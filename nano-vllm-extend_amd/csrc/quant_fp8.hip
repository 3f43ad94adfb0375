// bf16 or fp32 rows to e4m3 with one fp32 scale for each group of 128 columns of a
// row (activations), or of each 128 x 128 block (weights, once at load time).  The
// scale and the rounding: gdn::fp8_scale.  No counterpart in the reference, whose
// projections are bf16 (nanovllm/layers/linear.py:56-75, :133-158).
//
// Rows: 16 lanes per group, 8 values each; two bytes read and one written per value
// (and 4 / 128 of scale), nothing read twice: 16384 x 2048 19.6 us, 5.1 TB/s, a large
// copy's rate.  The scales go out with the caller's
// strides; the GEMM reads the scales of 64 consecutive rows at once, so its callers
// keep the rows of one group side by side.
#include "quant_fp8.h"

namespace {

template <bool kF32>
__global__ __launch_bounds__(256) void quant_rows_kernel(const void* __restrict__ x, int64_t sx,
                                                         uint8_t* __restrict__ y, int64_t sy,
                                                         float* __restrict__ scale, int64_t ss_row, int64_t ss_grp,
                                                         int64_t M, int G) {
  quant_group<kF32>(x, sx, y, sy, scale, ss_row, ss_grp, M, G, static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16,
                    threadIdx.x % 16);
}

// One workgroup per 128 x 128 block: 16 rows at a time, the largest magnitude of all
// of them first, then the values again.
template <bool kF32>
__global__ __launch_bounds__(256) void quant_blocks_kernel(const void* __restrict__ x, int64_t sx,
                                                           uint8_t* __restrict__ y, int64_t sy,
                                                           float* __restrict__ scale, int64_t ss_row, int64_t ss_grp,
                                                           int64_t M, int G) {
  __shared__ float part[4];
  const int g = static_cast<int>(blockIdx.x % G);
  const int64_t blk = blockIdx.x / G;
  const int c = g * gdn::kFp8Group + (threadIdx.x % 16) * 8;
  const int64_t r0 = blk * gdn::kFp8Group + threadIdx.x / 16;
  float v[8], m = 0.0f;
  for (int i = 0; i < gdn::kFp8Group; i += 16) {
    if (r0 + i >= M) break;
    load8<kF32>(x, (r0 + i) * sx + c, v);
    m = fmaxf(m, max8(v));
  }
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, 64));
  if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = m;
  __syncthreads();
  const float s = gdn::fp8_scale(fmaxf(fmaxf(part[0], part[1]), fmaxf(part[2], part[3])));
  const float inv = 1.0f / s;
  for (int i = 0; i < gdn::kFp8Group; i += 16) {
    if (r0 + i >= M) break;
    load8<kF32>(x, (r0 + i) * sx + c, v);
    *reinterpret_cast<uint2*>(y + (r0 + i) * sy + c) = pack8(v, inv);
  }
  if (threadIdx.x == 0) scale[blk * ss_row + g * ss_grp] = s;
}

}  // namespace

extern "C" int gdn_quantize_fp8(const void* x, int x_is_fp32, int64_t sx, uint8_t* y, int64_t sy, float* scale,
                                int64_t ss_row, int64_t ss_grp, int64_t M, int K, int rows_per_scale, void* stream) {
  if (M < 0 || K < 0 || K % gdn::kFp8Group || (rows_per_scale != 1 && rows_per_scale != gdn::kFp8Group))
    return GDN_ERR_INVALID_ARG;
  if (M == 0 || K == 0) return GDN_OK;
  // 16-byte reads and 8-byte writes of every row piece
  if (!x || !y || !scale || reinterpret_cast<uintptr_t>(x) % 16 || sx % (x_is_fp32 ? 4 : 8) || sx < K ||
      reinterpret_cast<uintptr_t>(y) % 8 || sy % 8 || sy < K || reinterpret_cast<uintptr_t>(scale) % 4)
    return GDN_ERR_INVALID_ARG;
  const int G = K / gdn::kFp8Group;
  const bool rows = rows_per_scale == 1;
  const int64_t blocks = rows ? (M * G + 15) / 16 : (M + gdn::kFp8Group - 1) / gdn::kFp8Group * G;
  if (blocks >= (1LL << 31)) return GDN_ERR_UNSUPPORTED;
  const dim3 grid(static_cast<unsigned>(blocks)), block(256);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (rows && x_is_fp32)
    quant_rows_kernel<true><<<grid, block, 0, st>>>(x, sx, y, sy, scale, ss_row, ss_grp, M, G);
  else if (rows)
    quant_rows_kernel<false><<<grid, block, 0, st>>>(x, sx, y, sy, scale, ss_row, ss_grp, M, G);
  else if (x_is_fp32)
    quant_blocks_kernel<true><<<grid, block, 0, st>>>(x, sx, y, sy, scale, ss_row, ss_grp, M, G);
  else
    quant_blocks_kernel<false><<<grid, block, 0, st>>>(x, sx, y, sy, scale, ss_row, ss_grp, M, G);
  return gdn_launch_status();
}
