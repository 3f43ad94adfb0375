// The layer's projections with 8-bit operands: C = A B^T, A and B in e4m3 (OCP), one
// fp32 scale for each row of A and 128 columns and for each 128 x 128 block of B,
// fp32 accumulation, bf16 result.  (The reference's projections are bf16:
// nanovllm/layers/linear.py:56-75, :133-158.)
//
//   C[m][n] = sum over blocks kb of  sa[m][kb] sb[n / 128][kb]  *  sum over k in kb of A[m][k] B[n][k]
//
// A block's inner sum is one matrix-core product (16 x 16 x 128, its own
// accumulator 0); the scaled sum over the blocks is fp32 in the vector ALUs, one fma
// per value and block.  Rows of 128 values are 128 bytes, as the bf16 GEMM's rows of
// 64, so the LDS layout, the loads and the stores are its own (gemm_tile.h).  A lane's
// 32 values of an operand are granules lg and 4 + lg of its row: the order of the
// values inside of a product is free as long as both operands have the same.
#include "gemm_tile.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kFp8Threads = 256;

// 32 values of a row from its LDS granules lg and 4 + lg
struct Frag8 {
  i32x4_t lo, hi;
};
__device__ __forceinline__ gdn::f32x4_t mfma_fp8(const Frag8& a, const Frag8& b) {
  const i32x8_t x = __builtin_shufflevector(a.lo, a.hi, 0, 1, 2, 3, 4, 5, 6, 7);
  const i32x8_t y = __builtin_shufflevector(b.lo, b.hi, 0, 1, 2, 3, 4, 5, 6, 7);
  // (formats 0, 0: e4m3 both; no block scales of the instruction's own)
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, gdn::f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}

struct Fp8Scales {
  const float* a;  // [M, K / 128], strides a_row, a_grp
  int64_t a_row, a_grp;
  const float* b;  // [ceil(N / 128), K / 128], row stride b_row
  int64_t b_row;
};

// 64 x 64 tiles, 4 waves of 32 x 32, one LDS stage: the plain kernel.
__global__ __launch_bounds__(kFp8Threads) void gemm_fp8_kernel(const uint8_t* __restrict__ A, int64_t lda,
                                                               const uint8_t* __restrict__ B, int64_t ldb,
                                                               Fp8Scales sc, GemmOut out, int M, int N, int K) {
  __shared__ __align__(16) uint8_t st[128 * 128];
  const int mb_n = (M + 63) / 64;
  const int64_t L = gdn::xcd_remap(blockIdx.x, static_cast<int64_t>(mb_n) * ((N + 63) / 64));
  if (L < 0) return;
  const int m0 = 64 * static_cast<int>(L % mb_n), n0 = 64 * static_cast<int>(L / mb_n);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave >> 1, wn = wave & 1;
  const int lr = lane & 15, lg = lane >> 4;
  const __amdgpu_buffer_rsrc_t ra = rsrc_of(A), rb = rsrc_of(B);
  // the wave's 1 KiB blocks: A rows 8 wave .. and 32 + 8 wave .., the same of B
  int va[2], vb[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * i + 8 * wave + (lane >> 3);
    va[i] = static_cast<int>(min(m0 + r, M - 1) * lda + 16 * ((lane & 7) ^ ((r >> 1) & 7)));
    vb[i] = static_cast<int>(min(n0 + r, N - 1) * ldb + 16 * ((lane & 7) ^ (((r >> 1) & 1) | (((r >> 3) & 3) << 1))));
  }
  gdn::f32x4_t acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[i][t] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
  const float* sa[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) sa[i] = sc.a + min(m0 + 32 * wm + 16 * i + lr, M - 1) * sc.a_row;
  const float* sb = sc.b + n0 / 128 * sc.b_row;
  for (int kb = 0; kb < K / 128; ++kb) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      dma16(ra, st + (32 * i + 8 * wave) * 128, va[i], 128 * kb);
      dma16(rb, st + (64 + 32 * i + 8 * wave) * 128, vb[i], 128 * kb);
    }
    __syncthreads();
    Frag8 fa[2], fb[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 32 * wm + 16 * i + lr;
      fa[i].lo = *reinterpret_cast<const i32x4_t*>(st + sw_off(r, lg));
      fa[i].hi = *reinterpret_cast<const i32x4_t*>(st + sw_off(r, 4 + lg));
      const int c = 32 * wn + 8 * (lr >> 2) + 4 * i + (lr & 3);
      fb[i].lo = *reinterpret_cast<const i32x4_t*>(st + 64 * 128 + swb_off(c, lg));
      fb[i].hi = *reinterpret_cast<const i32x4_t*>(st + 64 * 128 + swb_off(c, 4 + lg));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float s = sa[i][kb * sc.a_grp] * sb[kb];
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const gdn::f32x4_t p = mfma_fp8(fb[t], fa[i]);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][t][e] = fmaf(p[e], s, acc[i][t][e]);
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
    gemm_store16(acc[i][0], acc[i][1], out, M, N, m0 + 32 * wm + 16 * i, n0 + 32 * wn, lane, GemmGates{}, nullptr);
}

int fp8_launch(const uint8_t* A, int64_t lda, const uint8_t* B, int64_t ldb, const Fp8Scales& sc, const GemmOut& out,
               int M, int N, int K, hipStream_t st) {
  const int64_t tiles = static_cast<int64_t>((M + 63) / 64) * ((N + 63) / 64);
  const dim3 grid(static_cast<unsigned>(gdn::kNumXcd * ((tiles + gdn::kNumXcd - 1) / gdn::kNumXcd)));
  gemm_fp8_kernel<<<grid, dim3(kFp8Threads), 0, st>>>(A, lda, B, ldb, sc, out, M, N, K);
  return gdn_launch_status();
}

}  // namespace

extern "C" int gdn_gemm_fp8(const uint8_t* A, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_grp,
                            const uint8_t* B, int64_t ldb, const float* sb, int64_t sb_row, int M, int N, int K,
                            int n_parts, uint16_t* const* C, const int64_t* ldc, const int* col_end, void* stream) {
  if (M < 0 || N < 0 || K < 0 || n_parts < 1 || n_parts > kMaxParts || !C || !ldc || !col_end)
    return GDN_ERR_INVALID_ARG;
  if (M == 0 || N == 0) return GDN_OK;
  if (!A || !B || !sa || !sb) return GDN_ERR_INVALID_ARG;
  // K in whole groups; 16-byte row pieces of A and B; 32-bit buffer offsets
  const int64_t kLimit = 1LL << 31;
  const int64_t groups = K / gdn::kFp8Group;
  if (K == 0 || K % gdn::kFp8Group || lda % 16 || ldb % 16 || lda < K || ldb < K ||
      reinterpret_cast<uintptr_t>(A) % 16 || reinterpret_cast<uintptr_t>(B) % 16 || M * lda >= kLimit ||
      N * ldb >= kLimit || sa_row < 0 || sa_grp < 0 || sb_row < groups ||
      4 * ((M - 1) * sa_row + (groups - 1) * sa_grp) >= kLimit ||
      4 * ((N + 127) / 128 * sb_row) >= kLimit)
    return GDN_ERR_INVALID_ARG;
  GemmOut out{};
  if (!parts_of(out, n_parts, C, ldc, col_end, N)) return GDN_ERR_INVALID_ARG;
  return fp8_launch(A, lda, B, ldb, Fp8Scales{sa, sa_row, sa_grp, sb, sb_row}, out, M, N, K,
                    static_cast<hipStream_t>(stream));
}
