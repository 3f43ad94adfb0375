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
#include <algorithm>

#include "gemm_tile.h"

namespace {

typedef int i32x8_t __attribute__((ext_vector_type(8)));
typedef int i32x4_t __attribute__((ext_vector_type(4)));

constexpr int kFp8Threads = 256;
constexpr int kGroupM8 = 4;  // row blocks per tile group
constexpr int kCUs8 = gdn::kNumCu;

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

// ---- 256 x 256 tiles, 8 waves in two alternating groups ----
// gemm_tn_pp_kernel of the bf16 GEMM with K-steps of 128: the same bytes per step, the
// same sections and waits, one product where it has two.  What is added per section:
// 64 fmas that scale the products' results into the sums (4 per product of 32 cycles,
// 16 cycles of the vector ALU beside them), 10 LDS reads and 8 multiplies for the
// scales.  A step's scales (256 of A's rows, 2 of B's column halves) come into LDS
// like its operands: one 4-byte load per lane and wave (waves 0 to 3 a quarter of the
// rows each, wave 4 + h the column half h), two steps ahead.  The section after the one
// that read a step's scales loads those of the step two later, so that two sections
// in a row issue 9 loads.  An odd step past the last one repeats it with B's scale 0.
constexpr int kPPThreads = 512;
constexpr int kWaitPP8 = 9 | (7 << 4);    // s_waitcnt vmcnt(9) lgkmcnt(0)
constexpr int kWaitQ8 = 10 | (7 << 4);    // s_waitcnt vmcnt(10) lgkmcnt(0)

__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rsrc, void* lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 4, voff, soff, 0, 0);
}

__global__ __launch_bounds__(kPPThreads, 2) void gemm_fp8_pp_kernel(const uint8_t* __restrict__ A, int64_t lda,
                                                                    const uint8_t* __restrict__ B, int64_t ldb,
                                                                    Fp8Scales sc, GemmOut out, int M, int N, int K,
                                                                    int whole) {
  constexpr int kHalf = 128 * 128;  // bytes of a half tile
  __shared__ __align__(16) uint8_t a00[kHalf];
  __shared__ __align__(16) uint8_t a01[kHalf];
  __shared__ __align__(16) uint8_t a10[kHalf];
  __shared__ __align__(16) uint8_t a11[kHalf];
  __shared__ __align__(16) uint8_t b00[kHalf];
  __shared__ __align__(16) uint8_t b01[kHalf];
  __shared__ __align__(16) uint8_t b10[kHalf];
  __shared__ __align__(16) uint8_t b11[kHalf];
  // scales of a step: 256 rows, then 64 copies for each column half (and unused)
  __shared__ __align__(16) float sc0[512];
  __shared__ __align__(16) float sc1[512];
  __shared__ __align__(16) float sc2[512];
  __shared__ __align__(16) float sc3[512];

  const int mb_n = (M + 255) / 256, nb_n = (N + 255) / 256;
  const int xcd = blockIdx.x % gdn::kNumXcd, slot = blockIdx.x / gdn::kNumXcd, stride = gridDim.x / gdn::kNumXcd;
  const int tiles = mb_n * nb_n;
  const int per_xcd = (whole + gdn::kNumXcd - 1) / gdn::kNumXcd;
  const int xend = min((xcd + 1) * per_xcd, whole);

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wm = wave >> 2, wn = wave & 3;
  const int lr = lane & 15, lg = lane >> 4;

  auto tile_of = [&](int t, int& m0, int& n0) {
    const int per_group = kGroupM8 * nb_n;
    const int grp = t / per_group, in_grp = t % per_group;
    const int gm = min(kGroupM8, mb_n - grp * kGroupM8);
    m0 = 256 * (grp * kGroupM8 + in_grp % gm);
    n0 = 256 * (in_grp / gm);
  };
  const __amdgpu_buffer_rsrc_t ra = rsrc_of(A), rb = rsrc_of(B), rs = rsrc_of(wave < 4 ? sc.a : sc.b);
  const int s_step = wave < 4 ? static_cast<int>(sc.a_grp) * 4 : 4;
  const int ldrow = 8 * wave + (lane >> 3);
  const int gcol_a = 16 * ((lane & 7) ^ (((wave & 1) << 2) | (lane >> 4)));
  const int gcol_b = 16 * ((lane & 7) ^ (((wave & 3) << 1) | ((lane >> 4) & 1)));
  int va[2][2], vb[2][2], vs;
  auto set_offsets = [&](int m0, int n0) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        va[h][i] = static_cast<int>(min(m0 + 128 * h + 64 * i + ldrow, M - 1) * lda + gcol_a);
        vb[h][i] = static_cast<int>(min(n0 + 128 * h + 64 * i + ldrow, N - 1) * ldb + gcol_b);
      }
    vs = wave < 4 ? static_cast<int>(min(m0 + 64 * wave + lane, M - 1) * sc.a_row * 4)
                  : static_cast<int>(min(n0 / 128 + (wave & 1), (N - 1) / 128) * sc.b_row * 4);
  };
  auto dma = [&](const __amdgpu_buffer_rsrc_t& r, uint8_t* dst, const int (&v)[2], int kbyte) {
#pragma unroll
    for (int i = 0; i < 2; ++i) dma16(r, dst + (wave + 8 * i) * 1024, v[i], kbyte);
  };
  const int nk = K / 128;
  const int steps = (nk + 1) & ~1;
  auto kbyte = [&](int s) { return 128 * min(s, nk - 1); };
  auto dma_sc = [&](float* dst, int s) { dma4(rs, dst + 64 * wave, vs, s_step * min(s, nk - 1)); };
  auto read_a = [&](const uint8_t* h, Frag8 (&f)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      f[i].lo = *reinterpret_cast<const i32x4_t*>(h + sw_off(64 * wm + 16 * i + lr, lg));
      f[i].hi = *reinterpret_cast<const i32x4_t*>(h + sw_off(64 * wm + 16 * i + lr, 4 + lg));
    }
  };
  auto read_b = [&](const uint8_t* h, Frag8 (&f)[2]) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int r = 32 * wn + 8 * (lr >> 2) + 4 * t + (lr & 3);
      f[t].lo = *reinterpret_cast<const i32x4_t*>(h + swb_off(r, lg));
      f[t].hi = *reinterpret_cast<const i32x4_t*>(h + swb_off(r, 4 + lg));
    }
  };
  // the wave's scales of a step: of its rows (row half, 16-row tile), of the column halves
  float sa[2][4], sb[2];
  auto read_sc = [&](const float* p, int s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sa[h][i] = p[128 * h + 64 * wm + 16 * i + lr];
      sb[h] = s < nk ? p[256 + 64 * h] : 0.0f;
    }
  };
  gdn::f32x4_t acc[2][2][4][2];  // [row half][column half][16-row tile][column tile]
  // one row half of A against both column halves of B
  auto prod = [&](gdn::f32x4_t (&c)[2][4][2], const Frag8 (&fa)[4], const Frag8 (&f0)[2], const Frag8 (&f1)[2],
                  const float (&s)[4]) {
    float f[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b) f[b][i] = s[i] * sb[b];
    __builtin_amdgcn_s_setprio(1);
    // product j is scaled into its sum behind the issue of product j + 2, when its
    // result is there
    gdn::f32x4_t p[3];
#pragma unroll
    for (int j = 0; j < 18; ++j) {
      if (j < 16) p[j % 3] = mfma_fp8((j >> 1) & 1 ? f1[j & 1] : f0[j & 1], fa[j >> 2]);
      if (j >= 2) {
        const int d = j - 2, i = d >> 2, b = (d >> 1) & 1, t = d & 1;
#pragma unroll
        for (int e = 0; e < 4; ++e) c[b][i][t][e] = fmaf(p[d % 3][e], f[b][i], c[b][i][t][e]);
      }
    }
    __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // the scales
    __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
#pragma unroll
    for (int j = 2; j < 16; ++j) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);
    __builtin_amdgcn_s_setprio(0);
    half_barrier();
  };
  auto mem_end = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWaitPP8);
    half_barrier();
  };
  int L = xcd * per_xcd + slot;
  if (L < xend) {
    int m0, n0;
    tile_of(L, m0, n0);
    set_offsets(m0, n0);
    dma(rb, b00, vb[0], 0);
    dma_sc(sc0, 0);
    dma(ra, a00, va[0], 0);
    dma(rb, b01, vb[1], 0);
    dma(rb, b10, vb[0], kbyte(1));
    dma(ra, a01, va[1], 0);
    dma_sc(sc1, 1);
    dma(ra, a10, va[0], kbyte(1));
    dma(rb, b11, vb[1], kbyte(1));
    Frag8 fa[4], fb0[2], fb1[2], fbn[2];
    __builtin_amdgcn_s_waitcnt(14 | (7 << 4));
    half_barrier();
    read_b(b00, fb0);
    mem_end();
    for (;;) {
      const int Ln = L + stride;
      const int m0c = m0, n0c = n0;
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 2; ++t) acc[a][b][i][t] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
      if (wm) half_barrier();
      for (int s = 0; s < steps; s += 2) {
        const int ka = kbyte(s + 1);  // the current tile's
        const int v1[2] = {va[1][0], va[1][1]};
        int s2 = s + 2;
        if (s2 == steps) {
          // the next loads are the next tile's first steps (past the last tile
          // they repeat this one's)
          if (Ln < xend) {
            tile_of(Ln, m0, n0);
            set_offsets(m0, n0);
          }
          s2 = 0;
        }
        const int k2 = kbyte(s2), k3 = kbyte(s2 + 1);
        dma(rb, b00, vb[0], k2);
        dma(ra, a11, v1, ka);
        read_a(a00, fa);
        read_b(b01, fb1);
        read_sc(sc0, s);
        mem_end();
        prod(acc[0], fa, fb0, fb1, sa[0]);
        dma(ra, a00, va[0], k2);
        dma(rb, b01, vb[1], k2);
        dma_sc(sc0, s2);
        read_a(a01, fa);
        read_b(b10, fbn);
        mem_end();
        prod(acc[1], fa, fb0, fb1, sa[1]);
        dma(rb, b10, vb[0], k3);
        dma(ra, a01, va[1], k2);
        read_a(a10, fa);
        read_b(b11, fb1);
        read_sc(sc1, s + 1);
        mem_end();
        prod(acc[0], fa, fbn, fb1, sa[0]);
        dma(ra, a10, va[0], k3);
        dma(rb, b11, vb[1], k3);
        dma_sc(sc1, s2 + 1);
        read_a(a11, fa);
        read_b(b00, fb0);
        mem_end();
        prod(acc[1], fa, fbn, fb1, sa[1]);
      }
      if (!wm) half_barrier();
      // (the lane from an opaque copy, so that no address of the epilogue is
      // kept in registers across the loop)
      int tid_e = static_cast<int>(threadIdx.x);
      asm volatile("" : "+v"(tid_e));
#pragma unroll
      for (int a = 0; a < 2; ++a)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int b = 0; b < 2; ++b)
            gemm_store16(acc[a][b][i][0], acc[a][b][i][1], out, M, N, m0c + 128 * a + 64 * wm + 16 * i,
                         n0c + 128 * b + 32 * wn, tid_e & 63, GemmGates{}, nullptr);
      if (Ln >= xend) break;
      L = Ln;
    }
  }
  // The tiles after the whole ones as quarters of 128 x 128 (without whole tiles: the
  // 128 x 128 blocks of C in groups of as many rows), four steps in the LDS objects.
  const int mq_n = (M + 127) / 128, nq_n = (N + 127) / 128;
  const int nq = whole ? 4 * (tiles - whole) : mq_n * nq_n;
  const int q_xcd = (nq + gdn::kNumXcd - 1) / gdn::kNumXcd;
  const int qend = min((xcd + 1) * q_xcd, nq);
  for (int q = xcd * q_xcd + slot; q < qend; q += stride) {
    int m0, n0;
    if (whole) {
      tile_of(whole + (q >> 2), m0, n0);
      m0 += 128 * ((q >> 1) & 1);
      n0 += 128 * (q & 1);
      if (m0 >= M || n0 >= N) continue;  // (the whole workgroup)
    } else {
      const int per_group = 2 * kGroupM8 * nq_n;
      const int grp = q / per_group, in_grp = q % per_group;
      const int gm = min(2 * kGroupM8, mq_n - grp * 2 * kGroupM8);
      m0 = 128 * (grp * 2 * kGroupM8 + in_grp % gm);
      n0 = 128 * (in_grp / gm);
    }
    set_offsets(m0, n0);
    __builtin_amdgcn_s_waitcnt(7 << 4);  // loads into the stages, of a tile before
    half_barrier();
    auto load = [&](uint8_t* a, uint8_t* b, float* p, int step) {
      dma(ra, a, va[0], kbyte(step));
      dma(rb, b, vb[0], kbyte(step));
      dma_sc(p, step);
    };
    load(a00, b00, sc0, 0);
    load(a01, b01, sc1, 1);
    load(a10, b10, sc2, 2);
    gdn::f32x4_t c[4][2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int t = 0; t < 2; ++t) c[i][t] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
    Frag8 fa[4], fb[2];
    // step s from (a, b, p); the loads of step s + 3 into (an, bn, pn)
    auto step = [&](const uint8_t* a, const uint8_t* b, const float* p, uint8_t* an, uint8_t* bn, float* pn, int s) {
      load(an, bn, pn, s + 3);
      read_a(a, fa);
      read_b(b, fb);
      float f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) f[i] = p[64 * wm + 16 * i + lr];
      const float g = s < nk ? p[256] : 0.0f;
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kWaitQ8);
      half_barrier();
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float fg = f[i] * g;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const gdn::f32x4_t r = mfma_fp8(fb[t], fa[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) c[i][t][e] = fmaf(r[e], fg, c[i][t][e]);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      half_barrier();
    };
    __builtin_amdgcn_s_waitcnt(kWaitQ8);  // step 0
    half_barrier();
    if (wm) half_barrier();
    for (int s = 0; s < steps; s += 4) {
      step(a00, b00, sc0, a11, b11, sc3, s);
      step(a01, b01, sc1, a00, b00, sc0, s + 1);
      if (s + 2 >= steps) break;
      step(a10, b10, sc2, a01, b01, sc1, s + 2);
      step(a11, b11, sc3, a10, b10, sc2, s + 3);
    }
    if (!wm) half_barrier();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      gemm_store16(c[i][0], c[i][1], out, M, N, m0 + 64 * wm + 16 * i, n0 + 32 * wn, lane, GemmGates{}, nullptr);
  }
  __builtin_amdgcn_s_waitcnt(0);
}

int fp8_launch(const uint8_t* A, int64_t lda, const uint8_t* B, int64_t ldb, const Fp8Scales& sc, const GemmOut& out,
               int M, int N, int K, hipStream_t st) {
  const int64_t t256 = static_cast<int64_t>((M + 255) / 256) * ((N + 255) / 256);
  const int64_t t128 = static_cast<int64_t>((M + 127) / 128) * ((N + 127) / 128);
  const int64_t tiles = static_cast<int64_t>((M + 63) / 64) * ((N + 63) / 64);
  auto grid = [](int64_t wgs) {
    return dim3(static_cast<unsigned>(gdn::kNumXcd * ((wgs + gdn::kNumXcd - 1) / gdn::kNumXcd)));
  };
  if (tiles > kCUs8) {
    const int64_t rem = t256 % kCUs8;
    const int64_t whole = rem <= kCUs8 / 2 ? t256 - rem : t256;
    const int64_t wgs = std::min<int64_t>(kCUs8, whole ? std::max(whole, 4 * (t256 - whole)) : t128);
    gemm_fp8_pp_kernel<<<grid(wgs), dim3(kPPThreads), 0, st>>>(A, lda, B, ldb, sc, out, M, N, K,
                                                               static_cast<int>(whole));
    return gdn_launch_status();
  }
  gemm_fp8_kernel<<<grid(tiles), dim3(kFp8Threads), 0, st>>>(A, lda, B, ldb, sc, out, M, N, K);
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
