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
//
// Rounding: the matrix cores add a block's 128 products after shifting them to the
// exponent of the largest, and what lies below 2^-13 of that one is lost (measured: two
// large products that cancel leave a third of 2^-13 of them whole and lose one of 2^-14).
// What a result is off by beyond its rounding, of the sum of its products' magnitudes (the
// largest of 64 x 1024 results): normal data 2^-17.2 for K = 128 and 2^-19.4 for 2048; with 2 %
// of the columns 30 times as loud 2^-13.8 and 2^-14.5; values spread over 2^14 2^-12.8 and 2^-15.1.
// bf16's half step is 2^-9 of the result, so that a result of which most cancels can lose more
// to the products than to its rounding.  The instruction with 32 products per sum loses the same
// (in each of its parts) and runs at half the rate (2.4 against 4.8 PFLOP/s from registers); the
// alternative is the bf16 GEMM.  Everything after a block's sum is fp32, and one rounding to bf16.
#include <algorithm>
#include <cstddef>
#include <utility>

#include "gemm_tile.h"
#include "lora_tile.h"
#include "quant_fp8.h"

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

// ---- 256 x 256 tiles, 8 waves in two alternating groups ----
// gemm_tn_pp_kernel of the bf16 GEMM with K-steps of 128: the same bytes per step, the
// same sections and waits, one product where it has two.  What is added per section:
// 64 fmas that scale the products' results into the sums (4 per product of 32 cycles,
// 16 cycles of the vector ALU beside them), 10 LDS reads and 8 multiplies for the
// scales.  A step's scales (256 of A's rows, 2 of B's column halves) come into LDS
// like its operands: one 4-byte load per lane and wave (waves 0 to 3 a quarter of the
// rows each, wave 4 + h the column half h), two steps ahead.  The section after the one
// that read a step's scales loads those of the step two later, so that two sections
// in a row issue 9 loads.  An odd step past the last one repeats it with scales of 0 (both: a row's
// may be infinite).
//
// 16384 x 12288 x 2048 363 us (2.27 PFLOP/s; the library's product with one scale for each
// operand 399), 8192^3 418 us (2.63 PFLOP/s; library 2.65), 17001 x 2048 x 2048 70-75 us.  Bound
// by power (the clock falls to 1.6-2.0 GHz), no LDS conflicts; for 17001 x 2048 by 536 tiles
// in rounds of 256.  The 12 spilled registers that a first form reloaded between tiles, each
// behind a wait for every load and store in flight, cost 385, 432 and 79 us.  Not kept:
// row-block groups of 2, 8 and 16 (4 is 1-3 % faster), non-temporal stores (slower), a tile's
// first sections that do not wait for the stores of the tile before (no faster).
constexpr int kPPThreads = 512;
constexpr int kWaitPP8 = 9 | (7 << 4);    // s_waitcnt vmcnt(9) lgkmcnt(0)
constexpr int kWaitQ8 = 10 | (7 << 4);    // s_waitcnt vmcnt(10) lgkmcnt(0)

__device__ __forceinline__ void dma4(__amdgpu_buffer_rsrc_t rsrc, void* lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 4, voff, soff, 0, 0);
}

// kOdd: K is an odd number of steps.
template <bool kOdd, bool kLora>
__global__ __launch_bounds__(kPPThreads, 2) void gemm_fp8_pp_kernel(const uint8_t* __restrict__ A, int64_t lda,
                                                                    const uint8_t* __restrict__ B, int64_t ldb,
                                                                    Fp8Scales sc, GemmOut out, int M, int N, int K,
                                                                    int whole, LoraArg<kLora>) {
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
  __shared__ std::conditional_t<kLora, LoraTiles, int> tiles_l;

  struct Args {  // the kernel's
    const uint8_t* A;
    int64_t lda;
    const uint8_t* B;
    int64_t ldb;
    Fp8Scales sc;
    GemmOut out;
    int M, N, K, whole;
    Lora lo;
  };
  constexpr int kLoraAt = static_cast<int>(offsetof(Args, lo));
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
  // the lane's number found anew: nothing that only a new tile's offsets or an epilogue needs
  // is kept in registers across the loop (a spilled one comes back behind a wait for every
  // load and store in flight)
  auto new_lane = []() {
    int zero = 0;
    asm volatile("" : "+v"(zero));
    return static_cast<int>(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero)));
  };
  // (all byte offsets are below 2^31)
  const int a_ld = static_cast<int>(lda), b_ld = static_cast<int>(ldb);
  const int a_row = static_cast<int>(sc.a_row) * 4, b_row = static_cast<int>(sc.b_row) * 4;
  int va[2][2], vb[2][2], vs;
  auto set_offsets = [&](int m0, int n0) {
    const int l = new_lane();
    const int ldrow = 8 * wave + (l >> 3);
    const int gcol_a = 16 * ((l & 7) ^ (((wave & 1) << 2) | (l >> 4)));
    const int gcol_b = 16 * ((l & 7) ^ (((wave & 3) << 1) | ((l >> 4) & 1)));
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        va[h][i] = min(m0 + 128 * h + 64 * i + ldrow, M - 1) * a_ld + gcol_a;
        vb[h][i] = min(n0 + 128 * h + 64 * i + ldrow, N - 1) * b_ld + gcol_b;
      }
    vs = wave < 4 ? min(m0 + 64 * wave + l, M - 1) * a_row : min(n0 / 128 + (wave & 1), (N - 1) / 128) * b_row;
  };
  auto dma = [&](const __amdgpu_buffer_rsrc_t& r, uint8_t* dst, const int (&v)[2], int kbyte) {
#pragma unroll
    for (int i = 0; i < 2; ++i) dma16(r, dst + (wave + 8 * i) * 1024, v[i], kbyte);
  };
  const int nk = K / 128;
  const int steps = (nk + 1) & ~1;
  if constexpr (kLora) __builtin_assume(steps >= 2);
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
  // a product of scales of step s, or 0 past the last one (a mask: of a choice the compiler makes two
  // bodies of the loop, and spills).  In an instance of its own: it costs 1 to 2 % (8192^3 423 us
  // for 413), and so does the even one without the choice of sb above (426 for 420).
  auto kept = [&](float v, int s) {
    return kOdd ? __uint_as_float(__float_as_uint(v) & static_cast<uint32_t>((s - nk) >> 31)) : v;
  };
  gdn::f32x4_t acc[2][2][4][2];  // [row half][column half][16-row tile][column tile]
  // (kLora, which is short of registers: in a scalar one)
  auto uniform = [](float v) {
    return kLora ? __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(v))) : v;
  };
  // one row half of A against both column halves of B, in step `at`; odd: which may be past the last
  auto prod = [&](gdn::f32x4_t (&c)[2][4][2], const Frag8 (&fa)[4], const Frag8 (&f0)[2], const Frag8 (&f1)[2],
                  const float (&s)[4], int at, auto odd) {
    float f[2][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int b = 0; b < 2; ++b) f[b][i] = odd.value ? kept(s[i] * uniform(sb[b]), at) : s[i] * uniform(sb[b]);
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
    __builtin_amdgcn_sched_group_barrier(0x002, kOdd && odd.value ? 16 : 8, 0);  // the scales
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
  constexpr std::true_type yes;
  constexpr std::false_type no;
  auto mem_end = [&]() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWaitPP8);
    half_barrier();
  };
  int L = xcd * per_xcd + slot;
  int n_whole = 0, n_quarters = 0;
  if constexpr (kLora) {
    lora_tiles(tiles_l, kernel_arg<Lora>(kLoraAt), M, N, xcd * per_xcd, xend, slot, stride, tile_of);
    n_whole = __builtin_amdgcn_readfirstlane(tiles_l.whole);
    if (n_whole) L = __builtin_amdgcn_readfirstlane(tiles_l.tile[0]);
  }
  if (kLora ? n_whole > 0 : L < xend) {
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
    // (kLora) the pairs of bf16 steps behind K, as in the bf16 GEMM: v's rows and the adapters' B in
    // A's and B's place, 64 values of a row in its 128 bytes
    LoraBase na(A), nb(B);
    int lora_lo = 0;        // bytes to the low parts in a row of v; 0: none in the second step
    bool lora_all = false;  // a step's second half has values
    LoraSteps lt{LoraTiles::kNone, 0, false};
    auto set_lora_offsets = [&](int e, int m, int n) {
      if constexpr (kLora) {
        const Lora lo = kernel_arg<Lora>(kLoraAt);
        lora_offsets(tiles_l, lo, lt, lora_pair(tiles_l, lo, lt, e, N, n), M, N, m, n, wave, new_lane(), va, vb, na, nb, lora_lo, lora_all);
      }
    };
    int at = 0;
    // one row half of v against both column halves of the adapter's B; of ranks up to 32 the first half
    // of a step
    auto prod_lora = [&](gdn::f32x4_t (&c)[2][4][2], const Frag8 (&fa)[4], const Frag8 (&f0)[2], const Frag8 (&f1)[2],
                         bool any) {
      if constexpr (kLora) {
        auto bits = [](const i32x4_t& v) { return __builtin_bit_cast(gdn::s16x8_t, v); };
        if (any) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              c[b][i][t] = gdn::mfma16x16x32(bits(b ? f1[t].lo : f0[t].lo), bits(fa[i].lo), c[b][i][t]);
        }
        if (any && lora_all) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int t = 0; t < 2; ++t)
                c[b][i][t] = gdn::mfma16x16x32(bits(b ? f1[t].hi : f0[t].hi), bits(fa[i].hi), c[b][i][t]);
        }
        half_barrier();
      }
    };
    __builtin_amdgcn_s_waitcnt(14 | (7 << 4));
    half_barrier();
    read_b(b00, fb0);
    mem_end();
    for (;;) {
      int Ln = L + stride;
      if constexpr (kLora) {
        lt = lora_steps(tiles_l, at);
        Ln = ++at < n_whole ? __builtin_amdgcn_readfirstlane(tiles_l.tile[at]) : xend;
      }
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
        if constexpr (kLora) dma(ra, a11, v1, ka);  // (here for two registers less)
        int s2 = s + 2;
        const bool lora_next = kLora && s2 == steps && lt.pairs;
        if (s2 == steps) {
          // the next loads are the next tile's first steps (past the last tile
          // they repeat this one's)
          if (lora_next) {
            set_lora_offsets(0, m0, n0);
          } else if (Ln < xend) {
            tile_of(Ln, m0, n0);
            set_offsets(m0, n0);
          }
          s2 = 0;
        }
        const int k2 = kbyte(s2), k3 = lora_next ? lora_lo : kbyte(s2 + 1), k3b = lora_next ? 0 : k3;
        __amdgpu_buffer_rsrc_t ra_n = ra, rb_n = rb;
        if constexpr (kLora) ra_n = na.rsrc(), rb_n = nb.rsrc();
        dma(rb_n, b00, vb[0], k2);
        if constexpr (!kLora) dma(ra, a11, v1, ka);
        read_a(a00, fa);
        read_b(b01, fb1);
        read_sc(sc0, s);
        mem_end();
        prod(acc[0], fa, fb0, fb1, sa[0], s, no);
        dma(ra_n, a00, va[0], k2);
        dma(rb_n, b01, vb[1], k2);
        dma_sc(sc0, s2);
        read_a(a01, fa);
        read_b(b10, fbn);
        mem_end();
        prod(acc[1], fa, fb0, fb1, sa[1], s, no);
        dma(rb_n, b10, vb[0], k3b);
        dma(ra_n, a01, va[1], k2);
        read_a(a10, fa);
        read_b(b11, fb1);
        read_sc(sc1, s + 1);
        mem_end();
        prod(acc[0], fa, fbn, fb1, sa[0], s + 1, yes);
        dma(ra_n, a10, va[0], k3);
        dma(rb_n, b11, vb[1], k3b);
        dma_sc(sc1, s2 + 1);
        read_a(a11, fa);
        read_b(b00, fb0);
        mem_end();
        prod(acc[1], fa, fbn, fb1, sa[1], s + 1, yes);
      }
      if constexpr (kLora) {
        // the adapters' pairs of steps, as the loop's; the next loads are the next pair's or tile's
        for (int e = 0; e < lt.pairs; ++e) {
          dma(na.rsrc(), a11, va[1], lora_lo);
          int k3a = kbyte(1), k3b = k3a;
          if (e + 1 < lt.pairs) {
            set_lora_offsets(e + 1, m0, n0);
            k3a = lora_lo;
            k3b = 0;
          } else if (Ln < xend) {
            tile_of(Ln, m0, n0);
            set_offsets(m0, n0);
            na = LoraBase(A);
            nb = LoraBase(B);
          } else {
            k3a = k3b = 0;
          }
          const __amdgpu_buffer_rsrc_t ra_n = na.rsrc(), rb_n = nb.rsrc();
          dma(rb_n, b00, vb[0], 0);
          read_a(a00, fa);
          read_b(b01, fb1);
          mem_end();
          prod_lora(acc[0], fa, fb0, fb1, true);
          dma(ra_n, a00, va[0], 0);
          dma(rb_n, b01, vb[1], 0);
          dma_sc(sc0, 0);
          read_a(a01, fa);
          if (lora_lo) read_b(b10, fbn);
          mem_end();
          prod_lora(acc[1], fa, fb0, fb1, true);
          dma(rb_n, b10, vb[0], k3b);
          dma(ra_n, a01, va[1], 0);
          if (lora_lo) {
            read_a(a10, fa);
            read_b(b11, fb1);
          }
          mem_end();
          prod_lora(acc[0], fa, fbn, fb1, lora_lo);
          dma(ra_n, a10, va[0], k3a);
          dma(rb_n, b11, vb[1], k3b);
          dma_sc(sc1, 1);
          if (lora_lo) read_a(a11, fa);
          read_b(b00, fb0);
          mem_end();
          prod_lora(acc[1], fa, fbn, fb1, lora_lo);
        }
        if (lt.part) {
          float bad = 0.0f;
#pragma unroll
          for (int a = 0; a < 2; ++a)
#pragma unroll
            for (int b = 0; b < 2; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                  for (int x = 0; x < 4; ++x) bad = fmaf(acc[a][b][i][t][x], 0.0f, bad);
          if (bad != 0.0f) tiles_l.again[at - 1] = 1;
        }
      }
      if (!wm) half_barrier();
      const int lane_e = new_lane();
      if constexpr (kLora)
        gemm_store_tile<true>(acc, kernel_arg<GemmOut>(offsetof(Args, out)), M, N, m0c, n0c, wm, wn, lane_e, GemmGates{},
                              nullptr);
      else
#pragma unroll
        for (int a = 0; a < 2; ++a)
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int b = 0; b < 2; ++b)
              gemm_store16<true>(acc[a][b][i][0], acc[a][b][i][1], out, M, N, m0c + 128 * a + 64 * wm + 16 * i,
                           n0c + 128 * b + 32 * wn, lane_e, GemmGates{}, nullptr);
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
  // (kLora) the quarters of the workgroup's own tiles first: ql of them, then q as without
  int ql = 0;
  if constexpr (kLora) n_quarters = lora_quarters(tiles_l);
  for (int q = xcd * q_xcd + slot; q < qend || (kLora && ql < n_quarters); q += stride) {
    int m0 = 0, n0 = 0;
    bool own = false;
    if constexpr (kLora) {
      own = ql < n_quarters;
      if (own) {
        q -= stride;
        tile_of(__builtin_amdgcn_readfirstlane(tiles_l.in_quarters[ql >> 2]), m0, n0);
        m0 += 128 * ((ql >> 1) & 1);
        n0 += 128 * (ql & 1);
        ++ql;
        if (m0 >= M || n0 >= N) continue;  // (the whole workgroup)
      }
    }
    if (own) {
      // (m0 and n0 are there)
    } else if (whole) {
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
        const float fg = kept(f[i] * g, s);
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
    if constexpr (kLora)
      lora_add<4>(kernel_arg<Lora>(kLoraAt), M, N, m0 + 64 * wm, n0 + 32 * wn, new_lane(),
                  [&](int i, int t) -> gdn::f32x4_t& { return c[i][t]; });
    const GemmOut out_q = kLora ? kernel_arg<GemmOut>(offsetof(Args, out)) : out;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      gemm_store16<true>(c[i][0], c[i][1], out_q, M, N, m0 + 64 * wm + 16 * i, n0 + 32 * wn, new_lane(), GemmGates{}, nullptr);
  }
  __builtin_amdgcn_s_waitcnt(0);
}

// ---- columns with a bf16 weight beside the 8-bit ones ----
// The layer's gate projections are a few columns whose weight stays in bf16, read with
// the same rows.  A launch of their own costs more than they do (64 columns of 2048: 5
// us), so the kernels that quantize the rows take them along: 16 rows x 16 columns per
// workgroup, K-steps of 64 or 128 dealt to its waves, two stages per wave, as in the ring.
struct Fp8Wide {
  const uint16_t* b;  // [n, K] bf16, row stride ldb; columns N .. N + n - 1 of the output
  int64_t ldb;
  int n;              // a multiple of 16; 0: none
};

// Bytes of a stage of one wave: 16 rows of KS values of each operand.
constexpr int wide_stage(int KS) { return 2 * 16 * 2 * KS; }

template <int NW, int KS>
__device__ __forceinline__ void wide_tile(const void* __restrict__ A, int64_t lda, const Fp8Wide& wide,
                                          const GemmOut& out, int M, int N, int K, int m0, int n0, uint8_t* st0,
                                          uint8_t* st1) {
  constexpr int kRow = 2 * KS, kGran = kRow / 16;  // bytes and 16-byte granules of a row
  constexpr int kLoads = 16 * kRow / 1024;         // of an operand's stage
  constexpr int kWait = 2 * kLoads | (7 << 4) | (15 << 8);  // all but the newest stage
  static_assert(2 * kLoads < 16, "vmcnt field");
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const __amdgpu_buffer_rsrc_t ra = rsrc_of(A), rb = rsrc_of(wide.b);
  int voff[2 * kLoads];
#pragma unroll
  for (int i = 0; i < kLoads; ++i) {
    // granule c of row r at slot c ^ (r % kGran)
    const int r = 1024 / kRow * i + lane / kGran, at = 16 * ((lane % kGran) ^ (r % kGran));
    voff[i] = static_cast<int>(min(m0 + r, M - 1) * lda * 2 + at);
    voff[kLoads + i] = static_cast<int>((n0 + r) * wide.ldb * 2 + at);
  }
  const int nk = K / KS;
  auto issue = [&](uint8_t* st, int step) {
    uint8_t* w = st + wave * wide_stage(KS);
    const int s = kRow * min(step, nk - 1);
#pragma unroll
    for (int i = 0; i < 2 * kLoads; ++i) dma16(i < kLoads ? ra : rb, w + i * 1024, voff[i], s);
  };
  gdn::f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  auto one = [&](uint8_t* st, int step) {
    const uint8_t* a = st + wave * wide_stage(KS) + lr * kRow;
    gdn::s16x8_t fa[KS / 32], fb[KS / 32];
#pragma unroll
    for (int c = 0; c < KS / 32; ++c) {
      const int at = 16 * ((4 * c + lg) ^ (lr % kGran));
      fa[c] = *reinterpret_cast<const gdn::s16x8_t*>(a + at);
      fb[c] = *reinterpret_cast<const gdn::s16x8_t*>(a + 16 * kRow + at);
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWaitLds);
    __builtin_amdgcn_sched_barrier(0);
    issue(st, step + 2 * NW);
#pragma unroll
    for (int c = 0; c < KS / 32; ++c) acc = gdn::mfma16x16x32(fb[c], fa[c], acc);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWait);
    __builtin_amdgcn_sched_barrier(0);
  };
  issue(st0, wave);
  issue(st1, wave + NW);
  __builtin_amdgcn_s_waitcnt(kWait);
  int s = wave;
  for (; s + NW < nk; s += 2 * NW) {
    one(st0, s);
    one(st1, s + NW);
  }
  if (s < nk) one(st0, s);
  __builtin_amdgcn_s_waitcnt(0);  // the repeated loads past the last step
  __syncthreads();
  gdn::f32x4_t* red = reinterpret_cast<gdn::f32x4_t*>(st0);
  red[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave) return;
  acc = red[lane];
#pragma unroll
  for (int w = 1; w < NW; ++w) acc += red[w * 64 + lane];
  // lane (lr, lg): row m0 + lr, columns N + n0 + 4 lg .. + 3, all of one part
  const int n = N + n0;
  int p = 0;
#pragma unroll
  for (int i = 0; i + 1 < kMaxParts; ++i) p += n >= out.end[i] ? 1 : 0;
  auto pick = [&](auto a0, auto a1, auto a2, auto a3) { return p == 0 ? a0 : p == 1 ? a1 : p == 2 ? a2 : a3; };
  if (m0 + lr >= M) return;
  uint16_t* c = pick(out.c[0], out.c[1], out.c[2], out.c[3]) +
                static_cast<int64_t>(m0 + lr) * pick(out.ld[0], out.ld[1], out.ld[2], out.ld[3]) + n -
                pick(0, out.end[0], out.end[1], out.end[2]) + 4 * lg;
  const uint2 v = make_uint2(gdn::f2bf2(acc[0], acc[1]), gdn::f2bf2(acc[2], acc[3]));
  if (pick(out.vec[0], out.vec[1], out.vec[2], out.vec[3])) {
    *reinterpret_cast<uint2*>(c) = v;
  } else {
    c[0] = static_cast<uint16_t>(v.x);
    c[1] = static_cast<uint16_t>(v.x >> 16);
    c[2] = static_cast<uint16_t>(v.y);
    c[3] = static_cast<uint16_t>(v.y >> 16);
  }
}

// Rows to e4m3 for the kernels that take them so, and the bf16 columns: the first `groups`
// workgroups 16 groups of 128 each, then 16 x 16 tiles.
__global__ __launch_bounds__(256) void quant_wide_kernel(const uint16_t* __restrict__ A, int64_t lda,
                                                         uint8_t* __restrict__ y, float* __restrict__ scale,
                                                         Fp8Wide wide, GemmOut out, int M, int N, int K, int groups) {
  __shared__ __align__(16) uint8_t st0[4 * wide_stage(128)];
  __shared__ __align__(16) uint8_t st1[4 * wide_stage(128)];
  if (static_cast<int>(blockIdx.x) < groups) {
    quant_group<false>(A, lda, y, K, scale, 1, M, M, K / gdn::kFp8Group,
                       static_cast<int64_t>(blockIdx.x) * 16 + threadIdx.x / 16, threadIdx.x % 16);
    return;
  }
  const int t = blockIdx.x - groups, mb_n = (M + 15) / 16;
  wide_tile<4, 128>(A, lda, wide, out, M, N, K, 16 * (t % mb_n), 16 * (t / mb_n), st0, st1);
}

// the larger of each pair of 16-bit halves
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  const u16x2_t x = __builtin_bit_cast(u16x2_t, a), y = __builtin_bit_cast(u16x2_t, b);
  return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
}

// The waves' partial sums, added in wave order, into C.  red: [wave][row tile][column
// tile][lane], free of loads and readers.
template <int MT, int NT, int NW, class Order = SameRow>
__device__ __forceinline__ void ring_store(const gdn::f32x4_t (&acc)[MT][NT][2], gdn::f32x4_t* red, const GemmOut& out,
                                           int M, int N, int m0, int n0, const Order& order = {}) {
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) red[(((wave * MT + i) * NT + j) * 2 + t) * 64 + lane] = acc[i][j][t];
  __syncthreads();
  for (int ij = wave; ij < MT * NT; ij += NW) {
    gdn::f32x4_t c0 = red[(ij * 2) * 64 + lane], c1 = red[(ij * 2 + 1) * 64 + lane];
#pragma unroll
    for (int w = 1; w < NW; ++w) {
      c0 += red[((w * MT * NT + ij) * 2) * 64 + lane];
      c1 += red[((w * MT * NT + ij) * 2 + 1) * 64 + lane];
    }
    gemm_store16<true>(c0, c1, out, M, N, m0 + 16 * (ij / NT), n0 + 32 * (ij % NT), lane, GemmGates{}, nullptr,
                       order);
  }
}

// ---- few rows: a load ring per wave ----
// As the bf16 GEMM's ring kernel: BM rows x BN columns of C per workgroup, the K-steps
// of 128 dealt to its NW waves in turn, each wave with NS stages of its own in LDS and
// no barrier in the loop; the partial sums are added through LDS in wave order.  What
// bounds it: the loads' latency times the bytes in flight.
//
// kQuant: A is bf16 and is brought to e4m3 here (gdn::fp8_scale, the bits of
// gdn_quantize_fp8), a lane's 32 values of a row in its registers and the largest
// magnitude over the four lanes that share the row: no launch of its own and nothing
// written.  Every workgroup repeats it for its rows, so it is for few of them (fewer still:
// gemm_fp8_rows_kernel).
template <int BM, int BN, int NW, int NS, bool kQuant, bool kLora>
__global__ __launch_bounds__(64 * NW) void gemm_fp8_ring_kernel(const void* __restrict__ A, int64_t lda,
                                                                const uint8_t* __restrict__ B, int64_t ldb,
                                                                Fp8Scales sc, GemmOut out, int M, int N, int K,
                                                                Fp8Wide wide, LoraArg<kLora> lo) {
  constexpr int MT = BM / 16, NT = BN / 32;
  constexpr int kARow = kQuant ? 256 : 128;               // bytes of a row of A in LDS
  constexpr int kABytes = BM * kARow, kBBytes = BN * 128;
  constexpr int kStage = kABytes + kBBytes + 256 * (kQuant ? 1 : 2);
  constexpr int kAPer = kABytes / 1024, kBPer = kBBytes / 1024;
  constexpr int kPer = kAPer + kBPer + (kQuant ? 1 : 2);  // loads of a stage
  constexpr int kVm = (NS - 1) * kPer;
  static_assert(kVm < 64 && NS >= 2 && NS <= 3, "vmcnt field");
  constexpr int kWait = (kVm & 15) | (7 << 4) | (15 << 8) | ((kVm >> 4) << 14);
  __shared__ __align__(16) uint8_t st0[NW * kStage];
  __shared__ __align__(16) uint8_t st1[NW * kStage];
  __shared__ __align__(16) uint8_t st2[NS > 2 ? NW * kStage : 16];
  static_assert(MT * NT * 2048 <= kStage, "the partial sums fit a stage");
  const int mb_n = (M + BM - 1) / BM, nb_n = (N + BN - 1) / BN;
  // the row blocks of a column block on one XCD, so that its L2 reads the weights once
  const int64_t L = gdn::xcd_remap(blockIdx.x, static_cast<int64_t>(mb_n) * (nb_n + (kQuant ? wide.n / 16 : 0)));
  if (L < 0) return;
  if constexpr (kQuant) {
    static_assert(BM == 16 && kStage >= wide_stage(128), "wide tiles in the ring's stages");
    if (L >= static_cast<int64_t>(mb_n) * nb_n) {
      const int t = static_cast<int>(L - static_cast<int64_t>(mb_n) * nb_n);
      wide_tile<NW, 128>(A, lda, wide, out, M, N, K, 16 * (t % mb_n), 16 * (t / mb_n), st0, st1);
      return;
    }
  }
  const int m0 = BM * static_cast<int>(L % mb_n), n0 = BN * static_cast<int>(L / mb_n);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const __amdgpu_buffer_rsrc_t ra = rsrc_of(A), rb = rsrc_of(B), rsa = rsrc_of(sc.a), rsb = rsrc_of(sc.b);
  int goff[kAPer + kBPer];
#pragma unroll
  for (int i = 0; i < kAPer; ++i) {
    if constexpr (kQuant) {
      // 4 rows of 256 bytes; granule c of row r at slot c ^ (r % 16)
      const int r = 4 * i + (lane >> 4);
      goff[i] = static_cast<int>(min(m0 + r, M - 1) * lda * 2 + 16 * ((lane & 15) ^ (r & 15)));
    } else {
      const int r = 8 * i + (lane >> 3);
      goff[i] = static_cast<int>(lora_row<kLora>(lo, m0 + r, M) * lda + 16 * ((lane & 7) ^ ((r >> 1) & 7)));
    }
  }
#pragma unroll
  for (int i = 0; i < kBPer; ++i) {
    const int r = 8 * i + (lane >> 3);
    goff[kAPer + i] = static_cast<int>(min(n0 + r, N - 1) * ldb +
                                       16 * ((lane & 7) ^ (((r >> 1) & 1) | (((r >> 3) & 3) << 1))));
  }
  const int va = kQuant ? 0 : static_cast<int>(lora_row<kLora>(lo, m0 + lane % BM, M) * sc.a_row * 4);
  const int vb = static_cast<int>(n0 / 128 * sc.b_row * 4);
  const int nk = K / 128;
  auto issue = [&](uint8_t* st, int step) {
    const int s = min(step, nk - 1);
    uint8_t* w = st + wave * kStage;
#pragma unroll
    for (int i = 0; i < kAPer; ++i) dma16(ra, w + i * 1024, goff[i], kARow * s);
#pragma unroll
    for (int i = 0; i < kBPer; ++i) dma16(rb, w + kABytes + i * 1024, goff[kAPer + i], 128 * s);
    dma4(rsb, w + kABytes + kBBytes, vb, 4 * s);
    if constexpr (!kQuant) dma4(rsa, w + kABytes + kBBytes + 256, va, static_cast<int>(sc.a_grp) * 4 * s);
  };
  gdn::f32x4_t acc[MT][NT][2];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) acc[i][j][t] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto one = [&](uint8_t* st, int step) {
    const uint8_t* a = st + wave * kStage;
    const uint8_t* b = a + kABytes;
    const float* p = reinterpret_cast<const float*>(b + kBBytes);
    Frag8 fa[MT], fb[NT][2];
    float f[MT];
    uint4 raw[kQuant ? MT : 1][4];
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const int r = 16 * i + lr;
      if constexpr (kQuant) {
#pragma unroll
        for (int c = 0; c < 4; ++c)  // granules 2 lg, 2 lg + 1, 8 + 2 lg, 9 + 2 lg
          raw[i][c] = *reinterpret_cast<const uint4*>(a + r * 256 + 16 * ((8 * (c >> 1) + 2 * lg + (c & 1)) ^ (r & 15)));
      } else {
        fa[i].lo = *reinterpret_cast<const i32x4_t*>(a + sw_off(r, lg));
        fa[i].hi = *reinterpret_cast<const i32x4_t*>(a + sw_off(r, 4 + lg));
        f[i] = p[64 + r];
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 8 * (lr >> 2) + 4 * t + (lr & 3);
        fb[j][t].lo = *reinterpret_cast<const i32x4_t*>(b + 4096 * j + swb_off(r, lg));
        fb[j][t].hi = *reinterpret_cast<const i32x4_t*>(b + 4096 * j + swb_off(r, 4 + lg));
      }
    const float sb = p[0];
    // the reads have returned before the stage is loaded again
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWaitLds);
    __builtin_amdgcn_sched_barrier(0);
    issue(st, step + NS * NW);
    if constexpr (kQuant) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        // the largest magnitude, two values at a time in 16-bit integers (bf16 magnitudes
        // are ordered as such), then as a float; one at a time where there is a NaN,
        // which sorts above infinity there and must not count
        float v[32];
        uint32_t top = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t w[4] = {raw[i][c].x, raw[i][c].y, raw[i][c].z, raw[i][c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            v[8 * c + 2 * e] = __uint_as_float(w[e] << 16);
            v[8 * c + 2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
            top = max2(top, w[e] & 0x7fff7fffu);
          }
        }
        float m = __uint_as_float(max(top & 0xffffu, top >> 16) << 16);
        if (__builtin_expect(m != m, 0)) {
          m = 0.0f;
#pragma unroll
          for (int e = 0; e < 32; ++e) m = fmaxf(m, fabsf(v[e]));
        }
        m = fmaxf(m, __shfl_xor(m, 16, 64));
        m = fmaxf(m, __shfl_xor(m, 32, 64));
        f[i] = gdn::fp8_scale(m);
        const float inv = 1.0f / f[i];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          fa[i].lo[e] = gdn::f2fp8x4(v[4 * e] * inv, v[4 * e + 1] * inv, v[4 * e + 2] * inv, v[4 * e + 3] * inv);
          fa[i].hi[e] = gdn::f2fp8x4(v[16 + 4 * e] * inv, v[17 + 4 * e] * inv, v[18 + 4 * e] * inv,
                                     v[19 + 4 * e] * inv);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const float s = f[i] * sb;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const gdn::f32x4_t r = mfma_fp8(fb[j][t], fa[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][t][e] = fmaf(r[e], s, acc[i][j][t][e]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWait);
    __builtin_amdgcn_sched_barrier(0);
  };
  issue(st0, wave);
  issue(st1, wave + NW);
  if constexpr (NS == 3) issue(st2, wave + 2 * NW);
  if constexpr (kLora) {
    int cb[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) cb[j] = n0 + 32 * j;
    lora_init<MT, NT>(lo, M, N, m0, cb, lane, wave, NW,
                        [&](int i, int j, int t) -> gdn::f32x4_t& { return acc[i][j][t]; });
  }
  __builtin_amdgcn_s_waitcnt(kWait);
  int s = wave;
  for (; s + (NS - 1) * NW < nk; s += NS * NW) {
    one(st0, s);
    one(st1, s + NW);
    if constexpr (NS == 3) one(st2, s + 2 * NW);
  }
  if (s < nk) one(st0, s);
  if (NS == 3 && s + NW < nk) one(st1, s + NW);
  // the repeated loads past the last step land before the stages are reused
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  ring_store<MT, NT, NW>(acc, reinterpret_cast<gdn::f32x4_t*>(st0), out, M, N, m0, n0,
                         LoraOrder<kLora, LoraArg<kLora>>{lo, M});
}

// v of the lane D places on, around each 16 lanes
template <int D>
__device__ __forceinline__ float row_ror(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x120 + D, 15, 15, false));
}

template <class F, int... I>
__device__ __forceinline__ void each(const F& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>{}), ...);
}

// ---- up to 8 bf16 rows ----
// The ring of 16 rows for R (4 or 8) of them that come in bf16.  A wave has at most S K-steps: it
// asks for its rows' values of all of them first, 8 per lane, then for as many stages of B as LDS
// holds, and quantizes while B is on its way, into LDS rows as the ring's loads would leave them:
// R S / 4 passes of 55 instructions, where the ring's own way takes 140 for each of S steps,
// whether its 16 rows are there or not, and between the waits.  1 x 12288 x 2048 5.2 us (ring 6.7,
// e4m3 rows 5.1), 8 rows 5.7 (6.7), 1 x 2048 x 4096 4.7 (7.0), 8 rows 5.9 (7.2); for 16 rows 7.5 and
// 8.2 (6.8, 7.2).  Those are with the weights in the last-level cache; from memory 1 x 12288 x 2048
// takes 7.8, 8 rows 8.1, 1 x 2048 x 4096 6.1, 8 rows 7.1.
template <int BN, int NW, int NS, int S, int R>
__global__ __launch_bounds__(64 * NW) void gemm_fp8_rows_kernel(const uint16_t* __restrict__ A, int64_t lda,
                                                                const uint8_t* __restrict__ B, int64_t ldb,
                                                                Fp8Scales sc, GemmOut out, int M, int N, int K,
                                                                Fp8Wide wide) {
  constexpr int NT = BN / 32;
  constexpr int kBBytes = BN * 128, kStage = kBBytes + 256;
  constexpr int kBPer = kBBytes / 1024, kPer = kBPer + 1;  // loads of a stage
  static_assert(NS <= 4 && NS <= S && (NS - 1) * kPer < 64, "stages, vmcnt field");
  static_assert(kStage >= wide_stage(64) && NT * 2048 <= kStage, "wide tiles and partial sums fit a stage");
  __shared__ __align__(16) uint8_t st0[NW * kStage];
  __shared__ __align__(16) uint8_t st1[NW * kStage];
  __shared__ __align__(16) uint8_t st2[NS > 2 ? NW * kStage : 16];
  __shared__ __align__(16) uint8_t st3[NS > 3 ? NW * kStage : 16];
  __shared__ __align__(16) uint8_t rows[NW * S * 2048];  // [wave][step] 16 rows of 128 bytes
  __shared__ float scales[NW * S * 16];
  const int mb_n = (M + 15) / 16, nb_n = (N + BN - 1) / BN;
  const int64_t L = gdn::xcd_remap(blockIdx.x, static_cast<int64_t>(mb_n) * (nb_n + wide.n / 16));
  if (L < 0) return;
  if (L >= static_cast<int64_t>(mb_n) * nb_n) {
    const int t = static_cast<int>(L - static_cast<int64_t>(mb_n) * nb_n);
    wide_tile<NW, 64>(A, lda, wide, out, M, N, K, 16 * (t % mb_n), 16 * (t / mb_n), st0, st1);
    return;
  }
  const int m0 = 16 * static_cast<int>(L % mb_n), n0 = BN * static_cast<int>(L / mb_n);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const __amdgpu_buffer_rsrc_t ra = rsrc_of(A), rb = rsrc_of(B), rsb = rsrc_of(sc.b);
  const int nk = K / 128;
  // pass p: the 8 values l of step g % S of row g / S, g = 4 p + lane / 16
  constexpr int P = R * S / 4;
  static_assert(R * S % 4 == 0, "whole passes");
  const int l = lane & 15;
  auto row_of = [&](int p) { return (4 * p + lg) / S; };
  auto step_of = [&](int p) { return (4 * p + lg) % S; };
  i32x4_t raw[P];
#pragma unroll
  for (int p = 0; p < P; ++p)
    raw[p] = __builtin_bit_cast(
        i32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                     ra, static_cast<int>(min(m0 + row_of(p), M - 1) * lda * 2) + 16 * l +
                             256 * min(wave + NW * step_of(p), nk - 1), 0, 0));
  gdn::keep_loads_here();
  int goff[kBPer];
#pragma unroll
  for (int i = 0; i < kBPer; ++i) {
    const int r = 8 * i + (lane >> 3);
    goff[i] = static_cast<int>(min(n0 + r, N - 1) * ldb + 16 * ((lane & 7) ^ (((r >> 1) & 1) | (((r >> 3) & 3) << 1))));
  }
  const int vb = static_cast<int>(n0 / 128 * sc.b_row * 4);
  auto issue = [&](uint8_t* st, int i) {
    const int s = min(wave + NW * i, nk - 1);
    uint8_t* w = st + wave * kStage;
#pragma unroll
    for (int k = 0; k < kBPer; ++k) dma16(rb, w + k * 1024, goff[k], 128 * s);
    dma4(rsb, w + kBBytes, vb, 4 * s);
  };
  uint8_t* const st[4] = {st0, st1, st2, st3};
#pragma unroll
  for (int i = 0; i < NS; ++i) issue(st[i], i);
  __builtin_amdgcn_sched_barrier(0);
  // each group's largest magnitude, two values at a time in 16-bit integers (bf16 magnitudes
  // are ordered as such), then as a float; one at a time where there is a NaN, which sorts
  // above infinity there and must not count
  auto lo = [&](int p, int w) { return __uint_as_float(static_cast<uint32_t>(raw[p][w]) << 16); };
  auto hi = [&](int p, int w) { return __uint_as_float(raw[p][w] & 0xffff0000u); };
  float f[P];
  bool nan = false;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    uint32_t top = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) top = max2(top, raw[p][w] & 0x7fff7fffu);
    f[p] = __uint_as_float(max(top & 0xffffu, top >> 16) << 16);
    nan |= f[p] != f[p];
  }
  if (__builtin_expect(__any(nan), 0)) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      f[p] = 0.0f;
#pragma unroll
      for (int w = 0; w < 4; ++w) f[p] = fmaxf(f[p], fmaxf(fabsf(lo(p, w)), fabsf(hi(p, w))));
    }
  }
  uint8_t* my_rows = rows + wave * S * 2048;
  float* my_scales = scales + wave * S * 16;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    float m = f[p];  // over the 16 lanes
    m = fmaxf(m, row_ror<8>(m));
    m = fmaxf(m, row_ror<4>(m));
    m = fmaxf(m, row_ror<2>(m));
    m = fmaxf(m, row_ror<1>(m));
    const float s = gdn::fp8_scale(m), inv = 1.0f / s;
    const int r = row_of(p), i = step_of(p);
    *reinterpret_cast<uint2*>(my_rows + i * 2048 + sw_off(r, l >> 1) + 8 * (l & 1)) =
        make_uint2(gdn::f2fp8x4(lo(p, 0) * inv, hi(p, 0) * inv, lo(p, 1) * inv, hi(p, 1) * inv),
                   gdn::f2fp8x4(lo(p, 2) * inv, hi(p, 2) * inv, lo(p, 3) * inv, hi(p, 3) * inv));
    if (l == 0) my_scales[i * 16 + r] = s;
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  gdn::f32x4_t acc[1][NT][2];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int t = 0; t < 2; ++t) acc[0][j][t] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
  auto step = [&](auto at) {
    constexpr int i = decltype(at)::value;
    // stages behind stage i that have been asked for
    constexpr int behind = (i + NS <= S ? NS : S - i) - 1, vm = behind * kPer;
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt((vm & 15) | (7 << 4) | (15 << 8) | ((vm >> 4) << 14));
    __builtin_amdgcn_sched_barrier(0);
    const uint8_t* b = st[i % NS] + wave * kStage;
    Frag8 fa, fb[NT][2];
    fa.lo = *reinterpret_cast<const i32x4_t*>(my_rows + i * 2048 + sw_off(lr, lg));
    fa.hi = *reinterpret_cast<const i32x4_t*>(my_rows + i * 2048 + sw_off(lr, 4 + lg));
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 8 * (lr >> 2) + 4 * t + (lr & 3);
        fb[j][t].lo = *reinterpret_cast<const i32x4_t*>(b + 4096 * j + swb_off(r, lg));
        fb[j][t].hi = *reinterpret_cast<const i32x4_t*>(b + 4096 * j + swb_off(r, 4 + lg));
      }
    const float sb = *reinterpret_cast<const float*>(b + kBBytes);
    if constexpr (i + NS < S) {
      // the reads have returned before the stage is loaded again
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kWaitLds);
      __builtin_amdgcn_sched_barrier(0);
      issue(st[i % NS], i + NS);
    }
    if (wave + NW * i < nk) {
      const float s = my_scales[i * 16 + lr] * sb;
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const gdn::f32x4_t r = mfma_fp8(fb[j][t], fa);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[0][j][t][e] = fmaf(r[e], s, acc[0][j][t][e]);
        }
    }
  };
  each(step, std::make_integer_sequence<int, S>{});
  __syncthreads();
  ring_store<1, NT, NW>(acc, reinterpret_cast<gdn::f32x4_t*>(st0), out, M, N, m0, n0);
}

// ---- 64-row tiles with a deeper load pipeline ----
// As the bf16 GEMM's deep kernel: 64 x BN tiles, NS stages as objects of their own, the
// loads of step s + NS - 1 at the start of step s, the barrier before it waiting for
// step s alone.  The scales of a step come with its operands (wave 0 the rows', the
// others B's: a load each).
//
// H = 2: two groups of four waves, each with stages of its own, take the first and the second
// half of the K-steps (kOdd: one past the last repeats it with scale 0), which puts twice the
// loads in flight where a CU has one tile; the second's sums
// are added to the first's through LDS.
template <int BN, int NS, int H, bool kOdd, bool kLora>
__global__ __launch_bounds__(kFp8Threads * H, 2) void gemm_fp8_deep_kernel(const uint8_t* __restrict__ A, int64_t lda,
                                                                       const uint8_t* __restrict__ B, int64_t ldb,
                                                                       Fp8Scales sc, GemmOut out, int M, int N,
                                                                       int K, LoraArg<kLora> lo) {
  static_assert(NS == 3 || NS == 4, "three or four stages");
  constexpr int BM = 64, NJ = BN / 64;  // column pairs of 32 per wave
  constexpr int kStage = (BM + BN) * 128 + 1024;
  constexpr int kAPer = BM / 32, kBPer = BN / 32, kPer = kAPer + kBPer + 1;
  constexpr int kVm = (NS - 2) * kPer;
  static_assert(kVm < 64, "vmcnt field");
  constexpr int kWait = (kVm & 15) | (7 << 4) | ((kVm >> 4) << 14);
  __shared__ __align__(16) uint8_t st0[H * kStage];
  __shared__ __align__(16) uint8_t st1[H * kStage];
  __shared__ __align__(16) uint8_t st2[H * kStage];
  __shared__ __align__(16) uint8_t st3[NS == 4 ? H * kStage : 16];

  const int mb_n = (M + BM - 1) / BM, nb_n = (N + BN - 1) / BN;
  const int64_t L = gdn::xcd_remap(blockIdx.x, static_cast<int64_t>(mb_n) * nb_n);
  if (L < 0) return;
  const int64_t per_group = static_cast<int64_t>(kGroupM8) * nb_n;
  const int64_t grp = L / per_group, in_grp = L % per_group;
  const int gm = static_cast<int>(min<int64_t>(kGroupM8, mb_n - grp * kGroupM8));
  const int m0 = BM * static_cast<int>(grp * kGroupM8 + in_grp % gm), n0 = BN * static_cast<int>(in_grp / gm);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6 & 3);
  const int half = H == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 8);
  const int wm = wave >> 1, wn = wave & 1;
  const int lr = lane & 15, lg = lane >> 4;
  const __amdgpu_buffer_rsrc_t ra = rsrc_of(A), rb = rsrc_of(B), rs = rsrc_of(wave == 0 ? sc.a : sc.b);
  int goff[kAPer + kBPer];
#pragma unroll
  for (int i = 0; i < kAPer + kBPer; ++i) {
    const int r = 8 * wave + 32 * (i < kAPer ? i : i - kAPer) + (lane >> 3);
    goff[i] = i < kAPer ? static_cast<int>(lora_row<kLora>(lo, m0 + r, M) * lda + 16 * ((lane & 7) ^ ((r >> 1) & 7)))
                        : static_cast<int>(min(n0 + r, N - 1) * ldb +
                                           16 * ((lane & 7) ^ (((r >> 1) & 1) | (((r >> 3) & 3) << 1))));
  }
  const int vs = wave == 0 ? static_cast<int>(lora_row<kLora>(lo, m0 + lane, M) * sc.a_row * 4)
                           : static_cast<int>(n0 / 128 * sc.b_row * 4);
  const int s_step = wave == 0 ? static_cast<int>(sc.a_grp) * 4 : 4;
  const int nk = K / 128, trips = (nk + H - 1) / H, first = half * trips;
  auto issue = [&](uint8_t* st, int step) {
    const int s = min(first + step, nk - 1);
    st += half * kStage;
#pragma unroll
    for (int i = 0; i < kAPer + kBPer; ++i)
      dma16(i < kAPer ? ra : rb, st + (i < kAPer ? 0 : BM * 128) + (wave + 4 * (i < kAPer ? i : i - kAPer)) * 1024,
            goff[i], 128 * s);
    dma4(rs, st + (BM + BN) * 128 + 256 * wave, vs, s_step * s);
  };
  gdn::f32x4_t acc[2][NJ][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) acc[i][j][t] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
  // step s from `cur`, the loads of step s + NS - 1 into `nxt` (the stage of step
  // s - 1, which every wave has finished reading at the barrier)
  auto one = [&](const uint8_t* cur, uint8_t* nxt, int step) {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_waitcnt(kWait);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    issue(nxt, step + NS - 1);
    __builtin_amdgcn_sched_barrier(0);
    cur += half * kStage;
    const uint8_t* b = cur + BM * 128;
    const float* p = reinterpret_cast<const float*>(cur + (BM + BN) * 128);
    Frag8 fa[2], fb[NJ][2];
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = 32 * wm + 16 * i + lr;
      fa[i].lo = *reinterpret_cast<const i32x4_t*>(cur + sw_off(r, lg));
      fa[i].hi = *reinterpret_cast<const i32x4_t*>(cur + sw_off(r, 4 + lg));
      f[i] = p[r];
    }
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int r = 32 * (NJ * wn + j) + 8 * (lr >> 2) + 4 * t + (lr & 3);
        fb[j][t].lo = *reinterpret_cast<const i32x4_t*>(b + swb_off(r, lg));
        fb[j][t].hi = *reinterpret_cast<const i32x4_t*>(b + swb_off(r, 4 + lg));
      }
    const float sb = p[64];
    const bool on = !kOdd || first + step < nk;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float s = on ? f[i] * sb : 0.0f;
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          const gdn::f32x4_t r = mfma_fp8(fb[j][t], fa[i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][t][e] = fmaf(r[e], s, acc[i][j][t][e]);
        }
    }
  };
  issue(st0, 0);
  issue(st1, 1);
  if constexpr (NS == 4) issue(st2, 2);
  if constexpr (kLora) {
    int cb[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) cb[j] = n0 + 32 * (NJ * wn + j);
    lora_init<2, NJ>(lo, M, N, m0 + 32 * wm, cb, lane, half, H,
                       [&](int i, int j, int t) -> gdn::f32x4_t& { return acc[i][j][t]; });
  }
  // (no exit inside a trip: the compiler's load counting would merge its states at the
  // loop head and wait there for loads that are meant to stay in flight)
  int s = 0;
  if constexpr (NS == 4) {
    for (; s + 3 < trips; s += 4) {
      one(st0, st3, s);
      one(st1, st0, s + 1);
      one(st2, st1, s + 2);
      one(st3, st2, s + 3);
    }
    if (s < trips) one(st0, st3, s);
    if (s + 1 < trips) one(st1, st0, s + 1);
    if (s + 2 < trips) one(st2, st1, s + 2);
  } else {
    for (; s + 2 < trips; s += 3) {
      one(st0, st2, s);
      one(st1, st0, s + 1);
      one(st2, st1, s + 2);
    }
    if (s < trips) one(st0, st2, s);
    if (s + 1 < trips) one(st1, st0, s + 1);
  }
  if constexpr (H == 2) {
    static_assert(4 * NJ * 4096 <= H * kStage, "the second half's sums fit a stage");
    __builtin_amdgcn_s_waitcnt(0);  // the repeated loads past the last step
    __syncthreads();
    gdn::f32x4_t* red = reinterpret_cast<gdn::f32x4_t*>(st0) + (threadIdx.x & 255);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (half) red[256 * ((i * NJ + j) * 2 + t)] = acc[i][j][t];
    __syncthreads();
    if (half) return;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) acc[i][j][t] += red[256 * ((i * NJ + j) * 2 + t)];
  }
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
      gemm_store16<true>(acc[i][j][0], acc[i][j][1], out, M, N, m0 + 32 * wm + 16 * i, n0 + 32 * (NJ * wn + j), lane,
                         GemmGates{}, nullptr, LoraOrder<kLora, LoraArg<kLora>>{lo, M});
  __builtin_amdgcn_s_waitcnt(0);  // the repeated loads past the last step
}

// The kernels (fp8_plan says which is taken); the last four take bf16 rows.  Those and
// the two that take the same calls' e4m3 rows deal K to as many waves, so that a call from
// bf16 rows has the bits of gdn_quantize_fp8 and a call from e4m3 ones.  (Four waves of
// three stages for kRing16x32: 1 x 2048 3.6 us against 3.8, 64 x 2048 x 4096 4.8 / 5.1.)
enum Fp8Kernel {
  kPP, kDeep64, kDeep128, kDeep64x2, kRing16x32, kRing16x64, kRing32x32, kRing64x32,
  kRingQ16x32, kRingQ16x64, kRows16x32, kRows16x64
};

// Times: one launch replayed from a graph, operands in the caches, K = 2048 unless
// said.
Fp8Kernel fp8_plan(int M, int N, int K, bool quant) {
  auto blocks = [&](int bm, int bn) { return static_cast<int64_t>((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  // Ring tiles with at most one workgroup per CU, the fewest rows first: 1 x 2048 3.8 us
  // (64 x 64 tiles 6.5, 128 x 128 blocks 11.6), 64 x 2048 4.0 (6.9), 128 x 2048 4.7
  // (7.0), 256 x 2048 6.4 (7.1), 64 x 8192 6.2 (7.1); 37 x 2048 x 4096 4.6 (10.8).  With
  // more workgroups the 64 x 64 tiles move fewer bytes: 64 x 12288 7.2 against 10.8-12.
  // One row block of wide outputs takes 64 columns: 1 x 12288 4.8 (32 columns 5.2, 64 x
  // 64 tiles 6.9), 1 x 16384 5.2 (5.6, 7.3); past one workgroup per CU 1 x 32768 14.3,
  // 64 x 64 tiles 12.4.
  if (quant && K <= 4096) {
    // A bf16 A's own launch takes 2.0 to 2.8 us; in the ring it takes 0.5 per K-step of a
    // wave (2048 columns: two of them for each of 8 waves): 64 x 2048 5.9 against 7.0 in
    // two launches, 37 x 2048 x 4096 7.4 against 7.8, 16 x 12288 6.9 against 7.7.  Longer
    // rows take more, and so do row blocks past one workgroup per CU (64 x 8192 17.5
    // against 8.6).
    // Up to 8 rows quantize ahead, in at most 8 passes per wave (see there; with 16: 8 x 12288
    // x 4096 12.3 against 11.7).
    // K past 4096, in the ring against two launches: 2048 columns lose (1 row x 5120 7.7 against 6.9, x
    // 8192 10.2 / 8.1; 16 rows 7.8 / 8.0, 10.4 / 9.0), 8192 and 12288 ones would gain up to a
    // tenth (1 x 8192 x 5120 10.4 / 10.9, 16 x 12288 x 8192 18.8 / 20.2): the limit is for all.
    if (blocks(16, 32) <= kCUs8) return M <= 8 ? kRows16x32 : kRingQ16x32;
    if (M <= 16 && blocks(16, 64) <= kCUs8) return M <= 4 || (M <= 8 && K <= 2048) ? kRows16x64 : kRingQ16x64;
  }
  if (blocks(16, 32) <= kCUs8) return kRing16x32;
  if (M <= 16 && blocks(16, 64) <= kCUs8) return kRing16x64;
  if (blocks(32, 32) <= kCUs8) return kRing32x32;
  if (blocks(64, 32) <= kCUs8) return kRing64x32;
  // At most one 64 x 64 tile per CU, in two halves of K: 512 x 2048 x 4096 9.8 us (whole 11.4),
  // 512 x 2048 7.0 (7.5), 128 x 8192 7.2 (7.7); 300 x 2048 x 512 4.8 (4.3).
  if (blocks(64, 64) <= kCUs8 && K >= 2048) return kDeep64x2;
  // Up to two 64 x 64 tiles per CU: 200 x 8192 8.5 us (64 x 128 tiles 10.4, 128 x 128
  // blocks 13.1), 1024 x 2048 9.0 (10.3, 13.2), 128 x 12288 8.6 (10.3, 13.3); with three
  // 256 x 12288 14.5 (12.4, 14.3).
  if (blocks(64, 64) <= 2 * kCUs8) return kDeep64;
  // Up to nearly four 64 x 128 tiles per CU: 400 x 12288 21.2 (pp 24.7), 700 x 8192 21.3
  // (24.6), 600 x 12288 26.1 (28.3), 1500 x 2048 13.1 (14.1), 900 x 8192 26.0 (25.4); then
  // the large tiles: 700 x 12288 31.7 against 28.4.
  if (blocks(64, 128) <= 15 * kCUs8 / 4) return kDeep128;
  return kPP;
}

// Rows up to which the quantizing launch takes the bf16 columns along (each 16 x 16 tile
// reads its rows again).
constexpr int kWideRows = 1024;

template <bool kWant, class T>
LoraArg<kWant> ring_arg(const T& lo) {
  if constexpr (kWant) return lo;
  else return {};
}

bool fp8_quantizes(Fp8Kernel k) { return k >= kRingQ16x32; }

// kLora: e4m3 rows.
template <bool kLora>
int fp8_launch(Fp8Kernel kernel, const void* A, int64_t lda, const uint8_t* B, int64_t ldb, const Fp8Scales& sc,
               const GemmOut& out, int M, int N, int K, const Fp8Wide& wide, const LoraArg<kLora>& lo, hipStream_t st) {
  auto blocks = [&](int bm, int bn) { return static_cast<int64_t>((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  auto grid = [](int64_t wgs) {
    return dim3(static_cast<unsigned>(gdn::kNumXcd * ((wgs + gdn::kNumXcd - 1) / gdn::kNumXcd)));
  };
  // (few rows in their adapters' order keep to the small tiles: 200 x 49152 x 2048, rank 64, all one adapter's 52 us
  // and in large tiles 39, 32 at random 97 and 352)
  if constexpr (kLora)
    if (kernel == kPP && (!lora_tiles_fit(blocks(256, 256)) || lo.order)) kernel = kDeep128;
  const uint8_t* A8 = static_cast<const uint8_t*>(A);
  const uint16_t* A16 = static_cast<const uint16_t*>(A);
  auto rows_grid = [&](int bn) { return grid(blocks(16, bn) + blocks(16, 1 << 30) * (wide.n / 16)); };
  switch (kernel) {
    case kPP: {
      // whole 256 x 256 tiles for full rounds of the CUs, the rest (up to half a round)
      // as quarters; less than half a round: all of it in 128 x 128 blocks
      const int64_t t256 = blocks(256, 256), rem = t256 % kCUs8;
      const int64_t whole = rem <= kCUs8 / 2 ? t256 - rem : t256;
      const int64_t wgs = std::min<int64_t>(kCUs8, whole ? std::max(whole, 4 * (t256 - whole)) : blocks(128, 128));
      auto pp = K / gdn::kFp8Group % 2 ? gemm_fp8_pp_kernel<true, kLora> : gemm_fp8_pp_kernel<false, kLora>;
      pp<<<grid(wgs), dim3(kPPThreads), 0, st>>>(A8, lda, B, ldb, sc, out, M, N, K, static_cast<int>(whole), lo);
      break;
    }
#define GDN_DEEP(BN, NS, H, odd)                                                                                        \
  gemm_fp8_deep_kernel<BN, NS, H, odd, kLora><<<grid(blocks(64, BN)), dim3(kFp8Threads * H), 0, st>>>(A8, lda, B, ldb,   \
                                                                                                      sc, out, M, N, K, \
                                                                                                      lo)
    case kDeep64: GDN_DEEP(64, 4, 1, false); break;
    case kDeep128: GDN_DEEP(128, 3, 1, false); break;
    case kDeep64x2: K / gdn::kFp8Group % 2 ? GDN_DEEP(64, 4, 2, true) : GDN_DEEP(64, 4, 2, false); break;
#undef GDN_DEEP
#define GDN_RING(name, BM, BN, NW, NS, Q)                                                                            \
  case name:                                                                                                         \
    gemm_fp8_ring_kernel<BM, BN, NW, NS, Q, kLora && !Q>                                                             \
        <<<Q ? rows_grid(BN) : grid(blocks(BM, BN)), dim3(64 * NW), 0, st>>>(A, lda, B, ldb, sc, out, M, N, K, wide,  \
                                                                             ring_arg<kLora && !Q>(lo));             \
    break
      GDN_RING(kRing16x32, 16, 32, 8, 2, false);
      GDN_RING(kRing16x64, 16, 64, 4, 3, false);
      GDN_RING(kRing32x32, 32, 32, 4, 3, false);
      GDN_RING(kRing64x32, 64, 32, 4, 3, false);
      GDN_RING(kRingQ16x32, 16, 32, 8, 2, true);
      GDN_RING(kRingQ16x64, 16, 64, 4, 2, true);
#undef GDN_RING
#define GDN_ROWS(BN, NW, NS, S, R)                                                                                  \
  gemm_fp8_rows_kernel<BN, NW, NS, S, R><<<rows_grid(BN), dim3(64 * NW), 0, st>>>(A16, lda, B, ldb, sc, out, M, N, K, \
                                                                                  wide)
    case kRows16x32:
      if (K <= 2048)
        M <= 4 ? GDN_ROWS(32, 8, 2, 2, 4) : GDN_ROWS(32, 8, 2, 2, 8);
      else
        M <= 4 ? GDN_ROWS(32, 8, 2, 4, 4) : GDN_ROWS(32, 8, 2, 4, 8);
      break;
    case kRows16x64:
      if (K <= 2048)
        M <= 4 ? GDN_ROWS(64, 4, 3, 4, 4) : GDN_ROWS(64, 4, 3, 4, 8);
      else
        GDN_ROWS(64, 4, 2, 8, 4);
      break;
#undef GDN_ROWS
  }
  return gdn_launch_status();
}

// K in whole groups; 16-byte row pieces of A and B; 32-bit buffer offsets.
bool fp8_operands_ok(const void* A, bool a_is_bf16, int64_t lda, int64_t sa_row, int64_t sa_grp, const uint8_t* B,
                     int64_t ldb, int64_t sb_row, int M, int N, int K) {
  const int64_t kLimit = 1LL << 31;
  const int64_t groups = K / gdn::kFp8Group;
  if (K == 0 || K % gdn::kFp8Group || lda % (a_is_bf16 ? 8 : 16) || ldb % 16 || lda < K || ldb < K ||
      reinterpret_cast<uintptr_t>(A) % 16 || reinterpret_cast<uintptr_t>(B) % 16 ||
      M * lda * (a_is_bf16 ? 2 : 1) >= kLimit || N * ldb >= kLimit || sb_row < groups ||
      4 * ((N + 127) / 128 * sb_row) >= kLimit)
    return false;
  return a_is_bf16 || (sa_row >= 0 && sa_grp >= 0 && 4 * ((M - 1) * sa_row + (groups - 1) * sa_grp) < kLimit);
}

}  // namespace

// x's rows in e4m3 and their scales, of a call from bf16 rows that no kernel above quantizes itself.
extern "C" int64_t gdn_gemm_fp8_workspace_size(int M, int N, int K, int a_is_bf16) {
  if (M < 0 || N < 0 || K < 0 || K % gdn::kFp8Group) return -1;
  if (!a_is_bf16 || M == 0 || N == 0 || K == 0 || fp8_quantizes(fp8_plan(M, N, K, true))) return 0;
  return static_cast<int64_t>(M) * K + static_cast<int64_t>(M) * (K / gdn::kFp8Group) * 4;
}

extern "C" int gdn_gemm_fp8(const void* A, int a_is_bf16, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_grp,
                            const uint8_t* B, int64_t ldb, const float* sb, int64_t sb_row, const uint16_t* B2,
                            int64_t ldb2, int N2, int M, int N, int K, int n_parts, uint16_t* const* C,
                            const int64_t* ldc, const int* col_end, void* workspace, int64_t workspace_bytes,
                            void* stream) {
  if (M < 0 || N < 0 || K < 0 || N2 < 0 || n_parts < 1 || n_parts > kMaxParts || !C || !ldc || !col_end)
    return GDN_ERR_INVALID_ARG;
  if (M == 0 || N == 0) return GDN_OK;
  if (!A || !B || !sb || (!a_is_bf16 && !sa)) return GDN_ERR_INVALID_ARG;
  if (!fp8_operands_ok(A, a_is_bf16 != 0, lda, sa_row, sa_grp, B, ldb, sb_row, M, N, K)) return GDN_ERR_INVALID_ARG;
  const int64_t kLimit = 1LL << 31, groups = K / gdn::kFp8Group;
  GemmOut out{};
  if (!parts_of(out, n_parts, C, ldc, col_end, N + N2, true)) return GDN_ERR_INVALID_ARG;
  int first = n_parts;  // the first part of the bf16 columns
  if (N2) {
    if (!B2 || !a_is_bf16 || N2 % 16 || N % 16 || ldb2 % 8 || ldb2 < K || reinterpret_cast<uintptr_t>(B2) % 16 ||
        N2 * ldb2 * 2 >= kLimit)
      return GDN_ERR_INVALID_ARG;
    first = 0;
    while (first < n_parts && col_end[first] < N) ++first;
    if (first == n_parts || col_end[first++] != N) return GDN_ERR_INVALID_ARG;  // a part ends at N
    for (int i = first; i < n_parts; ++i)  // (the bf16 GEMM's rows, which writes them where M is large)
      if (!part_ok(C[i], ldc[i], 0)) return GDN_ERR_INVALID_ARG;
  }
  const Fp8Kernel kernel = fp8_plan(M, N, K, a_is_bf16 != 0);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const Fp8Wide wide{B2, ldb2, N2};
  if (a_is_bf16 && !fp8_quantizes(kernel)) {
    if (workspace_bytes < gdn_gemm_fp8_workspace_size(M, N, K, 1) || !workspace ||
        reinterpret_cast<uintptr_t>(workspace) % 16)
      return GDN_ERR_INVALID_ARG;
    uint8_t* x8 = static_cast<uint8_t*>(workspace);
    float* scale = reinterpret_cast<float*>(x8 + static_cast<int64_t>(M) * K);
    int rc;
    if (N2 && M <= kWideRows) {
      const int64_t quant = (M * groups + 15) / 16;
      quant_wide_kernel<<<dim3(static_cast<unsigned>(quant + (M + 15) / 16 * (N2 / 16))), dim3(256), 0, st>>>(
          static_cast<const uint16_t*>(A), lda, x8, scale, wide, out, M, N, K, static_cast<int>(quant));
      rc = gdn_launch_status();
    } else {
      rc = gdn_quantize_fp8(A, 0, lda, x8, K, scale, 1, M, M, K, 1, stream);
      if (rc == GDN_OK && N2) {
        int ends[kMaxParts];
        for (int i = first; i < n_parts; ++i) ends[i - first] = col_end[i] - N;
        rc = gdn_gemm_bf16_cols(static_cast<const uint16_t*>(A), lda, B2, ldb2, M, N2, K, n_parts - first, C + first,
                                ldc + first, ends, nullptr, nullptr, nullptr, nullptr, 0, 0, 0, stream);
      }
    }
    if (rc != GDN_OK) return rc;
    A = x8;
    lda = K;
    sa = scale;
    sa_row = 1;
    sa_grp = M;
  }
  return fp8_launch<false>(kernel, A, lda, B, ldb, Fp8Scales{sa, sa_row, sa_grp, sb, sb_row}, out, M, N, K, wide,
                           NoLora{}, st);
}

extern "C" int gdn_gemm_fp8_lora(const uint8_t* A, int64_t lda, const float* sa, int64_t sa_row, int64_t sa_grp,
                                 const uint8_t* B, int64_t ldb, const float* sb, int64_t sb_row, int M, int N, int K,
                                 int n_parts, uint16_t* const* C, const int64_t* ldc, const int* col_end,
                                 const uint16_t* v, int64_t ldv, const int32_t* groups, const uint16_t* lb,
                                 int64_t lb_slot, const int32_t* ids, int slots, int rank, int slices, const int* slice_end, void* stream) {
  if (M < 0 || N < 0 || K < 0 || n_parts < 1 || n_parts > kMaxParts || !C || !ldc || !col_end)
    return GDN_ERR_INVALID_ARG;
  if (M == 0 || N == 0) return GDN_OK;
  if (!A || !B || !sb || !sa || !fp8_operands_ok(A, false, lda, sa_row, sa_grp, B, ldb, sb_row, M, N, K))
    return GDN_ERR_INVALID_ARG;
  GemmOut out{};
  if (!parts_of(out, n_parts, C, ldc, col_end, N, true)) return GDN_ERR_INVALID_ARG;
  Lora lo{};
  if (!lora_of(lo, v, ldv, groups, lb, lb_slot, ids, slots, rank, slices, slice_end, M, N)) return GDN_ERR_INVALID_ARG;
  if (slots == 0)
    return fp8_launch<false>(fp8_plan(M, N, K, false), A, lda, B, ldb, Fp8Scales{sa, sa_row, sa_grp, sb, sb_row}, out, M, N,
                             K, Fp8Wide{}, NoLora{}, static_cast<hipStream_t>(stream));
  return fp8_launch<true>(fp8_plan(M, N, K, false), A, lda, B, ldb, Fp8Scales{sa, sa_row, sa_grp, sb, sb_row}, out, M, N,
                          K, Fp8Wide{}, lo, static_cast<hipStream_t>(stream));
}
