// What the bf16 and the 8-bit projection GEMMs share: the output's column parts and
// gate outputs, 128-byte LDS rows (swizzle, loads from global memory straight into
// them), the store of an accumulator block and the waits of the alternating waves.
#pragma once

#include "gdn_common.h"

namespace {

// The output: C's columns in up to four parts, part s holding columns
// [end[s - 1], end[s]) (end[-1] = 0) at c[s] with row stride ld[s]; vec[s]: its
// rows take 16-byte stores.  Every part boundary is a multiple of 16, so each
// 16-column half of a 32-column block (one store pair of every lane) lies in
// one part, and the part is the same for the whole wave.
constexpr int kMaxParts = 4;
struct GemmOut {
  uint16_t* c[kMaxParts];
  int64_t ld[kMaxParts];
  int end[kMaxParts];
  int vec[kMaxParts];
};

struct GemmGates {
  float* g;               // [M, Hv] fp32 (NULL: no gate outputs)
  uint16_t* beta;         // [M, Hv] bf16
  const void* A_log;      // [Hv], bf16 or fp32 (param_f32)
  const void* dt_bias;
  int param_f32;
  int gate_col;           // first b column of C
  int Hv;
};

// Byte offset of granule c (16 bytes) of row r in a 128-byte-row LDS tile.
// Granules are XOR-swizzled by (r / 2) % 8: a 16-byte read serves 16 lanes
// at a time from 256 bytes of banks (two rows), and the 16 lanes of a
// fragment read (16 consecutive rows, one granule) then hit 16 distinct
// 16-byte bank groups.
__device__ __forceinline__ int sw_off(int r, int c) { return r * 128 + ((c ^ ((r >> 1) & 7)) << 4); }

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc_of(const void* base) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0), 0x7fffffff, 0x00020000);
}

// Direct-to-LDS loads: one buffer_load_dwordx4 ... lds moves 64 lanes x 16
// bytes into the 1 KiB of LDS at M0 + 16 lane.  A stage holds the A tile (BM
// rows) then the B tile (256 rows), 128 bytes a row: 1 KiB block b is tile rows
// 8 b' .. 8 b' + 7 (b' = b for A, b - BM / 8 for B; BM / 8 is even).  Lane l
// fills row 8 b' + l / 8, slot l % 8, which under the swizzle holds the row's
// global granule (l % 8) ^ (4 (b % 2) + l / 16).  Wave w loads blocks w,
// w + 4, w + 8, ...
typedef __attribute__((address_space(3))) void* lds_ptr_t;

__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rsrc, uint8_t* lds, int voff, int soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (lds_ptr_t)lds, 16, voff, soff, 0, 0);
}

// ---- 16 rows x 32 columns of accumulators to the output (the 8-wave kernel) ----
// Lane (lr, lg) holds C[row0 + lr][cb + 8 lg .. + 7] in c0 (the first four) and
// c1: one 16-byte piece, four lanes filling 64 contiguous bytes of a row.  kAnyRow: the piece
// goes out whole in rows without 16-byte alignment too (the 8-bit GEMM's kernels: 8192 x
// 4001 x 256 36 us, value by value 77; 4002 columns 26).
template <bool kAnyRow = false>
__device__ __forceinline__ void gemm_store16(const gdn::f32x4_t& c0, const gdn::f32x4_t& c1, const GemmOut& out,
                                             int M, int N, int row0, int cb, int lane, const GemmGates& gt,
                                             uint16_t* gs) {
  const int lr = lane & 15, lg = lane >> 4;
  if (cb >= N || row0 >= M) return;  // wave-uniform
  auto pick = [](int t, auto a0, auto a1, auto a2, auto a3) { return t == 0 ? a0 : t == 1 ? a1 : t == 2 ? a2 : a3; };
  const uint4 w = make_uint4(gdn::f2bf2(c0[0], c0[1]), gdn::f2bf2(c0[2], c0[3]), gdn::f2bf2(c1[0], c1[1]),
                             gdn::f2bf2(c1[2], c1[3]));
  // the part of the block's first 16 columns (wave-uniform)
  const int s = cb < out.end[0] ? 0 : cb < out.end[1] ? 1 : cb < out.end[2] ? 2 : 3;
  const int cend = pick(s, out.end[0], out.end[1], out.end[2], out.end[3]);
  const int m = row0 + lr, n = cb + 8 * lg;
  if (pick(s, out.vec[0], out.vec[1], out.vec[2], out.vec[3]) && cb + 32 <= cend) {
    // the whole block in one part with 16-byte rows
    uint16_t* c = pick(s, out.c[0], out.c[1], out.c[2], out.c[3]) - pick(s, 0, out.end[0], out.end[1], out.end[2]);
    const int64_t ld = pick(s, out.ld[0], out.ld[1], out.ld[2], out.ld[3]);
    if (m < M) *reinterpret_cast<uint4*>(c + m * ld + n) = w;
  } else if (m < M) {
    // a part boundary inside the block, the last columns, or rows without
    // 16-byte alignment
    const int sp = n >= cend && cend < N ? s + 1 : s;
    const int pe = pick(sp, out.end[0], out.end[1], out.end[2], out.end[3]);
    const int pb = pick(sp, 0, out.end[0], out.end[1], out.end[2]);
    uint16_t* crow = pick(sp, out.c[0], out.c[1], out.c[2], out.c[3]) +
                     static_cast<int64_t>(m) * pick(sp, out.ld[0], out.ld[1], out.ld[2], out.ld[3]) - pb;
    if (kAnyRow && n + 8 <= pe) {
      __builtin_memcpy(crow + n, &w, 16);
    } else if (!kAnyRow && pick(sp, out.vec[0], out.vec[1], out.vec[2], out.vec[3]) && n + 8 <= pe) {
      *reinterpret_cast<uint4*>(crow + n) = w;
    } else {
      const uint32_t ww[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
      for (int t = 0; t < 8; ++t)
        if (n + t < pe) crow[n + t] = static_cast<uint16_t>(ww[t / 2] >> (16 * (t % 2)));
    }
  }
  // gate outputs from the bf16-rounded b and a columns of this block, through
  // the wave's own 1 KiB of LDS (see gemm_store)
  if (gt.g && cb + 32 > gt.gate_col && cb < gt.gate_col + 2 * gt.Hv) {
    *reinterpret_cast<uint4*>(gs + 32 * lr + 8 * lg) = w;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
#pragma unroll 1
    for (int e = lane; e < 16 * 32; e += 64) {
      const int r = e >> 5, c = e & 31;
      const int mm = row0 + r, nn = cb + c, col = nn - gt.gate_col;
      if (mm >= M || nn >= N || col < 0 || col >= 2 * gt.Hv) continue;
      const float v = gdn::bf2f(gs[32 * r + c]);
      if (col < gt.Hv) {
        gt.beta[static_cast<int64_t>(mm) * gt.Hv + col] = gdn::gate_beta(v);
      } else {
        const int h = col - gt.Hv;
        gt.g[static_cast<int64_t>(mm) * gt.Hv + h] =
            gdn::gate_g(v, gdn::load_param(gt.A_log, h, gt.param_f32), gdn::load_param(gt.dt_bias, h, gt.param_f32));
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
    __builtin_amdgcn_wave_barrier();
  }
}

__device__ __forceinline__ void half_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  asm volatile("" ::: "memory");
}

// s_waitcnt lgkmcnt(0) alone (vmcnt 63)
constexpr int kWaitLds = 15 | (7 << 4) | (3 << 14);

// LDS offset of granule c of row r in a half tile of B (see the column order
// below)
__device__ __forceinline__ int swb_off(int r, int c) {
  return r * 128 + ((c ^ (((r >> 1) & 1) | (((r >> 3) & 3) << 1))) << 4);
}

// One output part: rows of ld elements at c (16-byte stores when ld is a
// multiple of 8 and c 16-byte aligned, else element by element: c then only
// 2-byte aligned).
bool part_ok(const uint16_t* c, int64_t ld, int width) {
  return c && ld >= width && reinterpret_cast<uintptr_t>(c) % (ld % 8 ? 2 : 16) == 0;
}

// The n_parts (1 to kMaxParts) column parts of an output of N columns: increasing
// boundaries at multiples of 16, the last one at N.  any_row: rows of any alignment are taken
// (gemm_store16<true>), those with 16-byte stores among them.
bool parts_of(GemmOut& out, int n_parts, uint16_t* const* C, const int64_t* ldc, const int* col_end, int N,
              bool any_row = false) {
  int beg = 0;
  for (int s = 0; s < kMaxParts; ++s) {
    const int e = s < n_parts ? col_end[s] : N;
    if (s < n_parts) {
      if (e <= beg || (s + 1 < n_parts ? e % 16 != 0 || e >= N : e != N)) return false;
      const uintptr_t at = reinterpret_cast<uintptr_t>(C[s]);
      if (any_row ? !at || at % 2 || ldc[s] < e - beg : !part_ok(C[s], ldc[s], e - beg)) return false;
      out.c[s] = C[s];
      out.ld[s] = ldc[s];
      out.vec[s] = ldc[s] % 8 == 0 && at % 16 == 0;
    } else {
      out.c[s] = out.c[n_parts - 1];
      out.ld[s] = out.ld[n_parts - 1];
      out.vec[s] = out.vec[n_parts - 1];
    }
    out.end[s] = e;
    beg = e;
  }
  return true;
}

}  // namespace
