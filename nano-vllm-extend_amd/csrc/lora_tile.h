// What the projection GEMMs add for low-rank adapters: to a block of accumulators the products
// of the rows' shrunk values with their adapters' B.
//
// Row m has adapter s = ids[m] (none outside of 0 .. slots - 1); its columns are those of one or
// more slices (projections side by side), slice p with values of its own:
//   C[m][n] += sum over r of v[m][p][r] b[s][n][r],   v[m][p] = scale_s x[m] A_s^T  (lora.hip)
// v is held as the sum of two bf16 values (2^-16 of it is lost), the high parts of a slice's
// `rank` values, then the low ones: 2 rank values that meet b's rank ones twice, in K-steps of
// the matrix cores' depth; at rank 16 and less the low parts fill what is empty anyway.
#pragma once

#include <type_traits>

#include "gemm_tile.h"

namespace {

constexpr int kMaxRank = 256;

struct Lora {
  const uint16_t* v;    // [M, slices, 2, rank] bf16, row stride ldv
  int64_t ldv;
  const uint16_t* b;    // [slots][N, rank] bf16, slot stride b_slot
  int64_t b_slot;
  const int* ids;       // [M]
  int slots, rank, slices;
  int end[kMaxParts];   // slice p: columns end[p - 1] .. end[p] - 1; multiples of 16
};
struct NoLora {};
template <bool kLora>
using LoraArg = std::conditional_t<kLora, Lora, NoLora>;

// An offset past every buffer: the load gives 0.
constexpr int kNoOffset = static_cast<int>(0x80000000u);

__device__ __forceinline__ gdn::s16x8_t lora_load(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(gdn::s16x8_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t lora_b(const Lora& lo, int s, int N) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(lo.b + s * lo.b_slot), static_cast<short>(0),
                                           N * lo.rank * 2, 0x00020000);
}

// The adapters of a wave's rows, each once, in the rows' order: `mine` is the lane's row's, -1
// for none.  With `turns` waves that share the rows, wave `turn` takes every turns-th.
struct LoraIds {
  uint64_t todo;
  int turn, turns, at;
  // the next one, or -1 (wave-uniform)
  __device__ __forceinline__ int next(int mine) {
    while (todo) {
      const int s = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
      todo &= ~__ballot(mine == s);
      if (at++ % turns == turn) return s;
    }
    return -1;
  }
};

// RT tiles of 16 rows from row0 against CT blocks of 32 columns from cb[j]: at(i, j, t) is the
// accumulator of row tile i, block j and half t, C[row0 + 16 i + lr][cb[j] + 8 lg + 4 t ..
// + 3] in lane (lr, lg) (gemm_store16).  A row's sums take its own adapter's products only:
// what another one's give in its place (an infinity as well) is dropped.
template <int RT, int CT, int DEPTH, class At>
__device__ __forceinline__ void lora_add(const Lora& lo, int M, int N, int row0, const int (&cb)[CT], int lane, int turn,
                                         int turns, const At& at) {
  const int lr = lane & 15, lg = lane >> 4;
  int id[RT], voff[RT];
#pragma unroll
  for (int i = 0; i < RT; ++i) {
    const int r = row0 + 16 * i + lr, rc = min(r, M - 1);
    const int s = lo.ids[rc];
    id[i] = r < M && static_cast<unsigned>(s) < static_cast<unsigned>(lo.slots) ? s : -1;
    voff[i] = static_cast<int>(rc * lo.ldv * 2);
  }
  int mine = RT * 16 > lane ? id[0] : -1;  // row0 + lane's
#pragma unroll
  for (int i = 1; i < RT; ++i) mine = lg == i ? id[i] : mine;
  const uint64_t all = __ballot(mine >= 0);
  if (!all) return;
  const int half = lo.rank / 8, terms = 2 * half;  // granules of 8 values
  const int brow = 8 * (lr >> 2) + (lr & 3);
  for (int p = 0, beg = 0; p < lo.slices; beg = lo.end[p++]) {
    const int end = lo.end[p];
    bool in[CT], any = false, sel[CT];
#pragma unroll
    for (int j = 0; j < CT; ++j) {
      in[j] = cb[j] < end && cb[j] + 32 > beg && cb[j] < N;  // wave-uniform
      any |= in[j];
      sel[j] = cb[j] + 8 * lg >= beg && cb[j] + 8 * lg < end;
    }
    if (!any) continue;
    const __amdgpu_buffer_rsrc_t rv = rsrc_of(lo.v + 2 * p * lo.rank);
    for (int c = 0; c < terms; c += 4) {
      const int q = c + lg, qb = q < half ? q : q - half;
      gdn::s16x8_t va[RT];
#pragma unroll
      for (int i = 0; i < RT; ++i) va[i] = lora_load(rv, q < terms ? voff[i] + 16 * q : kNoOffset);
      int boff[CT][2];
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          boff[j][t] = q < terms ? (cb[j] + brow + 4 * t) * lo.rank * 2 + 16 * qb : kNoOffset;
      LoraIds it{all, turn, turns, 0};
      gdn::s16x8_t fb[DEPTH][CT][2];
      int sid[DEPTH];
      auto fetch = [&](int d) {
        sid[d] = it.next(mine);
        if (sid[d] < 0) return;
        const __amdgpu_buffer_rsrc_t rb = lora_b(lo, sid[d], N);
#pragma unroll
        for (int j = 0; j < CT; ++j)
#pragma unroll
          for (int t = 0; t < 2; ++t)
            if (in[j]) fb[d][j][t] = lora_load(rb, boff[j][t]);
      };
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) fetch(d);
      while (sid[0] >= 0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
          if (sid[d] < 0) continue;
#pragma unroll
          for (int j = 0; j < CT; ++j) {
            if (!in[j]) continue;
#pragma unroll
            for (int i = 0; i < RT; ++i) {
              const bool take = id[i] == sid[d] && sel[j];
#pragma unroll
              for (int t = 0; t < 2; ++t) {
                gdn::f32x4_t& acc = at(i, j, t);
                const gdn::f32x4_t sum = gdn::mfma16x16x32(fb[d][j][t], va[i], acc);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = take ? sum[e] : acc[e];
              }
            }
          }
          fetch(d);
        }
      }
    }
  }
}

// The arguments of the entry points, checked; slots == 0: no row has an adapter.
bool lora_of(Lora& lo, const uint16_t* v, int64_t ldv, const uint16_t* b, int64_t b_slot, const int* ids, int slots,
             int rank, int slices, const int* slice_end, int M, int N) {
  const int64_t kLimit = 1LL << 31;
  if (!ids || slots < 0 || rank < 8 || rank > kMaxRank || rank % 8 || slices < 1 || slices > kMaxParts || !slice_end)
    return false;
  if (slots && (!v || !b || reinterpret_cast<uintptr_t>(v) % 16 || reinterpret_cast<uintptr_t>(b) % 16)) return false;
  if (reinterpret_cast<uintptr_t>(ids) % 4 || ldv % 8 || ldv < 2LL * slices * rank || M * ldv * 2 >= kLimit ||
      b_slot % 8 || (slots > 1 && b_slot < static_cast<int64_t>(N) * rank) ||
      static_cast<int64_t>(N + 32) * rank * 2 >= kLimit)
    return false;
  lo = Lora{v, ldv, b, b_slot, ids, slots, rank, slices, {N, N, N, N}};
  for (int p = 0, beg = 0; p < slices; beg = slice_end[p++]) {
    const bool last = p + 1 == slices;
    if (slice_end[p] <= beg || (last ? slice_end[p] != N : slice_end[p] % 16 != 0 || slice_end[p] >= N)) return false;
    lo.end[p] = slice_end[p];
  }
  return true;
}

}  // namespace
