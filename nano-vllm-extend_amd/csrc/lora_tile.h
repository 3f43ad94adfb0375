// What the projection GEMMs add for low-rank adapters: the products of the rows' shrunk values
// with their adapters' B, in the accumulators before the projection's own.
//
// Row m has adapter s = ids[m] (none outside of 0 .. slots - 1); its columns are those of one or
// more slices (projections side by side), slice p with values of its own:
//   C[m][n] += sum over r of v[m][p][r] b[s][n][r],   v[m][p] = scale_s x[m] A_s^T  (lora.hip)
// v is held as the sum of two bf16 values (2^-16 of it is lost), the high parts of a slice's
// `rank` values, then the low ones, each of which meets the same value of b.
//
// A block of accumulators has up to 64 rows, and each adapter among them is multiplied with the
// tiles of 16 rows that have it, the others' values of v masked to 0.  That is right for finite
// numbers; where a result is not finite (an infinity times those zeros), all of the block is
// done again with the sums kept apart per row: a row never sees another one's adapter.
#pragma once

#include <algorithm>
#include <type_traits>

#include "gemm_tile.h"

namespace {

constexpr int kMaxRank = 256;
// Up to so many rows, and more than one tile's, are sorted by their adapters (lora.hip), and the kernels
// of few rows take them in that order: where lora_sorted is true the shrink writes it and the product reads it,
// whatever the columns of either.  200 rows of 32 adapters at random, 12352 columns of e4m3 x 2048, rank 32: 32 us,
// as they come 42.  (One tile's have nothing to gain: 1 row 16.0 us, sorted 17.3.  The counting grows
// with the square of the rows: 1.3 us for 256, 5 for 512.)
constexpr int kLoraSort = GDN_LORA_SORT;
__host__ __device__ constexpr bool lora_sorted(int M, int slots) {
  return M > 16 && M <= kLoraSort && slots < (1 << 23);  // (an adapter and a row in 32 bits)
}

struct Lora {
  const uint16_t* v;    // [M, slices, 2, rank] bf16, row stride ldv
  int64_t ldv;
  const uint16_t* b;    // [slots][N, rank] bf16, slot stride b_slot
  int64_t b_slot;
  const int* ids;       // [M]
  const int* groups;    // [ceil(M / 16)]: the adapter of 16 rows, -1 none, -2 not one for all (lora.hip)
  const int* order;     // lora_sorted: [M] the rows in the order of their adapters, [M] the adapters
  int slots, rank, slices;
  int end[kMaxParts];   // slice p: columns end[p - 1] .. end[p] - 1; multiples of 16
  int two;              // 256 x 256 tiles: two adapters to a pair of steps
};
struct NoLora {};
template <bool kLora>
using LoraArg = std::conditional_t<kLora, Lora, NoLora>;

// A pointer that is known to be one to global memory: by any other a store is a flat one, which
// the LDS reads behind it wait for as well (a tile's stores: 2.3 us of the next tile's products).
template <class T>
__device__ __forceinline__ void in_global(T*& p) {
  p = (T*)(__attribute__((address_space(1))) T*)reinterpret_cast<uintptr_t>(p);
}
__device__ __forceinline__ void in_global(GemmOut& o) {
#pragma unroll
  for (int i = 0; i < kMaxParts; ++i) in_global(o.c[i]);
}
__device__ __forceinline__ void in_global(GemmGates& g) {
  in_global(g.g);
  in_global(g.beta);
  in_global(g.A_log);
  in_global(g.dt_bias);
}
__device__ __forceinline__ void in_global(Lora& lo) {
  in_global(lo.v);
  in_global(lo.b);
  in_global(lo.ids);
  in_global(lo.groups);
  in_global(lo.order);
}

// A kernel's argument read from where the launch put it, `offset` bytes into its arguments: at the
// few places between tiles that need it, and not held in scalar registers across a loop that has
// none to spare (spilled ones made its loads late: 15 % of a large product).
template <class T>
__device__ __forceinline__ T kernel_arg(int offset) {
  typedef const __attribute__((address_space(4))) char* bytes_t;
  bytes_t p = (bytes_t)__builtin_amdgcn_kernarg_segment_ptr() + offset;
  asm volatile("" : "+s"(p));
  typedef const __attribute__((address_space(4))) uint32_t* words_t;
  static_assert(sizeof(T) % 4 == 0, "whole words");
  uint32_t w[sizeof(T) / 4];
#pragma unroll
  for (unsigned i = 0; i < sizeof(T) / 4; ++i) w[i] = ((words_t)p)[i];
  T value;
  __builtin_memcpy(&value, w, sizeof(T));
  in_global(value);
  return value;
}

// A buffer by its address, so that one of two can be chosen in scalar registers.
struct LoraBase {
  uint32_t lo, hi;
  __device__ __forceinline__ LoraBase() {}
  __device__ __forceinline__ explicit LoraBase(const void* p)
      : lo(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p))),
        hi(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(p) >> 32)) {}
  __device__ __forceinline__ __amdgpu_buffer_rsrc_t rsrc() const {
    return rsrc_of(reinterpret_cast<const void*>(
        static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(lo)))) |
        static_cast<uint64_t>(static_cast<uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(hi)))) << 32));
  }
};

// An offset past every buffer: the load gives 0.
constexpr int kNoOffset = static_cast<int>(0x80000000u);

__device__ __forceinline__ gdn::s16x8_t lora_load(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(gdn::s16x8_t, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0));
}

__device__ __forceinline__ __amdgpu_buffer_rsrc_t lora_b(const Lora& lo, int s, int N) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(lo.b + s * lo.b_slot), static_cast<short>(0),
                                           N * lo.rank * 2, 0x00020000);
}

__device__ __forceinline__ gdn::s16x8_t lora_mask(const gdn::s16x8_t& v, bool keep) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 w = __builtin_bit_cast(u32x4, v);
#pragma unroll
  for (int e = 0; e < 4; ++e) w[e] = keep ? w[e] : 0u;
  return __builtin_bit_cast(gdn::s16x8_t, w);
}

// The adapters of a wave's rows, each once, in the rows' order: `mine` is the lane's row's, -1
// for none.  With `turns` waves that share the rows, wave `turn` takes every turns-th adapter (by its
// number, and not by its place among the rows': which wave adds it shows in the result's last bits).
struct LoraIds {
  uint64_t todo;
  int turn, turns;
  // the next one and the lanes whose rows have it, or -1 (wave-uniform)
  __device__ __forceinline__ int next(int mine, uint64_t& rows) {
    while (todo) {
      const int s = __builtin_amdgcn_readlane(mine, __builtin_ctzll(todo));
      rows = __ballot(mine == s);
      todo &= ~rows;
      if (turns == 1 || s % turns == turn) return s;
    }
    rows = 0;
    return -1;
  }
};

// A row's adapter, -1 for none and for rows past M.
__device__ __forceinline__ int lora_id(const Lora& lo, int r, int M) {
  const int s = lo.ids[min(r, M - 1)];
  return r < M && static_cast<unsigned>(s) < static_cast<unsigned>(lo.slots) ? s : -1;
}

// What the kernels of few rows have as their r-th row, at most the last one: rows in the order of
// their adapters have few in a tile, and each is loaded and multiplied once there.
template <bool kOrder, class L>
__device__ __forceinline__ int lora_row(const L& lo, int r, int M) {
  r = min(r, M - 1);
  if constexpr (kOrder) r = lo.order ? lo.order[r] : r;
  return r;
}

template <bool kOrder, class L>
struct LoraOrder {
  const L& lo;
  int M;
  __device__ __forceinline__ int operator()(int r) const { return lora_row<kOrder>(lo, r, M); }
};

// One past the last column of slice p.
__device__ __forceinline__ int lora_end(const Lora& lo, int p) {
  return p == 0 ? lo.end[0] : p == 1 ? lo.end[1] : p == 2 ? lo.end[2] : lo.end[3];
}

// lora_init's products, CH times 32 values of the rank at once.  kSelect: the sums kept apart per row.
template <int RT, int CT, int DEPTH, int CH, bool kSelect, class At>
__device__ __forceinline__ void lora_pass(const Lora& lo, int N, const int (&id)[RT], int mine, uint64_t all,
                                          const int (&voff)[RT], const int (&cb)[CT], int lane, int turn, int turns,
                                          const At& at) {
  const int lr = lane & 15, lg = lane >> 4;
  const int half = lo.rank / 8;  // granules of 8 values
  const bool packed = half <= 2;  // high and low parts in one product
  const int brow = 8 * (lr >> 2) + (lr & 3);
  for (int p = 0, beg = 0, end = 0; p < lo.slices; ++p, beg = end) {
    end = lora_end(lo, p);
    bool in[CT], any = false, sel[CT];
#pragma unroll
    for (int j = 0; j < CT; ++j) {
      in[j] = cb[j] < end && cb[j] + 32 > beg && cb[j] < N;  // wave-uniform
      any |= in[j];
      sel[j] = cb[j] + 8 * lg >= beg && cb[j] + 8 * lg < end;
    }
    if (!any) continue;
    const __amdgpu_buffer_rsrc_t rv = rsrc_of(lo.v + 2 * p * lo.rank);
    for (int c0 = 0; c0 < half; c0 += 4 * CH) {
      gdn::s16x8_t vh[CH][RT], vl[CH][RT];
      int off[CH];
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        const int q = c0 + 4 * c + lg;
        off[c] = q < (packed ? 2 * half : half) ? 0 : kNoOffset;  // (or'ed: no branches)
#pragma unroll
        for (int i = 0; i < RT; ++i) vh[c][i] = lora_load(rv, (voff[i] + 16 * q) | off[c]);
        if (!packed) {
#pragma unroll
          for (int i = 0; i < RT; ++i) vl[c][i] = lora_load(rv, (voff[i] + 16 * (half + q)) | off[c]);
        }
      }
      const int q0 = c0 + lg, qb = packed && q0 >= half ? q0 - half : q0;
      int boff[CT][2];
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t)
          // (a column of another slice: 0, as its value of v is not this slice's)
          boff[j][t] = ((cb[j] + brow + 4 * t) * lo.rank * 2 + 16 * qb) |
                       (cb[j] + brow + 4 * t >= beg && cb[j] + brow + 4 * t < end ? 0 : kNoOffset);
      LoraIds it{all, turn, turns};
      gdn::s16x8_t fb[DEPTH][CH][CT][2];
      int sid[DEPTH];
      uint64_t rows[DEPTH];
      auto fetch = [&](int d) {
        sid[d] = it.next(mine, rows[d]);
        if (sid[d] < 0) return;
        const __amdgpu_buffer_rsrc_t rb = lora_b(lo, sid[d], N);
#pragma unroll
        for (int c = 0; c < CH; ++c)
#pragma unroll
          for (int j = 0; j < CT; ++j)
#pragma unroll
            for (int t = 0; t < 2; ++t)
              if (in[j]) fb[d][c][j][t] = lora_load(rb, (boff[j][t] + 64 * c) | (boff[j][t] & kNoOffset) | off[c]);
      };
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) fetch(d);
      while (sid[0] >= 0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
          if (sid[d] < 0) continue;
#pragma unroll
          for (int i = 0; i < RT; ++i) {
            if (!((rows[d] >> (16 * i)) & 0xffff)) continue;
            const bool own = id[i] == sid[d];
#pragma unroll
            for (int c = 0; c < CH; ++c) {
              if (c > 0 && c0 + 4 * c >= half) continue;
              const gdn::s16x8_t h = kSelect ? vh[c][i] : lora_mask(vh[c][i], own);
              gdn::s16x8_t l;
              if (!packed) l = kSelect ? vl[c][i] : lora_mask(vl[c][i], own);
#pragma unroll
              for (int j = 0; j < CT; ++j) {
                if (!in[j]) continue;
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                  gdn::f32x4_t& acc = at(i, j, t);
                  gdn::f32x4_t sum = gdn::mfma16x16x32(fb[d][c][j][t], h, acc);
                  if (!packed) sum = gdn::mfma16x16x32(fb[d][c][j][t], l, sum);
#pragma unroll
                  for (int e = 0; e < 4; ++e) acc[e] = !kSelect || (own && sel[j]) ? sum[e] : acc[e];
                }
              }
            }
          }
          fetch(d);
        }
      }
    }
  }
}

// The adapters of a lane's rows row0 + 16 i + lr and where their values are in v; `mine` is that of
// row0 + lane, `all` the lanes that have one.
template <int RT, bool kOrder>
struct LoraRows {
  int id[RT], voff[RT], mine;
  uint64_t all;
  __device__ __forceinline__ LoraRows(const Lora& lo, int M, int row0, int lane) {
    const int lr = lane & 15, lg = lane >> 4;
#pragma unroll
    for (int i = 0; i < RT; ++i) {
      const int r = row0 + 16 * i + lr;
      if (kOrder && lo.order)
        id[i] = r < M ? lo.order[M + r] : -1;
      else
        id[i] = lora_id(lo, r, M);
      voff[i] = static_cast<int>(lora_row<kOrder>(lo, r, M) * lo.ldv * 2);
    }
    mine = RT * 16 > lane ? id[0] : -1;
#pragma unroll
    for (int i = 1; i < RT; ++i) mine = lg == i ? id[i] : mine;
    all = __ballot(mine >= 0);
  }
};

// 64 rows from row0 against the 32 columns from cb, onto sums that are kept apart per row: at(i, t)
// as lora_init's at(i, 0, t).  A row's products in the order of the 256 x 256 tiles' steps: of each 64
// of the rank the high parts, then the low ones, of ranks up to 32 both one behind the other.
template <int DEPTH, class At>
__device__ __forceinline__ void lora_add(const Lora& lo, int M, int N, int row0, int cb, int lane, const At& at) {
  const LoraRows<4, false> r(lo, M, row0, lane);
  if (!r.all || cb >= N) return;
  const int lr = lane & 15, lg = lane >> 4, half = lo.rank / 8;
  const bool one = half <= 4;
  const int col = cb + 8 * (lr >> 2) + (lr & 3);
  for (int p = 0, beg = 0, end = 0; p < lo.slices; ++p, beg = end) {
    end = lora_end(lo, p);
    if (cb >= end || cb + 32 <= beg) continue;
    const bool sel = cb + 8 * lg >= beg && cb + 8 * lg < end;
    const __amdgpu_buffer_rsrc_t rv = rsrc_of(lo.v + 2 * p * lo.rank);
    for (int sub = 0; sub < (one ? (half + 1) / 2 : (half + 7) / 8 * 4); ++sub) {
      // granules q0 .. q0 + 3 of both parts, or of the high (or low) ones
      const int q0 = one ? 4 * sub : 8 * (sub >> 2) + 4 * (sub & 1), low = one ? 0 : (sub >> 1) & 1;
      if (!one && q0 >= half) continue;
      const int q = q0 + lg, off = q < (one ? 2 * half : half) ? 0 : kNoOffset;
      const int qb = one && q >= half ? q - half : q;
      gdn::s16x8_t v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = lora_load(rv, (r.voff[i] + 16 * (q + (low ? half : 0))) | off);
      LoraIds it{r.all, 0, 1};
      gdn::s16x8_t fb[DEPTH][2];
      int sid[DEPTH];
      uint64_t rows[DEPTH];
      auto fetch = [&](int d) {
        sid[d] = it.next(r.mine, rows[d]);
        if (sid[d] < 0) return;
        const __amdgpu_buffer_rsrc_t rb = lora_b(lo, sid[d], N);
#pragma unroll
        for (int t = 0; t < 2; ++t) fb[d][t] = lora_load(rb, ((col + 4 * t) * lo.rank * 2 + 16 * qb) | off);
      };
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) fetch(d);
      while (sid[0] >= 0) {
#pragma unroll
        for (int d = 0; d < DEPTH; ++d) {
          if (sid[d] < 0) continue;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (!((rows[d] >> (16 * i)) & 0xffff)) continue;
            const bool take = r.id[i] == sid[d] && sel;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
              gdn::f32x4_t& acc = at(i, t);
              const gdn::f32x4_t sum = gdn::mfma16x16x32(fb[d][t], v[i], acc);
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[e] = take ? sum[e] : acc[e];
            }
          }
          fetch(d);
        }
      }
    }
  }
}

// RT tiles of 16 rows from row0 against CT blocks of 32 columns from cb[j], into accumulators
// that are 0: at(i, j, t) is that of row tile i, block j and half t, C[row0 + 16 i + lr][cb[j] + 8
// lg + 4 t .. + 3] in lane (lr, lg) (gemm_store16).  B of the next adapters is on its way: of four,
// of ranks past 32 of two, 64 values of a row of B at once, which is its whole line.
template <int RT, int CT, class At>
__device__ __forceinline__ void lora_init(const Lora& lo, int M, int N, int row0, const int (&cb)[CT], int lane, int turn,
                                          int turns, const At& at) {
  const LoraRows<RT, true> r(lo, M, row0, lane);
  if (!r.all) return;
  if (lo.rank <= 32)
    lora_pass<RT, CT, 4, 1, false>(lo, N, r.id, r.mine, r.all, r.voff, cb, lane, turn, turns, at);
  else
    lora_pass<RT, CT, 2, 2, false>(lo, N, r.id, r.mine, r.all, r.voff, cb, lane, turn, turns, at);
  float bad = 0.0f;
#pragma unroll
  for (int i = 0; i < RT; ++i)
#pragma unroll
    for (int j = 0; j < CT; ++j)
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) bad = fmaf(at(i, j, t)[e], 0.0f, bad);
  if (__builtin_expect(__any(bad != 0.0f || bad != bad), 0)) {
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
      for (int j = 0; j < CT; ++j)
#pragma unroll
        for (int t = 0; t < 2; ++t) at(i, j, t) = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
    lora_pass<RT, CT, 1, 1, true>(lo, N, r.id, r.mine, r.all, r.voff, cb, lane, turn, turns, at);
  }
}

// ---- 256 x 256 tiles ----
// A tile takes its rows' adapters as more steps of 64 values behind K, in pairs: the high parts of
// 64 of the rank's values, then the low ones, for each adapter among its rows, each slice among
// its columns and each 64 of the rank; of ranks up to 32 both parts are in the first step, B's values
// twice, and the second one is empty; of ranks up to 16 the first step's halves are two adapters' (Lora::two: their slots must
// be within one 32-bit offset of each other).  Rows of other adapters and columns of other slices come as
// zeros.  Where that is not all of the tile, a result that is not finite may be the zeros' fault:
// the tile is then done again as quarters of 128 x 128, whose sums are kept apart per row
// (lora_add, the same products in the same order: a row has the same bits).  So are the tiles with
// more than kLoraMix adapters or kLoraPairs pairs, 2 to 3 us each (us, 768 rows, 12352 columns, 6 / 12 / 20 adapters
// a tile, in pairs: rank 16 47 / 58 / 73, one to a pair 54 / 71; in quarters 65 / 65 / 70; of bf16 rows 57 / 68 / 82,
// 62 / 78, 85 / 87 / 93), and those of at most 128 columns, which are two quarters and not four, with more than kLoraNarrow
// pairs (one to a pair, 2 / 4 / 6 adapters, the last 64 columns two slices: 42 / 47 / 53, all whole 43 / 54 / 65).
constexpr int kLoraMix = 20, kLoraPairs = 12, kLoraNarrow = 2, kLoraTiles = 448, kLoraMixed = 48;

// The tiles of a workgroup, made once: those that run whole with what they need, and those that
// run as quarters behind them.  (Found out tile by tile, a load waits for the stores of the tile
// before: 5 us a tile.)  Tile j of workgroup `slot` is number stride j + (slot + j) % stride of its
// XCD, so that a row block's tiles go to different workgroups.
struct LoraTiles {
  int whole, quarters;
  // code: the one adapter of all rows, kNone, or kMixed - i for entry i of mix
  int tile[kLoraTiles], code[kLoraTiles], in_quarters[kLoraTiles];
  int mix[kLoraMixed][kLoraMix + 1];  // how many, and which
  uint8_t which[kLoraMixed][256];     // each row's of them, kLoraMix: none
  uint8_t pairs[kLoraTiles];  // of steps, + kPart: of which not all rows or columns have the same
  uint8_t again[kLoraTiles];
  static constexpr int kNone = -1, kMixed = -2, kPart = 128;
};

// slices of columns n0 .. n1 - 1: the first, and one past the last
__device__ __forceinline__ void lora_slices(const Lora& lo, int n0, int n1, int& p0, int& p1) {
  p0 = 0;
#pragma unroll
  for (int i = 0; i + 1 < kMaxParts; ++i) p0 += n0 >= lo.end[i] ? 1 : 0;
  p1 = 1;
#pragma unroll
  for (int i = 0; i + 1 < kMaxParts; ++i) p1 += n1 > lo.end[i] ? 1 : 0;
}

template <class TileOf>
__device__ __forceinline__ void lora_tiles(LoraTiles& list, const Lora& lo, int M, int N, int first, int end, int slot,
                                           int stride, const TileOf& tile_of) {
  if (threadIdx.x < 64) {
    const int lane = static_cast<int>(threadIdx.x);
    const int last = (M - 1) / 16, parts = (lo.rank + 63) / 64;
    const uint64_t below = (uint64_t{1} << lane) - 1;
    int nw = 0, nq = 0, nm = 0;
    for (int j0 = 0; first + stride * j0 < end; j0 += 64) {
      const int j = j0 + lane, t = first + stride * j + (slot + j) % stride;
      const bool valid = t < end;
      int m0 = 0, n0 = 0, code = LoraTiles::kNone;
      bool quarters = false;
      int pairs = 0;
      if (valid) {
        tile_of(t, m0, n0);
        code = lo.groups[m0 / 16];
        int differ = 0;
#pragma unroll
        for (int i = 1; i < 16; ++i) differ |= lo.groups[min(m0 / 16 + i, last)] ^ code;
        if (differ || code < LoraTiles::kNone) code = LoraTiles::kMixed;
      }
      // the tiles whose rows differ, one after the other by the whole wave
      for (uint64_t todo = __ballot(code == LoraTiles::kMixed); todo; todo &= todo - 1) {
        const int at = __builtin_ctzll(todo), m = __builtin_amdgcn_readlane(m0, at);
        int id[4], which[4], n = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) id[i] = lora_id(lo, m + 64 * i + lane, M), which[i] = kLoraMix;
        for (;;) {
          int s = -1;
#pragma unroll
          for (int i = 3; i >= 0; --i) {
            const uint64_t left = __ballot(id[i] >= 0);
            if (left) s = __builtin_amdgcn_readlane(id[i], __builtin_ctzll(left));
          }
          if (s < 0) break;
          if (n < kLoraMix && nm < kLoraMixed && lane == 0) list.mix[nm][n + 1] = s;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            which[i] = id[i] == s ? n : which[i];
            id[i] = id[i] == s ? -1 : id[i];
          }
          if (++n > kLoraMix) break;
        }
        const bool fits = n <= kLoraMix && nm < kLoraMixed;
        if (fits && lane == 0) list.mix[nm][0] = n;
        if (fits) {
#pragma unroll
          for (int i = 0; i < 4; ++i) list.which[nm][64 * i + lane] = static_cast<uint8_t>(which[i]);
        }
        if (lane == at) {
          quarters = !fits;
          code = LoraTiles::kMixed - nm;
        }
        nm += fits ? 1 : 0;
      }
      if (valid && code != LoraTiles::kNone) {
        int p0, p1;
        lora_slices(lo, n0, min(n0 + 256, N), p0, p1);
        const int n = code >= 0 ? 1 : quarters ? 0 : list.mix[LoraTiles::kMixed - code][0];
        pairs = (lo.two ? (n + 1) / 2 : n) * (p1 - p0) * parts;
        quarters = quarters || pairs > (N - n0 <= 128 ? kLoraNarrow : kLoraPairs);
        pairs += code < LoraTiles::kNone || p1 - p0 > 1 ? LoraTiles::kPart : 0;
      }
      const uint64_t w = __ballot(valid && !quarters), q = __ballot(valid && quarters);
      if ((w >> lane) & 1) {
        const int at = nw + __builtin_popcountll(w & below);
        list.tile[at] = t;
        list.code[at] = code;
        list.pairs[at] = static_cast<uint8_t>(pairs);
        list.again[at] = 0;
      } else if ((q >> lane) & 1) {
        list.in_quarters[nq + __builtin_popcountll(q & below)] = t;
      }
      nw += __builtin_popcountll(w);
      nq += __builtin_popcountll(q);
    }
    if (lane == 0) list.whole = nw, list.quarters = nq;
  }
  __syncthreads();
}

// What tile `at` of the list takes behind K: `pairs` of steps, `part` that of a tile of which not
// all rows or columns have the same.
struct LoraSteps {
  int code, pairs;
  bool part;
};
__device__ __forceinline__ LoraSteps lora_steps(const LoraTiles& list, int at) {
  const int pairs = __builtin_amdgcn_readfirstlane(list.pairs[at]);
  return LoraSteps{__builtin_amdgcn_readfirstlane(list.code[at]), pairs % LoraTiles::kPart, pairs >= LoraTiles::kPart};
}
// Pair e of them: the adapter and its number among the tile's, the next one that goes with it (-1: none), the slice and its
// columns, the first of the rank's values.
struct LoraPair {
  int s, s2, of, p, beg, end, r0;
  bool both;  // a pair of the tile has a second one (the same for all of them: the next pair's is asked for before the products)
};
__device__ __forceinline__ LoraPair lora_pair(const LoraTiles& list, const Lora& lo, const LoraSteps& t, int e, int N,
                                              int n0) {
  int p0, p1;
  lora_slices(lo, n0, min(n0 + 256, N), p0, p1);
  const int parts = (lo.rank + 63) / 64, per = parts * (p1 - p0), i = e / per, r = e - i * per;
  LoraPair q;
  q.of = lo.two ? 2 * i : i;
  q.s = t.code;
  q.s2 = -1;
  q.both = false;
  if (t.code < LoraTiles::kNone) {
    const int* mix = list.mix[LoraTiles::kMixed - t.code];
    q.s = __builtin_amdgcn_readfirstlane(mix[1 + q.of]);
    const int n = __builtin_amdgcn_readfirstlane(mix[0]);
    q.both = lo.two && n > 1;
    if (lo.two && q.of + 1 < n) q.s2 = __builtin_amdgcn_readfirstlane(mix[2 + q.of]);
  }
  q.p = p0 + r / parts;
  q.r0 = 64 * (r % parts);
  q.beg = q.p == 0 ? 0 : lora_end(lo, q.p - 1);
  q.end = lora_end(lo, q.p);
  return q;
}
// Offsets of the wave's loads for a pair (rows m0 .., columns n0 ..; va and vb as the products'),
// the pointers in A's and B's place, the bytes from the high parts to the low ones (0: both are in the first
// step), and whether a step's second half has values.
__device__ __forceinline__ void lora_offsets(const LoraTiles& list, const Lora& lo, const LoraSteps& t, const LoraPair& q, int M, int N, int m0,
                                             int n0, int wave, int lane, int (&va)[2][2], int (&vb)[2][2], LoraBase& na,
                                             LoraBase& nb, int& low, bool& all) {
  const int half = lo.rank / 8, r = 8 * wave + (lane >> 3);
  const bool one = half <= 4;
  int ga = (lane & 7) ^ (((wave & 1) << 2) | (lane >> 4));
  int gb = (lane & 7) ^ (((wave & 3) << 1) | ((lane >> 4) & 1));
  const int to = one ? 2 * half : half - q.r0 / 8;
  // (a second adapter: its values in the step's second half)
  int base = q.s, of = q.of, more = 0;
  if (q.s2 >= 0) {
    base = min(q.s, q.s2);
    of += ga >> 2;
    more = ((gb >> 2 ? q.s2 : q.s) - base) * static_cast<int>(lo.b_slot) * 2;
    ga &= 3;
    gb &= 3;
  }
  const int oa = ga < to ? 0 : kNoOffset, ob = gb < to ? 0 : kNoOffset;
  gb -= one && gb >= half ? half : 0;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int row = m0 + 128 * h + 64 * i + r, col = n0 + 128 * h + 64 * i + r;
      va[h][i] = (min(row, M - 1) * static_cast<int>(lo.ldv) * 2 + 16 * ga) | oa;
      vb[h][i] = (min(col, N - 1) * lo.rank * 2 + 16 * gb + more) | ob | (col >= q.beg && col < q.end ? 0 : kNoOffset);
      // (a load from memory here would wait for all that are in flight, 0.5 us a pair)
      if (t.code < LoraTiles::kNone) va[h][i] |= list.which[LoraTiles::kMixed - t.code][row - m0] == of ? 0 : kNoOffset;
    }
  na = LoraBase(lo.v + 2 * q.p * lo.rank + q.r0);
  nb = LoraBase(lo.b + base * lo.b_slot + q.r0);
  low = one ? 0 : 2 * lo.rank;
  all = half > 2 || q.both;
}
// The tiles to be done again, behind the others' quarters; returns how many quarters.
__device__ __forceinline__ int lora_quarters(LoraTiles& list) {
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = list.quarters;
    for (int i = 0; i < list.whole; ++i)
      if (list.again[i]) list.in_quarters[n++] = list.tile[i];
    list.quarters = n;
  }
  __syncthreads();
  return 4 * __builtin_amdgcn_readfirstlane(list.quarters);
}
// Whether every workgroup's list holds its tiles.
bool lora_tiles_fit(int64_t whole) { return (whole + gdn::kNumCu - 1) / gdn::kNumCu + 1 < kLoraTiles; }

// The arguments of the entry points, checked; slots == 0: no row has an adapter.
bool lora_of(Lora& lo, const uint16_t* v, int64_t ldv, const int* groups, const uint16_t* b, int64_t b_slot,
             const int* ids, int slots, int rank, int slices, const int* slice_end, int M, int N) {
  const int64_t kLimit = 1LL << 31;
  if (!ids || slots < 0 || rank < 8 || rank > kMaxRank || rank % 8 || slices < 1 || slices > kMaxParts || !slice_end)
    return false;
  if (slots && (!v || !b || !groups || reinterpret_cast<uintptr_t>(v) % 16 || reinterpret_cast<uintptr_t>(b) % 16 ||
                reinterpret_cast<uintptr_t>(groups) % 4))
    return false;
  if (reinterpret_cast<uintptr_t>(ids) % 4 || ldv % 8 || ldv < 2LL * slices * rank || M * ldv * 2 >= kLimit ||
      b_slot % 8 || (slots > 1 && b_slot < static_cast<int64_t>(N) * rank) ||
      static_cast<int64_t>(N + 256) * rank * 2 >= kLimit)
    return false;
  lo = Lora{v, ldv, b, b_slot, ids, groups, lora_sorted(M, slots) ? groups + (M + 15) / 16 : nullptr, slots, rank, slices, {N, N, N, N},
            rank <= 16 && slots <= (kLimit / 2 - 1) / std::max<int64_t>(b_slot, 1)};
  for (int p = 0, beg = 0; p < slices; beg = slice_end[p++]) {
    const bool last = p + 1 == slices;
    if (slice_end[p] <= beg || (last ? slice_end[p] != N : slice_end[p] % 16 != 0 || slice_end[p] >= N)) return false;
    lo.end[p] = slice_end[p];
  }
  return true;
}

}  // namespace
