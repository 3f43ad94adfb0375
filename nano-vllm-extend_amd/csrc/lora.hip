// The first half of low-rank adapters beside a projection: the rows shrunk to their adapters'
// rank, v[m][j] = scale_s sum over k of x[m][k] A_s[j][k], s = ids[m] the row's adapter (none
// outside of 0 .. slots - 1: nothing is written for the row), j over the slices' ranks one
// after the other.  The GEMMs take v from there (lora_tile.h).  No counterpart in the
// reference.
//
// v is summed in fp32 and held as two bf16 values, high and low part (2^-16 of it is lost): one
// would cost the result as much again as its own rounding where an adapter's share is as large
// as the projection's.
//
// Prompts (lora_shrink_kernel): a workgroup has 16 MT rows and 16 NT of the columns j.  It goes
// through the adapters of its rows, each once: all rows times the adapter's A, K-steps dealt to
// the waves, each with a ring of NS stages of its own in LDS that loads fill directly (as in the
// GEMM's ring kernel), the waves' sums added in wave order, and the rows that have the adapter
// stored.
//
// Few rows (lora_few_kernel), most of them with adapters of their own, are bound by the reading
// of A: 16 rows and 16 columns to a workgroup, K dealt to its waves, all of their
// loads on their way at once.  Up to kLoraSort rows are taken in the order of their
// adapters, so that an adapter's A is read once for each 16 of its rows and not once for each 16
// rows that it is among; the GEMM takes its rows in the same order.
//
// x comes in bf16 (steps of 64 values) or in e4m3 with a scale for each row and 128 columns
// (steps of 128): e4m3 values are bf16 ones, so a group's sum is the matrix cores' and the
// scale is applied to it in fp32.
#include <algorithm>

#include "lora_tile.h"
#include "quant_fp8.h"

namespace {

typedef int i32x2_t __attribute__((ext_vector_type(2)));

struct Shrink {
  const void* x;
  int64_t ldx;
  const float* xs;  // kFp8: scale of row m, group g at xs[m xs_row + g xs_grp]
  int64_t xs_row, xs_grp;
  const uint16_t* a;  // [slots][cols, K] bf16
  int64_t a_slot;
  const float* scale;  // [slots]
  const int* ids;
  int slots, cols, rank, M, K;
  uint16_t* v;
  int64_t ldv;
  int* groups;  // [ceil(M / 16)]: the adapter of 16 rows, -1 none, -2 not one for all; up to kLoraSort rows: [M] the
                // rows in the order of their adapters, [M] these
  // lora_few_kernel: where x is bf16 and an 8-bit product reads it next, its e4m3 rows, by workgroups of their own
  // behind the `share` of the adapters' (one launch less: 2.3 us)
  uint8_t* x8;
  int64_t sx8;
  float* s8;
  int64_t s8_row, s8_grp;
  int share;
};

// 8 e4m3 values as bf16
__device__ __forceinline__ gdn::s16x8_t e4m3_to_bf16(const i32x2_t& w) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  uint32_t d[4];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
    d[2 * i] = gdn::f2bf2(lo[0], lo[1]);
    d[2 * i + 1] = gdn::f2bf2(hi[0], hi[1]);
  }
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(gdn::s16x8_t, u4{d[0], d[1], d[2], d[3]});
}

// Columns c .. c + 3 of row m (a slice's ranks are a multiple of 8).
__device__ __forceinline__ void store_v(const Shrink& p, int m, int c, const gdn::f32x4_t& sum, float scale) {
  if (c >= p.cols) return;
  float hi[4], lo[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float val = sum[e] * scale;
    hi[e] = gdn::bf2f(gdn::f2bf(val));
    // (what bf16 does not hold is infinite in the one part and has none in the other)
    lo[e] = fabsf(hi[e]) < __builtin_inff() ? val - hi[e] : 0.0f;
  }
  const int slice = c / p.rank;
  uint16_t* at = p.v + static_cast<int64_t>(m) * p.ldv + slice * p.rank + c;
  *reinterpret_cast<uint2*>(at) = make_uint2(gdn::f2bf2(hi[0], hi[1]), gdn::f2bf2(hi[2], hi[3]));
  *reinterpret_cast<uint2*>(at + p.rank) = make_uint2(gdn::f2bf2(lo[0], lo[1]), gdn::f2bf2(lo[2], lo[3]));
}

// A wave's share of 16 rows times 16 columns of one adapter: the K-steps wave, wave + NW, ...  Of C
// steps the loads are on their way at once, 8 lanes to a row's 128 bytes (straight in the
// matrix cores' layout, a row to a lane, they took 4 times as long); each step then goes through the wave's own rows of
// LDS.  A lane asks for rows (-1: none) and columns lane / 8 and 8 + lane / 8; steps past the end load zeros.
constexpr int kFewWaves = 8;  // (16 take as long, K up to 16384, and longer where there are more tiles than CUs)

template <bool kFp8>
__device__ __forceinline__ gdn::f32x4_t few_product(const Shrink& p, __amdgpu_buffer_rsrc_t rx, __amdgpu_buffer_rsrc_t ra,
                                                    __amdgpu_buffer_rsrc_t rs, const int (&row)[2], int own_row, int c0, int wave,
                                                    int lane, uint8_t* lds) {
  constexpr int NW = kFewWaves, C = kFp8 ? 2 : 4, kStep = kFp8 ? 128 : 64, kHalves = kFp8 ? 2 : 1;
  const int nk = p.K / kStep, lr = lane & 15, lg = lane >> 4;
  int xoff[2], aoff[2], at[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 8 * i + (lane >> 3);
    xoff[i] = row[i] < 0 ? kNoOffset : static_cast<int>(row[i] * p.ldx * (kFp8 ? 1 : 2)) + 16 * (lane & 7);
    aoff[i] = min(c0 + r, p.cols - 1) * p.K * 2 + 16 * (lane & 7);
    at[i] = sw_off(r, lane & 7);
  }
  const int soff = kFp8 ? static_cast<int>(own_row * p.xs_row * 4) : 0;
  gdn::f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = wave; k0 < nk; k0 += C * NW) {
    gdn::s16x8_t x[C][2], a[C][2 * kHalves];
    float f[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int k = k0 + i * NW, off = k < nk ? 0 : kNoOffset;
#pragma unroll
      for (int h = 0; h < 2; ++h) x[i][h] = lora_load(rx, (xoff[h] + 128 * k) | off | (xoff[h] & kNoOffset));
#pragma unroll
      for (int h = 0; h < 2 * kHalves; ++h) a[i][h] = lora_load(ra, (aoff[h & 1] + 128 * (kHalves * k + (h >> 1))) | off);
      if constexpr (kFp8)
        f[i] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(
                                             rs, (soff + static_cast<int>(p.xs_grp) * 4 * k) | off, 0, 0));
    }
#pragma unroll
    for (int i = 0; i < C; ++i) {
#pragma unroll
      for (int h = 0; h < 2; ++h) *reinterpret_cast<gdn::s16x8_t*>(lds + at[h]) = x[i][h];
#pragma unroll
      for (int h = 0; h < 2 * kHalves; ++h)
        *reinterpret_cast<gdn::s16x8_t*>(lds + 2048 * (1 + (h >> 1)) + at[h & 1]) = a[i][h];
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
      gdn::f32x4_t sum = kFp8 ? gdn::f32x4_t{0.f, 0.f, 0.f, 0.f} : acc;
#pragma unroll
      for (int ks = 0; ks < 2 * kHalves; ++ks) {
        const gdn::s16x8_t fa = *reinterpret_cast<const gdn::s16x8_t*>(lds + 2048 * (1 + (ks >> 1)) + sw_off(lr, 4 * (ks & 1) + lg));
        gdn::s16x8_t fx;
        if constexpr (kFp8)
          fx = e4m3_to_bf16(*reinterpret_cast<const i32x2_t*>(lds + sw_off(lr, 2 * ks + (lg >> 1)) + 8 * (lg & 1)));
        else
          fx = *reinterpret_cast<const gdn::s16x8_t*>(lds + sw_off(lr, 4 * ks + lg));
        sum = gdn::mfma16x16x32(fa, fx, sum);
      }
      if constexpr (kFp8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(sum[e], f[i], acc[e]);
      } else {
        acc = sum;
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
    }
  }
  return acc;
}

// kSort: 17 to kLoraSort rows in the order of their adapters, blockIdx.y and on every share-th
// of the runs of one adapter in 16 places of that order; the order is written for the GEMM.  Every
// workgroup finds it for itself: a row's place is the number of rows before it, counted by all
// threads (256 rows: 1 us, and none of it waits for memory).  Else: blockIdx.x has 16 rows and, of
// their adapters, the blockIdx.y-th and on every share-th.
template <bool kFp8, bool kSort>
__global__ __launch_bounds__(64 * kFewWaves) void lora_few_kernel(Shrink p) {
  constexpr int NW = kFewWaves;
  constexpr int kStepBytes = kFp8 ? 6144 : 4096;
  __shared__ __align__(16) unsigned key[kLoraSort];
  __shared__ int place[kLoraSort], s_row[kLoraSort], s_id[kLoraSort], s_item[kLoraSort], s_count[4];
  __shared__ __align__(16) uint8_t steps[NW * kStepBytes];
  gdn::f32x4_t* red = reinterpret_cast<gdn::f32x4_t*>(steps);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int tiles_n = (p.cols + 15) / 16;
  const int c0 = 16 * static_cast<int>(blockIdx.x % tiles_n), m0 = 16 * static_cast<int>(blockIdx.x / tiles_n);
  if constexpr (!kFp8)
    if (static_cast<int>(blockIdx.y) >= p.share) {
      const int64_t b = static_cast<int64_t>(blockIdx.y - p.share) * gridDim.x + blockIdx.x;
      quant_group<false>(p.x, p.ldx, p.x8, p.sx8, p.s8, p.s8_row, p.s8_grp, p.M, p.K / gdn::kFp8Group, b * (4 * NW) + tid / 16,
                         tid % 16);
      return;
    }
  const __amdgpu_buffer_rsrc_t rx = rsrc_of(p.x), rs = rsrc_of(p.xs);
  // rows: the ones that the lane loads
  auto run = [&](int s, const int (&rows)[2], int row, bool own) {
    const gdn::f32x4_t acc = few_product<kFp8>(p, rx, rsrc_of(p.a + s * p.a_slot), rs, rows, row, c0, wave, lane,
                                                   steps + wave * kStepBytes);
    const float scale = p.scale[s];
    __syncthreads();
    red[64 * wave + lane] = acc;
    __syncthreads();
    if (wave == 0) {
      gdn::f32x4_t sum = acc;
#pragma unroll
      for (int w = 1; w < NW; ++w) sum += red[64 * w + lane];
      if (own) store_v(p, row, c0 + 4 * lg, sum, scale);
    }
    __syncthreads();
  };
  if constexpr (kSort) {
    // a row's key: its adapter (0: none) and its number; the keys of P rows, T / P parts of them to a row
    const int P = p.M <= 64 ? 64 : p.M <= 128 ? 128 : 256, parts = 64 * NW / P;
    if (tid < P) {
      const int s = p.ids[min(tid, p.M - 1)];
      const unsigned id = static_cast<unsigned>(s) < static_cast<unsigned>(p.slots) ? s + 1 : 0;
      key[tid] = tid < p.M ? id * kLoraSort + tid : ~0u;
      place[tid] = 0;
    }
    __syncthreads();
    const int m = tid & (P - 1), per = (p.M + 4 * parts - 1) / (4 * parts);
    const unsigned own_key = key[m];
    const int mine = static_cast<int>(own_key / kLoraSort) - 1;
    if (m < p.M) {
      int count = 0;
      const uint4* keys = reinterpret_cast<const uint4*>(key);
      const int from = __builtin_amdgcn_readfirstlane(tid / P * per), to = min(from + per, P / 4);
#pragma unroll 8
      for (int j = from; j < to; ++j) {
        const uint4 k = keys[j];
        count += k.x < own_key ? 1 : 0;
        count += k.y < own_key ? 1 : 0;
        count += k.z < own_key ? 1 : 0;
        count += k.w < own_key ? 1 : 0;
      }
      atomicAdd(&place[m], count);
    }
    const uint64_t differ = __ballot(m < p.M && mine != static_cast<int>(key[m & ~15] / kLoraSort) - 1);
    __syncthreads();
    if (tid < p.M) {
      s_row[place[tid]] = tid;
      s_id[place[tid]] = mine;
    }
    __syncthreads();
    const bool first = tid < p.M && s_id[tid] >= 0 && (tid % 16 == 0 || s_id[tid] != s_id[tid - 1]);
    const uint64_t firsts = __ballot(first);
    if (wave < 4 && lane == 0) s_count[wave] = __builtin_popcountll(firsts);
    if (blockIdx.x == 0 && blockIdx.y == 0 && tid < p.M) {
      if (lr == 0) p.groups[tid / 16] = (differ >> lane) & 0xffff ? -2 : mine;
      int* order = p.groups + (p.M + 15) / 16;
      order[tid] = s_row[tid];
      order[p.M + tid] = s_id[tid];
    }
    __syncthreads();
    int before = 0, items = 0;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      before += w < wave ? s_count[w] : 0;
      items += s_count[w];
    }
    if (first) s_item[before + __builtin_popcountll(firsts & ((1ull << lane) - 1))] = tid;
    __syncthreads();
    for (int it = blockIdx.y; it < items; it += p.share) {
      const int at = s_item[it], to = min(at | 15, p.M - 1);
      const int s = __builtin_amdgcn_readfirstlane(s_id[at]);
      auto has = [&](int i) { return at + i <= to && s_id[min(at + i, to)] == s; };
      auto row = [&](int i) { return has(i) ? s_row[at + i] : -1; };
      const int rows[2] = {row(lane >> 3), row(8 + (lane >> 3))};
      run(s, rows, max(row(lr), 0), has(lr));
    }
  } else {
    const int r = m0 + lr, s0 = p.ids[min(r, p.M - 1)];
    const int id = r < p.M && static_cast<unsigned>(s0) < static_cast<unsigned>(p.slots) ? s0 : -1;
    const int first = __builtin_amdgcn_readfirstlane(id);
    const bool alike = !__any(r < p.M && id != first);
    if (c0 == 0 && blockIdx.y == 0 && tid == 0) p.groups[m0 / 16] = alike ? first : -2;
    LoraIds it{__ballot(id >= 0 && lane < 16), 0, 1};
    uint64_t rows;
    int turn = static_cast<int>(blockIdx.y);
    for (int s = it.next(id, rows); s >= 0; s = it.next(id, rows)) {
      if (turn-- > 0) continue;
      turn = p.share - 1;
      auto row = [&](int i) { return (rows >> i) & 1 ? m0 + i : -1; };
      const int mine[2] = {row(lane >> 3), row(8 + (lane >> 3))};
      run(s, mine, min(r, p.M - 1), id == s);
    }
  }
}

template <int MT, int NT, int NW, int NS, bool kFp8>
__global__ __launch_bounds__(64 * NW) void lora_shrink_kernel(Shrink p) {
  constexpr int BM = 16 * MT, BN = 16 * NT;
  constexpr int kStep = kFp8 ? 128 : 64;                   // values of a K-step
  constexpr int kHalves = kFp8 ? 2 : 1;                    // 128-byte rows of A in it
  constexpr int kXBytes = BM * 128, kABytes = BN * 128;    // (of one half)
  constexpr int kStage = kXBytes + kHalves * kABytes + (kFp8 ? 256 : 0);
  constexpr int kXPer = kXBytes / 1024, kAPer = kABytes / 1024;
  constexpr int kPer = kXPer + kHalves * kAPer + (kFp8 ? 1 : 0);
  constexpr int kVm = (NS - 1) * kPer;
  static_assert(kVm < 64 && (NS == 2 || NS == 3), "vmcnt field");
  constexpr int kWait = (kVm & 15) | (7 << 4) | (15 << 8) | ((kVm >> 4) << 14);
  static_assert(MT * NT * 1024 <= kStage, "the partial sums fit a stage");
  __shared__ __align__(16) uint8_t st0[NW * kStage];
  __shared__ __align__(16) uint8_t st1[NW * kStage];
  __shared__ __align__(16) uint8_t st2[NS > 2 ? NW * kStage : 16];
  // (the column tiles of a row tile one after the other on one XCD: x comes from its L2)
  const int tiles_n = (p.cols + BN - 1) / BN;
  const int64_t tile = gdn::xcd_remap(blockIdx.x, static_cast<int64_t>((p.M + BM - 1) / BM) * tiles_n);
  if (tile < 0) return;
  const int m0 = BM * static_cast<int>(tile / tiles_n), c0 = BN * static_cast<int>(tile % tiles_n);
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  int id[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    const int r = m0 + 16 * i + lr;
    const int s = p.ids[min(r, p.M - 1)];
    id[i] = r < p.M && static_cast<unsigned>(s) < static_cast<unsigned>(p.slots) ? s : -1;
    const int first = __builtin_amdgcn_readfirstlane(id[i]);
    const bool alike = !__any(r < p.M && id[i] != first);
    if (c0 == 0 && blockIdx.y == 0 && threadIdx.x == 0 && r < p.M) p.groups[m0 / 16 + i] = alike ? first : -2;
  }
  int mine = BM > lane ? id[0] : -1;  // row m0 + lane's
#pragma unroll
  for (int i = 1; i < MT; ++i) mine = lg == i ? id[i] : mine;
  LoraIds it{__ballot(mine >= 0), 0, 1};
  uint64_t rows;
  int turn = static_cast<int>(blockIdx.y);  // adapters before this workgroup's next
  auto next = [&]() {
    int s;
    do s = it.next(mine, rows);
    while (s >= 0 && turn-- > 0);
    turn = static_cast<int>(gridDim.y) - 1;
    return s;
  };
  int s = next();
  if (s < 0) return;  // (the workgroup)

  const __amdgpu_buffer_rsrc_t rx = rsrc_of(p.x), rs = rsrc_of(p.xs);
  int goff[kXPer + kAPer];
#pragma unroll
  for (int i = 0; i < kXPer + kAPer; ++i) {
    const int r = 8 * (i < kXPer ? i : i - kXPer) + (lane >> 3);
    const int gran = 16 * ((lane & 7) ^ ((r >> 1) & 7));
    goff[i] = i < kXPer ? static_cast<int>(min(m0 + r, p.M - 1) * p.ldx * (kFp8 ? 1 : 2)) + gran
                        : min(c0 + r, p.cols - 1) * p.K * 2 + gran;
  }
  const int vs = kFp8 ? static_cast<int>(min(m0 + lane % BM, p.M - 1) * p.xs_row * 4) : 0;
  const int nk = p.K / kStep;
  while (s >= 0) {
    const __amdgpu_buffer_rsrc_t ra = rsrc_of(p.a + s * p.a_slot);
    auto issue = [&](uint8_t* st, int step) {
      const int k = min(step, nk - 1);
      uint8_t* w = st + wave * kStage;
#pragma unroll
      for (int i = 0; i < kXPer; ++i) dma16(rx, w + i * 1024, goff[i], 128 * k);
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int i = 0; i < kAPer; ++i)
          dma16(ra, w + kXBytes + h * kABytes + i * 1024, goff[kXPer + i], 128 * (kHalves * k + h));
      if constexpr (kFp8)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr_t)(w + kXBytes + kHalves * kABytes), 4, vs,
                                                 static_cast<int>(p.xs_grp) * 4 * k, 0, 0);
    };
    gdn::f32x4_t acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) acc[i][j] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
    auto one = [&](uint8_t* st, int step) {
      const uint8_t* x = st + wave * kStage;
      const uint8_t* a = x + kXBytes;
      constexpr int kSub = kStep / 32;
      gdn::s16x8_t fa[kSub][NT];
      gdn::s16x8_t fx[kSub][MT];
      float f[MT];
#pragma unroll
      for (int ks = 0; ks < kSub; ++ks) {
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          const int r = 16 * i + lr;
          if constexpr (kFp8)
            fx[ks][i] = e4m3_to_bf16(*reinterpret_cast<const i32x2_t*>(x + sw_off(r, 2 * ks + (lg >> 1)) + 8 * (lg & 1)));
          else
            fx[ks][i] = *reinterpret_cast<const gdn::s16x8_t*>(x + sw_off(r, 4 * ks + lg));
        }
#pragma unroll
        for (int j = 0; j < NT; ++j)
          fa[ks][j] = *reinterpret_cast<const gdn::s16x8_t*>(a + (ks >> 1) * kABytes + sw_off(16 * j + lr, 4 * (ks & 1) + lg));
      }
      if constexpr (kFp8)
#pragma unroll
        for (int i = 0; i < MT; ++i) f[i] = reinterpret_cast<const float*>(a + kHalves * kABytes)[16 * i + lr];
      // the reads have returned before the stage is loaded again
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kWaitLds);
      __builtin_amdgcn_sched_barrier(0);
      issue(st, step + NS * NW);
#pragma unroll
      for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          gdn::f32x4_t sum = kFp8 ? gdn::f32x4_t{0.f, 0.f, 0.f, 0.f} : acc[i][j];
#pragma unroll
          for (int ks = 0; ks < kSub; ++ks) sum = gdn::mfma16x16x32(fa[ks][j], fx[ks][i], sum);
          if constexpr (kFp8) {
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][j][e] = fmaf(sum[e], f[i], acc[i][j][e]);
          } else {
            acc[i][j] = sum;
          }
        }
      __builtin_amdgcn_sched_barrier(0);
      __builtin_amdgcn_s_waitcnt(kWait);
      __builtin_amdgcn_sched_barrier(0);
    };
    issue(st0, wave);
    issue(st1, wave + NW);
    if constexpr (NS == 3) issue(st2, wave + 2 * NW);
    __builtin_amdgcn_s_waitcnt(kWait);
    int k = wave;
    for (; k + (NS - 1) * NW < nk; k += NS * NW) {
      one(st0, k);
      one(st1, k + NW);
      if constexpr (NS == 3) one(st2, k + 2 * NW);
    }
    if (k < nk) one(st0, k);
    if (NS == 3 && k + NW < nk) one(st1, k + NW);
    // the repeated loads past the last step land before the stages are reused
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    gdn::f32x4_t* red = reinterpret_cast<gdn::f32x4_t*>(st0);  // [wave][row tile][column tile][lane]
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
      for (int j = 0; j < NT; ++j) red[((wave * MT + i) * NT + j) * 64 + lane] = acc[i][j];
    __syncthreads();
    const float scale = p.scale[s];
#pragma unroll
    for (int ij = 0; ij < MT * NT; ++ij) {
      if (ij % NW != wave) continue;
      const int i = ij / NT, j = ij % NT;
      gdn::f32x4_t sum = red[ij * 64 + lane];
#pragma unroll
      for (int w = 1; w < NW; ++w) sum += red[(w * MT * NT + ij) * 64 + lane];
      if (id[i] == s) store_v(p, m0 + 16 * i + lr, c0 + 16 * j + 4 * lg, sum, scale);
    }
    s = next();
    if (s >= 0) __syncthreads();  // the sums have been read
  }
}

// Whether the kernel of few rows takes them: its 16 x 16 tiles read A and x again for each other, the prompts' 64-row
// tiles take 9 to 12 us for any number up to the CUs (us, few / prompts, 2048 columns of bf16 x, one adapter: 2000 x 64 8.8 /
// 11.6, 2000 x 128 14.8 / 12.2, 800 x 256 10.4 / 12.1, 1100 x 256 13.5 / 12.3, 800 x 512 15.5 / 12.5; of rows at random
// 1100 x 256 56 / 41).  Rows whose order the product goes by are its whatever their columns: it writes the order.
bool few_rows(int M, int cols, int slots) {
  return lora_sorted(M, slots) || (M <= 2048 && (M + 15) / 16 * ((cols + 15) / 16) <= 7 * gdn::kNumCu / 2);
}

template <bool kFp8>
int launch(Shrink p, hipStream_t st) {
  auto tiles = [](int n, int of) { return (n + of - 1) / of; };
  // Prompts: 64-row tiles, all columns up to 64 (32 of them where x is e4m3: its stages are the larger ones).
  // Four waves have a CU's LDS for themselves; with more tiles than CUs two waves and a
  // half of it, so that a second tile runs beside the first.  us, four waves / two, 2048 columns of bf16 x, all rows one
  // adapter's: 17001 x 64 (266 tiles) 26.3 / 21.5, 16384 x 128 (512) 25.9 / 20.9, 16384 x 64 (256) 18.1 / 18.0, 4096 x 128
  // (128) 12.5 / 15.1; e4m3, 16384 x 64 (512) 21.2 / 17.0, 16384 x 16 (256) 11.9 / 13.7, 4096 x 128 (256) 10.9 / 13.3.
  if (!few_rows(p.M, p.cols, p.slots)) {
    const int bn = !kFp8 && p.cols > 32 ? 64 : 32, n = tiles(p.M, 64) * tiles(p.cols, bn);
    const bool two = n > gdn::kNumCu;
    // Workgroups share a tile's adapters where that leaves no more of them than find room at once (one that finds
    // none ends): 17001 x 64 in 21 sequences 34.0 alone, 25.5 in two; 4096 x 16 in sequences of 700 12.7 and 8.7; 16384 x
    // 16 (256 tiles) 15.4 and 16.8.
    const int room = (two ? 2 : 1) * gdn::kNumCu;
    const int share = std::max(1, std::min(16, (room + n / 2) / n));
    const dim3 grid(static_cast<unsigned>(gdn::kNumXcd * tiles(n, gdn::kNumXcd)), static_cast<unsigned>(share));
    if constexpr (!kFp8)
      if (bn == 64) {
        two ? lora_shrink_kernel<4, 4, 2, 2, false><<<grid, dim3(128), 0, st>>>(p)
            : lora_shrink_kernel<4, 4, 4, 2, false><<<grid, dim3(256), 0, st>>>(p);
        return gdn_launch_status();
      }
    two ? lora_shrink_kernel<4, 2, 2, 2, kFp8><<<grid, dim3(128), 0, st>>>(p)
        : lora_shrink_kernel<4, 2, 4, 2, kFp8><<<grid, dim3(256), 0, st>>>(p);
    return gdn_launch_status();
  }
  // So many workgroups share the adapters (those that find none end).
  const int n = tiles(p.cols, 16), most = std::max(1, 512 / n);
  const bool sort = lora_sorted(p.M, p.slots);
  p.share = sort ? std::min(most, std::min(p.M, tiles(p.M, 16) + std::min(p.slots, p.M)))
                 : std::max(1, std::min(std::min(std::min(16, p.M), p.slots), 1024 / (n * tiles(p.M, 16))));
  const int across = sort ? n : n * tiles(p.M, 16);
  const int64_t quant = p.x8 ? (static_cast<int64_t>(p.M) * (p.K / gdn::kFp8Group) + 31) / 32 : 0;
  const dim3 grid(static_cast<unsigned>(across), static_cast<unsigned>(p.share + (quant + across - 1) / across));
  if (sort)
    lora_few_kernel<kFp8, true><<<grid, dim3(64 * kFewWaves), 0, st>>>(p);
  else
    lora_few_kernel<kFp8, false><<<grid, dim3(64 * kFewWaves), 0, st>>>(p);
  return gdn_launch_status();
}

}  // namespace

extern "C" int gdn_lora_shrink(const void* x, int x_is_bf16, int64_t ldx, const float* xs, int64_t xs_row, int64_t xs_grp,
                               const uint16_t* a, int64_t a_slot, const float* scale, const int32_t* ids, int slots,
                               int slices, int rank, int M, int K, uint16_t* v, int64_t ldv, int32_t* groups,
                               uint8_t* x8, int64_t sx8, float* x8_scale, int64_t s8_row, int64_t s8_grp, void* stream) {
  const int64_t kLimit = 1LL << 31;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (M < 0 || slots < 0 || slices < 1 || slices > kMaxParts || rank < 8 || rank > kMaxRank || rank % 8 || K <= 0 ||
      K % (x_is_bf16 ? 64 : gdn::kFp8Group))
    return GDN_ERR_INVALID_ARG;
  if (x8 && !x_is_bf16) return GDN_ERR_INVALID_ARG;
  if (M == 0) return GDN_OK;
  if (slots == 0) return x8 ? gdn_quantize_fp8(x, 0, ldx, x8, sx8, x8_scale, s8_row, s8_grp, M, K, 1, stream) : GDN_OK;
  const int cols = slices * rank;
  if (!x || !a || !scale || !ids || !v || !groups || (!x_is_bf16 && !xs)) return GDN_ERR_INVALID_ARG;
  if (reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(a) % 16 || reinterpret_cast<uintptr_t>(v) % 8 ||
      reinterpret_cast<uintptr_t>(scale) % 4 || reinterpret_cast<uintptr_t>(ids) % 4 || reinterpret_cast<uintptr_t>(groups) % 4 || ldx < K ||
      ldx % (x_is_bf16 ? 8 : 16) || M * ldx * (x_is_bf16 ? 2 : 1) >= kLimit || a_slot % 8 ||
      (slots > 1 && a_slot < static_cast<int64_t>(cols) * K) || static_cast<int64_t>(cols) * K * 2 >= kLimit ||
      ldv % 4 || ldv < 2LL * cols)
    return GDN_ERR_INVALID_ARG;
  if (!x_is_bf16 && (reinterpret_cast<uintptr_t>(xs) % 4 || xs_row < 0 || xs_grp < 0 ||
                     4 * ((M - 1) * xs_row + (K / gdn::kFp8Group - 1) * xs_grp) >= kLimit))
    return GDN_ERR_INVALID_ARG;
  if (x8 && (K % gdn::kFp8Group || !x8_scale || reinterpret_cast<uintptr_t>(x8) % 8 || sx8 % 8 || sx8 < K ||
             reinterpret_cast<uintptr_t>(x8_scale) % 4))
    return GDN_ERR_INVALID_ARG;
  if (x8 && !few_rows(M, cols, slots)) {
    const int status = gdn_quantize_fp8(x, 0, ldx, x8, sx8, x8_scale, s8_row, s8_grp, M, K, 1, stream);
    if (status != GDN_OK) return status;
  }
  const Shrink p{x, ldx, xs, xs_row, xs_grp, a, a_slot, scale, ids, slots, cols, rank, M, K, v, ldv, groups, x8, sx8, x8_scale, s8_row, s8_grp, 0};
  return x_is_bf16 ? launch<false>(p, st) : launch<true>(p, st);
}
