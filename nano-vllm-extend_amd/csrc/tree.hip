// Speculative verify over a tree of drafted tokens: the causal conv and the gated
// delta rule of T nodes per sequence against the slot pools, which they only read,
// and the accepted path's way into the pools.  (No counterpart in the reference:
// spec decode is disabled for qwen3_5, nanovllm/config.py:84; one token's update is
// nanovllm/models/qwen3_5.py:575-594.)
//
// parents[b][t] is the node before node t: -1 the sequence's own state, else a node
// s < t; any other value, or a parent that is itself unused, makes the node unused
// (output 0, no effect).  With E_t = e^{g_t}, W_t the product of E over the path from
// the root to t, and w(t, s) that over the nodes after s:
//   u_t = beta_t (v_t - W_t S^T k_t - sum over ancestors s of w(t, s) (k_s . k_t) u_s)
//   o_t = scale (W_t S^T q_t + sum over ancestors s and t itself of w(t, s) (k_s . q_t) u_s)
//   state after node a:  W_a S + sum over its path of w(a, s) k_s u_s^T
// so the states of the nodes are never stored: a verify reads S once, where the chain
// form (gdn_recurrent) writes one D x D state per token, and a commit forms one state
// from the path's k, g and u.  The weights are products of factors in [0, 1], never
// differences of sums: no cancellation, and a decay of 0 stays 0.  What has weight 0 is
// left out, not multiplied: a node sees nothing of what its path has forgotten, nor of
// unused nodes and other branches, infinities and NaN included.
#include <algorithm>
#include <type_traits>

#include "gdn_common.h"

namespace {

constexpr int kMaxNodes = 64;

// The links of two trees, by the 64 lanes of one wave, lane t with node t's parents: the
// parent (-1: the state), or kUnused (lanes past T too).  A node counts if the walk from it
// ends at -1; every lane jumps over its ancestor's jumps, so that the rounds are as many as
// the depth has bits.  (Jumps go to smaller nodes: they end.)
constexpr int kUnused = -2;
__device__ __forceinline__ void tree_links(int lane, int T0, int& link0, int T1, int& link1) {
  auto near = [&](int p, int T) { return lane < T && p >= -1 && p < lane ? p : kUnused; };
  link0 = near(link0, T0);
  link1 = near(link1, T1);
  int a0 = link0, a1 = link1;
  while (__any(a0 >= 0 || a1 >= 0)) {
    const int n0 = __shfl(a0, max(a0, 0), 64), n1 = __shfl(a1, max(a1, 0), 64);
    a0 = a0 >= 0 ? n0 : a0;
    a1 = a1 >= 0 ? n1 : a1;
  }
  if (a0 != -1) link0 = kUnused;
  if (a1 != -1) link1 = kUnused;
}

// The accepted node of a row, or -1: nothing was accepted.
__device__ __forceinline__ int accepted_node(int64_t want, int T, int link) {
  const int a = want >= 0 && want < T ? __builtin_amdgcn_readfirstlane(static_cast<int>(want)) : -1;
  return a >= 0 && __builtin_amdgcn_readlane(link, a) != kUnused ? a : -1;
}

// A step that was verified and is not yet in the pools.
struct RulePending {
  const uint16_t* k;       // [B, T, Hk, D], strides k_b, k_t
  int64_t k_b, k_t;
  const float* g;          // [B, T, Hv]
  const float* u;          // [B, T, Hv, D]
  const int32_t* parents;  // row stride p_b
  int64_t p_b;
  const int64_t* accepted;  // [B]; NULL: nothing pending
  int T;
};

struct ConvPending {
  const uint16_t* x;  // [B, T, C] raw rows, strides x_b, x_t
  int64_t x_b, x_t;
  const int32_t* parents;
  int64_t p_b;
  const int64_t* accepted;
  int T;
};

// Rows and tiles move through buffer loads and stores: the base, which the workgroup
// shares, in the descriptor, the lane's offset in one register, the rest in the
// instruction, so that no address pairs sit in registers.  bytes: from where on a load gives
// 0 and a store is dropped.
typedef __amdgpu_buffer_rsrc_t buf_t;
__device__ __forceinline__ buf_t buf_of(const void* base, int bytes = 0x7fffffff) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), static_cast<short>(0), bytes, 0x00020000);
}

// ---- conv ----
// The row before row r (one for the wave) of a tree: r >= 0 a node, -1, -2, -3 the taps from
// the newest.
__device__ __forceinline__ int row_before(int r, int link) {
  return r >= 0 ? __builtin_amdgcn_readlane(link, r) : r - 1;
}

// Eight channels' values (of a row, or of one tap).
struct Row8 {
  uint16_t v[8];
};
static_assert(sizeof(Row8) == 16, "one 16-byte piece");
__device__ __forceinline__ Row8 row8(const uint16_t* p) {
  return __builtin_bit_cast(Row8, *reinterpret_cast<const uint4*>(p));
}

// The three taps of channels c .. c + 7 of a slot, oldest first.  dense: the channels'
// taps lie one behind the other in 16-byte pieces.
struct Taps {
  Row8 tap[3];

  __device__ __forceinline__ void load(const uint16_t* p, int64_t sp_ch, bool dense) {
    if (dense) {
      Row8 raw[3];
#pragma unroll
      for (int i = 0; i < 3; ++i) raw[i] = row8(p + 8 * i);
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 3; ++j) tap[j].v[i] = raw[(3 * i + j) / 8].v[(3 * i + j) % 8];
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 3; ++j) tap[j].v[i] = p[i * sp_ch + j];
    }
  }
  __device__ __forceinline__ void store(uint16_t* p, int64_t sp_ch, bool dense) const {
    if (dense) {
      Row8 raw[3];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 3; ++j) raw[(3 * i + j) / 8].v[(3 * i + j) % 8] = tap[j].v[i];
#pragma unroll
      for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(p + 8 * i) = __builtin_bit_cast(uint4, raw[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 3; ++j) p[i * sp_ch + j] = tap[j].v[i];
    }
  }
  // The taps after the accepted node: its row (a), its parent's (r1) and its grandparent's (r0),
  // each a node or, below 0, one of the taps.
  __device__ __forceinline__ void advance(const ConvPending& pd, int b, int c, int a, int r1, int r0) {
    const uint16_t* x = pd.x + b * pd.x_b + c;
    // (masks: a choice among the taps becomes one among their addresses, with all of them in memory)
    typedef uint32_t words __attribute__((ext_vector_type(4)));
    const words t0 = __builtin_bit_cast(words, tap[0]), t1 = __builtin_bit_cast(words, tap[1]),
                t2 = __builtin_bit_cast(words, tap[2]);
    auto row = [&](int r) {
      words v = (t2 & (r == -1 ? ~0u : 0u)) | (t1 & (r == -2 ? ~0u : 0u)) | (t0 & (r == -3 ? ~0u : 0u));
      if (r >= 0) v = *reinterpret_cast<const words*>(x + r * pd.x_t);
      return __builtin_bit_cast(Row8, v);
    };
    tap[0] = row(r0);
    tap[1] = row(r1);
    tap[2] = row(a);
  }
};

__device__ __forceinline__ bool dense_taps(const uint16_t* pool, int64_t sp_slot, int64_t sp_ch) {
  return sp_ch == 3 && sp_slot % 8 == 0 && reinterpret_cast<uintptr_t>(pool) % 16 == 0;
}

// A workgroup is one wave: 128 channels of one sequence, two per thread, all nodes.  A
// thread's rows go through its own column of LDS, where their children find them: every
// row is read once, no wave waits for another, and a thread rolls its own channels' taps.
// Rows come 4 at a time, the next 8 on their way while these are worked on, 4 nodes' chains of
// operations side by side.  No branch in the loop: rows past T are past the buffers' ends, and
// the counts by which a wave waits for its rows stay known (else it waits for its stores too).
//
// Bound by the rows' way in and out (2 + 2 bytes per value) and, with few waves, by each
// node's own chain: 64 trees of 64 nodes, 8192 channels 35.3 us (4.1 TB/s), of 16 nodes 11.3,
// one tree of 64 nodes 5.5, of 16 nodes 4.1, of 8 nodes 3.9.  Before: with a branch per node
// 49.7 (64 x 64), 13.0 (64 x 16), 6.8 (1 x 16) and 5.1 (1 x 8); four channels per thread in
// place of two 57.4, 14.2, 8.1, 5.9.
//
// W: with few sequences W waves share a workgroup's channels and deal the groups of 4 nodes
// among them.  Wave 0 has the taps; every row is in LDS before the first node is worked on.
template <int W>
__global__ __launch_bounds__(64 * W) void conv_tree_kernel(const uint16_t* __restrict__ x, int64_t x_b, int64_t x_t,
                                                       uint16_t* __restrict__ pool, int64_t sp_slot, int64_t sp_ch,
                                                       int64_t n_slots, const int64_t* __restrict__ ids,
                                                       const uint16_t* __restrict__ w,
                                                       const int32_t* __restrict__ parents, int64_t p_b,
                                                       ConvPending pd, uint16_t* __restrict__ y, int T, int C) {
  // [3 + T up to whole groups][64], two channels per thread: the taps, oldest first, then the
  // nodes' rows, so that row r is at r + 3 (row_before)
  extern __shared__ uint32_t rows[];
  const int b = blockIdx.y, lane = threadIdx.x % 64;
  const int wave = W == 1 ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int c = 2 * (blockIdx.x * 64 + lane);
  const bool in = c < C;
  // (x_t < 2^24, C < 2^23: the rows of 64 nodes and a few more have 32-bit offsets, also from
  // 2^31 on, where the stores of channels past C are dropped)
  const buf_t by = buf_of(y + static_cast<int64_t>(b) * T * C, T * C * 2);
  const buf_t bx = buf_of(x + b * x_b, ((T - 1) * static_cast<int>(x_t) + C) * 2);
  const uint32_t y_row = 2 * C, x_row = 2 * static_cast<uint32_t>(x_t);
  const uint32_t y_at = in ? 2 * c : 0x80000000u, x_at = 2 * c;
  const int64_t slot = ids[b];
  if (slot < 0 || slot >= n_slots) {  // (the whole workgroup)
    for (int t = wave; t < T; t += W) __builtin_amdgcn_raw_buffer_store_b32(0u, by, y_at + t * y_row, 0, 0);
    return;
  }
  // what the links need first, then weights and rows, then the taps and the pending rows
  int link = parents[b * p_b + min(lane, T - 1)], last_link = kUnused;
  int64_t want = -1;
  if (pd.accepted) {
    last_link = pd.parents[b * pd.p_b + min(lane, pd.T - 1)];
    want = pd.accepted[b];
  }
  uint16_t* tp = pool + slot * sp_slot + (in ? c : 0) * sp_ch;
  const uint4 wv = *reinterpret_cast<const uint4*>(w + (in ? c : 0) * 4);
  auto pair = [](const uint16_t* p) { return *reinterpret_cast<const uint32_t*>(p); };
  constexpr int kG = 4;  // nodes at a time
  struct Group {
    uint32_t v[kG];
  };
  auto load = [&](int t0) {
    Group r;
#pragma unroll
    for (int i = 0; i < kG; ++i)
      r.v[i] = __builtin_amdgcn_raw_buffer_load_b32(bx, x_at + static_cast<uint32_t>(t0 + i) * x_row, 0, 0);
    return r;
  };
  Group next[W == 1 ? 2 : kMaxNodes / kG / W];
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(next) / sizeof(Group)); ++i) next[i] = load(kG * (wave + W * i));
  uint32_t tap[3] = {0u, 0u, 0u};  // of both channels, oldest first
  const bool dense = sp_ch == 3 && sp_slot % 2 == 0 && reinterpret_cast<uintptr_t>(pool) % 4 == 0;
  if (W > 1 && wave) {
  } else if (dense) {
    const uint32_t u0 = pair(tp), u1 = pair(tp + 2), u2 = pair(tp + 4);
    tap[0] = (u0 & 0xffffu) | (u1 & 0xffff0000u);
    tap[1] = (u0 >> 16) | (u2 << 16);
    tap[2] = (u1 & 0xffffu) | (u2 & 0xffff0000u);
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j) tap[j] = tp[j] | static_cast<uint32_t>(tp[sp_ch + j]) << 16;
  }
  gdn::keep_loads_here();
  tree_links(lane, T, link, pd.T, last_link);
  auto old = [&](int r) { return r == -1 ? tap[2] : r == -2 ? tap[1] : tap[0]; };
  const int a = wave ? -1 : accepted_node(want, pd.T, last_link);
  if (a >= 0) {
    // the taps after the accepted node: its row, its parent's and its grandparent's
    const uint16_t* lx = pd.x + b * pd.x_b + (in ? c : 0);
    const int r1 = row_before(a, last_link), r0 = row_before(r1, last_link);
    const uint32_t n2 = pair(lx + a * pd.x_t);
    const uint32_t n1 = r1 >= 0 ? pair(lx + r1 * pd.x_t) : old(r1);
    const uint32_t n0 = r0 >= 0 ? pair(lx + r0 * pd.x_t) : old(r0);
    tap[0] = n0;
    tap[1] = n1;
    tap[2] = n2;
  }
  float w0[4], w1[4];
  const uint32_t ww[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w0[j] = __uint_as_float(j % 2 ? ww[j / 2] & 0xffff0000u : ww[j / 2] << 16);
    w1[j] = __uint_as_float(j % 2 ? ww[2 + j / 2] & 0xffff0000u : ww[2 + j / 2] << 16);
  }
  if (W == 1 || wave == 0) {
#pragma unroll
    for (int j = 0; j < 3; ++j) rows[j * 64 + lane] = tap[j];
  }
  // lane t: the places of node t's three predecessors, a byte each; negative: unused
  auto up = [&](int r) {
    const int p = __shfl(link, max(r, 0), 64);
    return r >= 0 ? p : r - 1;
  };
  const int r2 = link, r1 = up(r2), r0 = up(r1);
  const int places = link == kUnused ? -1 : (r2 + 3) | (r1 + 3) << 8 | (r0 + 3) << 16;
  auto lo = [](uint32_t u) { return __uint_as_float(u << 16); };
  auto hi = [](uint32_t u) { return __uint_as_float(u & 0xffff0000u); };
  auto put = [&](int t0, const Group& now) {
#pragma unroll
    for (int i = 0; i < kG; ++i) rows[(3 + t0 + i) * 64 + lane] = now.v[i];
  };
  auto work = [&](int t0, const Group& now) {
    uint32_t x0[kG], x1[kG], x2[kG];
    int place[kG];
#pragma unroll
    for (int i = 0; i < kG; ++i) {
      place[i] = __builtin_amdgcn_readlane(places, t0 + i);
      const int at = max(place[i], 0);
      x2[i] = rows[(at & 255) * 64 + lane];
      x1[i] = rows[(at >> 8 & 255) * 64 + lane];
      x0[i] = rows[(at >> 16 & 255) * 64 + lane];
    }
#pragma unroll
    for (int i = 0; i < kG; ++i) {
      const uint32_t x3 = now.v[i];
      const uint32_t out = gdn::f2bf2(gdn::conv_decode_silu(lo(x3), lo(x0[i]), lo(x1[i]), lo(x2[i]), w0),
                                      gdn::conv_decode_silu(hi(x3), hi(x0[i]), hi(x1[i]), hi(x2[i]), w1));
      __builtin_amdgcn_raw_buffer_store_b32(place[i] < 0 ? 0u : out, by, y_at + static_cast<uint32_t>(t0 + i) * y_row,
                                            0, 0);
    }
  };
  if constexpr (W == 1) {
    for (int t0 = 0; t0 < T; t0 += kG) {
      const Group now = next[0];
      next[0] = next[1];
      next[1] = load(t0 + 2 * kG);
      put(t0, now);
      work(t0, now);
    }
  } else {
    constexpr int kGroups = kMaxNodes / kG / W;
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      if (kG * (wave + W * i) < T) put(kG * (wave + W * i), next[i]);
    gdn::lds_barrier();
#pragma unroll
    for (int i = 0; i < kGroups; ++i)
      if (kG * (wave + W * i) < T) work(kG * (wave + W * i), next[i]);
  }
  if (a < 0 || !in) return;
  if (dense) {
    uint32_t* q = reinterpret_cast<uint32_t*>(tp);
    q[0] = (tap[0] & 0xffffu) | (tap[1] << 16);
    q[1] = (tap[2] & 0xffffu) | (tap[0] & 0xffff0000u);
    q[2] = (tap[1] >> 16) | (tap[2] & 0xffff0000u);
  } else {
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      tp[j] = static_cast<uint16_t>(tap[j]);
      tp[sp_ch + j] = static_cast<uint16_t>(tap[j] >> 16);
    }
  }
}

// ---- rule ----
// One workgroup of D / 32 waves per (sequence, value head): wave w holds columns 32 w ..
// of the state, lane (lr, lg) = (lane % 16, lane / 16) columns 2 lr and 2 lr + 1 of rows
// 32 kk + 8 lg + e, in registers from the one read of it to the one write.  That is the
// second operand's layout of a 16 x 16 x 32 product over the rows, for the even columns
// and for the odd ones, with the nodes' raw bf16 rows as the first: S^T k and S^T q are
// products of 16 nodes, 32 rows and 16 columns.  S goes in as three bf16 terms that add
// up to it exactly (8 bits of the significand each), k and q are not normalised before
// (their norms scale the results), so the products are those of fp32 operands.
//
// The nodes' rows are loaded once, 8 values per lane ahead of the state, and go to LDS, where
// the coefficients (k_s . k_t, k_s . q_t, 16 x 16 nodes at a time, dealt to the waves) and the
// products with the state find them.  (Rows read by each wave from the caches: 64 x 64 nodes
// 120 us for 99, 1 x 64 21.4 for 17.7, 64 x 16 without a pending path 37.1 for 33.4.)
//
// The corrections u of 16 nodes are the product of the inverse of their 16 x 16 triangle
// (found by substitution while the state is on its way) with what the state, v and the
// nodes of earlier tiles give, and o adds the products of the second coefficients with u:
// fp32 products of 16 x 16 x 4, in which a lane's results are its part of the next
// operand (register r of lane group lg: node 4 lg + r), so that nothing goes through LDS.
//
// kLayer: the layer's gates before it and its gated norm behind it in the same launch.  Wave
// 0 finds the gates of the head's nodes.  A tile's outputs, rounded to bf16 as without the
// norm, meet in LDS, and D / 8 lanes per row take the norm in the order of its own kernel.
// Two launches and the outputs' way out and in less: 64 trees of 16 nodes 63 us for the 69
// of three launches, one of 8 nodes 12.0 for 15.4 (32 heads of 128, with a pending path).
//
// What bounds it: the state's way in (and out, where a path is pending).  The tree's
// weights, the nodes' norms and dot products (on the matrix cores as well) and the
// pending path's rows are worked on while the state is on its way.  32 heads of 128: 64
// trees of 16 nodes with a pending path 57.5 us (5.5 TB/s, a large copy's rate), without one
// 33.4; 30 trees of 24 nodes 33.5, 16 of 48 24.0; one tree of 8 nodes 6.6, the latency of its
// chain (ids, state, products, corrections).  64 nodes cost more than the state (64 trees
// 99 us, one 17.7: coefficients 4, products 2.2, corrections 3.3), and so do long paths: 21
// chains of 48 69 us, each row of the path a pass of the vector ALUs over the tile.
// Before: a thread per column of the state and one node at a time 249 us (64 x 16) and
// 32 (1 x 8).
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
constexpr float kEps = 1e-6f;
constexpr int kPathRows = 16;  // of a pending path in LDS at a time

constexpr int kNT = 2;  // cache policy: non-temporal
__device__ __forceinline__ gdn::s16x8_t buf_row(buf_t r, int voff) {
  return __builtin_bit_cast(gdn::s16x8_t, __builtin_amdgcn_raw_buffer_load_b128(r, voff, 0, 0));
}

__device__ __forceinline__ void wave_lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// The state tile of a workgroup: S[kk][e] = columns 2 lr, 2 lr + 1 of row 32 kk + 8 lg + e.
template <int D>
struct Tile {
  f32x2_t s[D / 32][8];

  // r: the tile; voff: byte offset of the lane's first row and column
  __device__ __forceinline__ void load(buf_t r, int voff) {
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        s[kk][e] = __builtin_bit_cast(
            f32x2_t, __builtin_amdgcn_raw_buffer_load_b64(r, voff + e * D * 4, 32 * kk * D * 4, kNT));
  }
  __device__ __forceinline__ void store(buf_t r, int voff) const {
    // (a region of its own: nothing overwrites a register whose store is being issued)
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, s[kk][e]), r, voff + e * D * 4,
                                              32 * kk * D * 4, kNT);
    asm volatile("s_nop 1");
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ void scale(float total) {
    if (total == 0.0f) {  // forgotten, whatever it held
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
        for (int e = 0; e < 8; ++e) s[kk][e] = f32x2_t{0.0f, 0.0f};
      return;
    }
#pragma unroll
    for (int kk = 0; kk < D / 32; ++kk)
#pragma unroll
      for (int e = 0; e < 8; ++e) s[kk][e] *= total;
  }
  // S += sum over count nodes of (w k)[row] u[column], both from LDS rows
  __device__ __forceinline__ void advance(int count, const float (&wk)[kPathRows][D], const float (&u)[kPathRows][D],
                                          int wave, int lr, int lg) {
    for (int p = 0; p < count; ++p) {
      const f32x2_t c = *reinterpret_cast<const f32x2_t*>(&u[p][32 * wave + 2 * lr]);
#pragma unroll
      for (int kk = 0; kk < D / 32; ++kk) {
        const float4 a = *reinterpret_cast<const float4*>(&wk[p][32 * kk + 8 * lg]);
        const float4 b = *reinterpret_cast<const float4*>(&wk[p][32 * kk + 8 * lg + 4]);
        const float r[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          s[kk][e].x = fmaf(r[e], c.x, s[kk][e].x);
          s[kk][e].y = fmaf(r[e], c.y, s[kk][e].y);
        }
      }
    }
  }
};

// A pending path in LDS: its nodes from the accepted one up to the root, the weight of
// each one's correction and that of the state.
struct Path {
  int node[kMaxNodes];
  float weight[kMaxNodes];
  float total;
  int count;  // 0: nothing was accepted
};

// By one wave, lane t with node t's parent and decay: the walk from the accepted node up,
// lane by lane in scalar registers.  What it reads comes as PathIn, so that it can be asked
// for ahead of the state.
struct PathIn {
  int64_t want;
  float g;
  int parent;

  __device__ __forceinline__ void load(const RulePending& pd, int b, int h, int Hv, int lane) {
    const int t = min(lane, pd.T - 1);
    want = pd.accepted[b];
    g = pd.g[(static_cast<int64_t>(b) * pd.T + t) * Hv + h];
    parent = pd.parents[b * pd.p_b + t];
  }
};
__device__ __forceinline__ float lane_f(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ void find_path(const PathIn& in, int T, int lane, Path& path) {
  const float dec = expf(in.g);
  int s = in.want >= 0 && in.want < T ? __builtin_amdgcn_readfirstlane(static_cast<int>(in.want)) : -1;
  int n = 0, node = 0;
  float w = 1.0f, weight = 0.0f;
  bool fine = s >= 0;
  while (s >= 0) {
    if (lane == n) {
      node = s;
      weight = w;
    }
    ++n;
    w *= lane_f(dec, s);
    const int p = __builtin_amdgcn_readlane(in.parent, s);
    fine = p >= -1 && p < s;  // (so that the walk ends; else node s is unused, and what follows it)
    s = fine ? p : -1;
  }
  if (lane < n) {
    path.node[lane] = node;
    path.weight[lane] = weight;
  }
  if (lane == 0) {
    path.total = w;
    path.count = fine ? n : 0;
  }
}

// Up to 16 rows of the path from the p0-th on into LDS, a wave per node: its normalised key
// times its weight, and its correction.
template <int D>
__device__ __forceinline__ void stage_path(const RulePending& pd, const Path& path, int first, int b, int h, int kh,
                                           int Hv, int wave, int waves, int lane, float (&wk)[kPathRows][D],
                                           float (&u)[kPathRows][D]) {
  typedef uint16_t halves __attribute__((ext_vector_type(D / 64)));
  typedef float floats __attribute__((ext_vector_type(D / 64)));
  constexpr int E = D / 64;
  const int rows = min(path.count - first, kPathRows);
  for (int p0 = wave; p0 < rows; p0 += 4 * waves) {
    halves kr[4];
    floats ur[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int s = path.node[first + min(p0 + i * waves, rows - 1)];
      kr[i] = *reinterpret_cast<const halves*>(pd.k + b * pd.k_b + s * pd.k_t + kh * D + lane * E);
      ur[i] = *reinterpret_cast<const floats*>(pd.u + ((static_cast<int64_t>(b) * pd.T + s) * Hv + h) * D + lane * E);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = p0 + i * waves;
      if (p >= rows) break;
      floats v;
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        v[e] = gdn::bf2f(kr[i][e]);
        ss = fmaf(v[e], v[e], ss);
      }
      const float weight = path.weight[first + p], norm = rsqrtf(gdn::wave_sum(ss) + kEps);
      const bool on = weight != 0.0f;
      *reinterpret_cast<floats*>(&u[p][lane * E]) = on ? ur[i] : floats(0.0f);
      *reinterpret_cast<floats*>(&wk[p][lane * E]) = on ? v * (weight * norm) : floats(0.0f);
    }
  }
}

// Three bf16 terms of two fp32 values that add up to them exactly: the leading 8 bits of
// the significand, the next 8, the last 8 (cut, not rounded), in the low and the high half.
__device__ __forceinline__ void split3(float a, float b, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  const uint32_t ua = __float_as_uint(a), ub = __float_as_uint(b);
  hi = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
  const float ra = a - __uint_as_float(ua & 0xffff0000u), rb = b - __uint_as_float(ub & 0xffff0000u);
  const uint32_t va = __float_as_uint(ra), vb = __float_as_uint(rb);
  mid = __builtin_amdgcn_perm(vb, va, 0x07060302u);
  const float sa = ra - __uint_as_float(va & 0xffff0000u), sb = rb - __uint_as_float(vb & 0xffff0000u);
  lo = __builtin_amdgcn_perm(__float_as_uint(sb), __float_as_uint(sa), 0x07060302u);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.4028234664e38f; }

// c += a b, 16 x 16 x 16 in fp32: a the lane's row lr, columns 4 lg .. + 3; b and c in the
// results' layout (register r of lane (lr, lg): row 4 lg + r, column lr).
__device__ __forceinline__ gdn::f32x4_t mul16(const gdn::f32x4_t& a, const gdn::f32x4_t& b, gdn::f32x4_t c) {
#pragma unroll
  for (int r = 0; r < 4; ++r) c = gdn::mfma16x16x4f32(a[r], b[r], c);
  return c;
}

// v added over N (8 or 16) neighbouring lanes
template <int kPerm>
__device__ __forceinline__ float lane_perm(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), kPerm, 15, 15, false));
}
template <int N>
__device__ __forceinline__ float row_sum(float v) {
  v += lane_perm<0xB1>(v);   // lane ^ 1
  v += lane_perm<0x4E>(v);   // lane ^ 2
  v += lane_perm<0x141>(v);  // the other half of 8
  if (N == 16) v += lane_perm<0x140>(v);
  return v;
}

__device__ __forceinline__ const gdn::f32x4_t& four(const float* p) { return *reinterpret_cast<const gdn::f32x4_t*>(p); }

// The layer around the rule: what the gates and the norm take and give.
struct TreeLayer {
  const uint16_t *b, *a;        // [B, T, Hv] contiguous
  const void *A_log, *dt_bias;  // [Hv]
  int param_f32;
  float* g;                     // out, [B, T, Hv]
  const uint16_t* z;            // [B, T, Hv D], strides z_b, z_t
  int64_t z_b, z_t;
  const uint16_t* w;            // [D]
  float eps;
  uint8_t* y8;                  // D = 128: [B, T, Hv, D] e4m3 in o's place (else NULL), with
  float* scale;                 // a scale per row, row i of head h at h M + i, M = B T
};

// NT: 16-node tiles of the tree.
template <int D, int NT, bool kLayer>
__global__ __launch_bounds__(2 * D, D == 128 ? (NT <= 2 ? 3 : 2) : NT == 1 ? 3 : NT == 2 ? 2 : 1) void rule_tree_kernel(
    const uint16_t* __restrict__ q, int64_t q_b, int64_t q_t, const uint16_t* __restrict__ k, int64_t k_b, int64_t k_t,
    const uint16_t* __restrict__ v, int64_t v_b, int64_t v_t, const float* __restrict__ g,
    const uint16_t* __restrict__ beta, float* __restrict__ pool, int64_t s_slot, int64_t n_slots,
    const int64_t* __restrict__ ids, const int32_t* __restrict__ parents, int64_t p_b, RulePending pd,
    uint16_t* __restrict__ o, float* __restrict__ u, int B, int T, int Hk, int Hv, float scale, TreeLayer L) {
  constexpr int NW = D / 32, KK = D / 32, TM = 16 * NT;
  // 16 x 16 tiles (I, J), J <= I, of a node t's row and an earlier node s's column
  constexpr int kTiles = NT * (NT + 1) / 2;
  auto tile = [](int I, int J) { return I * (I + 1) / 2 + J; };
  __shared__ __align__(16) float cu[kTiles][16][16];  // minus the coefficients of u_s in u_t
  __shared__ __align__(16) float co[kTiles][16][16];  // the coefficients of u_s in o_t
  __shared__ __align__(16) float inv[TM][16];         // the inverses of the 16-node triangles
  // The pending path's keys and corrections (and see the end).  With 64 nodes, where two
  // workgroups of a CU leave no room for both, in the weights' place once those are used.
  constexpr bool kShare = NT == 4;
  constexpr int kPathFloats = 2 * kPathRows * D;
  __shared__ __align__(16) float xbuf[kShare ? std::max(kPathFloats, 256 * kTiles) : kPathFloats];
  __shared__ __align__(16) float wbuf[kShare ? 4 : 256 * kTiles];
  float(*wt)[16][16] = reinterpret_cast<float(*)[16][16]>(kShare ? xbuf : wbuf);  // weights w(t, s)
  float(&xk)[kPathRows][D] = *reinterpret_cast<float(*)[kPathRows][D]>(xbuf);
  float(&xq)[kPathRows][D] = *reinterpret_cast<float(*)[kPathRows][D]>(xbuf + kPathRows * D);
  __shared__ __align__(16) int link[TM];
  __shared__ __align__(16) float bt[TM], total[TM], rk[TM], rq[TM];
  __shared__ __align__(16) float fv[TM], fk[TM], fq[TM];  // factors of v, S^T k, S^T q: 0 for an unused node
  __shared__ int any_cu[NT][NT];                // whether a tile of coefficients holds an ancestor
  __shared__ Path path;
  __shared__ __align__(16) uint16_t kq[2 * TM][D + 8];  // the nodes' keys, then their queries
  // (the layer's norm) a tile's outputs, two in turn, where the rows were
  uint16_t(*rows)[16][D + 8] = reinterpret_cast<uint16_t(*)[16][D + 8]>(&kq[0][0]);
  __shared__ int bad;                           // a correction is not finite

  const int64_t wi = gdn::xcd_remap(blockIdx.x, static_cast<int64_t>(B) * Hv);
  if (wi < 0) return;
  const int b = static_cast<int>(wi / Hv), h = static_cast<int>(wi % Hv), kh = h / (Hv / Hk);
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lr = lane & 15, lg = lane >> 4;
  const int col = 32 * wave + 2 * lr;                            // the lane's columns col, col + 1
  const int64_t out_t = static_cast<int64_t>(Hv) * D;
  const int64_t out0 = static_cast<int64_t>(b) * T * out_t + h * D;  // row t at out0 + t out_t
  const int64_t slot = ids[b];
  if (slot < 0 || slot >= n_slots) {  // (the whole workgroup)
    for (int t = tid / D; t < T; t += 2) {
      if (kLayer && L.y8) L.y8[out0 + t * out_t + tid % D] = 0;
      else o[out0 + t * out_t + tid % D] = 0;
      u[out0 + t * out_t + tid % D] = 0.0f;
    }
    if (kLayer && tid < T) {
      L.g[(static_cast<int64_t>(b) * T + tid) * Hv + h] = 0.0f;
      if (L.y8) L.scale[static_cast<int64_t>(h) * B * T + static_cast<int64_t>(b) * T + tid] = gdn::fp8_scale(0.0f);
    }
    return;
  }
  // Loads return in order: what the tree and the coefficients need goes out ahead of the
  // state, which is then on its way while they are worked on.
  const buf_t bk = buf_of(k + b * k_b + kh * D), bq = buf_of(q + b * q_b + kh * D);
  const buf_t bv = buf_of(v + b * v_b + static_cast<int64_t>(h) * D);
  const int k_row = static_cast<int>(k_t) * 2, q_row = static_cast<int>(q_t) * 2, v_row = static_cast<int>(v_t) * 2;
  int my_parent = 0;
  float my_g = 0.0f, my_beta = 0.0f, A_log = 0.0f, dt_bias = 0.0f;
  PathIn pin = {-1, 0.0f, 0};
  if (wave == 0) {
    const int64_t at = (static_cast<int64_t>(b) * T + min(lane, T - 1)) * Hv + h;
    // (with the layer: a and b as they are, until the loads are on their way)
    my_g = kLayer ? gdn::bf2f(L.a[at]) : g[at];
    my_beta = gdn::bf2f((kLayer ? L.b : beta)[at]);
    if (kLayer) {
      A_log = gdn::load_param(L.A_log, h, L.param_f32);
      dt_bias = gdn::load_param(L.dt_bias, h, L.param_f32);
    }
    my_parent = parents[b * p_b + min(lane, T - 1)];
  } else if (wave == 1 && pd.accepted) {
    pin.load(pd, b, h, Hv, lane);
  }
  // the nodes' rows, each once, 8 values per lane: the wave's share, keys first
  constexpr int kRowLanes = D / 8, kRowsPer = 64 / kRowLanes;
  const int rl = lane % kRowLanes, rr = wave * kRowsPer + lane / kRowLanes;  // of rows NW kRowsPer = 16
  gdn::s16x8_t raw[2 * NT];
#pragma unroll
  for (int p = 0; p < 2 * NT; ++p) {
    const int t = min(16 * (p % NT) + rr, T - 1);
    raw[p] = p < NT ? buf_row(bk, t * k_row + 16 * rl) : buf_row(bq, t * q_row + 16 * rl);
  }
  uint32_t vv[NT][4];  // rows 16 I + 4 lg + r, both columns
#pragma unroll
  for (int I = 0; I < NT; ++I)
#pragma unroll
    for (int r = 0; r < 4; ++r) 
      vv[I][r] = __builtin_amdgcn_raw_buffer_load_b32(bv, min(16 * I + 4 * lg + r, T - 1) * v_row + 2 * col, 0, 0);
  gdn::keep_loads_here();
  const buf_t bs = buf_of(pool + slot * s_slot + static_cast<int64_t>(h) * D * D);
  const int s_off = (8 * lg * D + col) * 4;
  Tile<D> S;
  S.load(bs, s_off);
  gdn::keep_loads_here();

  // --- the tree: lane t of wave 0 from node t up to the root; the pending path ---
  if (wave == 0) {
    for (int i = lane; i < 64 * kTiles; i += 64) reinterpret_cast<float4*>(wt)[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (kLayer) {
      my_g = gdn::gate_g(my_g, A_log, dt_bias);
      my_beta = gdn::bf2f(gdn::gate_beta(my_beta));
      if (lane < T) L.g[(static_cast<int64_t>(b) * T + lane) * Hv + h] = my_g;
      if (lane == 0) bad = 0;
    }
    const float dec = expf(my_g);
    bool fine = lane < T && my_parent >= -1 && my_parent < lane;
    int s = fine ? my_parent : -1;
    float w = dec;
    if (fine) wt[tile(lane >> 4, lane >> 4)][lane & 15][lane & 15] = 1.0f;
    while (__any(s >= 0)) {
      const int at = max(s, 0);
      const float d = __shfl(dec, at, 64);
      const int p = __shfl(my_parent, at, 64);
      if (s >= 0) {
        wt[tile(lane >> 4, s >> 4)][lane & 15][s & 15] = w;
        w *= d;
        fine = p >= -1 && p < s;  // (each step goes to an earlier node: the walk ends)
        s = fine ? p : -1;
      }
    }
    if (lane < TM) {
      link[lane] = fine ? my_parent : kUnused;
      bt[lane] = my_beta;
      total[lane] = w;
    }
  } else if (wave == 1 && pd.accepted) {
    find_path(pin, pd.T, lane, path);
  }
#pragma unroll
  for (int p = 0; p < 2 * NT; ++p) {
    const int t = 16 * (p % NT) + rr;
    *reinterpret_cast<gdn::s16x8_t*>(&kq[p < NT ? t : TM + t][8 * rl]) = raw[p];
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = gdn::bf2f(static_cast<uint16_t>(raw[p][e]));
      ss = fmaf(x, x, ss);
    }
    ss = row_sum<kRowLanes>(ss);
    if (rl == 0) (p < NT ? rk : rq)[t] = rsqrtf(ss + kEps);
  }
  gdn::lds_barrier();
  const bool pending = pd.accepted && path.count > 0;  // (the whole workgroup)
  if (pending && !kShare) stage_path<D>(pd, path, 0, b, h, kh, Hv, wave, NW, lane, xk, xq);
  if (tid < TM) {
    const bool on = link[tid] != kUnused;
    fv[tid] = on ? bt[tid] : 0.0f;
    fk[tid] = on ? -(bt[tid] * total[tid]) * rk[tid] : 0.0f;
    fq[tid] = on ? (scale * total[tid]) * rq[tid] : 0.0f;
  }

  // --- the nodes' products with each other: coefficients of u_s in u_t and in o_t ---
  // Tile (I, J), J <= I, of K K^T and of Q K^T: lane (lr, lg), register r: t = 16 I + 4 lg
  // + r, s = 16 J + lr.  A weight of 0 is not multiplied: nothing of an unused node, of
  // another branch or past T gets in.
  auto frag = [&](int row, int kk) { return *reinterpret_cast<const gdn::s16x8_t*>(&kq[row][32 * kk + 8 * lg]); };
  // of u_s in u_t, in o_t, or in both
  auto coefficients = [&](int I, int J, auto in_u, auto in_o) {
    gdn::f32x4_t c = {0.f, 0.f, 0.f, 0.f}, d = c;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      const gdn::s16x8_t key = frag(16 * J + lr, kk);
      if constexpr (in_u.value) c = gdn::mfma16x16x32(frag(16 * I + lr, kk), key, c);
      if constexpr (in_o.value) d = gdn::mfma16x16x32(frag(TM + 16 * I + lr, kk), key, d);
    }
    const int s = 16 * J + lr;
    const float rs = rk[s];
    bool some = false;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * I + 4 * lg + r;
      const float w = wt[tile(I, J)][4 * lg + r][lr];
      const bool on = w != 0.0f && link[t] != kUnused;
      if constexpr (in_o.value) co[tile(I, J)][4 * lg + r][lr] = on ? (scale * rq[t]) * (rs * w) * d[r] : 0.0f;
      if constexpr (in_u.value) {
        cu[tile(I, J)][4 * lg + r][lr] = on && s < t ? -(bt[t] * rk[t]) * (rs * w) * c[r] : 0.0f;
        some |= on && s < t;
      }
    }
    if constexpr (in_u.value) {
      some = __any(some);
      if (lane == 0) any_cu[I][J] = some;
    }
  };
  constexpr std::true_type yes;
  constexpr std::false_type no;
  // the inverse of a triangle by substitution: lane (lr, lg) rows 4 lg .. + 3 of its column lr;
  // four rows at a time are finished and handed to the later ones (in few registers: the state
  // is on its way into most of them)
  auto invert = [&](int I) {
    wave_lds_order();
    gdn::f32x4_t x;
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = 4 * lg + r == lr ? 1.0f : 0.0f;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      gdn::f32x4_t c[4], y = x;
#pragma unroll
      for (int r = 0; r < 4; ++r) c[r] = four(&cu[tile(I, I)][4 * lg + r][4 * p]);
      y[1] = fmaf(c[1][0], y[0], y[1]);
      y[2] = fmaf(c[2][1], y[1], fmaf(c[2][0], y[0], y[2]));
      y[3] = fmaf(c[3][2], y[2], fmaf(c[3][1], y[1], fmaf(c[3][0], y[0], y[3])));
      float z[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) z[e] = __shfl(y[e], 16 * p + lr, 64);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float n = x[r];
#pragma unroll
        for (int e = 0; e < 4; ++e) n = fmaf(c[r][e], z[e], n);
        x[r] = lg == p ? y[r] : n;
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) inv[16 * I + 4 * lg + r][lr] = x[r];
  };
  // a triangle and its inverse to one wave (from the last one on), the other tiles dealt out
  int turn = 0;
#pragma unroll 1
  for (int I = 0; I < NT; ++I) {
    if (wave == NW - 1 - I % NW) {
      coefficients(I, I, yes, no);
      invert(I);
    }
#pragma unroll 1
    for (int J = 0; J < I; ++J)
      if (turn++ % NW == wave) coefficients(I, J, yes, yes);
    if (turn++ % NW == wave) coefficients(I, I, no, yes);
  }

  // --- the state after the pending path; its products with the nodes' rows ---
  gdn::lds_barrier();
  if (pending) {
    S.scale(path.total);
    if (kShare) {
      stage_path<D>(pd, path, 0, b, h, kh, Hv, wave, NW, lane, xk, xq);
      gdn::lds_barrier();
    }
    S.advance(min(path.count, kPathRows), xk, xq, wave, lr, lg);
    for (int p = kPathRows; p < path.count; p += kPathRows) {
      gdn::lds_barrier();
      stage_path<D>(pd, path, p, b, h, kh, Hv, wave, NW, lane, xk, xq);
      gdn::lds_barrier();
      S.advance(min(path.count - p, kPathRows), xk, xq, wave, lr, lg);
    }
    S.store(bs, s_off);
    gdn::lds_barrier();  // the path's rows have been read
  }
  gdn::f32x4_t ak[NT][2], aq[NT][2];  // [node tile][even, odd columns]
#pragma unroll
  for (int I = 0; I < NT; ++I)
#pragma unroll
    for (int c = 0; c < 2; ++c) ak[I][c] = aq[I][c] = gdn::f32x4_t{0.f, 0.f, 0.f, 0.f};
  // What is written is dropped past the buffers' ends (rows past T): no branch, and the counts
  // by which a wave waits for its loads stay known (else it waits for its stores too).
  const int out_row = static_cast<int>(out_t), out_end = (T - 1) * out_row + D;
  const buf_t bu = buf_of(u + out0, 4 * out_end);
  const buf_t bo = kLayer && L.y8 ? buf_of(L.y8 + out0, out_end) : buf_of(o + out0, 2 * out_end);
  constexpr int kLanes = D / 8;  // of a row in the norm: 8 columns each
  const int row = tid / kLanes, c8 = tid % kLanes * 8;
  auto z_row = [&](int I) {
    return *reinterpret_cast<const uint4*>(L.z + b * L.z_b + min(16 * I + row, T - 1) * L.z_t +
                                           static_cast<int64_t>(h) * D + c8);
  };
  uint4 zv, wv;
  if constexpr (kLayer) {
    zv = z_row(0);
    wv = *reinterpret_cast<const uint4*>(L.w + c8);
  }
  // the gated norm of tile I's rows, as its own kernels take it
  auto norm_rows = [&](int I) {
    const int t = 16 * I + row;
    uint16_t xs[8], zs[8], ws[8];
    __builtin_memcpy(xs, &rows[I & 1][row][c8], 16);
    __builtin_memcpy(zs, &zv, 16);
    __builtin_memcpy(ws, &wv, 16);
    float v[8], ss = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = gdn::bf2f(xs[i]);
      ss += v[i] * v[i];
    }
#pragma unroll
    for (int m = kLanes / 2; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
    const float r = rsqrtf(ss / static_cast<float>(D) + L.eps);
    const bool on = link[t] != kUnused;
    const int at = t * out_row + c8;
    if (D == 128 && L.y8) {
      float top = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        v[i] = on ? v[i] * r * gdn::bf2f(ws[i]) * gdn::silu_ulp(gdn::bf2f(zs[i])) : 0.0f;
        top = fmaxf(top, fabsf(v[i]));
      }
#pragma unroll
      for (int m = 8; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
      const float s = gdn::fp8_scale(top), inv = 1.0f / s;
      const u32x2_t w8 = {gdn::f2fp8x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                          gdn::f2fp8x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv)};
      __builtin_amdgcn_raw_buffer_store_b64(w8, bo, at, 0, 0);
      const buf_t bs8 = buf_of(L.scale + (static_cast<int64_t>(h) * B + b) * T, 4 * T);
      __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(s), bs8, c8 == 0 ? 4 * t : 4 * kMaxNodes, 0, 0);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = on ? gdn::norm_gate(v[i], r, gdn::bf2f(ws[i]), gdn::bf2f(zs[i])) : 0.0f;
      const u32x4_t w16 = {gdn::f2bf2(v[0], v[1]), gdn::f2bf2(v[2], v[3]), gdn::f2bf2(v[4], v[5]),
                           gdn::f2bf2(v[6], v[7])};
      __builtin_amdgcn_raw_buffer_store_b128(w16, bo, 2 * at, 0, 0);
    }
  };
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) {
    u32x4_t f[2][3];
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t hi, mid, lo;
        split3(S.s[kk][2 * e][c], S.s[kk][2 * e + 1][c], hi, mid, lo);
        f[c][0][e] = hi;
        f[c][1][e] = mid;
        f[c][2][e] = lo;
      }
#pragma unroll
    for (int I = 0; I < NT; ++I) {
      const gdn::s16x8_t x = frag(16 * I + lr, kk), y = frag(TM + 16 * I + lr, kk);
#pragma unroll
      for (int n = 2; n >= 0; --n)  // (the smallest terms first)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          ak[I][c] = gdn::mfma16x16x32(x, __builtin_bit_cast(gdn::s16x8_t, f[c][n]), ak[I][c]);
          aq[I][c] = gdn::mfma16x16x32(y, __builtin_bit_cast(gdn::s16x8_t, f[c][n]), aq[I][c]);
        }
    }
  }

  // --- u and o, 16 nodes at a time ---
  if constexpr (kLayer) gdn::lds_barrier();  // the rows have been read
  gdn::f32x4_t uu[NT][2];
  bool fine = true;
#pragma unroll
  for (int I = 0; I < NT; ++I) {
    const gdn::f32x4_t xv = four(&fv[16 * I + 4 * lg]), xk4 = four(&fk[16 * I + 4 * lg]), xq4 = four(&fq[16 * I + 4 * lg]);
    gdn::f32x4_t rhs[2], out[2];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float x = __uint_as_float(c ? vv[I][r] & 0xffff0000u : vv[I][r] << 16);
        // (a factor of 0 keeps what its row holds out)
        rhs[c][r] = (xv[r] != 0.0f ? xv[r] * x : 0.0f) + (xk4[r] != 0.0f ? xk4[r] * ak[I][c][r] : 0.0f);
        out[c][r] = xq4[r] != 0.0f ? xq4[r] * aq[I][c][r] : 0.0f;
      }
#pragma unroll
    for (int J = 0; J < I; ++J) {
      if (!any_cu[I][J]) continue;
      const gdn::f32x4_t a = four(&cu[tile(I, J)][lr][4 * lg]), e = four(&co[tile(I, J)][lr][4 * lg]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        rhs[c] = mul16(a, uu[J][c], rhs[c]);
        out[c] = mul16(e, uu[J][c], out[c]);
      }
    }
    const gdn::f32x4_t a = four(&inv[16 * I + lr][4 * lg]), e = four(&co[tile(I, I)][lr][4 * lg]);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uu[I][c] = mul16(a, rhs[c], gdn::f32x4_t{0.f, 0.f, 0.f, 0.f});
      out[c] = mul16(e, uu[I][c], out[c]);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int t = 16 * I + 4 * lg + r;
      fine &= finite(uu[I][0][r]) && finite(uu[I][1][r]);
      const int at = t * out_row + col;
      __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2_t, f32x2_t{uu[I][0][r], uu[I][1][r]}), bu, 4 * at,
                                            0, 0);
      const uint32_t pair = gdn::f2bf2(out[0][r], out[1][r]);
      if constexpr (kLayer) *reinterpret_cast<uint32_t*>(&rows[I & 1][4 * lg + r][col]) = pair;
      else __builtin_amdgcn_raw_buffer_store_b32(pair, bo, 2 * at, 0, 0);
    }
    if constexpr (kLayer) {
      if (__any(!fine) && lane == 0) bad = 1;
      gdn::lds_barrier();
      const uint4 next = I + 1 < NT ? z_row(I + 1) : zv;
      norm_rows(I);
      zv = next;
    }
  }
  if constexpr (kLayer) {
    if (!bad) return;  // (the whole workgroup)
    gdn::lds_barrier();
  } else if (!__any(!fine)) {
    return;
  }

  // --- where a correction is not finite (an infinity or a NaN in a row or in the state): the
  // products above let it into every node of its column, coefficient 0 or not.  So the
  // wave's columns again, a column per lane, each node from its ancestors alone. ---
  const int mine = 32 * wave + (lane & 31);
#pragma unroll 1
  for (int I = 0; I < NT; ++I) {
#pragma unroll
    for (int J = 0; J < NT; ++J)
      if (J == I)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          *reinterpret_cast<f32x2_t*>(&xk[4 * lg + r][col]) = f32x2_t{ak[J][0][r], ak[J][1][r]};
          *reinterpret_cast<f32x2_t*>(&xq[4 * lg + r][col]) = f32x2_t{aq[J][0][r], aq[J][1][r]};
        }
    wave_lds_order();
#pragma unroll 1
    for (int t = 16 * I; t < min(T, 16 * I + 16); ++t) {
      float x = 0.0f, y = 0.0f;
      if (link[t] != kUnused) {
        if (fv[t] != 0.0f) x = fv[t] * gdn::bf2f(v[b * v_b + t * v_t + static_cast<int64_t>(h) * D + mine]);
        if (fk[t] != 0.0f) x += fk[t] * xk[t - 16 * I][mine];
        if (fq[t] != 0.0f) y = fq[t] * xq[t - 16 * I][mine];
        for (int s = link[t]; s >= 0; s = link[s]) {
          const float us = u[out0 + s * out_t + mine], a = cu[tile(I, s >> 4)][t & 15][s & 15],
                      e = co[tile(I, s >> 4)][t & 15][s & 15];
          if (a != 0.0f) x = fmaf(a, us, x);
          if (e != 0.0f) y = fmaf(e, us, y);
        }
        y = fmaf(co[tile(I, I)][t & 15][t & 15], x, y);
      }
      if (lane < 32) {
        u[out0 + t * out_t + mine] = x;
        if constexpr (kLayer) rows[I & 1][t - 16 * I][mine] = gdn::f2bf(y);
        else o[out0 + t * out_t + mine] = gdn::f2bf(y);
      }
    }
    wave_lds_order();
    if constexpr (kLayer) {
      gdn::lds_barrier();
      zv = z_row(I);
      norm_rows(I);
    }
  }
}

// ---- commit ----
// The first `states` workgroups: the state tiles, one each, as in the rule: read once, the
// path's rows 16 at a time through LDS, written once.  Then the taps, 8 channels per thread.
// 64 sequences of 32 heads of 128 51 us (5.6 TB/s, a large copy's rate), one 5.8.
template <int D>
__global__ __launch_bounds__(2 * D) void commit_tree_kernel(float* __restrict__ pool, int64_t s_slot,
                                                            uint16_t* __restrict__ cpool, int64_t sp_slot,
                                                            int64_t sp_ch, int64_t n_slots,
                                                            const int64_t* __restrict__ ids, RulePending pd,
                                                            ConvPending cd, int B, int Hk, int Hv, int C,
                                                            int states) {
  constexpr int NW = D / 32;
  __shared__ __align__(16) float wk[kPathRows][D];
  __shared__ __align__(16) float us[kPathRows][D];
  __shared__ Path path;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (static_cast<int>(blockIdx.x) >= states) {
    const int parts = (C + 16 * D - 1) / (16 * D);
    const int at = blockIdx.x - states, b = at / parts;
    const int64_t slot = ids[b];
    if (slot < 0 || slot >= n_slots) return;
    int link = cd.parents[b * cd.p_b + min(lane, cd.T - 1)], none = kUnused;
    tree_links(lane, cd.T, link, 0, none);
    const int a = accepted_node(cd.accepted[b], cd.T, link);
    if (a < 0) return;
    // (the path's rows while every lane, and with it every node's link, is there)
    const int r1 = row_before(a, link), r0 = row_before(r1, link);
    const int c0 = (at % parts * 2 * D + tid) * 8;
    if (c0 >= C) return;
    uint16_t* p = cpool + slot * sp_slot + c0 * sp_ch;
    const bool dense = dense_taps(cpool, sp_slot, sp_ch);
    Taps taps;
    taps.load(p, sp_ch, dense);
    taps.advance(cd, b, c0, a, r1, r0);
    taps.store(p, sp_ch, dense);
    return;
  }
  const int64_t wi = gdn::xcd_remap(blockIdx.x, static_cast<int64_t>(B) * Hv);
  if (wi < 0) return;
  const int b = static_cast<int>(wi / Hv), h = static_cast<int>(wi % Hv);
  const int lr = lane & 15, lg = lane >> 4;
  const int64_t slot = ids[b];
  if (slot < 0 || slot >= n_slots) return;
  const buf_t bs = buf_of(pool + slot * s_slot + static_cast<int64_t>(h) * D * D);
  const int s_off = (8 * lg * D + 32 * wave + 2 * lr) * 4;
  PathIn pin = {-1, 0.0f, 0};
  if (wave == 0) pin.load(pd, b, h, Hv, lane);
  gdn::keep_loads_here();
  Tile<D> S;
  S.load(bs, s_off);
  gdn::keep_loads_here();
  if (wave == 0) find_path(pin, pd.T, lane, path);
  gdn::lds_barrier();
  if (path.count == 0) return;  // (the whole workgroup)
  for (int p = 0; p < path.count; p += kPathRows) {
    if (p) gdn::lds_barrier();
    stage_path<D>(pd, path, p, b, h, h / (Hv / Hk), Hv, wave, NW, lane, wk, us);
    gdn::lds_barrier();
    if (p == 0) S.scale(path.total);
    S.advance(min(path.count - p, kPathRows), wk, us, wave, lr, lg);
  }
  S.store(bs, s_off);
}

bool rows_ok(const void* p, int64_t s_b, int64_t s_t, int width, int T) {
  // (kMaxNodes rows of below 2^24 values: 32-bit byte offsets)
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && s_b % 8 == 0 && s_t % 8 == 0 && s_t >= width &&
         s_t < (1 << 24) && s_b >= 0 && T >= 1 && T <= kMaxNodes;
}

struct RuleRows {
  const uint16_t* q;
  int64_t q_b, q_t;
  const uint16_t* k;
  int64_t k_b, k_t;
  const uint16_t* v;
  int64_t v_b, v_t;
};

int rule_check(const RuleRows& r, const float* s_pool, int64_t s_slot, int64_t n_slots, const int64_t* ids,
               const int32_t* parents, int64_t p_b, const RulePending& pd, const float* u, int B, int T, int Hk, int Hv,
               int D) {
  if (B < 0 || T < 0 || Hk <= 0 || Hv <= 0 || Hv % Hk || n_slots < 0) return GDN_ERR_INVALID_ARG;
  if (T > kMaxNodes || (pd.accepted && pd.T > kMaxNodes) || (D != 64 && D != 128)) return GDN_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return GDN_OK;
  if (!rows_ok(r.q, r.q_b, r.q_t, Hk * D, T) || !rows_ok(r.k, r.k_b, r.k_t, Hk * D, T) ||
      !rows_ok(r.v, r.v_b, r.v_t, Hv * D, T) || !s_pool || !ids || !parents || !u || p_b < 0 ||
      s_slot < static_cast<int64_t>(Hv) * D * D || s_slot % 4 || reinterpret_cast<uintptr_t>(s_pool) % 16 ||
      reinterpret_cast<uintptr_t>(u) % 16)
    return GDN_ERR_INVALID_ARG;
  if (pd.accepted && (!rows_ok(pd.k, pd.k_b, pd.k_t, Hk * D, pd.T) || !pd.g || !pd.u || !pd.parents || pd.p_b < 0 ||
                      reinterpret_cast<uintptr_t>(pd.u) % 16))
    return GDN_ERR_INVALID_ARG;
  // (Hv D below 2^23: 64 rows of u have 32-bit byte offsets)
  return static_cast<int64_t>(B) * Hv >= (1LL << 24) || static_cast<int64_t>(Hv) * D >= (1 << 23) ? GDN_ERR_UNSUPPORTED
                                                                                                   : GDN_OK;
}

template <bool kLayer>
int rule_launch(const RuleRows& r, const float* g, const uint16_t* beta, float* s_pool, int64_t s_slot, int64_t n_slots,
                const int64_t* ids, const int32_t* parents, int64_t p_b, const RulePending& pd, uint16_t* o, float* u,
                int B, int T, int Hk, int Hv, int D, float scale, const TreeLayer& layer, void* stream) {
  if (stream == GDN_CHECK_ONLY) return GDN_OK;
  const dim3 grid(static_cast<unsigned>(gdn::kNumXcd * ((B * Hv + gdn::kNumXcd - 1) / gdn::kNumXcd)));
  hipStream_t st = static_cast<hipStream_t>(stream);
#define GDN_RULE(DD, NT)                                                                                           \
  rule_tree_kernel<DD, NT, kLayer><<<grid, dim3(2 * DD), 0, st>>>(r.q, r.q_b, r.q_t, r.k, r.k_b, r.k_t, r.v, r.v_b,  \
                                                                  r.v_t, g, beta, s_pool, s_slot, n_slots, ids,      \
                                                                  parents, p_b, pd, o, u, B, T, Hk, Hv, scale, layer)
  if (D == 128)
    T <= 16 ? GDN_RULE(128, 1) : T <= 32 ? GDN_RULE(128, 2) : T <= 48 ? GDN_RULE(128, 3) : GDN_RULE(128, 4);
  else
    T <= 16 ? GDN_RULE(64, 1) : T <= 32 ? GDN_RULE(64, 2) : T <= 48 ? GDN_RULE(64, 3) : GDN_RULE(64, 4);
#undef GDN_RULE
  return gdn_launch_status();
}

}  // namespace

extern "C" int gdn_conv_tree(const uint16_t* x, int64_t x_b, int64_t x_t, uint16_t* pool, int64_t sp_slot,
                             int64_t sp_ch, int64_t n_slots, const int64_t* ids, const uint16_t* w,
                             const int32_t* parents, int64_t p_b, const uint16_t* last_x, int64_t lx_b, int64_t lx_t,
                             const int32_t* last_parents, int64_t lp_b, const int64_t* accepted, int last_T,
                             uint16_t* y, int B, int T, int C, void* stream) {
  if (B < 0 || T < 0 || C <= 0 || n_slots < 0) return GDN_ERR_INVALID_ARG;
  if (T > kMaxNodes || (accepted && last_T > kMaxNodes) || C % 8 || C >= 1 << 23) return GDN_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return GDN_OK;
  if (!rows_ok(x, x_b, x_t, C, T) || !pool || !ids || !w || !parents || !y || p_b < 0 || sp_ch < 3 ||
      sp_slot < static_cast<int64_t>(C - 1) * sp_ch + 3 || reinterpret_cast<uintptr_t>(w) % 16 ||
      reinterpret_cast<uintptr_t>(y) % 16)
    return GDN_ERR_INVALID_ARG;
  if (accepted && (!rows_ok(last_x, lx_b, lx_t, C, last_T) || !last_parents || lp_b < 0)) return GDN_ERR_INVALID_ARG;
  if (B > 65535) return GDN_ERR_UNSUPPORTED;
  if (stream == GDN_CHECK_ONLY) return GDN_OK;
  const ConvPending pd{last_x, lx_b, lx_t, last_parents, lp_b, accepted, last_T};
  const dim3 grid((C + 127) / 128, B);
  const int lds = ((T + 3) / 4 * 4 + 3) * 256;
  hipStream_t st = static_cast<hipStream_t>(stream);
  // Up to six workgroups per CU and more than one group of nodes: 1 x 8 3.9 us (one wave 4.2), 1 x
  // 64 5.5 (11.7), 8 x 64 7.4 (13.1), 16 x 16 5.6 (6.0); 1 x 4 3.8 against 3.6, 32 x 16 8.0 against
  // 7.4, 64 x 16 12.8 against 11.2 (8192 channels).
  if (T > 4 && static_cast<int64_t>(B) * ((C + 127) / 128) <= 6 * gdn::kNumCu)
    conv_tree_kernel<4><<<grid, dim3(256), lds, st>>>(x, x_b, x_t, pool, sp_slot, sp_ch, n_slots, ids, w, parents, p_b, pd,
                                                     y, T, C);
  else
    conv_tree_kernel<1><<<grid, dim3(64), lds, st>>>(x, x_b, x_t, pool, sp_slot, sp_ch, n_slots, ids, w, parents, p_b, pd,
                                                    y, T, C);
  return gdn_launch_status();
}

extern "C" int gdn_rule_tree(const uint16_t* q, int64_t q_b, int64_t q_t, const uint16_t* k, int64_t k_b, int64_t k_t,
                             const uint16_t* v, int64_t v_b, int64_t v_t, const float* g, const uint16_t* beta,
                             float* s_pool, int64_t s_slot, int64_t n_slots, const int64_t* ids,
                             const int32_t* parents, int64_t p_b, const uint16_t* last_k, int64_t lk_b, int64_t lk_t,
                             const float* last_g, const float* last_u, const int32_t* last_parents, int64_t lp_b,
                             const int64_t* accepted, int last_T, uint16_t* o, float* u, int B, int T, int Hk, int Hv,
                             int D, float scale, void* stream) {
  const RulePending pd{last_k, lk_b, lk_t, last_g, last_u, last_parents, lp_b, accepted, last_T};
  const RuleRows r{q, q_b, q_t, k, k_b, k_t, v, v_b, v_t};
  const int rc = rule_check(r, s_pool, s_slot, n_slots, ids, parents, p_b, pd, u, B, T, Hk, Hv, D);
  if (rc != GDN_OK || B == 0 || T == 0) return rc;
  if (!g || !beta || !o || reinterpret_cast<uintptr_t>(o) % 16) return GDN_ERR_INVALID_ARG;
  return rule_launch<false>(r, g, beta, s_pool, s_slot, n_slots, ids, parents, p_b, pd, o, u, B, T, Hk, Hv, D, scale,
                            TreeLayer{}, stream);
}

extern "C" int gdn_rule_tree_layer(const uint16_t* q, int64_t q_b, int64_t q_t, const uint16_t* k, int64_t k_b,
                                   int64_t k_t, const uint16_t* v, int64_t v_b, int64_t v_t, const uint16_t* b,
                                   const uint16_t* a, const void* A_log, const void* dt_bias, int param_is_fp32,
                                   float* s_pool, int64_t s_slot, int64_t n_slots, const int64_t* ids,
                                   const int32_t* parents, int64_t p_b, const uint16_t* last_k, int64_t lk_b,
                                   int64_t lk_t, const float* last_g, const float* last_u, const int32_t* last_parents,
                                   int64_t lp_b, const int64_t* accepted, int last_T, const uint16_t* z, int64_t z_b,
                                   int64_t z_t, const uint16_t* w, float eps, uint16_t* y, uint8_t* y8, float* y8_scale,
                                   float* u, float* g, int B, int T, int Hk, int Hv, int D, float scale, void* stream) {
  const RulePending pd{last_k, lk_b, lk_t, last_g, last_u, last_parents, lp_b, accepted, last_T};
  const RuleRows r{q, q_b, q_t, k, k_b, k_t, v, v_b, v_t};
  const int rc = rule_check(r, s_pool, s_slot, n_slots, ids, parents, p_b, pd, u, B, T, Hk, Hv, D);
  if (rc != GDN_OK || B == 0 || T == 0) return rc;
  if (!rows_ok(z, z_b, z_t, Hv * D, T) || !b || !a || !A_log || !dt_bias || !w || !g || (!y == !y8) ||
      reinterpret_cast<uintptr_t>(w) % 16 || reinterpret_cast<uintptr_t>(y) % 16 ||
      reinterpret_cast<uintptr_t>(y8) % 16 || (y8 && !y8_scale))
    return GDN_ERR_INVALID_ARG;
  if (y8 && D != gdn::kFp8Group) return GDN_ERR_UNSUPPORTED;  // a head per scale
  const TreeLayer layer{b, a, A_log, dt_bias, param_is_fp32 ? 1 : 0, g, z, z_b, z_t, w, eps, y8, y8_scale};
  return rule_launch<true>(r, nullptr, nullptr, s_pool, s_slot, n_slots, ids, parents, p_b, pd, y, u, B, T, Hk, Hv, D,
                           scale, layer, stream);
}

extern "C" int gdn_commit_tree(float* s_pool, int64_t s_slot, uint16_t* conv_pool, int64_t sp_slot, int64_t sp_ch,
                               int64_t n_slots, const int64_t* ids, const int32_t* parents, int64_t p_b,
                               const int64_t* accepted, const uint16_t* x, int64_t x_b, int64_t x_t, const uint16_t* k,
                               int64_t k_b, int64_t k_t, const float* g, const float* u, int B, int T, int Hk, int Hv,
                               int D, int C, void* stream) {
  if (B < 0 || T < 0 || Hk <= 0 || Hv <= 0 || Hv % Hk || C <= 0 || n_slots < 0) return GDN_ERR_INVALID_ARG;
  if (T > kMaxNodes || (D != 64 && D != 128) || C % 8) return GDN_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return GDN_OK;
  if (!s_pool || !conv_pool || !ids || !parents || !accepted || p_b < 0 || !g || !u || !rows_ok(x, x_b, x_t, C, T) ||
      !rows_ok(k, k_b, k_t, Hk * D, T) || s_slot < static_cast<int64_t>(Hv) * D * D || s_slot % 4 ||
      reinterpret_cast<uintptr_t>(s_pool) % 16 || sp_ch < 3 || sp_slot < static_cast<int64_t>(C - 1) * sp_ch + 3 ||
      reinterpret_cast<uintptr_t>(u) % 16)
    return GDN_ERR_INVALID_ARG;
  if (static_cast<int64_t>(B) * (Hv + (C + D - 1) / D) >= (1LL << 24)) return GDN_ERR_UNSUPPORTED;
  if (stream == GDN_CHECK_ONLY) return GDN_OK;
  const RulePending pd{k, k_b, k_t, g, u, parents, p_b, accepted, T};
  const ConvPending cd{x, x_b, x_t, parents, p_b, accepted, T};
  // (the conv workgroups after the states')
  const int states = gdn::kNumXcd * ((B * Hv + gdn::kNumXcd - 1) / gdn::kNumXcd);
  const dim3 grid(static_cast<unsigned>(states + B * ((C + 8 * 2 * D - 1) / (8 * 2 * D))));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (D == 128)
    commit_tree_kernel<128><<<grid, dim3(256), 0, st>>>(s_pool, s_slot, conv_pool, sp_slot, sp_ch, n_slots, ids, pd, cd,
                                                        B, Hk, Hv, C, states);
  else
    commit_tree_kernel<64><<<grid, dim3(128), 0, st>>>(s_pool, s_slot, conv_pool, sp_slot, sp_ch, n_slots, ids, pd, cd,
                                                       B, Hk, Hv, C, states);
  return gdn_launch_status();
}
