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
// differences of sums: no cancellation, and a decay of 0 stays 0.
#include "gdn_common.h"

namespace {

constexpr int kMaxNodes = 64;

// A tree's links, by the 64 lanes of one wave: link[t] the parent (-1: the state),
// or kUnused.  (Each walk goes to smaller nodes, so it ends.)
constexpr int kUnused = -2;
__device__ __forceinline__ void tree_links(const int32_t* __restrict__ parents, int T, int lane, int* raw, int* link) {
  if (lane < T) raw[lane] = parents[lane];
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
  if (lane < T) {
    int n = lane;
    while (n >= 0) {
      const int p = raw[n];
      n = p >= -1 && p < n ? p : kUnused;
    }
    link[lane] = n == -1 ? raw[lane] : kUnused;
  }
}

// The accepted node of a row, or -1: nothing was accepted.
__device__ __forceinline__ int accepted_node(int64_t a, int T, const int* link) {
  return a >= 0 && a < T && link[a] != kUnused ? static_cast<int>(a) : -1;
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

// ---- conv ----
// The row before row r of a tree: r >= 0 a node, -1, -2, -3 the taps from the newest.
__device__ __forceinline__ int row_before(int r, const int* link) { return r >= 0 ? link[r] : r - 1; }

// The taps of channel c after the accepted node: rows a, its parent and its grandparent.
__device__ __forceinline__ void advance_taps(uint16_t (&tap)[3], const ConvPending& pd, int b, int c, int a,
                                             const int* link) {
  uint16_t now[3];
  int r = a;
#pragma unroll
  for (int j = 2; j >= 0; --j) {
    now[j] = r >= 0 ? pd.x[b * pd.x_b + r * pd.x_t + c] : r == -1 ? tap[2] : r == -2 ? tap[1] : tap[0];
    r = row_before(r, link);
  }
#pragma unroll
  for (int j = 0; j < 3; ++j) tap[j] = now[j];
}

// grid (ceil(C / 256), B): a channel per thread
__global__ __launch_bounds__(256) void conv_tree_kernel(const uint16_t* __restrict__ x, int64_t x_b, int64_t x_t,
                                                        uint16_t* __restrict__ pool, int64_t sp_slot, int64_t sp_ch,
                                                        int64_t n_slots, const int64_t* __restrict__ ids,
                                                        const uint16_t* __restrict__ w,
                                                        const int32_t* __restrict__ parents, int64_t p_b,
                                                        ConvPending pd, uint16_t* __restrict__ y, int T, int C) {
  __shared__ int raw[2][kMaxNodes], link[2][kMaxNodes];
  const int b = blockIdx.y;
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (threadIdx.x < 64) {
    tree_links(parents + b * p_b, T, threadIdx.x, raw[0], link[0]);
  } else if (threadIdx.x < 128 && pd.accepted) {
    tree_links(pd.parents + b * pd.p_b, pd.T, threadIdx.x - 64, raw[1], link[1]);
  }
  __syncthreads();
  if (c >= C) return;
  const int64_t slot = ids[b];
  const bool row_ok = slot >= 0 && slot < n_slots;
  uint16_t tap[3] = {0, 0, 0};
  if (row_ok) {
    uint16_t* p = pool + slot * sp_slot + c * sp_ch;
#pragma unroll
    for (int j = 0; j < 3; ++j) tap[j] = p[j];
    const int a = pd.accepted ? accepted_node(pd.accepted[b], pd.T, link[1]) : -1;
    if (a >= 0) {
      advance_taps(tap, pd, b, c, a, link[1]);
#pragma unroll
      for (int j = 0; j < 3; ++j) p[j] = tap[j];
    }
  }
  float wk[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) wk[j] = gdn::bf2f(w[c * 4 + j]);
  for (int t = 0; t < T; ++t) {
    uint16_t out = 0;
    if (row_ok && link[0][t] != kUnused) {
      float s[3];
      int r = t;
#pragma unroll
      for (int j = 2; j >= 0; --j) {
        r = row_before(r, link[0]);
        s[j] = gdn::bf2f(r >= 0 ? x[b * x_b + r * x_t + c] : r == -1 ? tap[2] : r == -2 ? tap[1] : tap[0]);
      }
      out = gdn::f2bf(gdn::conv_decode_silu(gdn::bf2f(x[b * x_b + t * x_t + c]), s[0], s[1], s[2], wk));
    }
    y[(static_cast<int64_t>(b) * T + t) * C + c] = out;
  }
}

// ---- rule ----
// The path to an accepted node, newest first: its nodes and the weight w(a, s) of each
// one's correction; returns the weight of the state, W_a.  One thread.
__device__ __forceinline__ float path_of(int a, const int* link, const float* __restrict__ g, int64_t g_t, int* node,
                                         float* weight, int& n) {
  float w = 1.0f;
  n = 0;
  for (int s = a; s >= 0; s = link[s]) {
    node[n] = s;
    weight[n++] = w;
    w *= expf(g[s * g_t]);
  }
  return w;
}

// 1 / |row| of a bf16 row of D values for each lane of a wave (lane holds D / 64 values)
template <int D>
__device__ __forceinline__ void unit_row(const uint16_t* __restrict__ p, int lane, float* out) {
  constexpr int E = D / 64;
  float v[E], ss = 0.0f;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    v[e] = gdn::bf2f(p[lane * E + e]);
    ss += v[e] * v[e];
  }
  const float r = rsqrtf(gdn::wave_sum(ss) + 1e-6f);
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane * E + e] = v[e] * r;
}

// The column of S that a thread holds, after the pending path of row b (value head h).
template <int D>
__device__ __forceinline__ bool advance_column(float (&S)[D], const RulePending& pd, int b, int h, int kh, int Hv,
                                               const int* link, int* node, float* weight, float* total, int* count,
                                               float* key) {
  const int a = accepted_node(pd.accepted[b], pd.T, link);
  if (a < 0) return false;  // (the whole workgroup)
  if (threadIdx.x == 0) {
    int n;
    *total = path_of(a, link, pd.g + (static_cast<int64_t>(b) * pd.T) * Hv + h, Hv, node, weight, n);
    *count = n;
  }
  __syncthreads();
  const float w = *total;
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] *= w;
  for (int p = 0; p < *count; ++p) {
    const int s = node[p];
    __syncthreads();
    if (threadIdx.x < 64) unit_row<D>(pd.k + b * pd.k_b + s * pd.k_t + kh * D, threadIdx.x, key);
    __syncthreads();
    const float c = weight[p] * pd.u[((static_cast<int64_t>(b) * pd.T + s) * Hv + h) * D + threadIdx.x];
#pragma unroll
    for (int i = 0; i < D; ++i) S[i] = fmaf(c, key[i], S[i]);
  }
  return true;
}

// One workgroup of D threads per (sequence, value head); a thread holds a column of S.
template <int D>
__global__ __launch_bounds__(D) void rule_tree_kernel(const uint16_t* __restrict__ q, int64_t q_b, int64_t q_t,
                                                      const uint16_t* __restrict__ k, int64_t k_b, int64_t k_t,
                                                      const uint16_t* __restrict__ v, int64_t v_b, int64_t v_t,
                                                      const float* __restrict__ g, const uint16_t* __restrict__ beta,
                                                      float* __restrict__ pool, int64_t s_slot, int64_t n_slots,
                                                      const int64_t* __restrict__ ids,
                                                      const int32_t* __restrict__ parents, int64_t p_b,
                                                      RulePending pd, uint16_t* __restrict__ o, float* __restrict__ u,
                                                      int T, int Hk, int Hv, float scale) {
  __shared__ int raw[2][kMaxNodes], link[2][kMaxNodes], node[kMaxNodes];
  __shared__ float weight[kMaxNodes], dec[kMaxNodes], bt[kMaxNodes];
  __shared__ float key[D], qry[D], su[kMaxNodes][D], sk[kMaxNodes][D];
  __shared__ float total, kk[kMaxNodes], qk[kMaxNodes];
  __shared__ int count;
  const int b = blockIdx.x / Hv, h = blockIdx.x % Hv, kh = h / (Hv / Hk);
  const int j = threadIdx.x, wave = threadIdx.x / 64, lane = threadIdx.x % 64;
  const int64_t slot = ids[b];
  const bool row_ok = slot >= 0 && slot < n_slots;
  if (j < 64) {
    tree_links(parents + b * p_b, T, lane, raw[0], link[0]);
    if (pd.accepted) tree_links(pd.parents + b * pd.p_b, pd.T, lane, raw[1], link[1]);
    if (lane < T) {
      const int64_t at = (static_cast<int64_t>(b) * T + lane) * Hv + h;
      dec[lane] = expf(g[at]);
      bt[lane] = gdn::bf2f(beta[at]);
    }
  }
  for (int t = wave; t < T; t += D / 64) unit_row<D>(k + b * k_b + t * k_t + kh * D, lane, sk[t]);
  __syncthreads();
  float* S0 = pool + slot * s_slot + static_cast<int64_t>(h) * D * D + j;
  float S[D];
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] = row_ok ? S0[i * D] : 0.0f;
  if (pd.accepted && row_ok &&
      advance_column<D>(S, pd, b, h, kh, Hv, link[1], node, weight, &total, &count, key)) {
#pragma unroll
    for (int i = 0; i < D; ++i) S0[i * D] = S[i];
  }
  for (int t = 0; t < T; ++t) {
    const int64_t at = ((static_cast<int64_t>(b) * T + t) * Hv + h) * D + j;
    if (!row_ok || link[0][t] == kUnused) {  // (the whole workgroup)
      o[at] = 0;
      u[at] = 0.0f;
      continue;
    }
    __syncthreads();
    if (wave == 0) unit_row<D>(q + b * q_b + t * q_t + kh * D, lane, qry);
    __syncthreads();
    // the products with the path's keys: a wave per node
    if (j < 64) {
      for (int s = t; s >= 0; s = link[0][s]) {
        float a = 0.0f, c = 0.0f;
#pragma unroll
        for (int e = 0; e < D / 64; ++e) {
          a += sk[s][lane + 64 * e] * sk[t][lane + 64 * e];
          c += sk[s][lane + 64 * e] * qry[lane + 64 * e];
        }
        a = gdn::wave_sum(a);
        c = gdn::wave_sum(c);
        if (lane == 0) {
          kk[s] = a;
          qk[s] = c;
        }
      }
    }
    __syncthreads();
    float ks = 0.0f, qs = 0.0f;
#pragma unroll
    for (int i = 0; i < D; ++i) {
      ks = fmaf(sk[t][i], S[i], ks);
      qs = fmaf(qry[i], S[i], qs);
    }
    float w = dec[t], au = 0.0f, ao = 0.0f;
    for (int s = link[0][t]; s >= 0; s = link[0][s]) {
      au = fmaf(w * kk[s], su[s][j], au);
      ao = fmaf(w * qk[s], su[s][j], ao);
      w *= dec[s];
    }
    const float ut = bt[t] * (gdn::bf2f(v[b * v_b + t * v_t + h * D + j]) - fmaf(w, ks, au));
    su[t][j] = ut;
    u[at] = ut;
    o[at] = gdn::f2bf(scale * (fmaf(w, qs, ao) + qk[t] * ut));
  }
}

// Grid: B * Hv workgroups for the states, then B * ceil(C / D) for the taps.
template <int D>
__global__ __launch_bounds__(D) void commit_tree_kernel(float* __restrict__ pool, int64_t s_slot,
                                                        uint16_t* __restrict__ cpool, int64_t sp_slot, int64_t sp_ch,
                                                        int64_t n_slots, const int64_t* __restrict__ ids,
                                                        RulePending pd, ConvPending cd, int B, int Hk, int Hv, int C) {
  __shared__ int raw[kMaxNodes], link[kMaxNodes], node[kMaxNodes];
  __shared__ float weight[kMaxNodes], key[D], total;
  __shared__ int count;
  const int parts = (C + D - 1) / D;
  const bool conv = blockIdx.x >= static_cast<unsigned>(B * Hv);
  const int at = conv ? blockIdx.x - B * Hv : blockIdx.x;
  const int b = conv ? at / parts : at / Hv;
  const int64_t slot = ids[b];
  if (slot < 0 || slot >= n_slots) return;
  if (threadIdx.x < 64) tree_links(pd.parents + b * pd.p_b, pd.T, threadIdx.x, raw, link);
  __syncthreads();
  if (conv) {
    const int c = at % parts * D + threadIdx.x;
    const int a = accepted_node(cd.accepted[b], cd.T, link);
    if (c >= C || a < 0) return;
    uint16_t* p = cpool + slot * sp_slot + c * sp_ch;
    uint16_t tap[3];
#pragma unroll
    for (int j = 0; j < 3; ++j) tap[j] = p[j];
    advance_taps(tap, cd, b, c, a, link);
#pragma unroll
    for (int j = 0; j < 3; ++j) p[j] = tap[j];
    return;
  }
  const int h = at % Hv;
  float* S0 = pool + slot * s_slot + static_cast<int64_t>(h) * D * D + threadIdx.x;
  float S[D];
#pragma unroll
  for (int i = 0; i < D; ++i) S[i] = S0[i * D];
  if (advance_column<D>(S, pd, b, h, h / (Hv / Hk), Hv, link, node, weight, &total, &count, key)) {
#pragma unroll
    for (int i = 0; i < D; ++i) S0[i * D] = S[i];
  }
}

bool rows_ok(const void* p, int64_t s_b, int64_t s_t, int width, int T) {
  return p && reinterpret_cast<uintptr_t>(p) % 16 == 0 && s_b % 8 == 0 && s_t % 8 == 0 && s_t >= width && s_b >= 0 &&
         T >= 1 && T <= kMaxNodes;
}

}  // namespace

extern "C" int gdn_conv_tree(const uint16_t* x, int64_t x_b, int64_t x_t, uint16_t* pool, int64_t sp_slot,
                             int64_t sp_ch, int64_t n_slots, const int64_t* ids, const uint16_t* w,
                             const int32_t* parents, int64_t p_b, const uint16_t* last_x, int64_t lx_b, int64_t lx_t,
                             const int32_t* last_parents, int64_t lp_b, const int64_t* accepted, int last_T,
                             uint16_t* y, int B, int T, int C, void* stream) {
  if (B < 0 || T < 0 || C <= 0 || n_slots < 0) return GDN_ERR_INVALID_ARG;
  if (T > kMaxNodes || (accepted && last_T > kMaxNodes) || C % 8) return GDN_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return GDN_OK;
  if (!rows_ok(x, x_b, x_t, C, T) || !pool || !ids || !w || !parents || !y || p_b < 0 || sp_ch < 3 ||
      sp_slot < static_cast<int64_t>(C - 1) * sp_ch + 3 || reinterpret_cast<uintptr_t>(w) % 16 ||
      reinterpret_cast<uintptr_t>(y) % 16)
    return GDN_ERR_INVALID_ARG;
  if (accepted && (!rows_ok(last_x, lx_b, lx_t, C, last_T) || !last_parents || lp_b < 0)) return GDN_ERR_INVALID_ARG;
  if (B > 65535) return GDN_ERR_UNSUPPORTED;
  const ConvPending pd{last_x, lx_b, lx_t, last_parents, lp_b, accepted, last_T};
  conv_tree_kernel<<<dim3((C + 255) / 256, B), dim3(256), 0, static_cast<hipStream_t>(stream)>>>(
      x, x_b, x_t, pool, sp_slot, sp_ch, n_slots, ids, w, parents, p_b, pd, y, T, C);
  return gdn_launch_status();
}

extern "C" int gdn_rule_tree(const uint16_t* q, int64_t q_b, int64_t q_t, const uint16_t* k, int64_t k_b, int64_t k_t,
                             const uint16_t* v, int64_t v_b, int64_t v_t, const float* g, const uint16_t* beta,
                             float* s_pool, int64_t s_slot, int64_t n_slots, const int64_t* ids,
                             const int32_t* parents, int64_t p_b, const uint16_t* last_k, int64_t lk_b, int64_t lk_t,
                             const float* last_g, const float* last_u, const int32_t* last_parents, int64_t lp_b,
                             const int64_t* accepted, int last_T, uint16_t* o, float* u, int B, int T, int Hk, int Hv,
                             int D, float scale, void* stream) {
  if (B < 0 || T < 0 || Hk <= 0 || Hv <= 0 || Hv % Hk || n_slots < 0) return GDN_ERR_INVALID_ARG;
  if (T > kMaxNodes || (accepted && last_T > kMaxNodes) || (D != 64 && D != 128)) return GDN_ERR_UNSUPPORTED;
  if (B == 0 || T == 0) return GDN_OK;
  if (!rows_ok(q, q_b, q_t, Hk * D, T) || !rows_ok(k, k_b, k_t, Hk * D, T) || !rows_ok(v, v_b, v_t, Hv * D, T) || !g ||
      !beta || !s_pool || !ids || !parents || !o || !u || p_b < 0 || s_slot < static_cast<int64_t>(Hv) * D * D ||
      s_slot % 4 || reinterpret_cast<uintptr_t>(s_pool) % 16 || reinterpret_cast<uintptr_t>(o) % 16 ||
      reinterpret_cast<uintptr_t>(u) % 16)
    return GDN_ERR_INVALID_ARG;
  if (accepted && (!rows_ok(last_k, lk_b, lk_t, Hk * D, last_T) || !last_g || !last_u || !last_parents || lp_b < 0 ||
                   reinterpret_cast<uintptr_t>(last_u) % 16))
    return GDN_ERR_INVALID_ARG;
  if (static_cast<int64_t>(B) * Hv >= (1LL << 24)) return GDN_ERR_UNSUPPORTED;
  const RulePending pd{last_k, lk_b, lk_t, last_g, last_u, last_parents, lp_b, accepted, last_T};
  const dim3 grid(static_cast<unsigned>(B * Hv));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (D == 128)
    rule_tree_kernel<128><<<grid, dim3(128), 0, st>>>(q, q_b, q_t, k, k_b, k_t, v, v_b, v_t, g, beta, s_pool, s_slot,
                                                      n_slots, ids, parents, p_b, pd, o, u, T, Hk, Hv, scale);
  else
    rule_tree_kernel<64><<<grid, dim3(64), 0, st>>>(q, q_b, q_t, k, k_b, k_t, v, v_b, v_t, g, beta, s_pool, s_slot,
                                                    n_slots, ids, parents, p_b, pd, o, u, T, Hk, Hv, scale);
  return gdn_launch_status();
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
  const RulePending pd{k, k_b, k_t, g, u, parents, p_b, accepted, T};
  const ConvPending cd{x, x_b, x_t, parents, p_b, accepted, T};
  const dim3 grid(static_cast<unsigned>(B * (Hv + (C + D - 1) / D)));
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (D == 128)
    commit_tree_kernel<128><<<grid, dim3(128), 0, st>>>(s_pool, s_slot, conv_pool, sp_slot, sp_ch, n_slots, ids, pd,
                                                        cd, B, Hk, Hv, C);
  else
    commit_tree_kernel<64><<<grid, dim3(64), 0, st>>>(s_pool, s_slot, conv_pool, sp_slot, sp_ch, n_slots, ids, pd, cd,
                                                      B, Hk, Hv, C);
  return gdn_launch_status();
}
