// The residual stream between two blocks: the stream takes a block's output, and the next
// block reads the stream's RMSNorm (the decoder layer's norms, nanovllm/models/qwen3_5.py:99-118,
// :674-689; the norm behind a block, its gate and the scales are other models').
//
//   h = x                                                     the block's output
//   h = h rsqrt(mean(h^2) + eps) (offset + post_w)            where the block has a norm behind it
//   h = h gate, or h sigmoid(gate)                            per row, column or value
//   r = residual + scale h                                    the stream; scale h without a residual
//   y = r rsqrt(mean(r^2) + eps) (offset + w)                 in bf16, in e4m3 (gdn::fp8_scale), or both
//
// All of it in fp32 from the inputs' values; r is rounded once, to the stream's type, and y
// is formed from the r that was not rounded (as the reference forms it), so that y has one
// rounding.
#include <algorithm>
#include <type_traits>

#include "gdn_common.h"

namespace {

struct NormArgs {
  const uint16_t* x;
  int64_t sx;
  const void* residual;  // NULL: none
  int64_t sr;
  const void* w;
  const void* post_w;    // NULL: none
  const void* gate;      // NULL: none
  int64_t g_row, g_col;
  void* stream;          // r, dense; NULL: not written
  uint16_t* y;           // dense; NULL: not written
  uint8_t* y8;           // dense (kFp8)
  float* y8_scale;
  int64_t ss_row, ss_grp;
  int64_t M;
  int H;
  int stream_f32, w_f32, gate_f32, gate_sigmoid;
  float offset, scale, eps;
};

// 1 / (1 + e^-g): the hardware reciprocal and one Newton step; 0 below -88, where it is less
// than 2^-126.  The exponent is capped on both sides: exp_acc makes a NaN of one whose product with log2(e) is
// infinite, and past 88 e^-g adds nothing to 1.
__device__ __forceinline__ float sigmoid_ulp(float g) {
  const float d = 1.0f + gdn::exp_acc(fmaxf(fminf(0.0f - g, 88.0f), -88.0f));
  const float rc = __builtin_amdgcn_rcpf(d);
  return g < -88.0f ? 0.0f : g != g ? g : fmaf(rc, fmaf(-d, rc, 1.0f), rc);
}

constexpr int V = 8;  // values to a piece

// One value at p[at], bf16 or fp32.
__device__ __forceinline__ float load1(const void* p, int64_t at, bool f32) {
  return f32 ? static_cast<const float*>(p)[at] : gdn::bf2f(static_cast<const uint16_t*>(p)[at]);
}

// A piece at p[at].  kAny: at any address, its first n values (the others 0); else whole and aligned.
template <bool kAny>
__device__ __forceinline__ void load(const void* p, int64_t at, int n, bool f32, float (&v)[V]) {
  if (kAny && n < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = e < n ? load1(p, at + e, f32) : 0.0f;
  } else if (f32) {
    const float* q = static_cast<const float*>(p) + at;
    if constexpr (kAny) {
      __builtin_memcpy(v, q, sizeof(v));
    } else {
      const float4 a = *reinterpret_cast<const float4*>(q), b = *reinterpret_cast<const float4*>(q + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
  } else {
    const uint16_t* q = static_cast<const uint16_t*>(p) + at;
    uint4 a;
    if constexpr (kAny) __builtin_memcpy(&a, q, sizeof(a));
    else a = *reinterpret_cast<const uint4*>(q);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <bool kAny>
__device__ __forceinline__ void store(void* p, int64_t at, int n, bool f32, const float (&v)[V]) {
  if (kAny && n < V) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (e >= n) continue;
      if (f32) static_cast<float*>(p)[at + e] = v[e];
      else static_cast<uint16_t*>(p)[at + e] = gdn::f2bf(v[e]);
    }
  } else if (f32) {
    float* q = static_cast<float*>(p) + at;
    if constexpr (kAny) {
      __builtin_memcpy(q, v, sizeof(v));
    } else {
      reinterpret_cast<float4*>(q)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(q)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
    uint16_t* q = static_cast<uint16_t*>(p) + at;
    const uint4 w = make_uint4(gdn::f2bf2(v[0], v[1]), gdn::f2bf2(v[2], v[3]), gdn::f2bf2(v[4], v[5]), gdn::f2bf2(v[6], v[7]));
    if constexpr (kAny) __builtin_memcpy(q, &w, sizeof(w));
    else *reinterpret_cast<uint4*>(q) = w;
  }
}

// The sum over the T threads of a row (T: 64, or the whole workgroup).
template <int T>
__device__ __forceinline__ float row_sum(float v, float* part) {
  v = gdn::wave_sum(v);
  if constexpr (T > 64) {
    constexpr int W = T / 64;
    if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = v;
    __syncthreads();
    v = part[0];
#pragma unroll
    for (int i = 1; i < W; ++i) v += part[i];
  }
  return v;
}

// One pass: the row stays in registers between its sums.  What bounds it: HBM, 16384 x 2048 41 us (6.5
// TB/s; 4 bytes read and 4 written a value), with a norm behind the block and a gate 45, in bf16 and e4m3 56; a few rows one
// launch's latency (1 x 2048 2.8 to 4.4, 201 rows with both norms 3.8 to 4.3).
//
// T threads per row, N pieces of 8 values per thread: piece i of thread t is columns V (T i +
// t) .., so that 16 neighbouring lanes hold a group of 128.
template <bool kAny, int N, int T, bool kFp8>
__global__ __launch_bounds__(T > 256 ? T : 256) void block_norm_kernel(NormArgs a) {
  __shared__ float part[2][T > 64 ? T / 64 : 1];
  constexpr int kRows = T > 256 ? 1 : 256 / T;
  static_assert(T == 64 || kRows == 1, "a row's threads are a wave or the workgroup");
  const int t = threadIdx.x % T;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / T;
  if (row >= a.M) return;  // (a wave, or the workgroup)
  auto col = [&](int i) { return V * (T * i + t); };
  auto left = [&](int i) { return a.H - col(i); };  // values of the row from the piece on
  float h[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) h[i][e] = 0.0f;
    if (col(i) < a.H) load<kAny>(a.x, row * a.sx + col(i), left(i), false, h[i]);
  }
  float res[N][V];
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) res[i][e] = 0.0f;
    if (a.residual && col(i) < a.H) load<kAny>(a.residual, row * a.sr + col(i), left(i), a.stream_f32, res[i]);
  }
  const float inv_h = 1.0f / static_cast<float>(a.H);
  if (a.post_w) {
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) ss = fmaf(h[i][e], h[i][e], ss);
    const float r = rsqrtf(row_sum<T>(ss, part[0]) * inv_h + a.eps);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (col(i) >= a.H) continue;
      float w[V];
      load<kAny>(a.post_w, col(i), left(i), a.w_f32, w);
#pragma unroll
      for (int e = 0; e < V; ++e) h[i][e] *= r * (a.offset + w[e]);
    }
  }
  if (a.gate) {
    if (a.g_col == 0) {
      float g = load1(a.gate, row * a.g_row, a.gate_f32);
      if (a.gate_sigmoid) g = sigmoid_ulp(g);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int e = 0; e < V; ++e) h[i][e] *= g;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (col(i) >= a.H) continue;
        float g[V];
        load<kAny>(a.gate, row * a.g_row + col(i), left(i), a.gate_f32, g);
#pragma unroll
        for (int e = 0; e < V; ++e) h[i][e] *= a.gate_sigmoid ? sigmoid_ulp(g[e]) : g[e];
      }
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
      // (what lies past the row stays 0: a gate of infinity is one per row there)
      h[i][e] = (kAny ? e : 0) < left(i) ? fmaf(h[i][e], a.scale, res[i][e]) : 0.0f;
      ss = fmaf(h[i][e], h[i][e], ss);
    }
    if (a.stream && col(i) < a.H) store<kAny>(a.stream, row * a.H + col(i), left(i), a.stream_f32, h[i]);
  }
  const float r = rsqrtf(row_sum<T>(ss, part[1]) * inv_h + a.eps);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const bool in = col(i) < a.H;
    if (!kFp8 && !in) continue;
    float w[V];
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = 0.0f;
    if (in) load<kAny>(a.w, col(i), left(i), a.w_f32, w);
#pragma unroll
    for (int e = 0; e < V; ++e) h[i][e] *= r * (a.offset + w[e]);
    if (a.y && in) store<kAny>(a.y, row * a.H + col(i), left(i), false, h[i]);
    if constexpr (kFp8) {
      float top = 0.0f;
#pragma unroll
      for (int e = 0; e < V; ++e) top = fmaxf(top, fabsf(h[i][e]));
#pragma unroll
      for (int m = 8; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m, 64));
      const float s = gdn::fp8_scale(top), inv = 1.0f / s;
      if (in) {
        *reinterpret_cast<uint2*>(a.y8 + row * a.H + col(i)) =
            make_uint2(gdn::f2fp8x4(h[i][0] * inv, h[i][1] * inv, h[i][2] * inv, h[i][3] * inv),
                       gdn::f2fp8x4(h[i][4] * inv, h[i][5] * inv, h[i][6] * inv, h[i][7] * inv));
        if (t % 16 == 0) a.y8_scale[row * a.ss_row + col(i) / gdn::kFp8Group * a.ss_grp] = s;
      }
    }
  }
}

// Rows `first` .. first + rows - 1.
NormArgs rows_of(const NormArgs& a, int64_t first, int64_t rows) {
  auto at = [](auto* p, int64_t bytes) { return p ? (decltype(p))((uintptr_t)p + bytes) : p; };
  const int64_t dense = first * a.H;
  NormArgs part = a;
  part.x = a.x + first * a.sx;
  part.residual = at(a.residual, first * a.sr * (a.stream_f32 ? 4 : 2));
  part.gate = at(a.gate, first * a.g_row * (a.gate_f32 ? 4 : 2));
  part.stream = at(a.stream, dense * (a.stream_f32 ? 4 : 2));
  part.y = at(a.y, dense * 2);
  part.y8 = at(a.y8, dense);
  part.y8_scale = at(a.y8_scale, first * a.ss_row * 4);
  part.M = rows;
  return part;
}

template <bool kAny, int T, bool kFp8, int... N>
int launch(const NormArgs& a, hipStream_t st) {
  constexpr int kRows = T > 256 ? 1 : 256 / T;
  constexpr int kThreads = T > 256 ? T : 256;
  // (a launch has less than 2^32 threads: 2^26 rows of up to 1024 columns are past that, 2^24 of up to 2048)
  constexpr int64_t kMost = kRows * (((int64_t{1} << 32) - 1) / kThreads);
  bool done = false;
  auto one = [&](auto n) {
    if (done || a.H > V * T * n.value) return;
    for (int64_t first = 0; first < a.M; first += kMost) {
      const NormArgs part = rows_of(a, first, std::min(kMost, a.M - first));
      const dim3 grid(static_cast<unsigned>((part.M + kRows - 1) / kRows));
      block_norm_kernel<kAny, n.value, T, kFp8><<<grid, dim3(kThreads), 0, st>>>(part);
    }
    done = true;
  };
  (one(std::integral_constant<int, N>{}), ...);
  return done ? gdn_launch_status() : GDN_ERR_UNSUPPORTED;
}

template <bool kAny, bool kFp8>
int launch_rows(const NormArgs& a, hipStream_t st) {
  // One piece of 8 to a thread (past 8192 columns two), and so a row's workgroup grows with it: what is in flight is then
  // bounded by the rows that run at once and not by a thread's chain (us, replayed; 256 threads for all: 16 x 4096
  // 4.2, in 512 3.9; 16 x 16384 8.6, in 1024 4.7; 8192 x 16384 317 and 188, 8192 x 8192 107 and 97).  Many short
  // rows go to a wave each, without a barrier: 16384 x 1024 22.1 (256 threads 24.5), 4096 x 1024 7.4 (7.8); 16384 x 2048 45.3
  // (41.1), 1024 x 1024 4.7 (4.3).  What is just past a step pays for threads without a piece, and rows of odd widths
  // for pieces that straddle lines: 1031 x 4096 7.9, x 4296 9.7, x 4299 14.2, x 6144 11.6, x 8192 14.2; 4096 x 4096 22.4, x 4608 25.8,
  // x 6144 31.4, x 8192 41.0.
  if (a.M >= 2048 && a.H <= 1024) return launch<kAny, 64, kFp8, 1, 2>(a, st);
  if (a.H <= 2048) return launch<kAny, 256, kFp8, 1>(a, st);
  if (a.H <= 4096) return launch<kAny, 512, kFp8, 1>(a, st);
  return launch<kAny, 1024, kFp8, 1, 2>(a, st);
}

constexpr int kMostColumns = 16384;

}  // namespace

extern "C" int gdn_add_rms_norm(const uint16_t* x, int64_t sx, const void* residual, int64_t sr, int stream_is_fp32,
                                const void* w, const void* post_w, int w_is_fp32, float offset, const void* gate,
                                int gate_is_fp32, int64_t g_row, int64_t g_col, int gate_sigmoid, float scale, float eps,
                                void* stream_out, uint16_t* y, uint8_t* y8, float* y8_scale, int64_t ss_row,
                                int64_t ss_grp, int64_t M, int H, void* stream) {
  if (M < 0 || H <= 0 || g_col < 0 || g_col > 1 || g_row < 0) return GDN_ERR_INVALID_ARG;
  if (H > kMostColumns || M >= (1LL << 31)) return GDN_ERR_UNSUPPORTED;
  if (y8 && H % gdn::kFp8Group) return GDN_ERR_INVALID_ARG;
  if (M == 0) return GDN_OK;
  if (!x || !w || (!y && !y8) || (y8 && !y8_scale) || sx < H || (residual && sr < H)) return GDN_ERR_INVALID_ARG;
  if (gate && g_col == 1 && g_row != 0 && g_row < H) return GDN_ERR_INVALID_ARG;
  auto aligned = [](const void* p, uintptr_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  auto natural = [&](const void* p, int f32) { return aligned(p, f32 ? 4 : 2); };
  if (!aligned(x, 2) || !natural(residual, stream_is_fp32) || !natural(w, w_is_fp32) || !natural(post_w, w_is_fp32) ||
      !natural(gate, gate_is_fp32) || !natural(stream_out, stream_is_fp32) || !aligned(y, 2) || !aligned(y8_scale, 4))
    return GDN_ERR_INVALID_ARG;
  const NormArgs a{x, sx, residual, sr, w, post_w, gate, g_row, g_col, stream_out, y, y8, y8_scale, ss_row, ss_grp, M, H,
                   stream_is_fp32 ? 1 : 0, w_is_fp32 ? 1 : 0, gate_is_fp32 ? 1 : 0, gate_sigmoid ? 1 : 0, offset, scale,
                   eps};
  // rows of whole 16-byte pieces
  const bool whole = H % 8 == 0 && sx % 8 == 0 && (!residual || sr % 8 == 0) && aligned(x, 16) && aligned(residual, 16) &&
                     aligned(w, 16) && aligned(post_w, 16) && aligned(stream_out, 16) && aligned(y, 16) && aligned(y8, 8) &&
                     (!gate || g_col == 0 || (aligned(gate, 16) && g_row % 8 == 0));
  if (y8 && !whole) return GDN_ERR_INVALID_ARG;
  if (stream == GDN_CHECK_ONLY) return GDN_OK;
  const hipStream_t st = static_cast<hipStream_t>(stream);
  if (y8) return launch_rows<false, true>(a, st);
  // (any other row goes by the same pieces, which straddle lines, its last one value by value: value by value
  // throughout, 8192 x 1001 25.1 us, 1031 x 4299 360)
  return whole ? launch_rows<false, false>(a, st) : launch_rows<true, false>(a, st);
}
