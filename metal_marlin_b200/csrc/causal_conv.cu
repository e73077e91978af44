// Short causal depthwise convolution over a pool of per-sequence windows:
//   y[t, c] = act(b[c] + sum_{k < K} w[c, k] x[t - K + 1 + k, c]),
// where inputs in front of a sequence come from its window state[row, c, 0 .. K - 2] (oldest first), which afterwards holds the sequence's
// last K - 1 inputs.  2 K flops and two special functions (SiLU) against one value read and one written.
//
// Prompts.  A thread owns V = 4 neighbouring channels (one where the rows are not aligned for that) and walks TT tokens of one sequence in batches
// of U with the last K - 1 inputs in registers; the next batch is loaded before this one is computed, and a batch is converted, filtered,
// activated and stored as a whole, with one choice by type for each.  An input is read (TT + K - 1) / TT times, the repeats from L2.  Tiles are cut
// per sequence, not over the flat token axis: with TT >= K - 1 only a sequence's first tile reads its old window, and the same thread writes the
// new one (from x, or from the old window where the sequence is shorter than it), so the window is updated in place without a second launch.
// Tile i belongs to the sequence s with base(s) <= i < base(s + 1), base(s) = cu[s] / TT + s: at least ceil(len / TT) tiles a sequence, found by
// bisection, nothing counted on the host.  Measured, 8111 rows of 10240 channels, 4 taps, bf16: 72 us = 4.6 TB/s; two special functions a value
// take 37 us of it, the bytes 51 us (conversions between the loads of a batch: 332 us; a choice by type at every value: 93 us).
//
// Single tokens.  A thread owns V channels of RB rows: the taps are read once for RB rows, the window (V (K - 1) consecutive floats) moves
// through registers.  256 rows of 10240 channels: 14.6 us = 5.0 TB/s.
#include "api_ext.h"
#include "launch.h"
#include "typed_io.cuh"

namespace mmb {

constexpr int kConvThreads = 128;
constexpr int kConvSeqs = 1024;              // starts of this many sequences are kept in shared memory

__device__ __forceinline__ float conv_act(float y, int act) { return act == 1 ? silu(y) : y; }

// Taps and bias of V channels; taps that are compiled in but not used are zero.  The V K values of 16-bit weights lie together: whole words.
template <int KT, int V>
__device__ __forceinline__ void load_taps(const MmbCausalConvParams& p, int c0, int K, float (&w)[KT][V], float (&b)[V]) {
  const int skip = KT - K;
  const long long at = (long long)c0 * K;
  if (KT < 8 && KT * V % 8 == 0 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0) {
    float f[KT * V];
#pragma unroll
    for (int i = 0; i < KT * V / 8; ++i) ldv<8>(p.w, at + 8 * i, p.wt, f + 8 * i);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < KT; ++k) w[k][v] = f[v * KT + k];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < KT; ++k) w[k][v] = k >= skip ? ld1(p.w, at + v * K + k - skip, p.wt) : 0.f;
  }
#pragma unroll
  for (int v = 0; v < V; ++v) b[v] = p.bias ? ld1(p.bias, c0 + v, p.wt) : 0.f;
}

template <int U, int V, int ES>
__device__ __forceinline__ void cvt_batch(const Raw<V, ES> (&r)[U], int t, float (&x)[U][V]) {
  if (ES == 4 || t == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u) cvt_raw<V, ES>(r[u], 0, x[u]);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u) cvt_raw<V, ES>(r[u], 1, x[u]);
  }
}
template <int U, int V>
__device__ __forceinline__ void store_batch(void* out, long long at, long long ld, int n, int t, const float (&x)[U][V]) {
  if (t == 0) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < n) stv<V>(out, at + u * ld, 0, x[u]);
  } else if (t == 1) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < n) stv<V>(out, at + u * ld, 1, x[u]);
  } else {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < n) stv<V>(out, at + u * ld, 2, x[u]);
  }
}

// KT taps are compiled in; `K` of them are used (K < KT only for KT = 8), aligned to the newest input: tap KT - 1 meets the newest one.
template <int KT, int V, int ES>
__global__ void __launch_bounds__(kConvThreads) causal_conv_kernel(const MmbCausalConvParams p, int n_groups, int TT, long long n_tiles) {
  constexpr int U = V == 4 && ES == 4 ? 4 : 8;             // tokens loaded together
  constexpr int W = KT - 1;
  const int K = KT == 8 ? p.K : KT, skip = KT - K;
  pdl_launch_dependents();
  pdl_wait();
  // sequence starts in shared memory: the bisection would otherwise wait for global memory at every step
  __shared__ int starts[kConvSeqs + 1];
  const bool near = p.S <= kConvSeqs;
  if (near)
    for (int i = threadIdx.x; i <= p.S; i += kConvThreads) starts[i] = min(max(p.cu_seqlens[i], 0), p.T);
  const long long id = (long long)blockIdx.x * kConvThreads + threadIdx.x;
  const long long tile = id / n_groups;
  const int c0 = (int)(id - tile * n_groups) * V;
  float w[KT][V], b[V], win[W][V];
  if (tile < n_tiles) load_taps<KT, V>(p, c0, K, w, b);
  __syncthreads();
  if (tile >= n_tiles) return;
  auto start = [&](int s) { return near ? starts[s] : min(max(p.cu_seqlens[s], 0), p.T); };
  // last sequence whose first tile is at or before this one; number S is the rows behind the last sequence
  int lo = 0, hi = p.S;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start(mid) / TT + mid <= tile) lo = mid;
    else hi = mid - 1;
  }
  const int s = lo, begin = start(s), end = s < p.S ? max(begin, start(s + 1)) : p.T;
  const long long first = (tile - (begin / TT + s)) * TT;
  if (first < 0 || first >= end - begin) return;
  const int t0 = begin + (int)first, t1 = min(end, t0 + TT);
  Raw<V, ES> xr[U], wr[W];
  auto load = [&](int t) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u < t1) ld_raw<V, ES>(p.x, (long long)(t + u) * p.ldx + c0, xr[u]);
  };
  load(t0);
  if (first > 0) {
#pragma unroll
    for (int j = 0; j < W; ++j)
      if (j >= skip) ld_raw<V, ES>(p.x, (long long)(t0 - W + j) * p.ldx + c0, wr[j]);
  }
  long long row = -1;
  bool live = s < p.S;
  if (live && p.state) {
    row = pool_row(p.rows, s, p.pool_rows, p.status);
    live = row >= 0;
  }
  if (!live) {
    if (p.zero_dead) {
      float zero[V] = {};
      for (int t = t0; t < t1; ++t) stv<V>(p.out, (long long)t * p.ldo + c0, p.ot, zero);
    }
    return;
  }
  if (first == 0) {
    const bool old = p.state && !(p.fresh && p.fresh[s]);
    float* st = p.state ? p.state + (row * p.C + c0) * (K - 1) - skip : nullptr;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < W; ++j) win[j][v] = old && j >= skip ? st[v * (K - 1) + j] : 0.f;
    if (st) {
      const int len = end - begin;
#pragma unroll
      for (int j = 0; j < W; ++j) {
        if (j < skip) continue;
        const int at = len - W + j;              // place of the new window's element j in the sequence; before it, in the old window
        float nw[V];
        if (at >= 0) {
          ldv<V>(p.x, (long long)(begin + at) * p.ldx + c0, p.xt, nw);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) nw[v] = old ? st[v * (K - 1) + j + len] : 0.f;      // behind what has been overwritten
        }
#pragma unroll
        for (int v = 0; v < V; ++v) st[v * (K - 1) + j] = nw[v];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) {
      if (j >= skip) {
        cvt_raw<V, ES>(wr[j], p.xt, win[j]);
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) win[j][v] = 0.f;
      }
    }
  }
  // a batch is converted, filtered, activated and stored as a whole: one choice by type for each, none between its loads
  for (int t = t0; t < t1; t += U) {
    float x[U][V], last[W][V];
    cvt_batch<U, V, ES>(xr, p.xt, x);
    load(t + U);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) last[j][v] = U - W + j >= 0 ? x[U - W + j >= 0 ? U - W + j : 0][v] : win[j + U < W ? j + U : 0][v];
#pragma unroll
    for (int u = U - 1; u >= 0; --u)             // newest first: an output takes the place of its input, which only newer outputs saw
#pragma unroll
      for (int v = 0; v < V; ++v) {
        float a = fmaf(w[W][v], x[u][v], b[v]);
#pragma unroll
        for (int k = W - 1; k >= 0; --k) a = fmaf(w[k][v], u + k - W >= 0 ? x[u + k - W >= 0 ? u + k - W : 0][v] : win[u + k < W ? u + k : 0][v], a);
        x[u][v] = a;
      }
    if (p.act == 1) {
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int v = 0; v < V; ++v) x[u][v] = silu(x[u][v]);
    }
    store_batch<U, V>(p.out, (long long)t * p.ldo + c0, p.ldo, min(U, t1 - t), p.ot, x);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) win[j][v] = last[j][v];
  }
}

template <int KT, int V, int ES, int RB>
__global__ void __launch_bounds__(kConvThreads) causal_conv_step_kernel(const MmbCausalConvParams p, int n_groups) {
  constexpr int W = KT - 1;
  const int K = KT == 8 ? p.K : KT, skip = KT - K;
  constexpr bool kVecState = V == 4 && KT < 8;
  pdl_launch_dependents();
  pdl_wait();
  const int g = blockIdx.x * kConvThreads + threadIdx.x;
  if (g >= n_groups) return;
  const int c0 = g * V;
  const int r0 = blockIdx.y * RB;
  long long row[RB];
  float win[RB][V * W];
  Raw<V, ES> xr[RB];
  float w[KT][V], b[V];
  load_taps<KT, V>(p, c0, K, w, b);
#pragma unroll
  for (int r = 0; r < RB; ++r) row[r] = r0 + r < p.T ? pool_row(p.rows, r0 + r, p.pool_rows, p.status) : -1;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (row[r] < 0) continue;
    const float* st = p.state + (row[r] * p.C + c0) * (K - 1);
    if constexpr (kVecState) {
#pragma unroll
      for (int j = 0; j < W; ++j) {
        const float4 f = reinterpret_cast<const float4*>(st)[j];
        win[r][4 * j] = f.x, win[r][4 * j + 1] = f.y, win[r][4 * j + 2] = f.z, win[r][4 * j + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < W; ++j) win[r][v * W + j] = j >= skip ? st[v * (K - 1) + j - skip] : 0.f;
    }
    ld_raw<V, ES>(p.x, (long long)(r0 + r) * p.ldx + c0, xr[r]);
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (row[r] < 0) {
      if (p.zero_dead && r0 + r < p.T) {
        float zero[V] = {};
        stv<V>(p.out, (long long)(r0 + r) * p.ldo + c0, p.ot, zero);
      }
      continue;
    }
    float x[V], y[V], nw[V * W];
    cvt_raw<V, ES>(xr[r], p.xt, x);
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = fmaf(w[W][v], x[v], b[v]);
#pragma unroll
      for (int k = W - 1; k >= 0; --k) {
        a = fmaf(w[k][v], win[r][v * W + k], a);
        nw[v * W + k] = k + 1 < W ? win[r][v * W + k + 1] : x[v];
      }
      y[v] = conv_act(a, p.act);
    }
    float* st = p.state + (row[r] * p.C + c0) * (K - 1);
    if constexpr (kVecState) {
#pragma unroll
      for (int j = 0; j < W; ++j) reinterpret_cast<float4*>(st)[j] = make_float4(nw[4 * j], nw[4 * j + 1], nw[4 * j + 2], nw[4 * j + 3]);
    } else {
#pragma unroll
      for (int v = 0; v < V; ++v)
#pragma unroll
        for (int j = 0; j < W; ++j)
          if (j >= skip) st[v * (K - 1) + j - skip] = nw[v * W + j];
    }
    stv<V>(p.out, (long long)(r0 + r) * p.ldo + c0, p.ot, y);
  }
}

template <int KT, int V, int ES>
static int launch_conv_v(const MmbCausalConvParams& p, cudaStream_t stream) {
  const int groups = p.C / V;
  // long tiles read fewer inputs twice and start less often (8111 rows of 10240 channels, us for 8 / 16 / 32 / 64 tokens: 125 / 93 / 78 / 72), short
  // ones give more threads (500 rows of 2048: 4.5 / 5.8 / 6.6 / 9.5): the longest that leave 2^17 threads
  int TT = 8;
  while (TT < 64 && (long long)p.T * groups / (2 * TT) >= (1 << 17)) TT *= 2;
  const long long tiles = (long long)p.T / TT + p.S + 2;
  const long long blocks = (tiles * groups + kConvThreads - 1) / kConvThreads;
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  return launch(causal_conv_kernel<KT, V, ES>, dim3((unsigned)blocks), dim3(kConvThreads), 0, stream, 1, p, groups, TT, tiles);
}
template <int KT>
static int launch_conv(const MmbCausalConvParams& p, cudaStream_t stream) {
  const bool vec = p.C % 4 == 0 && rows_aligned(p.x, p.ldx, p.xt, 4) && rows_aligned(p.out, p.ldo, p.ot, 4);
  if (p.xt == 2) return vec ? launch_conv_v<KT, 4, 4>(p, stream) : launch_conv_v<KT, 1, 4>(p, stream);
  return vec ? launch_conv_v<KT, 4, 2>(p, stream) : launch_conv_v<KT, 1, 2>(p, stream);
}

template <int KT, int V, int ES>
static int launch_conv_step_v(const MmbCausalConvParams& p, cudaStream_t stream) {
  const int groups = p.C / V;
  const unsigned gx = (unsigned)((groups + kConvThreads - 1) / kConvThreads);
  // four rows a thread read the taps once (256 rows of 3001 channels: 4.7 us against 7.0) where that leaves enough threads (64 rows of 8192: 6.2 against 4.8)
  const bool many = (long long)groups * p.T >= (1 << 18);
  const long long gy = many ? ((long long)p.T + 3) / 4 : p.T;
  if (gy > 65535) return (int)cudaErrorInvalidValue;
  if (many) return launch(causal_conv_step_kernel<KT, V, ES, 4>, dim3(gx, (unsigned)gy), dim3(kConvThreads), 0, stream, 1, p, groups);
  return launch(causal_conv_step_kernel<KT, V, ES, 1>, dim3(gx, (unsigned)gy), dim3(kConvThreads), 0, stream, 1, p, groups);
}
template <int KT>
static int launch_conv_step(const MmbCausalConvParams& p, cudaStream_t stream) {
  const bool vec = p.C % 4 == 0 && rows_aligned(p.x, p.ldx, p.xt, 4) && rows_aligned(p.out, p.ldo, p.ot, 4) &&
                   reinterpret_cast<uintptr_t>(p.state) % 16 == 0;
  if (p.xt == 2) return vec ? launch_conv_step_v<KT, 4, 4>(p, stream) : launch_conv_step_v<KT, 1, 4>(p, stream);
  return vec ? launch_conv_step_v<KT, 4, 2>(p, stream) : launch_conv_step_v<KT, 1, 2>(p, stream);
}

}  // namespace mmb

MMB_API int mmb_causal_conv(const MmbCausalConvParams* pp, cudaStream_t stream) {
  const MmbCausalConvParams& p = *pp;
  if (p.T <= 0 || p.C <= 0) return 0;
  if (p.S < 0 || p.cu_seqlens == nullptr || p.K < 2 || p.K > 8) return (int)cudaErrorInvalidValue;
  switch (p.K) {
    case 2: return mmb::launch_conv<2>(p, stream);
    case 3: return mmb::launch_conv<3>(p, stream);
    case 4: return mmb::launch_conv<4>(p, stream);
    default: return mmb::launch_conv<8>(p, stream);
  }
}

MMB_API int mmb_causal_conv_step(const MmbCausalConvParams* pp, cudaStream_t stream) {
  const MmbCausalConvParams& p = *pp;
  if (p.T <= 0 || p.C <= 0) return 0;
  if (p.state == nullptr || p.K < 2 || p.K > 8) return (int)cudaErrorInvalidValue;
  switch (p.K) {
    case 2: return mmb::launch_conv_step<2>(p, stream);
    case 3: return mmb::launch_conv_step<3>(p, stream);
    case 4: return mmb::launch_conv_step<4>(p, stream);
    default: return mmb::launch_conv_step<8>(p, stream);
  }
}
