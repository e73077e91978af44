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
// Tile i belongs to the sequence s with base(s) <= i < base(s + 1), base(s) = cu[s] / TT + s + 1: at least ceil(len / TT) tiles a sequence, found by
// bisection, nothing counted on the host; the rows in front of the first sequence and behind the last one are sequences -1 and S.
// Measured, 8111 rows of 10240 channels, 4 taps, bf16: 72 us = 4.6 TB/s (the bytes 51 us, two special functions a value 37), 8 taps 91 us; fp32 109.5 us
// = 6.1 TB/s (the bytes 102 us).  What is left for 16-bit types is the work of a value, which does not overlap its loads and stores altogether: without
// the activation 66 us, while fp32 with as many bytes in flight a thread comes near the copy rate; 24 instead of 16 warps an SM or 16-byte instead of 8-byte
// loads changed nothing.  What it took: conversions between the loads of a batch 332 us; a choice by type at every value 93; arithmetic on one value instead
// of two an instruction 75.
//
// Single tokens.  A thread owns V channels of RB rows: the taps are read once for RB rows, the window (V (K - 1) consecutive floats) moves
// through registers.  256 rows of 10240 channels: 13.8 us = 4.9 TB/s, fp32 15.5 us = 5.0; 4096 channels of 8 taps, fp32: 17.2 us for 10.3 us of
// bytes (every lane moves 28 values of its own, so a warp's accesses cover their sectors in several steps; by single floats 55 us).
#include <atomic>

#include "api_ext.h"
#include "launch.h"
#include "typed_io.cuh"

namespace mmb {

constexpr int kConvThreads = 128;
constexpr int kConvSeqs = 1024;              // starts of this many sequences are kept in shared memory

// a = w x + a for V channels.
template <int V>
__device__ __forceinline__ void fma_v(float (&a)[V], const float (&w)[V], const float (&x)[V]) {
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      const float2 f = unpack2(fma2(pack2(w[v], w[v + 1]), pack2(x[v], x[v + 1]), pack2(a[v], a[v + 1])));
      a[v] = f.x, a[v + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) a[v] = fmaf(w[v], x[v], a[v]);
  }
}
// x / (1 + e^-x)
template <int V>
__device__ __forceinline__ void silu_v(float (&x)[V]) {
  constexpr float c = -1.4426950408889634f;
  if constexpr (V % 2 == 0) {
#pragma unroll
    for (int v = 0; v < V; v += 2) {
      const f32x2 xx = pack2(x[v], x[v + 1]);
      float2 f = unpack2(mul2(xx, pack2(c, c)));
      f = unpack2(add2(pack2(exp2_fast(f.x), exp2_fast(f.y)), pack2(1.f, 1.f)));
      f = unpack2(mul2(xx, pack2(rcp_fast(f.x), rcp_fast(f.y))));
      x[v] = f.x, x[v + 1] = f.y;
    }
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] *= rcp_fast(1.f + exp2_fast(c * x[v]));
  }
}

// Taps and bias of V channels.  The V K values of 16-bit weights lie together: whole words.
template <int K, int V>
__device__ __forceinline__ void load_taps(const MmbCausalConvParams& p, int c0, float (&w)[K][V], float (&b)[V]) {
  constexpr int P = K * V % 8 == 0 ? 8 : 4;                // values a load
  const long long at = (long long)c0 * K;
  if (V == 4 && reinterpret_cast<uintptr_t>(p.w) % 16 == 0) {
    float f[K * V];
#pragma unroll
    for (int i = 0; i < K * V / P; ++i) ldv<P>(p.w, at + P * i, p.wt, f + P * i);
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][v] = f[v * K + k];
  } else {
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int k = 0; k < K; ++k) w[k][v] = ld1(p.w, at + v * K + k, p.wt);
  }
#pragma unroll
  for (int v = 0; v < V; ++v) b[v] = p.bias ? ld1(p.bias, c0 + v, p.wt) : 0.f;
}

// The window of V channels: V W consecutive floats, in 16-byte pieces where it is aligned for that.
template <int W, int V>
__device__ __forceinline__ void ld_window(const float* st, bool vec, float (&win)[V * W]) {
  if (V == 4 && vec) {
#pragma unroll
    for (int j = 0; j < V * W / 4; ++j) {
      const float4 f = reinterpret_cast<const float4*>(st)[j];
      win[4 * j] = f.x, win[4 * j + 1] = f.y, win[4 * j + 2] = f.z, win[4 * j + 3] = f.w;
    }
  } else {
#pragma unroll
    for (int j = 0; j < V * W; ++j) win[j] = st[j];
  }
}
template <int W, int V>
__device__ __forceinline__ void st_window(float* st, bool vec, const float (&win)[V * W]) {
  if (V == 4 && vec) {
#pragma unroll
    for (int j = 0; j < V * W / 4; ++j) reinterpret_cast<float4*>(st)[j] = make_float4(win[4 * j], win[4 * j + 1], win[4 * j + 2], win[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < V * W; ++j) st[j] = win[j];
  }
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

template <int K, int V, int ES, int U>
__global__ void __launch_bounds__(kConvThreads) causal_conv_kernel(const MmbCausalConvParams p, int n_groups, int TT, long long n_tiles, bool vec_state) {
  constexpr int W = K - 1;
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
  float w[K][V], b[V], win[W][V];
  if (tile < n_tiles) load_taps<K, V>(p, c0, w, b);
  __syncthreads();
  if (tile >= n_tiles) return;
  auto start = [&](int s) { return near ? starts[s] : min(max(p.cu_seqlens[s], 0), p.T); };
  // last sequence whose first tile is at or before this one; number -1 is the rows in front of the first sequence, number S those behind the last
  int lo = -1, hi = p.S;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start(mid) / TT + mid + 1 <= tile) lo = mid;
    else hi = mid - 1;
  }
  const int s = lo, begin = s < 0 ? 0 : start(s), end = s < p.S ? max(begin, start(s + 1)) : p.T;
  const long long first = (tile - (begin / TT + s + 1)) * TT;
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
      ld_raw<V, ES>(p.x, (long long)(t0 - W + j) * p.ldx + c0, wr[j]);
  }
  long long row = -1;
  bool live = s >= 0 && s < p.S;
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
    float* st = p.state ? p.state + (row * p.C + c0) * W : nullptr;
    float was[V * W];
    if (old) {
      ld_window<W, V>(st, vec_state, was);
    } else {
#pragma unroll
      for (int i = 0; i < V * W; ++i) was[i] = 0.f;
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < W; ++j) win[j][v] = was[v * W + j];
    if (st) {
      const int len = end - begin;
      Raw<V, ES> tail[W];                            // element j of the new window is input len - W + j; in front of the sequence, element j + len of the old
#pragma unroll
      for (int j = 0; j < W; ++j)
        if (len - W + j >= 0) ld_raw<V, ES>(p.x, (long long)(end - W + j) * p.ldx + c0, tail[j]);
      float nw[V * W];
#pragma unroll
      for (int j = 0; j < W; ++j) {
        float x[V];
        cvt_raw<V, ES>(tail[j], p.xt, x);
#pragma unroll
        for (int v = 0; v < V; ++v) {
          nw[v * W + j] = x[v];
          if (len - W + j < 0) {
#pragma unroll
            for (int i = j + 1; i < W; ++i)
              if (i == j + len) nw[v * W + j] = was[v * W + i];
          }
        }
      }
      st_window<W, V>(st, vec_state, nw);
    }
  } else {
#pragma unroll
    for (int j = 0; j < W; ++j) cvt_raw<V, ES>(wr[j], p.xt, win[j]);
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
    {
      float a[V];
#pragma unroll
      for (int v = 0; v < V; ++v) a[v] = b[v];
      fma_v<V>(a, w[W], x[u]);
#pragma unroll
      for (int k = W - 1; k >= 0; --k) fma_v<V>(a, w[k], u + k - W >= 0 ? x[u + k - W >= 0 ? u + k - W : 0] : win[u + k < W ? u + k : 0]);
#pragma unroll
      for (int v = 0; v < V; ++v) x[u][v] = a[v];
    }
    if (p.act == 1) {
#pragma unroll
      for (int u = 0; u < U; ++u) silu_v<V>(x[u]);
    }
    store_batch<U, V>(p.out, (long long)t * p.ldo + c0, p.ldo, min(U, t1 - t), p.ot, x);
#pragma unroll
    for (int j = 0; j < W; ++j)
#pragma unroll
      for (int v = 0; v < V; ++v) win[j][v] = last[j][v];
  }
}

template <int K, int V, int ES, int RB>
__global__ void __launch_bounds__(kConvThreads) causal_conv_step_kernel(const MmbCausalConvParams p, int n_groups) {
  constexpr int W = K - 1;
  pdl_launch_dependents();
  pdl_wait();
  const int g = blockIdx.x * kConvThreads + threadIdx.x;
  if (g >= n_groups) return;
  const int c0 = g * V;
  const int r0 = blockIdx.y * RB;
  long long row[RB];
  float win[RB][V * W];
  Raw<V, ES> xr[RB];
  float w[K][V], b[V];
  load_taps<K, V>(p, c0, w, b);
#pragma unroll
  for (int r = 0; r < RB; ++r) row[r] = r0 + r < p.T ? pool_row(p.rows, r0 + r, p.pool_rows, p.status) : -1;
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    if (row[r] < 0) continue;
    const float* st = p.state + (row[r] * p.C + c0) * W;
    ld_window<W, V>(st, true, win[r]);
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
      y[v] = a;
    }
    float s[V];                                      // chosen without a branch, which would end the overlap of the rows (256 rows: 14.6 us against 16.1)
#pragma unroll
    for (int v = 0; v < V; ++v) s[v] = y[v];
    silu_v<V>(s);
#pragma unroll
    for (int v = 0; v < V; ++v) y[v] = p.act == 1 ? s[v] : y[v];
    float* st = p.state + (row[r] * p.C + c0) * W;
    st_window<W, V>(st, true, nw);
    stv<V>(p.out, (long long)(r0 + r) * p.ldo + c0, p.ot, y);
  }
}

template <int K, int V, int ES, int U>
static int launch_conv_u(const MmbCausalConvParams& p, cudaStream_t stream) {
  const int groups = p.C / V;
  static std::atomic<int> resident{0};
  int ctas = resident.load(std::memory_order_relaxed);
  if (ctas == 0) {
    const cudaError_t e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, causal_conv_kernel<K, V, ES, U>, kConvThreads, 0);
    if (e != cudaSuccess) return (int)e;
    resident.store(ctas, std::memory_order_relaxed);
  }
  // long tiles read fewer inputs twice and start less often (8111 rows of 10240 channels, us for 8 / 16 / 32 / 64 tokens: 128 / 95 / 78 / 72), short
  // ones give more threads (500 rows of 2048: 4.6 / 5.7 / 7.0 / 10.3): the longest that leave 2^17 threads
  int TT = 8;
  while (TT < 64 && (long long)p.T * groups / (2 * TT) >= (1 << 17)) TT *= 2;
  // then up to twice that where the last wave is fuller for it; a tile's start costs about six tokens (4096 rows of 8192: 64 tokens, 1.7 waves, 33 us;
  // 112 tokens, one wave, 30 us)
  long long best = -1;
  for (int t = TT, t1 = 2 * TT; t < t1; t += 8) {
    const long long b = (((long long)p.T + t - 1) / t + p.S / 2) * groups / kConvThreads, cost = (b / (148 * ctas) + (b % (148 * ctas) != 0)) * (t + 6);
    if (best < 0 || cost < best) best = cost, TT = t;
  }
  const long long tiles = (long long)p.T / TT + p.S + 2;
  const long long blocks = (tiles * groups + kConvThreads - 1) / kConvThreads;
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  return launch(causal_conv_kernel<K, V, ES, U>, dim3((unsigned)blocks), dim3(kConvThreads), 0, stream, 1, p, groups, TT, tiles, reinterpret_cast<uintptr_t>(p.state) % 16 == 0);
}
// U: tokens a thread loads together
template <int K, int V, int ES>
static int launch_conv_v(const MmbCausalConvParams& p, cudaStream_t stream) {
  constexpr int U = V == 4 && ES == 4 ? 4 : 8;
  if constexpr (V == 4 && ES == 2) {
    // short sequences are mostly starts: smaller batches take fewer registers, so more starts overlap (8192 channels, us for U = 8 / 4 / 2: 155 sequences
    // of 1 to 20 tokens 28 / 21 / 20, 64 of 20 to 40 tokens 30 / 27 / 28; 300 single tokens of 10240: 57 / 40 / 32; one prompt of 4096: 29 / 33 / -)
    if (p.S > 1 && p.T / p.S <= 8) return launch_conv_u<K, V, ES, 2>(p, stream);
    if (p.S > 1 && p.T / p.S <= 32) return launch_conv_u<K, V, ES, 4>(p, stream);
  }
  return launch_conv_u<K, V, ES, U>(p, stream);
}
template <int K>
static int launch_conv(const MmbCausalConvParams& p, cudaStream_t stream) {
  const bool vec = p.C % 4 == 0 && rows_aligned(p.x, p.ldx, p.xt, 4) && rows_aligned(p.out, p.ldo, p.ot, 4);
  if (p.xt == 2) return vec ? launch_conv_v<K, 4, 4>(p, stream) : launch_conv_v<K, 1, 4>(p, stream);
  return vec ? launch_conv_v<K, 4, 2>(p, stream) : launch_conv_v<K, 1, 2>(p, stream);
}

template <int K, int V, int ES>
static int launch_conv_step_v(const MmbCausalConvParams& p, cudaStream_t stream) {
  const int groups = p.C / V;
  const unsigned gx = (unsigned)((groups + kConvThreads - 1) / kConvThreads);
  // four rows a thread read the taps once (256 rows of 3001 channels: 4.7 us against 7.0) where that leaves enough threads (64 rows of 8192: 6.2 against 4.8)
  const bool many = (long long)groups * p.T >= (1 << 18);
  const long long gy = many ? ((long long)p.T + 3) / 4 : p.T;
  if (gy > 65535) return (int)cudaErrorInvalidValue;
  if (many) return launch(causal_conv_step_kernel<K, V, ES, 4>, dim3(gx, (unsigned)gy), dim3(kConvThreads), 0, stream, 1, p, groups);
  return launch(causal_conv_step_kernel<K, V, ES, 1>, dim3(gx, (unsigned)gy), dim3(kConvThreads), 0, stream, 1, p, groups);
}
template <int K>
static int launch_conv_step(const MmbCausalConvParams& p, cudaStream_t stream) {
  const bool vec = p.C % 4 == 0 && rows_aligned(p.x, p.ldx, p.xt, 4) && rows_aligned(p.out, p.ldo, p.ot, 4) &&
                   reinterpret_cast<uintptr_t>(p.state) % 16 == 0;
  if (p.xt == 2) return vec ? launch_conv_step_v<K, 4, 4>(p, stream) : launch_conv_step_v<K, 1, 4>(p, stream);
  return vec ? launch_conv_step_v<K, 4, 2>(p, stream) : launch_conv_step_v<K, 1, 2>(p, stream);
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
    case 5: return mmb::launch_conv<5>(p, stream);
    case 6: return mmb::launch_conv<6>(p, stream);
    case 7: return mmb::launch_conv<7>(p, stream);
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
    case 5: return mmb::launch_conv_step<5>(p, stream);
    case 6: return mmb::launch_conv_step<6>(p, stream);
    case 7: return mmb::launch_conv_step<7>(p, stream);
    default: return mmb::launch_conv_step<8>(p, stream);
  }
}
