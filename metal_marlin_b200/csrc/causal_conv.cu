// Short causal depthwise convolution over a pool of per-sequence windows:
//   y[t, c] = act(b[c] + sum_{k < K} w[c, k] x[t - K + 1 + k, c]),
// where inputs in front of a sequence come from its window state[row, c, 0 .. K - 2] (oldest first), which afterwards holds the sequence's
// last K - 1 inputs.  2 K flops against one value read and one written: bound by memory at every size that fills the GPU.
//
// Prompts.  A thread owns V neighbouring channels (16 bytes of a 16-bit type) and walks TT tokens of one sequence with the last K - 1
// inputs in registers, so an input is read (TT + K - 1) / TT times, the repeats from L2.  Tiles are cut per sequence, not over the flat
// token axis: with TT >= K - 1 only a sequence's first tile reads its old window, and the same thread writes the new one (from x, or from
// the old window where the sequence is shorter than it), so the window can be updated in place without a second launch.  Tile i belongs to
// the sequence s with base(s) <= i < base(s + 1), base(s) = cu[s] / TT + s: at least ceil(len / TT) tiles a sequence, found by bisection,
// nothing counted on the host.
//
// Single tokens.  A thread owns V channels of RB rows: the weights are read once for RB rows, the window (V (K - 1) consecutive floats) moves
// through registers.
#include "api_ext.h"
#include "launch.h"
#include "typed_io.cuh"

namespace mmb {

constexpr int kConvThreads = 128;

__device__ __forceinline__ float conv_act(float y, int act) { return act == 1 ? silu(y) : y; }

template <int K, int V>
__global__ void __launch_bounds__(kConvThreads) causal_conv_kernel(const MmbCausalConvParams p, int n_groups, int TT, long long n_tiles) {
  constexpr int U = V == 8 ? 4 : 8;        // tokens loaded together
  pdl_launch_dependents();
  pdl_wait();
  const long long id = (long long)blockIdx.x * kConvThreads + threadIdx.x;
  const long long tile = id / n_groups;
  if (tile >= n_tiles) return;
  const int c0 = (int)(id - tile * n_groups) * V;
  auto start = [&](int s) { return min(max(p.cu_seqlens[s], 0), p.T); };
  // last sequence whose first tile is at or before this one; number S is the rows behind the last sequence
  int lo = 0, hi = p.S;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if ((long long)start(mid) / TT + mid <= tile) lo = mid;
    else hi = mid - 1;
  }
  const int s = lo, begin = start(s), end = s < p.S ? max(begin, start(s + 1)) : p.T;
  const long long first = (tile - ((long long)begin / TT + s)) * TT;
  if (first < 0 || first >= end - begin) return;
  const int t0 = begin + (int)first, t1 = min(end, t0 + TT);
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
  float w[K][V], b[V], win[K - 1][V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][v] = ld1(p.w, (long long)(c0 + v) * K + k, p.wt);
    b[v] = p.bias ? ld1(p.bias, c0 + v, p.wt) : 0.f;
  }
  if (first == 0) {
    const bool old = p.state && !(p.fresh && p.fresh[s]);
    float* st = p.state ? p.state + (row * p.C + c0) * (K - 1) : nullptr;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
      for (int j = 0; j < K - 1; ++j) win[j][v] = old ? st[v * (K - 1) + j] : 0.f;
    if (st) {
      const int len = end - begin;
#pragma unroll
      for (int j = 0; j < K - 1; ++j) {
        const int at = len - (K - 1) + j;        // place of the new window's element j in the sequence
        float nw[V];
        if (at >= 0) {
          ldv<V>(p.x, (long long)(begin + at) * p.ldx + c0, p.xt, nw);
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) {
            nw[v] = 0.f;
#pragma unroll
            for (int i = 0; i < K - 1; ++i)
              if (i == j + len) nw[v] = win[i][v];
          }
        }
#pragma unroll
        for (int v = 0; v < V; ++v) st[v * (K - 1) + j] = nw[v];
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < K - 1; ++j) ldv<V>(p.x, (long long)(t0 - (K - 1) + j) * p.ldx + c0, p.xt, win[j]);
  }
  for (int t = t0; t < t1; t += U) {
    float x[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u < t1) ldv<V>(p.x, (long long)(t + u) * p.ldx + c0, p.xt, x[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (t + u < t1) {
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
          float a = b[v];
#pragma unroll
          for (int k = 0; k < K - 1; ++k) a = fmaf(w[k][v], win[k][v], a);
          y[v] = conv_act(fmaf(w[K - 1][v], x[u][v], a), p.act);
        }
        stv<V>(p.out, (long long)(t + u) * p.ldo + c0, p.ot, y);
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
          for (int k = 0; k + 1 < K - 1; ++k) win[k][v] = win[k + 1][v];
          win[K - 2][v] = x[u][v];
        }
      }
    }
  }
}

template <int K, int V, int RB>
__global__ void __launch_bounds__(kConvThreads) causal_conv_step_kernel(const MmbCausalConvParams p, int n_groups) {
  pdl_launch_dependents();
  pdl_wait();
  const int g = blockIdx.x * kConvThreads + threadIdx.x;
  if (g >= n_groups) return;
  const int c0 = g * V;
  float w[K][V], b[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][v] = ld1(p.w, (long long)(c0 + v) * K + k, p.wt);
    b[v] = p.bias ? ld1(p.bias, c0 + v, p.wt) : 0.f;
  }
  const int r0 = blockIdx.y * RB;
  float win[RB][V * (K - 1)], x[RB][V];
  long long row[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    row[r] = r0 + r < p.T ? pool_row(p.rows, r0 + r, p.pool_rows, p.status) : -1;
    if (row[r] >= 0) {
      const float* st = p.state + (row[r] * p.C + c0) * (K - 1);
      if constexpr (V == 4) {
#pragma unroll
        for (int j = 0; j < K - 1; ++j) {
          const float4 f = reinterpret_cast<const float4*>(st)[j];
          win[r][4 * j] = f.x, win[r][4 * j + 1] = f.y, win[r][4 * j + 2] = f.z, win[r][4 * j + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int j = 0; j < V * (K - 1); ++j) win[r][j] = st[j];
      }
      ldv<V>(p.x, (long long)(r0 + r) * p.ldx + c0, p.xt, x[r]);
    }
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
    float y[V], nw[V * (K - 1)];
#pragma unroll
    for (int v = 0; v < V; ++v) {
      float a = b[v];
#pragma unroll
      for (int k = 0; k < K - 1; ++k) {
        a = fmaf(w[k][v], win[r][v * (K - 1) + k], a);
        nw[v * (K - 1) + k] = k + 1 < K - 1 ? win[r][v * (K - 1) + k + 1] : x[r][v];
      }
      y[v] = conv_act(fmaf(w[K - 1][v], x[r][v], a), p.act);
    }
    float* st = p.state + (row[r] * p.C + c0) * (K - 1);
    if constexpr (V == 4) {
#pragma unroll
      for (int j = 0; j < K - 1; ++j) reinterpret_cast<float4*>(st)[j] = make_float4(nw[4 * j], nw[4 * j + 1], nw[4 * j + 2], nw[4 * j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < V * (K - 1); ++j) st[j] = nw[j];
    }
    stv<V>(p.out, (long long)(r0 + r) * p.ldo + c0, p.ot, y);
  }
}

template <int K>
static int launch_conv(const MmbCausalConvParams& p, cudaStream_t stream) {
  const bool vec = p.C % 8 == 0 && rows_aligned(p.x, p.ldx, p.xt, 8) && rows_aligned(p.out, p.ldo, p.ot, 8);
  const int groups = vec ? p.C / 8 : p.C;
  const int TT = (long long)p.T * groups >= (1 << 21) ? 32 : 8;
  const long long tiles = (long long)p.T / TT + p.S + 2;
  const long long blocks = (tiles * groups + kConvThreads - 1) / kConvThreads;
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  if (vec) return launch(causal_conv_kernel<K, 8>, dim3((unsigned)blocks), dim3(kConvThreads), 0, stream, 1, p, groups, TT, tiles);
  return launch(causal_conv_kernel<K, 1>, dim3((unsigned)blocks), dim3(kConvThreads), 0, stream, 1, p, groups, TT, tiles);
}

template <int K, int V>
static int launch_conv_step_v(const MmbCausalConvParams& p, cudaStream_t stream) {
  const int groups = p.C / V;
  const unsigned gx = (unsigned)((groups + kConvThreads - 1) / kConvThreads);
  const bool many = (long long)groups * p.T >= (1 << 17);
  const long long gy = many ? ((long long)p.T + 3) / 4 : p.T;
  if (gy > 65535) return (int)cudaErrorInvalidValue;
  if (many) return launch(causal_conv_step_kernel<K, V, 4>, dim3(gx, (unsigned)gy), dim3(kConvThreads), 0, stream, 1, p, groups);
  return launch(causal_conv_step_kernel<K, V, 1>, dim3(gx, (unsigned)gy), dim3(kConvThreads), 0, stream, 1, p, groups);
}
template <int K>
static int launch_conv_step(const MmbCausalConvParams& p, cudaStream_t stream) {
  const bool vec = p.C % 4 == 0 && rows_aligned(p.x, p.ldx, p.xt, 4) && rows_aligned(p.out, p.ldo, p.ot, 4) &&
                   reinterpret_cast<uintptr_t>(p.state) % 16 == 0;
  return vec ? launch_conv_step_v<K, 4>(p, stream) : launch_conv_step_v<K, 1>(p, stream);
}

}  // namespace mmb

MMB_API int mmb_causal_conv(const MmbCausalConvParams* pp, cudaStream_t stream) {
  const MmbCausalConvParams& p = *pp;
  if (p.T <= 0 || p.C <= 0) return 0;
  if (p.S < 0 || p.cu_seqlens == nullptr) return (int)cudaErrorInvalidValue;
  switch (p.K) {
    case 2: return mmb::launch_conv<2>(p, stream);
    case 3: return mmb::launch_conv<3>(p, stream);
    case 4: return mmb::launch_conv<4>(p, stream);
    case 5: return mmb::launch_conv<5>(p, stream);
    case 6: return mmb::launch_conv<6>(p, stream);
    case 7: return mmb::launch_conv<7>(p, stream);
    case 8: return mmb::launch_conv<8>(p, stream);
    default: return (int)cudaErrorInvalidValue;
  }
}

MMB_API int mmb_causal_conv_step(const MmbCausalConvParams* pp, cudaStream_t stream) {
  const MmbCausalConvParams& p = *pp;
  if (p.T <= 0 || p.C <= 0) return 0;
  if (p.state == nullptr) return (int)cudaErrorInvalidValue;
  switch (p.K) {
    case 2: return mmb::launch_conv_step<2>(p, stream);
    case 3: return mmb::launch_conv_step<3>(p, stream);
    case 4: return mmb::launch_conv_step<4>(p, stream);
    case 5: return mmb::launch_conv_step<5>(p, stream);
    case 6: return mmb::launch_conv_step<6>(p, stream);
    case 7: return mmb::launch_conv_step<7>(p, stream);
    case 8: return mmb::launch_conv_step<8>(p, stream);
    default: return (int)cudaErrorInvalidValue;
  }
}
