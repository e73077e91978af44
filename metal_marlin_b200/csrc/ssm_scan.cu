// Selective state space scan over a pool of per-sequence states:
//   d_t = softplus(dt_t + dt_bias)                       (or dt_t itself)
//   h_t[n] = exp(d_t A[c, n]) h_{t-1}[n] + d_t x_t B_t[n]
//   out_t = (sum_n h_t[n] C_t[n] + D[c] x_t) silu(z_t)
// with h fp32 in state[row, c, 0 .. N - 1], read when a sequence starts (zero when it is fresh) and written when it ends.
//
// Prompts.  Every step of every state takes one exponential and four fp32 multiply-adds; at 16 exponentials a clock and SM the special
// function unit bounds the scan (N = 16 and 16-bit activations: 3 x longer than moving the activations through memory).  The recurrence is
// one multiply-add deep, so a warp with a few states a lane already keeps that unit busy; the work is therefore split over channels and over
// the STATES of a channel, never over time (a second pass over time would double the exponentials).  S lanes share a channel, each with NPL
// states in registers; 128 threads own 128 / S channels of one sequence and walk it in tiles of TT = 8 S tokens (1024 values):
//   * the tile's x, dt, z, B, C arrive raw in shared memory by 16-byte cp.async, one tile ahead;
//   * every thread turns 8 values into (d, d x) pairs, so softplus is paid once per value, not once per lane;
//   * the warps scan: per token one broadcast pair and NPL values of B and C each;
//   * partial outputs of S tokens are summed over the S lanes by a transposing butterfly (S - 1 shuffles for S tokens) that leaves every
//     lane with the sum of one token;
//   * every thread adds the skip term, applies the gate and stores its 8 values.
// exp(d A) is taken as 2^(d (A log2 e)); A log2 e is rounded once, which shifts every exponent by the same relative 2^-24.
//
// Single tokens.  The state is the traffic: S lanes move a channel's N values in 16-byte pieces, RB rows at a time so that A stays in registers.
#include <atomic>

#include "api_ext.h"
#include "launch.h"
#include "typed_io.cuh"

namespace mmb {

constexpr int kSsmThreads = 128;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// log(1 + e^v) = max(v, 0) + log1p(e^-|v|): no overflow, and exact to fp32 for the small steps of strongly negative v
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(__expf(-fabsf(v))); }

__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Sums v[i] over the S lanes of a group for i < S; lane s of the group ends with the sum of v[s] in v[0].
template <int S>
__device__ __forceinline__ void transposed_sum(float (&v)[S], int s) {
#pragma unroll
  for (int m = S / 2; m >= 1; m >>= 1) {
    const bool up = s & m;
#pragma unroll
    for (int i = 0; i < m; ++i) {
      const float send = up ? v[i] : v[i + m], keep = up ? v[i + m] : v[i];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m);
    }
  }
}

// Byte offsets of the parts of a block's shared memory; two raw stages, then the fp32 tiles.
struct SsmLayout {
  int x, dt, z, b, c, stage, pair, bf, cf, total;
};
__host__ __device__ inline SsmLayout ssm_layout(int TT, int CH, int N, int NP, int xb, int dtb, int zb, int bb) {
  SsmLayout l;
  auto up = [](int v) { return (v + 15) / 16 * 16; };
  int at = 0;
  l.x = at, at += TT * CH * xb;
  l.dt = at, at += TT * CH * dtb;
  l.z = at, at += TT * CH * zb;
  l.b = at, at += up(TT * N * bb);
  l.c = at, at += up(TT * N * bb);
  l.stage = at;
  at *= 2;
  l.pair = at, at += TT * CH * 8;
  l.bf = at, at += TT * NP * 4;
  l.cf = at, at += TT * NP * 4;
  l.total = at;
  return l;
}

template <int S, int NPL>
__global__ void __launch_bounds__(kSsmThreads) ssm_scan_kernel(const MmbSsmParams p, int n_blocks, int vec_x, int vec_bc, int vec_out) {
  constexpr int CH = kSsmThreads / S, TT = 8 * S, NP = S * NPL;
  extern __shared__ __align__(16) unsigned char sm[];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x;
  const int seq = blockIdx.x / n_blocks, c0 = (blockIdx.x % n_blocks) * CH;
  auto start = [&](int s) { return min(max(p.cu_seqlens[s], 0), p.T); };
  const int begin = start(seq), end = seq < p.S ? max(begin, start(seq + 1)) : p.T;
  if (begin >= end) return;
  long long row = -1;
  bool live = seq < p.S;
  if (live && p.state) {
    row = pool_row(p.rows, seq, p.pool_rows, p.status);
    live = row >= 0;
  }
  if (!live) {                                    // rows of no live sequence
    if (p.zero_dead)
      for (long long i = tid; i < (long long)(end - begin) * CH; i += kSsmThreads) {
        const int c = c0 + (int)(i % CH);
        if (c < p.D) st1(p.out, (begin + i / CH) * p.ldo + c, p.ot, 0.f);
      }
    return;
  }
  const int xb = elt_bytes(p.xt), dtb = elt_bytes(p.dtt), zb = p.z ? elt_bytes(p.zt) : 0, bb = elt_bytes(p.bt), N = p.N;
  const SsmLayout L = ssm_layout(TT, CH, N, NP, xb, dtb, zb, bb);
  float2* pair = reinterpret_cast<float2*>(sm + L.pair);
  float* bf = reinterpret_cast<float*>(sm + L.bf);
  float* cf = reinterpret_cast<float*>(sm + L.cf);

  // rows t0 .. t0 + TT of a [*, width] tensor, `cols` of them from column `col`, into a dense [TT][cols] raw tile; zeros outside
  auto fetch = [&](unsigned char* dst, const void* src, long long ld, int es, int col, int cols, int width, int t0, bool vec) {
    if (vec) {
      const int per = cols * es / 16;             // 16-byte pieces a row
      for (int i = tid; i < TT * per; i += kSsmThreads) {
        const int r = i / per, q = i - r * per;
        const bool ok = t0 + r < end && col + q * 16 / es < width;
        const char* g = reinterpret_cast<const char*>(src) + (ok ? ((long long)(t0 + r) * ld + col) * es + q * 16 : 0);
        cp_async16(dst + i * 16, g, ok);
      }
    } else {
      for (int i = tid; i < TT * cols; i += kSsmThreads) {
        const int r = i / cols, q = i - r * cols;
        const bool ok = t0 + r < end && col + q < width;
        const long long at = (long long)(t0 + r) * ld + col + q;
        if (es == 2) reinterpret_cast<uint16_t*>(dst)[i] = ok ? reinterpret_cast<const uint16_t*>(src)[at] : (uint16_t)0;
        else reinterpret_cast<uint32_t*>(dst)[i] = ok ? reinterpret_cast<const uint32_t*>(src)[at] : 0u;
      }
    }
  };
  auto prefetch = [&](int t0, int stage) {
    unsigned char* st = sm + stage * L.stage;
    fetch(st + L.x, p.x, p.ldx, xb, c0, CH, p.D, t0, vec_x);
    fetch(st + L.dt, p.dt, p.lddt, dtb, c0, CH, p.D, t0, vec_x);
    if (p.z) fetch(st + L.z, p.z, p.ldz, zb, c0, CH, p.D, t0, vec_x);
    fetch(st + L.b, p.B, p.ldb, bb, 0, N, N, t0, vec_bc);
    fetch(st + L.c, p.C, p.ldc, bb, 0, N, N, t0, vec_bc);
    cp_async_commit();
  };
  prefetch(begin, 0);

  // this thread's 8 values of a tile: token vt, channels vc .. vc + 7
  const int vt = tid * 8 / CH, vc = tid * 8 % CH;
  float bias[8], skip[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const bool in = c0 + vc + i < p.D;
    bias[i] = in && p.dt_bias ? p.dt_bias[c0 + vc + i] : 0.f;
    skip[i] = in && p.Dskip ? p.Dskip[c0 + vc + i] : 0.f;
  }
  // this lane's states: channel ch, states s NPL .. s NPL + NPL - 1
  const int lane = tid & 31, s = lane % S, cl = (tid >> 5) * (32 / S) + lane / S, ch = c0 + cl;
  float h[NPL], a[NPL];
  const bool old = p.state && !(p.fresh && p.fresh[seq]);
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int n = s * NPL + j;
    const bool in = ch < p.D && n < N;
    a[j] = in ? p.A[(long long)ch * N + n] * kLog2e : 0.f;
    h[j] = in && old ? p.state[(row * p.D + ch) * N + n] : 0.f;
  }

  int stage = 0;
  for (int t0 = begin; t0 < end; t0 += TT, stage ^= 1) {
    const int valid = min(TT, end - t0);
    unsigned char* st = sm + stage * L.stage;
    cp_async_wait<0>();
    __syncthreads();                              // the raw tile is there; everybody is done with the other stage and the fp32 tiles
    if (t0 + TT < end) prefetch(t0 + TT, stage ^ 1);
    {
      float x[8], d[8];
      ldv<8>(st + L.x, tid * 8, p.xt, x);
      ldv<8>(st + L.dt, tid * 8, p.dtt, d);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = d[i] + bias[i];
        if (p.softplus) v = softplus(v);
        d[i] = v;
      }
      float4* dst = reinterpret_cast<float4*>(pair + tid * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) dst[i] = make_float4(d[2 * i], d[2 * i] * x[2 * i], d[2 * i + 1], d[2 * i + 1] * x[2 * i + 1]);
      for (int i = tid; i < TT * NP; i += kSsmThreads) {
        const int t = i / NP, n = i % NP;
        bf[i] = n < N ? ld1(st + L.b, t * N + n, p.bt) : 0.f;
        cf[i] = n < N ? ld1(st + L.c, t * N + n, p.bt) : 0.f;
      }
    }
    __syncthreads();
    auto token = [&](int t) {
      const float2 dd = pair[t * CH + cl];
      float acc = 0.f;
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        const float b = bf[t * NP + s * NPL + j], c = cf[t * NP + s * NPL + j];
        h[j] = fmaf(exp2_fast(dd.x * a[j]), h[j], dd.y * b);
        acc = fmaf(h[j], c, acc);
      }
      return acc;
    };
    for (int g = 0; g < valid; g += S) {
      float v[S];
      if (g + S <= valid) {
#pragma unroll
        for (int i = 0; i < S; ++i) v[i] = token(g + i);
      } else {
#pragma unroll
        for (int i = 0; i < S; ++i) v[i] = g + i < valid ? token(g + i) : 0.f;
      }
      transposed_sum<S>(v, s);
      __syncwarp();
      pair[(g + s) * CH + cl].x = v[0];           // all lanes of this channel have read the pairs of these tokens
    }
    __syncthreads();
    if (vt < valid) {
      float x[8], y[8];
      ldv<8>(st + L.x, tid * 8, p.xt, x);
      const float4* src = reinterpret_cast<const float4*>(pair + tid * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float4 f = src[i];
        y[2 * i] = fmaf(skip[2 * i], x[2 * i], f.x);
        y[2 * i + 1] = fmaf(skip[2 * i + 1], x[2 * i + 1], f.z);
      }
      if (p.z) {
        float z[8];
        ldv<8>(st + L.z, tid * 8, p.zt, z);
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] *= silu(z[i]);
      }
      const long long at = (long long)(t0 + vt) * p.ldo + c0 + vc;
      if (vec_out) {
        if (c0 + vc < p.D) stv<8>(p.out, at, p.ot, y);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (c0 + vc + i < p.D) st1(p.out, at + i, p.ot, y[i]);
      }
    }
  }
  if (p.state) {
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int n = s * NPL + j;
      if (ch < p.D && n < N) p.state[(row * p.D + ch) * N + n] = h[j];
    }
  }
}

// S lanes a channel, VEC states at a time (4: 16-byte pieces), CH_N pieces a lane, RB rows.
template <int S, int VEC, int PCS, int RB>
__global__ void __launch_bounds__(kSsmThreads) ssm_step_kernel(const MmbSsmParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % S, ch = blockIdx.x * (kSsmThreads / S) + threadIdx.x / S, N = p.N;
  const bool in = ch < p.D;
  float a[PCS][VEC];
#pragma unroll
  for (int i = 0; i < PCS; ++i) {
    const int n = (i * S + lane) * VEC;
    const bool ok = in && n < N;
#pragma unroll
    for (int v = 0; v < VEC; ++v) a[i][v] = 0.f;
    if (ok) ldv<VEC>(p.A, (long long)ch * N + n, 2, a[i]);
#pragma unroll
    for (int v = 0; v < VEC; ++v) a[i][v] *= kLog2e;
  }
  const float bias = in && p.dt_bias ? p.dt_bias[ch] : 0.f, skip = in && p.Dskip ? p.Dskip[ch] : 0.f;
  const int r0 = blockIdx.y * RB;
  long long row[RB];
  float h[RB][PCS][VEC];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    row[r] = r0 + r < p.T ? pool_row(p.rows, r0 + r, p.pool_rows, p.status) : -1;
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int n = (i * S + lane) * VEC;
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[r][i][v] = 0.f;
      if (in && n < N && row[r] >= 0) ldv<VEC>(p.state, (row[r] * p.D + ch) * N + n, 2, h[r][i]);
    }
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int t = r0 + r;
    if (row[r] < 0) {
      if (p.zero_dead && t < p.T && in && lane == 0) st1(p.out, (long long)t * p.ldo + ch, p.ot, 0.f);
      continue;
    }
    const float x = in ? ld1(p.x, (long long)t * p.ldx + ch, p.xt) : 0.f;
    float d = in ? ld1(p.dt, (long long)t * p.lddt + ch, p.dtt) + bias : 0.f;
    if (p.softplus) d = softplus(d);
    const float dx = d * x;
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int n = (i * S + lane) * VEC;
      if (in && n < N) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          const float b = ld1(p.B, (long long)t * p.ldb + n + v, p.bt), c = ld1(p.C, (long long)t * p.ldc + n + v, p.bt);
          h[r][i][v] = fmaf(exp2_fast(d * a[i][v]), h[r][i][v], dx * b);
          acc = fmaf(h[r][i][v], c, acc);
        }
        stv<VEC>(p.state, (row[r] * p.D + ch) * N + n, 2, h[r][i]);
      }
    }
#pragma unroll
    for (int m = S / 2; m >= 1; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
    if (in && lane == 0) {
      float y = fmaf(skip, x, acc);
      if (p.z) y *= silu(ld1(p.z, (long long)t * p.ldz + ch, p.zt));
      st1(p.out, (long long)t * p.ldo + ch, p.ot, y);
    }
  }
}

// Raises a kernel's shared memory limit once per device (the attribute belongs to a device, not to the process).
template <typename F>
static int allow_smem(F kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return 0;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return (int)e;
}

template <int S, int NPL>
static int launch_scan(const MmbSsmParams& p, cudaStream_t stream) {
  constexpr int CH = kSsmThreads / S, TT = 8 * S;
  const bool vx = p.D % 8 == 0 && rows_aligned(p.x, p.ldx, p.xt, 8) && rows_aligned(p.dt, p.lddt, p.dtt, 8) && rows_aligned(p.z, p.ldz, p.zt, 8);
  const bool vb = (p.N * elt_bytes(p.bt)) % 16 == 0 && rows_aligned(p.B, p.ldb, p.bt, 8) && rows_aligned(p.C, p.ldc, p.bt, 8);
  const bool vo = p.D % 8 == 0 && rows_aligned(p.out, p.ldo, p.ot, 8);
  const int nb = (p.D + CH - 1) / CH;
  const long long blocks = (long long)nb * (p.S + 1);
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  const SsmLayout L = ssm_layout(TT, CH, p.N, S * NPL, elt_bytes(p.xt), elt_bytes(p.dtt), p.z ? elt_bytes(p.zt) : 0, elt_bytes(p.bt));
  static std::atomic<unsigned long long> done{0};
  // the largest this instance can ask for: fp32 activations, all of its states
  const int e = allow_smem(ssm_scan_kernel<S, NPL>, ssm_layout(TT, CH, S * NPL, S * NPL, 4, 4, 4, 4).total, done);
  if (e) return e;
  return launch(ssm_scan_kernel<S, NPL>, dim3((unsigned)blocks), dim3(kSsmThreads), (size_t)L.total, stream, 1, p, nb, (int)vx, (int)vb, (int)vo);
}

template <int S, int VEC, int PCS>
static int launch_step(const MmbSsmParams& p, cudaStream_t stream) {
  const unsigned gx = (unsigned)((p.D + kSsmThreads / S - 1) / (kSsmThreads / S));
  const bool many = (long long)gx * p.T >= 8192;
  const long long gy = many ? ((long long)p.T + 1) / 2 : p.T;
  if (gy > 65535) return (int)cudaErrorInvalidValue;
  if (many) return launch(ssm_step_kernel<S, VEC, PCS, 2>, dim3(gx, (unsigned)gy), dim3(kSsmThreads), 0, stream, 1, p);
  return launch(ssm_step_kernel<S, VEC, PCS, 1>, dim3(gx, (unsigned)gy), dim3(kSsmThreads), 0, stream, 1, p);
}

}  // namespace mmb

MMB_API int mmb_ssm_scan(const MmbSsmParams* pp, cudaStream_t stream) {
  const MmbSsmParams& p = *pp;
  if (p.T <= 0 || p.D <= 0) return 0;
  if (p.S < 0 || p.N < 1 || p.N > 128 || p.cu_seqlens == nullptr) return (int)cudaErrorInvalidValue;
  if (p.N <= 8) return mmb::launch_scan<4, 2>(p, stream);
  if (p.N <= 16) return mmb::launch_scan<4, 4>(p, stream);
  if (p.N <= 32) return mmb::launch_scan<8, 4>(p, stream);
  if (p.N <= 64) return mmb::launch_scan<8, 8>(p, stream);
  return mmb::launch_scan<8, 16>(p, stream);
}

MMB_API int mmb_ssm_step(const MmbSsmParams* pp, cudaStream_t stream) {
  const MmbSsmParams& p = *pp;
  if (p.T <= 0 || p.D <= 0) return 0;
  if (p.N < 1 || p.N > 128 || p.state == nullptr) return (int)cudaErrorInvalidValue;
  const bool vec = p.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % 16 == 0 && reinterpret_cast<uintptr_t>(p.A) % 16 == 0;
  if (vec && p.N <= 16) return mmb::launch_step<4, 4, 1>(p, stream);
  if (vec && p.N <= 32) return mmb::launch_step<8, 4, 1>(p, stream);
  if (vec) return mmb::launch_step<16, 4, 2>(p, stream);
  return p.N <= 32 ? mmb::launch_step<16, 1, 2>(p, stream) : mmb::launch_step<16, 1, 8>(p, stream);
}
