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
#include <cstdlib>

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
// log(1 + e^v) = max(v, 0) + log1p(e), e = e^-|v| in (0, 1]: no overflow, and small steps keep their relative accuracy.  log1p(e) / e is smooth on
// [0, 1] (its singularity lies at -1), so a polynomial of degree 8 fitted to it is within 2^-24.9; with the roundings of its evaluation 2^-22.4.
__device__ __forceinline__ float softplus(float v) {
  const float e = exp2_fast(-kLog2e * fabsf(v));
  float q = 0.0052326880395412445f;
  q = fmaf(q, e, -0.029505213722586632f);
  q = fmaf(q, e, 0.07822591066360474f);
  q = fmaf(q, e, -0.13663242757320404f);
  q = fmaf(q, e, 0.19106005132198334f);
  q = fmaf(q, e, -0.2484298199415207f);
  q = fmaf(q, e, 0.3331909775733948f);
  q = fmaf(q, e, -0.4999949336051941f);
  q = fmaf(q, e, 0.9999999403953552f);
  return fmaf(q, e, fmaxf(v, 0.f));
}

// Two fp32 values in one 64-bit register: Blackwell multiplies and adds such pairs with one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float a, float b) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}

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
  int x, dt, z, b, c, stage, step, bf, cf, y, total;
};
__host__ __device__ inline SsmLayout ssm_layout(int TT, int CH, int NP, int xb, int dtb, int zb, int bb) {
  SsmLayout l;
  int at = 0;
  l.x = at, at += TT * CH * xb;
  l.dt = at, at += TT * CH * dtb;
  l.z = at, at += TT * CH * zb;
  l.b = at, at += TT * NP * bb;             // rows padded to NP values
  l.c = at, at += TT * NP * bb;
  l.stage = at;
  at *= 2;
  l.step = at, at += TT * CH * 16;          // {d, d, d x, d x}: both halves of the packed factors in one load
  l.bf = at, at += bb == 4 ? 0 : TT * NP * 4;   // fp32 tiles are used where they arrive
  l.cf = at, at += bb == 4 ? 0 : TT * NP * 4;
  l.y = at, at += TT * (CH + 8) * 4;        // the padding spreads the tokens that a warp writes at once over the banks
  l.total = at;
  return l;
}

template <int S, int NPL>
__global__ void __launch_bounds__(kSsmThreads) ssm_scan_kernel(const MmbSsmParams p, int n_blocks, int vec_x, int vec_bc, int vec_out) {
  constexpr int CH = kSsmThreads / S, TT = 8 * S, NP = S * NPL, YS = CH + 8;
  extern __shared__ __align__(16) unsigned char sm[];
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
  const SsmLayout L = ssm_layout(TT, CH, NP, xb, dtb, zb, bb);
  float4* steps = reinterpret_cast<float4*>(sm + L.step);
  float* bf = reinterpret_cast<float*>(sm + L.bf);
  float* cf = reinterpret_cast<float*>(sm + L.cf);
  float* yt = reinterpret_cast<float*>(sm + L.y);

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
    fetch(st + L.b, p.B, p.ldb, bb, 0, NP, N, t0, vec_bc);
    fetch(st + L.c, p.C, p.ldc, bb, 0, NP, N, t0, vec_bc);
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
  // this lane's states: channel ch, states s NPL .. s NPL + NPL - 1, in pairs
  const int lane = tid & 31, s = lane % S, cl = (tid >> 5) * (32 / S) + lane / S, ch = c0 + cl;
  f32x2 h[NPL / 2], a[NPL / 2];
  const bool old = p.state && !(p.fresh && p.fresh[seq]);
#pragma unroll
  for (int j = 0; j < NPL / 2; ++j) {
    float av[2], hv[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int n = s * NPL + 2 * j + e;
      const bool in = ch < p.D && n < N;
      av[e] = in ? p.A[(long long)ch * N + n] * kLog2e : 0.f;
      hv[e] = in && old ? p.state[(row * p.D + ch) * N + n] : 0.f;
    }
    a[j] = pack2(av[0], av[1]);
    h[j] = pack2(hv[0], hv[1]);
  }
  auto token = [&](int t) {
    const ulonglong2 dd = *reinterpret_cast<const ulonglong2*>(steps + t * CH + cl);
    f32x2 b[NPL / 2], c[NPL / 2];
    const float *bp = bf + t * NP + s * NPL, *cp = cf + t * NP + s * NPL;
    if constexpr (NPL == 2) {
      b[0] = *reinterpret_cast<const f32x2*>(bp);
      c[0] = *reinterpret_cast<const f32x2*>(cp);
    } else {
#pragma unroll
      for (int j = 0; j < NPL / 4; ++j) {
        const ulonglong2 u = reinterpret_cast<const ulonglong2*>(bp)[j], w = reinterpret_cast<const ulonglong2*>(cp)[j];
        b[2 * j] = u.x, b[2 * j + 1] = u.y, c[2 * j] = w.x, c[2 * j + 1] = w.y;
      }
    }
    f32x2 acc = 0;
#pragma unroll
    for (int j = 0; j < NPL / 2; ++j) {
      const float2 x = unpack2(mul2(dd.x, a[j]));
      h[j] = fma2(pack2(exp2_fast(x.x), exp2_fast(x.y)), h[j], mul2(dd.y, b[j]));
      acc = j ? fma2(h[j], c[j], acc) : mul2(h[j], c[j]);
    }
    const float2 y = unpack2(acc);
    return y.x + y.y;
  };

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
      for (int i = 0; i < 8; ++i) d[i] += bias[i];
      if (p.softplus) {
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = softplus(d[i]);
      }
      float4* dst = steps + tid * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) dst[i] = make_float4(d[i], d[i], d[i] * x[i], d[i] * x[i]);
      if (bb == 4) {
        bf = reinterpret_cast<float*>(st + L.b);
        cf = reinterpret_cast<float*>(st + L.c);
      } else {
        for (int i = tid; i < TT * NP / 4; i += kSsmThreads) {
          float v[4];
          ldv<4>(st + L.b, 4 * i, p.bt, v);
          reinterpret_cast<float4*>(bf)[i] = make_float4(v[0], v[1], v[2], v[3]);
          ldv<4>(st + L.c, 4 * i, p.bt, v);
          reinterpret_cast<float4*>(cf)[i] = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
    }
    __syncthreads();
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
      yt[(g + s) * YS + cl] = v[0];
    }
    __syncthreads();
    if (vt < valid) {
      float x[8], y[8];
      ldv<8>(st + L.x, tid * 8, p.xt, x);
      ldv<8>(yt, vt * YS + vc, 2, y);
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = fmaf(skip[i], x[i], y[i]);
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
    for (int j = 0; j < NPL / 2; ++j) {
      const float2 v = unpack2(h[j]);
      const int n = s * NPL + 2 * j;
      if (ch < p.D && n < N) p.state[(row * p.D + ch) * N + n] = v.x;
      if (ch < p.D && n + 1 < N) p.state[(row * p.D + ch) * N + n + 1] = v.y;
    }
  }
}

// S lanes a channel, each PCS pieces of VEC states (4: 16 bytes), RB rows.
template <int S, int VEC, int PCS, int RB>
__global__ void __launch_bounds__(kSsmThreads) ssm_step_kernel(const MmbSsmParams p) {
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x % S, ch = blockIdx.x * (kSsmThreads / S) + threadIdx.x / S, N = p.N;
  const bool in = ch < p.D;
  const int r0 = blockIdx.y * RB;
  long long row[RB];
#pragma unroll
  for (int r = 0; r < RB; ++r) row[r] = r0 + r < p.T ? pool_row(p.rows, r0 + r, p.pool_rows, p.status) : -1;
  float h[RB][PCS][VEC], a[PCS][VEC];
#pragma unroll
  for (int r = 0; r < RB; ++r)
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int n = (i * S + lane) * VEC;
#pragma unroll
      for (int v = 0; v < VEC; ++v) h[r][i][v] = 0.f;
      if (in && n < N && row[r] >= 0) ldv<VEC>(p.state, (row[r] * p.D + ch) * N + n, 2, h[r][i]);
    }
#pragma unroll
  for (int i = 0; i < PCS; ++i) {
    const int n = (i * S + lane) * VEC;
#pragma unroll
    for (int v = 0; v < VEC; ++v) a[i][v] = 0.f;
    if (in && n < N) ldv<VEC>(p.A, (long long)ch * N + n, 2, a[i]);
  }
  const float bias = in && p.dt_bias ? p.dt_bias[ch] : 0.f, skip = in && p.Dskip ? p.Dskip[ch] : 0.f;
  // everything of the rows in flight before the first conversion waits for its data
  uint32_t xr[RB], dr[RB], zr[RB], br[RB][PCS][VEC], cr[RB][PCS][VEC];
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const long long t = r0 + r;
    if (!in || row[r] < 0) continue;
    xr[r] = bits1(p.x, t * p.ldx + ch, p.xt);
    dr[r] = bits1(p.dt, t * p.lddt + ch, p.dtt);
    if (p.z) zr[r] = bits1(p.z, t * p.ldz + ch, p.zt);
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int n = (i * S + lane) * VEC;
      if (n < N) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) br[r][i][v] = bits1(p.B, t * p.ldb + n + v, p.bt), cr[r][i][v] = bits1(p.C, t * p.ldc + n + v, p.bt);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < RB; ++r) {
    const int t = r0 + r;
    if (row[r] < 0) {
      if (p.zero_dead && t < p.T && in && lane == 0) st1(p.out, (long long)t * p.ldo + ch, p.ot, 0.f);
      continue;
    }
    const float x = in ? value1(xr[r], p.xt) : 0.f;
    float d = in ? value1(dr[r], p.dtt) + bias : 0.f;
    if (p.softplus) d = softplus(d);
    const float dx = d * x, dl = d * kLog2e;
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int n = (i * S + lane) * VEC;
      if (in && n < N) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
          h[r][i][v] = fmaf(exp2_fast(dl * a[i][v]), h[r][i][v], dx * value1(br[r][i][v], p.bt));
          acc = fmaf(h[r][i][v], value1(cr[r][i][v], p.bt), acc);
        }
        stv<VEC>(p.state, (row[r] * p.D + ch) * N + n, 2, h[r][i]);
      }
    }
#pragma unroll
    for (int m = S / 2; m >= 1; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
    if (in && lane == 0) {
      float y = fmaf(skip, x, acc);
      if (p.z) y *= silu(value1(zr[r], p.zt));
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
  const SsmLayout L = ssm_layout(TT, CH, S * NPL, elt_bytes(p.xt), elt_bytes(p.dtt), p.z ? elt_bytes(p.zt) : 0, elt_bytes(p.bt));
  static std::atomic<unsigned long long> done{0};
  // the largest this instance can ask for: fp32 activations, all of its states
  const int e = allow_smem(ssm_scan_kernel<S, NPL>, ssm_layout(TT, CH, S * NPL, 4, 4, 4, 4).total, done);
  if (e) return e;
  // not a programmatic dependent launch: blocks that start while the previous kernel drains pile up on the SMs that it leaves first, and a scan
  // has too few blocks to even that out (4096 tokens, 8192 channels back to back: 1132 us against 837 us for a lone one, first version)
  ssm_scan_kernel<S, NPL><<<(unsigned)blocks, kSsmThreads, (size_t)L.total, stream>>>(p, nb, (int)vx, (int)vb, (int)vo);
  return (int)cudaGetLastError();
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
  const char* ev = getenv("SSM_V"); const int v = ev ? atoi(ev) : 0;
  if (p.N <= 8) return mmb::launch_scan<4, 2>(p, stream);
  if (p.N <= 16) return v == 1 ? mmb::launch_scan<2, 8>(p, stream) : v == 2 ? mmb::launch_scan<8, 2>(p, stream) : mmb::launch_scan<4, 4>(p, stream);
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
