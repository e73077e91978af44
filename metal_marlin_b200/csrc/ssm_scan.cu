// Selective state space scan over a pool of per-sequence states:
//   d_t = softplus(dt_t + dt_bias)                       (or dt_t itself)
//   h_t[n] = exp(d_t A[c, n]) h_{t-1}[n] + d_t x_t B_t[n]
//   out_t = (sum_n h_t[n] C_t[n] + D[c] x_t) silu(z_t)
// with h fp32 in state[row, c, 0 .. N - 1], read when a sequence starts (zero when it is fresh) and written when it ends.
//
// Prompts.  Every step of every state takes one exponential and four fp32 operations; at 16 exponentials a clock and SM the special function
// unit bounds the scan (16 states, 16-bit activations: 3 x longer than moving the activations through memory), closely followed by the
// 32 bytes a clock that shared memory returns to each scheduler's registers (8 bytes of B and C a state).  The recurrence itself is one
// multiply-add deep.  The work is split over channels and over the STATES of a channel, never over time: a second pass over time would
// double the exponentials, which is too much where they bound the scan.  It is what a narrow layer would need, whose few warps wait for one another's
// latency and leave that unit idle (2048 tokens of 1024 channels, 16 states: 56 us, the exponentials 7, the bytes 3; 8192 of 64: 210 us).  S lanes
// share a channel, each with NPL states in registers (of R channels where there are lanes to spare).  A block
// owns 32 W / S R channels of one sequence and walks it in tiles of 32 or 64 tokens with two roles that meet at named barriers, tile by tile:
//   * ST / 32 staging warps: the tile's x, dt, z, B, C arrive raw by 16-byte cp.async two tiles ahead; they turn x and dt into (d, d x) pairs, so
//     softplus is paid once per value and not once per lane, and later add the skip term, apply the gate and store the outputs;
//   * W scanning warps: G tokens at a time, all their exponentials before the recurrence, the next group's loads before both; partial sums of S
//     tokens are added over the S lanes by a transposing butterfly (S - 1 shuffles for S tokens) that leaves every lane with the sum of one token.
// What it took (4096 tokens of 8192 channels, 16 states, bf16): one role with runtime types 1132 us; blocks spread evenly over the SMs and loads of a
// batch issued before their conversions 772 -> 547; types at compile time, conflict-free staging 386; the two roles 327; groups of four
// tokens, unrolled 262; seven scanning warps on every SM instead of eight on most 244 us.
// exp(d A) is taken as 2^(d (A log2 e)); A log2 e is rounded once, which shifts every exponent by the same relative 2^-24.
//
// Single tokens.  The state is the traffic: see ssm_step_kernel.
#include <atomic>

#include "api_ext.h"
#include "launch.h"
#include "typed_io.cuh"

namespace mmb {

constexpr int kStepThreads = 128;
constexpr int kSsmSorted = 16;              // up to this many sequences are ordered by length
constexpr int kSsmSpread = 4;               // up to this many blocks an SM are all resident and spread evenly
constexpr float kLog2e = 1.4426950408889634f;

// log(1 + e^v) = max(v, 0) + log1p(e), e = e^-|v| in (0, 1]: no overflow, and small steps keep their relative accuracy.  log1p(e) / e is smooth on
// [0, 1] (its singularity lies at -1), so a polynomial of degree 8 fitted to it is, with its coefficients rounded to fp32, within 2^-23.7 of the value; with the roundings of its
// evaluation within 2^-22.4.
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

// softplus of two values; the polynomial takes one instruction a step for both.
__device__ __forceinline__ void softplus2(float (&v)[2]) {
  const float e0 = exp2_fast(-kLog2e * fabsf(v[0])), e1 = exp2_fast(-kLog2e * fabsf(v[1]));
  const f32x2 e = pack2(e0, e1);
  auto both = [](float c) { return pack2(c, c); };
  f32x2 q = both(0.0052326880395412445f);
  q = fma2(q, e, both(-0.029505213722586632f));
  q = fma2(q, e, both(0.07822591066360474f));
  q = fma2(q, e, both(-0.13663242757320404f));
  q = fma2(q, e, both(0.19106005132198334f));
  q = fma2(q, e, both(-0.2484298199415207f));
  q = fma2(q, e, both(0.3331909775733948f));
  q = fma2(q, e, both(-0.4999949336051941f));
  q = fma2(q, e, both(0.9999999403953552f));
  const float2 f = unpack2(fma2(q, e, pack2(fmaxf(v[0], 0.f), fmaxf(v[1], 0.f))));
  v[0] = f.x, v[1] = f.y;
}
// y silu(z) for two values
__device__ __forceinline__ void gate2(float (&y)[2], const float (&z)[2]) {
  const f32x2 zz = pack2(z[0], z[1]);
  float2 f = unpack2(mul2(zz, pack2(-kLog2e, -kLog2e)));
  f = unpack2(add2(pack2(exp2_fast(f.x), exp2_fast(f.y)), pack2(1.f, 1.f)));
  f = unpack2(mul2(mul2(zz, pack2(rcp_fast(f.x), rcp_fast(f.y))), pack2(y[0], y[1])));
  y[0] = f.x, y[1] = f.y;
}

// Sums v[i] over the S lanes of a group for i < S; lane s of the group ends with the sums of v[s] in v[0].
template <int S, int R>
__device__ __forceinline__ void transposed_sum(float (&v)[S][R], int s) {
#pragma unroll
  for (int m = S / 2; m >= 1; m >>= 1) {
    const bool up = s & m;
#pragma unroll
    for (int i = 0; i < m; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float send = up ? v[i][r] : v[i + m][r], keep = up ? v[i + m][r] : v[i][r];
        v[i][r] = keep + __shfl_xor_sync(0xffffffffu, send, m);
      }
  }
}

__device__ __forceinline__ void ld2(const void* p, int i, int t, float* v) {
  if (t == 2) {
    const float2 f = *reinterpret_cast<const float2*>(reinterpret_cast<const float*>(p) + i);
    v[0] = f.x, v[1] = f.y;
  } else {
    const uint32_t w = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const uint16_t*>(p) + i);
    unpack16<2>(&w, t, v);
  }
}
__device__ __forceinline__ void st2(void* p, long long i, int t, const float* v) {
  if (t == 2) *reinterpret_cast<float2*>(reinterpret_cast<float*>(p) + i) = make_float2(v[0], v[1]);
  else *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(p) + i) = pack16(v[0], v[1], t);
}

// N consecutive floats of shared memory, N a power of two or less than five, by the widest loads.
template <int N>
__device__ __forceinline__ void lds(const float* p, float* v) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const float4 f = reinterpret_cast<const float4*>(p)[i];
      v[4 * i] = f.x, v[4 * i + 1] = f.y, v[4 * i + 2] = f.z, v[4 * i + 3] = f.w;
    }
  } else if constexpr (N == 2) {
    const float2 f = *reinterpret_cast<const float2*>(p);
    v[0] = f.x, v[1] = f.y;
  } else {
    v[0] = *p;
  }
}
// Partial sums of SG tokens: SG / S times S tokens are summed over the S lanes of a channel, lane s stores token s of them.
template <int S, int R, int SG, int YS>
__device__ __forceinline__ void emit(float (&v)[SG][R], int s, float* yt) {
#pragma unroll
  for (int k = 0; k < SG; k += S) {
    float w[S][R];
#pragma unroll
    for (int i = 0; i < S; ++i)
#pragma unroll
      for (int r = 0; r < R; ++r) w[i][r] = v[k + i][r];
    transposed_sum<S, R>(w, s);
    float* y = yt + k * YS;
    if constexpr (R == 4) *reinterpret_cast<float4*>(y) = make_float4(w[0][0], w[0][1], w[0][2], w[0][3]);
    else if constexpr (R == 2) *reinterpret_cast<float2*>(y) = make_float2(w[0][0], w[0][1]);
    else *y = w[0][0];
  }
}

template <int V>
struct Int {
  static constexpr int value = V;
};

// Byte offsets of the parts of a block's shared memory.
struct SsmLayout {
  int x, dt, z, b, c, stage, step, bf, cf, y, total;
};
constexpr int kSsmStages = 3;               // raw tiles: one arriving, one being prepared, one whose outputs are being finished
// Row pitch of the partial outputs: eight more than a multiple of 32 spreads the tokens that a warp writes at once over the banks.
__host__ __device__ constexpr int ssm_y_pitch(int CH) { return CH < 32 ? CH + 8 : (CH + 31) / 32 * 32 + 8; }
__host__ __device__ inline SsmLayout ssm_layout(int TT, int CH, int NP, int xb, int dtb, int zb, int bb) {
  SsmLayout l;
  int at = 0;
  l.x = at, at += TT * CH * xb;
  l.dt = at, at += TT * CH * dtb;
  l.z = at, at += TT * CH * zb;
  l.b = at, at += TT * NP * bb;             // rows padded to NP values
  l.c = at, at += TT * NP * bb;
  l.stage = at;
  at *= kSsmStages;
  // two of each of the following
  l.step = at, at += 2 * TT * CH * 8;       // {d, d x}
  l.bf = at, at += bb == 4 ? 0 : 2 * TT * NP * 4;   // fp32 tiles are used where they arrive
  l.cf = at, at += bb == 4 ? 0 : 2 * TT * NP * 4;
  l.y = at, at += 2 * TT * ssm_y_pitch(CH) * 4;
  l.total = at;
  return l;
}

// Named barriers with constant numbers (a number in a register makes a block reserve all sixteen).  Full and done: one per buffer.
enum { kBarStage = 1, kBarFull = 2, kBarDone = 4 };
template <int ID, int N>
__device__ __forceinline__ void bar_sync() { asm volatile("bar.sync %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
template <int ID, int N>
__device__ __forceinline__ void bar_arrive() { asm volatile("bar.arrive %0, %1;" ::"n"(ID), "n"(N) : "memory"); }
template <int ID, int N>
__device__ __forceinline__ void bar_sync_of(int buffer) { buffer ? bar_sync<ID + 1, N>() : bar_sync<ID, N>(); }
template <int ID, int N>
__device__ __forceinline__ void bar_arrive_of(int buffer) { buffer ? bar_arrive<ID + 1, N>() : bar_arrive<ID, N>(); }

// XT: the type of x, dt, z, B, C and out where they have one type, else 3.
// W: scanning warps; ST: staging threads; TT: tokens of a tile.
template <int S, int NPL, int R, int G, int W, int ST, int TT, int XT>
__global__ void __launch_bounds__(32 * W + ST) ssm_scan_kernel(const MmbSsmParams p, int n_blocks, int vec_x, int vec_bc, int vec_out) {
  const int xt = XT < 3 ? XT : p.xt, dtt = XT < 3 ? XT : p.dtt, zt = XT < 3 ? XT : p.zt, bt = XT < 3 ? XT : p.bt, ot = XT < 3 ? XT : p.ot;
  constexpr int CH = 32 * W / S * R, NP = S * NPL, YS = ssm_y_pitch(CH), kScan = 32 * W, kAll = kScan + ST;
  constexpr int SG = 2 * G > S ? 2 * G : S;                 // tokens between two sums over the lanes: an even number of groups
  extern __shared__ __align__(16) unsigned char sm[];
  const int c0 = (blockIdx.x % n_blocks) * CH;
  int seq = blockIdx.x / n_blocks;
  auto start = [&](int s) { return min(max(p.cu_seqlens[s], 0), p.T); };
  if (p.S > 1 && p.S <= kSsmSorted && seq < p.S && (long long)n_blocks * p.S > 148 * kSsmSpread) {
    // the longest sequences first, so that none of them begins when the others end (10 sequences of 12 to 1500 tokens, 4096 channels: 165 -> 153 us;
    // shortest first 189).  Every block sorts for itself, about 1 us: not worth it for many short sequences (100 of them 94 -> 121 us).
    int* len = reinterpret_cast<int*>(sm);
    for (int i = threadIdx.x; i < p.S; i += kAll) len[i] = max(0, start(i + 1) - start(i));
    __syncthreads();
    for (int i = threadIdx.x; i < p.S; i += kAll) {
      int rank = 0;
      for (int j = 0; j < p.S; ++j) rank += len[j] > len[i] || (len[j] == len[i] && j < i);
      if (rank == seq) len[p.S] = i;
    }
    __syncthreads();
    seq = len[p.S];
    __syncthreads();
  }
  const int begin = start(seq), end = seq < p.S ? max(begin, start(seq + 1)) : p.T;
  const int front = seq < p.S ? 0 : start(0);     // the last block also has the rows in front of the first sequence
  if (begin >= end && front == 0) return;
  long long row = -1;
  bool live = seq < p.S;
  if (live && p.state) {
    row = pool_row(p.rows, seq, p.pool_rows, p.status);
    live = row >= 0;
  }
  if (!live) {                                    // rows of no live sequence
    if (p.zero_dead)
      for (long long i = threadIdx.x; i < ((long long)(end - begin) + front) * CH; i += kAll) {
        const int c = c0 + (int)(i % CH);
        const long long t = i / CH;
        if (c < p.D) st1(p.out, (t < front ? t : t - front + begin) * p.ldo + c, ot, 0.f);
      }
    return;
  }
  const int xb = elt_bytes(xt), dtb = elt_bytes(dtt), zb = p.z ? elt_bytes(zt) : 0, bb = elt_bytes(bt), N = p.N;
  const SsmLayout L = ssm_layout(TT, CH, NP, xb, dtb, zb, bb);
  const int tiles = (end - begin + TT - 1) / TT;

  if (threadIdx.x >= kScan) {
    // ------------------------------------------------------------------------------------------------ staging warps
    const int tid = threadIdx.x - kScan;
    // rows t0 .. t0 + TT of COLS columns of a [*, width] tensor into a dense raw tile; zeros outside.  16-byte pieces where the
    // rows are aligned for it: a thread's pieces lie in one column of pieces, so its addresses are one pointer and a stride.
    auto fetch16 = [&](auto cols, auto es, unsigned char* dst, const unsigned char* src, long long ld, int width, int t0) {
      constexpr int COLS = decltype(cols)::value, ES = decltype(es)::value, PER = COLS * ES / 16, RS = ST / PER;   // pieces a row, rows a pass
      const int r0 = tid / PER, q = tid % PER;
      const bool in = q * (16 / ES) < width;
      const unsigned char* g = src + (t0 + r0) * ld * ES + q * 16;
#pragma unroll
      for (int k = 0; k < (TT + RS - 1) / RS; ++k) {
        const int r = r0 + k * RS;
        if ((ST % PER == 0 || r0 < RS) && (TT % RS == 0 || r < TT)) {
          const bool ok = in && t0 + r < end;
          cp_async16(dst + (r * PER + q) * 16, ok ? g + k * RS * ld * ES : src, ok);
        }
      }
    };
    auto fetch = [&](auto cols, unsigned char* dst, const void* base, int col, long long ld, int es, int width, int t0, bool vec) {
      constexpr int COLS = decltype(cols)::value;
      const unsigned char* src = reinterpret_cast<const unsigned char*>(base) + (long long)col * es;
      width -= col;
      if (vec && COLS * es % 16 == 0) {
        if constexpr (COLS * 2 % 16 == 0) {
          if (es == 2) fetch16(cols, Int<2>{}, dst, src, ld, width, t0);
        }
        if constexpr (COLS * 4 % 16 == 0) {
          if (es == 4) fetch16(cols, Int<4>{}, dst, src, ld, width, t0);
        }
        return;
      }
      for (int i = tid; i < TT * COLS; i += ST) {
        const int r = i / COLS, q = i % COLS;
        const bool ok = t0 + r < end && q < width;
        const long long at = (long long)(t0 + r) * ld + q;
        if (es == 2) reinterpret_cast<uint16_t*>(dst)[i] = ok ? reinterpret_cast<const uint16_t*>(src)[at] : (uint16_t)0;
        else reinterpret_cast<uint32_t*>(dst)[i] = ok ? reinterpret_cast<const uint32_t*>(src)[at] : 0u;
      }
    };
    auto prefetch = [&](int i) {
      if (i < tiles) {
        const int t0 = begin + i * TT;
        unsigned char* st = sm + i % kSsmStages * L.stage;
        fetch(Int<CH>{}, st + L.x, p.x, c0, p.ldx, xb, p.D, t0, vec_x);
        fetch(Int<CH>{}, st + L.dt, p.dt, c0, p.lddt, dtb, p.D, t0, vec_x);
        if (p.z) fetch(Int<CH>{}, st + L.z, p.z, c0, p.ldz, zb, p.D, t0, vec_x);
        fetch(Int<NP>{}, st + L.b, p.B, 0, p.ldb, bb, N, t0, vec_bc);
        fetch(Int<NP>{}, st + L.c, p.C, 0, p.ldc, bb, N, t0, vec_bc);
      }
      cp_async_commit();
    };
    prefetch(0);
    prefetch(1);
    // this thread's values of a tile: channels vc, vc + 1 of the tokens vt, vt + VS, ..
    constexpr int VS = ST / (CH / 2), VN = (TT + VS - 1) / VS;
    constexpr bool kEven = ST % (CH / 2) == 0 && TT % VS == 0;            // every thread has VN tokens
    const int vt = tid / (CH / 2), vc = tid % (CH / 2) * 2;
    auto mine = [&](int k) { return kEven || (vt < VS && vt + k * VS < TT); };
    auto at = [&](int k) { return kEven ? vt + k * VS : min(vt + k * VS, TT - 1); };
    float bias[2], skip[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const bool in = c0 + vc + i < p.D;
      bias[i] = in && p.dt_bias ? p.dt_bias[c0 + vc + i] : 0.f;
      skip[i] = in && p.Dskip ? p.Dskip[c0 + vc + i] : 0.f;
    }
    // tile i: (d, d x) and fp32 B, C into buffer i & 1
    auto prepare = [&](int i) {
      const unsigned char* st = sm + i % kSsmStages * L.stage;
      float x[VN][2], d[VN][2];
#pragma unroll
      for (int k = 0; k < VN; ++k) {
        ld2(st + L.x, at(k) * CH + vc, xt, x[k]);
        ld2(st + L.dt, at(k) * CH + vc, dtt, d[k]);
      }
#pragma unroll
      for (int k = 0; k < VN; ++k) d[k][0] += bias[0], d[k][1] += bias[1];
      if (p.softplus) {
#pragma unroll
        for (int k = 0; k < VN; ++k) softplus2(d[k]);
      }
      float4* step = reinterpret_cast<float4*>(sm + L.step + (i & 1) * TT * CH * 8);
#pragma unroll
      for (int k = 0; k < VN; ++k)
        if (mine(k)) step[((vt + k * VS) * CH + vc) / 2] = make_float4(d[k][0], d[k][0] * x[k][0], d[k][1], d[k][1] * x[k][1]);
      if (bb == 2) {
        float4* bf = reinterpret_cast<float4*>(sm + L.bf) + (i & 1) * TT * NP / 4;
        float4* cf = reinterpret_cast<float4*>(sm + L.cf) + (i & 1) * TT * NP / 4;
        for (int q = tid; q < TT * NP / 4; q += ST) {
          float v[4];
          ldv<4>(st + L.b, 4 * q, bt, v);
          bf[q] = make_float4(v[0], v[1], v[2], v[3]);
          ldv<4>(st + L.c, 4 * q, bt, v);
          cf[q] = make_float4(v[0], v[1], v[2], v[3]);
        }
      }
    };
    // tile i: skip term, gate, output
    auto finish = [&](int i) {
      const unsigned char* st = sm + i % kSsmStages * L.stage;
      const float* yt = reinterpret_cast<const float*>(sm + L.y) + (i & 1) * TT * YS;
      const int t0 = begin + i * TT;
      float x[VN][2], y[VN][2];
#pragma unroll
      for (int k = 0; k < VN; ++k) {
        ld2(st + L.x, at(k) * CH + vc, xt, x[k]);
        const float2 f = *reinterpret_cast<const float2*>(yt + at(k) * YS + vc);
        y[k][0] = f.x, y[k][1] = f.y;
      }
#pragma unroll
      for (int k = 0; k < VN; ++k) y[k][0] = fmaf(skip[0], x[k][0], y[k][0]), y[k][1] = fmaf(skip[1], x[k][1], y[k][1]);
      if (p.z) {
        float z[VN][2];
#pragma unroll
        for (int k = 0; k < VN; ++k) ld2(st + L.z, at(k) * CH + vc, zt, z[k]);
#pragma unroll
        for (int k = 0; k < VN; ++k) gate2(y[k], z[k]);
      }
#pragma unroll
      for (int k = 0; k < VN; ++k) {
        if (mine(k) && t0 + vt + k * VS < end) {
          const long long at = (long long)(t0 + vt + k * VS) * p.ldo + c0 + vc;
          if (vec_out) {
            if (c0 + vc < p.D) st2(p.out, at, ot, y[k]);
          } else {
            if (c0 + vc < p.D) st1(p.out, at, ot, y[k][0]);
            if (c0 + vc + 1 < p.D) st1(p.out, at + 1, ot, y[k][1]);
          }
        }
      }
    };
    for (int i = 0; i < tiles; ++i) {
      cp_async_wait<1>();
      bar_sync<kBarStage, ST>();           // raw tile i is there
      prepare(i);
      bar_arrive_of<kBarFull, kAll>(i & 1);
      if (i > 0) {
        bar_sync_of<kBarDone, kAll>((i - 1) & 1);
        finish(i - 1);
      }
      bar_sync<kBarStage, ST>();           // everybody is done with raw tile i - 1
      prefetch(i + 2);
    }
    bar_sync_of<kBarDone, kAll>((tiles - 1) & 1);
    finish(tiles - 1);
    return;
  }

  // -------------------------------------------------------------------------------------------------- scanning warps
  // This lane: channels c0 + cl .. + R - 1, states s NPL .. s NPL + NPL - 1 of each.  The loads of the next G tokens are issued before the
  // exponentials of these, so that one warp alone keeps the special function unit busy.
  const int tid = threadIdx.x, lane = tid & 31, s = lane % S, cl = ((tid >> 5) * (32 / S) + lane / S) * R;
  float h[R][NPL], a[R][NPL];
  const bool old = p.state && !(p.fresh && p.fresh[seq]);
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int n = s * NPL + j, ch = c0 + cl + r;
      const bool in = ch < p.D && n < N;
      a[r][j] = in ? p.A[(long long)ch * N + n] * kLog2e : 0.f;
      h[r][j] = in && old ? p.state[(row * p.D + ch) * N + n] : 0.f;
    }
  struct Loaded {
    float d[G][R][2], b[G][NPL], c[G][NPL];
  };
  auto load = [&](const float2* step, const float* bp, const float* cp, int t, Loaded& v) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      lds<2 * R>(reinterpret_cast<const float*>(step + (t + g) * CH), &v.d[g][0][0]);
      lds<NPL>(bp + (t + g) * NP, v.b[g]);
      lds<NPL>(cp + (t + g) * NP, v.c[g]);
    }
  };
  // `n` of the G loaded tokens are there
  auto advance = [&](const Loaded& v, int n, float (*out)[R]) {
    float e[G][R][NPL];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < NPL; ++j) e[g][r][j] = exp2_fast(v.d[g][r][0] * a[r][j]);
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int r = 0; r < R; ++r) {
        out[g][r] = 0.f;
        if (g < n) {
          if constexpr (NPL % 2 == 0) {
            f32x2 acc = 0;
#pragma unroll
            for (int j = 0; j < NPL; j += 2) {
              const f32x2 u = pack2(v.d[g][r][1] * v.b[g][j], v.d[g][r][1] * v.b[g][j + 1]);
              const f32x2 hn = fma2(pack2(e[g][r][j], e[g][r][j + 1]), pack2(h[r][j], h[r][j + 1]), u);
              const f32x2 c = pack2(v.c[g][j], v.c[g][j + 1]);
              acc = j ? fma2(hn, c, acc) : mul2(hn, c);
              const float2 f = unpack2(hn);
              h[r][j] = f.x, h[r][j + 1] = f.y;
            }
            const float2 y = unpack2(acc);
            out[g][r] = y.x + y.y;
          } else {
#pragma unroll
            for (int j = 0; j < NPL; ++j) {
              h[r][j] = fmaf(e[g][r][j], h[r][j], v.d[g][r][1] * v.b[g][j]);
              out[g][r] = j ? fmaf(h[r][j], v.c[g][j], out[g][r]) : h[r][j] * v.c[g][j];
            }
          }
        }
      }
  };
  for (int i = 0; i < tiles; ++i) {
    const int valid = min(TT, end - begin - i * TT);
    const float2* step = reinterpret_cast<const float2*>(sm + L.step + (i & 1) * TT * CH * 8) + cl;
    const float* bp = (bb == 4 ? reinterpret_cast<const float*>(sm + i % kSsmStages * L.stage + L.b) : reinterpret_cast<const float*>(sm + L.bf) + (i & 1) * TT * NP) + s * NPL;
    const float* cp = (bb == 4 ? reinterpret_cast<const float*>(sm + i % kSsmStages * L.stage + L.c) : reinterpret_cast<const float*>(sm + L.cf) + (i & 1) * TT * NP) + s * NPL;
    float* yt = reinterpret_cast<float*>(sm + L.y) + (i & 1) * TT * YS + s * YS + cl;
    bar_sync_of<kBarFull, kAll>(i & 1);
    if (valid == TT) {
      Loaded ld[2];
      load(step, bp, cp, 0, ld[0]);
#pragma unroll
      for (int t = 0; t < TT; t += SG) {
        float v[SG][R];
#pragma unroll
        for (int k = 0; k < SG; k += G) {
          if (k + G < SG || t + SG < TT) load(step, bp, cp, t + k + G, ld[(k / G + 1) & 1]);
          advance(ld[(k / G) & 1], G, v + k);
        }
        emit<S, R, SG, YS>(v, s, yt + t * YS);
      }
    } else {
      for (int t = 0; t < valid; t += SG) {
        float v[SG][R];
#pragma unroll
        for (int k = 0; k < SG; k += G) {
          Loaded ld;
          load(step, bp, cp, t + k, ld);
          advance(ld, valid - t - k, v + k);
        }
        emit<S, R, SG, YS>(v, s, yt + t * YS);
      }
    }
    bar_arrive_of<kBarDone, kAll>(i & 1);
  }
  if (p.state) {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int j = 0; j < NPL; ++j) {
        const int n = s * NPL + j, ch = c0 + cl + r;
        if (ch < p.D && n < N) p.state[(row * p.D + ch) * N + n] = h[r][j];
      }
  }
}

// Inputs of the single-token kernel as raw bits.  XT: the type of x, dt, z, B and C where they have one type and whole pieces can be
// loaded, else 3; a choice at run time around every load would keep the loads from being issued together.
template <int XT, int W>
__device__ __forceinline__ void ld_quad(const void* p, long long i, int n, int t, uint32_t (&w)[W]) {
  if constexpr (XT < 2) {
    const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
    w[0] = u.x, w[1] = u.y;
  } else if constexpr (XT == 2) {
    const uint4 u = *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
#pragma unroll
    for (int v = 0; v < 4; ++v) w[v] = v < n ? bits1(p, i + v, t) : 0u;
  }
}
template <int XT, int W>
__device__ __forceinline__ void quad_values(const uint32_t (&w)[W], int t, float (&v)[4]) {
  if constexpr (XT < 2) {
    unpack16<4>(w, XT, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = XT == 2 ? __uint_as_float(w[e]) : value1(w[e], t);
  }
}
template <int XT>
__device__ __forceinline__ uint32_t ld_bits(const void* p, long long i, int t) {
  if constexpr (XT < 2) return reinterpret_cast<const uint16_t*>(p)[i];
  if constexpr (XT == 2) return reinterpret_cast<const uint32_t*>(p)[i];
  return bits1(p, i, t);
}

// S lanes a channel, each PCS pieces of four states; a block owns `per` neighbouring groups of channels of one row.  What bounds it is the state
// (read and written once); what keeps it from the memory's rate is the work around it, softplus, gate and sums, which every lane of a channel
// repeats: two pieces a lane instead of one together with the walk along the row make it 55 us, 4.8 TB/s (256 rows of 8192 channels, 16 states;
// walking the rows of one group of channels with A in registers instead, 65 us: the accesses of neighbouring blocks lie further apart).  Inputs of several
// types take the form XT = 3, which also moves the state and A by single values: bf16 x with fp32 dt, B and C 99 us.
template <int S, int PCS, int XT>
__global__ void __launch_bounds__(kStepThreads) ssm_step_kernel(const MmbSsmParams p, int per) {
  const int xt = XT < 3 ? XT : p.xt, dtt = XT < 3 ? XT : p.dtt, zt = XT < 3 ? XT : p.zt, bt = XT < 3 ? XT : p.bt;
  constexpr int CB = kStepThreads / S;
  const int lane = threadIdx.x % S, N = p.N, t = blockIdx.y;
  const int ch0 = blockIdx.x * per * CB + threadIdx.x / S;
  pdl_launch_dependents();
  pdl_wait();
  const long long row = pool_row(p.rows, t, p.pool_rows, p.status);
  if (row < 0) {
    if (p.zero_dead)
      for (int k = 0; k < per; ++k)
        if (ch0 + k * CB < p.D && lane == 0) st1(p.out, (long long)t * p.ldo + ch0 + k * CB, p.ot, 0.f);
    return;
  }
  float b[PCS][4], c[PCS][4];
#pragma unroll
  for (int i = 0; i < PCS; ++i) {
    const int n = (i * S + lane) * 4;
    uint32_t bw[XT < 2 ? 2 : 4] = {}, cw[XT < 2 ? 2 : 4] = {};
    if (n < N) {
      ld_quad<XT>(p.B, (long long)t * p.ldb + n, N - n, bt, bw);
      ld_quad<XT>(p.C, (long long)t * p.ldc + n, N - n, bt, cw);
    }
    quad_values<XT>(bw, bt, b[i]);
    quad_values<XT>(cw, bt, c[i]);
  }
  struct In {
    float h[PCS][4], a[PCS][4], bias, skip;
    uint32_t x, dt, z;
  };
  auto load = [&](int ch, In& q) {
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int n = (i * S + lane) * 4;
      if (n < N) {
        const float *hs = p.state + (row * p.D + ch) * N + n, *as = p.A + (long long)ch * N + n;
        if constexpr (XT < 3) {
          const float4 f = *reinterpret_cast<const float4*>(hs), g = *reinterpret_cast<const float4*>(as);
          q.h[i][0] = f.x, q.h[i][1] = f.y, q.h[i][2] = f.z, q.h[i][3] = f.w;
          q.a[i][0] = g.x, q.a[i][1] = g.y, q.a[i][2] = g.z, q.a[i][3] = g.w;
        } else {
#pragma unroll
          for (int v = 0; v < 4; ++v) q.h[i][v] = n + v < N ? hs[v] : 0.f, q.a[i][v] = n + v < N ? as[v] : 0.f;
        }
      }
    }
    q.dt = ld_bits<XT>(p.dt, (long long)t * p.lddt + ch, dtt);
    q.x = ld_bits<XT>(p.x, (long long)t * p.ldx + ch, xt);
    if (p.z) q.z = ld_bits<XT>(p.z, (long long)t * p.ldz + ch, zt);
    q.bias = p.dt_bias ? p.dt_bias[ch] : 0.f;
    q.skip = p.Dskip ? p.Dskip[ch] : 0.f;
  };
  for (int k = 0; k < per; ++k) {
    const int ch = ch0 + k * CB;
    const bool in = ch < p.D;
    In v;
    if (in) load(ch, v);
    const float x = in ? value1(v.x, xt) : 0.f;
    float d = in ? value1(v.dt, dtt) + v.bias : 0.f;
    if (p.softplus) d = softplus(d);
    const float dx = d * x, dl = d * kLog2e;
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < PCS; ++i) {
      const int n = (i * S + lane) * 4;
      if (in && n < N) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          v.h[i][e] = fmaf(exp2_fast(dl * v.a[i][e]), v.h[i][e], dx * b[i][e]);
          if (XT < 3 || n + e < N) acc = fmaf(v.h[i][e], c[i][e], acc);
        }
        float* dst = p.state + (row * p.D + ch) * N + n;
        if constexpr (XT < 3) {
          *reinterpret_cast<float4*>(dst) = make_float4(v.h[i][0], v.h[i][1], v.h[i][2], v.h[i][3]);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (n + e < N) dst[e] = v.h[i][e];
        }
      }
    }
#pragma unroll
    for (int m = S / 2; m >= 1; m >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, m);
    if (in && lane == 0) {
      float y = fmaf(v.skip, x, acc);
      if (p.z) y *= silu(value1(v.z, zt));
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

template <int S, int NPL, int R, int G, int W, int ST, int TT, int XT>
static int launch_scan_t(const MmbSsmParams& p, cudaStream_t stream) {
  constexpr int CH = 32 * W / S * R;
  const bool vx = p.D % 8 == 0 && rows_aligned(p.x, p.ldx, p.xt, 8) && rows_aligned(p.dt, p.lddt, p.dtt, 8) && rows_aligned(p.z, p.ldz, p.zt, 8);
  const bool vb = (p.N * elt_bytes(p.bt)) % 16 == 0 && rows_aligned(p.B, p.ldb, p.bt, 8) && rows_aligned(p.C, p.ldc, p.bt, 8);
  const bool vo = p.D % 2 == 0 && rows_aligned(p.out, p.ldo, p.ot, 2);
  const int nb = (p.D + CH - 1) / CH;
  const long long blocks = (long long)nb * (p.S + 1);
  if (blocks > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
  size_t smem = ssm_layout(TT, CH, S * NPL, elt_bytes(p.xt), elt_bytes(p.dtt), p.z ? elt_bytes(p.zt) : 0, elt_bytes(p.bt)).total;
  // a grid of a few blocks a SM is not spread evenly by itself: ask for so much shared memory that no SM takes more than its share
  constexpr int kSmem = 227 * 1024;
  const long long share = ((long long)nb * p.S + 147) / 148;
  if (share >= 1 && share <= kSsmSpread) smem = max(smem, (size_t)(kSmem / share - 1024) / 128 * 128);
  static std::atomic<unsigned long long> done{0};
  const int e = allow_smem(ssm_scan_kernel<S, NPL, R, G, W, ST, TT, XT>, kSmem, done);
  if (e) return e;
  // not a programmatic dependent launch: blocks that start while the previous kernel drains pile up on the SMs that it leaves first, and a scan
  // has too few blocks to even that out
  ssm_scan_kernel<S, NPL, R, G, W, ST, TT, XT><<<(unsigned)blocks, 32 * W + ST, smem, stream>>>(p, nb, (int)vx, (int)vb, (int)vo);
  return (int)cudaGetLastError();
}
template <int S, int NPL, int R, int G, int W, int ST, int TT>
static int launch_scan_w(const MmbSsmParams& p, cudaStream_t stream) {
  const bool same = p.dtt == p.xt && p.bt == p.xt && p.ot == p.xt && (p.z == nullptr || p.zt == p.xt);
  if (!same) return launch_scan_t<S, NPL, R, G, W, ST, TT, 3>(p, stream);
  return p.xt == 0   ? launch_scan_t<S, NPL, R, G, W, ST, TT, 0>(p, stream)
         : p.xt == 1 ? launch_scan_t<S, NPL, R, G, W, ST, TT, 1>(p, stream)
                     : launch_scan_t<S, NPL, R, G, W, ST, TT, 2>(p, stream);
}
// The same where x is fp32.
template <int S, int NPL, int R, int G, int W, int ST, int TT>
static int launch_scan_f(const MmbSsmParams& p, cudaStream_t stream) {
  const bool same = p.dtt == 2 && p.bt == 2 && p.ot == 2 && (p.z == nullptr || p.zt == 2);
  return same ? launch_scan_t<S, NPL, R, G, W, ST, TT, 2>(p, stream) : launch_scan_t<S, NPL, R, G, W, ST, TT, 3>(p, stream);
}
// Blocks of four scanning warps, unless some SMs would get two of them where wider blocks give every SM at most one: then the SM with the most
// work has W warps instead of eight.  A block that has its SM to itself needs more staging warps, or they are what the scan waits for, and the wide
// ones longer tiles, as there is no other block to run while the two roles hand over.  Measured (bf16, 16 states; us for four and for W warps):
// 4096 tokens of 8192 channels 263 / 244 (7), 2048 of 7000 136 / 117 (6), 2048 of 5120 134 / 112 (5).  33 to 64 states: six warps where x is fp32, at
// 1192 / 1400 / 1776 channels (1531 tokens, us for four and for six warps) 92 / 80, 92 / 81, 92 / 81, with bf16 B and C 104 / 90; with a 16-bit x a tile of six
// warps is 12 channels or 24 bytes wide, no whole 16-byte pieces: bf16 94 / 93 there and 27.7 / 29.3 for 400 tokens, so four.  One
// block of four warps an SM, with four and with eight staging warps: 2048 of 4096 94 / 84, 4096 of 1536 (eight lanes a channel) 134 / 129.
// fp32 inputs with a 16-bit gate and output: 2048 of 5120 160 / 138, 2048 of 4096 140 / 105.
template <int S, int NPL, int R, int G>
static int launch_scan(const MmbSsmParams& p, cudaStream_t stream) {
  constexpr int PER = 32 / S * R;                  // channels a warp
  auto one_each = [&](int warps) { return ((long long)p.D + warps * PER - 1) / (warps * PER) * p.S <= 148; };
  if constexpr (S == 4 && NPL == 4) {
    if (one_each(4)) return launch_scan_w<S, NPL, R, G, 4, 256, 32>(p, stream);
    if (one_each(5)) return launch_scan_w<S, NPL, R, G, 5, 384, 64>(p, stream);
    if (one_each(6)) return launch_scan_w<S, NPL, R, G, 6, 384, 64>(p, stream);
    // in fp32 a tile of seven warps does not fit the shared memory
    if (p.xt != 2 && one_each(7)) return launch_scan_w<S, NPL, R, G, 7, 256, 64>(p, stream);
  }
  if constexpr (S == 8 && NPL == 2) {
    if (one_each(4)) return launch_scan_w<S, NPL, R, G, 4, 256, 32>(p, stream);
  }
  if constexpr (S == 16 && NPL == 4 && R == 1) {
    if (p.xt == 2 && !one_each(4) && one_each(6)) return launch_scan_f<S, NPL, R, G, 6, 384, 64>(p, stream);
  }
  return launch_scan_w<S, NPL, R, G, 4, 128, 32>(p, stream);
}

template <int S, int PCS, int XT>
static int launch_step_t(const MmbSsmParams& p, cudaStream_t stream) {
  const int groups = (p.D + kStepThreads / S - 1) / (kStepThreads / S);
  // a few groups of channels a block share its row's B and C, while that leaves eight blocks for every SM
  int per = 1;
  while (per < 4 && (long long)p.T * ((groups + 2 * per - 1) / (2 * per)) >= 8 * 148) per *= 2;
  if (p.T > 65535) return (int)cudaErrorInvalidValue;
  return launch(ssm_step_kernel<S, PCS, XT>, dim3((unsigned)((groups + per - 1) / per), (unsigned)p.T), dim3(kStepThreads), 0, stream, 1, p, per);
}
template <int S, int PCS>
static int launch_step(const MmbSsmParams& p, cudaStream_t stream) {
  const bool vec = p.N % 4 == 0 && reinterpret_cast<uintptr_t>(p.state) % 16 == 0 && reinterpret_cast<uintptr_t>(p.A) % 16 == 0 &&
                   rows_aligned(p.B, p.ldb, p.bt, 4) && rows_aligned(p.C, p.ldc, p.bt, 4) && p.dtt == p.xt && p.bt == p.xt &&
                   (p.z == nullptr || p.zt == p.xt);
  if (!vec) return launch_step_t<S, PCS, 3>(p, stream);
  return p.xt == 0 ? launch_step_t<S, PCS, 0>(p, stream) : p.xt == 1 ? launch_step_t<S, PCS, 1>(p, stream) : launch_step_t<S, PCS, 2>(p, stream);
}

}  // namespace mmb

MMB_API int mmb_ssm_scan(const MmbSsmParams* pp, cudaStream_t stream) {
  const MmbSsmParams& p = *pp;
  if (p.T <= 0 || p.D <= 0) return 0;
  if (p.S < 0 || p.N < 1 || p.N > 128 || p.cu_seqlens == nullptr) return (int)cudaErrorInvalidValue;
  // Lanes a channel: as many as leave one block to an SM, for a warp alone on its scheduler waits less the fewer states its lanes have; four where
  // there is more work than that.  Measured (2048 tokens, bf16, 16 states; us for S = 4 / 8 / 16): 768 channels 84 / 67 / 58, 1024 84 / 66 / 58,
  // 1280 84 / 68 / 70, 2368 84 / 68 / 72, 2560 84 / 94 / 92, 3584 85 / 95 / 120; 4096 tokens of 8192 244 / 326 / 390.
  const long long width = (long long)p.D * (p.S > 0 ? p.S : 1);
  if (p.N <= 8) return width > 148 * 16 ? mmb::launch_scan<4, 2, 1, 4>(p, stream) : mmb::launch_scan<8, 1, 1, 4>(p, stream);
  if (p.N <= 16) {
    if (width > 148 * 16) return mmb::launch_scan<4, 4, 1, 4>(p, stream);
    return width > 148 * 8 ? mmb::launch_scan<8, 2, 1, 4>(p, stream) : mmb::launch_scan<16, 1, 1, 2>(p, stream);
  }
  if (p.N <= 32) return mmb::launch_scan<8, 4, 1, 4>(p, stream);
  // 64 states: two channels a lane halve the shared memory reads of B and C (2000 tokens of 4096 channels, bf16: 199 us against 248 us) once there are
  // enough lanes for it (1531 tokens of 1536 channels, fp32: 117 us against 94 us)
  if (p.N <= 64) return width >= 4096 ? mmb::launch_scan<16, 4, 2, 1>(p, stream) : mmb::launch_scan<16, 4, 1, 4>(p, stream);
  return mmb::launch_scan<16, 8, 1, 2>(p, stream);
}

MMB_API int mmb_ssm_step(const MmbSsmParams* pp, cudaStream_t stream) {
  const MmbSsmParams& p = *pp;
  if (p.T <= 0 || p.D <= 0) return 0;
  if (p.N < 1 || p.N > 128 || p.state == nullptr) return (int)cudaErrorInvalidValue;
  if (p.N <= 16) return mmb::launch_step<2, 2>(p, stream);
  if (p.N <= 32) return mmb::launch_step<4, 2>(p, stream);
  return p.N <= 64 ? mmb::launch_step<8, 2>(p, stream) : mmb::launch_step<8, 4>(p, stream);
}
