// Attention of one new token per sequence over a paged cache with a sliding window and sinks: a sequence of n cached tokens sees the keys
// p < sinks and p >= n - window,
//   o = sum_p softmax_p(scale q . k_p) v_p.
// The visible keys are numbered j = 0 .. m - 1 (the sinks first, then the window) and everything else of the cache is never touched.  Work is
// 4 flops a query head and cached value, 1 to 16 heads a value: bound by the bytes of the visible K and V rows.
//
// Split.  The visible keys of one (sequence, KV head) are cut over the CTAs of a cluster, theirs over four warps, and each warp walks tiles of 16
// or 32 keys on its own: a private ring of tiles filled by 16-byte cp.async straight from the pages, no block barrier inside the loop.  Every warp
// keeps a reference maximum and a sum (fp32, base 2) and an O accumulator in registers; the warps are joined in shared memory and the CTAs through
// distributed shared memory in the same launch.  No global workspace: captured graphs share nothing and no result depends on arrival order.
// The reference of a row moves only when a score exceeds it by more than 2^8 (one vote for all rows; the usual tile has no shuffles).
//
// Tensor cores (m16n8k16): eight query heads of a KV head are the columns of a product (9 to 16 heads: of two), so a key is read once.
//   S^T = K Q^T: the contraction may be permuted, so a lane reads 8 consecutive values (16 bytes of bf16) of a key and uses them as the A
//   fragments of two k-steps; Q is held in the same order.
//   O^T = V^T P^T: the output rows may be permuted, so a lane reads 8 consecutive columns of its four keys and pairs them up with byte permutes; P
//   is transposed inside the warp (movmatrix).
// With the heads as columns every accumulator belongs to a head; as rows (16 of them) up to 8 heads left half of the accumulators empty and took
// twice the products for S (fp8, 64 rows: 143 us against 135; 8-bit cache of 256-wide heads 75 against 69).
// P is split into 16-bit numbers whose sum keeps what its 32 bits hold: three in bf16 (8 bits each), two in f16 (11 each).  A single bf16 P would add as
// much error as rounding the output does; two leave up to 2^-17 of a probability, visible where values cancel.  The third costs its share of the
// products: 64 rows 164.6 -> 166.6 us, 16 rows of 256-wide heads 49.7 -> 50.7, 16 query heads a KV head (32 rows, 256 wide) 58.6 -> 63.5.
// The products cut off what they can not add to an accumulator (no rounding), always towards zero: a sum over thousands of keys would drift by 2^-17.  So
// they sum one tile from zero, and an ordinary addition, rounded to nearest, takes that to O: 64 rows 168.0 -> 169.1 us, fp8 134.8 -> 140.7, fp4 154 -> 156, int4
// 160 -> 164, 8-bit cache of 256-wide heads 69.3 -> 71.1.  Outputs that are not the nearest bf16 to the exact value (64 rows): 2.0 in 1000 before,
// 0.23 after; with 32-bit products and sums 0.9.
//
// Quantized pools: the codes of every format are exact in f16, so both products run in f16.  Q goes in divided by a power of two per row, undone in
// the score; the row scale of K multiplies the score and that of V the probability, both in fp32.  Probabilities times value scales are kept in f16's
// range by a reference for the scales (4 x the largest seen) and a factor of 2^7: 22 bits of each down to 2^-8 of the largest scale, and below that no
// key loses more than 2^-30 of the largest |v| seen (half of f16's smallest step, 2^-24, against 2^5).
//
// Measured (graph replays, heads 32 / 8 of 128, window 4096 + 4, three input sets in turn): 64 rows bf16 169 us = 6.4 TB/s, 97 % of the measured
// copy rate; 8 rows 27.1 us; 1 row 12.2 us.  64 rows int8 117 us and fp8 141 us, 1.4 and 1.7 x the time of their bytes: half the bytes a key, the
// same instructions a key plus the conversions, so the issue slots bound them (hardware conversions into f16 instead of bf16: 32 rows of int8 117 -> 76 us;
// 32 keys a tile 76 -> 64; rows padded instead of swizzled changed nothing, 62 -> 63).  fp4 156 us and int4 164 us for 44 us of bytes: the same
// bound, with more instructions a conversion.
#include <atomic>
#include <cuda_fp4.h>

#include "api_ext.h"
#include "launch.h"
#include "typed_io.cuh"

namespace mmb {

constexpr float kSdLazy = 8.f;              // log2 units
constexpr int kSdWarps = 4, kSdThreads = kSdWarps * 32;

enum { kSdBf16 = 0, kSdFp8 = 1, kSdInt8 = 2, kSdFp4 = 3, kSdInt4 = 4 };

template <int D, int F>
struct SdCfg {
  static constexpr int row_bytes = F == kSdBf16 ? D * 2 : (F <= kSdInt8 ? D : D / 2);
  static constexpr int T = F == kSdBf16 || D == 256 ? 16 : 32;          // keys a tile
  static constexpr int U = row_bytes / 16;                       // 16-byte units a row
  static constexpr int piece = row_bytes * 8 / D;                // bytes of 8 values
  static constexpr int tile_bytes = 2 * T * row_bytes;     // K and V
  static constexpr int scale_bytes = F == kSdBf16 ? 0 : 2 * T * 4;
  static constexpr int stage_bytes = tile_bytes + scale_bytes;
  // as many stages as fit next to two more CTAs on the SM, two to four (more stages and fewer CTAs were slower: the warps, not the copies, are short)
  static constexpr int fit = (72 * 1024) / (kSdWarps * stage_bytes);
  static constexpr int NST = fit < 2 ? 2 : (fit > 4 ? 4 : fit);
  static constexpr int ring_bytes = kSdWarps * NST * stage_bytes;
};

// Where 16-byte unit u of row r lies in its row, so that the lanes of one fragment load fall into different banks.
template <int U, int PIECE>
__device__ __forceinline__ int sd_unit_k(int r, int u) {
  if constexpr (PIECE == 16) return u ^ ((r & 1) << 2);
  if constexpr (PIECE == 8) return u ^ (U >= 8 ? (r & 3) << 1 : (r & 2));
  return u ^ (U >= 8 ? (r & 7) : (U == 4 ? (r >> 1) & 3 : (r >> 2) & 1));
}
template <int U, int PIECE>
__device__ __forceinline__ int sd_unit_v(int r, int u) {
  if constexpr (U >= 8) return u ^ (r & 6);
  if constexpr (U == 4) return u ^ (r & 2);
  return u;
}

// 8 cached codes at `p` as four f16 pairs (all formats are exact in it).  int8: 0x6400 + u is the f16 number 1024 + u for 0 <= u < 256.
template <int F>
__device__ __forceinline__ void sd_load8_f16(const unsigned char* p, uint32_t (&w)[4]) {
  if constexpr (F == kSdFp8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)((i < 2 ? u.x : u.y) >> (16 * (i & 1))), __NV_E4M3);
      w[i] = (uint32_t)h.x | (uint32_t)h.y << 16;
    }
  } else if constexpr (F == kSdInt8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    const __half2 off = __half2half2(__ushort_as_half(0x6480));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t m = __byte_perm((i < 2 ? u.x : u.y) ^ 0x80808080u, 0x64646464u, i & 1 ? 0x4342 : 0x4140);
      const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&m), off);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  } else if constexpr (F == kSdFp4) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2_raw h = __nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)((u >> (8 * i)) & 0xff), __NV_E2M1);
      w[i] = (uint32_t)h.x | (uint32_t)h.y << 16;
    }
  } else {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p) ^ 0x88888888u;
    const __half2 off = __half2half2(__ushort_as_half(0x6408));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t n = u >> (8 * i);
      const uint32_t m = (n & 0xfu) | (n & 0xf0u) << 12 | 0x64006400u;
      const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&m), off);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
}
template <int F>
__device__ __forceinline__ void sd_load8(const unsigned char* p, uint32_t (&w)[4]) {
  if constexpr (F == kSdBf16) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else {
    sd_load8_f16<F>(p, w);
  }
}
// 8 x 8 matrix of 16-bit values, two of a row in each lane, transposed.
__device__ __forceinline__ uint32_t sd_transpose(uint32_t a) {
  uint32_t d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(a));
  return d;
}
template <int N>
__device__ __forceinline__ float sd_max(const float (&v)[N]) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  return m;
}
template <int F>
__device__ __forceinline__ void sd_mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F == kSdBf16) mma_bf16_16816(d, a0, a1, a2, a3, b0, b1);
  else mma_f16_16816(d, a0, a1, a2, a3, b0, b1);
}

__device__ __forceinline__ void sd_cp4(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ uint32_t sd_remote(uint32_t addr, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float sd_remote_f(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 sd_remote_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// CTAs an SM that the compiler leaves registers for.  Left alone, 128-wide heads of fp8, fp4 and int4 take 180 to 190 registers, which is two CTAs; held to
// three they need no spills (9 rows, window 4096, us for two and for three: fp8 39.0 / 36.4, fp4 40.5 / 36.9, int4 42.4 / 38.1; 64 rows 143.6 / 144.5, 162.6 /
// 156.5, 171.7 / 164).  int8 loses by it (64 rows 121 / 157).
constexpr int sd_ctas(int D, int F, bool wide) { return !wide && D == 128 && (F == kSdFp8 || F >= kSdFp4) ? 3 : 1; }

// grid (splits, Hkv * head groups, B), clusters of `splits`.  WIDE: 16 query heads a CTA, else 8.
template <int D, int F, bool WIDE>
__global__ void __launch_bounds__(kSdThreads, sd_ctas(D, F, WIDE)) sink_decode_kernel(const MmbSinkDecodeParams p, int splits, int head_groups, int bs_shift) {
  using Cfg = SdCfg<D, F>;
  constexpr int R = WIDE ? 16 : 8, U = Cfg::U, NST = Cfg::NST, NI = D / 32, NJ = D / 64, T = Cfg::T, NT = T / 8, KT = T / 16;
  constexpr bool kScaled = F != kSdBf16;
  constexpr int kParts = kScaled ? 2 : 3;                        // 16-bit numbers that hold a probability
  extern __shared__ __align__(16) unsigned char sm[];
  __shared__ __align__(16) unsigned char q_sm[R * D * 2];        // 16-byte pieces, placed like the units of K
  __shared__ float ml[kSdWarps][R][2], ml_cta[R][2];
  __shared__ unsigned ok_sm[kSdWarps][NST];
  __shared__ float q_scale[R];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  const int rank = blockIdx.x, hk = blockIdx.y / head_groups, hg = blockIdx.y % head_groups, b = blockIdx.z;
  const int G = p.Hq / p.Hkv, head0 = hk * G + hg * R, heads = min(R, G - hg * R);

  // visible keys: j < n_sink at position j, the others at position j + shift
  const long long room = (long long)p.max_blocks * p.block_size;
  const int n = max(0, (int)min((long long)p.ctx_lens[b], room));
  if (p.ctx_lens[b] > room && tid == 0 && p.status) atomicExch(p.status, 131);      // more tokens than its table has places for
  const int lo = max(0, n - p.window), n_sink = min(p.sinks, lo), shift = lo - n_sink, m = n - shift;
  const int per = ((m + splits - 1) / splits + T - 1) / T * T;
  const int j_begin = min(m, rank * per), j_end = min(m, j_begin + per);
  const int tiles = (j_end - j_begin + T - 1) / T;
  const int mine = tiles > warp ? (tiles - warp + kSdWarps - 1) / kSdWarps : 0;

  for (int i = tid; i < R * D / 8; i += kSdThreads) {
    const int r = i / (D / 8), c = i % (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < heads) v = reinterpret_cast<const uint4*>(p.q)[((long long)b * p.Hq + head0 + r) * (D / 8) + c];
    *reinterpret_cast<uint4*>(q_sm + (r * (D / 8) + (c ^ ((r & 1) << 2))) * 16) = v;
  }
  __syncthreads();
  if constexpr (kScaled) {
    // f16 products take q divided by the power of two at its row's largest magnitude (nothing below 2^-24 of that matters to a score)
    for (int r = warp; r < R; r += kSdWarps) {
      bf16* row = reinterpret_cast<bf16*>(q_sm) + r * D;
      float m = 0.f;
      for (int i = lane; i < D; i += 32) m = fmaxf(m, fabsf(__bfloat162float(row[i])));
      m = warp_max(m);
      const int e = m > 0.f && m < INFINITY ? (int)(__float_as_uint(m) >> 23) - 127 : 0;
      const int half_e = e / 2;                                   // two factors: 2^-e alone can overflow
      const float f0 = __uint_as_float((uint32_t)(127 - half_e) << 23), f1 = __uint_as_float((uint32_t)(127 - (e - half_e)) << 23);
      for (int i = lane; i < D; i += 32) reinterpret_cast<__half*>(row)[i] = __float2half_rn(__bfloat162float(row[i]) * f0 * f1);
      if (lane == 0) q_scale[r] = 1.f / f0 / f1;
    }
    __syncthreads();
  }

  const long long row_stride = (long long)p.Hkv * Cfg::row_bytes;
  const int head_at = hk * Cfg::row_bytes;
  unsigned char* ring = sm + warp * NST * Cfg::stage_bytes;
  const int* table = p.block_tables + (long long)b * p.max_blocks;
  // cache slot of key `lane % T` of tile t of this warp, -1 where there is none
  auto slot_of = [&](int t) -> int {
    const int j = j_begin + (warp + t * kSdWarps) * T + lane % T;
    if (t >= mine || j >= j_end) return -1;
    const int pos = j < n_sink ? j : j + shift;
    const int blk = bs_shift >= 0 ? pos >> bs_shift : pos / p.block_size;
    const long long slot = (long long)table[blk] * p.block_size + (pos - blk * p.block_size);
    if (slot >= 0 && slot < p.n_slots) return (int)slot;
    if (p.status) atomicExch(p.status, 131);
    return -1;
  };
  auto issue = [&](int t, int slot) {
    if (t < mine) {
      unsigned char* st = ring + (t % NST) * Cfg::stage_bytes;
      const unsigned ok = __ballot_sync(0xffffffffu, slot >= 0);
      if (lane == 0) ok_sm[warp][t % NST] = ok;
#pragma unroll
      for (int i = 0; i < T * U / 32; ++i) {
        const int e = i * 32 + lane, r = e / U, u = e % U;
        const int sl = __shfl_sync(0xffffffffu, slot, r);
        const long long at = (long long)max(sl, 0) * row_stride + (head_at + u * 16);
        cp_async16(st + (r * U + sd_unit_k<U, Cfg::piece>(r, u)) * 16, reinterpret_cast<const unsigned char*>(p.k) + at, sl >= 0);
        cp_async16(st + Cfg::tile_bytes / 2 + (r * U + sd_unit_v<U, Cfg::piece>(r, u)) * 16, reinterpret_cast<const unsigned char*>(p.v) + at, sl >= 0);
      }
      if constexpr (kScaled) {
        const long long at = slot >= 0 ? (long long)slot * p.Hkv + hk : 0;
        if constexpr (T == 16) {
          sd_cp4(st + Cfg::tile_bytes + lane * 4, (lane < 16 ? p.k_scale : p.v_scale) + at, slot >= 0);
        } else {
          sd_cp4(st + Cfg::tile_bytes + lane * 4, p.k_scale + at, slot >= 0);
          sd_cp4(st + Cfg::tile_bytes + (T + lane) * 4, p.v_scale + at, slot >= 0);
        }
      }
    }
    cp_async_commit();
  };

  constexpr int HT = R / 8;                                      // tiles of eight heads
  constexpr bool kQReg = D <= 128;
  uint4 qr[kQReg ? NI : 1][HT];
  if constexpr (kQReg) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int h = 0; h < HT; ++h) qr[i][h] = *reinterpret_cast<const uint4*>(q_sm + ((gid + 8 * h) * (D / 8) + ((tig + 4 * i) ^ ((gid & 1) << 2))) * 16);
  }
  float o[NJ * 4][HT][4];
#pragma unroll
  for (int i = 0; i < NJ * 4; ++i)
#pragma unroll
    for (int h = 0; h < HT; ++h) o[i][h][0] = o[i][h][1] = o[i][h][2] = o[i][h][3] = 0.f;
  float v_ref = 0.f;                                             // quantized: reference of the value scales
  // this lane's heads: 8 h + 2 tig, + 1
  float mx[2 * HT], l[2 * HT], cr[2 * HT];
#pragma unroll
  for (int h = 0; h < 2 * HT; ++h) {
    mx[h] = -INFINITY;
    l[h] = 0.f;
    cr[h] = p.scale * 1.4426950408889634f;
    if constexpr (kScaled) cr[h] *= q_scale[8 * (h >> 1) + 2 * tig + (h & 1)];
  }

#pragma unroll
  for (int t = 0; t < NST - 1; ++t) issue(t, slot_of(t));
  int next = slot_of(NST - 1);
  for (int t = 0; t < mine; ++t) {
    issue(t + NST - 1, next);
    next = slot_of(t + NST);
    cp_async_wait<NST - 1>();
    __syncwarp();
    const unsigned char* st = ring + (t % NST) * Cfg::stage_bytes;
    const unsigned char* vt = st + Cfg::tile_bytes / 2;
    const unsigned ok = ok_sm[warp][t % NST];
    // S^T = K Q^T, two chains a tile
    float s[KT][HT][4] = {}, s2[KT][HT][4] = {};
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int pc = tig + 4 * i;
      uint4 q[HT];
#pragma unroll
      for (int h = 0; h < HT; ++h) {
        if constexpr (kQReg) q[h] = qr[i][h];
        else q[h] = *reinterpret_cast<const uint4*>(q_sm + ((gid + 8 * h) * (D / 8) + (pc ^ ((gid & 1) << 2))) * 16);
      }
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint32_t w[2][4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 16 * kt + 8 * e + gid;
          sd_load8<F>(st + (r * U + sd_unit_k<U, Cfg::piece>(r, pc * Cfg::piece / 16)) * 16 + pc * Cfg::piece % 16, w[e]);
        }
#pragma unroll
        for (int h = 0; h < HT; ++h) {
          sd_mma<F>(s[kt][h], w[0][0], w[1][0], w[0][1], w[1][1], q[h].x, q[h].y);
          sd_mma<F>(s2[kt][h], w[0][2], w[1][2], w[0][3], w[1][3], q[h].z, q[h].w);
        }
      }
    }
    // scores in units of log2; this lane's keys are 8 k + gid
    float p4[2 * HT][NT];                                        // [head][key]
    bool grew = false;
    float vs[NT] = {};
#pragma unroll
    for (int k = 0; k < NT; ++k) {
      const int key = 8 * k + gid;
      float f = 1.f;
      if constexpr (kScaled) {
        f = reinterpret_cast<const float*>(st + Cfg::tile_bytes)[key];
        vs[k] = reinterpret_cast<const float*>(st + Cfg::tile_bytes)[T + key];
        grew |= vs[k] > v_ref;
      }
      const bool in = ok >> key & 1;
#pragma unroll
      for (int h = 0; h < 2 * HT; ++h) {
        const int c = 2 * (k & 1) + (h & 1);
        p4[h][k] = in ? (s[k >> 1][h >> 1][c] + s2[k >> 1][h >> 1][c]) * (cr[h] * f) : -INFINITY;
      }
    }
    // the reference of a head moves only when one of its scores is more than kSdLazy above it; the test is one vote for all heads
#pragma unroll
    for (int h = 0; h < 2 * HT; ++h) grew |= sd_max(p4[h]) > mx[h] + kSdLazy;
    if (__any_sync(0xffffffffu, grew)) {
      float alpha[2 * HT], beta = 1.f;
      auto lanes_max = [](float m) {                             // over the lanes that hold other keys of the same heads
#pragma unroll
        for (int d = 4; d < 32; d *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, d));
        return m;
      };
      if constexpr (kScaled) {
        const float m = lanes_max(sd_max(vs));
        if (m > v_ref) {
          beta = v_ref / (4.f * m);
          v_ref = 4.f * m;
        }
      }
#pragma unroll
      for (int h = 0; h < 2 * HT; ++h) {
        const float m = lanes_max(sd_max(p4[h]));
        alpha[h] = beta;
        if (m > mx[h]) {
          const float f = exp2_fast(mx[h] - m);
          mx[h] = m;
          l[h] *= f;
          alpha[h] *= f;
        }
      }
#pragma unroll
      for (int i = 0; i < NJ * 4; ++i)
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[i][h][e] *= alpha[2 * h + (e & 1)];
    }
    const float inv = kScaled && v_ref > 0.f ? 128.f / v_ref : 0.f;
#pragma unroll
    for (int h = 0; h < 2 * HT; ++h) {
      const float ref = mx[h] == -INFINITY ? 0.f : mx[h];
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        p4[h][k] = exp2_fast(p4[h][k] - ref);
        l[h] += p4[h][k];
        if constexpr (kScaled) p4[h][k] *= vs[k] * inv;
      }
    }
    // P as B fragments: [8 keys][8 heads] of this layout, in kParts numbers whose sum it is, transposed inside the warp
    uint32_t pf[kParts][HT][NT];
#pragma unroll
    for (int h = 0; h < HT; ++h)
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        float x = p4[2 * h][k], y = p4[2 * h + 1][k];
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          uint32_t a;
          if constexpr (kScaled) {
            a = pack16(x, y, 1);
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&a));
            x -= f.x, y -= f.y;
          } else {
            a = pack16(x, y, 0);
            x -= __uint_as_float(a << 16), y -= __uint_as_float(a & 0xffff0000u);
          }
          pf[i][h][k] = sd_transpose(a);
        }
      }
    // O^T += V^T P^T.  A tile's products are summed from zero, the smallest parts of P first, and added to O once: every product that adds to O itself would
    // cut O's last bit off
#pragma unroll
    for (int jj = 0; jj < NJ; ++jj) {
      const int pc = gid + 8 * jj;
      float d[4][HT][4] = {};
#pragma unroll
      for (int kt = 0; kt < KT; ++kt) {
        uint32_t v[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = 16 * kt + 2 * tig + (k & 1) + 8 * (k >> 1);
          sd_load8<F>(vt + (r * U + sd_unit_v<U, Cfg::piece>(r, pc * Cfg::piece / 16)) * 16 + pc * Cfg::piece % 16, v[k]);
        }
#pragma unroll
        for (int m = 0; m < 4; ++m) {                            // rows gid: column 2 m of the piece, rows gid + 8: column 2 m + 1
          const uint32_t a0 = __byte_perm(v[0][m], v[1][m], 0x5410), a1 = __byte_perm(v[0][m], v[1][m], 0x7632);
          const uint32_t a2 = __byte_perm(v[2][m], v[3][m], 0x5410), a3 = __byte_perm(v[2][m], v[3][m], 0x7632);
#pragma unroll
          for (int h = 0; h < HT; ++h)
#pragma unroll
            for (int i = kParts - 1; i >= 0; --i) sd_mma<F>(d[m][h], a0, a1, a2, a3, pf[i][h][2 * kt], pf[i][h][2 * kt + 1]);
        }
      }
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int h = 0; h < HT; ++h)
#pragma unroll
          for (int e = 0; e < 4; e += 2) {
            float(&x)[4] = o[jj * 4 + m][h];
            const float2 f = unpack2(add2(pack2(x[e], x[e + 1]), pack2(d[m][h][e], d[m][h][e + 1])));
            x[e] = f.x, x[e + 1] = f.y;
          }
    }
    __syncwarp();                                                // the stage may be refilled
  }

  // ---- join the warps.  Head r of warp w: maximum and sum in ml, O in the (idle) ring as [w][r][D]
  cp_async_wait<0>();
  __syncthreads();
#pragma unroll
  for (int h = 0; h < 2 * HT; ++h) {
#pragma unroll
    for (int d = 4; d < 32; d *= 2) l[h] += __shfl_xor_sync(0xffffffffu, l[h], d);
    if (gid == 0) ml[warp][8 * (h >> 1) + 2 * tig + (h & 1)][0] = mx[h], ml[warp][8 * (h >> 1) + 2 * tig + (h & 1)][1] = l[h];
  }
  float* os = reinterpret_cast<float*>(sm);
  const float back = kScaled ? v_ref * (1.f / 128.f) : 1.f;
#pragma unroll
  for (int jj = 0; jj < NJ; ++jj)
#pragma unroll
    for (int h = 0; h < HT; ++h)
#pragma unroll
      for (int e = 0; e < 2; ++e) {                              // head 8 h + 2 tig + e, columns 8 (gid + 8 jj) .. + 7
        float4* dst = reinterpret_cast<float4*>(os + ((warp * R + 8 * h + 2 * tig + e) * D + (gid + 8 * jj) * 8));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const float(&x)[4] = o[jj * 4 + 2 * q][h];
          const float(&y)[4] = o[jj * 4 + 2 * q + 1][h];
          dst[q] = make_float4(x[e] * back, x[2 + e] * back, y[e] * back, y[2 + e] * back);
        }
      }
  __syncthreads();
  // weights of the warps of row r: 2^(m_w - M)
  auto weight = [](float mw, float M) { return mw == -INFINITY ? 0.f : exp2_fast(mw - M); };
  if (splits == 1) {
    for (int i = tid; i < heads * D / 4; i += kSdThreads) {
      const int r = i / (D / 4), col = i % (D / 4) * 4;
      float M = -INFINITY, L = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kSdWarps; ++w) M = fmaxf(M, ml[w][r][0]);
#pragma unroll
      for (int w = 0; w < kSdWarps; ++w) {
        const float f = weight(ml[w][r][0], M);
        const float4 x = *reinterpret_cast<const float4*>(os + (w * R + r) * D + col);
        L = fmaf(f, ml[w][r][1], L);
        a.x = fmaf(f, x.x, a.x), a.y = fmaf(f, x.y, a.y), a.z = fmaf(f, x.z, a.z), a.w = fmaf(f, x.w, a.w);
      }
      const float inv = L == 0.f ? 0.f : 1.f / L;                // a row that sees nothing is zero
      uint2 w2 = make_uint2(pack16(a.x * inv, a.y * inv, 0), pack16(a.z * inv, a.w * inv, 0));
      *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(p.out) + ((long long)b * p.Hq + head0 + r) * D + col) = w2;
    }
    return;
  }
  // this CTA's rows into warp 0's place, then every CTA of the cluster joins its share of the columns
  for (int i = tid; i < R * D / 4; i += kSdThreads) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kSdWarps; ++w) M = fmaxf(M, ml[w][r][0]);
#pragma unroll
    for (int w = 0; w < kSdWarps; ++w) {
      const float f = weight(ml[w][r][0], M);
      const float4 x = *reinterpret_cast<const float4*>(os + (w * R + r) * D + col);
      L = fmaf(f, ml[w][r][1], L);
      a.x = fmaf(f, x.x, a.x), a.y = fmaf(f, x.y, a.y), a.z = fmaf(f, x.z, a.z), a.w = fmaf(f, x.w, a.w);
    }
    *reinterpret_cast<float4*>(os + r * D + col) = a;
    if (col == 0) ml_cta[r][0] = M, ml_cta[r][1] = L;
  }
  cluster_arrive();
  cluster_wait();
  const uint32_t os_addr = smem_u32(os), ml_addr = smem_u32(&ml_cta[0][0]);
  for (int i = rank * kSdThreads + tid; i < heads * D / 4; i += splits * kSdThreads) {
    const int r = i / (D / 4), col = i % (D / 4) * 4;
    float M = -INFINITY, L = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < splits; ++k) M = fmaxf(M, sd_remote_f(sd_remote(ml_addr + r * 8, k)));
    for (int k = 0; k < splits; ++k) {
      const uint32_t mk = sd_remote(ml_addr + r * 8, k);
      const float f = weight(sd_remote_f(mk), M);
      const float4 x = sd_remote_f4(sd_remote(os_addr + (r * D + col) * 4, k));
      L = fmaf(f, sd_remote_f(mk + 4), L);
      a.x = fmaf(f, x.x, a.x), a.y = fmaf(f, x.y, a.y), a.z = fmaf(f, x.z, a.z), a.w = fmaf(f, x.w, a.w);
    }
    const float inv = L == 0.f ? 0.f : 1.f / L;
    uint2 w2 = make_uint2(pack16(a.x * inv, a.y * inv, 0), pack16(a.z * inv, a.w * inv, 0));
    *reinterpret_cast<uint2*>(reinterpret_cast<bf16*>(p.out) + ((long long)b * p.Hq + head0 + r) * D + col) = w2;
  }
  cluster_arrive();                                              // nobody leaves while its shared memory is still read
  cluster_wait();
}

template <int D, int F, bool WIDE>
static int launch_sinks(const MmbSinkDecodeParams& p, cudaStream_t stream) {
  using Cfg = SdCfg<D, F>;
  constexpr int R = WIDE ? 16 : 8;
  constexpr int join = kSdWarps * R * D * 4;
  constexpr int smem = Cfg::ring_bytes > join ? Cfg::ring_bytes : join;
  auto kern = sink_decode_kernel<D, F, WIDE>;
  // the shared memory limit and how many CTAs an SM takes belong to a device: CTAs + 1 of each, 0 = not asked yet
  static std::atomic<int> resident[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  int ctas = dev < 64 ? resident[dev].load(std::memory_order_relaxed) - 1 : -1;
  if (ctas < 0) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kern, kSdThreads, smem);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) resident[dev].store(ctas + 1, std::memory_order_relaxed);
  }
  const int G = p.Hq / p.Hkv, hg = (G + R - 1) / R;
  if ((long long)p.Hkv * hg > 65535 || p.B > 65535) return (int)cudaErrorInvalidValue;
  int splits = p.splits;
  if (splits == 0) {
    const long long most = min((long long)p.window + p.sinks, (long long)p.max_blocks * p.block_size);
    const long long tiles = (most + Cfg::T - 1) / Cfg::T, rows = (long long)p.B * p.Hkv * hg;
    // as many as the SMs hold at once: a second wave costs more than idle slots (24 rows of 8 KV heads: 1 split 73 us, 3 splits 88), a larger cluster
    // more than it saves once the SMs are full (64 rows: 1 split 166 us, 2 splits 180, 8 splits 236)
    splits = 1;
    while (splits < 8 && rows * (splits + 1) <= 148 * ctas && (splits + 1) * kSdWarps <= tiles) ++splits;
  }
  int shift = -1;
  if ((p.block_size & (p.block_size - 1)) == 0)
    for (shift = 0; (1 << shift) < p.block_size; ++shift) {
    }
  return launch(kern, dim3((unsigned)splits, (unsigned)(p.Hkv * hg), (unsigned)p.B), dim3(kSdThreads), (size_t)smem, stream, splits, p, splits, hg, shift);
}

template <int D, int F>
static int launch_sinks_g(const MmbSinkDecodeParams& p, cudaStream_t stream) {
  return p.Hq / p.Hkv > 8 ? launch_sinks<D, F, true>(p, stream) : launch_sinks<D, F, false>(p, stream);
}
template <int D>
static int launch_sinks_f(const MmbSinkDecodeParams& p, cudaStream_t stream) {
  switch (p.fmt) {
    case -1: return launch_sinks_g<D, kSdBf16>(p, stream);
    case 0: return launch_sinks_g<D, kSdFp8>(p, stream);
    case 1: return launch_sinks_g<D, kSdInt8>(p, stream);
    case 2: return launch_sinks_g<D, kSdFp4>(p, stream);
    case 3: return launch_sinks_g<D, kSdInt4>(p, stream);
    default: return (int)cudaErrorInvalidValue;
  }
}

}  // namespace mmb

MMB_API int mmb_sink_decode(const MmbSinkDecodeParams* pp, cudaStream_t stream) {
  const MmbSinkDecodeParams& p = *pp;
  if (p.B <= 0) return 0;
  if (p.Hkv < 1 || p.Hq < 1 || p.Hq % p.Hkv != 0 || p.window < 1 || p.sinks < 0 || p.block_size < 1 || p.max_blocks < 0 || p.n_slots < 0 ||
      p.splits < 0 || p.splits > 8)
    return (int)cudaErrorInvalidValue;
  switch (p.D) {
    case 64: return mmb::launch_sinks_f<64>(p, stream);
    case 128: return mmb::launch_sinks_f<128>(p, stream);
    case 256: return mmb::launch_sinks_f<256>(p, stream);
    default: return (int)cudaErrorInvalidValue;
  }
}
