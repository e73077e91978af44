// Attention of one new token per sequence over a paged cache with a sliding window and sinks: a sequence of n cached tokens sees the keys
// p < sinks and p >= n - window,
//   o = sum_p softmax_p(scale q . k_p) v_p.
// The visible keys are numbered j = 0 .. m - 1 (the sinks first, then the window) and everything else of the cache is never touched.  Work is
// 4 flops a query head and cached value, 1 to 16 heads a value: bound by the bytes of the visible K and V rows.
//
// Split.  The visible keys of one (sequence, KV head) are cut over the CTAs of a cluster, theirs over four warps, and each warp walks tiles of 16
// keys on its own: a private ring of tiles filled by 16-byte cp.async straight from the pages, no block barrier inside the loop.  Every warp keeps
// a running maximum and sum (fp32, base 2) and an O accumulator in registers; the warps are joined in shared memory and the CTAs through
// distributed shared memory in the same launch.  No global workspace: captured graphs share nothing and no result depends on arrival order.
//
// Tensor cores (m16n8k16): all query heads of a KV head are the rows of one product, so a key is read once.
//   S = Q K^T: the contraction may be permuted, so a lane reads 8 consecutive values (16 bytes of bf16) of its key and uses them as the B
//   fragments of two k-steps; Q is held in the same order.
//   O = P V: the output columns may be permuted, so a lane reads 8 consecutive columns of its four keys and pairs them up with byte permutes.
// P is split into two bf16 numbers (P = hi + lo to 2^-17): a single bf16 P would add as much error as rounding the output does.  Up to 8 heads fill
// only half of the 16 rows; hi and lo then take rows 0-7 and 8-15 of ONE product.  9 to 16 heads take two products.
// Quantized pools: the codes are exact in bf16; the row scale of K multiplies the score and that of V the probability, both in fp32.
#include <atomic>
#include <cuda_fp4.h>

#include "api_ext.h"
#include "launch.h"
#include "typed_io.cuh"

namespace mmb {

constexpr int kSdWarps = 4, kSdThreads = kSdWarps * 32, kSdTile = 16;

enum { kSdBf16 = 0, kSdFp8 = 1, kSdInt8 = 2, kSdFp4 = 3, kSdInt4 = 4 };

template <int D, int F>
struct SdCfg {
  static constexpr int row_bytes = F == kSdBf16 ? D * 2 : (F <= kSdInt8 ? D : D / 2);
  static constexpr int U = row_bytes / 16;                       // 16-byte units a row
  static constexpr int piece = row_bytes * 8 / D;                // bytes of 8 values
  static constexpr int tile_bytes = 2 * kSdTile * row_bytes;     // K and V
  static constexpr int scale_bytes = F == kSdBf16 ? 0 : 2 * kSdTile * 4;
  static constexpr int stage_bytes = tile_bytes + scale_bytes;
  // as many stages as fit next to a second CTA on the SM, at least three
  static constexpr int fit = (100 * 1024) / (kSdWarps * stage_bytes);
  static constexpr int NST = fit < 3 ? 3 : (fit > 6 ? 6 : fit);
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

__device__ __forceinline__ float sd_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t sd_pack(float a, float b) {
  const bf162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// 8 cached values at `p` as four bf16 pairs.
template <int F>
__device__ __forceinline__ void sd_load8(const unsigned char* p, uint32_t (&w)[4]) {
  if constexpr (F == kSdBf16) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
  } else if constexpr (F == kSdFp8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_fp8x2_storage_t c = (__nv_fp8x2_storage_t)((i < 2 ? u.x : u.y) >> (16 * (i & 1)));
      const __half2 h = __half2(__nv_cvt_fp8x2_to_halfraw2(c, __NV_E4M3));
      const float2 f = __half22float2(h);
      w[i] = sd_pack(f.x, f.y);
    }
  } else if constexpr (F == kSdInt8) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = (int)((i < 2 ? u.x : u.y) >> (16 * (i & 1)));
      w[i] = sd_pack((float)(signed char)(c & 0xff), (float)(signed char)((c >> 8) & 0xff));
    }
  } else if constexpr (F == kSdFp4) {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __half2(__nv_cvt_fp4x2_to_halfraw2((__nv_fp4x2_storage_t)((u >> (8 * i)) & 0xff), __NV_E2M1));
      const float2 f = __half22float2(h);
      w[i] = sd_pack(f.x, f.y);
    }
  } else {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int lo = (int)(u << (28 - 8 * i)) >> 28, hi = (int)(u << (24 - 8 * i)) >> 28;
      w[i] = sd_pack((float)lo, (float)hi);
    }
  }
}

__device__ __forceinline__ void sd_cp16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void sd_cp4(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void sd_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void sd_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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

// grid (splits, Hkv * head groups, B), clusters of `splits`.  WIDE: 16 query heads a CTA, else 8.
template <int D, int F, bool WIDE>
__global__ void __launch_bounds__(kSdThreads) sink_decode_kernel(const MmbSinkDecodeParams p, int splits, int head_groups, int bs_shift) {
  using Cfg = SdCfg<D, F>;
  constexpr int R = WIDE ? 16 : 8, U = Cfg::U, NST = Cfg::NST, NI = D / 32, NJ = D / 64;
  constexpr bool kScaled = F != kSdBf16;
  extern __shared__ __align__(16) unsigned char sm[];
  __shared__ __align__(16) unsigned char q_sm[R * D * 2];        // 16-byte pieces, placed like the units of K
  __shared__ float ml[kSdWarps][R][2], ml_cta[R][2];
  __shared__ unsigned ok_sm[kSdWarps][NST];
  pdl_launch_dependents();
  pdl_wait();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gid = lane >> 2, tig = lane & 3;
  const int rank = blockIdx.x, hk = blockIdx.y / head_groups, hg = blockIdx.y % head_groups, b = blockIdx.z;
  const int G = p.Hq / p.Hkv, head0 = hk * G + hg * R, heads = min(R, G - hg * R);

  // visible keys: j < n_sink at position j, the others at position j + shift
  const int n = max(0, (int)min((long long)p.ctx_lens[b], (long long)p.max_blocks * p.block_size));
  const int lo = max(0, n - p.window), n_sink = min(p.sinks, lo), shift = lo - n_sink, m = n - shift;
  const int per = ((m + splits - 1) / splits + kSdTile - 1) / kSdTile * kSdTile;
  const int j_begin = min(m, rank * per), j_end = min(m, j_begin + per);
  const int tiles = (j_end - j_begin + kSdTile - 1) / kSdTile;
  const int mine = tiles > warp ? (tiles - warp + kSdWarps - 1) / kSdWarps : 0;

  for (int i = tid; i < R * D / 8; i += kSdThreads) {
    const int r = i / (D / 8), c = i % (D / 8);
    uint4 v = make_uint4(0, 0, 0, 0);
    if (r < heads) v = reinterpret_cast<const uint4*>(p.q)[((long long)b * p.Hq + head0 + r) * (D / 8) + c];
    *reinterpret_cast<uint4*>(q_sm + (r * (D / 8) + (c ^ ((r & 1) << 2))) * 16) = v;
  }
  __syncthreads();

  unsigned char* ring = sm + warp * NST * Cfg::stage_bytes;
  const int* table = p.block_tables + (long long)b * p.max_blocks;
  // cache slot of key `lane % 16` of tile t of this warp, -1 where there is none
  auto slot_of = [&](int t) -> long long {
    const int j = j_begin + (warp + t * kSdWarps) * kSdTile + (lane & 15);
    if (t >= mine || j >= j_end) return -1;
    const int pos = j < n_sink ? j : j + shift;
    const int blk = bs_shift >= 0 ? pos >> bs_shift : pos / p.block_size;
    const long long slot = (long long)table[blk] * p.block_size + (pos - blk * p.block_size);
    if (slot >= 0 && slot < p.n_slots) return slot;
    if (p.status) atomicExch(p.status, 131);
    return -1;
  };
  auto issue = [&](int t, long long slot) {
    if (t < mine) {
      unsigned char* st = ring + (t % NST) * Cfg::stage_bytes;
      const unsigned ok = __ballot_sync(0xffffffffu, slot >= 0) & 0xffffu;
      if (lane == 0) ok_sm[warp][t % NST] = ok;
#pragma unroll
      for (int i = 0; i < kSdTile * U / 32; ++i) {
        const int e = i * 32 + lane, r = e / U, u = e % U;
        const long long sl = __shfl_sync(0xffffffffu, slot, r);
        const long long at = sl >= 0 ? (sl * p.Hkv + hk) * Cfg::row_bytes + u * 16 : 0;
        sd_cp16(st + (r * U + sd_unit_k<U, Cfg::piece>(r, u)) * 16, reinterpret_cast<const unsigned char*>(p.k) + at, sl >= 0);
        sd_cp16(st + Cfg::tile_bytes / 2 + (r * U + sd_unit_v<U, Cfg::piece>(r, u)) * 16, reinterpret_cast<const unsigned char*>(p.v) + at, sl >= 0);
      }
      if constexpr (kScaled) {
        const long long at = slot >= 0 ? slot * p.Hkv + hk : 0;
        sd_cp4(st + Cfg::tile_bytes + lane * 4, (lane < 16 ? p.k_scale : p.v_scale) + at, slot >= 0);
      }
    }
    sd_commit();
  };

  float o[NJ * 8][4];
#pragma unroll
  for (int i = 0; i < NJ * 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float mx[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};      // rows gid and (WIDE) gid + 8
  const float c = p.scale * 1.4426950408889634f;

#pragma unroll
  for (int t = 0; t < NST - 1; ++t) issue(t, slot_of(t));
  long long next = slot_of(NST - 1);
  for (int t = 0; t < mine; ++t) {
    issue(t + NST - 1, next);
    next = slot_of(t + NST);
    sd_wait<NST - 1>();
    __syncwarp();
    const unsigned char* st = ring + (t % NST) * Cfg::stage_bytes;
    const unsigned char* vt = st + Cfg::tile_bytes / 2;
    const unsigned ok = ok_sm[warp][t % NST];
    float s[2][4] = {};
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int pc = tig + 4 * i;
      const uint4 qa = *reinterpret_cast<const uint4*>(q_sm + (gid * (D / 8) + (pc ^ ((gid & 1) << 2))) * 16);
      uint4 qb = make_uint4(0, 0, 0, 0);
      if constexpr (WIDE) qb = *reinterpret_cast<const uint4*>(q_sm + ((gid + 8) * (D / 8) + (pc ^ ((gid & 1) << 2))) * 16);
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const int r = gid + 8 * nt;
        uint32_t w[4];
        sd_load8<F>(st + (r * U + sd_unit_k<U, Cfg::piece>(r, pc * Cfg::piece / 16)) * 16 + pc * Cfg::piece % 16, w);
        mma_bf16_16816(s[nt], qa.x, qb.x, qa.y, qb.y, w[0], w[1]);
        mma_bf16_16816(s[nt], qa.z, qb.z, qa.w, qb.w, w[2], w[3]);
      }
    }
    // scores in units of log2; this lane's keys are 2 tig, 2 tig + 1 (nt 0) and 8 more (nt 1)
    float p4[2][4];                                              // [row half][key]
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int key = 8 * nt + 2 * tig + e;
        float f = c;
        if constexpr (kScaled) f *= reinterpret_cast<const float*>(st + Cfg::tile_bytes)[key];
        const bool in = ok >> key & 1;
        p4[0][2 * nt + e] = in ? s[nt][e] * f : -INFINITY;
        p4[1][2 * nt + e] = in ? s[nt][2 + e] * f : -INFINITY;
      }
    bool grew = false;
    float alpha[2] = {1.f, 1.f};
#pragma unroll
    for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
      float t4 = fmaxf(fmaxf(p4[h][0], p4[h][1]), fmaxf(p4[h][2], p4[h][3]));
      t4 = fmaxf(t4, __shfl_xor_sync(0xffffffffu, t4, 1));
      t4 = fmaxf(t4, __shfl_xor_sync(0xffffffffu, t4, 2));
      if (t4 > mx[h]) {
        alpha[h] = sd_exp2(mx[h] - t4);
        mx[h] = t4;
        grew = true;
      }
      const float ref = mx[h] == -INFINITY ? 0.f : mx[h];
      float sum = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        p4[h][k] = sd_exp2(p4[h][k] - ref);
        sum += p4[h][k];
      }
      l[h] = l[h] * alpha[h] + sum;
    }
    if (__any_sync(0xffffffffu, grew)) {
      const float a1 = WIDE ? alpha[1] : alpha[0];
#pragma unroll
      for (int i = 0; i < NJ * 8; ++i) o[i][0] *= alpha[0], o[i][1] *= alpha[0], o[i][2] *= a1, o[i][3] *= a1;
    }
    if constexpr (kScaled) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float f = reinterpret_cast<const float*>(st + Cfg::tile_bytes)[16 + 8 * (k >> 1) + 2 * tig + (k & 1)];
        p4[0][k] *= f;
        if constexpr (WIDE) p4[1][k] *= f;
      }
    }
    uint32_t hi[2][2], lw[2][2];                                 // [row half][key half]
#pragma unroll
    for (int h = 0; h < (WIDE ? 2 : 1); ++h)
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float x = p4[h][2 * k], y = p4[h][2 * k + 1];
        hi[h][k] = sd_pack(x, y);
        lw[h][k] = sd_pack(x - __uint_as_float(hi[h][k] << 16), y - __uint_as_float(hi[h][k] & 0xffff0000u));
      }
#pragma unroll
    for (int jj = 0; jj < NJ; ++jj) {
      const int pc = gid + 8 * jj;
      uint32_t v[4][4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int r = 2 * tig + (k & 1) + 8 * (k >> 1);
        sd_load8<F>(vt + (r * U + sd_unit_v<U, Cfg::piece>(r, pc * Cfg::piece / 16)) * 16 + pc * Cfg::piece % 16, v[k]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = e & 1 ? 0x7632u : 0x5410u;
        const uint32_t b0 = __byte_perm(v[0][e >> 1], v[1][e >> 1], sel), b1 = __byte_perm(v[2][e >> 1], v[3][e >> 1], sel);
        if constexpr (WIDE) {
          mma_bf16_16816(o[jj * 8 + e], hi[0][0], hi[1][0], hi[0][1], hi[1][1], b0, b1);
          mma_bf16_16816(o[jj * 8 + e], lw[0][0], lw[1][0], lw[0][1], lw[1][1], b0, b1);
        } else {
          mma_bf16_16816(o[jj * 8 + e], hi[0][0], lw[0][0], hi[0][1], lw[0][1], b0, b1);
        }
      }
    }
    __syncwarp();                                                // the stage may be refilled
  }

  // ---- join the warps.  Row r of warp w: maximum and sum in ml, O in the (idle) ring as [w][r][D]
  sd_wait<0>();
  __syncthreads();
#pragma unroll
  for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
    l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
    if (tig == 0) ml[warp][gid + 8 * h][0] = mx[h], ml[warp][gid + 8 * h][1] = l[h];
  }
  float* os = reinterpret_cast<float*>(sm);
#pragma unroll
  for (int jj = 0; jj < NJ; ++jj)
#pragma unroll
    for (int e = 0; e < 2; ++e) {                                // columns (2 tig + e + 8 jj) 8 .. + 7
      const int col = (2 * tig + e + 8 * jj) * 8;
#pragma unroll
      for (int h = 0; h < (WIDE ? 2 : 1); ++h) {
        float4* dst = reinterpret_cast<float4*>(os + ((warp * R + gid + 8 * h) * D + col));
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          float f[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float (&x)[4] = o[jj * 8 + q * 4 + i];
            f[i] = WIDE ? x[2 * h + e] : x[e] + x[2 + e];
          }
          dst[q] = make_float4(f[0], f[1], f[2], f[3]);
        }
      }
    }
  __syncthreads();
  // weights of the warps of row r: 2^(m_w - M)
  auto weight = [](float mw, float M) { return mw == -INFINITY ? 0.f : sd_exp2(mw - M); };
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
      uint2 w2 = make_uint2(sd_pack(a.x * inv, a.y * inv), sd_pack(a.z * inv, a.w * inv));
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
    uint2 w2 = make_uint2(sd_pack(a.x * inv, a.y * inv), sd_pack(a.z * inv, a.w * inv));
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
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return (int)e;
  if (dev >= 64 || !(done.load(std::memory_order_relaxed) >> dev & 1)) {       // the limit belongs to a device
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  }
  const int G = p.Hq / p.Hkv, hg = (G + R - 1) / R;
  if ((long long)p.Hkv * hg > 65535 || p.B > 65535) return (int)cudaErrorInvalidValue;
  int splits = p.splits;
  if (splits == 0) {
    const long long most = min((long long)p.window + p.sinks, (long long)p.max_blocks * p.block_size);
    const long long tiles = (most + kSdTile - 1) / kSdTile, rows = (long long)p.B * p.Hkv * hg;
    splits = 1;
    while (splits < 8 && rows * splits < 2 * 148 && splits * 2 * kSdWarps <= tiles) splits *= 2;
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
      (p.splits != 0 && p.splits != 1 && p.splits != 2 && p.splits != 4 && p.splits != 8))
    return (int)cudaErrorInvalidValue;
  switch (p.D) {
    case 64: return mmb::launch_sinks_f<64>(p, stream);
    case 128: return mmb::launch_sinks_f<128>(p, stream);
    case 256: return mmb::launch_sinks_f<256>(p, stream);
    default: return (int)cudaErrorInvalidValue;
  }
}
