// Loads and stores of activations whose element type is a run-time choice (0 bf16, 1 fp16, 2 fp32), as fp32 values.  The type is the
// same for every thread of a launch, so the branches are uniform.
#pragma once
#include "common.cuh"

namespace mmb {

__host__ __device__ __forceinline__ int elt_bytes(int t) { return t == 2 ? 4 : 2; }

__device__ __forceinline__ float ld1(const void* p, long long i, int t) {
  if (t == 0) return __bfloat162float(reinterpret_cast<const bf16*>(p)[i]);
  if (t == 1) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void st1(void* p, long long i, int t, float v) {
  if (t == 0) reinterpret_cast<bf16*>(p)[i] = __float2bfloat16(v);
  else if (t == 1) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<float*>(p)[i] = v;
}
// V consecutive values; V > 1 needs V * element size bytes of alignment (at most 16).
template <int V>
__device__ __forceinline__ void unpack16(const uint32_t* w, int t, float* v) {
#pragma unroll
  for (int i = 0; i < V / 2; ++i) {
    float2 f;
    if (t == 0) f = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    else f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
template <int V>
__device__ __forceinline__ void ldv(const void* p, long long i, int t, float* v) {
  if constexpr (V == 1) {
    v[0] = ld1(p, i, t);
  } else if (t == 2) {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
#pragma unroll
    for (int j = 0; j < V / 4; ++j) {
      const float4 f = q[j];
      v[4 * j] = f.x, v[4 * j + 1] = f.y, v[4 * j + 2] = f.z, v[4 * j + 3] = f.w;
    }
  } else {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p) + i;
    uint32_t w[V / 2];
    if constexpr (V == 8) {
      const uint4 u = *reinterpret_cast<const uint4*>(h);
      w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
    } else {
      const uint2 u = *reinterpret_cast<const uint2*>(h);
      w[0] = u.x, w[1] = u.y;
    }
    unpack16<V>(w, t, v);
  }
}
__device__ __forceinline__ uint32_t pack16(float a, float b, int t) {
  if (t == 0) {
    const bf162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <int V>
__device__ __forceinline__ void stv(void* p, long long i, int t, const float* v) {
  if constexpr (V == 1) {
    st1(p, i, t, v[0]);
  } else if (t == 2) {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
#pragma unroll
    for (int j = 0; j < V / 4; ++j) q[j] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
    uint16_t* h = reinterpret_cast<uint16_t*>(p) + i;
    if constexpr (V == 8) {
      *reinterpret_cast<uint4*>(h) = make_uint4(pack16(v[0], v[1], t), pack16(v[2], v[3], t), pack16(v[4], v[5], t), pack16(v[6], v[7], t));
    } else {
      *reinterpret_cast<uint2*>(h) = make_uint2(pack16(v[0], v[1], t), pack16(v[2], v[3], t));
    }
  }
}
// The same in two halves: raw bits first, so that a batch of loads is in flight before the first conversion waits for its data (a branch
// on the type around load and conversion together would wait load by load).  ES: bytes of an element; V values are V * ES / 4 words (V * ES >= 4)
// or one half word.
template <int V, int ES>
struct Raw {
  uint32_t w[V * ES >= 4 ? V * ES / 4 : 1];
};
template <int V, int ES>
__device__ __forceinline__ void ld_raw(const void* p, long long i, Raw<V, ES>& r) {
  const unsigned char* a = reinterpret_cast<const unsigned char*>(p) + i * ES;
  if constexpr (V * ES == 2) {
    r.w[0] = *reinterpret_cast<const uint16_t*>(a);
  } else if constexpr (V * ES == 4) {
    r.w[0] = *reinterpret_cast<const uint32_t*>(a);
  } else if constexpr (V * ES == 8) {
    const uint2 u = *reinterpret_cast<const uint2*>(a);
    r.w[0] = u.x, r.w[1] = u.y;
  } else {
#pragma unroll
    for (int j = 0; j < V * ES / 16; ++j) {
      const uint4 u = reinterpret_cast<const uint4*>(a)[j];
      r.w[4 * j] = u.x, r.w[4 * j + 1] = u.y, r.w[4 * j + 2] = u.z, r.w[4 * j + 3] = u.w;
    }
  }
}
template <int V, int ES>
__device__ __forceinline__ void cvt_raw(const Raw<V, ES>& r, int t, float* v) {
  if constexpr (ES == 4) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = __uint_as_float(r.w[i]);
  } else if constexpr (V == 1) {
    v[0] = t == 0 ? __uint_as_float(r.w[0] << 16) : __half2float(__ushort_as_half((unsigned short)r.w[0]));
  } else {
    unpack16<V>(r.w, t, v);
  }
}

__device__ __forceinline__ uint32_t bits1(const void* p, long long i, int t) {
  return t == 2 ? reinterpret_cast<const uint32_t*>(p)[i] : reinterpret_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float value1(uint32_t w, int t) {
  return t == 0 ? __uint_as_float(w << 16) : t == 1 ? __half2float(__ushort_as_half((unsigned short)w)) : __uint_as_float(w);
}

// Whether rows of a [*, n] tensor can be read or written in pieces of `v` values.
inline bool rows_aligned(const void* p, long long ld, int t, int v) {
  const int bytes = v * elt_bytes(t) < 16 ? v * elt_bytes(t) : 16;
  return p == nullptr || (reinterpret_cast<uintptr_t>(p) % bytes == 0 && (ld * elt_bytes(t)) % bytes == 0);
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
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 16 bytes from global to shared memory, zeros where they do not exist.
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Pool row of a sequence, or -1 where it is skipped.
__device__ __forceinline__ long long pool_row(const long long* rows, int s, int pool_rows, int* status) {
  const long long r = rows ? rows[s] : s;
  if (r >= 0 && r < pool_rows) return r;
  if (r >= 0 && status) atomicExch(status, 130);
  return -1;
}

}  // namespace mmb
