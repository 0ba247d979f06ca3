// kv4_rows.cuh — what the two attention kernels of the paged 4-bit cache
// (kv4_attn.cu, kv4_prompt.cu) share: reading query rows and sequences,
// writing output rows, the values' binary16 forms.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "kv4.h"

namespace zgpu {

// 2^x, 0 below 2^-126: without .ftz every exponential costs three more
// operations for subnormals, which no probability here can be.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ uint32_t h2bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits2h(uint32_t u) { return *reinterpret_cast<__half2 *>(&u); }

template <class T>
__device__ __forceinline__ float4 q4(const T *p);
template <>
__device__ __forceinline__ float4 q4<float>(const float *p) {
  return __ldg(reinterpret_cast<const float4 *>(p));
}
template <>
__device__ __forceinline__ float4 q4<__half>(const __half *p) {
  const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
  const float2 a = __half22float2(bits2h(u.x)), b = __half22float2(bits2h(u.y));
  return make_float4(a.x, a.y, b.x, b.y);
}
template <>
__device__ __forceinline__ float4 q4<__nv_bfloat16>(const __nv_bfloat16 *p) {
  const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p));
  return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                     __uint_as_float(u.y & 0xFFFF0000u));
}
__device__ __forceinline__ void put4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void put4(__half *p, float4 v) {
  *reinterpret_cast<uint2 *>(p) = make_uint2(h2bits(__floats2half2_rn(v.x, v.y)), h2bits(__floats2half2_rn(v.z, v.w)));
}
__device__ __forceinline__ void put4(__nv_bfloat16 *p, float4 v) {
  __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
  *reinterpret_cast<uint2 *>(p) = make_uint2(*reinterpret_cast<uint32_t *>(&a), *reinterpret_cast<uint32_t *>(&b));
}

// The factor of a row's scores, scale log2(e) 2^e with e in -252..252, applied
// in two halves: 2^e alone may lie outside the normal numbers.  It is at
// least the smallest normal number: the prompt kernel's masked scores are -inf
// before it is applied, and -inf times 0 would be NaN.  A score that the floor
// makes larger is below 2^-88 all the same.
__device__ __forceinline__ float score_factor(float scale, int e) {
  const int a = e >> 1, b = e - a;
  const float half = scale * __uint_as_float(static_cast<uint32_t>(127 + a) << 23) * 1.44269504088896341f;
  return fmaxf(half * __uint_as_float(static_cast<uint32_t>(127 + b) << 23), 0x1p-126f);
}

// One sequence as the call gives it, with lengths that cannot lead outside
// the buffers; *bad says that they would have.
struct Kv4Seq {
  uint32_t q0, nq, len;
};
__device__ __forceinline__ Kv4Seq kv4_seq(const Kv4AttnParams &p, uint32_t i, bool *bad) {
  Kv4Seq s;
  s.q0 = p.starts[i];
  const uint32_t q1 = p.starts[i + 1];
  s.len = p.kv_lens[i];
  s.nq = q1 - s.q0;
  if (q1 < s.q0 || q1 > p.n_rows || s.nq > p.max_q) {
    s.nq = 0;
    *bad = true;
  }
  const uint64_t most = static_cast<uint64_t>(p.table_width) << p.bt_log2;
  if (s.len > most) {
    s.len = static_cast<uint32_t>(most);
    *bad = true;
  }
  return s;
}

// The exponents of 16 and 256, read back from shared memory so that they stay
// in registers: a logical operation takes one constant, and where both
// operands are known the compiler makes two operations of it.
struct Magic {
  uint32_t x16, x256;
};
__device__ __forceinline__ Magic magic(uint32_t saddr) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(saddr), "r"(0x4C004C00u), "r"(0x5C005C00u) : "memory");
  Magic g;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(g.x16), "=r"(g.x256) : "r"(saddr) : "memory");
  return g;
}
// Likewise those of 1024 and 64, for K.
struct KMagic {
  uint32_t x1024, x64;
};
__device__ __forceinline__ KMagic k_magic(uint32_t saddr) {
  asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(saddr), "r"(0x64006400u), "r"(0x54005400u) : "memory");
  KMagic g;
  asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(g.x1024), "=r"(g.x64) : "r"(saddr) : "memory");
  return g;
}
// The four V nibbles of both halves of w as (n - 8) d, exactly.
__device__ __forceinline__ void v_values(uint32_t w, __half2 d, __half2 m24d, const Magic &g, uint32_t (&v)[4]) {
  const uint32_t x = __byte_perm(w, 0u, 0x2301u);
  const __half2 m264 = __half2half2(__ushort_as_half(0xDC20));
  v[0] = h2bits(__hfma2(bits2h((w & 0x03C003C0u) | g.x16), d, m24d));
  v[1] = h2bits(__hmul2(__hadd2(bits2h((w & 0x003C003Cu) | g.x256), m264), d));
  v[2] = h2bits(__hmul2(__hadd2(bits2h((x & 0x003C003Cu) | g.x256), m264), d));
  v[3] = h2bits(__hfma2(bits2h((x & 0x03C003C0u) | g.x16), d, m24d));
}

}  // namespace zgpu
