// e4m3 values of a 1 x 128 group and 8-element access, shared by the kernels that quantise rows.
#pragma once
#include "common.cuh"

namespace b200moe {

// A group's scale: max(amax, 1e-10) / 448 (what per_token_group_quant_fp8 stores).  The divisor is known: the product with its
// reciprocal, corrected once by the exact remainder (Brisebarre, Muller and Raina, "Accelerating correctly rounded floating-point division when
// the divisor is known in advance", 2004).  Compared with a division for every mantissa, at both ends of
// the range too.
__device__ __forceinline__ float group_scale(float amax) {
  const float x = fmaxf(amax, 1e-10f), q = x * (1.0f / 448.0f);
  return x < INFINITY ? fmaf(fmaf(-448.0f, q, x), 1.0f / 448.0f, q) : x;
}
__device__ __forceinline__ unsigned long long mul2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {
  return __nv_cvt_float2_to_fp8x2(make_float2(lo, hi), __NV_SATFINITE, __NV_E4M3);
}

// e4m3(v / s), the quotient as an IEEE division rounds it (but for a negative zero, which comes out positive): the product with the
// reciprocal, corrected by the quotient's exact remainder (Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990).  The reciprocal is the correctly rounded one: an approximate one and a step of Newton's iteration, compared
// with __frcp_rn for every mantissa.  An infinite scale divides every number to zero and infinities to NaN.  The product alone is off by up to
// 1.5 ulp, with the same error of the reciprocal for a whole group, which moved values of the norms and the activation over boundaries of e4m3;
// and 16-bit values over a scale of their own are ties so often (every second warp held one) that redoing the division where the
// product lies next to a boundary doubled the kernel's instructions.
struct Divisor {
  unsigned long long inv2, neg2;
};
__device__ __forceinline__ Divisor divisor_of(float s, float inv) {
  const float neg = s < INFINITY ? -s : 0.f;
  return {pack_f32x2(inv, inv), pack_f32x2(neg, neg)};
}
__device__ __forceinline__ Divisor divisor_of(float s) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  return divisor_of(s, s < INFINITY ? fmaf(r, fmaf(-s, r, 1.0f), r) : 0.f);
}
__device__ __forceinline__ uint32_t e4m3_pair(unsigned long long v2, const Divisor& d) {
  const unsigned long long r = mul2(v2, d.inv2);
  float a, b;
  unpack_f32x2(fma2(fma2(d.neg2, r, v2), d.inv2, r), a, b);
  return e4m3x2(a, b);
}
__device__ __forceinline__ uint2 e4m3_divided(const unsigned long long (&v)[4], const Divisor& d) {
  return make_uint2(e4m3_pair(v[0], d) | e4m3_pair(v[1], d) << 16, e4m3_pair(v[2], d) | e4m3_pair(v[3], d) << 16);
}
__device__ __forceinline__ uint2 e4m3_divided(const float (&v)[8], const Divisor& d) {
  const unsigned long long v2[4] = {pack_f32x2(v[0], v[1]), pack_f32x2(v[2], v[3]), pack_f32x2(v[4], v[5]), pack_f32x2(v[6], v[7])};
  return e4m3_divided(v2, d);
}

__device__ __forceinline__ float amax8(const float (&v)[8]) {
  float m = fabsf(v[0]);
#pragma unroll
  for (int i = 1; i < 8; ++i) m = fmaxf(m, fabsf(v[i]));
  return m;
}
// Largest of 16 neighbouring lanes (a group of 128 elements, eight to a lane).  Whole warp.
__device__ __forceinline__ float max16(float m) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
// The same for N groups at once: shuffles keep their order, so group after group their latencies would add up.
template <int N>
__device__ __forceinline__ void max16(float (&m)[N]) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
}

template <>
__device__ __forceinline__ float to_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}

// Eight elements as they lie in memory: one 16-byte load of a 16-bit type, two of fp32.
template <typename T>
struct Raw8 {
  uint4 a[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ void unpack8(const Raw8<T>& r, float (&v)[8]) {
  const T* e = reinterpret_cast<const T*>(&r);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = to_f32<T>(e[i]);
}
// `n` elements of eight are there (VEC: all eight, neighbours, aligned; else 32 apart); the others read as zero.
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* __restrict__ p, int n, Raw8<T>& r) {
  if (VEC) {
    const uint4* src = reinterpret_cast<const uint4*>(p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) r.a[i] = n > 0 ? src[i] : make_uint4(0, 0, 0, 0);
  } else {
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = i < n ? p[32 * i] : from_f32<T>(0.f);
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* __restrict__ p, int n, const float (&v)[8]) {
  if (n <= 0) return;
  if (VEC) {
    Raw8<T> r;
    T* e = reinterpret_cast<T*>(&r);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f32<T>(v[i]);
    uint4* dst = reinterpret_cast<uint4*>(p);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) dst[i] = r.a[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[32 * i] = from_f32<T>(v[i]);
  }
}
// The same as four pairs of fp32, for packed arithmetic.
template <typename T>
__device__ __forceinline__ void unpack4x2(const Raw8<T>& r, unsigned long long (&v)[4]) {
  float f[8];
  unpack8<T>(r, f);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pack_f32x2(f[2 * i], f[2 * i + 1]);
}
__device__ __forceinline__ void split4x2(const unsigned long long (&v)[4], float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) unpack_f32x2(v[i], f[2 * i], f[2 * i + 1]);
}
// Quantised eight: one 8-byte store (VEC), or byte by byte.
template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* __restrict__ p, int n, uint2 q) {
  if (n <= 0) return;
  if (VEC) {
    *reinterpret_cast<uint2*>(p) = q;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[32 * i] = static_cast<uint8_t>((i < 4 ? q.x : q.y) >> (8 * (i & 3)));
  }
}

// Where the eight elements of a lane's chunk start in a row of `len`, and how many of them there are.  VEC: eight neighbours, one load.  Else a
// warp's 256 elements lie 32 apart in a lane, so that its lanes load and store side by side.  (With neighbours there too, 1000 rows of 2601
// before a block took 14.1 us, 8.3 so; 4096 rows of 2047 through silu 25.4 and 9.4.)
template <bool VEC>
__device__ __forceinline__ void chunk_at(int chunk, int lane, int len, int& e0, int& n) {
  e0 = VEC ? chunk * 8 : (chunk - lane) * 8 + lane;
  n = VEC ? max(0, min(8, len - e0)) : e0 < len ? min(8, (len - e0 + 31) >> 5) : 0;
}

// A lane's chunk in e4m3 with the scales of its 1 x 128 groups.  Whole warp; what lies beyond the row is zero.
template <bool VEC>
__device__ __forceinline__ void quantise8(const float (&v)[8], uint8_t* q, float* scale, int e0, int n, int lane) {
  if (VEC) {
    const float s = group_scale(max16(amax8(v)));
    store_q8<true>(q + e0, n, e4m3_divided(v, divisor_of(s)));
    if ((lane & 15) == 0 && n > 0) scale[e0 >> 7] = s;
  } else {
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) m[i >> 2] = fmaxf(m[i >> 2], fabsf(v[i]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      m[0] = fmaxf(m[0], __shfl_xor_sync(0xffffffffu, m[0], o));
      m[1] = fmaxf(m[1], __shfl_xor_sync(0xffffffffu, m[1], o));
    }
    const float s0 = group_scale(m[0]), s1 = group_scale(m[1]);
    store_q8<false>(q + e0, n, make_uint2(e4m3_divided(v, divisor_of(s0)).x, e4m3_divided(v, divisor_of(s1)).y));
    if (lane == 0 && n > 0) scale[e0 >> 7] = s0;
    if (lane == 0 && n > 4) scale[(e0 >> 7) + 1] = s1;
  }
}

}  // namespace b200moe
