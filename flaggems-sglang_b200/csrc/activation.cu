// Gated activation of [M, 2I] rows (gate, then linear), its result in the rows' type or quantised to e4m3 per 1 x 128 group.
//
//   silu        y = g / (1 + exp(-g)) * u
//   gelu        y = g Phi(g) u,  Phi the normal distribution
//   swiglu_oai  g clamped from above, u to [-limit, limit];  y = g / (1 + exp(-alpha g)) * (u + 1)
//
// y is fp32 until it is rounded once, to its type or to e4m3.  Bound by HBM: 4 bytes in and 2 (or 1 + 1/32) out per
// element; 4096 rows of 18432, silu, in 67.2 us (6.7 TB/s), quantised in 63.3 (6.0 TB/s, 92 % of a copy's rate), swiglu_oai in 74.3 and 77.4.  GELU
// is bound by its instructions: 77.6 and 82.3.
// A thread takes two chunks of eight columns of a row; sixteen neighbours (rows off 16 bytes: a warp) hold a
// group, so its maximum is found by shuffles.
// Rows along the grid's x: no index needs a division.
#include <algorithm>

#include "block_ops.cuh"
#include "quant.cuh"

namespace b200moe {

namespace {

__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ unsigned long long both(float v) { return pack_f32x2(v, v); }

// exp(-a), exp(-b) for a, b in [0, 128].  The exponent -a log2 e is -h + l: h the rounded product, l what its rounding and that of log2 e leave,
// put back as 2^-h (1 + l ln 2).  (2^-h alone is off by a 2^-24: 2^-19 of the result where a is 32.)
__device__ __forceinline__ unsigned long long exp_neg2(float a, float b) {
  constexpr float kHigh = 1.44269502162933349609375f, kLow = 1.92596299e-8f;      // log2 e
  const unsigned long long x = pack_f32x2(a, b), h = mul2(x, both(kHigh));
  const unsigned long long l = fma2(x, both(-kLow), fma2(x, both(-kHigh), h));
  float ha, hb;
  unpack_f32x2(h, ha, hb);
  const unsigned long long e = pack_f32x2(exp2_fast(-ha), exp2_fast(-hb));
  return fma2(e, mul2(l, both(0.693147181f)), e);
}

// Two columns at once (packed fp32: what does not have to go through the special functions costs one instruction for both).
// EXACT: fp32 rows.  Their results show what 16-bit ones and e4m3 round away (within 2^-24 (8 + |z|) of the result; over normally distributed rows
// as few e4m3 values lie on the other side of a boundary either way), and their loads and stores take longer than the arithmetic:
// 16-bit rows of 4096 x 18432, quantised, take 80 us this way and 63 without.
template <int ACT, bool EXACT>
__device__ __forceinline__ unsigned long long activate2(float g0, float g1, float u0, float u1, float alpha, float limit) {
  if (ACT == B200MOE_ACT_GELU) {
    // (max(g, 0) - a Phi(-a)) u with a = |g| and Phi(-a) = exp(-a^2 / 2) t P(t), t = 1 / (1 + 0.306 a): P is a polynomial of degree seven, fitted
    // to the least relative error over [0, 15], 2^-23.2 (in fp32 2^-21.2 at most, 2^-23.2 in the mean).  Relative to the result, so that
    // negative g keep their digits: from 1 + erf(g / sqrt 2) they lose all of them down to -5, and erff takes 104 us where this takes 82,
    // 4096 rows of 18432, quantised.  fp32 rows put the roundings of a^2 and of its product with log2 e / 2 back behind the exponential, as
    // above; for others they are a^2 2^-24 of a small result.
    constexpr float kHigh = 0.721347510814666748046875f, kLow = 9.62981495e-9f;        // log2 e / 2
    const float a0 = fminf(fabsf(g0), 15.f), a1 = fminf(fabsf(g1), 15.f);             // (exp(-15^2 / 2) is zero in fp32)
    const unsigned long long x = pack_f32x2(a0, a1), w = mul2(x, x), h = mul2(w, both(kHigh));
    float a, b;
    unpack_f32x2(fma2(x, both(0.306f), both(1.f)), a, b);
    const unsigned long long t = pack_f32x2(rcp_fast(a), rcp_fast(b));
    unsigned long long p = fma2(t, both(-0.0365375467f), both(0.150698751f));          // -P
    p = fma2(p, t, both(-0.179383159f));
    p = fma2(p, t, both(0.0330344141f));
    p = fma2(p, t, both(-0.118628524f));
    p = fma2(p, t, both(-0.104367673f));
    p = fma2(p, t, both(-0.122772224f));
    p = fma2(p, t, both(-0.122044101f));
    unpack_f32x2(h, a, b);
    unsigned long long e = pack_f32x2(exp2_fast(-a), exp2_fast(-b));
    if (EXACT) {
      unsigned long long l = fma2(w, both(-kLow), fma2(w, both(-kHigh), h));
      l = fma2(fma2(pack_f32x2(-a0, -a1), x, w), both(kHigh), l);
      e = fma2(e, mul2(l, both(0.693147181f)), e);
    }
    unpack_f32x2(mul2(pack_f32x2(g0, g1), both(0.5f)), a, b);        // (g + |g|) / 2: NaN where g is NaN or minus infinity, as g Phi(g) is
    const unsigned long long positive = pack_f32x2(fmaf(0.5f, fabsf(g0), a), fmaf(0.5f, fabsf(g1), b));
    return mul2(fma2(mul2(mul2(p, t), e), x, positive), pack_f32x2(u0, u1));
  }
  if (ACT == B200MOE_ACT_SWIGLU_OAI && limit > 0.f) {
    // (not fminf / fmaxf alone: they drop a NaN)
    g0 = g0 > limit ? limit : g0;
    g1 = g1 > limit ? limit : g1;
    u0 = u0 > limit ? limit : u0 < -limit ? -limit : u0;
    u1 = u1 > limit ? limit : u1 < -limit ? -limit : u1;
  }
  const unsigned long long g = pack_f32x2(g0, g1);
  unsigned long long u = pack_f32x2(u0, u1);
  if (ACT == B200MOE_ACT_SWIGLU_OAI) u = add2(u, both(1.f));
  float a, b;
  if (EXACT) {
    // g sigmoid(z) = (z < 0 ? g e : g) / (1 + e) with e = exp(-|z|), z = alpha g: nothing overflows.  1 / (1 + e) takes a step of Newton's
    // iteration.
    float z0, z1;
    unpack_f32x2(mul2(g, both(ACT == B200MOE_ACT_SWIGLU_OAI ? alpha : 1.f)), z0, z1);
    const unsigned long long e = exp_neg2(fminf(fabsf(z0), 128.f), fminf(fabsf(z1), 128.f));
    const unsigned long long neg = fma2(e, both(-1.f), both(-1.f));
    unpack_f32x2(neg, a, b);
    unsigned long long r = pack_f32x2(rcp_fast(-a), rcp_fast(-b));
    r = fma2(fma2(neg, r, both(1.f)), r, r);
    unpack_f32x2(mul2(g, e), a, b);
    return mul2(mul2(pack_f32x2(z0 < 0.f ? a : g0, z1 < 0.f ? b : g1), r), u);
  }
  unpack_f32x2(mul2(g, both(-1.44269504f * (ACT == B200MOE_ACT_SWIGLU_OAI ? alpha : 1.f))), a, b);
  unpack_f32x2(add2(pack_f32x2(exp2_fast(a), exp2_fast(b)), both(1.f)), a, b);
  return mul2(mul2(g, pack_f32x2(rcp_fast(a), rcp_fast(b))), u);
}

constexpr int kRuns = 2;      // chunks of a thread, all loads in flight at once
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(256)
gated_activation_kernel(const ActArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const long long row = blockIdx.x;
  const int first = blockIdx.y * blockDim.x * kRuns + threadIdx.x, lane = threadIdx.x & 31;
  const T* src = static_cast<const T*>(a.x) + row * a.ldx;
  Raw8<T> gr[kRuns], ur[kRuns];
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    int e0, n;
    chunk_at<VEC>(first + r * blockDim.x, lane, a.I, e0, n);
    load8<T, VEC>(src + e0, n, gr[r]);
    load8<T, VEC>(src + a.I + e0, n, ur[r]);
  }
#pragma unroll
  for (int r = 0; r < kRuns; ++r) {
    // Whole warps stay: the shuffles below are the warp's.  One whose chunks all lie beyond the row leaves: half of the last CTA's of a row of
    // 18432, and GELU took 94 us with their arithmetic and takes 82 without.
    if ((first + r * static_cast<int>(blockDim.x) - lane) * 8 >= a.I) break;
    int e0, n;
    chunk_at<VEC>(first + r * blockDim.x, lane, a.I, e0, n);
    float g[8], u[8];
    unpack8<T>(gr[r], g);
    unpack8<T>(ur[r], u);
#pragma unroll
    for (int i = 0; i < 8; i += 2) unpack_f32x2(activate2<ACT, sizeof(T) == 4>(g[i], g[i + 1], u[i], u[i + 1], a.alpha, a.limit), g[i], g[i + 1]);
    if (a.y_scale == nullptr) {
      store8<T, VEC>(static_cast<T*>(a.y) + row * a.I + e0, n, g);
      continue;
    }
    quantise8<VEC>(g, static_cast<uint8_t*>(a.y) + row * a.I, a.y_scale + row * ((a.I + 127) >> 7), e0, n, lane);
  }
}

template <typename T, int ACT>
int launch_typed(const ActArgs& a, cudaStream_t stream) {
  const int chunks = (a.I + 7) / 8;
  const int threads = std::min(256, ((chunks + kRuns - 1) / kRuns + 31) / 32 * 32), per_cta = threads * kRuns;
  const int segments = (chunks + per_cta - 1) / per_cta;      // (B200MOE_ACT_MAX_I: at most 65535)
  note_launch("gated_activation_kernel");
  const dim3 grid(a.M, segments);
  cudaError_t err = a.vec ? launch_kernel(gated_activation_kernel<T, ACT, true>, grid, dim3(threads), 0, stream, a.pdl != 0, a)
                          : launch_kernel(gated_activation_kernel<T, ACT, false>, grid, dim3(threads), 0, stream, a.pdl != 0, a);
  return err == cudaSuccess ? B200MOE_OK : B200MOE_ERR_CUDA;
}

template <typename T>
int launch_act(const ActArgs& a, int activation, cudaStream_t stream) {
  switch (activation) {
    case B200MOE_ACT_SILU: return launch_typed<T, B200MOE_ACT_SILU>(a, stream);
    case B200MOE_ACT_GELU: return launch_typed<T, B200MOE_ACT_GELU>(a, stream);
    case B200MOE_ACT_SWIGLU_OAI: return launch_typed<T, B200MOE_ACT_SWIGLU_OAI>(a, stream);
    default: return B200MOE_ERR_BAD_ARG;
  }
}

}  // namespace

int launch_gated_activation(const ActArgs& a, int activation, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case B200MOE_DTYPE_BF16: return launch_act<__nv_bfloat16>(a, activation, stream);
    case B200MOE_DTYPE_FP16: return launch_act<__half>(a, activation, stream);
    case B200MOE_DTYPE_FP32: return launch_act<float>(a, activation, stream);
    default: return B200MOE_ERR_BAD_ARG;
  }
}

}  // namespace b200moe
