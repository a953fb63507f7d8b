// Norms before and after a block, fused with the block's gate, the residual scale and the residual add.
//
//   z      = norm(x; w_post, b_post)  or  x
//   h      = residual + scale * gate * z                       the residual stream after the block
//   y      = norm(h; w_pre, b_pre)                             the next block's input, in 16 bits or e4m3 per 1 x 128 group
//   norm(v) = (v - mean) * rsqrt(mean((v - mean)^2) + eps) * (offset + w) + b        (RMS norm: mean = 0)
//
// Everything between the loads and the stores is fp32; h and y are each rounded once, y from the h that was not yet rounded.
// A row is read once: its elements stay in registers over both norms, eight to a chunk, CH chunks to a thread, `team` threads to a
// row.  Variances are taken around the mean in a second pass over the registers, and what the
// mean's own rounding left there is taken off both, so rows with a large mean lose nothing.
// Sums: shuffles within a warp, then one exchange through shared memory, always in the same order.
//
// Bound by HBM where there are many rows (of a copy's 6.54 TB/s): before a block, 4096 x 7168 quantised, 206.5 MB in 35.8 us, 88 %; after
// a block, 8192 x 5120 with a gate per token, 251.7 MB in 40.4 us, 95 %; 2000 x 16384, 43.9 us, 91 %.  Two norms in one pass hold the
// rows through four round trips of sums and reach 60 % (4096 x 4096, quantised, 30.1 us).  By a launch and one round trip to memory where
// there are few: one row of 7168 in 2.5 us, 33 of 4096 with both norms in 3.0.
#include <algorithm>
#include <type_traits>

#include "block_ops.cuh"
#include "quant.cuh"

namespace b200moe {

namespace {

constexpr int kRingBytes = 220 * 1024, kSmBytes = 226 * 1024;     // shared memory of a CTA's ring, of an SM's
constexpr int kNormSums = 3;    // block-wide sums of a norm of one row: the mean; the mean of the differences from it, and their squares


// Sum over the row's team.  `s`: one slot per warp of the CTA, used once.
__device__ __forceinline__ float team_sum(float v, float* s, int warps, int warp0, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps == 1) return v;
  if (lane == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = lane < warps ? s[warp0 + lane] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Two sums in the shuffles of one: after the first of them a half warp carries each.  `s`: `slots` apart.
__device__ __forceinline__ void team_sum(float& a, float& b, float* s, int slots, int warps, int warp0, int lane) {
  const bool upper = (lane & 16) != 0;
  float v = (upper ? b : a) + __shfl_xor_sync(0xffffffffu, upper ? a : b, 16);
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (warps > 1) {
    float* mine = s + (upper ? slots : 0);
    const int l = lane & 15;
    if (l == 0) mine[threadIdx.x >> 5] = v;
    __syncthreads();
    v = l < warps ? mine[warp0 + l] : 0.f;
    if (l + 16 < warps) v += mine[warp0 + l + 16];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  }
  const float other = __shfl_xor_sync(0xffffffffu, v, 16);
  a = upper ? other : v;
  b = upper ? v : other;
}

// A layer norm's mean is off by some roundings of itself, which can be many times the deviation where rows are nearly constant.  So the
// differences' own mean `d` is summed beside their squares and taken off both: of equal elements nothing is left.
__device__ __forceinline__ float variance(float squares, float d) {
  const float v = fmaf(-d, d, squares);
  return v < 0.f ? 0.f : v;
}

// Weights, biases and per-channel gates come in the rows' type or in fp32.
template <typename T>
struct Vector8 {
  Raw8<float> r;      // (a 16-bit type uses half of it)
};
template <typename T, bool VEC>
__device__ __forceinline__ void load_vector(const void* p, bool f32, int e, int n, Vector8<T>& v) {
  if (f32) load8<float, VEC>(static_cast<const float*>(p) + e, n, v.r);
  else load8<T, VEC>(static_cast<const T*>(p) + e, n, *reinterpret_cast<Raw8<T>*>(&v.r));
}
template <typename T>
__device__ __forceinline__ void unpack_vector(const Vector8<T>& v, bool f32, float (&o)[8]) {
  if (f32) unpack8<float>(v.r, o);
  else unpack8<T>(*reinterpret_cast<const Raw8<T>*>(&v.r), o);
}

template <int CH>
__device__ __forceinline__ float chunk_sum(const float (&v)[CH][8]) {
  float s = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) s += v[c][i];
  return s;
}

// v = norm(v); elements beyond the row (n[c] of eight are there) are zero on entry and left as they come out
// EARLY: the weights are on their way during the sums (few rows, where that is a round trip); else they are read where they are used
template <typename T, bool VEC, int CH, bool EARLY, bool LAYER>
__device__ __forceinline__ void normalise(float (&v)[CH][8], const int (&n)[CH], const int (&e0)[CH], const NormArgs& a,
                                          const void* w, const void* b, bool w_f32, bool b_f32, float* sums, int slots, int warps,
                                          int warp0, int lane) {
  Vector8<T> wr[EARLY ? CH : 1];
  if (EARLY && w != nullptr) {
#pragma unroll
    for (int c = 0; c < CH; ++c) load_vector<T, VEC>(w, w_f32, e0[c], n[c], wr[c]);
  }
  const float h = static_cast<float>(a.H);
  if (LAYER) {
    const float mean = team_sum(chunk_sum<CH>(v), sums, warps, warp0, lane) / h;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = i < n[c] ? v[c][i] - mean : 0.f;
  }
  float q = 0.f;
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int i = 0; i < 8; ++i) q = fmaf(v[c][i], v[c][i], q);
  float r, shift = 0.f;
  if (LAYER) {
    float d = chunk_sum<CH>(v);
    team_sum(d, q, sums + slots, slots, warps, warp0, lane);
    d /= h;
    r = rsqrtf(variance(q / h, d) + a.eps);
    shift = -d * r;
  } else {
    r = rsqrtf(team_sum(q, sums, warps, warp0, lane) / h + a.eps);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[c][i] = LAYER ? fmaf(v[c][i], r, (VEC ? n[c] > 0 : i < n[c]) ? shift : 0.f) : v[c][i] * r;
    if (w != nullptr) {
      float f[8];
      if (!EARLY) load_vector<T, VEC>(w, w_f32, e0[c], n[c], wr[0]);
      unpack_vector<T>(wr[EARLY ? c : 0], w_f32, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] *= a.offset + f[i];
    }
    if (b != nullptr) {
      Vector8<T> br;
      float f[8];
      load_vector<T, VEC>(b, b_f32, e0[c], n[c], br);
      unpack_vector<T>(br, b_f32, f);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] += f[i];
    }
    // (what lies beyond the row stays zero: its weights and biases were read as zero, its elements are)
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_gate_chunk(const NormArgs& a, long long row, int n, int e0, Vector8<T>& g) {
  const long long at = a.gate_mode == B200MOE_GATE_FULL ? row * a.ldg : 0;
  const void* p = a.gate_f32 ? static_cast<const void*>(static_cast<const float*>(a.gate) + at)
                             : static_cast<const void*>(static_cast<const T*>(a.gate) + at);
  load_vector<T, VEC>(p, a.gate_f32, e0, n, g);
}

// A row from its loaded elements to its stores.
template <typename T, typename R, bool VEC, int CH, bool EARLY, bool LAYER, bool POST = true, bool PRE = true>
__device__ __forceinline__ void finish_row(const NormArgs& a, long long row, const int (&n)[CH], const int (&e0)[CH], const Raw8<T> (&xr)[CH],
                                           const Raw8<R> (&rr)[CH], const Vector8<T> (&gr)[EARLY ? CH : 1], float* sums, int slots, int warps,
                                           int warp0, int lane) {
  float v[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) unpack8<T>(xr[c], v[c]);
  if (POST && a.post)
    normalise<T, VEC, CH, EARLY, LAYER>(v, n, e0, a, a.w_post, a.b_post, a.w_post_f32, a.b_post_f32, sums, slots, warps, warp0, lane);

  float scale = a.scale;
  if (a.gate_mode == B200MOE_GATE_TOKEN && row < a.M)
    scale *= a.gate_f32 ? static_cast<const float*>(a.gate)[row * a.ldg] : to_f32<T>(static_cast<const T*>(a.gate)[row * a.ldg]);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    if (a.gate_mode == B200MOE_GATE_CHANNEL || a.gate_mode == B200MOE_GATE_FULL) {
      float g[8];
      if (EARLY) {
        unpack_vector<T>(gr[EARLY ? c : 0], a.gate_f32, g);
      } else {
        Vector8<T> now;
        load_gate_chunk<T, VEC>(a, row, n[c], e0[c], now);
        unpack_vector<T>(now, a.gate_f32, g);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] *= g[i];
    }
    if (a.residual != nullptr) {
      float r[8];
      unpack8<R>(rr[c], r);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = fmaf(scale, v[c][i], r[i]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] *= scale;
    }
    if (a.hidden != nullptr) store8<R, VEC>(static_cast<R*>(a.hidden) + row * a.ldh + e0[c], n[c], v[c]);
  }
  if (!PRE || !a.pre) return;
  normalise<T, VEC, CH, EARLY, LAYER>(v, n, e0, a, a.w_pre, a.b_pre, a.w_pre_f32, a.b_pre_f32, sums + kNormSums * slots, slots, warps, warp0, lane);
  if (a.y_scale == nullptr) {
#pragma unroll
    for (int c = 0; c < CH; ++c) store8<T, VEC>(static_cast<T*>(a.y) + row * a.H + e0[c], n[c], v[c]);
  } else {
    const int groups = (a.H + 127) >> 7;
#pragma unroll
    for (int c = 0; c < CH; ++c) quantise8<VEC>(v[c], static_cast<uint8_t*>(a.y) + row * a.H, a.y_scale + row * groups, e0[c], n[c], lane);
  }
}

// POST, PRE: norms that the call may have
template <typename T, typename R, bool VEC, int CH, int THREADS, bool LAYER, bool POST, bool PRE>
__global__ void __launch_bounds__(THREADS, THREADS == 512 && CH == 1 ? 3 : 0)
block_norm_kernel(const NormArgs a) {
  __shared__ float s_sum[2 * kNormSums * 32];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int t = threadIdx.x % a.team;
  const int warps = a.team >> 5, warp0 = (threadIdx.x / a.team) * warps;
  const long long row = static_cast<long long>(blockIdx.x) * a.rows_per_cta + threadIdx.x / a.team;
  int n[CH], e0[CH];
  Raw8<T> xr[CH];
  Raw8<R> rr[CH];
  Vector8<T> gr[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    chunk_at<VEC>(c * a.team + t, lane, row < a.M ? a.H : 0, e0[c], n[c]);
    load8<T, VEC>(static_cast<const T*>(a.x) + row * a.ldx + e0[c], n[c], xr[c]);
    if (a.residual != nullptr) load8<R, VEC>(static_cast<const R*>(a.residual) + row * a.ldr + e0[c], n[c], rr[c]);
  }
  if (a.gate_mode == B200MOE_GATE_CHANNEL || a.gate_mode == B200MOE_GATE_FULL) {
#pragma unroll
    for (int c = 0; c < CH; ++c) load_gate_chunk<T, VEC>(a, row, n[c], e0[c], gr[c]);
  }
  finish_row<T, R, VEC, CH, true, LAYER, POST, PRE>(a, row, n, e0, xr, rr, gr, s_sum, 32, warps, warp0, lane);
}

__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Many rows: every thread keeps its elements of the next S - 1 rows on their way into shared memory while the CTA works on one, so
// that memory stays busy through the sums' round trips however few CTAs fit.  Weights, biases and a gate per channel are copied once and
// stay there (from L2 each of them cost a row another round trip).  A thread reads only what it has copied itself.
template <typename T, typename R, int CH, int S, bool LAYER>
__global__ void __launch_bounds__(512, 1)
block_norm_ring_kernel(const NormArgs args, int stage_bytes) {
  NormArgs a = args;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float s_sum[2][2 * kNormSums * 16];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warps = a.team >> 5;
  const long long step = gridDim.x;
  const uint32_t base = smem_u32(ring), r_at = static_cast<uint32_t>(a.H * sizeof(T));
  int n[CH], e0[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    e0[c] = (c * a.team + threadIdx.x) * 8;
    n[c] = e0[c] < a.H ? 8 : 0;
  }
  auto fetch = [&](long long row, int s) {
    if (row < a.M) {
      const uint32_t at = base + s * stage_bytes;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (n[c] == 0) continue;
        const T* x = static_cast<const T*>(a.x) + row * a.ldx + e0[c];
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) copy16_async(at + e0[c] * sizeof(T) + 16 * i, x + 16 / sizeof(T) * i);
        if (a.residual != nullptr) {
          const R* r = static_cast<const R*>(a.residual) + row * a.ldr + e0[c];
#pragma unroll
          for (int i = 0; i < static_cast<int>(sizeof(R) / 2); ++i) copy16_async(at + r_at + e0[c] * sizeof(R) + 16 * i, r + 16 / sizeof(R) * i);
        }
      }
    }
    copies_commit();
  };
  {
    uint32_t off = static_cast<uint32_t>(S * stage_bytes);
    auto keep = [&](const void*& p, bool f32) {
      if (p == nullptr) return;
      const uint32_t size = f32 ? 4 : sizeof(T);
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (n[c] != 0)
          for (uint32_t i = 0; i < size / 2; ++i)
            copy16_async(base + off + e0[c] * size + 16 * i, static_cast<const uint8_t*>(p) + e0[c] * size + 16 * i);
      p = ring + off;
      off += a.H * size;
    };
    keep(a.w_post, a.w_post_f32);
    keep(a.b_post, a.b_post_f32);
    keep(a.w_pre, a.w_pre_f32);
    keep(a.b_pre, a.b_pre_f32);
    if (a.gate_mode == B200MOE_GATE_CHANNEL) keep(a.gate, a.gate_f32);
  }
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(blockIdx.x + s * step, s);
  int s = 0, turn = 0;
  for (long long row = blockIdx.x; row < a.M; row += step) {
    fetch(row + (S - 1) * step, s == 0 ? S - 1 : s - 1);
    const Vector8<T> gr[1] = {};
    copies_wait<S - 1>();
    Raw8<T> xr[CH];
    Raw8<R> rr[CH];
    const uint8_t* at = ring + s * stage_bytes;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      load8<T, true>(reinterpret_cast<const T*>(at) + e0[c], n[c], xr[c]);
      if (a.residual != nullptr) load8<R, true>(reinterpret_cast<const R*>(at + r_at) + e0[c], n[c], rr[c]);
    }
    finish_row<T, R, true, CH, false, LAYER>(a, row, n, e0, xr, rr, gr, s_sum[turn], 16, warps, 0, lane);
    turn ^= 1;
    if (++s == S) s = 0;
  }
}

// The same for rows of up to 8192, with the form of the call known when it is compiled and the arithmetic packed two to an instruction.
enum Form { kBefore, kAfter, kBetween };
// FAST: every thread has all of its chunks (H a multiple of 512) and the vectors have the rows' type: no test of either per chunk.
template <typename T, typename R, int FORM, bool QUANT, bool LAYER, bool FAST>
__global__ void __launch_bounds__(512, 2)
block_norm_stream_kernel(const NormArgs a, int stages, int stage_bytes) {
  constexpr int CH = 2;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ float s_sum[2][2 * kNormSums * 16];
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31, warps = a.team >> 5;
  const long long step = gridDim.x;
  const uint32_t base = smem_u32(ring), r_at = static_cast<uint32_t>(a.H * sizeof(T));
  bool there[CH];
  int e0[CH];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    e0[c] = (c * a.team + static_cast<int>(threadIdx.x)) * 8;
    there[c] = e0[c] < a.H;
  }
  // Pointers step from row to row; what a chunk adds to them is one 32-bit number.  (Indexed by row and column, the addresses took a
  // third of the instructions.)
  const bool add = a.residual != nullptr, keep = a.hidden != nullptr;
  const uint8_t* px = reinterpret_cast<const uint8_t*>(static_cast<const T*>(a.x) + blockIdx.x * a.ldx + e0[0]);
  const uint8_t* pr = reinterpret_cast<const uint8_t*>(static_cast<const R*>(a.residual) + (add ? blockIdx.x * a.ldr + e0[0] : 0));
  const long long step_x = step * a.ldx * sizeof(T), step_r = step * a.ldr * sizeof(R);
  const uint32_t to_x = base + e0[0] * sizeof(T), to_r = base + r_at + e0[0] * sizeof(R), hop = a.team * 8;     // elements from chunk to chunk
  int ahead = blockIdx.x;                      // row that px and pr point to
  auto fetch = [&](uint32_t stage_at) {
    if (ahead < a.M) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        if (!FAST && !there[c]) continue;
        const uint32_t ox = c * hop * static_cast<uint32_t>(sizeof(T)), orr = c * hop * static_cast<uint32_t>(sizeof(R));
#pragma unroll
        for (int i = 0; i < static_cast<int>(sizeof(T) / 2); ++i) copy16_async(to_x + stage_at + ox + 16 * i, px + ox + 16 * i);
        if (add) {
#pragma unroll
          for (int i = 0; i < static_cast<int>(sizeof(R) / 2); ++i) copy16_async(to_r + stage_at + orr + 16 * i, pr + orr + 16 * i);
        }
      }
    }
    copies_commit();
    ahead += static_cast<int>(step);
    px += step_x;
    pr += step_r;
  };
  for (int s = 0; s < stages - 1; ++s) fetch(s * stage_bytes);

  const bool channel = a.gate_mode == B200MOE_GATE_CHANNEL;
  const float per = 1.f / static_cast<float>(a.H);      // (rounded: the mean is corrected, and nothing else sees more than 2^-24 of it)
  // v = (v - mean) * rsqrt(var + eps) * (offset + w) + b.  The vectors stay in L1.
  const unsigned long long offset2 = pack_f32x2(a.offset, a.offset);
  auto normalise2 = [&](unsigned long long (&v)[CH][4], const void* w, bool w_f32, const void* b, bool b_f32, float* sums) {
    constexpr bool EARLY = FAST && FORM != kBetween;      // (two norms: the registers for it are not there, 30.2 us became 33.5)
    Raw8<T> early[EARLY ? CH : 1];
    if (EARLY && w != nullptr) {
#pragma unroll
      for (int c = 0; c < CH; ++c) load8<T, true>(static_cast<const T*>(w) + e0[c], 8, early[EARLY ? c : 0]);
    }
    if (LAYER) {
      unsigned long long t = 0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) t = add2(t, v[c][i]);
      float lo, hi;
      unpack_f32x2(t, lo, hi);
      const float mean = team_sum(lo + hi, sums, warps, 0, lane) * per;
      const unsigned long long m2 = pack_f32x2(-mean, -mean);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = FAST || there[c] ? add2(v[c][i], m2) : 0;
    }
    unsigned long long t = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) t = fma2(v[c][i], v[c][i], t);
    float lo, hi;
    unpack_f32x2(t, lo, hi);
    float r, shift = 0.f;
    if (LAYER) {
      unsigned long long t1 = 0;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 4; ++i) t1 = add2(t1, v[c][i]);
      float q = lo + hi, d;
      unpack_f32x2(t1, lo, hi);
      d = lo + hi;
      team_sum(d, q, sums + 16, 16, warps, 0, lane);
      d *= per;
      r = rsqrtf(variance(q * per, d) + a.eps);
      shift = -d * r;
    } else {
      r = rsqrtf(team_sum(lo + hi, sums, warps, 0, lane) * per + a.eps);
    }
    const unsigned long long shift2 = pack_f32x2(shift, shift);
    const unsigned long long r2 = pack_f32x2(r, r);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (!FAST && !there[c]) continue;
      if (w != nullptr) {
        float f[8];
        if (FAST) {
          if (!EARLY) load8<T, true>(static_cast<const T*>(w) + e0[c], 8, early[0]);
          unpack8<T>(early[EARLY ? c : 0], f);
        } else {
          Vector8<T> wr;
          load_vector<T, true>(w, w_f32, e0[c], 8, wr);
          unpack_vector<T>(wr, w_f32, f);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = mul2(LAYER ? fma2(v[c][i], r2, shift2) : mul2(v[c][i], r2), add2(pack_f32x2(f[2 * i], f[2 * i + 1]), offset2));
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = LAYER ? fma2(v[c][i], r2, shift2) : mul2(v[c][i], r2);
      }
      if (b != nullptr) {
        Vector8<T> br;
        float f[8];
        load_vector<T, true>(b, b_f32, e0[c], 8, br);
        unpack_vector<T>(br, b_f32, f);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = add2(v[c][i], pack_f32x2(f[2 * i], f[2 * i + 1]));
      }
    }
  };

  uint8_t* ph = reinterpret_cast<uint8_t*>(static_cast<R*>(a.hidden) + (keep ? blockIdx.x * a.ldh + e0[0] : 0));
  constexpr uint32_t kOut = QUANT ? 1 : sizeof(T);
  uint8_t* py = static_cast<uint8_t*>(a.y) + (static_cast<size_t>(blockIdx.x) * a.H + e0[0]) * kOut;
  const int groups = (a.H + 127) >> 7;
  float* ps = a.y_scale + (QUANT ? static_cast<size_t>(blockIdx.x) * groups + (e0[0] >> 7) : 0);
  const long long step_h = step * a.ldh * sizeof(R), step_y = step * a.H * kOut, step_s = step * groups;
  const bool full = a.gate_mode == B200MOE_GATE_FULL, token = a.gate_mode == B200MOE_GATE_TOKEN;
  const uint32_t stage_end = stages * stage_bytes;
  uint32_t now = 0, next = (stages - 1) * stage_bytes;       // stage of this row, of the one that is fetched
  int turn = 0;
  // The next row's gate, as it lies in memory: turned into a number where it was read it would be waited for there.
  auto token_gate = [&](int row) -> uint32_t {
    if (!token || row >= a.M) return 0;
    return a.gate_f32 || sizeof(T) == 4 ? static_cast<const uint32_t*>(a.gate)[row * a.ldg] : static_cast<const uint16_t*>(a.gate)[row * a.ldg];
  };
  auto gate_value = [&](uint32_t bits) {
    if (!token) return 1.f;
    if (a.gate_f32 || sizeof(T) == 4) return __uint_as_float(bits);
    const uint16_t low = static_cast<uint16_t>(bits);
    return to_f32<T>(*reinterpret_cast<const T*>(&low));
  };
  uint32_t gate_next = token_gate(blockIdx.x);
#pragma unroll 1
  for (int row = blockIdx.x; row < a.M; row += static_cast<int>(step)) {
    fetch(next);
    next = now;
    const float scale = a.scale * gate_value(gate_next);
    gate_next = token_gate(row + static_cast<int>(step));
    if (stages == 4) copies_wait<3>();
    else if (stages == 3) copies_wait<2>();
    else copies_wait<1>();
    const uint8_t* at = ring + now;
    unsigned long long v[CH][4] = {};
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (!FAST && !there[c]) continue;
      Raw8<T> x;
      load8<T, true>(reinterpret_cast<const T*>(at) + e0[c], 8, x);
      unpack4x2<T>(x, v[c]);
    }
    if (FORM != kBefore) normalise2(v, a.w_post, a.w_post_f32, a.b_post, a.b_post_f32, s_sum[turn]);
    const unsigned long long s2 = pack_f32x2(scale, scale);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      if (!FAST && !there[c]) continue;
      if (full || channel) {
        Vector8<T> r;
        float g[8];
        load_gate_chunk<T, true>(a, row, 8, e0[c], r);
        unpack_vector<T>(r, a.gate_f32, g);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = mul2(v[c][i], pack_f32x2(g[2 * i], g[2 * i + 1]));
      }
      if (add) {
        unsigned long long r2[4];
        Raw8<R> r;
        load8<R, true>(reinterpret_cast<const R*>(at + r_at) + e0[c], 8, r);
        unpack4x2<R>(r, r2);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = fma2(v[c][i], s2, r2[i]);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[c][i] = mul2(v[c][i], s2);
      }
      if (keep) {
        float h[8];
        split4x2(v[c], h);
        store8<R, true>(reinterpret_cast<R*>(ph) + c * hop, 8, h);
      }
    }
    ph += step_h;
    if (FORM != kAfter) {
      normalise2(v, a.w_pre, a.w_pre_f32, a.b_pre, a.b_pre_f32, s_sum[turn] + kNormSums * 16);
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        float y[8];
        split4x2(v[c], y);
        if (!QUANT) {
          if (FAST || there[c]) store8<T, true>(reinterpret_cast<T*>(py) + c * hop, 8, y);
          continue;
        }
        const float sc = group_scale(max16(amax8(y)));     // (zeros beyond the row)
        if (!FAST && !there[c]) continue;
        store_q8<true>(py + c * hop, 8, e4m3_divided(v[c], divisor_of(sc)));
        if ((lane & 15) == 0) ps[c * (hop >> 7)] = sc;
      }
      py += step_y;
      ps += step_s;
    }
    turn ^= 1;
    now += stage_bytes;
    if (now == stage_end) now = 0;
  }
}

template <typename T, typename R, int FORM, bool QUANT>
cudaError_t launch_stream(const NormArgs& a, int ctas, int stages, int stage_bytes, int num_sms, cudaStream_t stream) {
  const bool fast = a.H == a.team * 16 && !a.w_post_f32 && !a.w_pre_f32;
  auto kernel = a.layer ? (fast ? block_norm_stream_kernel<T, R, FORM, QUANT, true, true> : block_norm_stream_kernel<T, R, FORM, QUANT, true, false>)
                        : (fast ? block_norm_stream_kernel<T, R, FORM, QUANT, false, true> : block_norm_stream_kernel<T, R, FORM, QUANT, false, false>);
  const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
  if (err != cudaSuccess) return err;
  const int grid = static_cast<int>(std::min<long long>(a.M, static_cast<long long>(ctas) * num_sms));
  note_launch("block_norm_stream_kernel");
  return launch_kernel(kernel, dim3(grid), dim3(a.team), stages * stage_bytes, stream, a.pdl != 0, a, stages, stage_bytes);
}

template <typename T, typename R, int CH, int S>
cudaError_t launch_ring(const NormArgs& a, int ctas, int stage_bytes, int kept_bytes, int num_sms, cudaStream_t stream) {
  auto kernel = a.layer ? block_norm_ring_kernel<T, R, CH, S, true> : block_norm_ring_kernel<T, R, CH, S, false>;
  const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingBytes);
  if (err != cudaSuccess) return err;
  const int grid = static_cast<int>(std::min<long long>(a.M, static_cast<long long>(ctas) * num_sms));
  note_launch("block_norm_ring_kernel");
  return launch_kernel(kernel, dim3(grid), dim3(a.team), S * stage_bytes + kept_bytes, stream, a.pdl != 0, a, stage_bytes);
}

template <typename T, typename R, bool VEC>
int launch_rows(NormArgs a, int num_sms, cudaStream_t stream) {
  // Few elements: a CTA to a row and as many threads as it has chunks, for the shortest way from load to store.  More: the rows stream
  // through CTAs with two chunks to a thread, four where the row is longer than 8192.  Few is up to 700 thousand where the streaming
  // kernel needs no tests, else up to three million.  (us, a CTA to a row / as a stream; before a block, quantised: 100 x 4096 2.28 / 2.29,
  // 200 x 4096 2.90 / 2.77, 600 x 4096 5.9 / 4.3, 300 x 7168 6.5 / 4.7, but 300 x 2600 2.9 / 3.5, 1100 x 2600 6.3 / 7.9; after a block
  // 200 x 4096 2.66 / 2.35, both norms 200 x 4096 3.73 / 3.72.)  Rows off 16 bytes do not stream, so each has its CTA (two chunks to a thread: 3000 x 4097
  // after a block 51.5 us, one 31.6).
  const int chunks = (a.H + 7) / 8;
  const bool fast = VEC && a.H % 512 == 0 && !a.w_post_f32 && !a.w_pre_f32;
  const int ch = chunks > 1024 ? 4 : !VEC || static_cast<long long>(a.M) * a.H <= (fast ? 700000 : 3000000) ? 1 : 2;
  a.team = ((chunks + ch - 1) / ch + 31) / 32 * 32;
  cudaError_t err;
  if (VEC && ch > 1 && a.team >= 64) {
    const int stage = a.H * static_cast<int>(sizeof(T) + (a.residual != nullptr ? sizeof(R) : 0));
    auto bytes = [&](const void* p, int f32) { return p == nullptr ? 0 : a.H * (f32 ? 4 : static_cast<int>(sizeof(T))); };
    const int kept = bytes(a.w_post, a.w_post_f32) + bytes(a.b_post, a.b_post_f32) + bytes(a.w_pre, a.w_pre_f32) +
                     bytes(a.b_pre, a.b_pre_f32) + (a.gate_mode == B200MOE_GATE_CHANNEL ? bytes(a.gate, a.gate_f32) : 0);
    // as many CTAs as registers allow (64 a thread; four chunks: 128) and two stages each
    auto deep = [&](int c, int bytes_kept) { return std::min(4, (std::min(kSmBytes / c - 2048, kRingBytes) - bytes_kept) / stage); };
    if (ch == 2) {
      int most = std::min(16, 1024 / a.team);
      while (most > 1 && deep(most, 0) < 2) --most;
      const int stages = deep(most, 0);
      if (stages >= 2) {
        const bool quant = a.y_scale != nullptr;
        if (!a.post) err = quant ? launch_stream<T, R, kBefore, true>(a, most, stages, stage, num_sms, stream)
                                 : launch_stream<T, R, kBefore, false>(a, most, stages, stage, num_sms, stream);
        else if (!a.pre) err = launch_stream<T, R, kAfter, false>(a, most, stages, stage, num_sms, stream);
        else err = quant ? launch_stream<T, R, kBetween, true>(a, most, stages, stage, num_sms, stream)
                         : launch_stream<T, R, kBetween, false>(a, most, stages, stage, num_sms, stream);
        return err == cudaSuccess ? B200MOE_OK : B200MOE_ERR_CUDA;
      }
    }
    const int stages = ch == 4 ? deep(1, kept) : 0;
    if (stages >= 2) {
      err = stages >= 3 ? launch_ring<T, R, 4, 3>(a, 1, stage, kept, num_sms, stream) : launch_ring<T, R, 4, 2>(a, 1, stage, kept, num_sms, stream);
      return err == cudaSuccess ? B200MOE_OK : B200MOE_ERR_CUDA;
    }
  }
  a.rows_per_cta = a.M > 2 * num_sms && a.team < 128 ? 128 / a.team : 1;
  const dim3 grid((a.M + a.rows_per_cta - 1) / a.rows_per_cta), block(a.team * a.rows_per_cta);
  note_launch("block_norm_kernel");
  // Four chunks to a thread (rows of more than 8192 that the ring does not take: off 16 bytes, or fp32 beside their vectors) hold 128 registers and spill
  // 8 to 184 bytes; a row is bound by its way from load to store all the same (2000 x 16384, fp32 residual, after a block 84.7 us).
  // A layer norm before a block needs a few registers more than the RMS norm; with 40 four of its CTAs of 352 threads share an SM, and three with
  // more (1001 x 2600, fp16: 7.3 us and 9.1).  Rows of 16-bit types fit into 40 without spills.
  constexpr bool SLIM = VEC && sizeof(T) == 2 && sizeof(R) == 2;
  const bool slim = SLIM && block.x <= 512;
  auto pick = [&](auto layer) {
    constexpr bool L = decltype(layer)::value;
    return ch == 4   ? block_norm_kernel<T, R, VEC, 4, 512, L, true, true>
           : ch == 2 ? block_norm_kernel<T, R, true, 2, 512, L, true, true>      // (rows of up to 512, too narrow to stream)
           : !a.post ? (L && slim ? block_norm_kernel<T, R, VEC, 1, SLIM && L ? 512 : 1024, L, false, true>
                                  : block_norm_kernel<T, R, VEC, 1, 1024, L, false, true>)
           : !a.pre  ? block_norm_kernel<T, R, VEC, 1, 1024, L, true, false>
                     : block_norm_kernel<T, R, VEC, 1, 1024, L, true, true>;
  };
  auto kernel = a.layer ? pick(std::true_type{}) : pick(std::false_type{});
  err = launch_kernel(kernel, grid, block, 0, stream, a.pdl != 0, a);
  return err == cudaSuccess ? B200MOE_OK : B200MOE_ERR_CUDA;
}

template <typename T, typename R>
int launch_typed(const NormArgs& a, int num_sms, cudaStream_t stream) {
  return a.vec ? launch_rows<T, R, true>(a, num_sms, stream) : launch_rows<T, R, false>(a, num_sms, stream);
}

}  // namespace

int launch_block_norm(const NormArgs& a, int dtype, int residual_f32, int num_sms, cudaStream_t stream) {
  switch (dtype) {
    case B200MOE_DTYPE_BF16:
      return residual_f32 ? launch_typed<__nv_bfloat16, float>(a, num_sms, stream)
                          : launch_typed<__nv_bfloat16, __nv_bfloat16>(a, num_sms, stream);
    case B200MOE_DTYPE_FP16:
      return residual_f32 ? launch_typed<__half, float>(a, num_sms, stream) : launch_typed<__half, __half>(a, num_sms, stream);
    case B200MOE_DTYPE_FP32:
      return launch_typed<float, float>(a, num_sms, stream);
    default:
      return B200MOE_ERR_BAD_ARG;
  }
}

}  // namespace b200moe
