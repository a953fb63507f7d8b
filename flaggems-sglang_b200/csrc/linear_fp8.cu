// Linear layer with block-quantised FP8 weights: out[m][n] = sum_g xs[m][g] ws[n / 128][g] sum_{k in group g} x[m][k] w[n][k] + bias[n].
//
// The scales are fp32 numbers per 128 k, so no MMA can apply them: each 128-wide slice of the reduction is multiplied into a fresh
// partial accumulator in tensor memory (4 x tcgen05.mma.kind::f8f6f4, K = 32), read back, scaled and added to fp32 sums in
// registers by the promotion warps while the next slices are multiplied.
#include <algorithm>
#include <atomic>

#include "block_ops.cuh"
#include "cluster.cuh"
#include "quant.cuh"

namespace b200moe {

namespace {

constexpr int kSlice = 128;                    // k per slice: one swizzled row of e4m3, one scale
constexpr int kWTile = 128 * kSlice;           // 128 weight rows of a slice
constexpr size_t kSmemMost = 227 * 1024 - 1024;

__device__ __forceinline__ void store_out(void* out, int dtype, size_t at, float v) {
  if (dtype == B200MOE_DTYPE_BF16) static_cast<__nv_bfloat16*>(out)[at] = __float2bfloat16_rn(v);
  else if (dtype == B200MOE_DTYPE_FP16) static_cast<__half*>(out)[at] = __float2half_rn(v);
  else static_cast<float*>(out)[at] = v;
}

__device__ __forceinline__ float bias_at(const LinearArgs& a, int n) {
  if (a.bias == nullptr) return 0.f;
  if (a.bias_dtype == B200MOE_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(a.bias)[n]);
  if (a.bias_dtype == B200MOE_DTYPE_FP16) return __half2float(static_cast<const __half*>(a.bias)[n]);
  return static_cast<const float*>(a.bias)[n];
}

// ---------------------------------------------------------------- activations quantised ahead
// Sixteen lanes to a group, eight elements to a lane; kQuantRuns groups of a half warp in flight at once.  Rows along the grid's x, so
// that no index needs a division.  4096 x 7168 in 18.5 us: 88 MB, 4.8 TB/s.  The division by the scale, exact to the bit, is most of its
// arithmetic.
constexpr int kQuantRuns = 4;
template <typename T>
__global__ void __launch_bounds__(256)
linear_quant_kernel(const T* x, long long ldx, uint8_t* q, float* scales, int K, int G) {
  griddep_wait();
  griddep_launch_dependents();
  const int halves = blockDim.x >> 4, g0 = blockIdx.y * halves * kQuantRuns + (threadIdx.x >> 4), l16 = threadIdx.x & 15;
  const long long row = blockIdx.x;
  const T* src = x + row * ldx + l16 * 8;
  Raw8<T> r[kQuantRuns];
#pragma unroll
  for (int u = 0; u < kQuantRuns; ++u) {
    const int e0 = (g0 + u * halves) * kSlice;
    load8<T, true>(src + e0, e0 + l16 * 8 < K ? 8 : 0, r[u]);       // (K is a multiple of 16)
  }
  float v[kQuantRuns][8], m[kQuantRuns];
#pragma unroll
  for (int u = 0; u < kQuantRuns; ++u) {
    unpack8<T>(r[u], v[u]);
    m[u] = amax8(v[u]);
  }
  max16<kQuantRuns>(m);
#pragma unroll
  for (int u = 0; u < kQuantRuns; ++u) {
    const int g = g0 + u * halves, e0 = g * kSlice + l16 * 8;
    const float s = group_scale(m[u]);
    // (the division's own reciprocal: with divisor_of's the compiler takes the groups one after the other, 0.6 us more for 48 rows of 2048)
    store_q8<true>(q + row * K + e0, e0 < K ? 8 : 0, e4m3_divided(v[u], divisor_of(s, __frcp_rn(s))));
    if (l16 == 0 && g < G) scales[row * G + g] = s;
  }
}

// ---------------------------------------------------------------- few rows: weights on the MMA's M side
// A CTA takes 128 weight rows, NT tokens and a share of the reduction; the CTAs of a cluster share a tile's reduction and join
// their sums through distributed shared memory, in rank order.
// Bound by a launch's fixed way, then by memory: one row on 4096 x K takes 4.6 us at K = 896, 5.6 at 1792, 8.6 at 7168 (29.4 MB, 3.4 TB/s;
// 4.5 us at the rate of a copy) and 22.1 at 28672 (117 MB, 5.3 TB/s).  Hence a ring as deep as half an SM's shared memory allows, two
// CTAs to an SM, weights asked for in L2 ahead of the wait for the kernel before, and the reduction split over a cluster.
struct DecodeSmem {
  int stages, slices;       // ring stages; slices of the longest share
  int sums;                 // tokens whose sums a CTA of a cluster receives at most
  uint32_t x_off, t_off, sum_off, bar_off;
  size_t bytes;
};
// TMA producer, MMA issuer and promotion: four warps, or two groups of four that take half of the tokens each
__host__ __device__ constexpr int decode_groups(int nt) { return nt >= 32 ? 2 : 1; }
__host__ __device__ constexpr int decode_threads(int nt) { return 64 + 128 * decode_groups(nt); }
constexpr int kDecodeStages = 14;
constexpr int kOwnGroups = 4;                  // groups that a half warp quantises, where the kernel does that itself
constexpr int kPartCols = 256;                 // tensor memory of a CTA
// slices of a share at most, for the scales' table
constexpr int most_slices(int nt) { return 16384 / nt; }
// fused: the kernel quantises up to eight tokens itself and keeps them, in eight rows a slice, which the MMA's sixteen columns read twice (a
// stride of zero between groups of eight): the upper half of the results is not looked at.
constexpr int kFusedSlice = 8 * kSlice;
DecodeSmem decode_smem(int nt, bool fused, int slices, int split, int tokens, size_t budget) {
  DecodeSmem d;
  const size_t stage = kWTile + (fused ? 0 : nt * kSlice);
  const size_t table = static_cast<size_t>(slices) * nt * 4;
  const size_t resident = fused ? static_cast<size_t>(slices) * kFusedSlice : 0;
  d.sums = (std::min(nt, tokens) + split - 1) / split;
  const size_t sums = split > 1 ? static_cast<size_t>(split) * d.sums * 512 : 0;
  const size_t taken = 1024 + table + resident + sums + 512;
  d.slices = slices;
  d.stages = taken < budget ? static_cast<int>((budget - taken) / stage) : 0;
  if (d.stages > slices) d.stages = slices;
  if (d.stages > kDecodeStages) d.stages = kDecodeStages;
  d.x_off = static_cast<uint32_t>(d.stages * stage);
  d.t_off = static_cast<uint32_t>(d.x_off + resident);
  d.sum_off = static_cast<uint32_t>(d.t_off + table);
  d.bar_off = static_cast<uint32_t>(d.sum_off + sums);
  d.bytes = 1024 + d.bar_off + 512;
  // A cluster's CTAs wait for one another, and a third CTA on an SM would wait for tensor memory: with that much shared memory there is
  // none.
  if (split > 1) d.bytes = std::max<size_t>(d.bytes, 78 * 1024);
  return d;
}

constexpr int decode_tokens(int m) { return m <= 16 ? 16 : m <= 32 ? 32 : 64; }
int decode_seats(int split, bool two, int num_sms);      // clusters of that many CTAs, one or two to an SM, that the GPU holds at once
// As many CTAs to a tile as all tiles' clusters have seats for at once, and one to spare, with four slices or more each.  (us on K = 7168,
// splits of 1 to 8, one row: 32 tiles 16.5 11.6 10.7 10.2 10.4 9.6 8.5 8.7; 48 tiles 17.0 13.2 13.2 12.1 10.9, and with six, seats for 45,
// 16.7; 56 tiles with four 12.5, with five, seats for 56, 14.9.  On K = 2048, 32 tiles with 8, 4, 2 slices to a CTA 6.0 5.5 5.6.)  With
// more than 16 rows a second CTA on the SMs has to save five slices: their sums are more.  (64 rows on K = 2048, 36 tiles: three CTAs to a
// tile, one to an SM, 6.7, four 7.8; on K = 7168 three 12.4, seven 11.2.)  Over 7 to 200 tiles, K of 2048, 4096 and 7168 and 1 to 64 rows
// this is 1 to 2 % behind the best split.
// False: sizes beyond the kernel, or, fused, no room for three stages.
bool plan_decode(const LinearArgs& a, bool fused, int num_sms, int* split_out, DecodeSmem* d) {
  const int nt = decode_tokens(a.M), tiles = (a.N + 127) / 128, mt = (a.M + nt - 1) / nt;
  const long long all = static_cast<long long>(tiles) * mt;
  int split = a.split;
  if (split <= 0) {
    int seated[2];      // with one CTA to an SM, with two
    for (int two = 0; two < 2; ++two) {
      int c = 8;
      while (c > 1 && (a.G / c < 4 || all >= decode_seats(c, two != 0, num_sms))) --c;
      seated[two] = c;
    }
    split = nt > 16 && (a.G + seated[0] - 1) / seated[0] < (a.G + seated[1] - 1) / seated[1] + 5 ? seated[0] : seated[1];
  }
  split = std::max(split, (a.G + most_slices(nt) - 1) / most_slices(nt));
  split = std::min(std::max(std::min(split, a.G), 1), 8);
  const int slices = (a.G + split - 1) / split;
  if (slices > most_slices(nt) || mt > 65535 || all * split > 0x7fffffffll) return false;
  *split_out = split;
  *d = decode_smem(nt, fused, slices, split, a.M, (kSmemMost - 1024) / 2);
  if (d->stages >= std::min(slices, 3)) return true;
  if (fused) return false;
  *d = decode_smem(nt, fused, slices, split, a.M, kSmemMost);
  return d->stages >= 1;
}

__device__ __forceinline__ void tmem_ld_f32(uint32_t taddr, float (&v)[16]) { tmem_ld16_wait(taddr, v); }
__device__ __forceinline__ void tmem_ld_f32(uint32_t taddr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : B200MOE_R32(r, 0)
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

template <int NT, bool FUSED, typename T>
__global__ void __launch_bounds__(decode_threads(NT), 2)
fp8_linear_decode_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const LinearArgs a,
                         const DecodeSmem d, const int split) {
  constexpr int NPB = kPartCols / NT, NG = decode_groups(NT), WARPS = 4 * NG, CT = NT / NG;     // CT: tokens of a promotion thread
  constexpr int X_BYTES = FUSED ? 0 : NT * kSlice;
  constexpr int STAGE = kWTile + X_BYTES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* s_x = smem + d.x_off;                                       // FUSED: [slice][8][128]
  float* s_t = reinterpret_cast<float*>(smem + d.t_off);               // [slice][NT] xs * ws
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(smem + d.bar_off);
  uint64_t* bar_empty = bar_full + kDecodeStages;
  uint64_t* bar_pfull = bar_empty + kDecodeStages;
  uint64_t* bar_pempty = bar_pfull + 16;
  uint64_t* bar_ready = bar_pempty + 16;                               // tables (and FUSED: the tokens) are there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_ready + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const int tile = static_cast<int>(blockIdx.x) / split, rank = static_cast<int>(blockIdx.x) - tile * split;
  const int n0 = tile * 128, m0 = static_cast<int>(blockIdx.y) * NT;
  const int kb0 = a.G * rank / split, kb1 = a.G * (rank + 1) / split;
  const int nsl = kb1 - kb0;

  // The thread that loads sets the barriers up itself and starts the ring at once; tensor memory and tables follow meanwhile.
  const int first = min(nsl, d.stages);
  auto load_slice = [&](int i, int s) {
    const uint32_t full = smem_u32(&bar_full[s]), sw = smem_u32(smem + static_cast<size_t>(s) * STAGE);
    mbar_arrive_expect_tx(full, STAGE);
    tma_load_2d(sw, &tm_w, full, (kb0 + i) * kSlice, n0);
    if (!FUSED) tma_load_2d(sw + kWTile, &tm_x, full, (kb0 + i) * kSlice, m0);
  };
  if (warp == 0) {
    // (a barrier to a lane: one after the other they took 0.4 us)
    for (int i = lane; i < 2 * kDecodeStages + 33; i += 32)
      mbar_init(smem_u32(&bar_full[i]), i < 2 * kDecodeStages + 16 ? 1 : WARPS);
    fence_mbar_init();
    fence_proxy_async_smem();
    __syncwarp();
    if (elect_one()) {
      *abort_flag = 0;
      if (a.pdl) {
        for (int i = 0; i < first; ++i) tma_prefetch_2d(&tm_w, (kb0 + i) * kSlice, n0);
      }
      griddep_wait();
      for (int i = 0; i < first; ++i) load_slice(i, i);
    }
    __syncwarp();
  } else if (warp == 1) {
    tmem_alloc(smem_u32(tmem_slot), kPartCols);
    tmem_relinquish();
  } else if (warp == 2 && elect_one()) {
    prefetch_tmap(&tm_w);
    if (!FUSED) prefetch_tmap(&tm_x);
  }
  // FUSED: sixteen lanes to a (token, slice) group of the CTA's share, at most kOwnGroups to a half warp; they are asked for while the CTA
  // sets up.
  const int live = min(NT, a.M - m0), l16 = lane & 15, half = (warp - 2) * 2 + (lane >> 4);
  Raw8<T> xr[kOwnGroups];
  int xt[kOwnGroups], xi[kOwnGroups];
  if (FUSED && warp >= 2) {
    griddep_wait();
#pragma unroll
    for (int u = 0; u < kOwnGroups; ++u) {
      const int it = half + u * 2 * WARPS;
      xt[u] = it / nsl;
      xi[u] = it - xt[u] * nsl;
      const int k = (kb0 + xi[u]) * kSlice + l16 * 8;
      load8<T, true>(static_cast<const T*>(a.x) + static_cast<long long>(m0 + xt[u]) * a.ldx + k, xt[u] < live && k < a.K ? 8 : 0, xr[u]);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (split > 1) cluster_arrive();        // (waited for before this CTA writes into another)
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  if (warp == 0 && elect_one()) {
    // =============================== TMA producer ===============================
    bool ok = true;
    int i = first, s = 0;
    uint32_t phase = 0;
    for (; i < nsl; ++i) {
      if (!mbar_wait(smem_u32(&bar_empty[s]), phase, abort_flag, DEV_TIMEOUT_PRODUCER)) {
        ok = false;
        break;
      }
      load_slice(i, s);
      if (++s == d.stages) {
        s = 0;
        phase ^= 1;
      }
    }
    if (!ok || *abort_flag != 0)      // copies in flight land before the CTA leaves
      for (int j = i - 1; j >= 0 && j >= i - d.stages; --j) mbar_wait_brief(smem_u32(&bar_full[j % d.stages]), (j / d.stages) & 1);
  } else if (warp == 1 && elect_one()) {
    // =============================== MMA issuer ===============================
    const uint32_t idesc = make_idesc(0, 128, NT);
    if (!FUSED || mbar_wait(smem_u32(bar_ready), 0, abort_flag, DEV_TIMEOUT_MMA)) {
      // (stage and phase are counted: two divisions by the number of stages per slice set this thread's pace)
      int s = 0;
      uint32_t phase = 0, sw = smem_u32(smem), sx = smem_u32(s_x);
      for (int i = 0; i < nsl; ++i) {
        const int p = i % NPB;
        if (!mbar_wait(smem_u32(&bar_pempty[p]), ((i / NPB) & 1) ^ 1, abort_flag, DEV_TIMEOUT_MMA)) break;
        if (!mbar_wait(smem_u32(&bar_full[s]), phase, abort_flag, DEV_TIMEOUT_MMA)) break;
        tc_fence_after();
        const uint64_t dw = smem_desc_k_sw128(sw);
        const uint64_t dx = FUSED ? smem_desc_k_sw128(sx) & ~(0x3fffull << 32) : smem_desc_k_sw128(sw + kWTile);
#pragma unroll
        for (int k = 0; k < 4; ++k) tc_mma_f8(tmem_base + p * NT, dw + 2 * k, dx + 2 * k, idesc, k > 0);
        tc_commit(smem_u32(&bar_empty[s]));
        tc_commit(smem_u32(&bar_pfull[p]));
        sw += STAGE;
        sx += kFusedSlice;
        if (++s == d.stages) {
          s = 0;
          phase ^= 1;
          sw = smem_u32(smem);
        }
      }
    }
  }
  __syncwarp();
  float acc[CT];
#pragma unroll
  for (int t = 0; t < CT; ++t) acc[t] = 0.f;
  const int quad = warp & 3, row = quad * 32 + lane, first_t = ((warp - 2) >> 2) * CT;      // first token of the thread
  if (warp >= 2) {
    // =============================== promotion ===============================
    const float* ws = a.w_scale + static_cast<size_t>(tile) * a.G + kb0;
    if (FUSED) {
      float v[kOwnGroups][8], m[kOwnGroups];
#pragma unroll
      for (int u = 0; u < kOwnGroups; ++u) {
        unpack8<T>(xr[u], v[u]);
        m[u] = amax8(v[u]);
      }
      max16<kOwnGroups>(m);
#pragma unroll
      for (int u = 0; u < kOwnGroups; ++u) {
        const float s = group_scale(m[u]);
        const uint2 q = e4m3_divided(v[u], divisor_of(s));
        if (xt[u] < live) {
          *reinterpret_cast<uint2*>(s_x + xi[u] * kFusedSlice + xt[u] * kSlice + (((l16 >> 1) ^ xt[u]) << 4) + (l16 & 1) * 8) = q;
          if (l16 == 0) s_t[xi[u] * NT + xt[u]] = s * ws[xi[u]];
        }
      }
      fence_proxy_async_smem();
    } else {
      for (int it = threadIdx.x - 64; it < live * nsl; it += 32 * WARPS) {
        const int t = it / nsl, i = it - t * nsl;
        s_t[i * NT + t] = a.x_scale[static_cast<long long>(m0 + t) * a.G + kb0 + i] * ws[i];
      }
    }
    __syncwarp();
    if (lane == 0) mbar_arrive(smem_u32(bar_ready));
    bool ok = mbar_wait(smem_u32(bar_ready), 0, abort_flag, DEV_TIMEOUT_EPILOGUE);
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + first_t;
    for (int i = 0; ok && i < nsl; ++i) {
      const int p = i % NPB;
      if (!(ok = mbar_wait(smem_u32(&bar_pfull[p]), (i / NPB) & 1, abort_flag, DEV_TIMEOUT_EPILOGUE))) break;
      tc_fence_after();
      const float4* sc = reinterpret_cast<const float4*>(s_t + i * NT + first_t);
      constexpr int LD = CT < 32 ? CT : 32;
#pragma unroll
      for (int c = 0; c < CT; c += LD) {
        float v[LD];
        tmem_ld_f32(taddr + p * NT + c, v);
#pragma unroll
        for (int j = 0; j < LD / 4; ++j) {
          const float4 f = sc[c / 4 + j];
          acc[c + 4 * j] = fmaf(v[4 * j], f.x, acc[c + 4 * j]);
          acc[c + 4 * j + 1] = fmaf(v[4 * j + 1], f.y, acc[c + 4 * j + 1]);
          acc[c + 4 * j + 2] = fmaf(v[4 * j + 2], f.z, acc[c + 4 * j + 2]);
          acc[c + 4 * j + 3] = fmaf(v[4 * j + 3], f.w, acc[c + 4 * j + 3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_pempty[p]));
    }
  }
  // ---- each CTA of the cluster owns every split-th token: the others write their sums of it into its shared memory, it adds them in rank
  // order.  One barrier, after which no CTA touches another's memory.  (Read from the others after a barrier, with a second one
  // before leaving: 1.3 us more.)
  const int n = n0 + row;
  if (split > 1) {
    const int mine = d.sums;
    float* s_sum = reinterpret_cast<float*>(smem + d.sum_off);      // [rank][token][128]
    cluster_wait();
    if (warp >= 2) {
      uint32_t to = smem_u32(s_sum + (rank * mine + first_t / split) * 128 + row);
      int owner = first_t % split;
#pragma unroll
      for (int t = 0; t < CT; ++t) {
        if (first_t + t < live) st_cluster_f32(mapa_u32(to, owner), acc[t]);
        if (++owner == split) {
          owner = 0;
          to += 512;
        }
      }
    }
    cluster_arrive();
    cluster_wait();
    if (warp >= 2 && n < a.N) {
      const float b = bias_at(a, n);
      // (own tokens to the promotion groups in turn)
      const int grp = (warp - 2) >> 2;
      const float* from = s_sum + grp * 128 + row;
#pragma unroll 2
      for (int t = rank + grp * split; t < live; t += NG * split, from += NG * 128) {
        float part[8], v = 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) part[q] = q < split ? from[q * mine * 128] : 0.f;
#pragma unroll
        for (int q = 0; q < 8; ++q) v += part[q];
        store_out(a.out, a.out_dtype, static_cast<size_t>(m0 + t) * a.N + n, v + b);
      }
    }
  } else if (warp >= 2 && n < a.N) {
    const float b = bias_at(a, n);
#pragma unroll
    for (int t = 0; t < CT; ++t)
      if (first_t + t < live) store_out(a.out, a.out_dtype, static_cast<size_t>(m0 + first_t + t) * a.N + n, acc[t] + b);
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kPartCols);
  }
  if (threadIdx.x == 0 && *abort_flag != 0) atomicCAS(a.status, 0, *abort_flag);
}

// Clusters of `size` CTAs that the GPU holds at once, which is less than its SMs would have room for: a cluster lies within one group of SMs,
// and the groups' sizes are no multiples of it (two CTAs to an SM, sizes 2 to 8: 148 93 71 56 45 37 33).  Asked for once per device and size, for
// a kernel without tensor memory: of those with it the runtime counts one CTA to an SM, where two run.
__global__ void seats_kernel() {}
enum SeatKind { kHalfSeats, kWholeSeats };      // of an SM
int cluster_seats(SeatKind kind, int size, int threads, size_t smem, int room) {
  constexpr int kDevices = 64;
  static std::atomic<int> known[2][kDevices][9];
  int device = 0, seats = 0;
  if (cudaGetDevice(&device) == cudaSuccess && device < kDevices) {
    if ((seats = known[kind][device][size].load(std::memory_order_relaxed)) > 0) return seats;
    cudaLaunchAttribute shape;
    shape.id = cudaLaunchAttributeClusterDimension;
    shape.val.clusterDim.x = size;
    shape.val.clusterDim.y = shape.val.clusterDim.z = 1;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(size);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.attrs = &shape;
    config.numAttrs = 1;
    if (cudaFuncSetAttribute(seats_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMost)) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&seats, seats_kernel, &config) == cudaSuccess && seats > 0) {
      known[kind][device][size].store(seats, std::memory_order_relaxed);
      return seats;
    }
  }
  (void)cudaGetLastError();
  return std::max(1, room / size * 7 / 8);
}
// (by shared memory, half an SM's or all of it: every kernel of the family has the same seats)
int decode_seats(int split, bool two, int num_sms) {
  return two ? cluster_seats(kHalfSeats, split, decode_threads(64), (kSmemMost - 1024) / 2, 2 * num_sms)
             : cluster_seats(kWholeSeats, split, decode_threads(64), kSmemMost, num_sms);
}

template <int NT, bool FUSED, typename T>
int launch_decode(const LinearArgs& a, const DecodeSmem& d, int split, const CUtensorMap& tm_w, const CUtensorMap& tm_x, cudaStream_t stream) {
  auto kernel = fp8_linear_decode_kernel<NT, FUSED, T>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMost)) != cudaSuccess)
    return B200MOE_ERR_CUDA;
  note_launch("fp8_linear_decode_kernel");
  cudaError_t err = launch_kernel_cluster(kernel, dim3((a.N + 127) / 128 * split, (a.M + NT - 1) / NT), split, dim3(decode_threads(NT)),
                                          d.bytes, stream, a.pdl != 0, tm_w, tm_x, a, d, split);
  return err == cudaSuccess ? B200MOE_OK : B200MOE_ERR_CUDA;
}
// ---------------------------------------------------------------- many rows: tokens on the MMA's M side
// A CTA takes 128 tokens, a pair of CTAs (PAIR: tcgen05.mma.cta_group::2, issued by the leader for both) 256, by TN weight rows.  An
// accumulator lane is a token, so a slice's scale is one number per thread, and promotion is one fma per element.  Two promotion
// groups of four warps take TN / 2 columns each.
// `split` CTAs or pairs of a cluster share a tile's reduction; each of them owns a part of the tile's columns, gets the others' sums of
// it written into its shared memory and adds them in rank order.
// A pair's 256 x 256 tile takes 900 cycles a slice (4096 x 4096 x 7168, 115 us, 2090 TFLOP/s; 8192 x 18432 x 7168, 1.09 ms, 1990).  Its
// MMAs are 512 of them, its operands, 32 KB a CTA, take 620 from L2, and the way of a promotion warp through a slice 870: two loads of
// 64 columns with 330 cycles of latency each, and 32 packed fmas behind each, for which the 128 sums leave no registers to load
// ahead (loads of 32 columns, one ahead, have nearly the same latency: 1040 cycles; sixteen promotion warps with half of the sums
// each: 141 us where this took 121).  In long trains the power limit sets the clock, to 1.5 GHz there: without any promotion the same
// MMAs run at 1.35 GHz and take 860 us.
// A single CTA's 128 x 128 tile moves 32 KB into shared memory and 32 KB out of it per slice, 512 cycles at 128 bytes a cycle, for 256
// cycles of MMA; so it is for results of few tiles.
// Tiles that fill less than half of the last wave are not cut in two for it: 115.6 us for 115.3, and 1114 for 1089, since a wave with idle
// SMs runs faster as it is.
constexpr int kTokenThreads = 384;             // TMA producer, MMA issuer, two warps for the scales, promotion
constexpr int kTokenRing = 6;                  // operand stages at most; four or five where a split needs the room

template <int TN, bool PAIR>
constexpr int kTokenStage = kWTile + (PAIR ? TN / 2 : TN) * kSlice;     // per CTA: 128 tokens, its weight rows
template <int TN>
constexpr int kScaleSlots = 512 / TN + 2;               // two more than partial accumulators

// Columns of a lane, loaded and waited for in one statement: no use of the registers can move ahead of the wait.
__device__ __forceinline__ void tmem_ld_wait(uint32_t taddr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
      "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
      "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : B200MOE_R32(r, 0), B200MOE_R32(r, 32)
      : "r"(taddr)
      : "memory");
}
// c += r * s2, two columns to an instruction
template <int N>
__device__ __forceinline__ void fma_columns(unsigned long long* c, const uint32_t (&r)[N], unsigned long long s2) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) ffma2_packed(c[i], r[2 * i], r[2 * i + 1], s2);
}

// Tiles in bands of kBand token tiles, so that a band's tokens and the weights that sweep past them meet in L2.
constexpr int kBand = 16;
__device__ __forceinline__ void token_tile_at(int id, int mt, int nt, int& m, int& n) {
  const int band = id / (kBand * nt), first = band * kBand, rows = min(kBand, mt - first), in = id - band * kBand * nt;
  n = in / rows;
  m = first + in - n * rows;
}

// A warp's 32 rows (lane: row0 + lane, `live`: inside the result) of 32 columns from n on, `left` of which are inside.  Whole sectors straight
// from the registers where every row starts on 32 bytes; else turned in shared memory (`turn`, this warp's), so that the lanes of a
// store lie side by side: from lanes that each write two bytes of a row of their own a
// store touches 32 sectors.
constexpr int kTurnBytes = 32 * 34 * 2;        // 16-bit: 34 to a row; fp32: 17, half of the columns at a time
__device__ __forceinline__ void store_rows32(const LinearArgs& a, uint8_t* turn, int row0, bool live, int n, int left, const float (&v)[32]) {
  const int eb = a.out_dtype == B200MOE_DTYPE_FP32 ? 4 : 2, lane = threadIdx.x & 31;
  uint8_t* p = static_cast<uint8_t*>(a.out) + (static_cast<size_t>(row0 + lane) * a.N + n) * eb;
  if (left >= 32 && (static_cast<size_t>(a.N) * eb & 31) == 0 && (reinterpret_cast<uintptr_t>(a.out) & 31) == 0) {
    if (!live) return;
    if (eb == 4) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(v) + 8 * q;
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + 32 * q), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
      }
    } else {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        uint32_t w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float lo = v[16 * q + 2 * i], hi = v[16 * q + 2 * i + 1];
          if (a.out_dtype == B200MOE_DTYPE_BF16) {
            const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
            w[i] = *reinterpret_cast<const uint32_t*>(&b);
          } else {
            const __half2 h = __floats2half2_rn(lo, hi);
            w[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
        }
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p + 32 * q), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                     "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                     : "memory");
      }
    }
    return;
  }
  const unsigned rows = __ballot_sync(0xffffffffu, live);
  if (eb == 2) {
    uint32_t* words = reinterpret_cast<uint32_t*>(turn);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
      words[lane * 17 + i] = a.out_dtype == B200MOE_DTYPE_BF16 ? *reinterpret_cast<const uint32_t*>(&b) : *reinterpret_cast<const uint32_t*>(&h);
    }
    __syncwarp();
    const uint16_t* from = reinterpret_cast<const uint16_t*>(turn) + lane;
    uint16_t* to = static_cast<uint16_t*>(a.out) + static_cast<size_t>(row0) * a.N + n + lane;
#pragma unroll 8
    for (int r = 0; r < 32; ++r, to += a.N)
      if (lane < left && (rows >> r & 1)) *to = from[r * 34];
    __syncwarp();
  } else {
    float* words = reinterpret_cast<float*>(turn);
    const int col = lane & 15, up = lane >> 4;
#pragma unroll
    for (int c = 0; c < 32; c += 16) {
#pragma unroll
      for (int i = 0; i < 16; ++i) words[lane * 17 + i] = v[c + i];
      __syncwarp();
      float* to = static_cast<float*>(a.out) + static_cast<size_t>(row0 + up) * a.N + n + c + col;
#pragma unroll 8
      for (int r = 0; r < 32; r += 2, to += 2 * static_cast<size_t>(a.N))
        if (c + col < left && (rows >> (r + up) & 1)) *to = words[(r + up) * 17 + col];
      __syncwarp();
    }
  }
}

// The same with the bias, and nothing where the columns lie outside.  Whole warp.
__device__ __forceinline__ void store_columns(const LinearArgs& a, uint8_t* turn, int row0, bool live, int n, float (&v)[32]) {
  const int left = a.N - n;
  if (left <= 0) return;
  if (a.bias != nullptr) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] += i < left ? bias_at(a, n + i) : 0.f;
  }
  store_rows32(a, turn, row0, live, n, left, v);
}

template <int TN, bool PAIR>
__global__ void __launch_bounds__(kTokenThreads, 1)
fp8_linear_token_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_x, const LinearArgs a,
                        const int split, const int stages) {
  constexpr int NBUF = 512 / TN, CW = TN / 2, BLOCKS = TN / 128, SLOTS = kScaleSlots<TN>;
  constexpr int CTAS = PAIR ? 2 : 1, ROWS = 128 * CTAS;
  constexpr int STAGE = kTokenStage<TN, PAIR>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  float* s_sum = reinterpret_cast<float*>(smem + stages * STAGE);             // [other share][own columns][128 tokens]
  float* s_scale = s_sum + (split - 1) * (TN / split) * 128;                   // [slot][weight block][128 tokens]
  uint8_t* s_turn = reinterpret_cast<uint8_t*>(s_scale + SLOTS * BLOCKS * 128);      // [promotion warp]
  uint64_t* bar_full = reinterpret_cast<uint64_t*>(s_turn + 8 * kTurnBytes);
  uint64_t* bar_empty = bar_full + kTokenRing;
  uint64_t* bar_pfull = bar_empty + kTokenRing;
  uint64_t* bar_pempty = bar_pfull + NBUF;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bar_pempty + NBUF);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_index();
  const int lane = threadIdx.x & 31;
  const bool clustered = PAIR || split > 1;
  const uint32_t crank = clustered ? cluster_ctarank() : 0;
  const uint32_t rank = PAIR ? crank & 1 : 0, lead = crank - rank;     // in the pair; the leader's rank in the cluster
  const int share = static_cast<int>(crank) / CTAS;                    // of the reduction
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);      // the leader announces the bytes of both CTAs
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int s = 0; s < NBUF; ++s) {
      mbar_init(smem_u32(&bar_pfull[s]), 3);             // the MMAs are done, and both scale warps
      mbar_init(smem_u32(&bar_pempty[s]), 8 * CTAS);     // leader: the promotion warps of both CTAs
    }
    *abort_flag = 0;
    fence_mbar_init();
    fence_proxy_async_smem();
    prefetch_tmap(&tm_w);
    prefetch_tmap(&tm_x);
  }
  __syncwarp();
  if (clustered) {
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    if (PAIR) {
      tmem_alloc2(smem_u32(tmem_slot), 512u);
      tmem_relinquish2();
    } else {
      tmem_alloc(smem_u32(tmem_slot), 512u);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();
  griddep_launch_dependents();

  const int mt = (a.M + ROWS - 1) / ROWS, nt = (a.N + TN - 1) / TN, total = mt * nt;
  const int worker = static_cast<int>(blockIdx.x) / (CTAS * split), workers = static_cast<int>(gridDim.x) / (CTAS * split);
  const int kb0 = static_cast<int>(static_cast<long long>(a.G) * share / split);
  const int kb1 = static_cast<int>(static_cast<long long>(a.G) * (share + 1) / split);

  // registers after the split: 4 x 32 x 56 + 8 x 32 x 224 = 64512 = 384 x 168 at launch
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == 0 && elect_one()) {
      // =============================== TMA producer (every CTA, its own operands) ===============================
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      for (int id = worker; ok && id < total; id += workers) {
        int m, n;
        token_tile_at(id, mt, nt, m, n);
        const int xrow = m * ROWS + static_cast<int>(rank) * 128;
        const int wrow = n * TN + static_cast<int>(rank) * (TN / 2);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(smem_u32(&bar_empty[stage]), phase ^ 1, abort_flag, DEV_TIMEOUT_PRODUCER)) {
            ok = false;
            break;
          }
          const uint32_t s = smem_u32(smem + static_cast<size_t>(stage) * STAGE);
          if (PAIR) {
            const uint32_t full = mapa_u32(smem_u32(&bar_full[stage]), lead);
            if (leader) mbar_arrive_expect_tx(smem_u32(&bar_full[stage]), 2 * STAGE);
            tma_load_2d_pair(s, &tm_x, full, kb * kSlice, xrow);
            tma_load_2d_pair(s + kWTile, &tm_w, full, kb * kSlice, wrow);
          } else {
            const uint32_t full = smem_u32(&bar_full[stage]);
            mbar_arrive_expect_tx(full, STAGE);
            tma_load_2d(s, &tm_x, full, kb * kSlice, xrow);
            tma_load_2d(s + kWTile, &tm_w, full, kb * kSlice, wrow);
          }
          ++issued;
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
        // copies in flight land before the CTA leaves: the leader sees them on its barriers, the other CTA waits a while
        if (leader) {
          const int n = static_cast<int>(issued < stages ? issued : stages);
          for (int i = 1; i <= n; ++i) {
            const int s2 = stage - i < 0 ? stage - i + stages : stage - i;
            mbar_wait_brief(smem_u32(&bar_full[s2]), stage - i < 0 ? phase ^ 1 : phase);
          }
        } else {
          const unsigned long long t0 = globaltimer_ns();
          while (globaltimer_ns() - t0 < 20000ull) {
          }
        }
      }
    } else if (warp == 1 && leader && elect_one()) {
      // =============================== MMA issuer ===============================
      const uint32_t idesc = make_idesc(0, ROWS, TN);
      const uint16_t mask = static_cast<uint16_t>(3u << lead);
      int stage = 0, buf = 0;
      uint32_t phase = 0, bphase = 0;
      bool ok = true;
      for (int id = worker; ok && id < total; id += workers) {
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!(ok = mbar_wait(smem_u32(&bar_full[stage]), phase, abort_flag, DEV_TIMEOUT_MMA))) break;
          if (!(ok = mbar_wait(smem_u32(&bar_pempty[buf]), bphase ^ 1, abort_flag, DEV_TIMEOUT_MMA))) break;
          tc_fence_after();
          const uint32_t s = smem_u32(smem + static_cast<size_t>(stage) * STAGE);
          const uint64_t dx = smem_desc_k_sw128(s), dw = smem_desc_k_sw128(s + kWTile);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (PAIR) tc_mma2_f8(tmem_base + buf * TN, dx + 2 * k, dw + 2 * k, idesc, k > 0);
            else tc_mma_f8(tmem_base + buf * TN, dx + 2 * k, dw + 2 * k, idesc, k > 0);
          }
          if (PAIR) {
            tc_commit2(smem_u32(&bar_empty[stage]), mask);
            tc_commit2(smem_u32(&bar_pfull[buf]), mask);
          } else {
            tc_commit(smem_u32(&bar_empty[stage]));
            tc_commit(smem_u32(&bar_pfull[buf]));
          }
          if (++buf == NBUF) {
            buf = 0;
            bphase ^= 1;
          }
          if (++stage == stages) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
    } else if (warp >= 2) {
      // =============================== scales: x_scale * w_scale of each slice, a slot ahead ===============================
      // Slice k - 2 is multiplied: its buffer was then given back by every reader of slice k - 2 - NBUF, whose slot is the one that
      // slice k takes.
      const int t0 = threadIdx.x - 64;        // tokens t0 and t0 + 64
      long long k = 0;
      bool ok = true;
      for (int id = worker; ok && id < total; id += workers) {
        int m, n;
        token_tile_at(id, mt, nt, m, n);
        const int row0 = m * ROWS + static_cast<int>(rank) * 128 + t0;
        const bool l0 = row0 < a.M, l1 = row0 + 64 < a.M;
        const float* x0 = a.x_scale + (l0 ? static_cast<size_t>(row0) * a.G : 0);
        const float* x1 = a.x_scale + (l1 ? static_cast<size_t>(row0 + 64) * a.G : 0);
        const float* ws[BLOCKS];
        bool lw[BLOCKS];
#pragma unroll
        for (int b = 0; b < BLOCKS; ++b) {
          lw[b] = (n * BLOCKS + b) * 128 < a.N;
          ws[b] = a.w_scale + (lw[b] ? static_cast<size_t>(n * BLOCKS + b) * a.G : 0);
        }
        for (int kb = kb0; kb < kb1; ++kb, ++k) {
          // (no read-only loads: the kernel before may still write the scales when this one starts)
          const float v0 = l0 ? x0[kb] : 0.f, v1 = l1 ? x1[kb] : 0.f;
          float w[BLOCKS];
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) w[b] = lw[b] ? ws[b][kb] : 0.f;
          if (k >= 2) {
            const long long p = k - 2;
            if (!(ok = mbar_wait(smem_u32(&bar_pfull[p % NBUF]), static_cast<uint32_t>(p / NBUF) & 1, abort_flag, DEV_TIMEOUT_EPILOGUE))) break;
          }
          float* slot = s_scale + (k % SLOTS) * (BLOCKS * 128) + t0;
#pragma unroll
          for (int b = 0; b < BLOCKS; ++b) {
            slot[b * 128] = v0 * w[b];
            slot[b * 128 + 64] = v1 * w[b];
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_pfull[k % NBUF]));
        }
      }
    }
    __syncwarp();
    if (split > 1) {        // (where the promotion warps join their sums)
      cluster_arrive();
      cluster_wait();
    }
  } else {
    // =============================== promotion ===============================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
    const int grp = (warp - 4) >> 2, quad = warp & 3;
    const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quad * 32) << 16) + grp * CW;
    const float* my_scale = s_scale + (grp * CW >> 7) * 128 + quad * 32 + lane;
    int buf = 0, slot = 0;
    uint32_t bphase = 0;
    bool done = true;
    for (int id = worker; done && id < total; id += workers) {
      unsigned long long acc[CW / 2];
#pragma unroll
      for (int i = 0; i < CW / 2; ++i) acc[i] = 0;
#pragma unroll 1
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!(done = mbar_wait(smem_u32(&bar_pfull[buf]), bphase, abort_flag, DEV_TIMEOUT_EPILOGUE))) break;
        tc_fence_after();
        const float sc = my_scale[slot * (BLOCKS * 128)];
        const uint32_t t = taddr + buf * TN;
        const unsigned long long s2 = pack_f32x2(sc, sc);
#pragma unroll
        for (int c = 0; c < CW; c += 64) {
          uint32_t r[64];
          tmem_ld_wait(t + c, r);
          if (c + 64 == CW) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if (PAIR) mbar_arrive_remote_read(mapa_u32(smem_u32(&bar_pempty[buf]), lead));
              else mbar_arrive(smem_u32(&bar_pempty[buf]));
            }
          }
          fma_columns<64>(acc + c / 2, r, s2);
        }
        if (++slot == SLOTS) slot = 0;
        if (++buf == NBUF) {
          buf = 0;
          bphase ^= 1;
        }
      }
      int m, n;
      token_tile_at(id, mt, nt, m, n);
      const int row = quad * 32 + lane, row0 = m * ROWS + static_cast<int>(rank) * 128 + quad * 32;
      const bool live = row0 + lane < a.M;
      uint8_t* turn = s_turn + (warp - 4) * kTurnBytes;
      const int n0 = n * TN + grp * CW;
      if (split == 1) {
        if (!done) continue;
#pragma unroll
        for (int c = 0; c < CW; c += 32) {
          float v[32];
#pragma unroll
          for (int i = 0; i < 16; ++i) unpack_f32x2(acc[c / 2 + i], v[2 * i], v[2 * i + 1]);
          store_columns(a, turn, row0, live, n0 + c, v);
        }
        continue;
      }
      // The shares' sums meet (a cluster of several shares has one tile): each is written into the shared memory of the columns' owner.
      const int own = TN / split;
#pragma unroll
      for (int c = 0; c < CW; c += 32) {
        const int at = grp * CW + c, owner = at / own;
        if (owner == share) continue;
        const uint32_t to = mapa_u32(smem_u32(s_sum + ((share < owner ? share : share - 1) * own + at - owner * own) * 128 + row), owner * CTAS + rank);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float lo, hi;
          unpack_f32x2(acc[c / 2 + i], lo, hi);
          st_cluster_f32(to + i * 1024, lo);
          st_cluster_f32(to + i * 1024 + 512, hi);
        }
      }
      __syncwarp();
      cluster_arrive();
      cluster_wait();
#pragma unroll
      for (int c = 0; c < CW; c += 32) {
        const int at = grp * CW + c;
        if (!done || at / own != share) continue;
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0.f;
#pragma unroll 1
        for (int q = 0; q < split; ++q) {
          if (q == share) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float lo, hi;
              unpack_f32x2(acc[c / 2 + i], lo, hi);
              v[2 * i] += lo;
              v[2 * i + 1] += hi;
            }
          } else {
            const float* from = s_sum + ((q < share ? q : q - 1) * own + at - share * own) * 128 + row;
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] += from[i * 128];
          }
        }
        store_columns(a, turn, row0, live, n0 + c, v);
      }
    }
  }
  // ---- no CTA of a pair leaves while the other can still signal its barriers or read its shared memory.  (Without pairs the shares
  // have met for the last time.)
  tc_fence_before();
  __syncthreads();
  if (PAIR) {
    cluster_arrive();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after();
    if (PAIR) tmem_dealloc2(tmem_base, 512u);
    else tmem_dealloc(tmem_base, 512u);
  }
  if (threadIdx.x == 0 && *abort_flag != 0) atomicCAS(a.status, 0, *abort_flag);
}

template <int TN, bool PAIR>
int launch_tokens(const LinearArgs& a, int split, int num_sms, cudaStream_t stream) {
  constexpr int CTAS = PAIR ? 2 : 1;
  auto kernel = fp8_linear_token_kernel<TN, PAIR>;
  CUtensorMap tm_w, tm_x;
  int rc = make_tmap_bytes(&tm_w, a.w, a.K, a.N, a.ldw, TN / CTAS);
  if (rc == B200MOE_OK) rc = make_tmap_bytes(&tm_x, a.x, a.K, a.M, a.ldx, 128);
  if (rc != B200MOE_OK) return rc;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kSmemMost)) != cudaSuccess)
    return B200MOE_ERR_CUDA;
  const long long tiles = static_cast<long long>((a.M + 128 * CTAS - 1) / (128 * CTAS)) * ((a.N + TN - 1) / TN);
  if (tiles > 0x7ffffff) return B200MOE_ERR_TOO_LARGE;
  split = split >= 4 ? 4 : split >= 2 ? 2 : 1;
  while (split > a.G) split >>= 1;
  const int fixed = 1024 + (split - 1) * (TN / split) * 512 + kScaleSlots<TN> * TN * 4 + 8 * kTurnBytes + 512;
  const int stages = std::min(kTokenRing, (static_cast<int>(kSmemMost) - fixed) / kTokenStage<TN, PAIR>);
  const int smem = fixed + stages * kTokenStage<TN, PAIR>;
  const int workers = split > 1 ? static_cast<int>(tiles) : static_cast<int>(std::min<long long>(tiles, num_sms / CTAS));
  note_launch("fp8_linear_token_kernel");
  cudaError_t err = launch_kernel_cluster(kernel, dim3(CTAS * split * workers), CTAS * split, dim3(kTokenThreads), smem, stream, a.pdl != 0,
                                          tm_w, tm_x, a, split, stages);
  return err == cudaSuccess ? B200MOE_OK : B200MOE_ERR_CUDA;
}

template <typename T>
int launch_quant(const LinearArgs& a, cudaStream_t stream) {
  // (a row of up to 64 groups is one CTA's)
  const int threads = std::min(256, ((a.G + kQuantRuns - 1) / kQuantRuns * 16 + 31) / 32 * 32), per_cta = threads / 16 * kQuantRuns;
  note_launch("linear_quant_kernel");
  cudaError_t err = launch_kernel(linear_quant_kernel<T>, dim3(a.M, (a.G + per_cta - 1) / per_cta), dim3(threads), 0, stream, a.pdl != 0,
                                  static_cast<const T*>(a.x), a.ldx, a.ws_q, a.ws_scale, a.K, a.G);
  return err == cudaSuccess ? B200MOE_OK : B200MOE_ERR_CUDA;
}

struct Plan {
  int tile, split;
};
// Up to 64 rows: weights on the MMA's M side, mostly.  Beyond, the tile and split of the shortest estimate: waves of clusters times a cluster's
// slices and its fixed part (start, drain; with a split the meeting of the sums), in cycles measured per slice.  (us of PAIR_256 / PAIR_128 /
// TOKENS with a split of 1, 2, 4, on K = 7168: 100 x 4096 28 / 20 / 19.8, 13.6, 11.1; 333 x 2112 29 / 20.5 / 20.6, 14.5, 20.8; 600 x 4096
// 30 / 40 / 41, 45; 4096 x 4096 114 / 133 / 141.)
Plan pick_plan(const LinearArgs& a, int num_sms) {
  if (a.tile != 0) return {a.tile, a.split};
  if (a.M <= 64) {
    // (more than 32 rows and tiles for most SMs: 64 rows on 18432 x 7168 take 25.3 us with the tokens on M and 28.8 with the weights there,
    // on 12288 x 7168 21.8 and 23.5; on 10240 x 7168 21.5 and 17.9)
    const int tiles = (a.N + 127) / 128;
    if (a.M > 32 && a.split == 0 && tiles > 3 * num_sms / 5 && tiles <= num_sms) return {B200MOE_LINEAR_TILE_TOKENS, 1};
    return {B200MOE_LINEAR_TILE_WEIGHTS, a.split};
  }
  // Results so small that clusters of eight, with four slices or more to a CTA, hold little more than the SMs: only the weights' kernel
  // splits that far.  (us, weights / tokens on M: 128 x 1024 x 7168 8.0 / 9.8, 256 x 576 8.1 / 9.5; 500 x 512 10.1 / 9.9.)
  if (a.split == 0 && a.G >= 32 && static_cast<long long>((a.M + 63) / 64) * ((a.N + 127) / 128) * 6 <= num_sms)
    return {B200MOE_LINEAR_TILE_WEIGHTS, 0};
  struct Kind {
    int tile, rows, columns, ctas, slice, splits;
  };
  const Kind kinds[3] = {{B200MOE_LINEAR_TILE_PAIR_256, 256, 256, 2, 850, 2},
                         {B200MOE_LINEAR_TILE_PAIR_128, 256, 128, 2, 560, 2},
                         {B200MOE_LINEAR_TILE_TOKENS, 128, 128, 1, 540, 4}};
  Plan best = {0, 1};
  double least = 0;
  for (const Kind& k : kinds) {
    const long long tiles = static_cast<long long>((a.M + k.rows - 1) / k.rows) * ((a.N + k.columns - 1) / k.columns);
    for (int s = 1; s <= k.splits && s <= a.G; s *= 2) {
      if (a.split > 0 && s != a.split) continue;
      const int size = k.ctas * s;
      const long long seats = size <= 2 ? num_sms / size
                                        : cluster_seats(kWholeSeats, size, kTokenThreads, kSmemMost, num_sms);
      const long long waves = (tiles + seats - 1) / seats;
      const double t = static_cast<double>(waves) * ((a.G + s - 1) / s * k.slice + 3000 + (s > 1 ? 5000 : 0));
      if (best.tile == 0 || t < least) {
        best = {k.tile, s};
        least = t;
      }
    }
  }
  return best.tile != 0 ? best : Plan{B200MOE_LINEAR_TILE_TOKENS, a.split};
}

// 16-bit rows that the decode kernel quantises itself: every CTA its share of the slices, one batch of loads.  (With three batches, 12 rows
// on 4096 x 7168, it took 11.3 us where a launch for the quantisation took 10.1; with one, 4 rows, 9.5 and 9.6, and the launch less.)
bool quantised_within(const LinearArgs& a, int num_sms, int* split, DecodeSmem* d) {
  return a.x_dtype >= 0 && a.M <= 8 && a.tile == 0 && plan_decode(a, true, num_sms, split, d) && a.M * d->slices <= 8 * kOwnGroups;
}

}  // namespace

size_t linear_workspace_bytes(const LinearArgs& a, int num_sms) {
  int split;
  DecodeSmem d;
  if (a.x_dtype < 0 || a.M == 0 || quantised_within(a, num_sms, &split, &d)) return 0;
  return (static_cast<size_t>(a.M) * a.K + 255) / 256 * 256 + static_cast<size_t>(a.M) * a.G * 4;
}

int launch_fp8_linear(const LinearArgs& args, int num_sms, cudaStream_t stream) {
  LinearArgs a = args;
  CUtensorMap tm_w, tm_x;
  int rc, split;
  DecodeSmem d;
  if (quantised_within(a, num_sms, &split, &d)) {
    if ((rc = make_tmap_bytes(&tm_w, a.w, a.K, a.N, a.ldw, 128)) != B200MOE_OK) return rc;
    return a.x_dtype == B200MOE_DTYPE_BF16 ? launch_decode<16, true, __nv_bfloat16>(a, d, split, tm_w, tm_w, stream)
                                           : launch_decode<16, true, __half>(a, d, split, tm_w, tm_w, stream);
  }
  if (a.x_dtype >= 0) {
    rc = a.x_dtype == B200MOE_DTYPE_BF16 ? launch_quant<__nv_bfloat16>(a, stream) : launch_quant<__half>(a, stream);
    if (rc != B200MOE_OK) return rc;
    a.x = a.ws_q;
    a.x_scale = a.ws_scale;
    a.ldx = a.K;
  }
  const Plan p = pick_plan(a, num_sms);
  if (p.tile == B200MOE_LINEAR_TILE_PAIR_256) return launch_tokens<256, true>(a, p.split, num_sms, stream);
  if (p.tile == B200MOE_LINEAR_TILE_PAIR_128) return launch_tokens<128, true>(a, p.split, num_sms, stream);
  if (p.tile == B200MOE_LINEAR_TILE_TOKENS) return launch_tokens<128, false>(a, p.split, num_sms, stream);
  if (!plan_decode(a, false, num_sms, &split, &d)) return B200MOE_ERR_TOO_LARGE;
  if ((rc = make_tmap_bytes(&tm_w, a.w, a.K, a.N, a.ldw, 128)) != B200MOE_OK) return rc;
  const int nt = decode_tokens(a.M);
  if ((rc = make_tmap_bytes(&tm_x, a.x, a.K, a.M, a.ldx, nt)) != B200MOE_OK) return rc;
  return nt == 16   ? launch_decode<16, false, __half>(a, d, split, tm_w, tm_x, stream)
         : nt == 32 ? launch_decode<32, false, __half>(a, d, split, tm_w, tm_x, stream)
                    : launch_decode<64, false, __half>(a, d, split, tm_w, tm_x, stream);
}

}  // namespace b200moe
