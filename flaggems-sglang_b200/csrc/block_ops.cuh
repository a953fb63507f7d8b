// Operators around the experts: norms on either side of a block, the gated activation and the block-scaled FP8 linear layer.
// Argument blocks and launchers.
#pragma once
#include "common.cuh"

namespace b200moe {

struct NormArgs {
  const void* x;
  const void* residual;         // or null
  const void* gate;
  const void* w_post;           // norm of the block's output (post != 0); null weights count as ones, null biases as zeros
  const void* b_post;
  const void* w_pre;            // norm of the stream for the next block (pre != 0)
  const void* b_pre;
  void* hidden;                 // [M] rows, or null; may be `residual`
  void* y;                      // [M, H]
  float* y_scale;               // not null: y is e4m3, these its scales [M, ceil(H / 128)]
  long long ldx, ldr, ldg, ldh; // row strides in elements
  int M, H;
  int post, pre, layer;
  int gate_mode;                // B200MOE_GATE_*
  int gate_f32, w_post_f32, b_post_f32, w_pre_f32, b_pre_f32;
  float eps, scale, offset;
  int vec;                      // every row starts on 16 bytes (e4m3: 8) and holds whole chunks of eight elements
  int pdl;
  int team, rows_per_cta;       // set by the launcher
};
int launch_block_norm(const NormArgs& a, int dtype, int residual_f32, int num_sms, cudaStream_t stream);

struct ActArgs {
  const void* x;                // [M] rows of 2 I: gate, then linear
  long long ldx;
  void* y;                      // [M, I]
  float* y_scale;               // not null: y is e4m3, these its scales [M, ceil(I / 128)]
  int M, I;
  float alpha, limit;           // B200MOE_ACT_SWIGLU_OAI; limit <= 0: no clamps
  int vec, pdl;
};
int launch_gated_activation(const ActArgs& a, int activation, int dtype, cudaStream_t stream);

struct LinearArgs {
  int M, N, K, G;               // G = ceil(K / 128)
  const void* x;                // 16-bit or e4m3 rows
  long long ldx;
  int x_dtype;                  // B200MOE_DTYPE_*, or B200MOE_X_E4M3 with x_scale
  const float* x_scale;         // [M, G]
  const uint8_t* w;             // e4m3 [N] rows of K
  long long ldw;
  const float* w_scale;         // [ceil(N / 128), G]
  const void* bias;             // [N] or null
  int bias_dtype;
  void* out;                    // [M, N]
  int out_dtype;
  int* status;
  int tile, split;              // 0: choose
  int pdl;
  uint8_t* ws_q;                // 16-bit x of more rows than the kernel quantises itself: room for its e4m3 rows and scales
  float* ws_scale;
};
size_t linear_workspace_bytes(const LinearArgs& a, int num_sms);
int launch_fp8_linear(const LinearArgs& a, int num_sms, cudaStream_t stream);

// api.cu
int make_tmap_bytes(CUtensorMap* m, const void* base, uint64_t inner, uint64_t rows, uint64_t ld, uint32_t box_rows);

}  // namespace b200moe
