// Row norms around a block, fused with the block's gate and the residual scales:
//   r = x_scale x + y_scale gate (.) Npost(y),   h = Npre(r),   N = none | LayerNorm | RMS norm
// Host interface (block_norm.cu); the kernel and its reasons are there.
#pragma once

#include <cuda_runtime.h>

#include <cstdint>

namespace gp {

struct BlockNormArgs {
  int64_t m;
  int64_t gate_rows;   // consecutive rows that share a gate row (0: one gate row for all)
  int width;
  int post, pre;       // gp_norm
  float x_scale, y_scale, post_eps, pre_eps;
  const void* x;       // stream rows [m, width] (T or fp32), or null
  const void* y;       // block output rows [m, width] (T or fp32), or null
  const void* gate;    // T, or null
  const void* post_gamma;
  const void* post_beta;
  const void* pre_gamma;
  const void* pre_beta;
  void* r;             // stream rows out (type of x), or null
  void* h;             // normed rows out (T), or null
};

constexpr int kBlockNormMaxWidth = 32768;

// dtype: GP_F16 / GP_BF16 (T); x_f32 / y_f32: the stream / the block output are fp32. One launch.
int launch_block_norm(const BlockNormArgs& a, int dtype, bool x_f32, bool y_f32, cudaStream_t stream);

}  // namespace gp
