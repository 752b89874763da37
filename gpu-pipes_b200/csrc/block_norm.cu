// Row norms around a block (attention, feed-forward), fused with its gate and residual scales.
//
//   r[i] = x_scale x[i] + y_scale gate[i / gate_rows] (.) Npost(y[i])
//   h[i] = Npre(r[i])
//   LayerNorm: (v - mean) / sqrt(mean((v - mean)^2) + eps) gamma + beta;  RMS: v / sqrt(mean(v^2) + eps) gamma + beta
//
// The work is bytes: each of x, y is read once and each of r, h written once; the row stays in
// registers between the passes over it, so LayerNorm takes its statistics in two passes (mean, then
// squared deviations) as the chains' tails do. All arithmetic is fp32 and h is computed from the
// unrounded r: each output is rounded once.
#include "block_norm.cuh"

#include "../../include/gpipes.h"
#include "chain_registry.h"
#include "gp_ptx.cuh"

namespace gp {
namespace {

// 8 consecutive elements, as loaded and as fp32
template <typename T>
struct Vec8 {
  uint4 u[sizeof(T) / 2];
  __device__ __forceinline__ void load(const void* base, int64_t i) {
    const uint4* p = reinterpret_cast<const uint4*>(static_cast<const T*>(base) + i);
    u[0] = p[0];
    if constexpr (sizeof(T) == 4) u[1] = p[1];
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
    if constexpr (sizeof(T) == 4) {
      v[0] = __uint_as_float(u[0].x), v[1] = __uint_as_float(u[0].y), v[2] = __uint_as_float(u[0].z), v[3] = __uint_as_float(u[0].w);
      v[4] = __uint_as_float(u[1].x), v[5] = __uint_as_float(u[1].y), v[6] = __uint_as_float(u[1].z), v[7] = __uint_as_float(u[1].w);
    } else {
      const float2 a = Elem<T>::unpack(u[0].x), b = Elem<T>::unpack(u[0].y), c = Elem<T>::unpack(u[0].z), d = Elem<T>::unpack(u[0].w);
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y, v[4] = c.x, v[5] = c.y, v[6] = d.x, v[7] = d.y;
    }
  }
};

template <typename T>
__device__ __forceinline__ void load8(const void* base, int64_t i, float (&v)[8]) {
  Vec8<T> r;
  r.load(base, i);
  r.get(v);
}

template <typename T>
__device__ __forceinline__ void store8(void* base, int64_t i, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    float4* p = reinterpret_cast<float4*>(static_cast<float*>(base) + i);
    p[0] = make_float4(v[0], v[1], v[2], v[3]);
    p[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    uint4 u;
    u.x = Elem<T>::pack(v[0], v[1]);
    u.y = Elem<T>::pack(v[2], v[3]);
    u.z = Elem<T>::pack(v[4], v[5]);
    u.w = Elem<T>::pack(v[6], v[7]);
    *reinterpret_cast<uint4*>(static_cast<T*>(base) + i) = u;
  }
}

// Sum over the TPR threads of a row, in a fixed order. red: TPR / 32 floats; a row of one warp
// needs no shared memory. Consecutive calls alternate between two buffers, so one barrier per
// call keeps a slot from being rewritten before every thread has read it.
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int w = 0; w < TPR / 32; ++w) v += red[w];
  }
  return v;
}

// TPR threads per row, NV vectors of 8 elements per thread; rows of one warp share a CTA of 256.
template <typename T, typename X, typename Y, int TPR, int NV>
__global__ void __launch_bounds__(TPR == 32 ? 256 : TPR) block_norm_kernel(const __grid_constant__ BlockNormArgs a) {
  __shared__ float red[2][32];
  constexpr int kRows = TPR == 32 ? 8 : 1;  // rows per CTA: eight of a warp each, or one
  const int lane = threadIdx.x % TPR;
  const int width = a.width;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int64_t row = static_cast<int64_t>(blockIdx.x) * kRows + threadIdx.x / TPR;
  if (row >= a.m) return;  // whole warps (TPR = 32), or never (one row per CTA)
  const int64_t base = row * width;
  float v[NV][8];
  const float inv = 1.0f / static_cast<float>(width);
  int buf = 0;
  auto total = [&](float s) {
    buf ^= 1;
    return row_sum<TPR>(s, red[buf]);
  };
  // v <- N(v) gamma + beta over the row; columns past the width stay zero
  auto norm = [&](int kind, float eps, const void* gamma, const void* beta) {
    if (kind == GP_NORM_LAYER) {
      float s = 0.0f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) s += v[j][e];
      const float mean = total(s) * inv;
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if ((lane + j * TPR) * 8 < width)
#pragma unroll
          for (int e = 0; e < 8; ++e) v[j][e] -= mean;
    }
    float q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < 8; ++e) q = fmaf(v[j][e], v[j][e], q);
    const float rs = rsqrtf(total(q) * inv + eps);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (lane + j * TPR) * 8;
      if (c >= width) continue;
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] *= rs;
      if (gamma != nullptr) {
        load8<T>(gamma, c, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= p[e];
      }
      if (beta != nullptr) {
        load8<T>(beta, c, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] += p[e];
      }
    }
  };

  // both operands are on their way before either is used
  Vec8<X> xv[NV];
  Vec8<Y> yv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (lane + j * TPR) * 8;
    if (c < width && a.y != nullptr) yv[j].load(a.y, base + c);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (lane + j * TPR) * 8;
    if (c < width && a.x != nullptr) xv[j].load(a.x, base + c);
  }
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[j][e] = 0.0f;
  if (a.y != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if ((lane + j * TPR) * 8 < width) yv[j].get(v[j]);
    if (a.post != GP_NORM_NONE) norm(a.post, a.post_eps, a.post_gamma, a.post_beta);
    const int64_t grow = a.gate_rows > 0 ? row / a.gate_rows : 0;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (lane + j * TPR) * 8;
      if (c >= width) continue;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] *= a.y_scale;
      if (a.gate != nullptr) {
        float p[8];
        load8<T>(a.gate, grow * width + c, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[j][e] *= p[e];
      }
    }
  }
  if (a.x != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if ((lane + j * TPR) * 8 >= width) continue;
      float p[8];
      xv[j].get(p);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[j][e] = fmaf(a.x_scale, p[e], v[j][e]);
    }
  }
  if (a.r != nullptr) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (lane + j * TPR) * 8;
      if (c < width) store8<X>(a.r, base + c, v[j]);
    }
  }
  if (a.h != nullptr) {
    if (a.pre != GP_NORM_NONE) norm(a.pre, a.pre_eps, a.pre_gamma, a.pre_beta);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = (lane + j * TPR) * 8;
      if (c < width) store8<T>(a.h, base + c, v[j]);
    }
  }
}

template <typename T, typename X, typename Y, int TPR, int NV>
int launch_t(const BlockNormArgs& a, cudaStream_t stream) {
  constexpr int kThreads = TPR == 32 ? 256 : TPR;
  constexpr int kRows = TPR == 32 ? 8 : 1;
  const int64_t grid = (a.m + kRows - 1) / kRows;
  const uint64_t h = static_cast<uint64_t>(a.width), rows = static_cast<uint64_t>(a.m) * h;
  PdlIo io;
  io.add(PdlIo::kWrite, a.r, rows * sizeof(X));
  io.add(PdlIo::kWrite, a.h, rows * sizeof(T));
  PdlLaunch pdl(stream);
  launch_chain_kernel(&block_norm_kernel<T, X, Y, TPR, NV>, static_cast<int>(grid), kThreads, 0, stream, a);
  pdl.record(io);
  cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? GP_OK : set_error(GP_ERR_CUDA, "block norm launch: %s", cudaGetErrorString(e));
}

// A row is one warp up to 1,024 columns (no barrier, eight rows in flight per CTA), one CTA above. The
// CTA's size keeps two vectors per thread up to 4,096 columns, four above: a row's two reductions are
// latency, which other CTAs on the SM cover, and more threads per row leave fewer of them; fewer threads
// leave single rows slower. Measured on bf16 rows with a norm on both sides (TB/s of x, y, r, h; the other
// split in brackets): 32,768 x 2,048 6.3 (256 x 1: 5.4); 16,384 x 4,096 6.0 (128 x 4: 6.3) and one such row 2.8 us
// (3.5); 8,192 x 8,192 5.9 (512 x 2: 5.8), in fp16 with gates 5.0 (5.4); 4,096 x 16,384 3.8. Above 16,384
// columns 1,024 threads leave 64 registers for four vectors and some spill: 2,048 x 32,768 4.2, fp32 stream 3.7.
template <typename T, typename X, typename Y>
int launch_w(const BlockNormArgs& a, cudaStream_t s) {
  const int h = a.width;
  if (h <= 256) return launch_t<T, X, Y, 32, 1>(a, s);
  if (h <= 512) return launch_t<T, X, Y, 32, 2>(a, s);
  if (h <= 1024) return launch_t<T, X, Y, 32, 4>(a, s);
  if (h <= 2048) return launch_t<T, X, Y, 128, 2>(a, s);
  if (h <= 4096) return launch_t<T, X, Y, 256, 2>(a, s);
  if (h <= 8192) return launch_t<T, X, Y, 256, 4>(a, s);
  if (h <= 16384) return launch_t<T, X, Y, 512, 4>(a, s);
  return launch_t<T, X, Y, 1024, 4>(a, s);
}

template <typename T>
int launch_d(const BlockNormArgs& a, bool x_f32, bool y_f32, cudaStream_t s) {
  if (x_f32) return y_f32 ? launch_w<T, float, float>(a, s) : launch_w<T, float, T>(a, s);
  return y_f32 ? launch_w<T, T, float>(a, s) : launch_w<T, T, T>(a, s);
}

}  // namespace

int launch_block_norm(const BlockNormArgs& a, int dtype, bool x_f32, bool y_f32, cudaStream_t stream) {
  return dtype == GP_BF16 ? launch_d<__nv_bfloat16>(a, x_f32, y_f32, stream)
                          : launch_d<__half>(a, x_f32, y_f32, stream);
}

}  // namespace gp
