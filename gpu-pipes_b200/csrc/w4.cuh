// 4-bit weights with group scales: W[k][n] = s[k / G][n] (q[k][n] - z[k / G][n]), q in 0..15, G = 32, 64
// or 128, s in the activations' 16-bit type T, z an integer 0..15 (8 everywhere without zero points).
//
// Packed form (one buffer, two sections). Weights are held in the order in which a warp's matrix
// instructions take them, so a product reads them in 16-byte pieces and rearranges nothing:
//   codes   [n-tile of 16][k-block of 64][lane 32][word 4]   512 bytes per tile and block
//     lane = 4 g + t holds columns n = 16 tile + 2 g + r (r = 0, 1) and, of each 32-half h of the
//     block, rows k = 64 block + 32 h + 8 t + 4 j + i (word = 2 h + j, i = 0..3). In a word the code
//     of (r, i) is nibble 4 (i & 1) + 2 (i >> 1) + r: pairs (i, i + 1) sit 16 bits apart, so one
//     mask takes the two values of a packed 16-bit pair.
//   scales  [n-tile][group][16] T; with zero points [n-tile][group][8 g] {s0, s1, z0, z1} T, the
//     two columns of a lane next to each other. Z is held in T (exact).
// Padding (n >= N, k >= K) has code 0, scale 0, zero point 0; every byte of the buffer is defined.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "gp_ptx.cuh"

namespace gp {

constexpr int64_t kW4MaxK = 1 << 16;
constexpr int64_t kW4MaxN = 1 << 24;

struct W4Layout {
  int k, n, group;
  int zeros;         // 1: zero points stored
  int n_tiles;       // 16 columns each
  int k_blocks;      // 64 rows each
  int groups;        // groups stored per tile: those of k_blocks whole blocks
  int64_t scale_off; // bytes from the start of the buffer
  int64_t bytes;

  __host__ __device__ static W4Layout make(int64_t k, int64_t n, int group, int zeros) {
    W4Layout l;
    l.k = static_cast<int>(k);
    l.n = static_cast<int>(n);
    l.group = group;
    l.zeros = zeros != 0;
    l.n_tiles = static_cast<int>((n + 15) / 16);
    l.k_blocks = static_cast<int>((k + 63) / 64);
    l.groups = (l.k_blocks * 64 + group - 1) / group;
    l.scale_off = static_cast<int64_t>(l.n_tiles) * l.k_blocks * 512;
    l.bytes = l.scale_off + static_cast<int64_t>(l.n_tiles) * l.groups * 16 * (l.zeros ? 4 : 2);
    return l;
  }
};

__host__ __device__ constexpr int w4_nibble(int r, int i) { return 4 * (i & 1) + 2 * (i >> 1) + r; }

// Integers 0..15 as T pairs out of a word of codes, minus the zero point, exactly: a code ORed into
// the mantissa of 1024 (half) or 128 (bf16) is 1024 + q (128 + q), and the difference to 1024 + z
// is exact. In half the upper nibble of a byte is taken in place as 1024 + 16 q and scaled by 1/16
// in the same instruction that subtracts 64 + z, which saves the shift; bf16's mantissa is too
// short for that.
template <typename T>
struct W4Deq;

template <>
struct W4Deq<__half> {
  // zero points of the lane's two columns -> the constants of pairs()
  __device__ __forceinline__ static void consts(uint32_t z01, uint32_t& c0, uint32_t& c1) {
    const __half2 z = *reinterpret_cast<const __half2*>(&z01);
    const __half2 a = __hadd2(__low2half2(z), __float2half2_rn(1024.0f));
    const __half2 b = __hneg2(__hadd2(__high2half2(z), __float2half2_rn(64.0f)));
    c0 = *reinterpret_cast<const uint32_t*>(&a);
    c1 = *reinterpret_cast<const uint32_t*>(&b);
  }
  static constexpr uint32_t kC0 = 0x64086408u;  // 1024 + 8
  static constexpr uint32_t kC1 = 0xD480D480u;  // -(64 + 8)
  // p[0], p[2]: column 0, rows (0, 1) and (2, 3); p[1], p[3]: column 1
  __device__ __forceinline__ static void pairs(uint32_t w, uint32_t c0, uint32_t c1, uint32_t (&p)[4]) {
    const __half2 z0 = *reinterpret_cast<const __half2*>(&c0), z1 = *reinterpret_cast<const __half2*>(&c1);
    const __half2 s = __float2half2_rn(0.0625f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = i == 0 ? w : w >> 8;
      const uint32_t lo = (v & 0x000F000Fu) | 0x64006400u, hi = (v & 0x00F000F0u) | 0x64006400u;
      const __half2 a = __hsub2(*reinterpret_cast<const __half2*>(&lo), z0);
      const __half2 b = __hfma2(*reinterpret_cast<const __half2*>(&hi), s, z1);
      p[2 * i] = *reinterpret_cast<const uint32_t*>(&a);
      p[2 * i + 1] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
};

template <>
struct W4Deq<__nv_bfloat16> {
  __device__ __forceinline__ static void consts(uint32_t z01, uint32_t& c0, uint32_t& c1) {
    const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&z01);
    const __nv_bfloat162 o = __float2bfloat162_rn(128.0f);
    const __nv_bfloat162 a = __hadd2(__low2bfloat162(z), o), b = __hadd2(__high2bfloat162(z), o);
    c0 = *reinterpret_cast<const uint32_t*>(&a);
    c1 = *reinterpret_cast<const uint32_t*>(&b);
  }
  static constexpr uint32_t kC0 = 0x43084308u;  // 128 + 8
  static constexpr uint32_t kC1 = 0x43084308u;
  __device__ __forceinline__ static void pairs(uint32_t w, uint32_t c0, uint32_t c1, uint32_t (&p)[4]) {
    const __nv_bfloat162 z0 = *reinterpret_cast<const __nv_bfloat162*>(&c0);
    const __nv_bfloat162 z1 = *reinterpret_cast<const __nv_bfloat162*>(&c1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = ((w >> (4 * i)) & 0x000F000Fu) | 0x43004300u;
      const __nv_bfloat162 a = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), (i & 1) ? z1 : z0);
      p[i] = *reinterpret_cast<const uint32_t*>(&a);
    }
  }
};

// ---- host interface (w4_pack.cu, w4_linear.cu); dtype is GP_F16 / GP_BF16
int launch_w4_quantize(const W4Layout& l, int dtype, const void* w, void* packed, cudaStream_t s);
int launch_w4_pack(const W4Layout& l, int dtype, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                   void* packed, cudaStream_t s);
int launch_w4_unpack(const W4Layout& l, int dtype, const void* packed, uint8_t* codes, void* scales, uint8_t* zeros,
                     cudaStream_t s);
int launch_w4_dequantize(const W4Layout& l, int dtype, const void* packed, void* w, cudaStream_t s);

// out [m, n] = act(x [m, k] W + bias), out in T or fp32 (out_f32); x rows are read 16 bytes at a time
int launch_w4_linear(const W4Layout& l, int dtype, int64_t m, const void* x, const void* packed, const void* bias,
                     int act, void* out, bool out_f32, cudaStream_t s, int sm_count);

}  // namespace gp
