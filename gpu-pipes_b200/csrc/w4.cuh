// 4-bit weights with group scales: W[k][n] = s[k / G][n] (q[k][n] - z[k / G][n]), q in 0..15, G = 32, 64
// or 128, s in the activations' 16-bit type T, z an integer 0..15 (8 everywhere without zero points).
//
// Packed form (one buffer, two sections). Weights are held in the order in which a warp's matrix
// instructions take them, so a product reads them in 16-byte pieces and rearranges nothing:
//   codes   [n-tile of 16][k-block of 128][64-row part 2][lane 32][word 4]   1,024 bytes per block
//     lane = 4 g + t holds columns n = 16 tile + 2 g + r (r = 0, 1) and, of each 32-row half h of a
//     part, rows k = 32 h + 16 j + 4 t + i (word = 2 h + j, i = 0..3). The code of (r, i) is nibble
//     4 (i & 1) + 2 (i >> 1) + r of the word: rows i, i + 1 sit 16 bits apart, so one mask takes
//     both values of a 16-bit pair. bf16 words are rotated left by 3 bits (see W4Deq).
//   scales  [n-tile][k-block][g 8][group of the block][r 2] T; with zero points [..][group]{s0, s1, z0, z1}
//     (Z in T, exact): what a lane needs for a block is contiguous.
// Padding (n >= N, k >= K) has code 0, scale 0, zero point 0; every byte of the buffer is defined.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>

#include "chain_registry.h"
#include "gp_ptx.cuh"

namespace gp {

constexpr int64_t kW4MaxK = 1 << 16;
constexpr int64_t kW4MaxN = 1 << 24;
constexpr int kW4Block = 128;       // rows of a k-block
constexpr int kW4BlockBytes = 1024; // codes of a k-block of 16 columns

struct W4Layout {
  int k, n, group;
  int zeros;         // 1: zero points stored
  int n_tiles;       // 16 columns each
  int blocks;        // k-blocks of 128 rows
  int units;         // groups per block: 128 / group
  int64_t scale_off; // bytes from the start of the buffer
  int64_t bytes;

  __host__ __device__ static W4Layout make(int64_t k, int64_t n, int group, int zeros) {
    W4Layout l;
    l.k = static_cast<int>(k);
    l.n = static_cast<int>(n);
    l.group = group;
    l.zeros = zeros != 0;
    l.n_tiles = static_cast<int>((n + 15) / 16);
    l.blocks = static_cast<int>((k + kW4Block - 1) / kW4Block);
    l.units = kW4Block / group;
    const int64_t cells = static_cast<int64_t>(l.n_tiles) * l.blocks;
    l.scale_off = cells * kW4BlockBytes;
    l.bytes = l.scale_off + cells * l.scale_bytes();
    return l;
  }
  // bytes of the scales of one k-block of one n-tile
  __host__ __device__ int scale_bytes() const { return 16 * units * (zeros ? 4 : 2); }
};

__host__ __device__ constexpr int w4_nibble(int r, int i) { return 4 * (i & 1) + 2 * (i >> 1) + r; }

// A word of eight codes as four packed pairs unit_r (q - z) of T for the matrix unit: p[0], p[2] column 0, rows
// (0, 1) and (2, 3); p[1], p[3] column 1. A pair costs one mask (and every other one a shift) and one sum,
// both exact; the power of two leaves once per output.
//   half: a code masked into the low mantissa bits of 1024 is 1024 + q (column 0), or 1024 + 16 q four bits
//     higher (column 1)
//   bf16: the four upper mantissa bits of 16 are q: 16 + q
// z leaves before the product, so an x that meets q = z adds exactly nothing, an infinite x stays infinite, and a
// row's error does not depend on how many rows there are. (Products with q plus a constant, which leaves
// through sums of x over each group, save the sum here and are off by 2^-24 |x| (q + z + twice the constant)
// per term: 26.5 us against 28.2 at 1 x 8,192 x 28,672 fp16, 43.5 against 41.8 at 16 rows; bf16 34.9 / 30.0 and
// 49.0 / 43.4.)
// The words of bf16 weights are stored rotated left by 3, which puts code 0 on those bits.
template <typename T>
struct W4Deq;

// (w & MASK) | base in one instruction (as an expression it was two: 32.7 us against 28.2 at 1 x 8,192 x 28,672)
template <uint32_t MASK>
__device__ __forceinline__ uint32_t w4_mask_or(uint32_t w, uint32_t base) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(w), "n"(MASK), "r"(base));
  return r;
}

template <>
struct W4Deq<__half> {
  static constexpr int kRotate = 0;
  __half2 c[2];
  __host__ __device__ static constexpr float unit(int r) { return r == 0 ? 1.0f : 16.0f; }
  // z01: the two columns' zero points in T (8 if not ZP)
  template <bool ZP>
  __device__ __forceinline__ void set(uint32_t z01) {
    if constexpr (ZP) {
      const __half2 z = *reinterpret_cast<const __half2*>(&z01), o = __float2half2_rn(-1024.0f);
      c[0] = __hsub2(o, __low2half2(z));
      c[1] = __hfma2(__high2half2(z), __float2half2_rn(-16.0f), o);
    } else {
      c[0] = __float2half2_rn(-1032.0f), c[1] = __float2half2_rn(-1152.0f);
    }
  }
  __device__ __forceinline__ static void masked(uint32_t w, uint32_t (&p)[4]) {
    const uint32_t v = w >> 8;
    p[0] = w4_mask_or<0x000F000Fu>(w, 0x64006400u);
    p[1] = w4_mask_or<0x00F000F0u>(w, 0x64006400u);
    p[2] = w4_mask_or<0x000F000Fu>(v, 0x64006400u);
    p[3] = w4_mask_or<0x00F000F0u>(v, 0x64006400u);
  }
  __device__ __forceinline__ void pairs(uint32_t w, uint32_t (&p)[4]) const {
    masked(w, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 q = __hadd2(*reinterpret_cast<const __half2*>(&p[i]), c[i & 1]);
      p[i] = *reinterpret_cast<const uint32_t*>(&q);
    }
  }
};

template <>
struct W4Deq<__nv_bfloat16> {
  static constexpr int kRotate = 3;
  __nv_bfloat162 c[2];
  __host__ __device__ static constexpr float unit(int) { return 1.0f; }
  template <bool ZP>
  __device__ __forceinline__ void set(uint32_t z01) {
    if constexpr (ZP) {
      const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&z01), o = __float2bfloat162_rn(-16.0f);
      c[0] = __hsub2(o, __low2bfloat162(z));
      c[1] = __hsub2(o, __high2bfloat162(z));
    } else {
      c[0] = c[1] = __float2bfloat162_rn(-24.0f);
    }
  }
  __device__ __forceinline__ static void masked(uint32_t w, uint32_t (&p)[4]) {
    p[0] = w4_mask_or<0x00780078u>(w, 0x41804180u);
#pragma unroll
    for (int i = 1; i < 4; ++i) p[i] = w4_mask_or<0x00780078u>(__funnelshift_r(w, w, 4 * i), 0x41804180u);
  }
  __device__ __forceinline__ void pairs(uint32_t w, uint32_t (&p)[4]) const {
    masked(w, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 q = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&p[i]), c[i & 1]);
      p[i] = *reinterpret_cast<const uint32_t*>(&q);
    }
  }
};

// codes as stored <-> nibble i at bits 4 i
template <typename T>
__device__ __forceinline__ uint32_t w4_store_word(uint32_t v) {
  return __funnelshift_l(v, v, W4Deq<T>::kRotate);
}
template <typename T>
__device__ __forceinline__ uint32_t w4_load_word(uint32_t v) {
  return __funnelshift_r(v, v, W4Deq<T>::kRotate);
}

// Codes of a lane as T, s (q - z) rounded once: for the two columns r, the scale twice and the constant that takes the
// zero point and the code's offset away (both steps exact before the scale).
//   half: 1024 + q minus 1024 + z; column 1 four bits higher: (1024 + 16 q) / 16 - (64 + z)
//   bf16: 16 + q minus 16 + z
// As two T (with `rest`) a weight past T's largest number is that number and the rest of it, infinite only past
// twice the largest: the rounded product alone would be infinite and its rest minus infinity.
template <typename T>
struct W4Exact;

// Whether 15 times one of two scales may round to infinity: only then need the products be limited. (Limiting
// always: 46 -> 49 us at 64 rows of 4,096 -> 14,336 -> 4,096; a warp that looks first: 46.4.)
template <typename T>
__device__ __forceinline__ bool w4_large(uint32_t s01) {
  constexpr uint32_t kMost = Elem<T>::kIsBf16 ? 0x7D88u : 0x6C43u;  // 1.0625 2^124, 4,364
  const uint32_t a = s01 & 0x7FFF7FFFu;
  return (a & 0xFFFFu) > kMost || (a >> 16) > kMost;
}

// a pair of T, each limited to T's largest number in magnitude; a NaN stays
template <typename T>
__device__ __forceinline__ uint32_t w4_limit(uint32_t a) {
  uint32_t r;
  if constexpr (Elem<T>::kIsBf16)
    asm("min.NaN.xorsign.abs.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x7F7F7F7Fu));
  else
    asm("min.NaN.xorsign.abs.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(0x7BFF7BFFu));
  return r;
}

template <>
struct W4Exact<__half> {
  __half2 s[2], c[2];
  __device__ __forceinline__ void set(uint32_t s01, uint32_t z01, bool zp) {
    const __half2 sv = *reinterpret_cast<const __half2*>(&s01);
    s[0] = __low2half2(sv), s[1] = __high2half2(sv);
    if (zp) {
      const __half2 z = *reinterpret_cast<const __half2*>(&z01);
      c[0] = __hneg2(__hadd2(__low2half2(z), __float2half2_rn(1024.0f)));
      c[1] = __hneg2(__hadd2(__high2half2(z), __float2half2_rn(64.0f)));
    } else {
      c[0] = __float2half2_rn(-1032.0f), c[1] = __float2half2_rn(-72.0f);
    }
  }
  // r[2 column + j]: rows (0, 1) (j = 0) and (2, 3) of the word, as tcgen05.st 16x256b takes them. rest: what
  // each rounding took away, itself exact in T (s (q - z) has four bits more than T) but for weights
  // below T's smallest normal value or past its largest: there it may be rounded once more, by at most half a
  // step of the weight in the second case. large: some scale of the group is w4_large.
  __device__ __forceinline__ void word(uint32_t w, uint32_t* r, uint32_t* rest = nullptr, bool large = false) const {
    const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = i == 0 ? w : w >> 8;
      const uint32_t lo = w4_mask_or<0x000F000Fu>(v, 0x64006400u), hi = w4_mask_or<0x00F000F0u>(v, 0x64006400u);
      const __half2 qa = __hadd2(*reinterpret_cast<const __half2*>(&lo), c[0]);
      const __half2 qb = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, c[1]);
      __half2 a = __hmul2(qa, s[0]), b = __hmul2(qb, s[1]);
      r[i] = *reinterpret_cast<const uint32_t*>(&a);
      r[2 + i] = *reinterpret_cast<const uint32_t*>(&b);
      if (rest != nullptr) {
        if (large) {
          r[i] = w4_limit<__half>(r[i]);
          r[2 + i] = w4_limit<__half>(r[2 + i]);
          a = *reinterpret_cast<const __half2*>(&r[i]);
          b = *reinterpret_cast<const __half2*>(&r[2 + i]);
        }
        const __half2 ea = __hfma2(qa, s[0], __hneg2(a)), eb = __hfma2(qb, s[1], __hneg2(b));
        rest[i] = *reinterpret_cast<const uint32_t*>(&ea);
        rest[2 + i] = *reinterpret_cast<const uint32_t*>(&eb);
      }
    }
  }
};

template <>
struct W4Exact<__nv_bfloat16> {
  __nv_bfloat162 s[2], c[2];
  __device__ __forceinline__ void set(uint32_t s01, uint32_t z01, bool zp) {
    const __nv_bfloat162 sv = *reinterpret_cast<const __nv_bfloat162*>(&s01);
    s[0] = __low2bfloat162(sv), s[1] = __high2bfloat162(sv);
    if (zp) {
      const __nv_bfloat162 z = *reinterpret_cast<const __nv_bfloat162*>(&z01), o = __float2bfloat162_rn(16.0f);
      c[0] = __hneg2(__hadd2(__low2bfloat162(z), o));
      c[1] = __hneg2(__hadd2(__high2bfloat162(z), o));
    } else {
      c[0] = c[1] = __float2bfloat162_rn(-24.0f);
    }
  }
  __device__ __forceinline__ void word(uint32_t w, uint32_t* r, uint32_t* rest = nullptr, bool large = false) const {
    uint32_t p[4];
    W4Deq<__nv_bfloat16>::masked(w, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // p[2 j + column], j: rows (0, 1) / (2, 3)
      const __nv_bfloat162 q = __hadd2(*reinterpret_cast<const __nv_bfloat162*>(&p[i]), c[i & 1]);
      __nv_bfloat162 a = __hmul2(q, s[i & 1]);
      r[2 * (i & 1) + (i >> 1)] = *reinterpret_cast<const uint32_t*>(&a);
      if (rest != nullptr) {
        if (large) {
          r[2 * (i & 1) + (i >> 1)] = w4_limit<__nv_bfloat16>(r[2 * (i & 1) + (i >> 1)]);
          a = *reinterpret_cast<const __nv_bfloat162*>(&r[2 * (i & 1) + (i >> 1)]);
        }
        const __nv_bfloat162 e = __hfma2(q, s[i & 1], __hneg2(a));
        rest[2 * (i & 1) + (i >> 1)] = *reinterpret_cast<const uint32_t*>(&e);
      }
    }
  }
};

// v as two T, in the low halves; an infinity (a value past T's range) has no second part.
template <typename T>
__device__ __forceinline__ void w4_two(float v, uint16_t& hi, uint16_t& lo) {
  hi = static_cast<uint16_t>(Elem<T>::pack(v, 0.0f));
  const float f = Elem<T>::unpack(hi).x;
  lo = static_cast<uint16_t>(fabsf(f) <= 3.4028235e38f ? Elem<T>::pack(v - f, 0.0f) : 0u);
}

// W words from shared memory in one access (two for W = 8)
template <int W>
__device__ __forceinline__ void w4_lds(uint32_t p, uint32_t (&v)[W]) {
  if constexpr (W == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(p) : "memory");
  } else if constexpr (W == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(p) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4)
      asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
                   : "r"(p + 4 * i)
                   : "memory");
  }
}

// Activations of the epilogues in fp32: v sigmoid(u) with u = v (SiLU) or, for GELU's tanh form, twice
// its argument (0.5 (1 + tanh(t)) = sigmoid(2 t)). The fast exponential and quotient are within a few
// units of 2^-22 |u| of the exact ones, far below the 16-bit rounding that follows (results smaller than
// 1e-36, u below -87, become zero). Written without
// calls: expf, tanhf and divisions in the epilogues took 36 of 98 us at 512 x 4,096 x 14,336.
// The choice is made once for N values, whose arithmetic then overlaps.
template <int N>
__device__ __forceinline__ void w4_act(int act, float (&v)[N]) {
  if (act == kActNone) return;
  if (act == kActRelu) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = v[i] > 0.0f ? v[i] : (v[i] == v[i] ? 0.0f : v[i]);
    return;
  }
  float e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = -v[i];
  if (act == kActGeluTanh)
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = -1.5957691216057308f * fmaf(0.044715f * v[i], v[i] * v[i], v[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = __fdividef(act == kActSigmoid ? 1.0f : v[i], 1.0f + __expf(e[i]));
}

// ---- host interface (w4_pack.cu, w4_linear.cu); dtype is GP_F16 / GP_BF16
int launch_w4_quantize(const W4Layout& l, int dtype, const void* w, void* packed, cudaStream_t s);
int launch_w4_pack(const W4Layout& l, int dtype, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                   void* packed, cudaStream_t s);
int launch_w4_unpack(const W4Layout& l, int dtype, const void* packed, uint8_t* codes, void* scales, uint8_t* zeros,
                     cudaStream_t s);
int launch_w4_dequantize(const W4Layout& l, int dtype, const void* packed, void* w, cudaStream_t s);

// out [m, n] = act(x [m, k] W + bias), out in T or fp32 (out_f32); x rows are read 16 bytes at a time.
// Two planes hold a value as two T, [2][m][width]: its rounding, and what that took away.
struct W4LinearArgs {
  W4Layout l;
  int dtype;
  int64_t m;
  const void* x;
  const void* packed;
  const void* bias;
  int act;
  void* out;
  bool out_f32;
  int x_planes = 1, out_planes = 1;
  bool exact = false;  // no weight is rounded, at any m
};
// How many clusters of ck CTAs (one CTA per SM) the device holds at a time: fewer than SMs / ck, as a
// cluster stays within a GPC. `cache` is the caller's, one entry per device and log2(ck), zero at first.
int w4_max_clusters(const void* kern, int threads, int smem, int ck, int sm_count, std::atomic<int> (*cache)[4]);
int launch_w4_rows(const W4LinearArgs& a, cudaStream_t s, const DeviceInfo& dev);   // few rows (w4_linear.cu)
int launch_w4_tiles(const W4LinearArgs& a, cudaStream_t s, const DeviceInfo& dev);  // more rows (w4_tiles.cu)
int launch_w4_linear(const W4LinearArgs& a, cudaStream_t s, const DeviceInfo& dev);

}  // namespace gp
