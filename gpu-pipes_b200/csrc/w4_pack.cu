// Quantising 16-bit weights to 4 bits with group scales, and the ways in and out of the packed
// form (w4.cuh): from codes and scales made elsewhere, back to them, and to 16-bit weights.
//
// Every kernel has the same shape: a thread owns two neighbouring columns (a lane's column pair g
// of the packed layout) and one group of rows. A warp's 32 column pairs make 128-byte rows of the
// 16-bit matrix, so its reads (or writes) are whole lines, and a pair's rows of a 64-row block are
// 64 consecutive bytes of the packed form. The quantiser keeps the group's values in registers
// between the range and the codes, so the matrix is read once; all of it is bound by those bytes.
#include "../../include/gpipes.h"
#include "chain_registry.h"
#include "w4.cuh"

namespace gp {
namespace {

constexpr int kPackThreads = 128;

// Two neighbouring elements of a row of n columns (c even; one element when c + 1 == n or the row
// is not 4-byte aligned). VEC: n is even and the base 4-byte aligned.
template <bool VEC, typename E>
__device__ __forceinline__ uint32_t load_pair(const E* p, int64_t row, int n, int c) {
  static_assert(sizeof(E) == 2, "16-bit elements");
  const uint16_t* q = reinterpret_cast<const uint16_t*>(p) + row * n + c;
  if constexpr (VEC) return *reinterpret_cast<const uint32_t*>(q);
  return static_cast<uint32_t>(q[0]) | (c + 1 < n ? static_cast<uint32_t>(q[1]) << 16 : 0u);
}

template <bool VEC, typename E>
__device__ __forceinline__ void store_pair(E* p, int64_t row, int n, int c, uint32_t v) {
  uint16_t* q = reinterpret_cast<uint16_t*>(p) + row * n + c;
  if constexpr (VEC) {
    *reinterpret_cast<uint32_t*>(q) = v;
  } else {
    q[0] = static_cast<uint16_t>(v);
    if (c + 1 < n) q[1] = static_cast<uint16_t>(v >> 16);
  }
}

struct Where {
  int tile, g, c;  // n-tile, column pair in it, first column
  bool in;         // the pair's tile exists
};

__device__ __forceinline__ Where where(const W4Layout& l) {
  const int pair = blockIdx.x * kPackThreads + threadIdx.x;
  Where w;
  w.tile = pair >> 3;
  w.g = pair & 7;
  w.c = 2 * pair;
  w.in = w.tile < l.n_tiles;
  return w;
}

// part: 64-row part of the whole matrix (block = part / 2)
__device__ __forceinline__ uint4* code_ptr(const W4Layout& l, void* packed, int tile, int part, int g) {
  return reinterpret_cast<uint4*>(static_cast<char*>(packed) +
                                  ((static_cast<int64_t>(tile) * l.blocks * 2 + part) * (kW4BlockBytes / 2) + g * 64));
}

__device__ __forceinline__ uint32_t* scale_ptr(const W4Layout& l, void* packed, int tile, int group, int g) {
  const int64_t cell = static_cast<int64_t>(tile) * l.blocks + group / l.units;
  const int64_t i = (cell * 8 + g) * l.units + group % l.units;
  return reinterpret_cast<uint32_t*>(static_cast<char*>(packed) + l.scale_off) + (l.zeros ? 2 * i : i);
}

// Codes of one 32-row half of a block for a column pair: q(r, k) gives the code of row k (0..31) of
// the half. Word 2 h + j of lane 4 g + t.
template <typename T, class F>
__device__ __forceinline__ void put_half(uint4* block_pair, int h, F&& q) {
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    uint32_t w[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      w[j] = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) w[j] |= q(r, 16 * j + 4 * t + i) << (4 * w4_nibble(r, i));
    }
    reinterpret_cast<uint2*>(block_pair + t)[h] = make_uint2(w4_store_word<T>(w[0]), w4_store_word<T>(w[1]));
  }
}

// Codes and scale of a group of G rows (largest magnitude to 7, or the range with zero to 15).
// s is rounded to T first and the codes are taken against the rounded scale; quotients are IEEE
// divisions, rounded half to even. A group whose scale rounds to zero has code = zero point. A
// group with a NaN or an infinity has a scale that is not finite, and so has what it stands for.
template <typename T, int G, bool ZP, bool VEC>
__global__ void __launch_bounds__(kPackThreads) w4_quantize_kernel(const __grid_constant__ W4Layout l,
                                                                   const T* __restrict__ w, void* packed) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const Where at = where(l);
  if (!at.in) return;
  for (int64_t grp = blockIdx.y; grp < l.blocks * l.units; grp += gridDim.y) {
    const int k0 = static_cast<int>(grp) * G;
    uint32_t v[G];
#pragma unroll
    for (int i = 0; i < G; ++i) v[i] = (at.c < l.n && k0 + i < l.k) ? load_pair<VEC>(w, k0 + i, l.n, at.c) : 0u;
    float hi[2] = {0.0f, 0.0f}, lo[2] = {0.0f, 0.0f}, bad[2] = {0.0f, 0.0f};
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const float2 f = Elem<T>::unpack(v[i]);
      hi[0] = fmaxf(hi[0], f.x), lo[0] = fminf(lo[0], f.x), bad[0] += f.x * 0.0f;
      hi[1] = fmaxf(hi[1], f.y), lo[1] = fminf(lo[1], f.y), bad[1] += f.y * 0.0f;
    }
    float s[2], z[2];
    uint32_t s01 = 0, z01 = 0;
    {
      float raw[2];
#pragma unroll
      for (int r = 0; r < 2; ++r)  // max and min drop a NaN: bad (0, or NaN from a NaN or infinity) brings it back
        raw[r] = (ZP ? __fdiv_rn(hi[r] - lo[r], 15.0f) : __fdiv_rn(fmaxf(hi[r], -lo[r]), 7.0f)) + bad[r];
      s01 = Elem<T>::pack(raw[0], raw[1]);
      const float2 f = Elem<T>::unpack(s01);
      s[0] = f.x, s[1] = f.y;
    }
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      z[r] = ZP ? (s[r] > 0.0f ? fminf(fmaxf(rintf(__fdiv_rn(-lo[r], s[r])), 0.0f), 15.0f) : 0.0f) : 8.0f;
    }
    const bool real = at.c < l.n && k0 < l.k;
    if (ZP) z01 = Elem<T>::pack(z[0], z[1]);
    if (!real) s01 = 0, z01 = 0;
    if (at.c + 1 >= l.n) s01 &= 0xFFFFu, z01 &= 0xFFFFu;
    uint32_t* sp = scale_ptr(l, packed, at.tile, static_cast<int>(grp), at.g);
    if (ZP) *reinterpret_cast<uint2*>(sp) = make_uint2(s01, z01);
    else *sp = s01;
#pragma unroll
    for (int hh = 0; hh < G / 32; ++hh) {
      const int k = k0 + hh * 32;
      put_half<T>(code_ptr(l, packed, at.tile, k / 64, at.g), (k / 32) & 1, [&](int r, int kk) {
        const float2 f = Elem<T>::unpack(v[hh * 32 + kk]);
        const float x = r == 0 ? f.x : f.y;
        float q = z[r];
        if (s[r] > 0.0f) q = fminf(fmaxf(rintf(__fdiv_rn(x, s[r])) + z[r], 0.0f), 15.0f);
        const bool pad = k + kk >= l.k || at.c + r >= l.n;
        return pad ? 0u : static_cast<uint32_t>(q);
      });
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kPackThreads) w4_pack_kernel(const __grid_constant__ W4Layout l,
                                                               const uint8_t* __restrict__ codes,
                                                               const T* __restrict__ scales,
                                                               const uint8_t* __restrict__ zeros, void* packed) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const Where at = where(l);
  if (!at.in) return;
  for (int64_t b = blockIdx.y; b < l.blocks * 2; b += gridDim.y) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k = static_cast<int>(b) * 64 + h * 32;
      put_half<T>(code_ptr(l, packed, at.tile, static_cast<int>(b), at.g), h, [&](int r, int kk) {
        const bool pad = k + kk >= l.k || at.c + r >= l.n;
        return pad ? 0u : static_cast<uint32_t>(codes[static_cast<int64_t>(k + kk) * l.n + at.c + r]) & 15u;
      });
    }
    // the scales of the groups that begin in this block
    for (int grp = (static_cast<int>(b) * 64 + l.group - 1) / l.group; grp * l.group < (b + 1) * 64; ++grp) {
      const bool real = at.c < l.n && grp * l.group < l.k;
      const uint32_t s01 = real ? load_pair<VEC>(scales, grp, l.n, at.c) : 0u;
      uint32_t* sp = scale_ptr(l, packed, at.tile, grp, at.g);
      if (l.zeros) {
        uint32_t z[2] = {0, 0};
        for (int r = 0; r < 2; ++r)
          if (real && at.c + r < l.n) z[r] = zeros[static_cast<int64_t>(grp) * l.n + at.c + r] & 15u;
        *reinterpret_cast<uint2*>(sp) = make_uint2(s01, Elem<T>::pack(static_cast<float>(z[0]), static_cast<float>(z[1])));
      } else {
        *sp = s01;
      }
    }
  }
}

template <typename T, bool VEC>
__global__ void __launch_bounds__(kPackThreads) w4_unpack_kernel(const __grid_constant__ W4Layout l, void* packed,
                                                                 uint8_t* __restrict__ codes, T* __restrict__ scales,
                                                                 uint8_t* __restrict__ zeros) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const Where at = where(l);
  if (!at.in || at.c >= l.n) return;
  for (int64_t b = blockIdx.y; b < l.blocks * 2; b += gridDim.y) {
    if (codes != nullptr) {
      const uint4* p = code_ptr(l, packed, at.tile, static_cast<int>(b), at.g);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint4 u = p[t];
        const uint32_t w[4] = {w4_load_word<T>(u.x), w4_load_word<T>(u.y), w4_load_word<T>(u.z), w4_load_word<T>(u.w)};
#pragma unroll
        for (int e = 0; e < 16; ++e) {  // word 2 h + j, row i of it
          const int wi = e >> 2, i = e & 3;
          const int k = static_cast<int>(b) * 64 + (wi >> 1) * 32 + 16 * (wi & 1) + 4 * t + i;
#pragma unroll
          for (int r = 0; r < 2; ++r)
            if (k < l.k && at.c + r < l.n)
              codes[static_cast<int64_t>(k) * l.n + at.c + r] = (w[wi] >> (4 * w4_nibble(r, i))) & 15u;
        }
      }
    }
    for (int grp = (static_cast<int>(b) * 64 + l.group - 1) / l.group; grp * l.group < (b + 1) * 64; ++grp) {
      if (grp * l.group >= l.k) break;
      const uint32_t* sp = scale_ptr(l, packed, at.tile, grp, at.g);
      if (scales != nullptr) store_pair<VEC>(scales, grp, l.n, at.c, sp[0]);
      if (zeros != nullptr && l.zeros) {
        const float2 z = Elem<T>::unpack(sp[1]);
        zeros[static_cast<int64_t>(grp) * l.n + at.c] = static_cast<uint8_t>(z.x);
        if (at.c + 1 < l.n) zeros[static_cast<int64_t>(grp) * l.n + at.c + 1] = static_cast<uint8_t>(z.y);
      }
    }
  }
}

// s (q - z) in fp32 (exact: at most 11 + 5 bits), rounded once to T
template <typename T, bool VEC>
__global__ void __launch_bounds__(kPackThreads) w4_dequantize_kernel(const __grid_constant__ W4Layout l, void* packed,
                                                                     T* __restrict__ w) {
  pdl_wait_prior();
  pdl_launch_dependents();
  const Where at = where(l);
  if (!at.in || at.c >= l.n) return;
  for (int64_t b = blockIdx.y; b < l.blocks * 2; b += gridDim.y) {
    const uint4* p = code_ptr(l, packed, at.tile, static_cast<int>(b), at.g);
    uint4 u[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) u[t] = p[t];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int k0 = static_cast<int>(b) * 64 + h * 32;
      const uint32_t* sp = scale_ptr(l, packed, at.tile, k0 / l.group, at.g);
      const float2 s = Elem<T>::unpack(sp[0]);
      float2 z = make_float2(8.0f, 8.0f);
      if (l.zeros) z = Elem<T>::unpack(sp[1]);
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const uint32_t wd[2] = {w4_load_word<T>(h == 0 ? u[t].x : u[t].z), w4_load_word<T>(h == 0 ? u[t].y : u[t].w)};
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int j = e >> 2, i = e & 3, k = k0 + 16 * j + 4 * t + i;
          const float q0 = static_cast<float>((wd[j] >> (4 * w4_nibble(0, i))) & 15u);
          const float q1 = static_cast<float>((wd[j] >> (4 * w4_nibble(1, i))) & 15u);
          if (k < l.k) store_pair<VEC>(w, k, l.n, at.c, Elem<T>::pack(s.x * (q0 - z.x), s.y * (q1 - z.y)));
        }
      }
    }
  }
}

// Launch over column pairs (x) and 64-row parts or groups (y, with a stride past the grid's limit).
// `out` / `bytes`: what the launch writes.
template <typename... KArgs, typename... Args>
int launch_pack(void (*kern)(KArgs...), const W4Layout& l, int rows, cudaStream_t s, const PdlIo& io, Args... args) {
  cudaLaunchConfig_t cfg = {};
  const int pairs = l.n_tiles * 8;
  cfg.gridDim = dim3(static_cast<unsigned>((pairs + kPackThreads - 1) / kPackThreads),
                     static_cast<unsigned>(rows < 65535 ? rows : 65535), 1);
  cfg.blockDim = dim3(kPackThreads, 1, 1);
  cfg.stream = s;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = pdl_enabled() ? 1 : 0;
  PdlLaunch pdl(s);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, l, args...);
  pdl.record(io);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GP_OK : set_error(GP_ERR_CUDA, "w4 launch: %s", cudaGetErrorString(e));
}

bool even_rows(const W4Layout& l, const void* p) { return l.n % 2 == 0 && reinterpret_cast<uintptr_t>(p) % 4 == 0; }

template <typename T, int G>
int quantize_g(const W4Layout& l, const T* w, void* packed, cudaStream_t s) {
  PdlIo io;
  io.add(PdlIo::kWrite, packed, static_cast<uint64_t>(l.bytes));
  const bool vec = even_rows(l, w);
  auto kern = l.zeros ? (vec ? &w4_quantize_kernel<T, G, true, true> : &w4_quantize_kernel<T, G, true, false>)
                      : (vec ? &w4_quantize_kernel<T, G, false, true> : &w4_quantize_kernel<T, G, false, false>);
  return launch_pack(kern, l, l.blocks * l.units, s, io, w, packed);
}

template <typename T>
int quantize_t(const W4Layout& l, const void* w, void* packed, cudaStream_t s) {
  const T* p = static_cast<const T*>(w);
  return l.group == 32 ? quantize_g<T, 32>(l, p, packed, s)
         : l.group == 64 ? quantize_g<T, 64>(l, p, packed, s)
                         : quantize_g<T, 128>(l, p, packed, s);
}

template <typename T>
int pack_t(const W4Layout& l, const uint8_t* codes, const void* scales, const uint8_t* zeros, void* packed,
           cudaStream_t s) {
  PdlIo io;
  io.add(PdlIo::kWrite, packed, static_cast<uint64_t>(l.bytes));
  auto kern = even_rows(l, scales) ? &w4_pack_kernel<T, true> : &w4_pack_kernel<T, false>;
  return launch_pack(kern, l, l.blocks * 2, s, io, codes, static_cast<const T*>(scales), zeros, packed);
}

template <typename T>
int unpack_t(const W4Layout& l, const void* packed, uint8_t* codes, void* scales, uint8_t* zeros, cudaStream_t s) {
  const uint64_t ng = static_cast<uint64_t>((l.k + l.group - 1) / l.group) * l.n;
  PdlIo io;
  io.add(PdlIo::kWrite, codes, static_cast<uint64_t>(l.k) * l.n);
  io.add(PdlIo::kWrite, scales, ng * 2);
  io.add(PdlIo::kWrite, zeros, ng);
  auto kern = scales != nullptr && even_rows(l, scales) ? &w4_unpack_kernel<T, true> : &w4_unpack_kernel<T, false>;
  return launch_pack(kern, l, l.blocks * 2, s, io, const_cast<void*>(packed), codes, static_cast<T*>(scales), zeros);
}

template <typename T>
int dequantize_t(const W4Layout& l, const void* packed, void* w, cudaStream_t s) {
  PdlIo io;
  io.add(PdlIo::kWrite, w, static_cast<uint64_t>(l.k) * l.n * 2);
  auto kern = even_rows(l, w) ? &w4_dequantize_kernel<T, true> : &w4_dequantize_kernel<T, false>;
  return launch_pack(kern, l, l.blocks * 2, s, io, const_cast<void*>(packed), static_cast<T*>(w));
}

}  // namespace

int launch_w4_quantize(const W4Layout& l, int dtype, const void* w, void* packed, cudaStream_t s) {
  return dtype == GP_BF16 ? quantize_t<__nv_bfloat16>(l, w, packed, s) : quantize_t<__half>(l, w, packed, s);
}

int launch_w4_pack(const W4Layout& l, int dtype, const uint8_t* codes, const void* scales, const uint8_t* zeros,
                   void* packed, cudaStream_t s) {
  return dtype == GP_BF16 ? pack_t<__nv_bfloat16>(l, codes, scales, zeros, packed, s)
                          : pack_t<__half>(l, codes, scales, zeros, packed, s);
}

int launch_w4_unpack(const W4Layout& l, int dtype, const void* packed, uint8_t* codes, void* scales, uint8_t* zeros,
                     cudaStream_t s) {
  return dtype == GP_BF16 ? unpack_t<__nv_bfloat16>(l, packed, codes, scales, zeros, s)
                          : unpack_t<__half>(l, packed, codes, scales, zeros, s);
}

int launch_w4_dequantize(const W4Layout& l, int dtype, const void* packed, void* w, cudaStream_t s) {
  return dtype == GP_BF16 ? dequantize_t<__nv_bfloat16>(l, packed, w, s) : dequantize_t<__half>(l, packed, w, s);
}

}  // namespace gp
