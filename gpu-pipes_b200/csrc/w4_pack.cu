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

#include <type_traits>

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

// Range of packed pairs, column by column; a NaN stays.
template <typename T>
struct Pair;
template <>
struct Pair<__half> {
  using V = __half2;
  __device__ __forceinline__ static V max(V a, V b) { return __hmax2_nan(a, b); }
  __device__ __forceinline__ static V min(V a, V b) { return __hmin2_nan(a, b); }
};
template <>
struct Pair<__nv_bfloat16> {
  using V = __nv_bfloat162;
  __device__ __forceinline__ static V max(V a, V b) { return __hmax2_nan(a, b); }
  __device__ __forceinline__ static V min(V a, V b) { return __hmin2_nan(a, b); }
};

// rint(x / s) + z, without a division per weight, as the bits of the float 1.5 2^23 + rint(x / s) + z.
// x and s are T: their quotient is either exactly half way between two integers or, for quotients
// below 16, at least 2^-13 away from there (2 x - (2 k + 1) s is a multiple of half the last place of
// s, and s has 11 bits). below and above are 1 / s less and more 2^-22 of it, so x below and x above lie
// within 2^-17 of the quotient on both sides: they round to the same integer, or, at a tie, to its two
// neighbours, of which the even one is wanted. The fused sum rounds the exact products to integers.
// Below fp32's normal range (bf16 only) 1 / s may be past its largest number: there x and s are both
// taken 2^24 times, which is exact.
constexpr float kMagic = 12582912.0f;  // 1.5 2^23: its last place is 1
constexpr uint32_t kMagicBits = 0x4B400000u;

__device__ __forceinline__ uint32_t w4_code_bits(float x, float below, float above, float magic_z, uint32_t z) {
  const uint32_t a = __float_as_uint(fmaf(x, below, magic_z)), b = __float_as_uint(fmaf(x, above, magic_z));
  return ((a ^ z) & 1u) ? b : a;
}

// (hi - lo) / 15 in fp32. bf16's hi - lo may be past fp32's largest number, where the halves' difference is not:
// then it is taken from those (halving and doubling are exact there). Infinities and NaN stay.
template <typename T>
__device__ __forceinline__ float w4_span_step(float hi, float lo) {
  const float span = hi - lo;
  if (Elem<T>::kIsBf16 && !(span <= 3.4028235e38f)) return 2.0f * __fdiv_rn(0.5f * hi - 0.5f * lo, 15.0f);
  return __fdiv_rn(span, 15.0f);
}

// Codes and scale of a group of G rows (largest magnitude to 7, or the range with zero to 15).
// s is rounded to T first and the codes are taken against the rounded scale. A group whose scale
// rounds to zero has code = zero point; one with a NaN or an infinity has a scale that is not
// finite, and so has what it stands for. A thread takes 64 rows, so two threads of a warp share a
// group of 128 (128 values did not fit a thread's registers); 32 rows where pairs are loaded as two
// elements.
template <typename T, int G, bool ZP, bool VEC>
__global__ void __launch_bounds__(kPackThreads) w4_quantize_kernel(const __grid_constant__ W4Layout l,
                                                                   const T* __restrict__ w, void* packed) {
  using P = Pair<T>;
  using V = typename P::V;
  constexpr int kPer = VEC && G >= 64 ? 64 : 32, kSplit = G / kPer, kSeg = 32 / kSplit;
  pdl_wait_prior();
  pdl_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int part = lane / kSeg;
  const int pair = (blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5)) * kSeg + lane % kSeg;
  const int tile = pair >> 3, g = pair & 7, c = 2 * pair;
  const bool in = tile < l.n_tiles;
  for (int64_t grp = blockIdx.y; grp < l.blocks * l.units; grp += gridDim.y) {
    const int k0 = static_cast<int>(grp) * G + part * kPer;
    uint32_t v[kPer];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = (in && c < l.n && k0 + i < l.k) ? load_pair<VEC>(w, k0 + i, l.n, c) : 0u;
    const uint32_t zero = 0;
    V hi = *reinterpret_cast<const V*>(&zero), lo = hi;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const V x = *reinterpret_cast<const V*>(&v[i]);
      hi = P::max(hi, ZP ? x : __habs2(x));
      if (ZP) lo = P::min(lo, x);
    }
    uint32_t hb = *reinterpret_cast<const uint32_t*>(&hi), lb = *reinterpret_cast<const uint32_t*>(&lo);
#pragma unroll
    for (int o = kSeg; o < 32; o *= 2) {
      const uint32_t ho = __shfl_xor_sync(0xffffffffu, hb, o), lo_o = __shfl_xor_sync(0xffffffffu, lb, o);
      hi = P::max(hi, *reinterpret_cast<const V*>(&ho));
      lo = P::min(lo, *reinterpret_cast<const V*>(&lo_o));
      hb = *reinterpret_cast<const uint32_t*>(&hi), lb = *reinterpret_cast<const uint32_t*>(&lo);
    }
    if (!in) continue;
    const float2 h = Elem<T>::unpack(hb), b = Elem<T>::unpack(lb);
    uint32_t s01 = ZP ? Elem<T>::pack(w4_span_step<T>(h.x, b.x), w4_span_step<T>(h.y, b.y))
                      : Elem<T>::pack(__fdiv_rn(h.x, 7.0f), __fdiv_rn(h.y, 7.0f));
    const float2 sv = Elem<T>::unpack(s01);
    const float s[2] = {sv.x, sv.y}, low[2] = {b.x, b.y};
    float below[2], above[2], up[2];
    int z[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      up[r] = Elem<T>::kIsBf16 && s[r] < 0x1p-126f ? 0x1p24f : 1.0f;
      const float inv = s[r] > 0.0f ? __fdiv_rn(1.0f, s[r] * up[r]) : 0.0f;
      below[r] = inv * (1.0f - 0x1p-22f);
      above[r] = inv * (1.0f + 0x1p-22f);
      z[r] = 8;
      if (ZP) {
        const uint32_t q = w4_code_bits(-low[r] * up[r], below[r], above[r], kMagic, 0) - kMagicBits;
        z[r] = s[r] > 0.0f ? static_cast<int>(q > 15u ? 15u : q) : 0;
      }
    }
    const bool real = c < l.n && static_cast<int>(grp) * G < l.k;
    uint32_t z01 = ZP ? Elem<T>::pack(static_cast<float>(z[0]), static_cast<float>(z[1])) : 0u;
    if (!real) s01 = 0, z01 = 0;
    if (c + 1 >= l.n) s01 &= 0xFFFFu, z01 &= 0xFFFFu;
    if (part == 0) {
      uint32_t* sp = scale_ptr(l, packed, tile, static_cast<int>(grp), g);
      if (ZP) *reinterpret_cast<uint2*>(sp) = make_uint2(s01, z01);
      else *sp = s01;
    }
    const float mz[2] = {kMagic + static_cast<float>(z[0]), kMagic + static_cast<float>(z[1])};
    // Lowest code: rint is odd, so rint(lo / s) + z is not below 0. Highest: s is within half a step of
    // its unrounded value, so without zero points |x / s| stays below 7.5; with them two roundings can
    // make 16. A subnormal s is rounded more coarsely, and the edge's columns and rows are zeros: those
    // take every test.
    auto put = [&](auto edge) {
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        uint32_t word[kPer / 16];  // (half, j)
#pragma unroll
        for (int hj = 0; hj < kPer / 16; ++hj) {
          // the sum of the codes' bits 16^nibble apart; what 1.5 2^23 adds to it is constant
          uint32_t acc = 0u - kMagicBits * 0x11111111u;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = 16 * hj + 4 * t + i;
            const float2 f = Elem<T>::unpack(v[kk]);
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              float x = r == 0 ? f.x : f.y;
              if (edge) x *= up[r];
              uint32_t q = w4_code_bits(x, below[r], above[r], mz[r], static_cast<uint32_t>(z[r]));
              if (edge) {
                q = q < kMagicBits ? kMagicBits : q > kMagicBits + 15u ? kMagicBits + 15u : q;
                if (k0 + kk >= l.k || c + r >= l.n) q = kMagicBits;
              } else if (ZP) {
                q = q > kMagicBits + 15u ? kMagicBits + 15u : q;
              }
              acc += q * (1u << (4 * w4_nibble(r, i)));
            }
          }
          word[hj] = w4_store_word<T>(acc);
        }
        uint4* to = code_ptr(l, packed, tile, k0 / 64, g) + t;
        if constexpr (kPer == 64) *to = make_uint4(word[0], word[1], word[2], word[3]);
        else reinterpret_cast<uint2*>(to)[(k0 / 32) & 1] = make_uint2(word[0], word[1]);
      }
    };
    constexpr float kNormal = Elem<T>::kIsBf16 ? 0x1p-126f : 0x1p-14f;
    const bool plain = s[0] >= kNormal && s[1] >= kNormal && s[0] < 1e30f && s[1] < 1e30f;  // false for NaN
    if (plain && c + 1 < l.n && k0 + kPer <= l.k) put(std::false_type{});
    else put(std::true_type{});
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

// s (q - z), rounded once to T, in packed arithmetic
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
      W4Exact<T> dq;
      dq.set(sp[0], l.zeros ? sp[1] : 0u, l.zeros != 0);
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          uint32_t r[4];  // rows (0, 1) and (2, 3) of column 0, then of column 1
          dq.word(h == 0 ? (j == 0 ? u[t].x : u[t].y) : (j == 0 ? u[t].z : u[t].w), r);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int k = k0 + 16 * j + 4 * t + i;
            if (k < l.k) store_pair<VEC>(w, k, l.n, at.c, __byte_perm(r[i >> 1], r[2 + (i >> 1)], (i & 1) ? 0x7632 : 0x5410));
          }
        }
    }
  }
}

// Launch over column pairs (x) and 64-row parts or groups (y, with a stride past the grid's limit).
// `out` / `bytes`: what the launch writes.
template <typename... KArgs, typename... Args>
int launch_pack(void (*kern)(KArgs...), const W4Layout& l, int rows, int threads_per_pair, cudaStream_t s,
                const PdlIo& io, Args... args) {
  cudaLaunchConfig_t cfg = {};
  const int pairs = l.n_tiles * 8 * threads_per_pair;
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
  return launch_pack(kern, l, l.blocks * l.units, vec ? (G > 64 ? 2 : 1) : G / 32, s, io, w, packed);
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
  return launch_pack(kern, l, l.blocks * 2, 1, s, io, codes, static_cast<const T*>(scales), zeros, packed);
}

template <typename T>
int unpack_t(const W4Layout& l, const void* packed, uint8_t* codes, void* scales, uint8_t* zeros, cudaStream_t s) {
  const uint64_t ng = static_cast<uint64_t>((l.k + l.group - 1) / l.group) * l.n;
  PdlIo io;
  io.add(PdlIo::kWrite, codes, static_cast<uint64_t>(l.k) * l.n);
  io.add(PdlIo::kWrite, scales, ng * 2);
  io.add(PdlIo::kWrite, zeros, ng);
  auto kern = scales != nullptr && even_rows(l, scales) ? &w4_unpack_kernel<T, true> : &w4_unpack_kernel<T, false>;
  return launch_pack(kern, l, l.blocks * 2, 1, s, io, const_cast<void*>(packed), codes, static_cast<T*>(scales), zeros);
}

template <typename T>
int dequantize_t(const W4Layout& l, const void* packed, void* w, cudaStream_t s) {
  PdlIo io;
  io.add(PdlIo::kWrite, w, static_cast<uint64_t>(l.k) * l.n * 2);
  auto kern = even_rows(l, w) ? &w4_dequantize_kernel<T, true> : &w4_dequantize_kernel<T, false>;
  return launch_pack(kern, l, l.blocks * 2, 1, s, io, const_cast<void*>(packed), static_cast<T*>(w));
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
