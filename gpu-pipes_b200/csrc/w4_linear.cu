// Products with 4-bit weights for few rows: out [m, N] = act(x [m, K] W + b), W = s (q - z) (w4.cuh).
//
// With few rows the time is the weights' bytes (half a byte each), so the kernel is a stream over
// the packed codes. The matrix instruction is mma.sync m16n8k16 with the WEIGHTS as its 16-row
// operand (16 columns of W) and up to 8 rows of x as its 8-column operand: a warp turns 1,024
// weights into instruction operands with about 1.3 integer and half instructions each, one to
// eight rows cost the same, and the sums are fp32. (tcgen05 takes its weights from shared memory,
// which for so few rows only adds a store and a load per weight.) The codes enter as the exact
// integers q - z; the group's scale multiplies the fp32 sum of its 32 or 64 products, so no weight
// is rounded.
//
//   - A CTA of 16 warps owns a slice of K (one of `ck` CTAs of a cluster does; ck = 1: all of it),
//     keeps its part of the x rows in shared memory and goes over column tiles of 16. `ws` warps
//     share a tile, each taking every ws-th 64-row block, so together they read whole stretches.
//   - Every lane copies its own 16 bytes of codes (and its scales) into a private ring of kDepth
//     slots with cp.async and reads back only what it copied: the ring needs no barrier, and the
//     loads of the next tiles are in flight while the sums of this one are joined.
//   - The warps' sums are joined in shared memory, the CTAs' through distributed shared memory,
//     both in a fixed order: results do not depend on timing.
#include <climits>

#include "../../include/gpipes.h"
#include "chain_registry.h"
#include "w4.cuh"

namespace gp {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kDepth = 8;           // ring slots per warp
constexpr int kPartStride = 20;     // floats per row of a warp's 16 x rows sums: conflict-free float2 stores
constexpr int kMaxCluster = 8;

struct W4RowsArgs {
  W4Layout l;
  const void* x;
  const void* packed;
  const void* bias;
  void* out;
  int64_t m;
  int act;
  int ck;            // CTAs of a cluster, along K
  int slice;         // 64-row blocks of a CTA
  int ws;            // warps that share a column tile
  int iters;         // column tile groups per cluster
  int rows;          // x rows of a pass (at most 8 TT)
  int x_stride;      // bytes between x rows in shared memory
};

// exact forms: with few rows the epilogue costs nothing, so nothing is approximated
__device__ __forceinline__ float act_exact(int act, float v) {
  switch (act) {
    case GP_ACT_RELU: return v > 0.0f ? v : (v == v ? 0.0f : v);
    case GP_ACT_GELU_TANH: return 0.5f * v * (1.0f + tanhf(0.7978845608028654f * fmaf(0.044715f * v, v * v, v)));
    case GP_ACT_SILU: return v / (1.0f + expf(-v));
    case GP_ACT_SIGMOID: return 1.0f / (1.0f + expf(-v));
    default: return v;
  }
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (Elem<T>::kIsBf16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}

// TT: tiles of 8 x rows. UNIT: rows of W per scale step (32 or 64; groups of 128 use 64).
template <typename T, int TT, int UNIT, bool ZP, typename OutT>
__global__ void __launch_bounds__(kThreads, 1) w4_rows_kernel(const __grid_constant__ W4RowsArgs a) {
  constexpr int kUnits = 64 / UNIT;
  constexpr int kScale = ZP ? 8 : 4;                          // bytes of scales per lane and unit
  constexpr int kSlot = 32 * (16 + kUnits * kScale);          // bytes of a ring slot
  constexpr int kPart = TT * 8 * kPartStride;                 // floats of a warp's sums
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* ring = smem;                                       // [kWarps][kDepth][kSlot]
  float* part = reinterpret_cast<float*>(ring + kWarps * kDepth * kSlot);  // [2][kWarps][kPart]
  float* red = part + 2 * kWarps * kPart;                     // [2][TT * 128 * kWarps / ws] at most, clusters only
  const int np = kWarps / a.ws;                               // tiles at a time
  const int outs = np * TT * 128;                             // sums of a tile group
  uint8_t* xs = reinterpret_cast<uint8_t*>(red + (a.ck > 1 ? 2 * outs : 0));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = a.ck > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int cluster = blockIdx.x / a.ck, clusters = gridDim.x / a.ck;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * a.rows;
  const int rows = static_cast<int>(a.m - row0 < a.rows ? a.m - row0 : a.rows);
  const int b0 = rank * a.slice;
  const int nb = min(a.slice, a.l.k_blocks - b0);             // blocks of this CTA (may be <= 0)
  const int sub = warp % a.ws, slot_tile = warp / a.ws;
  const int steps = (a.slice + a.ws - 1) / a.ws;              // blocks of a warp per tile

  const uint8_t* codes = static_cast<const uint8_t*>(a.packed);
  const uint8_t* scales = codes + a.l.scale_off;
  const uint32_t my_ring = smem_u32(ring) + warp * (kDepth * kSlot);

  // the step that is loaded next: tile group it_i, block b_i of this warp's
  int it_i = 0, b_i = 0;
  auto src = [&](int it, int b, const uint8_t*& c, const uint8_t*& s) {
    const int tile = (cluster + it * clusters) * np + slot_tile;
    const int rel = sub + b * a.ws;
    if (it >= a.iters || tile >= a.l.n_tiles || rel >= nb) return false;
    const int blk = b0 + rel;
    c = codes + (static_cast<int64_t>(tile) * a.l.k_blocks + blk) * 512 + lane * 16;
    s = scales + (static_cast<int64_t>(tile) * a.l.groups + blk * 64 / a.l.group) * (8 * kScale) + g * kScale;
    return true;
  };
  auto issue = [&](int slot) {
    const uint8_t *c, *s;
    if (src(it_i, b_i, c, s)) {
      const uint32_t d = my_ring + slot * kSlot;
      cp_async<16>(d + lane * 16, c);
#pragma unroll
      for (int u = 0; u < kUnits; ++u) cp_async<kScale>(d + 512 + (u * 32 + lane) * kScale, s + u * 8 * kScale);
    }
    cp_commit();
    if (++b_i == steps) b_i = 0, ++it_i;
  };

  // The first codes go into L2 while the previous kernel of the stream drains (a hint: nothing is
  // read into the program before the wait).
  {
    const uint8_t *c, *s;
    for (int i = 0, it = 0, b = 0; i < kDepth; ++i) {
      if ((lane & 7) == 0 && src(it, b, c, s)) asm volatile("prefetch.global.L2 [%0];" ::"l"(c));
      if (++b == steps) b = 0, ++it;
    }
  }
  pdl_wait_prior();
  pdl_launch_dependents();
#pragma unroll
  for (int i = 0; i < kDepth - 1; ++i) issue(i);

  // x rows of this CTA's slice; zero past K
  {
    const int chunks = a.slice * 8;  // 16-byte pieces of a row
    for (int i = threadIdx.x; i < rows * chunks; i += kThreads) {
      const int r = i / chunks, c = i % chunks;
      const int k = b0 * 64 + c * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (k < a.l.k) v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (row0 + r) * a.l.k + k);
      *reinterpret_cast<uint4*>(xs + r * a.x_stride + c * 16) = v;
    }
  }
  __syncthreads();
  // every CTA of the cluster runs before one writes into another's shared memory
  if (a.ck > 1) cluster_sync_all();

  const uint8_t* xr[TT];
  bool live[TT];
#pragma unroll
  for (int i = 0; i < TT; ++i) {
    live[i] = i * 8 + g < rows;
    xr[i] = xs + (live[i] ? i * 8 + g : 0) * a.x_stride + t * 16;
  }

  int slot = 0;
  for (int it = 0; it < a.iters; ++it) {
    float acc[TT][4];
#pragma unroll
    for (int i = 0; i < TT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
    const int tile0 = (cluster + it * clusters) * np;
    const bool has_tile = tile0 + slot_tile < a.l.n_tiles;
    for (int b = 0; b < steps; ++b) {
      issue((slot + kDepth - 1) % kDepth);
      cp_wait<kDepth - 1>();
      const int rel = sub + b * a.ws;
      if (has_tile && rel < nb) {
        const uint32_t d = my_ring + slot * kSlot;
        uint32_t w[4];
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(d + lane * 16) : "memory");
        float sum[TT][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int u = h * kUnits / 2;
          uint32_t s01, z01 = 0, c0 = W4Deq<T>::kC0, c1 = W4Deq<T>::kC1;
          if constexpr (ZP) {
            asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(s01), "=r"(z01)
                         : "r"(d + 512 + (u * 32 + lane) * kScale) : "memory");
            W4Deq<T>::consts(z01, c0, c1);
          } else {
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(s01) : "r"(d + 512 + (u * 32 + lane) * kScale) : "memory");
          }
          if (kUnits == 2 || h == 0)
#pragma unroll
            for (int i = 0; i < TT; ++i) sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = 0.0f;
          uint32_t p0[4], p1[4];
          W4Deq<T>::pairs(w[2 * h], c0, c1, p0);
          W4Deq<T>::pairs(w[2 * h + 1], c0, c1, p1);
#pragma unroll
          for (int i = 0; i < TT; ++i) {
            uint4 xv = make_uint4(0, 0, 0, 0);
            if (live[i]) xv = *reinterpret_cast<const uint4*>(xr[i] + rel * 128 + h * 64);
            mma16816<T>(sum[i], p0, xv.x, xv.y);
            mma16816<T>(sum[i], p1, xv.z, xv.w);
          }
          if (kUnits == 2 || h == 1) {
            const float2 s = Elem<T>::unpack(s01);
#pragma unroll
            for (int i = 0; i < TT; ++i) {
              acc[i][0] = fmaf(s.x, sum[i][0], acc[i][0]);
              acc[i][1] = fmaf(s.x, sum[i][1], acc[i][1]);
              acc[i][2] = fmaf(s.y, sum[i][2], acc[i][2]);
              acc[i][3] = fmaf(s.y, sum[i][3], acc[i][3]);
            }
          }
        }
      }
      slot = slot + 1 == kDepth ? 0 : slot + 1;
    }
    // join: part[warp][row][column]; a buffer is written again two groups on, after the next
    // group's barrier, when everyone has read it
    float* pb = part + (it & 1) * (kWarps * kPart);
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      float* p = pb + warp * kPart + (i * 8 + 2 * t) * kPartStride + 2 * g;
      *reinterpret_cast<float2*>(p) = make_float2(acc[i][0], acc[i][2]);
      *reinterpret_cast<float2*>(p + kPartStride) = make_float2(acc[i][1], acc[i][3]);
    }
    __syncthreads();
    auto warps_sum = [&](int o) {
      const int tl = o / (TT * 128), r = (o >> 4) % (TT * 8), n = o & 15;
      const float* p = pb + tl * a.ws * kPart + r * kPartStride + n;
      float v = 0.0f;
      for (int i = 0; i < a.ws; ++i) v += p[i * kPart];
      return v;
    };
    auto finish = [&](int o, float v) {
      const int tl = o / (TT * 128), r = (o >> 4) % (TT * 8);
      const int64_t n = static_cast<int64_t>(tile0 + tl) * 16 + (o & 15);
      if (r >= rows || n >= a.l.n) return;
      if (a.bias != nullptr) v += Elem<T>::to_f(static_cast<const T*>(a.bias)[n]);
      v = act_exact(a.act, v);
      const int64_t at = (row0 + r) * a.l.n + n;
      if constexpr (sizeof(OutT) == 4) {
        static_cast<float*>(a.out)[at] = v;
      } else {
        const uint32_t u = Elem<T>::pack(v, 0.0f);
        static_cast<uint16_t*>(a.out)[at] = static_cast<uint16_t>(u);
      }
    };
    if (a.ck == 1) {
      for (int o = threadIdx.x; o < outs; o += kThreads)
        if ((o >> 4) % (TT * 8) < rows) finish(o, warps_sum(o));
    } else {
      // CTA r of the cluster finishes outputs [r outs / ck, (r + 1) outs / ck): the others send
      // their sums there; the buffer alternates like part, with the cluster's barrier in between
      const int own = outs / a.ck;
      float* rb = red + (it & 1) * outs;
      for (int o = threadIdx.x; o < outs; o += kThreads)
        if ((o >> 4) % (TT * 8) < rows)
          st_cluster_f32(mapa_shared(smem_u32(rb + rank * own + o % own), static_cast<uint32_t>(o / own)), warps_sum(o));
      cluster_sync_all();
      for (int o = threadIdx.x; o < own; o += kThreads) {
        const int oo = rank * own + o;
        if ((oo >> 4) % (TT * 8) >= rows) continue;
        float v = 0.0f;
        for (int i = 0; i < a.ck; ++i) v += rb[i * own + o];
        finish(oo, v);
      }
    }
  }
  // cp.async copies still in flight are none: every group past the last step is empty
}

constexpr int rows_slot(int units, bool zp) { return 32 * (16 + units * (zp ? 8 : 4)); }

// Shared memory of a CTA: ring, warps' sums, clusters' sums, x rows
int64_t rows_smem(int tt, int units, bool zp, int ck, int ws, int rows, int x_stride) {
  const int64_t outs = static_cast<int64_t>(kWarps / ws) * tt * 128;
  return static_cast<int64_t>(kWarps) * kDepth * rows_slot(units, zp) + 2ll * kWarps * tt * 8 * kPartStride * 4 +
         (ck > 1 ? 2 * outs * 4 : 0) + static_cast<int64_t>(rows) * x_stride;
}

template <typename T, int TT, int UNIT, bool ZP, typename OutT>
int rows_launch(const W4RowsArgs& a, int smem, int clusters, int64_t row_tiles, cudaStream_t s, const PdlIo& io) {
  static unsigned long long done_mask = 0;
  auto kern = &w4_rows_kernel<T, TT, UNIT, ZP, OutT>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), kSmemLimit, &done_mask);
  if (rc != GP_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(clusters * a.ck), static_cast<unsigned>(row_tiles), 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = static_cast<size_t>(smem);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int na = 0;
  if (a.ck > 1) {
    attr[na].id = cudaLaunchAttributeClusterDimension;
    attr[na].val.clusterDim.x = static_cast<unsigned>(a.ck);
    attr[na].val.clusterDim.y = 1;
    attr[na].val.clusterDim.z = 1;
    ++na;
  }
  if (pdl_enabled()) {
    attr[na].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[na].val.programmaticStreamSerializationAllowed = 1;
    ++na;
  }
  cfg.attrs = attr;
  cfg.numAttrs = static_cast<unsigned>(na);
  PdlLaunch pdl(s);
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, a);
  pdl.record(io);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GP_OK : set_error(GP_ERR_CUDA, "w4 linear launch: %s", cudaGetErrorString(e));
}

template <typename T, int TT, typename OutT>
int rows_dispatch(const W4RowsArgs& a, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  if (a.l.group == 32)
    return a.l.zeros ? rows_launch<T, TT, 32, true, OutT>(a, smem, clusters, rt, s, io)
                     : rows_launch<T, TT, 32, false, OutT>(a, smem, clusters, rt, s, io);
  return a.l.zeros ? rows_launch<T, TT, 64, true, OutT>(a, smem, clusters, rt, s, io)
                   : rows_launch<T, TT, 64, false, OutT>(a, smem, clusters, rt, s, io);
}

template <typename T, typename OutT>
int rows_tt(const W4RowsArgs& a, int tt, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  return tt == 1 ? rows_dispatch<T, 1, OutT>(a, smem, clusters, rt, s, io)
                 : rows_dispatch<T, 2, OutT>(a, smem, clusters, rt, s, io);
}

}  // namespace

int launch_w4_linear(const W4Layout& l, int dtype, int64_t m, const void* x, const void* packed, const void* bias,
                     int act, void* out, bool out_f32, cudaStream_t s, int sm_count) {
  W4RowsArgs a;
  a.l = l;
  a.x = x;
  a.packed = packed;
  a.bias = bias;
  a.out = out;
  a.act = act;
  const int units = l.group == 32 ? 2 : 1;
  // Split of the work: ck CTAs of a cluster along K, ws warps per column tile. A tile group costs
  // its warps' blocks plus a join (about one block's time within a CTA, about three more across a
  // cluster); the fewest rounds of that over the GPU's SMs win. A pass takes up to 16 rows, fewer
  // where they would not fit in shared memory even spread over eight CTAs.
  int per_pass = m > 8 ? 16 : 8;
  for (;; per_pass /= 2) {
    const int rows = static_cast<int>(m < per_pass ? m : per_pass), tt = per_pass > 8 ? 2 : 1;
    int64_t best = LLONG_MAX;
    for (int ck = 1; ck <= kMaxCluster; ck *= 2) {
      const int slice = (l.k_blocks + ck - 1) / ck;
      if (ck > 1 && (ck - 1) * slice >= l.k_blocks) break;  // a CTA without work
      for (int ws = 1; ws <= kWarps; ws *= 2) {
        if (ws > 1 && ws / 2 >= slice) break;
        if (rows_smem(tt, units, l.zeros != 0, ck, ws, rows, slice * 128 + 64) > kSmemLimit) continue;
        const int groups = (l.n_tiles + kWarps / ws - 1) / (kWarps / ws);
        const int clusters = groups < sm_count / ck ? groups : sm_count / ck;
        const int64_t iters = (groups + clusters - 1) / clusters;
        const int64_t cost = iters * ((slice + ws - 1) / ws + 1 + (ck > 1 ? 3 : 0));
        if (cost >= best) continue;
        best = cost;
        a.ck = ck;
        a.slice = slice;
        a.ws = ws;
        a.iters = static_cast<int>(iters);
      }
    }
    if (best != LLONG_MAX) break;
    if (per_pass == 1) return set_error(GP_ERR_UNSUPPORTED, "w4 linear: K = %d", l.k);
  }
  a.rows = per_pass;
  a.x_stride = a.slice * 128 + 64;
  const int tt = per_pass > 8 ? 2 : 1;
  const int smem = static_cast<int>(rows_smem(tt, units, l.zeros != 0, a.ck, a.ws,
                                              static_cast<int>(m < per_pass ? m : per_pass), a.x_stride));
  const int groups = (l.n_tiles + kWarps / a.ws - 1) / (kWarps / a.ws);
  const int clusters = groups < sm_count / a.ck ? groups : sm_count / a.ck;
  PdlIo io;
  io.add(PdlIo::kWrite, out, static_cast<uint64_t>(m) * l.n * (out_f32 ? 4 : 2));
  // the grid's y dimension holds 65,535 row tiles; longer inputs go in several launches
  const int64_t step = 65535ll * per_pass;
  for (int64_t r0 = 0; r0 < m; r0 += step) {
    W4RowsArgs c = a;
    c.m = m - r0 < step ? m - r0 : step;
    c.x = static_cast<const char*>(x) + r0 * l.k * 2;
    c.out = static_cast<char*>(out) + r0 * l.n * (out_f32 ? 4 : 2);
    const int64_t rt = (c.m + per_pass - 1) / per_pass;
    int rc;
    if (dtype == GP_BF16)
      rc = out_f32 ? rows_tt<__nv_bfloat16, float>(c, tt, smem, clusters, rt, s, io)
                   : rows_tt<__nv_bfloat16, __nv_bfloat16>(c, tt, smem, clusters, rt, s, io);
    else
      rc = out_f32 ? rows_tt<__half, float>(c, tt, smem, clusters, rt, s, io)
                   : rows_tt<__half, __half>(c, tt, smem, clusters, rt, s, io);
    if (rc != GP_OK) return rc;
    count_launches(1);
  }
  return GP_OK;
}

}  // namespace gp
