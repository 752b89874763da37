// Products with 4-bit weights for few rows: out [m, N] = act(x [m, K] W + b), W = s (q - z) (w4.cuh).
//
// With few rows the time is the weights' bytes (half a byte each), and what stands between them and
// the memory's rate is the number of instructions per weight. So:
//   - The matrix instruction is mma.sync m16n8k16 with the WEIGHTS as its 16-row operand (16 columns
//     of W) and up to 8 rows of x as its 8-column operand; one to eight rows cost the same and the
//     sums are fp32. (tcgen05 takes 16-bit weights from shared memory, which for so few rows only
//     adds a store and a load per weight.)
//   - A code becomes an operand with one mask (w4.cuh): the operand is q plus a constant, scaled by a
//     power of two. sum_k x (q - z) = sum_k x (q + c) - (c + z) sum_k x, and the second term starts
//     the accumulator; the sums of x over each group are taken once per CTA. The group's scale
//     multiplies the fp32 sum, so no weight is rounded. A first form that subtracted z from each
//     weight, took codes through a cp.async ring and divided to find the group ran 174 instructions
//     per 1,024 weights and 57 us at 1 x 8192 x 28672.
//
//   - A CTA of 16 warps owns a slice of K (one of `ck` CTAs of a cluster does; ck = 1: all of it),
//     keeps its part of the x rows in shared memory and goes over column tiles of 16. `ws` warps
//     share a tile, each taking every ws-th 128-row block, so together they read whole stretches.
//   - Every warp streams its blocks through a ring of its own in shared memory: one lane starts the
//     bulk copies (a block's codes and its scales, contiguous both), the warp waits on the slot's
//     mbarrier, takes the slot into registers and hands it back at once. The loads of the next tiles
//     go on while the sums of this one are joined. (Loads straight to registers, four blocks ahead,
//     ended up waiting for one another: 40 us at 1 x 8192 x 28672.)
//   - The warps' sums are joined in shared memory, the CTAs' through distributed shared memory,
//     both in a fixed order: results do not depend on timing.
#include <climits>

#include "../../include/gpipes.h"
#include "chain_registry.h"
#include "w4.cuh"

namespace gp {
namespace {

// Warps of a CTA (one CTA per SM): kWarps turn codes into sums, kJoinWarps add the sums up and store.
constexpr int kWarps = 16;
constexpr int kJoinWarps = 4;
constexpr int kJoiners = 32 * kJoinWarps;
constexpr int kThreads = 32 * (kWarps + kJoinWarps);
constexpr int kPartStride = 20;     // floats per row of a warp's 16 x rows sums: conflict-free float2 stores
constexpr int kMaxCluster = 8;
constexpr int kMaxDepth = 8;        // ring slots per warp
constexpr int kMinDepth = 3;
constexpr int kRowsSmem = kSmemLimit - 3072;  // dynamic: the barriers are static
constexpr int kZeroBytes = 256;     // zeros in shared memory, read in place of absent x rows

struct W4RowsArgs {
  W4Layout l;
  const void* x;
  const void* packed;
  const void* bias;
  void* out;
  int64_t m;
  int act;
  int ck;            // CTAs of a cluster, along K
  int slice;         // k-blocks of a CTA
  int run;           // k-blocks of a ring slot (1 or 2), neighbours in the packed codes
  int ws;            // warps that share a column tile
  int iters;         // column tile groups per cluster
  int rows;          // x rows of a pass (at most 8 TT)
  int x_stride;      // bytes between x rows in shared memory
  int depth;         // ring slots per warp
  int* status;
  unsigned long long timeout_ns;
  int inject;        // fault injection: 1 = no block is ever loaded
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

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

__device__ __forceinline__ uint4 lds128(uint32_t p) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(p) : "memory");
  return v;
}

template <int W>
__device__ __forceinline__ void lds_words(uint32_t p, uint32_t (&v)[W]) {
  if constexpr (W == 1) {
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v[0]) : "r"(p) : "memory");
  } else if constexpr (W == 2) {
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v[0]), "=r"(v[1]) : "r"(p) : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < W; i += 4) {
      const uint4 u = lds128(p + 4 * i);
      v[i] = u.x, v[i + 1] = u.y, v[i + 2] = u.z, v[i + 3] = u.w;
    }
  }
}

// Named barriers of the CTA (0 is __syncthreads): waiting, and arriving without waiting.
__device__ __forceinline__ void bar_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id) {
  __syncwarp();
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(kThreads) : "memory");
}
constexpr int kBarFull = 1, kBarFree = 3;  // + buffer 0 / 1 of the warps' sums

// 16 bytes into the shared memory of a CTA of the cluster, counted on that CTA's mbarrier: the
// reader needs no other signal and the writer no fence.
__device__ __forceinline__ void st_async_f32x4(uint32_t addr, uint32_t bar, float4 v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%2, %3, %4, %5}, [%1];" ::"r"(addr),
               "r"(bar), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// TT: tiles of 8 x rows. UNITS: groups per k-block of 128.
template <typename T, int TT, int UNITS, bool ZP, typename OutT>
__global__ void __launch_bounds__(kThreads, 1) w4_rows_kernel(const __grid_constant__ W4RowsArgs a) {
  constexpr int kWords = UNITS * (ZP ? 2 : 1);                // scale words of a lane per block
  constexpr int kPart = TT * 8 * kPartStride;                 // floats of a warp's sums
  constexpr int kScaleBytes = 32 * kWords;                    // scales of a block
  constexpr int kSlot = kW4BlockBytes + kScaleBytes;
  constexpr float kUnit0 = W4Deq<T>::unit(0), kUnit1 = W4Deq<T>::unit(1);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kWarps + kJoinWarps][kMaxDepth];
  __shared__ __align__(8) uint64_t red_full[2];
  __shared__ int abort_flag, join_abort;
  float* part = reinterpret_cast<float*>(smem + kWarps * a.depth * a.run * kSlot);  // [2][kWarps][kPart]
  const int np = kWarps / a.ws;                               // tiles at a time
  const int outs = np * TT * 128;                             // sums of a tile group
  float* red = part + 2 * kWarps * kPart;                     // [2][outs], clusters only
  float* xsum = red + (a.ck > 1 ? 2 * outs : 0);              // [slice * UNITS][8 TT]
  uint8_t* zeros = reinterpret_cast<uint8_t*>(xsum + a.slice * UNITS * 8 * TT);
  uint8_t* xs = zeros + kZeroBytes;                           // [rows][x_stride]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = a.ck > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int cluster = blockIdx.x / a.ck, clusters = gridDim.x / a.ck;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * a.rows;
  const int rows = static_cast<int>(a.m - row0 < a.rows ? a.m - row0 : a.rows);
  const int b0 = rank * a.slice;
  const int nb = min(a.slice, a.l.blocks - b0);               // blocks of this CTA
  const int sub = warp % a.ws, slot_tile = warp / a.ws;

  // the run of blocks that is loaded next: tile and first block (relative to the slice) of this
  // warp's; a warp without a block in the slice (and a joining one) loads nothing
  const int tile_step = clusters * np, lead = sub * a.run, stride = a.ws * a.run, slot_bytes = a.run * kSlot;
  int ld_tile = warp < kWarps && lead < nb ? cluster * np + slot_tile : INT_MAX, ld_rel = lead, ld_slot = 0;
  const uint32_t ring = smem_u32(smem) + warp * a.depth * slot_bytes, bars = smem_u32(full[warp]);
  const uint8_t* const codes0 = static_cast<const uint8_t*>(a.packed) + static_cast<int64_t>(b0) * kW4BlockBytes;
  const uint8_t* const scales0 = static_cast<const uint8_t*>(a.packed) + a.l.scale_off + static_cast<int64_t>(b0) * kScaleBytes;
  int64_t ld_cell = static_cast<int64_t>(cluster * np + slot_tile) * a.l.blocks;
  // one lane: the next run of the warp's sequence into the next slot
  auto load = [&] {
    if (ld_tile >= a.l.n_tiles || a.inject != 0) return;
    const uint32_t bar = bars + ld_slot * 8, dst = ring + ld_slot * slot_bytes;
    const int n = min(a.run, nb - ld_rel);
    mbar_arrive_expect_tx(bar, n * kSlot);
    bulk_load(dst, codes0 + (ld_cell + ld_rel) * kW4BlockBytes, n * kW4BlockBytes, bar);
    bulk_load(dst + a.run * kW4BlockBytes, scales0 + (ld_cell + ld_rel) * kScaleBytes, n * kScaleBytes, bar);
    ld_slot = ld_slot + 1 == a.depth ? 0 : ld_slot + 1;
    ld_rel += stride;
    if (ld_rel >= nb) {
      ld_rel = lead;
      ld_tile = tile_step < a.l.n_tiles - ld_tile ? ld_tile + tile_step : INT_MAX;
      ld_cell += static_cast<int64_t>(tile_step) * a.l.blocks;
    }
  };

  // The first codes go into L2 while the previous kernel of the stream drains (a hint: nothing is
  // read into the program before the wait).
  if (ld_tile < a.l.n_tiles)
    for (int i = 0; i < a.depth && lead + i * stride < nb; ++i) {
      const int n = min(a.run, nb - lead - i * stride);
      if (lane < 8 * n)
        asm volatile("prefetch.global.L2 [%0];" ::"l"(codes0 + (ld_cell + lead + i * stride) * kW4BlockBytes + lane * 128));
    }
  if (lane == 0 && warp < kWarps)
    for (int i = 0; i < a.depth; ++i) mbar_init(bars + i * 8, 1);
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&red_full[0]), 1);
    mbar_init(smem_u32(&red_full[1]), 1);
    abort_flag = join_abort = 0;
  }
  if (lane == 0) fence_mbar_init();
  pdl_wait_prior();
  pdl_launch_dependents();
  if (lane == 0)
    for (int i = 0; i < a.depth; ++i) load();

  // x rows of this CTA's slice (zero past K) and their sums over each group. Sixteen lanes hold a
  // block of a row; absent rows have sums of zero and are read from the zeros.
  if (threadIdx.x < kZeroBytes / 16) reinterpret_cast<uint4*>(zeros)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  {
    const int pieces = a.slice * 16;  // 16-byte pieces of a row
    for (int i = threadIdx.x; i < (8 * TT - rows) * a.slice * UNITS; i += kThreads) {
      const int dead = 8 * TT - rows;
      xsum[i / dead * (8 * TT) + rows + i % dead] = 0.0f;
    }
    for (int i0 = 0; i0 < rows * pieces; i0 += kThreads) {
      const int i = i0 + threadIdx.x;
      const int r = i / pieces, c = i % pieces;
      const int k = b0 * kW4Block + c * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < rows && k < a.l.k) v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.x) + (row0 + r) * a.l.k + k);
      if (r < rows) *reinterpret_cast<uint4*>(xs + r * a.x_stride + c * 16) = v;
      const float2 f0 = Elem<T>::unpack(v.x), f1 = Elem<T>::unpack(v.y), f2 = Elem<T>::unpack(v.z), f3 = Elem<T>::unpack(v.w);
      float sum = ((f0.x + f0.y) + (f1.x + f1.y)) + ((f2.x + f2.y) + (f3.x + f3.y));
#pragma unroll
      for (int o = 1; o < 16 / UNITS; o *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (r < rows && c % (16 / UNITS) == 0) xsum[(c / (16 / UNITS)) * (8 * TT) + r] = sum;
    }
  }
  __syncthreads();
  // every CTA of the cluster runs before one writes into another's shared memory
  if (a.ck > 1) cluster_sync_all();

  const WaitCtx wctx{a.status, &abort_flag, a.timeout_ns};
  int slot = 0, phase = 0;
  bool ok = true;
  if (warp >= kWarps) {
    // ---- joining: part[warp][row][column] of a tile group, summed over its warps (and CTAs)
    const int j = threadIdx.x - 32 * kWarps;
    // Sums go four neighbouring columns at a time: quad q is tile q / (32 TT), row (q / 4) % (8 TT),
    // columns 4 (q % 4) .. + 3. CTA r of a cluster finishes quads [r own, (r + 1) own).
    // The wait for another CTA has its own abort flag: a lost copy of codes ends no join, whose sums
    // are all sent and so arrive before any CTA leaves.
    const WaitCtx jctx{a.status, &join_abort, a.timeout_ns};
    const int quads = outs / 4, own = quads / a.ck;
    const bool vec = a.l.n % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (4 * sizeof(OutT)) == 0;
    for (int it = 0; it < a.iters; ++it) {
      const int tile0 = (cluster + it * clusters) * np, buf = it & 1;
      const float* pb = part + buf * (kWarps * kPart);
      auto row_of = [&](int q) { return (q >> 2) % (TT * 8); };
      auto warps_sum = [&](int q) {
        const float* p = pb + q / (TT * 32) * a.ws * kPart + row_of(q) * kPartStride + 4 * (q & 3);
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int i = 0; i < a.ws; ++i) {
          const float4 u = *reinterpret_cast<const float4*>(p + i * kPart);
          v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
        }
        return v;
      };
      auto finish = [&](int q, float4 u) {
        const int64_t n = static_cast<int64_t>(tile0 + q / (TT * 32)) * 16 + 4 * (q & 3);
        if (n >= a.l.n) return;
        float v[4] = {u.x, u.y, u.z, u.w};
        const int live = a.l.n - n < 4 ? static_cast<int>(a.l.n - n) : 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (a.bias != nullptr && i < live) v[i] += Elem<T>::to_f(static_cast<const T*>(a.bias)[n + i]);
          v[i] = act_exact(a.act, v[i]);
        }
        OutT* to = static_cast<OutT*>(a.out) + (row0 + row_of(q)) * a.l.n + n;
        if constexpr (sizeof(OutT) == 4) {
          if (vec) {
            *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
            for (int i = 0; i < live; ++i) to[i] = v[i];
          }
        } else {
          const uint32_t lo = Elem<T>::pack(v[0], v[1]), hi = Elem<T>::pack(v[2], v[3]);
          if (vec) {
            *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
          } else {
            uint16_t* h = reinterpret_cast<uint16_t*>(to);
            const uint16_t e[4] = {static_cast<uint16_t>(lo), static_cast<uint16_t>(lo >> 16), static_cast<uint16_t>(hi),
                                   static_cast<uint16_t>(hi >> 16)};
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < live) h[i] = e[i];
          }
        }
      };
      bar_sync(kBarFull + buf);
      if (a.ck == 1) {
        for (int q = j; q < quads; q += kJoiners)
          if (row_of(q) < rows) finish(q, warps_sum(q));
        if (it + 2 < a.iters) bar_arrive(kBarFree + buf);
      } else {
        // A buffer of sums is written again two groups on. The sender has then received the group in
        // between from the buffer's reader, whose threads all passed a barrier after their reads.
        const uint32_t bar = smem_u32(&red_full[buf]), to = smem_u32(red + buf * outs) + rank * own * 16;
        if (j == 0) mbar_arrive_expect_tx(bar, outs * 4);
        for (int q = j; q < quads; q += kJoiners) {
          const uint32_t dst = static_cast<uint32_t>(q / own);
          st_async_f32x4(mapa_shared(to + q % own * 16, dst), mapa_shared(bar, dst), warps_sum(q));
        }
        if (it + 2 < a.iters) bar_arrive(kBarFree + buf);
        if (!mbar_wait<true>(bar, (it >> 1) & 1, jctx, kDevTimeoutEpilogue)) continue;
        for (int o = j; o < own; o += kJoiners) {
          if (row_of(rank * own + o) >= rows) continue;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          for (int i = 0; i < a.ck; ++i) {
            const float4 u = *reinterpret_cast<const float4*>(red + buf * outs + (i * own + o) * 4);
            v.x += u.x, v.y += u.y, v.z += u.z, v.w += u.w;
          }
          finish(rank * own + o, v);
        }
      }
    }
  } else {
    // ---- codes to sums
    uint32_t xr[TT], xmask[TT];
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const bool live = i * 8 + g < rows;
      xr[i] = smem_u32(live ? xs + (i * 8 + g) * a.x_stride : zeros) + t * 16;
      xmask[i] = live ? 0xffffffffu : 0u;
    }
    float acc[TT][4];
    // block `i` of the run in ring slot d; rel: its place in the slice
    auto block = [&](uint32_t d, int i, int rel) {
      const uint4 cbuf[2] = {lds128(d + i * kW4BlockBytes + lane * 16),
                             lds128(d + i * kW4BlockBytes + kW4BlockBytes / 2 + lane * 16)};
      uint32_t sbuf[kWords];
      lds_words<kWords>(d + a.run * kW4BlockBytes + i * kScaleBytes + g * (4 * kWords), sbuf);
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        float sum[TT][4];
        const float2 s = Elem<T>::unpack(sbuf[ZP ? 2 * u : u]);
        float2 z = make_float2(-8.0f - W4Deq<T>::kOffset, -8.0f - W4Deq<T>::kOffset);
        if constexpr (ZP) {
          z = Elem<T>::unpack(sbuf[2 * u + 1]);
          z.x = -W4Deq<T>::kOffset - z.x;
          z.y = -W4Deq<T>::kOffset - z.y;
        }
        z.x *= kUnit0;
        z.y *= kUnit1;
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          const float2 xv = *reinterpret_cast<const float2*>(xsum + (rel * UNITS + u) * (8 * TT) + i * 8 + 2 * t);
          sum[i][0] = z.x * xv.x;
          sum[i][1] = z.x * xv.y;
          sum[i][2] = z.y * xv.x;
          sum[i][3] = z.y * xv.y;
        }
#pragma unroll
        for (int h = u * (4 / UNITS); h < (u + 1) * (4 / UNITS); ++h) {  // 32 rows at a time
          const uint4 c = cbuf[h >> 1];
          uint32_t p0[4], p1[4];
          W4Deq<T>::pairs((h & 1) ? c.z : c.x, p0);
          W4Deq<T>::pairs((h & 1) ? c.w : c.y, p1);
#pragma unroll
          for (int i = 0; i < TT; ++i) {
            const uint4 xv = lds128(xr[i] + (static_cast<uint32_t>(rel * (kW4Block * 2)) & xmask[i]) + h * 64);
            mma16816<T>(sum[i], p0, xv.x, xv.y);
            mma16816<T>(sum[i], p1, xv.z, xv.w);
          }
        }
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          acc[i][0] = fmaf(s.x, sum[i][0], acc[i][0]);
          acc[i][1] = fmaf(s.x, sum[i][1], acc[i][1]);
          acc[i][2] = fmaf(s.y, sum[i][2], acc[i][2]);
          acc[i][3] = fmaf(s.y, sum[i][3], acc[i][3]);
        }
      }
    };
    for (int it = 0, tile = cluster * np + slot_tile; it < a.iters; ++it, tile += tile_step) {
#pragma unroll
      for (int i = 0; i < TT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
      if (tile < a.l.n_tiles)
        for (int rel = lead; rel < nb; rel += stride) {
          if (!mbar_wait(bars + slot * 8, phase, wctx, kDevTimeoutProducer)) ok = false;
          ok = __all_sync(0xffffffffu, ok) != 0;
          if (!ok) break;  // nothing is read; the joins go on, so no barrier is missed
          const uint32_t d = ring + slot * slot_bytes;
          block(d, 0, rel);
          if (a.run == 2 && rel + 1 < nb) block(d, 1, rel + 1);
          if (++slot == a.depth) slot = 0, phase ^= 1;
          __syncwarp();
          if (lane == 0) load();
        }
      const int buf = it & 1;
      float* pb = part + buf * (kWarps * kPart) + warp * kPart;
      if (it >= 2) bar_sync(kBarFree + buf);
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        float* p = pb + (i * 8 + 2 * t) * kPartStride + 2 * g;
        *reinterpret_cast<float2*>(p) = make_float2(acc[i][0] * (1.0f / kUnit0), acc[i][2] * (1.0f / kUnit1));
        *reinterpret_cast<float2*>(p + kPartStride) = make_float2(acc[i][1] * (1.0f / kUnit0), acc[i][3] * (1.0f / kUnit1));
      }
      bar_arrive(kBarFull + buf);
    }
  }
  // After a wait that ran out, the copies that were started are waited for (again with a limit)
  // before the CTA's shared memory goes away; otherwise every copy has been taken above.
  if (!ok && lane == 0 && a.inject == 0) {
    for (int i = 0; i < a.depth; ++i) {
      const uint64_t t0 = globaltimer_ns();
      while (!mbar_try_wait(bars + slot * 8, phase) && globaltimer_ns() - t0 < a.timeout_ns) {
      }
      if (++slot == a.depth) slot = 0, phase ^= 1;
    }
  }
  // no CTA leaves while another may still write into its shared memory
  if (a.ck > 1) {
    __syncwarp();
    cluster_sync_all();
  }
}

int rows_x_stride(int slice) { return slice * (kW4Block * 2) + 64; }  // conflict-free: 64 past a multiple of 128

// Shared memory of a CTA: rings, warps' sums, clusters' sums, group sums of x, zeros, x rows
int64_t rows_smem(const W4Layout& l, int tt, int ck, int ws, int slice, int rows, int slots) {
  const int64_t outs = static_cast<int64_t>(kWarps / ws) * tt * 128;
  return static_cast<int64_t>(kWarps) * slots * (kW4BlockBytes + l.scale_bytes()) + 2ll * kWarps * tt * 8 * kPartStride * 4 + (ck > 1 ? 2 * outs * 4 : 0) + 32ll * slice * l.units * tt +
         kZeroBytes + static_cast<int64_t>(rows) * rows_x_stride(slice);
}

template <typename T, int TT, int UNITS, bool ZP, typename OutT>
int rows_launch(const W4RowsArgs& a, int smem, int clusters, int64_t row_tiles, cudaStream_t s, const PdlIo& io) {
  static unsigned long long done_mask = 0;
  auto kern = &w4_rows_kernel<T, TT, UNITS, ZP, OutT>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), kRowsSmem, &done_mask);
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

template <typename T, int TT, int UNITS, typename OutT>
int rows_zeros(const W4RowsArgs& a, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  return a.l.zeros ? rows_launch<T, TT, UNITS, true, OutT>(a, smem, clusters, rt, s, io)
                   : rows_launch<T, TT, UNITS, false, OutT>(a, smem, clusters, rt, s, io);
}

template <typename T, int TT, typename OutT>
int rows_dispatch(const W4RowsArgs& a, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  return a.l.units == 1   ? rows_zeros<T, TT, 1, OutT>(a, smem, clusters, rt, s, io)
         : a.l.units == 2 ? rows_zeros<T, TT, 2, OutT>(a, smem, clusters, rt, s, io)
                          : rows_zeros<T, TT, 4, OutT>(a, smem, clusters, rt, s, io);
}

template <typename T, typename OutT>
int rows_tt(const W4RowsArgs& a, int tt, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  return tt == 1 ? rows_dispatch<T, 1, OutT>(a, smem, clusters, rt, s, io)
                 : rows_dispatch<T, 2, OutT>(a, smem, clusters, rt, s, io);
}

}  // namespace

int launch_w4_linear(const W4Layout& l, int dtype, int64_t m, const void* x, const void* packed, const void* bias,
                     int act, void* out, bool out_f32, cudaStream_t s, const DeviceInfo& dev) {
  const int sm_count = dev.sm_count;
  W4RowsArgs a;
  a.status = dev.status;
  a.timeout_ns = current_timeout_ns();
  a.inject = current_fault_injection();
  a.l = l;
  a.x = x;
  a.packed = packed;
  a.bias = bias;
  a.out = out;
  a.act = act;
  // Split of the work: ck CTAs of a cluster along K, ws warps per column tile. A tile group costs
  // its warps' blocks plus a join (about one block's time within a CTA, about three more across a
  // cluster); the fewest rounds of that over the GPU's SMs win. A pass takes up to 16 rows, fewer
  // where they would not fit in shared memory even spread over eight CTAs.
  int per_pass = m > 8 ? 16 : 8;
  for (;; per_pass /= 2) {
    const int rows = static_cast<int>(m < per_pass ? m : per_pass), tt = per_pass > 8 ? 2 : 1;
      int64_t best = LLONG_MAX;
    for (int ck = 1; ck <= kMaxCluster; ck *= 2) {
      const int slice = (l.blocks + ck - 1) / ck;
      if (ck > 1 && (ck - 1) * slice >= l.blocks) break;  // a CTA without work
      for (int ws = 1; ws <= kWarps; ws *= 2) {
        if (ws > 1 && ws / 2 >= slice) break;
        const int run = slice >= 4 * ws ? 2 : 1;
        if (rows_smem(l, tt, ck, ws, slice, rows, run * kMinDepth) > kRowsSmem) continue;
        const int groups = (l.n_tiles + kWarps / ws - 1) / (kWarps / ws);
        const int clusters = groups < sm_count / ck ? groups : sm_count / ck;
        const int64_t iters = (groups + clusters - 1) / clusters;
        const int64_t cost = iters * ((slice + ws - 1) / ws + 1 + (ck > 1 ? 3 : 0));
        if (cost >= best) continue;
        best = cost;
        a.ck = ck;
        a.slice = slice;
        a.run = run;
        a.ws = ws;
        a.iters = static_cast<int>(iters);
      }
    }
    if (best != LLONG_MAX) break;
    if (per_pass == 1) return set_error(GP_ERR_UNSUPPORTED, "w4 linear: K = %d", l.k);
  }
  a.rows = per_pass;
  a.x_stride = rows_x_stride(a.slice);
  const int tt = per_pass > 8 ? 2 : 1;
  const int rows = static_cast<int>(m < per_pass ? m : per_pass);
  a.depth = kMaxDepth;
  while (rows_smem(l, tt, a.ck, a.ws, a.slice, rows, a.run * a.depth) > kRowsSmem) --a.depth;
  const int smem = static_cast<int>(rows_smem(l, tt, a.ck, a.ws, a.slice, rows, a.run * a.depth));
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
