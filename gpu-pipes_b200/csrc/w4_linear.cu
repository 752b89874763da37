// Products with 4-bit weights for few rows (one token to 16): out [m, N] = act(x [m, K] W + b),
// W = s (q - z) (w4.cuh).
//
// With few rows the time is the weights' bytes (half a byte each), and what stands between them and
// the memory's rate is the number of instructions per weight. So:
//   - The matrix instruction is mma.sync m16n8k16 with the WEIGHTS as its 16-row operand (16 columns
//     of W) and 8 or 16 rows of x on the other side; one to eight rows cost the same and the sums are
//     fp32. (tcgen05 wants 16-bit weights in TMEM or shared memory, a store and a read per weight
//     more: that form is w4_tiles.cu, for more rows.)
//   - A code becomes an operand q - z with one mask and one packed sum per two weights, both exact
//     (w4.cuh). The group's scale multiplies the fp32 sum, so no weight is rounded. A first form that
//     worked weight by weight and divided to find the group ran 348 instructions per 2,048 weights and 57 us at
//     1 x 8,192 x 28,672 (fp16, groups of 128), where the bytes take 18.5.
//
//   - A CTA of 16 computing warps owns a slice of K (one of `ck` CTAs of a cluster does; ck = 1: all of
//     it), keeps its part of the x rows in shared memory and goes over column tiles of 16. `ws` warps
//     share a tile; a warp takes RUN neighbouring 128-row blocks at a time.
//   - One thread streams the codes and scales through a ring of stages in shared memory. A stage is
//     what the 16 warps take next: for each tile one stretch of ws * RUN neighbouring blocks, one bulk
//     copy each for codes and scales. (Copies of a block at a time, started by each warp for itself,
//     were slower in two ways: the copy engine took about 35 ns a piece, and waiting and loading
//     were 42 of the computing warps' 143 instructions per 2,048 weights. 31.5 us.)
//   - The codes of the next tiles are in flight while the sums of this one are joined by warps of
//     their own, in shared memory and across a cluster through st.async, both in a fixed order:
//     results do not depend on timing.
// Measured (CUDA-graph replays over more weights than L2 holds): 1 x 8,192 x 28,672 fp16 28.2 us, 4.3
// TB/s of 121 MB; 16 rows 41.8 us; 1 x 1,024 x 4,096 bf16 3.3 us. What is left at one row: about 3.5 us of
// launch and first latency, 13 tiles on the busiest SM for 12.1 on average, and latency between
// (issue at 54%, the busiest pipe at 43%).
#include <climits>

#include "../../include/gpipes.h"
#include "chain_registry.h"
#include "w4.cuh"

namespace gp {
namespace {

// Warps of a CTA (one CTA per SM): kWarps turn codes into sums, kJoinWarps add the sums up and store,
// one more loads.
constexpr int kWarps = 16;
constexpr int kJoinWarps = 3;
constexpr int kJoiners = 32 * kJoinWarps;
constexpr int kThreads = 32 * (kWarps + kJoinWarps + 1);
constexpr int kPartStride = 20;     // floats per row of a warp's 16 x rows sums: conflict-free float2 stores
constexpr int kMaxCluster = 8;
constexpr int64_t kRowsMax = 16;    // rows that go to this kernel
constexpr int kMaxDepth = 8;        // ring stages
constexpr int kMinDepth = 2;
constexpr int kRowsSmem = kSmemLimit - 2048;  // dynamic: the barriers are static
constexpr int kZeroBytes = 256;     // zeros in shared memory, read in place of absent x rows

struct W4RowsArgs {
  W4Layout l;
  const void* x;
  const void* packed;
  const void* bias;
  void* out;
  int64_t m;
  int out_f32;
  int out_planes;
  int act;
  int ck;            // CTAs of a cluster, along K
  int slice;         // k-blocks of a CTA
  int ws;            // warps that share a column tile
  int iters;         // column tile groups per cluster
  int rows;          // x rows of a pass (at most 8 TT)
  int x_stride;      // bytes between x rows in shared memory
  int depth;         // ring stages
  int* status;
  unsigned long long timeout_ns;
  int inject;        // fault injection: 1 = no block is ever loaded
};

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

// Named barriers of the CTA (0 is __syncthreads): waiting, and arriving without waiting.
__device__ __forceinline__ void bar_sync(int id) {
  __syncwarp();
  asm volatile("bar.sync %0, %1;" ::"r"(id), "n"(32 * (kWarps + kJoinWarps)) : "memory");
}
__device__ __forceinline__ void bar_arrive(int id) {
  __syncwarp();
  asm volatile("bar.arrive %0, %1;" ::"r"(id), "n"(32 * (kWarps + kJoinWarps)) : "memory");
}
constexpr int kBarFull = 1, kBarFree = 3;  // + buffer 0 / 1 of the warps' sums

// 16 bytes into the shared memory of a CTA of the cluster, counted on that CTA's mbarrier: the
// reader needs no other signal and the writer no fence.
__device__ __forceinline__ void st_async_f32x4(uint32_t addr, uint32_t bar, float4 v) {
  asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.v4.f32 [%0], {%2, %3, %4, %5}, [%1];" ::"r"(addr),
               "r"(bar), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

// TT: tiles of 8 x rows. UNITS: groups per k-block of 128. RUN: k-blocks of a ring slot, neighbours in the
// packed codes. PLANES: x rows as one T or as two (in a chain), with a product each on the same codes.
template <typename T, int TT, int UNITS, bool ZP, int RUN, int PLANES>
__global__ void __launch_bounds__(kThreads, 1) w4_rows_kernel(const __grid_constant__ W4RowsArgs a) {
  constexpr int kWords = UNITS * (ZP ? 2 : 1);                // scale words of a lane per block
  constexpr int kPart = TT * 8 * kPartStride;                 // floats of a warp's sums
  constexpr int kScaleBytes = 32 * kWords;                    // scales of a block
  constexpr int kStageCodes = kWarps * RUN * kW4BlockBytes;   // a stage: codes of every warp, then scales
  constexpr int kStage = kWarps * RUN * (kW4BlockBytes + kScaleBytes);
  constexpr float kUnit0 = W4Deq<T>::unit(0), kUnit1 = W4Deq<T>::unit(1);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kMaxDepth], empty[kMaxDepth];
  __shared__ __align__(8) uint64_t red_full[2];
  __shared__ int abort_flag, join_abort;
  float* part = reinterpret_cast<float*>(smem + a.depth * kStage);  // [2][kWarps][kPart]
  const int np = kWarps / a.ws;                               // tiles at a time
  const int outs = np * TT * 128;                             // sums of a tile group
  float* red = part + 2 * kWarps * kPart;                     // [2][outs], clusters only
  uint8_t* zeros = reinterpret_cast<uint8_t*>(red + (a.ck > 1 ? 2 * outs : 0));
  uint8_t* xs = zeros + kZeroBytes;                           // [rows][x_stride]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int rank = a.ck > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int cluster = blockIdx.x / a.ck, clusters = gridDim.x / a.ck;
  const int64_t row0 = static_cast<int64_t>(blockIdx.y) * a.rows;
  const int rows = static_cast<int>(a.m - row0 < a.rows ? a.m - row0 : a.rows);
  const int b0 = rank * a.slice;
  const int nb = min(a.slice, a.l.blocks - b0);               // blocks of this CTA
  const int sub = warp % a.ws, slot_tile = warp / a.ws;

  const int tile_step = clusters * np, lead = sub * RUN, stride = a.ws * RUN;
  const WaitCtx wctx{a.status, &abort_flag, a.timeout_ns};
  bool ok = true;
  // codes and scales of block `rel` of the slice in column tile `tile`
  auto codes_at = [&](int tile, int rel) {
    return static_cast<const uint8_t*>(a.packed) + (static_cast<int64_t>(tile) * a.l.blocks + b0 + rel) * kW4BlockBytes;
  };
  auto scales_at = [&](int tile, int rel) {
    return static_cast<const uint8_t*>(a.packed) + a.l.scale_off +
           (static_cast<int64_t>(tile) * a.l.blocks + b0 + rel) * kScaleBytes;
  };

  if (threadIdx.x == 0) {
    for (int i = 0; i < a.depth; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), kWarps);
    }
    mbar_init(smem_u32(&red_full[0]), 1);
    mbar_init(smem_u32(&red_full[1]), 1);
    abort_flag = join_abort = 0;
    fence_mbar_init();
  }
  // The first codes go into L2 while the previous kernel of the stream drains (a hint: nothing is
  // read into the program before the wait).
  if (warp < np && cluster * np + warp < a.l.n_tiles)
    for (int i = lane; i < min(nb, a.depth * stride); i += 32)
      asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(codes_at(cluster * np + warp, i)), "n"(kW4BlockBytes));
  pdl_wait_prior();
  pdl_launch_dependents();
  __syncthreads();  // barriers
  // every CTA of the cluster runs before one writes into another's shared memory
  if (a.ck > 1) cluster_sync_all();

  if (warp == kWarps + kJoinWarps) {
    // ---- loading, by one thread
    if (lane == 0 && a.inject == 0) {
      int stage = 0, phase = 0, issued = 0;
      for (int it = 0; it < a.iters && ok; ++it)
        for (int rel = 0; rel < nb; rel += stride) {
          if (issued >= a.depth && !mbar_wait(smem_u32(&empty[stage]), phase ^ 1, wctx, kDevTimeoutProducer)) {
            ok = false;
            break;
          }
          const int n = min(stride, nb - rel);
          const int tile0 = (cluster + it * clusters) * np, tiles = min(np, a.l.n_tiles - tile0);
          const uint32_t bar = smem_u32(&full[stage]), dst = smem_u32(smem) + stage * kStage;
          mbar_arrive_expect_tx(bar, max(tiles, 0) * n * (kW4BlockBytes + kScaleBytes));
          for (int i = 0; i < tiles; ++i) {
            bulk_load(dst + i * stride * kW4BlockBytes, codes_at(tile0 + i, rel), n * kW4BlockBytes, bar);
            bulk_load(dst + kStageCodes + i * stride * kScaleBytes, scales_at(tile0 + i, rel), n * kScaleBytes, bar);
          }
          ++issued;
          if (++stage == a.depth) stage = 0, phase ^= 1;
        }
      // After a wait that ran out somewhere, the copies under way are waited for (again with a limit)
      // before the CTA's shared memory goes away; otherwise the computing warps take every stage.
      if (!ok)
        for (int i = 0; i < a.depth; ++i) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(smem_u32(&full[stage]), phase ^ 1) && globaltimer_ns() - t0 < a.timeout_ns) {
          }
          if (++stage == a.depth) stage = 0, phase ^= 1;
        }
    }
  } else {
  // x rows of this CTA's slice (zero past K); absent rows are read from the zeros.
  constexpr int kStagers = 32 * (kWarps + kJoinWarps);
  if (threadIdx.x < kZeroBytes / 16) reinterpret_cast<uint4*>(zeros)[threadIdx.x] = make_uint4(0, 0, 0, 0);
  {
    const int pieces = a.slice * 16;  // 16-byte pieces of a row
    for (int i = threadIdx.x; i < rows * pieces; i += kStagers) {
      const int r = i / pieces, c = i % pieces;
      const int k = b0 * kW4Block + c * 8;
      uint4 v = make_uint4(0, 0, 0, 0);
      const T* from = static_cast<const T*>(a.x) + (row0 + r) * a.l.k + k;
      if (k < a.l.k) v = *reinterpret_cast<const uint4*>(from);
      // rows 16 j + 4 t + i of a 32-row half where lane t reads them as 16 bytes, j by j
      uint8_t* to = xs + r * a.x_stride + (c >> 2) * 64 + (c & 1) * 32 + ((c >> 1) & 1) * 8;
      *reinterpret_cast<uint2*>(to) = make_uint2(v.x, v.y);
      *reinterpret_cast<uint2*>(to + 16) = make_uint2(v.z, v.w);
      if constexpr (PLANES == 2) {
        uint4 u = make_uint4(0, 0, 0, 0);
        if (k < a.l.k) u = *reinterpret_cast<const uint4*>(from + a.m * a.l.k);
        to += rows * a.x_stride;
        *reinterpret_cast<uint2*>(to) = make_uint2(u.x, u.y);
        *reinterpret_cast<uint2*>(to + 16) = make_uint2(u.z, u.w);
      }
    }
  }
  bar_sync(kBarFull);  // x is in place (this barrier's first use as a buffer's comes after)

  if (warp >= kWarps) {
    // ---- joining: part[warp][row][column] of a tile group, summed over its warps (and CTAs)
    const int j = threadIdx.x - 32 * kWarps;
    // Sums go four neighbouring columns at a time: quad q is tile q / (32 TT), row (q / 4) % (8 TT),
    // columns 4 (q % 4) .. + 3. CTA r of a cluster finishes quads [r own, (r + 1) own).
    // The wait for another CTA has its own abort flag: a lost copy of codes ends no join, whose sums
    // are all sent and so arrive before any CTA leaves.
    const WaitCtx jctx{a.status, &join_abort, a.timeout_ns};
    const int quads = outs / 4, own = quads / a.ck;
    const bool vec = a.l.n % 4 == 0 && reinterpret_cast<uintptr_t>(a.out) % (a.out_f32 ? 16 : 8) == 0;
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
        for (int i = 0; i < 4; ++i)
          if (a.bias != nullptr && i < live) v[i] += Elem<T>::to_f(static_cast<const T*>(a.bias)[n + i]);
        w4_act(a.act, v);
        const int64_t at = (row0 + row_of(q)) * a.l.n + n;
        if (a.out_f32) {
          float* to = static_cast<float*>(a.out) + at;
          if (vec) {
            *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (i < live) to[i] = v[i];
          }
        } else {
          uint16_t* to = static_cast<uint16_t*>(a.out) + at;
          auto put = [&](uint32_t lo, uint32_t hi) {
            if (vec) {
              *reinterpret_cast<uint2*>(to) = make_uint2(lo, hi);
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (i < live) to[i] = static_cast<uint16_t>((i < 2 ? lo : hi) >> (16 * (i & 1)));
            }
          };
          put(Elem<T>::pack(v[0], v[1]), Elem<T>::pack(v[2], v[3]));
          if (a.out_planes == 2) {
            uint16_t first, rest[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w4_two<T>(v[i], first, rest[i]);
            to += a.m * a.l.n;
            put(rest[0] | static_cast<uint32_t>(rest[1]) << 16, rest[2] | static_cast<uint32_t>(rest[3]) << 16);
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
    // ---- codes to sums. Addresses run along: this loop is bound by its integer instructions.
    uint32_t xa0[TT], xstep[TT], xsecond[TT];  // xsecond: bytes to the second plane
#pragma unroll
    for (int i = 0; i < TT; ++i) {  // absent rows read the zeros again and again
      const bool live = i * 8 + g < rows;
      xa0[i] = smem_u32(live ? xs + (i * 8 + g) * a.x_stride + lead * (kW4Block * 2) : zeros) + t * 16;
      xstep[i] = live ? kW4Block * 2 : 0;
      xsecond[i] = live ? rows * a.x_stride : 0;
    }
    float acc[TT][4];
    // a block: codes and scales at c and s, x rows at xa
    auto block = [&](uint32_t c, uint32_t s, const uint32_t (&xa)[TT]) {
      const uint4 cbuf[2] = {lds128(c), lds128(c + kW4BlockBytes / 2)};
      uint32_t sbuf[kWords];
      w4_lds<kWords>(s, sbuf);
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        float sum[TT][4];
        W4Deq<T> dq;
        dq.template set<ZP>(ZP ? sbuf[2 * u + 1] : 0u);
#pragma unroll
        for (int i = 0; i < TT; ++i) sum[i][0] = sum[i][1] = sum[i][2] = sum[i][3] = 0.0f;
#pragma unroll
        for (int h = u * (4 / UNITS); h < (u + 1) * (4 / UNITS); ++h) {  // 32 rows at a time
          const uint4 cw = cbuf[h >> 1];
          uint32_t p0[4], p1[4];
          dq.pairs((h & 1) ? cw.z : cw.x, p0);
          dq.pairs((h & 1) ? cw.w : cw.y, p1);
#pragma unroll
          for (int i = 0; i < TT; ++i) {
            const uint4 xv = lds128(xa[i] + h * 64);
            mma16816<T>(sum[i], p0, xv.x, xv.y);
            mma16816<T>(sum[i], p1, xv.z, xv.w);
            if constexpr (PLANES == 2) {
              const uint4 xl = lds128(xa[i] + xsecond[i] + h * 64);
              mma16816<T>(sum[i], p0, xl.x, xl.y);
              mma16816<T>(sum[i], p1, xl.z, xl.w);
            }
          }
        }
        const float2 sc = Elem<T>::unpack(sbuf[ZP ? 2 * u : u]);
#pragma unroll
        for (int i = 0; i < TT; ++i) {
          acc[i][0] = fmaf(sc.x, sum[i][0], acc[i][0]);
          acc[i][1] = fmaf(sc.x, sum[i][1], acc[i][1]);
          acc[i][2] = fmaf(sc.y, sum[i][2], acc[i][2]);
          acc[i][3] = fmaf(sc.y, sum[i][3], acc[i][3]);
        }
      }
    };
    // this warp's place in a stage
    const uint32_t c0 = smem_u32(smem) + (slot_tile * stride + lead) * kW4BlockBytes + lane * 16;
    const uint32_t to_scales = smem_u32(smem) + kStageCodes + (slot_tile * stride + lead) * kScaleBytes + g * (4 * kWords) - c0;
    int stage = 0, phase = 0;
    uint32_t cs = c0;
    for (int it = 0, tile = cluster * np + slot_tile; it < a.iters; ++it, tile += tile_step) {
#pragma unroll
      for (int i = 0; i < TT; ++i) acc[i][0] = acc[i][1] = acc[i][2] = acc[i][3] = 0.0f;
      uint32_t xa[TT];
#pragma unroll
      for (int i = 0; i < TT; ++i) xa[i] = xa0[i];
      // blocks left for this warp from `lead` on, run by run; every warp takes part in every stage
      int left = tile < a.l.n_tiles ? nb - lead : 0;
      for (int rel = 0; rel < nb && ok; rel += stride) {
        if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&full[stage]), phase, wctx, kDevTimeoutProducer))) {
          ok = false;  // nothing is read; the joins go on, so no barrier is missed
          break;
        }
        const uint32_t s = cs + to_scales;
        uint32_t xb[TT];
#pragma unroll
        for (int i = 0; i < TT; ++i) xb[i] = xa[i];
#pragma unroll
        for (int b = 0; b < RUN; ++b) {
          if (b >= left) break;
          block(cs + b * kW4BlockBytes, s + b * kScaleBytes, xb);
#pragma unroll
          for (int i = 0; i < TT; ++i) xb[i] += xstep[i];
        }
        left -= stride;
#pragma unroll
        for (int i = 0; i < TT; ++i) xa[i] += stride * xstep[i];
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&empty[stage]));
        cs += kStage;
        if (++stage == a.depth) stage = 0, phase ^= 1, cs = c0;
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
  }  // not loading
  // no CTA leaves while another may still write into its shared memory
  if (a.ck > 1) {
    __syncwarp();
    cluster_sync_all();
  }
}

int rows_x_stride(int slice) { return slice * (kW4Block * 2) + 64; }  // conflict-free: 64 past a multiple of 128

// Shared memory of a CTA: rings, warps' sums, clusters' sums, zeros, x rows
// (`rows` times its planes)
int64_t rows_smem(const W4Layout& l, int tt, int ck, int ws, int slice, int rows, int slots) {
  const int64_t outs = static_cast<int64_t>(kWarps / ws) * tt * 128;
  return static_cast<int64_t>(kWarps) * slots * (kW4BlockBytes + l.scale_bytes()) + 2ll * kWarps * tt * 8 * kPartStride * 4 + (ck > 1 ? 2 * outs * 4 : 0) +
         kZeroBytes + static_cast<int64_t>(rows) * rows_x_stride(slice);
}

template <typename T, int TT, int UNITS, bool ZP, int RUN, int PLANES>
int rows_launch(const W4RowsArgs& a, int smem, int clusters, int64_t row_tiles, cudaStream_t s, const PdlIo& io) {
  static unsigned long long done_mask = 0;
  auto kern = &w4_rows_kernel<T, TT, UNITS, ZP, RUN, PLANES>;
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

template <typename T, int TT, int UNITS, bool ZP>
int rows_run(const W4RowsArgs& a, int run, int planes, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  if (planes == 2) return rows_launch<T, TT, UNITS, ZP, 2, 2>(a, smem, clusters, rt, s, io);
  return run == 4 ? rows_launch<T, TT, UNITS, ZP, 4, 1>(a, smem, clusters, rt, s, io)
                  : rows_launch<T, TT, UNITS, ZP, 2, 1>(a, smem, clusters, rt, s, io);
}

template <typename T, int TT, int UNITS>
int rows_zeros(const W4RowsArgs& a, int run, int planes, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  return a.l.zeros ? rows_run<T, TT, UNITS, true>(a, run, planes, smem, clusters, rt, s, io)
                   : rows_run<T, TT, UNITS, false>(a, run, planes, smem, clusters, rt, s, io);
}

template <typename T, int TT>
int rows_units(const W4RowsArgs& a, int run, int planes, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  return a.l.units == 1   ? rows_zeros<T, TT, 1>(a, run, planes, smem, clusters, rt, s, io)
         : a.l.units == 2 ? rows_zeros<T, TT, 2>(a, run, planes, smem, clusters, rt, s, io)
                          : rows_zeros<T, TT, 4>(a, run, planes, smem, clusters, rt, s, io);
}

template <typename T>
int rows_tt(const W4RowsArgs& a, int tt, int run, int planes, int smem, int clusters, int64_t rt, cudaStream_t s, const PdlIo& io) {
  return tt == 1 ? rows_units<T, 1>(a, run, planes, smem, clusters, rt, s, io)
                 : rows_units<T, 2>(a, run, planes, smem, clusters, rt, s, io);
}

}  // namespace

int w4_max_clusters(const void* kern, int threads, int smem, int ck, int sm_count, std::atomic<int> (*cache)[4]) {
  if (ck == 1) return sm_count;
  int dev = 0;
  cudaGetDevice(&dev);
  std::atomic<int>& slot = cache[dev & 63][ck == 2 ? 1 : ck == 4 ? 2 : 3];  // racing first calls store the same value
  int n = slot.load(std::memory_order_relaxed);
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(sm_count / ck * ck), 1, 1);
    cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(ck);
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = sm_count / ck;
    }
    slot.store(n, std::memory_order_relaxed);
  }
  return n;
}

int launch_w4_rows(const W4LinearArgs& in, cudaStream_t s, const DeviceInfo& dev) {
  const W4Layout& l = in.l;
  const int64_t m = in.m;
  // the number of CTAs that run at a time, from one instance at its full shared memory
  static std::atomic<int> cluster_cache[64][4];
  static unsigned long long probe_mask = 0;
  auto probe = &w4_rows_kernel<__half, 1, 1, false, 2, 1>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(probe), kRowsSmem, &probe_mask);
  if (rc != GP_OK) return rc;
  auto resident = [&](int ck) {
    return w4_max_clusters(reinterpret_cast<const void*>(probe), kThreads, kRowsSmem, ck, dev.sm_count, cluster_cache);
  };
  W4RowsArgs a;
  a.status = dev.status;
  a.timeout_ns = current_timeout_ns();
  a.inject = current_fault_injection();
  a.l = l;
  a.packed = in.packed;
  a.bias = in.bias;
  a.out_f32 = in.out_f32;
  a.out_planes = in.out_planes;
  const int planes = in.x_planes;
  a.act = in.act;
  // Split of the work. A pass takes up to 16 rows (8 and fewer for the kernel of one row tile), fewer
  // where they would not fit in shared memory even spread over eight CTAs. Of the splits into ck CTAs
  // along K and ws warps per tile, the one with the least time on the busiest SM: per tile group its
  // warps' blocks and about one and a half blocks more, three more in all where a cluster joins. A warp has at
  // most four blocks of a tile if there are warps for that: with more, few tiles are long under way
  // (1 x 4,096 x 14,336: 9.3 us with ws = 8, 10.1 with 4, 10.8 with 2).
  int per_pass = m > 8 ? 16 : 8, run = 2, clusters = 1;
  for (;; per_pass /= 2) {
    const int rows = static_cast<int>(m < per_pass ? m : per_pass), tt = per_pass > 8 ? 2 : 1;
    int64_t best = LLONG_MAX;
    for (int ck = 1; ck <= kMaxCluster; ck *= 2) {
      const int slice = (l.blocks + ck - 1) / ck;
      if (ck > 1 && (ck - 1) * slice >= l.blocks) break;  // a CTA without work
      const int at_once = resident(ck);
      for (int ws = kWarps; ws >= 1; ws /= 2) {
        if (ws > 1 && ws / 2 >= slice) continue;  // warps without a block
        if (slice > 4 * ws && ws < kWarps) break;
        const int per_warp = (slice + ws - 1) / ws;
        int r = per_warp > 2 && planes == 1 ? 4 : 2;
        if (rows_smem(l, tt, ck, ws, slice, rows * planes, 4 * 3) > kRowsSmem) r = 2;
        if (rows_smem(l, tt, ck, ws, slice, rows * planes, r * kMinDepth) > kRowsSmem) continue;
        const int groups = (l.n_tiles + kWarps / ws - 1) / (kWarps / ws);
        const int n = groups < at_once ? groups : at_once;
        const int64_t iters = (groups + n - 1) / n;
        const int64_t cost = iters * (2 * per_warp + 3) + (ck > 1 ? 6 : 0);
        if (cost >= best) continue;
        best = cost;
        a.ck = ck;
        a.slice = slice;
        a.ws = ws;
        a.iters = static_cast<int>(iters);
        run = r;
        clusters = n;
      }
    }
    if (best != LLONG_MAX) break;
    if (per_pass == 1) return set_error(GP_ERR_UNSUPPORTED, "w4 linear: K = %d", l.k);
  }
  const int rows = static_cast<int>(m < per_pass ? m : per_pass), tt = per_pass > 8 ? 2 : 1;
  a.m = m;
  a.rows = per_pass;
  a.x = in.x;
  a.out = in.out;
  a.x_stride = rows_x_stride(a.slice);
  a.depth = kMaxDepth;
  while (rows_smem(l, tt, a.ck, a.ws, a.slice, rows * planes, run * a.depth) > kRowsSmem) --a.depth;
  const int smem = static_cast<int>(rows_smem(l, tt, a.ck, a.ws, a.slice, rows * planes, run * a.depth));
  PdlIo io;
  io.add(PdlIo::kWrite, in.out, static_cast<uint64_t>(m) * l.n * (in.out_f32 ? 4 : 2 * in.out_planes));
  const int64_t passes = (m + per_pass - 1) / per_pass;
  rc = in.dtype == GP_BF16 ? rows_tt<__nv_bfloat16>(a, tt, run, planes, smem, clusters, passes, s, io)
                           : rows_tt<__half>(a, tt, run, planes, smem, clusters, passes, s, io);
  if (rc == GP_OK) count_launches(1);
  return rc;
}

// Up to 16 rows the row kernel, from 17 on the tile kernel. Measured on either side of the border (CUDA-graph
// replays, fp16, groups of 128; us, row / tile kernel; 9, 16, 17 and 64 rows): 4,096 x 14,336 14.0 / 15.0, 16.3 / 15.0,
// 29 / 15.2, 63 / 16.7; 8,192 x 28,672 39 / 54, 42 / 54, 82 / 55, 166 / 58; 1,024 x 4,096 4.1 / 5.3, 4.4 / 5.3, 7.4 / 5.8,
// 17 / 6.7.
int launch_w4_linear(const W4LinearArgs& a, cudaStream_t s, const DeviceInfo& dev) {
  return a.m <= kRowsMax ? launch_w4_rows(a, s, dev) : launch_w4_tiles(a, s, dev);
}

}  // namespace gp
