// Products with 4-bit weights for more rows than the row kernel takes at a time (decode batches,
// prompts): out [m, N] = act(x [m, K] W + b) on the 5th-generation tensor cores.
//
// A CTA makes a tile of 128 columns of W times up to 256 rows of x, with the WEIGHTS as the 128-row
// operand A and the rows of x as the N side: D[n, row] = sum_k W[k, n] x[row, k]. The codes are turned
// into T once per tile and written straight to TMEM, where tcgen05.mma takes A from; shared memory
// carries only codes and x (through it, the 16-bit weights would be written once and read once more
// and its bandwidth would bound the kernel). The packed order is that of tcgen05.st 16x256b, so a
// lane's codes become its registers without a shuffle.
//
// Rounding: here a weight s (q - z) is rounded to T (q - z is exact, one multiplication), as
// w4_dequantize gives it; the sums are fp32. Scaling the sums instead, group by group, as the row
// kernel does, would read the accumulator once per group: more time than the tile's product.
//
//   loader (1 warp)     x panels by TMA, codes and scales by bulk copies, a ring of 128-row stages
//   16 dequantising warps  four groups of four (one warp per TMEM lane quarter); a group takes every
//                       fourth 64-row part: codes -> T -> its TMEM stage of 32 columns
//   MMA issuer (1 thread) four K = 16 products per part; commits free the TMEM stage and the ring stage
//   epilogue            the dequantising warps: bias, activation, store
// Where there are fewer tiles than SMs, a cluster of ck CTAs splits K and sums over distributed
// shared memory in a fixed order.
#include "../../include/gpipes.h"
#include "chain_registry.h"
#include "w4.cuh"

namespace gp {
namespace {

constexpr int kDeqGroups = 4;      // of four warps, one per TMEM lane quarter
constexpr int kDeqWarps = 4 * kDeqGroups;
constexpr int kTileThreads = 32 * (2 + kDeqWarps);
constexpr int kTileN = 128;        // columns of W per tile: the TMEM lanes
constexpr int kTileTiles = kTileN / 16;
constexpr int kAStages = kDeqGroups;  // TMEM stages of dequantised weights, 32 columns (64 rows of W) each
constexpr int kMaxStages = 8;
constexpr int kMaxTileRows = 256;

struct W4TileArgs {
  W4Layout l;
  const void* packed;
  const void* bias;
  void* out;
  int64_t m;
  int out_f32;
  int act;
  int rows;        // x rows of a tile: a multiple of 16 up to 256
  int row_tiles;
  int ck;          // CTAs of a cluster, along K
  int slice;       // k-blocks of a CTA
  int stages;
  int tmem_cols;
  int* status;
  unsigned long long timeout_ns;
  int inject;
};

__device__ __forceinline__ void tile_bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}

// 16 lanes x 32 columns: thread 4 g + t holds, per 8 columns, columns 2t and 2t + 1 of lane g, then of lane g + 8
__device__ __forceinline__ void tmem_st_16x256b_x4(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x4.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// Codes of a lane as T: for the two columns r, the scale twice and the constant that takes the
// zero point and the code's offset away (both steps exact before the scale).
//   half: 1024 + q minus 1024 + z; column 1 four bits higher: (1024 + 16 q) / 16 - (64 + z)
//   bf16: 16 + q minus 16 + z
template <typename T>
struct TileDeq;

template <>
struct TileDeq<__half> {
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
  // registers of one 8-column piece of tcgen05.st 16x256b
  __device__ __forceinline__ void word(uint32_t w, uint32_t* r) const {
    const __half2 sixteenth = __float2half2_rn(0.0625f);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t v = i == 0 ? w : w >> 8;
      const uint32_t lo = (v & 0x000F000Fu) | 0x64006400u, hi = (v & 0x00F000F0u) | 0x64006400u;
      const __half2 a = __hmul2(__hadd2(*reinterpret_cast<const __half2*>(&lo), c[0]), s[0]);
      const __half2 b = __hmul2(__hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, c[1]), s[1]);
      r[i] = *reinterpret_cast<const uint32_t*>(&a);
      r[2 + i] = *reinterpret_cast<const uint32_t*>(&b);
    }
  }
};

template <>
struct TileDeq<__nv_bfloat16> {
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
  __device__ __forceinline__ void word(uint32_t w, uint32_t* r) const {
    uint32_t p[4];
    W4Deq<__nv_bfloat16>::pairs(w, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // p[2 j + column], j: rows (0, 1) / (2, 3)
      const __nv_bfloat162 a = __hmul2(__hadd2(*reinterpret_cast<const __nv_bfloat162*>(&p[i]), c[i & 1]), s[i & 1]);
      r[2 * (i & 1) + (i >> 1)] = *reinterpret_cast<const uint32_t*>(&a);
    }
  }
};

// TMEM lane of a tile <-> column: lane 16 i + r holds column 16 i + 2 (r % 8) + r / 8
__device__ __forceinline__ int tile_column(int lane) { return (lane & ~15) + 2 * (lane & 7) + ((lane >> 3) & 1); }

template <typename T, int UNITS, bool ZP>
__global__ void __launch_bounds__(kTileThreads, 2)
    w4_tile_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ W4TileArgs a) {
  constexpr int kWords = UNITS * (ZP ? 2 : 1);
  constexpr int kScaleBytes = 32 * kWords;            // of a block of 16 columns
  constexpr int kCodes = kTileTiles * kW4BlockBytes;  // of a stage
  constexpr int kScales = kTileTiles * kScaleBytes;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], a_full[kAStages], a_empty[kAStages], d_full;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;
  const int panel = a.rows * 128;                     // x rows of 64 columns, SWIZZLE_128B
  const int stage_bytes = 2 * panel + kCodes + (kScales + 1023) / 1024 * 1024;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.ck > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / a.ck;
  const int tile0 = unit / a.row_tiles * kTileTiles;  // first 16-column tile
  const int64_t row0 = static_cast<int64_t>(unit % a.row_tiles) * a.rows;
  const int b0 = rank * a.slice, nb = min(a.slice, a.l.blocks - b0);
  const int tiles = min(kTileTiles, a.l.n_tiles - tile0);

  if ((smem_u32(smem) & 1023u) != 0) {  // the same in every CTA of the grid
    pdl_wait_prior();
    if (threadIdx.x == 0) atomicCAS(a.status, 0, kDevBadSmemAlign);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), 2 * 4 + 1);  // a block's two groups, and its products
    }
    for (int i = 0; i < kAStages; ++i) {
      mbar_init(smem_u32(&a_full[i]), 4);
      mbar_init(smem_u32(&a_empty[i]), 1);
    }
    mbar_init(smem_u32(&d_full), 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) prefetch_tmap(&tx);
  pdl_wait_prior();
  pdl_launch_dependents();
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_holder), a.tmem_cols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t d_tmem = tmem_holder, a_tmem = d_tmem + (a.tmem_cols - kAStages * 32);
  const WaitCtx wctx{a.status, &abort_flag, a.timeout_ns};
  bool ok = true;  // of this role

  if (warp == 0) {
    // lanes 0-7 the codes of a column tile each, lanes 8-15 its scales, lanes 16 and 17 the x panels:
    // one thread issuing all eighteen copies of a stage took longer than the copies
    if (a.inject == 0) {
      const uint64_t keep = l2_policy_evict_last();  // x is read by every column tile
      const int i = lane & 7;
      const int64_t cell = static_cast<int64_t>(tile0 + i) * a.l.blocks + b0;
      const uint8_t* src = static_cast<const uint8_t*>(a.packed) +
                           (lane < 8 ? cell * kW4BlockBytes : a.l.scale_off + cell * kScaleBytes);
      const uint32_t bytes = lane < 8 ? kW4BlockBytes : kScaleBytes;
      const uint32_t to = 2 * panel + (lane < 8 ? i * kW4BlockBytes : kCodes + i * kScaleBytes);
      int s = 0, ph = 0;
      for (int b = 0; b < nb; ++b) {
        if (b >= a.stages) {
          ok = mbar_wait(smem_u32(&empty[s]), ph ^ 1, wctx, kDevTimeoutProducer);
          if (!__all_sync(0xffffffffu, ok)) {
            ok = false;
            break;
          }
        }
        const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(smem) + s * stage_bytes;
        if (lane == 0) mbar_arrive_expect_tx(bar, 2 * panel + tiles * (kW4BlockBytes + kScaleBytes));
        __syncwarp();
        if (lane < 16) {
          if (i < tiles) tile_bulk_load(dst + to, src + b * static_cast<int64_t>(bytes), bytes, bar);
        } else if (lane < 18) {
          const int p = lane - 16;
          tma_load_2d_hint(dst + p * panel, &tx, bar, (b0 + b) * kW4Block + p * 64, static_cast<int>(row0), keep);
        }
        if (++s == a.stages) s = 0, ph ^= 1;
      }
      if (!ok && lane == 0)  // copies under way end (waited for with a limit) before their memory is used again or goes away
        for (int j = 0; j < a.stages; ++j) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(smem_u32(&full[s]), ph ^ 1) && globaltimer_ns() - t0 < a.timeout_ns) {
          }
          if (++s == a.stages) s = 0, ph ^= 1;
        }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      const uint32_t idesc = make_idesc_f16(kTileN, a.rows, Elem<T>::kIsBf16, 0, 0);
      int s = 0, ph = 0, as = 0, aph = 0;
      for (int b = 0; b < nb && ok; ++b) {
        if (!mbar_wait(smem_u32(&full[s]), ph, wctx, kDevTimeoutMma)) break;
        for (int p = 0; p < 2; ++p) {
          if (!mbar_wait(smem_u32(&a_full[as]), aph, wctx, kDevTimeoutMma)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint64_t bdesc = make_sdesc_sw128(smem_u32(smem) + s * stage_bytes + p * panel, 16, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(d_tmem, a_tmem + as * 32 + k * 8, bdesc + static_cast<uint64_t>(k * 2), idesc, (b | p | k) != 0 ? 1u : 0u);
          mma_commit(smem_u32(&a_empty[as]));
          if (++as == kAStages) as = 0, aph ^= 1;
        }
        if (ok) mma_commit(smem_u32(&empty[s]));
        if (++s == a.stages) s = 0, ph ^= 1;
      }
      // every product issued has completed before TMEM is read or released
      mma_commit(smem_u32(&d_full));
      volatile int no_abort = 0;
      const WaitCtx drain{a.status, &no_abort, a.timeout_ns};
      mbar_wait(smem_u32(&d_full), 0, drain, kDevTimeoutMma);
    }
  } else {
    const int q = warp & 3, group = (warp - 2) >> 2, g = lane >> 2;
    int s = 0, ph = 0;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    // this group's parts are group, group + 4, ...: every other block, always the same TMEM stage
    const int as = group;
    auto next_stage = [&] {
      if (++s == a.stages) s = 0, ph ^= 1;
    };
    if (group >= 2) next_stage();
    for (int b = group >> 1, use = 0; b < nb; b += kDeqGroups / 2, ++use) {
      ok = mbar_wait(smem_u32(&full[s]), ph, wctx, kDevTimeoutProducer) &&
           (use == 0 || mbar_wait(smem_u32(&a_empty[as]), (use - 1) & 1, wctx, kDevTimeoutEpilogue));
      if (!__all_sync(0xffffffffu, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint8_t* st = smem + s * stage_bytes + 2 * panel;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int nt = 2 * q + i;  // column tile of this 16-lane half; absent ones hold old bytes: zeroed
        uint4 c = make_uint4(0, 0, 0, 0);
        uint32_t sw[kWords];
#pragma unroll
        for (int w = 0; w < kWords; ++w) sw[w] = 0;
        if (nt < tiles) {
          c = *reinterpret_cast<const uint4*>(st + nt * kW4BlockBytes + (group & 1) * (kW4BlockBytes / 2) + lane * 16);
#pragma unroll
          for (int w = 0; w < kWords; ++w)
            sw[w] = *reinterpret_cast<const uint32_t*>(st + kCodes + nt * kScaleBytes + (g * kWords + w) * 4);
        }
        uint32_t r[16];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int u = UNITS == 1 ? 0 : UNITS == 2 ? group & 1 : 2 * (group & 1) + h;
          TileDeq<T> dq;
          if constexpr (UNITS == 1) {
            dq.set(sw[0], sw[ZP ? 1 : 0], ZP);
          } else {  // constant indices: sw stays in registers
            uint32_t s01 = 0, z01 = 0;
#pragma unroll
            for (int v = 0; v < UNITS; ++v)
              if (v == u) s01 = sw[ZP ? 2 * v : v], z01 = ZP ? sw[2 * v + (ZP ? 1 : 0)] : 0u;
            dq.set(s01, z01, ZP);
          }
          dq.word(h == 0 ? c.x : c.z, r + 8 * h);
          dq.word(h == 0 ? c.y : c.w, r + 8 * h + 4);
        }
        tmem_st_16x256b_x4(a_tmem + as * 32 + lanes + (static_cast<uint32_t>(i * 16) << 16), r);
      }
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(smem_u32(&a_full[as]));
        mbar_arrive(smem_u32(&empty[s]));
      }
      for (int i = 0; i < kDeqGroups / 2; ++i) next_stage();
    }
    if (ok) ok = mbar_wait(smem_u32(&d_full), 0, wctx, kDevTimeoutEpilogue);
    ok = __all_sync(0xffffffffu, ok) != 0;
    tc_fence_after();
  }

  // ---- epilogue: each quarter's warps take every fourth 32 rows of x
  const int q = warp & 3, part = (warp - 2) >> 2, n = tile0 * 16 + q * 32 + tile_column(lane);
  auto store = [&](int64_t row, float v, float bias) {
    v = w4_act(a.act, v + bias);
    if (a.out_f32) {
      static_cast<float*>(a.out)[row * a.l.n + n] = v;
    } else {
      static_cast<uint16_t*>(a.out)[row * a.l.n + n] = static_cast<uint16_t>(Elem<T>::pack(v, 0.0f));
    }
  };
  const bool has_n = warp >= 2 && n < a.l.n;
  const float bias = has_n && a.bias != nullptr ? Elem<T>::to_f(static_cast<const T*>(a.bias)[n]) : 0.0f;
  if (a.ck == 1) {
    if (warp >= 2 && ok)  // a wait that ran out leaves the rows unwritten
      for (int c0 = part * 32; c0 < a.rows; c0 += 32 * kDeqGroups) {
        if (row0 + c0 >= a.m) break;
        uint32_t v[32];
        tmem_ld32(d_tmem + (static_cast<uint32_t>(q * 32) << 16) + c0, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i)
          if (has_n && c0 + i < a.rows && row0 + c0 + i < a.m) store(row0 + c0 + i, __uint_as_float(v[i]), bias);
      }
  } else {
    // CTA r of the cluster finishes rows [r share, (r + 1) share) of the tile: sums [source][row][128]
    // in its ring, which nothing uses after the first barrier
    const int share = a.rows / a.ck;
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2)
      for (int c0 = part * 32; c0 < a.rows; c0 += 32 * kDeqGroups) {
        uint32_t v[32];
        tmem_ld32(d_tmem + (static_cast<uint32_t>(q * 32) << 16) + c0, v);
        tmem_wait_ld();
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int c = c0 + i;
          if (c >= a.rows) break;
          const uint32_t at = smem_u32(smem) + ((rank * share + c % share) * kTileN + q * 32 + lane) * 4;
          asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_shared(at, static_cast<uint32_t>(c / share))), "r"(v[i])
                       : "memory");
        }
      }
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2 && ok)
      for (int c = part; c < share; c += kDeqGroups) {
        const int64_t row = row0 + rank * share + c;
        float v = 0.0f;
        for (int i = 0; i < a.ck; ++i)
          v += reinterpret_cast<const float*>(smem)[(i * share + c) * kTileN + q * 32 + lane];
        if (has_n && row < a.m) store(row, v, bias);
      }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(d_tmem, a.tmem_cols);
  }
}

int tile_stage_bytes(const W4Layout& l, int rows) {
  return 2 * rows * 128 + kTileTiles * kW4BlockBytes + (kTileTiles * l.scale_bytes() + 1023) / 1024 * 1024;
}

template <typename T, int UNITS, bool ZP>
int tile_launch(const W4TileArgs& a, const CUtensorMap& tx, int64_t ctas, int smem, cudaStream_t s, const PdlIo& io) {
  static unsigned long long done_mask = 0;
  auto kern = &w4_tile_kernel<T, UNITS, ZP>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), kSmemLimit - 1024, &done_mask);
  if (rc != GP_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kTileThreads, 1, 1);
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
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, tx, a);
  pdl.record(io);
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? GP_OK : set_error(GP_ERR_CUDA, "w4 tile launch: %s", cudaGetErrorString(e));
}

template <typename T, int UNITS>
int tile_zeros(const W4TileArgs& a, const CUtensorMap& tx, int64_t ctas, int smem, cudaStream_t s, const PdlIo& io) {
  return a.l.zeros ? tile_launch<T, UNITS, true>(a, tx, ctas, smem, s, io)
                   : tile_launch<T, UNITS, false>(a, tx, ctas, smem, s, io);
}

template <typename T>
int tile_units(const W4TileArgs& a, const CUtensorMap& tx, int64_t ctas, int smem, cudaStream_t s, const PdlIo& io) {
  return a.l.units == 1   ? tile_zeros<T, 1>(a, tx, ctas, smem, s, io)
         : a.l.units == 2 ? tile_zeros<T, 2>(a, tx, ctas, smem, s, io)
                          : tile_zeros<T, 4>(a, tx, ctas, smem, s, io);
}

}  // namespace

int launch_w4_tiles(const W4LinearArgs& in, cudaStream_t s, const DeviceInfo& dev) {
  W4TileArgs a;
  a.l = in.l;
  a.packed = in.packed;
  a.bias = in.bias;
  a.out = in.out;
  a.m = in.m;
  a.out_f32 = in.out_f32;
  a.act = in.act;
  a.status = dev.status;
  a.timeout_ns = current_timeout_ns();
  a.inject = current_fault_injection();
  // rows per tile: as even as multiples of 16 up to 256 allow
  const int64_t row_tiles = (in.m + kMaxTileRows - 1) / kMaxTileRows;
  a.rows = static_cast<int>(((in.m + row_tiles - 1) / row_tiles + 15) / 16 * 16);
  a.row_tiles = static_cast<int>((in.m + a.rows - 1) / a.rows);
  a.tmem_cols = a.rows + kAStages * 32 <= 256 ? 256 : 512;
  const int64_t units = static_cast<int64_t>((a.l.n_tiles + kTileTiles - 1) / kTileTiles) * a.row_tiles;
  // CTAs along K: the fewest rounds over the SMs, a round costing its blocks and about four more
  // (six more with the sums across a cluster)
  int64_t best = -1;
  for (int ck = 1; ck <= 8; ck *= 2) {
    const int slice = (a.l.blocks + ck - 1) / ck;
    if (ck > 1 && ((ck - 1) * slice >= a.l.blocks || a.rows % ck != 0)) break;
    const int64_t cost = (units * ck + dev.sm_count - 1) / dev.sm_count * (slice + (ck > 1 ? 10 : 4));
    if (best >= 0 && cost >= best) continue;
    best = cost;
    a.ck = ck;
    a.slice = slice;
  }
  if (units * a.ck >= (int64_t(1) << 31)) return set_error(GP_ERR_SHAPE, "w4 linear: m = %lld", (long long)in.m);
  // two CTAs share an SM up to 64 rows
  const int stage = tile_stage_bytes(a.l, a.rows);
  const int budget = a.rows <= 64 ? kSmemLimit / 2 - 2048 : kSmemLimit - 1024;
  a.stages = budget / stage;
  if (a.stages > kMaxStages) a.stages = kMaxStages;
  int smem = a.stages * stage;
  const int sums = a.ck > 1 ? a.rows * kTileN * 4 : 0;
  if (smem < sums) smem = sums;
  CUtensorMap tx;
  int rc = make_tmap_2d(&tx, in.x, in.dtype, static_cast<uint64_t>(in.m), static_cast<uint64_t>(a.l.k), 64,
                        static_cast<uint32_t>(a.rows), 128);
  if (rc != GP_OK) return rc;
  PdlIo io;
  io.add(PdlIo::kWrite, in.out, static_cast<uint64_t>(in.m) * a.l.n * (in.out_f32 ? 4 : 2));
  rc = in.dtype == GP_BF16 ? tile_units<__nv_bfloat16>(a, tx, units * a.ck, smem, s, io)
                           : tile_units<__half>(a, tx, units * a.ck, smem, s, io);
  if (rc == GP_OK) count_launches(1);
  return rc;
}

}  // namespace gp
