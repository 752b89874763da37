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
// kernel does, would read the accumulator once per group: more time than the tile's product. In a
// chain (EXACT), whose layers' errors add up, the operand is two T per weight instead, the rounded one
// and what rounding took away, with a product each: the weight is then exact. Likewise x may be two T
// (planes): its second part meets the first part of the weights (second by second is at most 2^-16 of
// a bf16 product, a 256th of what the output's rounding takes; 2^-22 for fp16).
//
// The unit is a k-block of 128 rows of W:
//   loader (1 thread)   x panels (two of 64 columns) by TMA into a ring of stages
//   dequantising warps  four groups of four (one warp per TMEM lane quarter); the groups take the
//                       blocks in turn. Each lane copies its own codes and scales with cp.async into a
//                       private ring, one or two blocks ahead, turns them into T in registers and
//                       stores them to the group's TMEM stage of 64 columns. A turn's waits and
//                       fences take as long as the conversion of 64 rows does, hence whole blocks
//                       (half of one where a weight is two T: as many columns).
//   MMA issuer (1 thread) eight K = 16 products per block; commits free the TMEM stage and the x stage.
//                       With two T per weight there are two issuers, as a turn then is half a block
//                       and an issuer's wait is answered behind its own products (4,096 -> 14,336 ->
//                       4,096 at 32 rows: 53 us with one, 41 with two; single layers gain nothing): up to
//                       128 rows they take the turns alternately, each with an accumulator; above,
//                       each has half of the rows.
//   epilogue            the dequantising warps: bias, activation, store
// Where there are fewer tiles than SMs, a cluster of ck CTAs splits K and sums over distributed
// shared memory in a fixed order.
#include "../../include/gpipes.h"
#include "chain_registry.h"
#include "w4.cuh"

#include <type_traits>

namespace gp {
namespace {

// Groups of four dequantising warps, one warp per TMEM lane quarter: four, but two above 128 rows of x with
// zero points in groups of 32. There the code rings of four groups leave no room for two x stages of 256
// rows (512 x 4,096 x 14,336: 97 us in tiles of 128 rows, 76 with two groups), and the products of a
// block take longer than its conversion anyway. Elsewhere four are no slower (62 us; two: 65).
constexpr int tile_threads(int groups, bool exact) { return 32 * ((exact ? 3 : 2) + 4 * groups); }
constexpr int kTileN = 128;        // columns of W per tile: the TMEM lanes
constexpr int kTileTiles = kTileN / 16;
// a TMEM stage of dequantised weights per group: 64 columns, a block
constexpr int kACols = 64;
constexpr int kTmemCols = 512;            // 256 for the sums, 256 for the weights
constexpr int kMaxStages = 4;       // x stages
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
  int planes;      // of x
  int out_planes;
  int stages;      // x stages
  int depth;       // slots of a warp's code ring (2 or 3)
  int groups;
  int exact;
  int* status;
  unsigned long long timeout_ns;
  int inject;
};

template <int BYTES>
__device__ __forceinline__ void cp_async(uint32_t dst, const void* src) {
  if constexpr (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES) : "memory");
}

// Words of scales that a lane needs per turn (a block, or with two T per weight a 64-row part of it), and a
// warp's slot: for its two column tiles, a turn's codes and scales of each lane
constexpr int turn_words(int units, bool zp, bool exact) { return (exact && units > 1 ? units / 2 : units) * (zp ? 2 : 1); }
constexpr int code_slot(int units, bool zp, bool exact) {
  return 2 * 32 * ((exact ? 16 : 32) + 4 * turn_words(units, zp, exact));
}

// One lane of the (converged) warp, always the same one.
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
  return e != 0;
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

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr));
}

// TMEM lane of a tile <-> column: lane 16 i + r holds column 16 i + 2 (r % 8) + r / 8
__device__ __forceinline__ int tile_column(int lane) { return (lane & ~15) + 2 * (lane & 7) + ((lane >> 3) & 1); }

template <typename T, int UNITS, bool ZP, int GROUPS, bool EXACT>
__global__ void __launch_bounds__(tile_threads(GROUPS, EXACT), 1)
    w4_tile_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ W4TileArgs a) {
  constexpr int kWords = UNITS * (ZP ? 2 : 1);
  constexpr int kScaleBytes = 32 * kWords;            // of a block of 16 columns
  constexpr int kUse = turn_words(UNITS, ZP, EXACT);
  constexpr int kSlot = code_slot(UNITS, ZP, EXACT);
  constexpr int kTurns = EXACT ? 2 : 1;               // turns per block: the groups then take 64-row parts in turn
  static_assert(!EXACT || GROUPS == 4, "a group keeps to one part of its blocks");
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ __align__(8) uint64_t full[kMaxStages], empty[kMaxStages], a_full[GROUPS], a_empty[GROUPS], d_full;
  __shared__ uint32_t tmem_holder;
  __shared__ int abort_flag;
  const int panel = a.rows * 128, stage_bytes = 2 * panel * a.planes;  // x rows of 64 columns, SWIZZLE_128B
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = a.ck > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / a.ck;
  const int tile0 = unit / a.row_tiles * kTileTiles;  // first 16-column tile
  const int64_t row0 = static_cast<int64_t>(unit % a.row_tiles) * a.rows;
  const int b0 = rank * a.slice, nb = min(a.slice, a.l.blocks - b0);
  const int tiles = min(kTileTiles, a.l.n_tiles - tile0);

  // With as many x stages as TMEM stages, a block's x panels and weights share one barrier for "full" and
  // one for "free": one wait and one commit less per turn of the MMA issuer, whose turns bound the kernel
  // at few rows.
  const bool merged = !EXACT && a.stages == GROUPS;
  const bool split = EXACT && a.rows > 128;  // the two issuers take half of the rows each; else every other turn
  const uint32_t full0 = smem_u32(merged ? a_full : full), empty0 = smem_u32(merged ? a_empty : empty);

  if ((smem_u32(smem) & 1023u) != 0) {  // the same in every CTA of the grid
    pdl_wait_prior();
    if (threadIdx.x == 0) atomicCAS(a.status, 0, kDevBadSmemAlign);
    return;
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < a.stages; ++i) {
      mbar_init(smem_u32(&full[i]), 1);
      mbar_init(smem_u32(&empty[i]), EXACT ? 2 : 1);
    }
    for (int i = 0; i < GROUPS; ++i) {
      mbar_init(smem_u32(&a_full[i]), merged ? 5 : 4);  // the group's warps (and the x panels)
      mbar_init(smem_u32(&a_empty[i]), split ? 2 : 1);
    }
    mbar_init(smem_u32(&d_full), EXACT ? 2 : 1);
    abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0 && lane == 0) prefetch_tmap(&tx);
  // The first codes go into L2 while the previous kernel of the stream drains (a hint: nothing is
  // read into the program before the wait).
  if (warp >= 2 && warp < 2 + tiles && lane < min(2 * nb, 16))
    asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(
                     static_cast<const uint8_t*>(a.packed) +
                     (static_cast<int64_t>(tile0 + warp - 2) * a.l.blocks + b0) * kW4BlockBytes + lane * (kW4BlockBytes / 2)),
                 "n"(kW4BlockBytes / 2));
  pdl_wait_prior();
  pdl_launch_dependents();
  if (warp == 1) {
    tmem_alloc(smem_u32(&tmem_holder), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t d_tmem = tmem_holder, a_tmem = d_tmem + (kTmemCols - GROUPS * kACols);
  const WaitCtx wctx{a.status, &abort_flag, a.timeout_ns};
  const bool worker = warp >= 2 && warp < 2 + 4 * GROUPS;  // dequantises, then stores
  bool ok = true;  // of this role

  if (warp == 0) {
    if (lane == 0 && a.inject == 0) {
      const uint64_t keep = l2_policy_evict_last();  // x is read by every column tile
      int s = 0, ph = 0;
      for (int b = 0; b < nb; ++b) {
        if (b >= a.stages && !mbar_wait(empty0 + s * 8, ph ^ 1, wctx, kDevTimeoutProducer)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(full0 + s * 8, stage_bytes);
        for (int p = 0; p < 2 * a.planes; ++p)  // rows past m of the first plane are not stored
          tma_load_2d_hint(smem_u32(smem) + s * stage_bytes + p * panel, &tx, full0 + s * 8,
                           (b0 + b) * kW4Block + (p & 1) * 64, static_cast<int>(row0 + (p >> 1) * a.m), keep);
        if (++s == a.stages) s = 0, ph ^= 1;
      }
      if (!ok)  // copies under way end (waited for with a limit) before their memory is used again or goes away
        for (int j = 0; j < a.stages; ++j) {
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(full0 + s * 8, ph ^ 1) && globaltimer_ns() - t0 < a.timeout_ns) {
          }
          if (++s == a.stages) s = 0, ph ^= 1;
        }
    }
    __syncwarp();
  } else if (!worker) {
    // The whole warp runs the loop and one elected lane issues: the compiler then sees addresses and
    // descriptors that are the same in all lanes and keeps them in uniform registers, where the
    // product wants them (from a branch on lane 0, each product took 72 cycles to issue).
    const int me = warp == 1 ? 0 : 1, mine = split ? a.rows / 2 : a.rows;  // rows of this issuer's products
    const uint32_t idesc = make_idesc_f16(kTileN, mine, Elem<T>::kIsBf16, 0, 0);
    const uint32_t d = __shfl_sync(0xffffffffu, d_tmem + me * mine, 0), at0 = __shfl_sync(0xffffffffu, a_tmem, 0);
    const uint64_t desc0 = make_sdesc_sw128(smem_u32(smem) + (split ? me * mine * 128 : 0), 16, 1024);
    const int turn0 = split ? 0 : me, step = EXACT && !split ? 2 : 1;
    const uint32_t a_full0 = smem_u32(a_full), a_empty0 = smem_u32(a_empty);
    int s = 0, ph = 0, as = turn0, aph = 0;
    for (int turn = turn0; turn < kTurns * nb; turn += step) {
      const int part = EXACT ? turn & 1 : 0;
      const bool both = EXACT && split;  // the turns of a block's two parts are this issuer's
      ok = mbar_wait(a_full0 + as * 8, aph, wctx, kDevTimeoutMma) &&
           (merged || (both && part != 0) || mbar_wait(full0 + s * 8, ph, wctx, kDevTimeoutMma));
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint64_t bdesc = desc0 + static_cast<uint64_t>((s * stage_bytes + part * panel) >> 4);
      if (elect_one()) {
        const uint32_t stage = at0 + as * kACols;
        auto more = [&](int k) { return (turn != turn0 || k > 0) ? 1u : 0u; };
        if constexpr (EXACT) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(d, stage + k * 8, bdesc + static_cast<uint64_t>(k * 2), idesc, more(k));
#pragma unroll
          for (int k = 0; k < 4; ++k)
            mma_ts(d, stage + 32 + k * 8, bdesc + static_cast<uint64_t>(k * 2), idesc, 1u);
          if (a.planes == 2)
#pragma unroll
            for (int k = 0; k < 4; ++k)
              mma_ts(d, stage + k * 8, bdesc + static_cast<uint64_t>((panel >> 3) + k * 2), idesc, 1u);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_ts(d, stage + k * 8,
                   bdesc + static_cast<uint64_t>((k >> 2) * (panel >> 4) + (k & 3) * 2), idesc, more(k));
        }
        mma_commit(a_empty0 + as * 8);
        if (!merged && (!both || part == 1)) mma_commit(empty0 + s * 8);
      }
      __syncwarp();
      as += step;
      if (as >= GROUPS) as -= GROUPS, aph ^= 1;
      if (!both || part == 1)
        if (++s == a.stages) s = 0, ph ^= 1;
    }
    // every product issued has completed before TMEM is read or released
    if (elect_one()) mma_commit(smem_u32(&d_full));
    __syncwarp();
    volatile int no_abort = 0;
    const WaitCtx drain{a.status, &no_abort, a.timeout_ns};
    mbar_wait(smem_u32(&d_full), 0, drain, kDevTimeoutMma);
    __syncwarp();
  } else {
    const int q = warp & 3, group = (warp - 2) >> 2, g = lane >> 2;
    const uint32_t lanes = static_cast<uint32_t>(q * 32) << 16;
    const uint32_t ring = smem_u32(smem) + a.stages * stage_bytes + (warp - 2) * (a.depth * kSlot);
    // this warp's two column tiles of the tile's eight; an absent one stays zero
    const bool have[2] = {2 * q < tiles, 2 * q + 1 < tiles};
    const uint8_t *codes[2], *scales[2];
    const int my_part = EXACT ? group & 1 : 0, first = EXACT ? group >> 1 : group;
    constexpr int kStep = GROUPS / kTurns;  // blocks from a turn of this group to its next
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t cell = static_cast<int64_t>(tile0 + 2 * q + i) * a.l.blocks + b0 + first;
      codes[i] = static_cast<const uint8_t*>(a.packed) + cell * kW4BlockBytes + my_part * (kW4BlockBytes / 2) + lane * 16;
      scales[i] = static_cast<const uint8_t*>(a.packed) + a.l.scale_off + cell * kScaleBytes + g * (4 * kWords) +
                  (kUse < kWords ? my_part * (4 * kUse) : 0);
    }
    constexpr int kTurnCodes = kW4BlockBytes / kTurns;  // of a column tile
    const uint32_t my_codes = ring + lane * 16, my_scales = ring + 2 * kTurnCodes + lane * (4 * kUse);
    const uint32_t ring_end = a.depth * kSlot;
    int ld_b = first;
    uint32_t ld_at = 0;  // byte offset of the slot that is filled next
    auto load = [&] {
      if (ld_b < nb) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (have[i]) {
            cp_async<16>(my_codes + ld_at + i * kTurnCodes, codes[i]);
            if constexpr (!EXACT) cp_async<16>(my_codes + ld_at + i * kTurnCodes + 512, codes[i] + kW4BlockBytes / 2);
            if constexpr (kUse == 8) {
              cp_async<16>(my_scales + ld_at + i * (128 * kUse), scales[i]);
              cp_async<16>(my_scales + ld_at + i * (128 * kUse) + 16, scales[i] + 16);
            } else {
              cp_async<4 * kUse>(my_scales + ld_at + i * (128 * kUse), scales[i]);
            }
          }
          codes[i] += kStep * kW4BlockBytes;
          scales[i] += kStep * kScaleBytes;
        }
      }
      ld_b += kStep;
      ld_at = ld_at + kSlot == ring_end ? 0 : ld_at + kSlot;
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int i = 1; i < a.depth; ++i) load();
    uint32_t at = 0;
    const uint32_t a_stage = a_tmem + group * kACols + lanes;
    int parity = 1;  // of the stage's last use
    // codes and scales of a column tile's 64 rows to T: r, and with two T per weight rest
    auto convert = [&](int i, int part, uint32_t* r, uint32_t* rest) {
      uint32_t c[4] = {0, 0, 0, 0}, sw[kUse];
#pragma unroll
      for (int w = 0; w < kUse; ++w) sw[w] = 0;
      if (have[i]) {
        w4_lds<4>(my_codes + at + i * kTurnCodes + part * 512, c);
        w4_lds<kUse>(my_scales + at + i * (128 * kUse), sw);
      }
      auto words = [&](auto large) {
        W4Exact<T> dq;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          constexpr int kPer = ZP ? 2 : 1;
          const int u = (UNITS == 1 ? 0 : UNITS == 2 ? part : 2 * part + h) * kPer;
          if (UNITS == 4 || h == 0) dq.set(sw[u], sw[u + kPer - 1], ZP);
          dq.word(c[2 * h], r + 8 * h, rest == nullptr ? nullptr : rest + 8 * h, large);
          dq.word(c[2 * h + 1], r + 8 * h + 4, rest == nullptr ? nullptr : rest + 8 * h + 4, large);
        }
      };
      bool large = false;
      if constexpr (EXACT)
#pragma unroll
        for (int w = 0; w < kUse; w += ZP ? 2 : 1) large |= w4_large<T>(sw[w]);
      if (EXACT && __any_sync(0xffffffffu, large)) words(std::true_type{});
      else words(std::false_type{});
    };
    // the TMEM stage is free: its last products have completed
    auto stage_free = [&](bool never_used) {
      ok = never_used || mbar_wait(smem_u32(&a_empty[group]), parity, wctx, kDevTimeoutEpilogue);
      ok = __all_sync(0xffffffffu, ok) != 0;
      if (ok) tc_fence_after();
      return ok;
    };
    for (int b = first; b < nb; b += kStep, parity ^= 1) {
      load();
      if (a.depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
      else asm volatile("cp.async.wait_group 1;" ::: "memory");
      // in registers first; the stage is only then waited for
      if constexpr (EXACT) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t r[16], rest[16];
          convert(i, 0, r, rest);
          if (i == 0 && !stage_free(b == first)) break;
          tmem_st_16x256b_x4(a_stage + (static_cast<uint32_t>(i * 16) << 16), r);
          tmem_st_16x256b_x4(a_stage + 32 + (static_cast<uint32_t>(i * 16) << 16), rest);
        }
      } else {
#pragma unroll
        for (int part = 0; part < 2; ++part) {
          uint32_t r[2][16];
          convert(0, part, r[0], nullptr);
          convert(1, part, r[1], nullptr);
          if (part == 0 && !stage_free(b == first)) break;
#pragma unroll
          for (int i = 0; i < 2; ++i)
            tmem_st_16x256b_x4(a_stage + part * 32 + (static_cast<uint32_t>(i * 16) << 16), r[i]);
        }
      }
      if (!ok) break;
      at = at + kSlot == ring_end ? 0 : at + kSlot;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&a_full[group]));
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (ok) ok = mbar_wait(smem_u32(&d_full), 0, wctx, kDevTimeoutEpilogue);
    ok = __all_sync(0xffffffffu, ok) != 0;
    tc_fence_after();
  }

  // ---- epilogue: each quarter's warps take every fourth 8 rows of x (short loops: their code runs
  // once per CTA, so its length is its cost)
  const int q = warp & 3, quarter = (warp - 2) >> 2, n = tile0 * 16 + q * 32 + tile_column(lane);
  const bool has_n = worker && n < a.l.n;
  const float bias = has_n && a.bias != nullptr ? Elem<T>::to_f(static_cast<const T*>(a.bias)[n]) : 0.0f;
  // rows row, row + 1, ... of column n: the first `live` of v
  auto store = [&](int64_t row, auto& v, int live) {
    constexpr int kN = sizeof(v) / sizeof(float);
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] += bias;
    w4_act(a.act, v);
    const int64_t at = row * a.l.n + n;
    if (a.out_f32) {
      float* to = static_cast<float*>(a.out) + at;
#pragma unroll
      for (int i = 0; i < kN; ++i, to += a.l.n)
        if (i < live) *to = v[i];
    } else {
      uint16_t* to = static_cast<uint16_t*>(a.out) + at;
      const int64_t plane = a.m * a.l.n;
#pragma unroll
      for (int i = 0; i < kN; ++i, to += a.l.n) {
        uint16_t hi, lo;
        w4_two<T>(v[i], hi, lo);
        if (i < live) *to = hi;
        if (EXACT && i < live && a.out_planes == 2) to[plane] = lo;
      }
    }
  };
  const uint32_t d_lanes = d_tmem + (static_cast<uint32_t>(q * 32) << 16);
  auto load_sums = [&](int c0, float (&v)[8]) {
    uint32_t u[8], w[8];
    const bool two = EXACT && !split;  // an accumulator of each issuer (a block has a turn for both)
    tmem_ld8(d_lanes + c0, u);
    if (two) tmem_ld8(d_lanes + a.rows + c0, w);
    tmem_wait_ld();
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u[i]) + (two ? __uint_as_float(w[i]) : 0.0f);
  };
  if (a.ck == 1) {
    if (worker && ok)  // a wait that ran out leaves the rows unwritten
#pragma unroll 1
      for (int c0 = quarter * 8; c0 < a.rows && row0 + c0 < a.m; c0 += 8 * GROUPS) {
        float v[8];
        load_sums(c0, v);
        store(row0 + c0, v, has_n ? static_cast<int>(min(static_cast<int64_t>(8), a.m - row0 - c0)) : 0);
      }
  } else {
    // CTA r of the cluster finishes rows [r share, (r + 1) share) of the tile: sums [source][row][128]
    // in its shared memory, which nothing else uses after the first barrier
    const int share = a.rows / a.ck;
    __syncwarp();
    cluster_sync_all();
    if (worker)
#pragma unroll 1
      for (int c0 = quarter * 8; c0 < a.rows; c0 += 8 * GROUPS) {
        float v[8];
        load_sums(c0, v);
        int owner = c0 / share, r = c0 % share;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const uint32_t at = smem_u32(smem) + ((rank * share + r) * kTileN + q * 32 + lane) * 4;
          asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(at, static_cast<uint32_t>(owner))), "f"(v[i])
                       : "memory");
          if (++r == share) r = 0, ++owner;
        }
      }
    __syncwarp();
    cluster_sync_all();
    if (worker && ok)
#pragma unroll 1
      for (int c = quarter; c < share; c += GROUPS) {
        const int64_t row = row0 + rank * share + c;
        float v[1] = {0.0f};
        for (int i = 0; i < a.ck; ++i)
          v[0] += reinterpret_cast<const float*>(smem)[(i * share + c) * kTileN + q * 32 + lane];
        store(row, v, has_n && row < a.m ? 1 : 0);
      }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(d_tmem, kTmemCols);
  }
}

template <typename T, int UNITS, bool ZP, int GROUPS, bool EXACT>
int tile_launch(const W4TileArgs& a, const CUtensorMap& tx, int64_t ctas, int smem, cudaStream_t s, const PdlIo& io) {
  static unsigned long long done_mask = 0;
  auto kern = &w4_tile_kernel<T, UNITS, ZP, GROUPS, EXACT>;
  int rc = ensure_smem_attr(reinterpret_cast<const void*>(kern), kSmemLimit - 2048, &done_mask);
  if (rc != GP_OK) return rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(tile_threads(GROUPS, EXACT), 1, 1);
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

template <typename T, int UNITS, bool ZP>
int tile_groups(const W4TileArgs& a, const CUtensorMap& tx, int64_t ctas, int smem, cudaStream_t s, const PdlIo& io) {
  if (a.exact) return tile_launch<T, UNITS, ZP, 4, true>(a, tx, ctas, smem, s, io);
  if constexpr (UNITS == 4 && ZP)
    if (a.groups == 2) return tile_launch<T, UNITS, ZP, 2, false>(a, tx, ctas, smem, s, io);
  return tile_launch<T, UNITS, ZP, 4, false>(a, tx, ctas, smem, s, io);
}

template <typename T, int UNITS>
int tile_zeros(const W4TileArgs& a, const CUtensorMap& tx, int64_t ctas, int smem, cudaStream_t s, const PdlIo& io) {
  return a.l.zeros ? tile_groups<T, UNITS, true>(a, tx, ctas, smem, s, io)
                   : tile_groups<T, UNITS, false>(a, tx, ctas, smem, s, io);
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
  a.planes = in.x_planes;
  a.out_planes = in.out_planes;
  a.exact = in.exact || in.x_planes == 2 || in.out_planes == 2;
  a.status = dev.status;
  a.timeout_ns = current_timeout_ns();
  a.inject = current_fault_injection();
  static std::atomic<int> cluster_cache[64][4];
  static unsigned long long probe_mask = 0;
  const void* probe = reinterpret_cast<const void*>(&w4_tile_kernel<__half, 1, false, 4, false>);
  int rc = ensure_smem_attr(probe, kSmemLimit - 2048, &probe_mask);
  if (rc != GP_OK) return rc;
  // Rows per tile and CTAs along K, by time in hundredths of a microsecond. A round of what runs at once
  // costs 280 and a row's share to start and end, 180 more with sums across a cluster, and per block 34 (two T per
  // weight: 42) and what its rows add, as measured at 32 to 256 rows. Rows: as even as multiples of 16
  // (32 where two issuers halve them) allow, up to 256, or 128 where x is two T (a stage of 256 such rows
  // takes 128 KB); fewer, down to 64, where that puts more SMs to work.
  const int64_t most = a.planes == 2 ? kMaxTileRows / 2 : kMaxTileRows, columns = (a.l.n_tiles + kTileTiles - 1) / kTileTiles;
  int64_t best = -1, units = 0;
  for (int64_t row_tiles = (in.m + most - 1) / most;; row_tiles *= 2) {
    int rows = static_cast<int>(((in.m + row_tiles - 1) / row_tiles + 15) / 16 * 16);
    if (a.exact && rows > 128) rows = (rows + 31) / 32 * 32;
    const int64_t n = columns * ((in.m + rows - 1) / rows);
    for (int ck = 1; ck <= 8; ck *= 2) {
      const int slice = (a.l.blocks + ck - 1) / ck;
      if (ck > 1 && ((ck - 1) * slice >= a.l.blocks || rows % ck != 0)) break;
      const int at_once = w4_max_clusters(probe, tile_threads(4, false), kSmemLimit - 2048, ck, dev.sm_count, cluster_cache);
      const int64_t block = a.exact ? 42 + rows / 3 : 34 + rows / 6;
      const int64_t cost = (n + at_once - 1) / at_once * (block * slice + rows / 2 + (ck > 1 ? 460 : 280));
      if (best >= 0 && cost >= best) continue;
      best = cost;
      units = n;
      a.rows = rows;
      a.ck = ck;
      a.slice = slice;
    }
    if (rows <= 64) break;
  }
  a.row_tiles = static_cast<int>(units / columns);
  if (units * a.ck >= (int64_t(1) << 31)) return set_error(GP_ERR_SHAPE, "w4 linear: m = %lld", (long long)in.m);
  const int stage = 2 * a.rows * 128 * a.planes;
  a.groups = !a.exact && a.rows > 128 && a.l.units == 4 && a.l.zeros != 0 ? 2 : 4;
  const int slot = 4 * a.groups * code_slot(a.l.units, a.l.zeros != 0, a.exact != 0);
  // as many x stages as groups where that fits; then code slots, three if possible
  const int budget = kSmemLimit - 2048;
  a.depth = a.groups * stage + 3 * slot <= budget ? 3 : 2;
  const int rings = a.depth * slot;
  a.stages = (budget - rings) / stage;
  if (a.stages > a.groups) a.stages = a.groups;
  int smem = a.stages * stage + rings;
  const int sums = a.ck > 1 ? a.rows * kTileN * 4 : 0;
  if (smem < sums) smem = sums;
  CUtensorMap tx;
  rc = make_tmap_2d(&tx, in.x, in.dtype, static_cast<uint64_t>(in.m) * a.planes, static_cast<uint64_t>(a.l.k), 64,
                        static_cast<uint32_t>(a.rows), 128);
  if (rc != GP_OK) return rc;
  PdlIo io;
  io.add(PdlIo::kWrite, in.out, static_cast<uint64_t>(in.m) * a.l.n * (in.out_f32 ? 4 : 2 * a.out_planes));
  rc = in.dtype == GP_BF16 ? tile_units<__nv_bfloat16>(a, tx, units * a.ck, smem, s, io)
                           : tile_units<__half>(a, tx, units * a.ck, smem, s, io);
  if (rc == GP_OK) count_launches(1);
  return rc;
}

}  // namespace gp
