// Feed-forward products on 2-CTA pairs (tcgen05, TMEM), and their gradients.
//
//   gated  H[r, n]      = act(sum_k A[r, k] Wg[e, n, k]) * sum_k A[r, k] Wu[e, n, k]
//   act    C[r, n]      = act(sum_k A[r, k] W[n, k] + bias[n]) + R[r, n]
//   dA     dA[r, k]     = sum_h sum_n dz[h, r, n] Wh[e, n, k]
//   dW     dW[h, e, n, k] = sum_r dz[h, r, n] A[r, k]       r over expert e's rows
//
// As in grouped_gemm.cuh the weight's axis is the MMA's M = 256 and the tokens
// are its N (a multiple of 32, up to 256), so a ragged group of rows costs its
// rows rounded up to 32, and an operand whose contraction runs along rows is read
// MN-major as it lies.
//
// gated: a CTA's 128 accumulator lanes are 64 gate rows and the 64 up rows of the
// same features -- two boxes of a stage's weight tile -- so one MMA makes both
// products and a tile's traffic is that of a plain product of 2N columns.
// A feature's two values lie 64 lanes apart: the epilogue brings them together in
// shared memory (ffn_epilogue.cuh).  dA takes both weights in one contraction of
// 2N, so the sum over the halves is made in TMEM.
//
// Tiles that would leave pairs idle in a last wave are divided along the contraction
// into equal ranges, one per pair, and come first, so that joining them hides behind
// the others' products.  Whichever CTA arrives last adds the parts up in their order:
// the sums do not depend on which one it was, and nobody waits for another.
//
// Bound by the tensor pipe (84 to 90 % active): 4095 rows, 28672 x 4096, gated 597 us, dA
// 672, dW 617 (1.61, 1.43, 1.56 PFLOP/s, 0.87 to 0.98 of a large library product's rate).
//
// Eight epilogue warps, two groups of four: a group takes every other 16 tokens of its
// tile.  gated and dA have sixteen, eight for each accumulator, because a round of 16
// tokens mostly waits (4096 rows x 8192 x 256 gated 33.5 us with eight, 29.8 so); act's
// epilogue does not fit the registers that leaves (8192 x 1024 50.1 and 54.1), so it stages
// its rounds in turn in two places instead.
#pragma once
#include "ffn_epilogue.cuh"

namespace b200 {

enum FfnMode : int { kFfnGated = 0, kFfnAct = 1, kFfnDA = 2, kFfnDW = 3 };

struct FfnArgs {
  const int* offsets;  // null: one group of all rows
  int experts, rows;
  int feat;    // extent of the MMA's M axis: N (gated, act, dW: of one half) or K (dA)
  int red;     // contraction extent: K (gated, act) or N (dA: of one half); unused in dW
  int cols;    // dW: extent of the MMA's N axis, K
  int halves;  // dA, dW: 1 or 2
  int group;   // raster band
  int tile_n;  // tokens (dW: columns) of a tile, at the most
  FfnOut o;    // dW: out where TMA cannot write it (contiguous), else null
  float* slots;          // [CTA][2][256][128] partial sums, or null: no tile is divided
  unsigned int* counts;  // [pair][16], zero between launches
  const CUtensorMap* maps;  // dW with offsets: dz's and A's map of each expert
  int* status;
  unsigned long long timeout_ns;
};

// Four stagings of 16 tokens: one to a group of epilogue warps, or two where there are two
// groups; dW stages 64 columns of a warp's 32 rows.  For many experts (kMany) a stage is
// given up for the table of their rows.
template <int kMode, bool kMany = false>
struct FfnCfg {
  static constexpr int kStages = kMany ? 5 : 6;
  static constexpr int kOperand = 128 * kSlabK * 2;
  static constexpr int kStageBytes = 2 * kOperand;
  static constexpr int kSets = kMode == kFfnGated || kMode == kFfnDA ? 2 : 1;  // of eight warps
  static constexpr int kThreads = 32 * (2 + 8 * kSets);
  static constexpr int kStaging = kMode == kFfnDW ? 8 * kStoreBufBytes : 4 * kFfnStageBytes;
  static constexpr int kFeat = kMode == kFfnGated ? 128 : 256;  // output features of a tile
  static constexpr int smem_bytes(int experts) {
    return kStages * kStageBytes + kStaging + group_table_bytes(experts) + 1024;
  }
};

// The table of rows by expert; without offsets, one group of all of them.
__device__ __forceinline__ void ffn_groups(const int* offsets, int experts, int rows, int tile,
                                           int* status, int* s_off, int* s_tiles) {
  if (offsets != nullptr) {
    const bool bad = build_groups(offsets, experts, rows, tile, s_off, s_tiles);
    if (bad && blockIdx.x == 0 && (threadIdx.x & 31) == 0) atomicCAS(status, 0, kErrOffsets);
  } else if ((threadIdx.x & 31) == 0) {
    s_off[0] = s_tiles[0] = 0;
    s_off[1] = rows;
    s_tiles[1] = (rows + tile - 1) / tile;
  }
}

// dW: maps[2 e] and maps[2 e + 1] are dz's (n, r, half) and A's (k, r) tensor maps,
// ended at the last row of expert e, so that the rows past it read as zero.
template <int kUnused = 0>
__global__ void __launch_bounds__(32)
ffn_maps_kernel(const __grid_constant__ CUtensorMap tmap_dz,
                const __grid_constant__ CUtensorMap tmap_a, const int* offsets, int rows,
                CUtensorMap* maps) {
  __shared__ alignas(128) CUtensorMap map[2];
  grid_wait();
  grid_launch_next();
  const int e = blockIdx.x, lane = threadIdx.x;
  uint32_t* words = reinterpret_cast<uint32_t*>(map);
  words[lane] = reinterpret_cast<const uint32_t*>(&tmap_dz)[lane];
  words[32 + lane] = reinterpret_cast<const uint32_t*>(&tmap_a)[lane];
  // The end of expert e as build_groups has it: the largest of the clamped
  // offsets up to its own.
  int end = 0;
  for (int i = lane; i <= e + 1; i += 32) end = max(end, min(offsets[i], rows));
  end = __reduce_max_sync(0xffffffffu, end);
  __syncwarp();
  if (lane == 0) {
    // (an extent is at least 1; an expert that ends at row 0 has no rows)
    tmap_set_rows(smem_u32(&map[0]), end > 0 ? (uint32_t)end : 1u);
    tmap_set_rows(smem_u32(&map[1]), end > 0 ? (uint32_t)end : 1u);
  }
  __syncwarp();
  tmap_publish(maps + 2 * e, smem_u32(&map[0]));
  tmap_publish(maps + 2 * e + 1, smem_u32(&map[1]));
}

struct FfnUnit {
  int e, half;     // half: dW
  int row0, rows;  // the expert's rows (dW), or the tile's
  int feat0, col0;
  int blocks;  // 64-long contraction blocks
  int mma_n;
};

// a / b for 0 <= a < 2^30, b > 0.  Three of them find a unit's place, on the way of
// every tile: by the reciprocal they take a third of the compiler's division.
__device__ __forceinline__ int quick_div(int a, int b) {
  if (a >= 1 << 22) return a / b;
  int q = __float2int_rz(__fdividef((float)a, (float)b));  // off by one at the most
  const int r = a - q * b;
  q += r >= b ? 1 : r < 0 ? -1 : 0;
  return q;
}

// tile_coord's bands of tile-rows.
__device__ __forceinline__ void band_coord(int t, int tiles_m, int tiles_n, int group, int* tm,
                                           int* tn) {
  const int band = quick_div(t, group * tiles_n);
  const int first = band * group, width = min(tiles_m - first, group);
  const int r = t - band * group * tiles_n;
  const int b = quick_div(r, width);
  *tm = first + r - b * width;
  *tn = (band & 1) ? tiles_n - 1 - b : b;
}

// What a pair does of a unit: contraction blocks [kb0, kb1).
struct FfnSegment : FfnUnit {
  int kb0, kb1;
  int c0, c1;  // the first and last pair with a part of it
  __device__ __forceinline__ bool whole() const { return kb0 == 0 && kb1 == blocks; }
};

// A pair's parts of the divided units, then its whole ones.  The expert of the last
// unit found is remembered, so a walk over increasing units costs one pass over the table.
template <int kMode>
struct FfnWalk {
  static constexpr int kLeastBlocks = 8;  // of a part
  static constexpr int kJoinBlocks = 12;
  const int* off;
  const int* tiles;
  int tf, tc;  // feature tiles; dW: column tiles
  int e;
  int next_unit, pairs, undivided;  // units [0, undivided) are dealt whole
  int blocks;                       // of a divided unit
  long long items, pos, hi;
  int ranges;
  __device__ __forceinline__ void init(const FfnArgs& a, const int* s_off, const int* s_tiles) {
    constexpr int kFeat = FfnCfg<kMode>::kFeat;
    off = s_off;
    tiles = s_tiles;
    tf = (a.feat + kFeat - 1) / kFeat;
    tc = (a.cols + 255) / 256;
    e = 0;
    const int total = kMode == kFfnDW ? a.experts * a.halves * tf * tc : tiles[a.experts] * tf;
    const int pair = blockIdx.x >> 1;
    pairs = gridDim.x >> 1;
    next_unit = pair;
    undivided = total;
    pos = hi = 0;
    ranges = 0;
    if (a.slots == nullptr) return;
    const int rest = total % pairs;
    blocks = ((kMode == kFfnDW ? a.rows : a.red) + kSlabK - 1) / kSlabK *
             (kMode == kFfnDA ? a.halves : 1);
    items = (long long)rest * blocks;
    ranges = (int)min(items / kLeastBlocks, (long long)pairs);
    undivided = total - rest;
    // Joining costs, in contraction blocks, what the parts' way through L2 takes (there
    // are about ranges + rest of them): dividing has to save more, and whole tiles must
    // follow that hide it.  Measured, us, divided / not: 28672 x 4096 gated, 96 rows (38
    // tiles left of 112) 48 / 51, 384 rows (2 of 224) 79 / 87; 8192 x 8192, 1024 rows (54 of
    // 128, not divided by this) 105 / 100, 2048 rows (34 of 256) 189 / 193.
    const long long join = kJoinBlocks + (ranges + rest) * a.tile_n / 896ll;
    if (ranges == 0 || undivided == 0 || (items + ranges - 1) / ranges + join >= blocks) {
      ranges = 0;
      undivided = total;
      return;
    }
    if (pair < ranges) sk_range(pair, items, ranges, &pos, &hi);
  }

  __device__ __forceinline__ void unit(const FfnArgs& a, int u, FfnUnit* r) {
    int x, y;
    if constexpr (kMode == kFfnDW) {
      const int per = a.halves * tf * tc;
      r->e = quick_div(u, per);
      band_coord(u - r->e * per, a.halves * tf, tc, a.group, &x, &y);
      r->half = x >= tf;
      r->row0 = off[r->e];
      r->rows = off[r->e + 1] - r->row0;
      r->feat0 = (x - r->half * tf) * 256;
      r->col0 = y * 256;
      r->blocks = (r->rows + kSlabK - 1) / kSlabK;
      r->mma_n = 256;
    } else {
      while (u >= tiles[e + 1] * tf) ++e;
      r->e = e;
      r->half = 0;
      const int first = off[e], count = off[e + 1] - first;
      const int tt = tiles[e + 1] - tiles[e];
      const int size = (quick_div(count + tt - 1, tt) + 31) & ~31;
      band_coord(u - tiles[e] * tf, tt, tf, a.group, &x, &y);
      r->row0 = first + x * size;
      r->rows = min(size, count - x * size);
      r->feat0 = y * FfnCfg<kMode>::kFeat;
      r->col0 = 0;
      r->blocks = (a.red + kSlabK - 1) / kSlabK * (kMode == kFfnDA ? a.halves : 1);
      r->mma_n = (r->rows + 31) & ~31;
    }
  }
  __device__ __forceinline__ bool next(const FfnArgs& a, FfnSegment* s) {
    if (pos < hi) {
      const int v = (int)(pos / blocks);
      const long long first = (long long)v * blocks;
      unit(a, undivided + v, s);
      s->kb0 = (int)(pos - first);
      s->kb1 = (int)min((long long)blocks, hi - first);
      s->c0 = sk_owner(first, items, ranges);
      s->c1 = sk_owner(first + blocks - 1, items, ranges);
      pos = first + s->kb1;
      if (pos >= hi) e = 0;  // (the whole units come before these)
      return true;
    }
    if (next_unit >= undivided) return false;
    unit(a, next_unit, s);
    next_unit += pairs;
    s->kb0 = 0;
    s->kb1 = s->blocks;
    return true;
  }
  // next() for those whom the segment does not concern.
  __device__ __forceinline__ bool skip() {
    if (pos < hi) {
      const long long end = (pos / blocks + 1) * blocks;
      pos = end < hi ? end : hi;
      if (pos >= hi) e = 0;
      return true;
    }
    if (next_unit >= undivided) return false;
    next_unit += pairs;
    return true;
  }
};

// tmap_w0, tmap_w1: the banks (k, n, e); gated: gate and up, box 64 x 64; act: box
// 64 x 128 (w1 unused); dA: box 64 x 64, w1 the second half's.  dW: dz (n, r, half)
// and A (k, r), boxes 64 x 64, without offsets.
// tmap_t: the token operand (gated, act A, dA dz: columns, rows, half), box 64 x 128;
// tmap_h: the same with box 64 x 64 (unused in dW);
// tmap_s: the same with box 64 x 16; dW: dW (k, n, half * experts + e), box 64 x 32.
template <int kMode, bool kMany, class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(FfnCfg<kMode>::kThreads, 1)
ffn_pair_kernel(const __grid_constant__ CUtensorMap tmap_w0,
                const __grid_constant__ CUtensorMap tmap_w1,
                const __grid_constant__ CUtensorMap tmap_t,
                const __grid_constant__ CUtensorMap tmap_h,
                const __grid_constant__ CUtensorMap tmap_s, const FfnArgs args) {
  using C = FfnCfg<kMode, kMany>;
  constexpr int kStages = C::kStages;
  constexpr bool kMnA = kMode == kFfnDA || kMode == kFfnDW;  // the M operand lies along rows
  constexpr bool kMnB = kMode == kFfnDW;
  constexpr bool kGated = kMode == kFfnGated;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[kStages];
  __shared__ alignas(8) uint64_t bar_empty[kStages];
  __shared__ alignas(8) uint64_t bar_acc_full[2];
  __shared__ alignas(8) uint64_t bar_acc_empty[2];
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;
  __shared__ uint32_t last_word[4];

  cluster_arrive_started();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t store_base = smem_base + kStages * C::kStageBytes;
  int* s_off = reinterpret_cast<int*>(smem_raw + (store_base + C::kStaging - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 2);  // each CTA's producer
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_acc_full[b]), 1);
      mbar_init(smem_u32(&bar_acc_empty[b]), 2 * 8);  // of both CTAs
    }
    mbar_init(smem_u32(&bar_drain), 1);
    abort_word = 0;
    fence_mbar_init_cluster();
    prefetch_tmap(&tmap_w0);
    prefetch_tmap(&tmap_w1);
    if (kMode != kFfnDW) {
      prefetch_tmap(&tmap_t);
      prefetch_tmap(&tmap_h);
    }
    prefetch_tmap(&tmap_s);
  }
  __syncwarp();
  cluster_wait_started();
  if (warp == 1) tmem_alloc_pair(smem_u32(&tmem_slot), kTmemCols);
  grid_wait();
  if (warp == 2)
    ffn_groups(args.offsets, args.experts, args.rows, 256, args.status, s_off, s_tiles);
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  grid_launch_next();
  const uint32_t tmem_base = tmem_slot;

  WaitCtx wctx;
  wctx.status = args.status;
  wctx.timeout_ns = args.timeout_ns;
  wctx.abort_local = smem_u32(&abort_word);
  wctx.abort_peer = cluster_map(smem_u32(&abort_word), rank ^ 1u);

  FfnWalk<kMode> walk;
  walk.init(args, s_off, s_tiles);
  FfnSegment w;
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      const uint32_t full_leader = cluster_map(smem_u32(&bar_full[0]), 0);
      const uint64_t keep = l2_policy_evict_last();
      uint32_t stage = 0, phase = 0, filled = 0;
      int last_e = -1;
      bool ok = true;
      while (ok && walk.next(args, &w)) {
        const int f0 = w.feat0 + (int)rank * (C::kFeat / 2);
        const int half = w.mma_n / 2;
        const int t0 = kMode == kFfnDW ? w.col0 + (int)rank * 128 : w.row0 + (int)rank * half;
        // Few large boxes: past the tile's rows they bring the next ones, or zeros.
        const int box = half > 64 ? 128 : half > 32 ? 64 : 16;
        const uint32_t bytes = C::kOperand + (box == 16 ? half : box) * 128;
        const int per_half = kMode == kFfnDA && args.halves == 2 ? w.blocks / 2 : w.blocks;
        const CUtensorMap *dz = &tmap_w0, *a = &tmap_w1;
        if constexpr (kMode == kFfnDW) {
          if (args.maps != nullptr) {
            // A new expert's maps are fetched a unit ahead of their use.
            for (int i = 0; i < 2; ++i) {
              FfnUnit v = w;
              if (i == 1) {
                if (walk.next_unit >= walk.undivided) break;
                walk.unit(args, walk.next_unit, &v);
              }
              if (v.e <= last_e) continue;
              tmap_acquire(args.maps + 2 * v.e);
              tmap_acquire(args.maps + 2 * v.e + 1);
              prefetch_tmap(args.maps + 2 * v.e);
              prefetch_tmap(args.maps + 2 * v.e + 1);
              last_e = v.e;
            }
            dz = args.maps + 2 * w.e;
            a = dz + 1;
          }
        }
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!wait_ready(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          ++filled;
          const uint32_t fb = full_leader + stage * 8u;
          const uint32_t sa = smem_base + stage * C::kStageBytes;
          const uint32_t sb = sa + C::kOperand;
          mbar_arrive_expect_tx_cluster(fb, bytes);
          const int second = kb >= per_half;  // dA: which weight
          const int k0 = (kb - second * per_half) * kSlabK;
          if constexpr (kMode == kFfnGated) {
            tma_load_3d_pair_hint(sa, &tmap_w0, k0, f0, w.e, fb, keep);
            tma_load_3d_pair_hint(sa + C::kOperand / 2, &tmap_w1, k0, f0, w.e, fb, keep);
          } else if constexpr (kMode == kFfnAct) {
            tma_load_3d_pair_hint(sa, &tmap_w0, k0, f0, w.e, fb, keep);
          } else if constexpr (kMode == kFfnDA) {
            const CUtensorMap* bank = second ? &tmap_w1 : &tmap_w0;
            tma_load_3d_pair_hint(sa, bank, f0, k0, w.e, fb, keep);
            tma_load_3d_pair_hint(sa + C::kOperand / 2, bank, f0 + 64, k0, w.e, fb, keep);
          } else {
            tma_load_3d_pair_hint(sa, dz, f0, w.row0 + k0, w.half, fb, keep);
            tma_load_3d_pair_hint(sa + C::kOperand / 2, dz, f0 + 64, w.row0 + k0, w.half, fb, keep);
          }
          if constexpr (kMode == kFfnDW) {
            tma_load_2d_pair_hint(sb, a, t0, w.row0 + k0, fb, keep);
            tma_load_2d_pair_hint(sb + C::kOperand / 2, a, t0 + 64, w.row0 + k0, fb, keep);
          } else if (box == 128) {
            tma_load_3d_pair_hint(sb, &tmap_t, k0, t0, second, fb, keep);
          } else if (box == 64) {
            tma_load_3d_pair_hint(sb, &tmap_h, k0, t0, second, fb, keep);
          } else {
            for (int r = 0; r < half; r += 16)
              tma_load_3d_pair_hint(sb + r * 128, &tmap_s, k0, t0 + r, second, fb, keep);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // Before a CTA leaves: its copies have landed (the leader's barriers count both
      // CTAs'), and the leader's last arrivals on the other's barriers.
      drain_copies<kStages>(smem_u32(rank == 0 ? &bar_full[0] : &bar_empty[0]), stage, phase,
                            filled, wctx);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (rank == 0 && elect_one()) {
      const uint32_t accf_self = cluster_map(smem_u32(&bar_acc_full[0]), 0);
      const uint32_t accf_peer = cluster_map(smem_u32(&bar_acc_full[0]), 1);
      uint32_t stage = 0, phase = 0;
      int it = 0;
      bool ok = true;
      while (ok && walk.next(args, &w)) {
        if (w.blocks == 0) continue;
        const int red = kMode == kFfnDW ? w.rows : args.red;
        const int per_half = kMode == kFfnDA && args.halves == 2 ? w.blocks / 2 : w.blocks;
        const uint32_t idesc = make_idesc_16bit(kPairM, w.mma_n, kFormat<T>, kMnA, kMnB);
        const uint32_t buf = it & 1, acc_phase = (it >> 1) & 1;
        ++it;
        if (!wait_ready(smem_u32(&bar_acc_empty[buf]), acc_phase ^ 1u, wctx, kErrWaitAccEmpty))
          break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + buf * 256;
        for (int kb = w.kb0; kb < w.kb1; ++kb) {
          if (!wait_ready(smem_u32(&bar_full[stage]), phase, wctx, kErrWaitFull)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem_base + stage * C::kStageBytes;
          const uint32_t sb = sa + C::kOperand;
          const uint64_t adesc =
              kMnA ? make_sdesc_mn128(sa, C::kOperand / 2) : make_sdesc_k128(sa);
          const uint64_t bdesc =
              kMnB ? make_sdesc_mn128(sb, C::kOperand / 2) : make_sdesc_k128(sb);
          const int left = red - (kb >= per_half ? kb - per_half : kb) * kSlabK;
          const int steps = left >= kSlabK ? kSlabK / kMmaK : (left + kMmaK - 1) / kMmaK;
#pragma unroll
          for (int k = 0; k < kSlabK / kMmaK; ++k) {
            if (k < steps)
              umma_bf16_pair(d_tmem, adesc + (kMnA ? 128ull : 2ull) * k,
                             bdesc + (kMnB ? 128ull : 2ull) * k, idesc,
                             (kb != w.kb0 || k != 0) ? 1u : 0u);
          }
          umma_commit_both(smem_u32(&bar_empty[0]) + stage * 8u, 3);
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_pair(accf_self + buf * 8u);
        umma_commit_pair(accf_peer + buf * 8u);
      }
      umma_commit_pair(cluster_map(smem_u32(&bar_drain), 0));
      if (!mbar_try_wait(smem_u32(&bar_drain), 0))
        wait_slow(smem_u32(&bar_drain), 0, wctx, kErrWaitDrain, false);
    }
    __syncwarp();
  } else {
    // ----------------------------------------------------------- epilogue
    // warps 2..9 take the tiles of the first accumulator, 10..17 of the second
    const int quarter = warp & 3, set = (warp - 2) >> 3, group = ((warp - 2) >> 2) & 1;
    const int tid = ((warp - 2) & 3) * 32 + lane;
    const int crew = 2 * set + group;  // whose staging, barrier and word
    const uint32_t acc_empty_leader = cluster_map(smem_u32(&bar_acc_empty[0]), 0);
    T* out = static_cast<T*>(args.o.out);
    if constexpr (kMode != kFfnDW)
      zero_unowned_rows(out, args.o.ldo, args.feat, s_off[0], s_off[args.experts], args.rows,
                        (long long)blockIdx.x * (256 * C::kSets) + (threadIdx.x - 64),
                        gridDim.x * (256ll * C::kSets));
    const uint32_t box = store_base + (uint32_t)(warp - 2) * kStoreBufBytes;
    constexpr bool kTwo = C::kSets == 1;
    const uint32_t staging = store_base + (uint32_t)crew * (kTwo ? 2 : 1) * kFfnStageBytes;
    uint32_t turn = 0;
    int it = 0;
    int ok = 1;
    const int cta = blockIdx.x;
    // What the groups of all the CTAs with a part of a divided tile count in at: true
    // for the last, who takes the sum.
    auto joined = [&]() {
      named_bar_sync(1 + crew, 128);
      if (tid == 0) {
        unsigned int* count = args.counts + w.c0 * 16 + (int)rank * 2 + group;
        const bool last = atomic_add_acq_rel(count, 1u) == (unsigned int)(w.c1 - w.c0);
        if (last) atomicExch(count, 0u);
        last_word[crew] = last;
      }
      named_bar_sync(1 + crew, 128);
      return last_word[crew] != 0;
    };
    // Column `col` of this lane's accumulator row in the slot of pair c: a pair begins at
    // most one divided tile (slot 1) and ends or crosses at most one that an
    // earlier pair began (slot 0).
    auto slot = [&](int c, int col) {
      return args.slots + (((long long)(2 * c + (int)rank) * 2 + (c == w.c0 ? 1 : 0)) * 256 + col) *
                              128 + quarter * 32 + lane;
    };
    // acc = the parts' sum, `kN` columns from col on, 32 loads in flight, added in order.
    auto add_parts = [&](int col, auto& acc) {
      constexpr int kN = sizeof(acc) / sizeof(float), kParts = 32 / kN;
#pragma unroll
      for (int j = 0; j < kN; ++j) acc[j] = 0.0f;
#pragma unroll 1
      for (int c = w.c0; c <= w.c1; c += kParts) {
        float v[kParts][kN];
#pragma unroll
        for (int i = 0; i < kParts; ++i) {
          const float* from = slot(c + i <= w.c1 ? c + i : c, col);
#pragma unroll
          for (int j = 0; j < kN; ++j) v[i][j] = c + i <= w.c1 ? __ldcg(from + j * 128) : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
          for (int j = 0; j < kN; ++j) acc[j] += v[i][j];
      }
    };
    for (;;) {
      if (C::kSets == 2 && (it & 1) != set) {
        if (!walk.skip()) break;
        ++it;
        continue;
      }
      if (!walk.next(args, &w)) break;
      const uint32_t buf = it & 1, acc_phase = (it >> 1) & 1;
      const bool any = w.blocks != 0;
      if (any) {
        ++it;
        if (ok) {
          if (lane == 0)
            ok = wait_ready(smem_u32(&bar_acc_full[buf]), acc_phase, wctx, kErrWaitAccFull);
          ok = __shfl_sync(0xffffffffu, ok, 0);
        }
        tc_fence_after_sync();
      }
      const uint32_t tbase = tmem_base + buf * 256 + ((uint32_t)(quarter * 32) << 16);
      const bool whole = w.whole();
      if constexpr (kMode == kFfnDW) {
        // Lane = n, 64 columns of k at a time through a swizzled 32 x 64 box.
        const int f0 = w.feat0 + (int)rank * kCtaM + quarter * 32;
        auto load = [&](int c, int h, uint32_t (&v)[32]) {
          if (any) {
            tmem_ld_32x32b_x32(tbase + c * kStoreCols + 32 * h, v);
            tmem_wait_ld();
            if ((c & 1) && h) {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(acc_empty_leader + buf * 8u);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = 0;
          }
        };
        if (!whole) {
#pragma unroll 1
          for (int c = 4 * group; c < 4 * group + 4; ++c) {
            uint32_t v[32];
            load(c >> 1, c & 1, v);
            float* to = slot(cta >> 1, c * 32);
#pragma unroll
            for (int j = 0; j < 32; ++j) __stcg(to + j * 128, __uint_as_float(v[j]));
          }
          if (!joined()) continue;
        }
        if (!ok) continue;
#pragma unroll 1
        for (int c = 2 * group; c < 2 * group + 2; ++c) {
          uint32_t p[2][16];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (whole) {
              uint32_t v[32];
              load(c, h, v);
#pragma unroll
              for (int j = 0; j < 16; ++j)
                p[h][j] = pack_pair<T>(__uint_as_float(v[2 * j]), __uint_as_float(v[2 * j + 1]));
            } else {
              float v[32];
              add_parts(c * kStoreCols + 32 * h, v);
#pragma unroll
              for (int j = 0; j < 16; ++j) p[h][j] = pack_pair<T>(v[2 * j], v[2 * j + 1]);
            }
          }
          if (lane == 0) bulk_wait_group_read<0>();  // the store before has read the box
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t* q = p[j >> 2] + 4 * (j & 3);
            st_shared_v4(box + lane * 128u + ((uint32_t)(j ^ (lane & 7)) << 4), q[0], q[1], q[2],
                         q[3]);
          }
          const int z = w.half * args.experts + w.e;
          if (out == nullptr) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              // (a box that starts past the matrix has nothing to write)
              if (f0 < args.feat && w.col0 + c * kStoreCols < args.cols)
                tma_store_3d(&tmap_s, box, w.col0 + c * kStoreCols, f0, z);
              bulk_commit_group();
            }
          } else {
            // Rows that TMA cannot write: the box row by row, 64 bytes a store.
            __syncwarp();
            const int col = w.col0 + c * kStoreCols + lane;
            T* to = out + ((long long)z * args.feat + f0) * args.cols + col;
            for (int r = 0; r < 32 && f0 + r < args.feat; ++r, to += args.cols) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int j = h * 32 + lane;  // element j of row r: 16-byte chunk j / 8
                const uint16_t v = ld_shared_u16(box + r * 128 + (((j >> 3) ^ (r & 7)) << 4) +
                                                 (j & 7) * 2);
                if (col + h * 32 < args.cols) reinterpret_cast<uint16_t*>(to)[h * 32] = v;
              }
            }
            __syncwarp();
          }
        }
      } else {
        // (a warp whose wait ran out still comes to its group's barriers, and
        // writes nothing)
        const int f0 = w.feat0 + (int)rank * (C::kFeat / 2);
        FfnTile<kGated, T> tile;
        ffn_tile<kGated, T>(args.o, f0, w.row0, tid, tile);
        auto load = [&](int c, float (&acc)[kStageTokens]) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(tbase + c, v);
          tmem_wait_ld();
          if (c + 2 * kStageTokens >= w.mma_n) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty_leader + buf * 8u);
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[j] = __uint_as_float(v[j]);
        };
        if (!whole) {
#pragma unroll 1
          for (int c = group * kStageTokens; c < w.mma_n; c += 2 * kStageTokens) {
            float acc[kStageTokens];
            load(c, acc);
            float* to = slot(cta >> 1, c);
#pragma unroll
            for (int j = 0; j < 16; ++j) __stcg(to + j * 128, acc[j]);
          }
          if (!joined()) continue;
        }
        auto finish = [&](auto code) {
          constexpr int kAct = decltype(code)::value;
          FfnResidual<kGated, T> now, next;
          next.fetch(args.o, group * kStageTokens, w.rows - group * kStageTokens, tile);
#pragma unroll 1
          for (int c = group * kStageTokens; c < w.mma_n; c += 2 * kStageTokens) {
            now = next;
            next.fetch(args.o, c + 2 * kStageTokens, w.rows - c - 2 * kStageTokens, tile);
            float acc[kStageTokens];
            if (whole)
              load(c, acc);
            else
              add_parts(c, acc);
            ffn_finish<kGated, kAct, T, kTwo>(args.o, staging, &turn, 1 + crew, quarter, acc,
                                              w.row0, c, ok ? w.rows - c : 0, f0, tid, tile,
                                              now);
          }
        };
        if constexpr (kMode == kFfnDA)
          finish(ActCode<B200_ACT_NONE>());
        else
          with_act(args.o.act, finish);
      }
    }
    if (kMode == kFfnDW && lane == 0) bulk_wait_group_read<0>();
    __syncwarp();
  }

  // ------------------------------------------------------------- teardown
  tc_fence_before_sync();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_pair(tmem_base, kTmemCols);
  }
  cluster_sync_all();
}

}  // namespace b200
