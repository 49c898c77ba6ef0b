// Products grouped by expert, large groups: 2-CTA pairs, tcgen05, TMEM.
//
//   forward  C[r, n]     = sum_k A[r, k] B[e, n, k]     r among expert e's rows
//   dA       dA[r, k]    = sum_n dC[r, n] B[e, n, k]
//   dB       dB[e, n, k] = sum_r dC[r, n] A[r, k]       r over expert e's rows
//
// The pair kernel of gemm_kernel.cuh (same ring, same warp roles, bounded
// waits) with the operands turned round: the weight's axis (n in forward, k
// in dA) is the MMA's M = 256 and the tokens are its N, because N may be any
// multiple of 32 from one instruction to the next.  An expert's rows are cut
// into ceil(count / 256) equal tiles, so a ragged group costs its rows
// rounded up to 32 and not to 256, and no row needs padding in memory.  The
// accumulator then holds C transposed: a TMEM lane is one n, a column one
// token, and the epilogue writes it back the right way round.
//
// No operand is copied or transposed in memory.  Where the contraction runs
// along rows (B in dA; both operands in dB) the tile is loaded as it lies
// and the MMA reads it MN-major (make_sdesc_mn128).
//
// dB's contraction is ragged: an expert's last 64-row block reaches into the
// next expert's rows, which must read as zero in both operands (0 x inf is
// NaN).  TMA fills what lies beyond a tensor's end with zeros, so a small
// kernel first makes two tensor maps per expert that end at its last row
// (grouped_maps_kernel).  (Clearing the rows in shared memory instead, by a
// warp of its own between the load and the MMA, cost each tile 1.3 us: 8
// experts x 1023 rows, 14336 x 4096, took 800 us where 1024 rows took 663.)
// An expert without rows gets zeros.
//
// Bound by the tensor pipe: 8 experts, 8192 rows, 4096 x 4096, bf16: forward
// 200 us, dA 198, dB 192 (1.37 to 1.43 PFLOP/s, 0.81 to 0.84 of a large
// library product's rate), the pipe 87, 89 and 77 % active.  What is lost is
// the last wave of tiles, the filling of each CTA's ring and, in dB, the
// store of a whole weight tile.
#pragma once
#include <cuda_fp16.h>

#include "moe_groups.cuh"

namespace b200 {

enum GroupedMode : int { kGroupedFwd = 0, kGroupedDA = 1, kGroupedDB = 2 };

struct GroupedArgs {
  const int* offsets;
  int experts, rows;
  int feat;      // extent of the MMA's M axis: N (forward, dB) or K (dA)
  int red;       // contraction extent: K (forward) or N (dA); unused in dB
  int cols;      // dB: extent of the MMA's N axis, K
  void* out;     // forward, dA: rows x feat; dB: null, or dB where TMA cannot write it
  long long ldo;
  long long expert_stride;  // of out, dB
  int group;     // raster band
  const CUtensorMap* maps;  // dB: dC's and A's map of each expert, box 64 x 64
  int* status;
  unsigned long long timeout_ns;
};

// dB stages its output in shared memory, two boxes to an epilogue warp; for
// many experts (kMany) it gives up a stage for the table of their rows.
template <int kMode, bool kMany = false>
struct GroupedCfg {
  static constexpr int kStages = kMany ? 5 : 6;
  static constexpr int kOperand = 128 * kSlabK * 2;  // 16 KiB: 128 x 64 of either operand
  static constexpr int kStageBytes = 2 * kOperand;
  static constexpr int kThreads = 32 * 6;
  static constexpr int kStaging = kMode == kGroupedDB ? 4 * 2 * kStoreBufBytes : 0;
  static constexpr int smem_bytes(int experts) {
    return kStages * kStageBytes + kStaging + group_table_bytes(experts) + 1024;
  }
};

// dB: maps[2 e] and maps[2 e + 1] are dC's and A's tensor maps, ended at the
// last row of expert e.  One warp per expert, 5 us: its parts follow one
// another (two maps read, changed in shared memory, written, fenced).
__global__ void __launch_bounds__(32)
grouped_maps_kernel(const __grid_constant__ CUtensorMap tmap_dc,
                    const __grid_constant__ CUtensorMap tmap_a, const int* offsets, int rows,
                    CUtensorMap* maps) {
  __shared__ alignas(128) CUtensorMap map[2];
  grid_wait();
  grid_launch_next();
  const int e = blockIdx.x, lane = threadIdx.x;
  uint32_t* words = reinterpret_cast<uint32_t*>(map);
  words[lane] = reinterpret_cast<const uint32_t*>(&tmap_dc)[lane];
  words[32 + lane] = reinterpret_cast<const uint32_t*>(&tmap_a)[lane];
  // The end of expert e as the other kernels read it (build_groups): the
  // largest of the clamped offsets up to its own.
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

// One work unit: a tile of one expert's product.
struct GroupedUnit {
  int e;
  int row0, rows;  // the expert's rows (dB), or the tile's (forward, dA)
  int feat0;       // first index of the tile on the MMA's M axis
  int col0;        // dB: first index on the N axis
  int blocks;      // 64-long contraction blocks
  int mma_n;
};

// Units in order; the expert of the last one found is remembered, so a walk
// over increasing units costs one pass over the table.
template <int kMode>
struct GroupedWalk {
  const int* off;
  const int* tiles;
  int tf, tc;  // tiles on the MMA's M axis; dB: on its N axis
  int e;
  __device__ __forceinline__ void init(const GroupedArgs& a, const int* s_off, const int* s_tiles) {
    off = s_off;
    tiles = s_tiles;
    tf = (a.feat + kPairM - 1) / kPairM;
    tc = (a.cols + 255) / 256;
    e = 0;
  }
  __device__ __forceinline__ int total(const GroupedArgs& a) const {
    return kMode == kGroupedDB ? a.experts * tf * tc : tiles[a.experts] * tf;
  }
  __device__ __forceinline__ GroupedUnit unit(const GroupedArgs& a, int u) {
    GroupedUnit r;
    int x, y;
    if constexpr (kMode == kGroupedDB) {
      r.e = u / (tf * tc);
      tile_coord(u - r.e * tf * tc, tf, tc, a.group, &x, &y);
      r.row0 = off[r.e];
      r.rows = off[r.e + 1] - r.row0;
      r.feat0 = x * kPairM;
      r.col0 = y * 256;
      r.blocks = (r.rows + kSlabK - 1) / kSlabK;
      r.mma_n = 256;
    } else {
      while (u >= tiles[e + 1] * tf) ++e;
      r.e = e;
      const int first = off[e], count = off[e + 1] - first;
      const int tt = tiles[e + 1] - tiles[e];
      const int size = ((count + tt - 1) / tt + 31) & ~31;
      tile_coord(u - tiles[e] * tf, tt, tf, a.group, &x, &y);
      r.row0 = first + x * size;
      r.rows = min(size, count - x * size);
      r.feat0 = y * kPairM;
      r.col0 = 0;
      r.blocks = (a.red + kSlabK - 1) / kSlabK;
      r.mma_n = (r.rows + 31) & ~31;
    }
    return r;
  }
};

// tmap_w: forward the bank (k, n, e), box 64 x 128; dA the bank, box 64 x 64.
// tmap_t: the token operand (forward A, dA dC), box 64 x 128.
// tmap_s: forward, dA: the token operand, box 64 x 16; dB: dB (k, n, e), box 64 x 32.
template <int kMode, bool kMany, class T>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(GroupedCfg<kMode>::kThreads, 1)
grouped_pair_kernel(const __grid_constant__ CUtensorMap tmap_w,
                    const __grid_constant__ CUtensorMap tmap_t,
                    const __grid_constant__ CUtensorMap tmap_s, const GroupedArgs args) {
  using C = GroupedCfg<kMode, kMany>;
  constexpr int kStages = C::kStages;
  constexpr bool kMnA = kMode != kGroupedFwd;  // the M operand lies along rows
  constexpr bool kMnB = kMode == kGroupedDB;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[kStages];
  __shared__ alignas(8) uint64_t bar_empty[kStages];
  __shared__ alignas(8) uint64_t bar_acc_full[2];
  __shared__ alignas(8) uint64_t bar_acc_empty[2];
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;

  cluster_arrive_started();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int pair = blockIdx.x >> 1;
  const int npairs = gridDim.x >> 1;
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
      mbar_init(smem_u32(&bar_acc_empty[b]), 8);  // every epilogue warp of the pair
    }
    mbar_init(smem_u32(&bar_drain), 1);
    abort_word = 0;
    fence_mbar_init_cluster();
    if (kMode != kGroupedDB) {
      prefetch_tmap(&tmap_w);
      prefetch_tmap(&tmap_t);
    }
    prefetch_tmap(&tmap_s);
  }
  __syncwarp();
  cluster_wait_started();
  if (warp == 1) tmem_alloc_pair(smem_u32(&tmem_slot), kTmemCols);
  grid_wait();
  if (warp == 2) {
    const bool bad = build_groups(args.offsets, args.experts, args.rows, 256, s_off, s_tiles);
    if (bad && blockIdx.x == 0 && lane == 0) atomicCAS(args.status, 0, kErrOffsets);
  }
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

  GroupedWalk<kMode> walk;
  walk.init(args, s_off, s_tiles);
  const int total = walk.total(args);
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (elect_one()) {
      const uint32_t full_leader = cluster_map(smem_u32(&bar_full[0]), 0);
      const uint32_t empty_peer = cluster_map(smem_u32(&bar_empty[0]), 1);
      const uint64_t keep = l2_policy_evict_last();
      uint32_t stage = 0, phase = 0, filled = 0;
      int last_e = -1;
      bool ok = true;
      for (int u = pair; ok && u < total; u += npairs) {
        const GroupedUnit w = walk.unit(args, u);
        const int f0 = w.feat0 + (int)rank * kCtaM;
        const int half = w.mma_n / 2;
        const int t0 = kMode == kGroupedDB ? w.col0 + (int)rank * 128 : w.row0 + (int)rank * half;
        const uint32_t bytes = C::kOperand + (half == 128 ? C::kOperand : half * 128);
        const CUtensorMap* maps = args.maps + 2 * w.e;
        if constexpr (kMode == kGroupedDB) {
          // A new expert's maps are fetched a unit ahead of their use.
          for (int v = u; v < total && v <= u + npairs; v += npairs) {
            const int e = v == u ? w.e : walk.unit(args, v).e;
            if (e <= last_e) continue;
            tmap_acquire(args.maps + 2 * e);
            tmap_acquire(args.maps + 2 * e + 1);
            prefetch_tmap(args.maps + 2 * e);
            prefetch_tmap(args.maps + 2 * e + 1);
            last_e = e;
          }
        }
        for (int kb = 0; kb < w.blocks; ++kb) {
          if (!wait_ready(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          if (rank == 0 && filled >= (uint32_t)kStages) mbar_arrive_cluster(empty_peer + stage * 8u);
          ++filled;
          const uint32_t fb = full_leader + stage * 8u;
          const uint32_t sa = smem_base + stage * C::kStageBytes;
          const uint32_t sb = sa + C::kOperand;
          mbar_arrive_expect_tx_cluster(fb, bytes);
          const int k0 = kb * kSlabK;
          if constexpr (kMode == kGroupedFwd) {
            tma_load_3d_pair_hint(sa, &tmap_w, k0, f0, w.e, fb, keep);
          } else if constexpr (kMode == kGroupedDA) {
            tma_load_3d_pair_hint(sa, &tmap_w, f0, k0, w.e, fb, keep);
            tma_load_3d_pair_hint(sa + C::kOperand / 2, &tmap_w, f0 + 64, k0, w.e, fb, keep);
          } else {
            tma_load_2d_pair_hint(sa, maps, f0, w.row0 + k0, fb, keep);
            tma_load_2d_pair_hint(sa + C::kOperand / 2, maps, f0 + 64, w.row0 + k0, fb, keep);
          }
          if constexpr (kMode == kGroupedDB) {
            tma_load_2d_pair_hint(sb, maps + 1, t0, w.row0 + k0, fb, keep);
            tma_load_2d_pair_hint(sb + C::kOperand / 2, maps + 1, t0 + 64, w.row0 + k0, fb, keep);
          } else if (half == 128) {
            tma_load_2d_pair_hint(sb, &tmap_t, k0, t0, fb, keep);
          } else {
            for (int r = 0; r < half; r += 16)
              tma_load_2d_pair_hint(sb + r * 128, &tmap_s, k0, t0 + r, fb, keep);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // (the leader's barriers count both CTAs' copies)
      if (rank == 0) drain_copies<kStages>(smem_u32(&bar_full[0]), stage, phase, filled, wctx);
    }
    __syncwarp();
  } else if (warp == 1) {
    // ---------------------------------------------------------------- MMA
    if (rank == 0 && elect_one()) {
      const uint32_t empty_self = cluster_map(smem_u32(&bar_empty[0]), 0);
      const uint32_t accf_self = cluster_map(smem_u32(&bar_acc_full[0]), 0);
      const uint32_t accf_peer = cluster_map(smem_u32(&bar_acc_full[0]), 1);
      uint32_t stage = 0, phase = 0;
      int it = 0;
      bool ok = true;
      for (int u = pair; ok && u < total; u += npairs) {
        const GroupedUnit w = walk.unit(args, u);
        if (w.blocks == 0) continue;
        const int red = kMode == kGroupedDB ? w.rows : args.red;
        const uint32_t idesc = make_idesc_16bit(kPairM, w.mma_n, kFormat<T>, kMnA, kMnB);
        const uint32_t buf = it & 1, acc_phase = (it >> 1) & 1;
        ++it;
        if (!wait_ready(smem_u32(&bar_acc_empty[buf]), acc_phase ^ 1u, wctx, kErrWaitAccEmpty))
          break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + buf * 256;
        for (int kb = 0; kb < w.blocks; ++kb) {
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
          const int left = red - kb * kSlabK;
          const int steps = left >= kSlabK ? kSlabK / kMmaK : (left + kMmaK - 1) / kMmaK;
#pragma unroll
          for (int k = 0; k < kSlabK / kMmaK; ++k) {
            if (k < steps)
              umma_bf16_pair(d_tmem, adesc + (kMnA ? 128ull : 2ull) * k,
                             bdesc + (kMnB ? 128ull : 2ull) * k, idesc,
                             (kb != 0 || k != 0) ? 1u : 0u);
          }
          umma_commit_pair(empty_self + stage * 8u);
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
    const int quarter = warp & 3;
    const uint32_t acc_empty_leader = cluster_map(smem_u32(&bar_acc_empty[0]), 0);
    T* out = static_cast<T*>(args.out);
    if constexpr (kMode != kGroupedDB)
      zero_unowned_rows(out, args.ldo, args.feat, s_off[0], s_off[args.experts], args.rows,
                        (long long)blockIdx.x * 128 + (threadIdx.x - 64), gridDim.x * 128ll);
    // rows on 4 bytes take two elements at a time
    const bool even_rows = (args.ldo & 1) == 0 && (reinterpret_cast<uintptr_t>(out) & 3u) == 0;
    const uint32_t my_store = store_base + (uint32_t)(warp - 2) * 2 * kStoreBufBytes;
    int it = 0;
    for (int u = pair; u < total; u += npairs) {
      const GroupedUnit w = walk.unit(args, u);
      const uint32_t buf = it & 1, acc_phase = (it >> 1) & 1;
      const bool any = w.blocks != 0;
      if (any) {
        ++it;
        int ok = 0;
        if (lane == 0)
          ok = wait_ready(smem_u32(&bar_acc_full[buf]), acc_phase, wctx, kErrWaitAccFull);
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        tc_fence_after_sync();
      }
      const uint32_t tbase = tmem_base + buf * 256 + ((uint32_t)(quarter * 32) << 16);
      const int f0 = w.feat0 + (int)rank * kCtaM + quarter * 32;
      if constexpr (kMode == kGroupedDB) {
        // Lane = n, 64 columns of k at a time through a swizzled 32 x 64 box.
#pragma unroll 1
        for (int c = 0; c < 256 / kStoreCols; ++c) {
          uint32_t v0[32], v1[32];
          if (any) {
            tmem_ld_32x32b_x32(tbase + c * kStoreCols, v0);
            tmem_ld_32x32b_x32(tbase + c * kStoreCols + 32, v1);
            tmem_wait_ld();
            if (c == 256 / kStoreCols - 1) {
              tc_fence_before_sync();
              __syncwarp();
              if (lane == 0) mbar_arrive_cluster(acc_empty_leader + buf * 8u);
            }
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v0[j] = v1[j] = 0;
          }
          const uint32_t box = my_store + (c & 1) * kStoreBufBytes;
          if (lane == 0) bulk_wait_group_read<1>();  // the store before last has read it
          __syncwarp();
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const uint32_t* v = j < 4 ? v0 + 8 * j : v1 + 8 * (j - 4);
            uint32_t p[4];
#pragma unroll
            for (int q = 0; q < 4; ++q)
              p[q] = pack_pair<T>(__uint_as_float(v[2 * q]), __uint_as_float(v[2 * q + 1]));
            st_shared_v4(box + lane * 128u + ((uint32_t)(j ^ (lane & 7)) << 4), p[0], p[1], p[2],
                         p[3]);
          }
          if (args.out == nullptr) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              // (a box that starts past the matrix has nothing to write)
              if (f0 < args.feat && w.col0 + c * kStoreCols < args.cols)
                tma_store_3d(&tmap_s, box, w.col0 + c * kStoreCols, f0, w.e);
              bulk_commit_group();
            }
          } else {
            // Rows that TMA cannot write: the box row by row, 64 bytes a store.
            __syncwarp();
            const int col = w.col0 + c * kStoreCols + lane;
            T* to = out + w.e * args.expert_stride + (long long)f0 * args.ldo + col;
            for (int r = 0; r < 32 && f0 + r < args.feat; ++r, to += args.ldo) {
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
        // Lane = feature, column = token.  Neighbouring lanes trade values so
        // that each holds two features of one token (even lanes even tokens):
        // a store instruction then writes 64 bytes of each of two rows.
        const int odd = lane & 1;
        const int f = f0 + (lane & ~1);
        T* row = out + (long long)(w.row0 + odd) * args.ldo + f;
        const bool in = f < args.feat, second = f + 1 < args.feat;
        const bool both = second && even_rows;
#pragma unroll 1
        for (int c = 0; c < w.mma_n; c += 32) {
          uint32_t v[32];
          tmem_ld_32x32b_x32(tbase + c, v);
          tmem_wait_ld();
          if (c + 32 >= w.mma_n) {
            tc_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty_leader + buf * 8u);
          }
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const float give = __uint_as_float(odd ? v[j] : v[j + 1]);
            const float keep = __uint_as_float(odd ? v[j + 1] : v[j]);
            const float got = __shfl_xor_sync(0xffffffffu, give, 1);
            const uint32_t pair = odd ? pack_pair<T>(got, keep) : pack_pair<T>(keep, got);
            if (in && c + j + odd < w.rows) {
              if (both) {
                *reinterpret_cast<uint32_t*>(row) = pair;
              } else {
                uint16_t* half = reinterpret_cast<uint16_t*>(row);
                half[0] = (uint16_t)pair;
                if (second) half[1] = (uint16_t)(pair >> 16);
              }
            }
            row += 2 * args.ldo;
          }
        }
      }
    }
    if (kMode == kGroupedDB && lane == 0) bulk_wait_group_read<0>();
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
