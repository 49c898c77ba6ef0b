// Feed-forward products with fewer tiles than SMs: a tile's contraction is divided
// over the CTAs of a cluster, which add their parts up in shared memory.
//
// A cluster holds `splits` parts of one tile; a part is a CTA (128 accumulator rows) or
// a 2-CTA pair (256).  Each part multiplies its share of the contraction, 16 tokens of
// the result at a time belong to one part in turn, and every part writes the other
// parts' tokens of its accumulator into their shared memory -- where the ring of operands
// was, which a cluster barrier has shown to be done with.  Each then adds up the parts
// in their order and finishes its tokens, so the epilogue is divided as well, and
// nothing goes through global memory.
//
// Bound by HBM as long as the weights are most of what is read: the streaming kernel
// spreads them over every SM evenly but joins parts through L2, which took 10 to 25 us
// from 64 tokens on.  128 rows x 4096 x 14336: 25.5 us (4.7 TB/s; streaming 44, pairs 68),
// 256 rows x 2048 x 8192: 17 us (50 and 48).
#pragma once
#include "ffn_gemm.cuh"

namespace b200 {

struct FfnClusterArgs {
  int rows, feat;  // feat: output features, N (gated, act) or K (dA)
  int red;         // contraction extent (dA: of one half)
  int halves;      // dA: 1 or 2
  int splits;      // parts of a tile
  int tiles_t;     // token tiles, of `tokens` rows each but the last
  int tokens;      // a multiple of 16 (pairs: 32), up to 256
  int stages, stage_bytes;
  int box;         // rows of a token box: a part's tokens of a stage are one box
  FfnOut o;
  int* status;
  unsigned long long timeout_ns;
};

template <bool kPair>
struct FfnClusterCfg {
  static constexpr int kWeight = 128 * kSlabK * 2;  // per CTA and stage
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (2 + kEpiWarps);
  // The ring takes all the shared memory; when its work is done (every product has
  // completed, so every copy has landed) the parts' exchange, at most 14 x 8 KiB at 8 parts
  // of 256 tokens, and behind it the epilogue's stagings take its place.  A stage is 18 KiB
  // (boxes of 16 tokens) to 48 (256), so there are 12 of them to 4.  Against stagings of
  // their own beside a ring of 192 KiB (10 to 4): 4096 x 14336 at 200 rows 33.2 -> 30.3 us,
  // at 128 rows 26.1 -> 25.5; 16384 x 4096 at 128 rows 29.1 -> 28.2; one row the same within 3%.
  static constexpr int kRing = 224 * 1024;
  static constexpr int kMaxStages = kRing / (kWeight + 16 * 128);
  static constexpr int kStagingAt = 8 * kWeight;
  static constexpr int kSmem = kRing + 1024;
  static_assert(14 * kFfnStageBytes <= kStagingAt &&
                kStagingAt + 2 * 2 * kFfnStageBytes <= kRing, "what takes the ring's place");
};

// tmap_w0, tmap_w1: the weights (k, n, 1): gated gate and up, box 64 x 64; act box
// 64 x 128; dA box 64 x 64.  tmap_t: the token operand (columns, rows, half), box 64 x
// args.box.
template <int kMode, bool kPair, class T>
__global__ void __launch_bounds__(FfnClusterCfg<kPair>::kThreads, 1)
ffn_cluster_kernel(const __grid_constant__ CUtensorMap tmap_w0,
                   const __grid_constant__ CUtensorMap tmap_w1,
                   const __grid_constant__ CUtensorMap tmap_t, const FfnClusterArgs args) {
  using C = FfnClusterCfg<kPair>;
  constexpr bool kGated = kMode == kFfnGated;
  constexpr bool kMnA = kMode == kFfnDA;
  constexpr int kCtas = kPair ? 2 : 1;      // of a part
  constexpr int kFeat = kGated ? 64 : 128;  // output features of a CTA
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[C::kMaxStages];
  __shared__ alignas(8) uint64_t bar_empty[C::kMaxStages];
  __shared__ alignas(8) uint64_t bar_acc_full;
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;

  cluster_arrive_started();
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t crank = cluster_ctarank();
  const uint32_t rank = kPair ? crank & 1u : 0u;
  const uint32_t leader = kPair ? crank & ~1u : crank;
  const int part = (int)(crank / kCtas), splits = args.splits;
  const int tile = blockIdx.x / (splits * kCtas);
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t staging_base = smem_base + C::kStagingAt;
  const uint32_t stages = args.stages;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), kCtas);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    mbar_init(smem_u32(&bar_acc_full), 1);
    mbar_init(smem_u32(&bar_drain), 1);
    abort_word = 0;
    fence_mbar_init_cluster();
    prefetch_tmap(&tmap_w0);
    prefetch_tmap(&tmap_w1);
    prefetch_tmap(&tmap_t);
  }
  __syncwarp();
  cluster_wait_started();
  if (warp == 1) {
    if constexpr (kPair) {
      tmem_alloc_pair(smem_u32(&tmem_slot), 256);
    } else {
      tmem_alloc_1(smem_u32(&tmem_slot), 256);
      tmem_relinquish_1();
    }
  }
  grid_wait();
  tc_fence_before_sync();
  cluster_sync_all();
  tc_fence_after_sync();
  grid_launch_next();
  const uint32_t tmem_base = tmem_slot;

  WaitCtx wctx;
  wctx.status = args.status;
  wctx.timeout_ns = args.timeout_ns;
  wctx.abort_local = smem_u32(&abort_word);
  wctx.abort_peer = cluster_map(smem_u32(&abort_word), kPair ? crank ^ 1u : crank);

  const int tf = tile / args.tiles_t, tt = tile - tf * args.tiles_t;
  const int row0 = tt * args.tokens, rows = min(args.tokens, args.rows - row0);
  const int mma_n = kPair ? (rows + 31) & ~31 : (rows + 15) & ~15;
  const int f0 = (tf * kCtas + (int)rank) * kFeat;
  const int per_half = (args.red + kSlabK - 1) / kSlabK;
  const int blocks = per_half * (kMode == kFfnDA ? args.halves : 1);
  const int kb0 = (int)((long long)part * blocks / splits);
  const int kb1 = (int)((long long)(part + 1) * blocks / splits);
  const uint32_t stage_bytes = args.stage_bytes;

  if (warp == 0) {
    if (elect_one()) {
      const uint32_t full_leader = cluster_map(smem_u32(&bar_full[0]), leader);
      // (weights that another token tile reads as well stay)
      const uint64_t once = args.tiles_t > 1 ? l2_policy_evict_normal() : l2_policy_evict_first();
      const uint64_t keep = l2_policy_evict_last();
      const uint32_t bytes = C::kWeight + args.box * 128;
      const int t0 = row0 + (int)rank * (mma_n / 2);
      uint32_t stage = 0, phase = 0, filled = 0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!wait_ready(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty)) break;
        ++filled;
        const uint32_t sa = smem_base + stage * stage_bytes, sb = sa + C::kWeight;
        const int second = kb >= per_half;  // dA: which weight
        const int k0 = (kb - second * per_half) * kSlabK;
        const CUtensorMap* bank = kMode == kFfnDA && second ? &tmap_w1 : &tmap_w0;
        if constexpr (kPair) {
          const uint32_t fb = full_leader + stage * 8u;
          mbar_arrive_expect_tx_cluster(fb, bytes);
          if constexpr (kMode == kFfnGated) {
            tma_load_3d_pair_hint(sa, &tmap_w0, k0, f0, 0, fb, once);
            tma_load_3d_pair_hint(sa + C::kWeight / 2, &tmap_w1, k0, f0, 0, fb, once);
          } else if constexpr (kMode == kFfnAct) {
            tma_load_3d_pair_hint(sa, bank, k0, f0, 0, fb, once);
          } else {
            tma_load_3d_pair_hint(sa, bank, f0, k0, 0, fb, once);
            tma_load_3d_pair_hint(sa + C::kWeight / 2, bank, f0 + 64, k0, 0, fb, once);
          }
          tma_load_3d_pair_hint(sb, &tmap_t, k0, t0, second, fb, keep);
        } else {
          const uint32_t fb = smem_u32(&bar_full[stage]);
          mbar_arrive_expect_tx(fb, bytes);
          if constexpr (kMode == kFfnGated) {
            tma_load_3d_hint(sa, &tmap_w0, k0, f0, 0, fb, once);
            tma_load_3d_hint(sa + C::kWeight / 2, &tmap_w1, k0, f0, 0, fb, once);
          } else if constexpr (kMode == kFfnAct) {
            tma_load_3d_hint(sa, bank, k0, f0, 0, fb, once);
          } else {
            tma_load_3d_hint(sa, bank, f0, k0, 0, fb, once);
            tma_load_3d_hint(sa + C::kWeight / 2, bank, f0 + 64, k0, 0, fb, once);
          }
          tma_load_3d_hint(sb, &tmap_t, k0, t0, second, fb, keep);
        }
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
      // Before the ring is written by others: its copies have landed (the leader's barriers
      // count both CTAs'), and the leader's last arrivals on the other's barriers.
      const uint32_t last = smem_u32(rank == 0 ? &bar_full[0] : &bar_empty[0]);
#pragma unroll 1
      for (uint32_t i = 0; i < stages && i < filled; ++i) {
        if (stage == 0) { stage = stages; phase ^= 1u; }
        --stage;
        if (!wait_inline(last + stage * 8u, phase, wctx, kErrWaitDrain, true)) break;
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0 && elect_one()) {
      const uint32_t idesc = make_idesc_16bit(kPair ? 256 : 128, mma_n, kFormat<T>, kMnA, false);
      uint32_t stage = 0, phase = 0;
      bool ok = true;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!wait_ready(smem_u32(&bar_full[stage]), phase, wctx, kErrWaitFull)) {
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t sa = smem_base + stage * stage_bytes;
        const uint64_t adesc = kMnA ? make_sdesc_mn128(sa, C::kWeight / 2) : make_sdesc_k128(sa);
        const uint64_t bdesc = make_sdesc_k128(sa + C::kWeight);
#pragma unroll
        for (int k = 0; k < kSlabK / kMmaK; ++k) {
          const uint64_t a = adesc + (kMnA ? 128ull : 2ull) * k, b = bdesc + 2ull * k;
          const uint32_t add = (kb != kb0 || k != 0) ? 1u : 0u;
          if constexpr (kPair)
            umma_bf16_pair(tmem_base, a, b, idesc, add);
          else
            umma_bf16_1(tmem_base, a, b, idesc, add);
        }
        if constexpr (kPair)
          umma_commit_both(smem_u32(&bar_empty[0]) + stage * 8u, (uint16_t)(3u << leader));
        else
          umma_commit_1(smem_u32(&bar_empty[stage]));
        if (++stage == stages) { stage = 0; phase ^= 1u; }
      }
      if constexpr (kPair) {
        if (ok) {
          umma_commit_pair(cluster_map(smem_u32(&bar_acc_full), leader));
          umma_commit_pair(cluster_map(smem_u32(&bar_acc_full), leader + 1));
        }
        umma_commit_pair(cluster_map(smem_u32(&bar_drain), leader));
      } else {
        if (ok) umma_commit_1(smem_u32(&bar_acc_full));
        umma_commit_1(smem_u32(&bar_drain));
      }
      if (!mbar_try_wait(smem_u32(&bar_drain), 0))
        wait_slow(smem_u32(&bar_drain), 0, wctx, kErrWaitDrain, false);
    }
    __syncwarp();
  }
  const int quarter = warp & 3, group = (warp - 2) >> 2;
  const int tid = ((warp - 2) & 3) * 32 + lane;
  const uint32_t tbase = tmem_base + ((uint32_t)(quarter * 32) << 16);
  const int chunks = (rows + kStageTokens - 1) / kStageTokens;
  int ok = 1;
  if (warp >= 2) {
    if (lane == 0) ok = wait_ready(smem_u32(&bar_acc_full), 0, wctx, kErrWaitAccFull);
    ok = __shfl_sync(0xffffffffu, ok, 0);
    tc_fence_after_sync();
  }
  __syncwarp();
  if (splits > 1) {
    cluster_sync_all();  // every ring is done with
    if (warp >= 2) {
      // Chunk c belongs to part c % splits; there it is number c / splits, and this part's
      // place among the others' is its number, one less after the owner's.
      for (int c = group; c < chunks; c += 2) {
        const int owner = c % splits;
        if (owner == part) continue;
        uint32_t v[16];
        tmem_ld_32x32b_x16(tbase + c * kStageTokens, v);
        tmem_wait_ld();
        const int place = (c / splits) * (splits - 1) + (part < owner ? part : part - 1);
        const uint32_t to =
            cluster_map(smem_base + (uint32_t)place * kFfnStageBytes, owner * kCtas + rank) +
            (uint32_t)(quarter * 32 + lane) * 16u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          st_shared_cluster_v4(to + j * 2048u, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
      }
    }
    __syncwarp();
    cluster_sync_all();  // every part has arrived
  }
  if (warp >= 2) {
    FfnTile<kGated, T> s;
    ffn_tile<kGated, T>(args.o, f0, row0, tid, s);
    const uint32_t staging = staging_base + (uint32_t)group * 2 * kFfnStageBytes;
    uint32_t turn = 0;
    auto finish = [&](auto code) {
      constexpr int kAct = decltype(code)::value;
      FfnResidual<kGated, T> now, next;
      auto fetch = [&](int c) {
        next.fetch(args.o, c * kStageTokens, rows - c * kStageTokens, s);
      };
      fetch(part + group * splits);
#pragma unroll 1
      for (int i = group; part + i * splits < chunks; i += 2) {
        const int c = part + i * splits;
        now = next;
        fetch(c + 2 * splits);
        uint32_t v[16];
        tmem_ld_32x32b_x16(tbase + c * kStageTokens, v);
        tmem_wait_ld();
        float acc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = splits == 1 ? __uint_as_float(v[j]) : 0.0f;
        if (splits > 1) {
          uint32_t from = smem_base + (uint32_t)(i * (splits - 1)) * kFfnStageBytes +
                          (uint32_t)(quarter * 32 + lane) * 16u;
#pragma unroll 1
          for (int p = 0; p < splits; ++p) {
            if (p == part) {
#pragma unroll
              for (int j = 0; j < 16; ++j) acc[j] += __uint_as_float(v[j]);
              continue;
            }
            float w[16];
#pragma unroll
            for (int j = 0; j < 4; ++j)
              ld_shared_v4_f32(from + j * 2048u, w[4 * j], w[4 * j + 1], w[4 * j + 2],
                               w[4 * j + 3]);
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[j] += w[j];
            from += kFfnStageBytes;
          }
        }
        ffn_finish<kGated, kAct, T, true>(args.o, staging, &turn, 1 + group, quarter, acc, row0,
                                          c * kStageTokens, ok ? rows - c * kStageTokens : 0, f0,
                                          tid, s, now);
      }
    };
    if constexpr (kMode == kFfnDA)
      finish(ActCode<B200_ACT_NONE>());
    else
      with_act(args.o.act, finish);
  }
  __syncwarp();
  tc_fence_before_sync();
  if constexpr (kPair) {
    cluster_sync_all();
    if (warp == 1) {
      tc_fence_after_sync();
      tmem_dealloc_pair(tmem_base, 256);
    }
    cluster_sync_all();
  } else {
    __syncthreads();
    if (warp == 1) {
      tc_fence_after_sync();
      tmem_dealloc_1(tmem_base, 256);
    }
  }
}

}  // namespace b200
