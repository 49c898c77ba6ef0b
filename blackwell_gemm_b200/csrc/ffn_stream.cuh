// Feed-forward products for few rows: the weights are read once and everything
// else is small, so what counts is that every SM streams an equal share of them.
//
// Work is cut as in moe_stream.cuh: items in the order expert, 128-row block of
// the weight, token tile, block of the contraction, one contiguous range per CTA.
// gated: a block is 64 gate rows and the same 64 rows of the up weight.  A tile
// whose contraction falls into several ranges is joined by whichever of its CTAs
// finishes last, in range order, so sums do not depend on which one that was, and no
// CTA waits for another.  Here four epilogue warps count in together, because the
// activation needs a feature's both products; two such groups take every other 16 tokens
// (96 rows x 28672 x 4096 gated 51.4 us, with one group 53.4).  The end is the pair kernel's
// (ffn_epilogue.cuh).
//
// Bound by HBM: one row x 28672 x 4096 gated, 235 MB, 41 us (5.7 TB/s, 0.88 of the measured
// copy rate); 122 rows over 8 experts of that size, 1.88 GB, 281 us (6.7 TB/s).
#pragma once
#include "ffn_epilogue.cuh"
#include "moe_stream.cuh"

namespace b200 {

template <int kTok>
struct FfnStreamCfg {
  static constexpr int kWeight = 128 * kSlabK * 2;  // 16 KiB per item
  static constexpr int kTokens = kTok * kSlabK * 2;
  static constexpr int kStageBytes = kWeight + kTokens;
  static constexpr int kStages = (196 * 1024) / kStageBytes;
  static constexpr int kEpiWarps = 8;
  static constexpr int kThreads = 32 * (2 + kEpiWarps);
  static constexpr int smem_bytes(int experts) {
    return kStages * kStageBytes + 2 * kFfnStageBytes + group_table_bytes(experts) + 1024;
  }
};

// tmap_w0, tmap_w1: the banks (k, n, e), box 64 x 128, or gated gate and up, box
// 64 x 64.  tmap_t: the token operand, box 64 x 16.
template <bool kGated, int kTok, class T>
__global__ void __launch_bounds__(FfnStreamCfg<kTok>::kThreads, 1)
ffn_stream_kernel(const __grid_constant__ CUtensorMap tmap_w0,
                  const __grid_constant__ CUtensorMap tmap_w1,
                  const __grid_constant__ CUtensorMap tmap_t,
                  const __grid_constant__ CUtensorMap tmap_h, const StreamArgs args,
                  const FfnOut o) {
  using C = FfnStreamCfg<kTok>;
  constexpr int kStages = C::kStages;
  constexpr int kFeat = kGated ? 64 : 128;  // output features of a block
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[kStages];
  __shared__ alignas(8) uint64_t bar_empty[kStages];
  __shared__ alignas(8) uint64_t bar_acc_full[2];
  __shared__ alignas(8) uint64_t bar_acc_empty[2];
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;
  __shared__ uint32_t last_word[2];
  constexpr uint32_t kCols = 2 * kTok < 32 ? 32 : 2 * kTok;  // two accumulators

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t staging_base = smem_base + kStages * C::kStageBytes;
  int* s_off = reinterpret_cast<int*>(
      smem_raw + (staging_base + 2 * kFfnStageBytes - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_acc_full[b]), 1);
      mbar_init(smem_u32(&bar_acc_empty[b]), C::kEpiWarps);
    }
    mbar_init(smem_u32(&bar_drain), 1);
    abort_word = 0;
    fence_mbar_init_cluster();
    prefetch_tmap(&tmap_w0);
    prefetch_tmap(&tmap_w1);
    prefetch_tmap(&tmap_t);
    if (kTok > 16) prefetch_tmap(&tmap_h);
  }
  if (warp == 1) {
    tmem_alloc_1(smem_u32(&tmem_slot), kCols);
    tmem_relinquish_1();
  }
  grid_wait();
  if (warp == 2) stream_groups(args, kTok, s_off, s_tiles);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  grid_launch_next();
  const uint32_t tmem_base = tmem_slot;

  WaitCtx wctx;
  wctx.status = args.status;
  wctx.timeout_ns = args.timeout_ns;
  wctx.abort_local = smem_u32(&abort_word);
  wctx.abort_peer = cluster_map(smem_u32(&abort_word), 0);

  StreamWalk<kTok> walk;
  walk.init(args, s_off, s_tiles);
  StreamSegment s;

  if (warp == 0) {
    if (elect_one()) {
      const uint64_t once = l2_policy_evict_first(), keep = l2_policy_evict_last();
      uint32_t stage = 0, phase = 0;
      long long issued = 0;
      bool ok = true;
      while (ok && walk.next(&s)) {
        const int f0 = s.block * kFeat;
        const bool tall = kTok > 16 && s.rows > 32;
        const int box = tall ? 64 : 16, boxes = (s.rows + box - 1) / box;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (!wait_ready(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&bar_full[stage]);
          const uint32_t sa = smem_base + stage * C::kStageBytes;
          mbar_arrive_expect_tx(fb, C::kWeight + boxes * box * 128);
          const int k0 = kb * kSlabK;
          tma_load_3d_hint(sa, &tmap_w0, k0, f0, s.e, fb, once);
          if constexpr (kGated)
            tma_load_3d_hint(sa + C::kWeight / 2, &tmap_w1, k0, f0, s.e, fb, once);
          for (int i = 0; i < boxes; ++i)
            tma_load_2d_hint(sa + C::kWeight + i * box * 128, tall ? &tmap_h : &tmap_t, k0,
                             s.row0 + i * box, fb, keep);
          ++issued;
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      drain_copies<kStages>(smem_u32(&bar_full[0]), stage, phase, issued, wctx);
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0;
      int it = 0;
      bool ok = true;
      while (ok && walk.next(&s)) {
        const uint32_t idesc = make_idesc_16bit(128, (s.rows + 15) & ~15, kFormat<T>, false, false);
        const uint32_t buf = it & 1, acc_phase = (it >> 1) & 1;
        ++it;
        if (!wait_ready(smem_u32(&bar_acc_empty[buf]), acc_phase ^ 1u, wctx, kErrWaitAccEmpty))
          break;
        tc_fence_after_sync();
        const uint32_t d_tmem = tmem_base + buf * kTok;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (!wait_ready(smem_u32(&bar_full[stage]), phase, wctx, kErrWaitFull)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sa = smem_base + stage * C::kStageBytes;
          const uint64_t adesc = make_sdesc_k128(sa), bdesc = make_sdesc_k128(sa + C::kWeight);
#pragma unroll
          for (int k = 0; k < kSlabK / kMmaK; ++k)
            umma_bf16_1(d_tmem, adesc + 2ull * k, bdesc + 2ull * k, idesc,
                        (kb != s.kb0 || k != 0) ? 1u : 0u);
          umma_commit_1(smem_u32(&bar_empty[stage]));
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
        if (!ok) break;
        umma_commit_1(smem_u32(&bar_acc_full[buf]));
      }
      umma_commit_1(smem_u32(&bar_drain));
      if (!mbar_try_wait(smem_u32(&bar_drain), 0))
        wait_slow(smem_u32(&bar_drain), 0, wctx, kErrWaitDrain, false);
    }
    __syncwarp();
  } else {
    const int quarter = warp & 3, group = (warp - 2) >> 2;
    const int tid = ((warp - 2) & 3) * 32 + lane;
    const uint32_t staging = staging_base + (uint32_t)group * kFfnStageBytes;
    zero_unowned_rows(static_cast<T*>(o.out), o.ldo, o.feat, s_off[0], s_off[args.experts],
                      args.rows, (long long)blockIdx.x * 256 + (threadIdx.x - 64),
                      gridDim.x * 256ll);
    int it = 0;
    int ok = 1;
    while (walk.next(&s)) {
      const uint32_t buf = it & 1, acc_phase = (it >> 1) & 1;
      ++it;
      if (ok) {
        if (lane == 0)
          ok = wait_ready(smem_u32(&bar_acc_full[buf]), acc_phase, wctx, kErrWaitAccFull);
        ok = __shfl_sync(0xffffffffu, ok, 0);
      }
      tc_fence_after_sync();
      const int c_first = group * kStageTokens;
      if (c_first >= s.rows) {  // nothing for this group
        if (lane == 0) mbar_arrive_local(smem_u32(&bar_acc_empty[buf]));
        continue;
      }
      const uint32_t tbase = tmem_base + buf * kTok + ((uint32_t)(quarter * 32) << 16);
      const bool whole = s.kb0 == 0 && s.kb1 == walk.red_blocks;
      const int f0 = s.block * kFeat;
      // The parts of a divided tile: this CTA's and the others' slots.
      const long long first = s.unit * walk.red_blocks;
      const int c0 = sk_owner(first, walk.items, walk.ranges);
      const int c1 = sk_owner(first + walk.red_blocks - 1, walk.items, walk.ranges);
      auto slot = [&](int c) {
        // a CTA begins at most one divided tile (slot 1) and ends or crosses
        // at most one that an earlier CTA began (slot 0)
        return args.slots + ((long long)c * 2 + (c == c0 ? 1 : 0)) * kTok * 128 + quarter * 32 +
               lane;
      };
      FfnTile<kGated, T> tile;
      ffn_tile<kGated, T>(o, f0, s.row0, tid, tile);
      auto load = [&](int c, float (&acc)[kStageTokens]) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tbase + c, v);
        tmem_wait_ld();
        if (c + 2 * kStageTokens >= s.rows) {
          tc_fence_before_sync();
          __syncwarp();
          if (lane == 0) mbar_arrive_local(smem_u32(&bar_acc_empty[buf]));
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = __uint_as_float(v[j]);
      };
      if (!whole) {
        float* mine = slot(blockIdx.x);
#pragma unroll 1
        for (int c = c_first; c < s.rows; c += 2 * kStageTokens) {
          float acc[kStageTokens];
          load(c, acc);
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (c + j < s.rows) __stcg(mine + (c + j) * 128, acc[j]);
        }
        named_bar_sync(1 + group, 128);
        if (tid == 0) {
          unsigned int* count = args.counts + c0 * 16 + group;
          const bool last = atomic_add_acq_rel(count, 1u) == (unsigned int)(c1 - c0);
          if (last) atomicExch(count, 0u);
          last_word[group] = last;
        }
        named_bar_sync(1 + group, 128);
        if (last_word[group] == 0) continue;
      }
      with_act(o.act, [&](auto code) {
        constexpr int kAct = decltype(code)::value;
#pragma unroll 1
        for (int c = c_first; c < s.rows; c += 2 * kStageTokens) {
          float acc[kStageTokens];
          if (whole) {
            load(c, acc);
          } else {
            // Four parts' loads in flight at a time, added in order.
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[j] = 0.0f;
#pragma unroll 1
            for (int p = c0; p <= c1; p += 4) {
              float v[4][16];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float* from = slot(p + i <= c1 ? p + i : c1) + c * 128;
#pragma unroll
                for (int j = 0; j < 16; ++j)
                  v[i][j] = c + j < s.rows && p + i <= c1 ? __ldcg(from + j * 128) : 0.0f;
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[j] += v[i][j];
            }
          }
          FfnResidual<kGated, T> res;
          res.fetch(o, c, s.rows - c, tile);
          ffn_finish<kGated, kAct, T, false>(o, staging, nullptr, 1 + group, quarter, acc, s.row0,
                                             c, ok ? s.rows - c : 0, f0, tid, tile, res);
        }
      });
    }
    __syncwarp();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_1(tmem_base, kCols);
  }
}

}  // namespace b200
