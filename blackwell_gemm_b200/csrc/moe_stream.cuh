// Products grouped by expert, small groups: the weights are read once and
// everything else is small, so what counts is that every SM streams an equal
// share of them.
//
// Work is a list of items in a fixed order -- expert, 128-row block of the
// weight, token tile, block of the contraction -- cut into one contiguous
// range per CTA.  A (block, token tile) whose contraction falls into several
// ranges is summed by whichever of its CTAs finishes last: each leaves its
// fp32 partial in a slot and counts itself in; the last one adds the slots
// in range order, so the sum does not depend on which CTA that was, and no
// CTA ever waits for another.  The count goes back to zero with the last.
//
// The accumulator holds the output transposed (lane = weight row, column =
// token): an SM reads 128 rows of the weight whatever the number of tokens.
//
// Bound by HBM: 16 rows over 6 experts of 4096 x 4096, 203 MB, take 43 us
// (4.7 TB/s, 0.73 of the measured copy rate); 122 rows over 8
// experts of 4096 x 14336, 944 MB, 149 us (6.3 TB/s, 0.98).  The difference is
// the launch, the first loads' way and the joining of divided tiles, about
// 8 us a call.
#pragma once
#include <cuda_fp16.h>

#include "moe_groups.cuh"

namespace b200 {

struct StreamArgs {
  const int* offsets;     // experts + 1, or null: one group of all rows
  int experts, rows;
  int feat;               // weight rows: columns of the output
  int feat_blocks;        // ceil(feat / 128)
  int red;                // contraction extent
  int red_blocks;         // items per (block, token tile)
  int min_items;          // a range is at least this long
  void* out;
  long long ldo;
  float* slots;           // [CTA][2][tok][128]
  unsigned int* counts;   // [CTA][16], zero between launches
  int* status;
  unsigned long long timeout_ns;
  const uint8_t* packed;  // 4-bit weights (moe_w4.cuh)
  long long expert_bytes;
  int record_bytes;
};

// A CTA's part of one (expert, weight block, token tile).
struct StreamSegment {
  int e, block, row0, rows;
  int kb0, kb1;
  long long unit;
};

template <int kTok>
struct StreamWalk {
  const int* off;
  const int* tiles;
  int feat_blocks, red_blocks, experts;
  long long items, lo, hi, pos;
  int ranges, e;
  __device__ __forceinline__ void init(const StreamArgs& a, const int* s_off, const int* s_tiles) {
    off = s_off;
    tiles = s_tiles;
    feat_blocks = a.feat_blocks;
    red_blocks = a.red_blocks;
    experts = a.experts;
    items = (long long)tiles[experts] * feat_blocks * red_blocks;
    long long r = items / a.min_items;
    ranges = (int)(r < 1 ? 1 : r < gridDim.x ? r : gridDim.x);
    lo = hi = 0;
    if ((int)blockIdx.x < ranges && items > 0)
      sk_range(blockIdx.x, items, ranges, &lo, &hi);
    pos = lo;
    e = 0;
  }
  __device__ __forceinline__ bool next(StreamSegment* s) {
    if (pos >= hi) return false;
    s->unit = pos / red_blocks;
    s->kb0 = (int)(pos - s->unit * red_blocks);
    const long long left = hi - pos;
    s->kb1 = left < red_blocks - s->kb0 ? s->kb0 + (int)left : red_blocks;
    pos += s->kb1 - s->kb0;
    while (s->unit >= (long long)tiles[e + 1] * feat_blocks) ++e;
    const int tt = tiles[e + 1] - tiles[e];
    const int r = (int)(s->unit - (long long)tiles[e] * feat_blocks);
    s->e = e;
    s->block = r / tt;
    const int t = r - s->block * tt;
    s->row0 = off[e] + t * kTok;
    s->rows = min(kTok, off[e + 1] - s->row0);
    return true;
  }
};

// The group table of one warp; without offsets, one group of all rows.
__device__ __forceinline__ void stream_groups(const StreamArgs& a, int tile, int* s_off,
                                              int* s_tiles) {
  if (a.offsets != nullptr) {
    const bool bad = build_groups(a.offsets, a.experts, a.rows, tile, s_off, s_tiles);
    if (bad && blockIdx.x == 0 && (threadIdx.x & 31) == 0) atomicCAS(a.status, 0, kErrOffsets);
  } else if ((threadIdx.x & 31) == 0) {
    s_off[0] = s_tiles[0] = 0;
    s_off[1] = a.rows;
    s_tiles[1] = (a.rows + tile - 1) / tile;
  }
}

// One warp's 32 weight rows of a finished segment: acc[c] is lane's row,
// token tok0 + c of the tile's kTile.  A whole contraction is rounded and
// stored; a part is left in this CTA's slot, and the last contributor to
// arrive stores the sum.  `piece` numbers the warps of a CTA that finish.
// valid = false (a wait ran out): the part is only counted, so that the
// counts are zero again when the launch ends.  kParts: fewer where registers
// are short.
template <int kTok, class T, int kParts = 4, int kTile>
__device__ __forceinline__ void stream_finish(const StreamArgs& a, const StreamWalk<kTile>& walk,
                                              const StreamSegment& s, int quarter, int piece,
                                              int tok0, float (&acc)[kTok], bool valid) {
  const int lane = threadIdx.x & 31;
  const int f = s.block * 128 + quarter * 32 + lane;
  const int rows = s.rows - tok0;  // of this warp's tokens (may be none)
  if (s.kb0 != 0 || s.kb1 != walk.red_blocks) {
    const long long first = s.unit * walk.red_blocks;
    const int c0 = sk_owner(first, walk.items, walk.ranges);
    const int c1 = sk_owner(first + walk.red_blocks - 1, walk.items, walk.ranges);
    const int me = blockIdx.x;
    auto slot = [&](int c) {
      // a CTA begins at most one divided tile (slot 1) and ends or crosses
      // at most one that an earlier CTA began (slot 0)
      return a.slots + (((long long)c * 2 + (c == c0 ? 1 : 0)) * kTile + tok0) * 128 +
             quarter * 32 + lane;
    };
    if (valid) {
      float* mine = slot(me);
#pragma unroll
      for (int c = 0; c < kTok; ++c)
        if (c < rows) __stcg(mine + c * 128, acc[c]);
    }
    __syncwarp();
    unsigned int before = 0;
    if (lane == 0) before = atomic_add_acq_rel(a.counts + c0 * 16 + piece, 1u);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (before != (unsigned int)(c1 - c0)) return;
    __syncwarp();
    if (lane == 0) atomicExch(a.counts + c0 * 16 + piece, 0u);
#pragma unroll
    for (int c = 0; c < kTok; ++c) acc[c] = 0.0f;
    // kParts parts' loads in flight at a time, added in order.
    constexpr int kBatch = kTok < 16 ? kTok : kParts == 4 ? 16 : 8;
    for (int p = c0; p <= c1; p += kParts) {
      const float* from[kParts];
#pragma unroll
      for (int i = 0; i < kParts; ++i) from[i] = slot(p + i <= c1 ? p + i : c1);
#pragma unroll
      for (int b = 0; b < kTok; b += kBatch) {
        if (b >= rows) break;
        float v[kParts][kBatch];
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
          for (int c = 0; c < kBatch; ++c)
            v[i][c] = b + c < rows && p + i <= c1 ? __ldcg(from[i] + (b + c) * 128) : 0.0f;
#pragma unroll
        for (int i = 0; i < kParts; ++i)
#pragma unroll
          for (int c = 0; c < kBatch; ++c) acc[b + c] += v[i][c];
      }
    }
  }
  if (!valid || f >= a.feat) return;
  T* col = static_cast<T*>(a.out) + (long long)(s.row0 + tok0) * a.ldo + f;
#pragma unroll
  for (int c = 0; c < kTok; ++c)
    if (c < rows) col[c * a.ldo] = round_one<T>(acc[c]);
}

// ----------------------------------------------- 16-bit weights, few tokens
// kMode kGroupedFwd: contraction over K, the bank's rows as they lie;
// kGroupedDA: contraction over N, the bank read MN-major.
// Warps: 0 TMA, 1 MMA (M = 128, N = tokens rounded up to 16), 2-5 epilogue.
template <int kTok>
struct StreamCfg {
  static constexpr int kWeight = 128 * kSlabK * 2;  // 16 KiB per item
  static constexpr int kTokens = kTok * kSlabK * 2;
  static constexpr int kStageBytes = kWeight + kTokens;
  static constexpr int kStages = (200 * 1024) / kStageBytes;
  static constexpr int kThreads = 192;
  static constexpr int smem_bytes(int experts) {
    return kStages * kStageBytes + group_table_bytes(experts) + 1024;
  }
};

// tmap_w: the bank (k, n, e), box 64 x 128 (forward) or 64 x 64 (dA).
// tmap_t: the token operand, box 64 x 16.
template <bool kDA, int kTok, class T>
__global__ void __launch_bounds__(StreamCfg<kTok>::kThreads, 1)
grouped_stream_kernel(const __grid_constant__ CUtensorMap tmap_w,
                      const __grid_constant__ CUtensorMap tmap_t, const StreamArgs args) {
  using C = StreamCfg<kTok>;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[kStages];
  __shared__ alignas(8) uint64_t bar_empty[kStages];
  __shared__ alignas(8) uint64_t bar_acc_full[2];
  __shared__ alignas(8) uint64_t bar_acc_empty[2];
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;
  constexpr uint32_t kCols = 2 * kTok < 32 ? 32 : 2 * kTok;  // two accumulators

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  int* s_off =
      reinterpret_cast<int*>(smem_raw + (smem_base + kStages * C::kStageBytes - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(smem_u32(&bar_acc_full[b]), 1);
      mbar_init(smem_u32(&bar_acc_empty[b]), 4);
    }
    mbar_init(smem_u32(&bar_drain), 1);
    abort_word = 0;
    fence_mbar_init_cluster();
    prefetch_tmap(&tmap_w);
    prefetch_tmap(&tmap_t);
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
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (!wait_ready(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&bar_full[stage]);
          const uint32_t sa = smem_base + stage * C::kStageBytes;
          const int boxes = (s.rows + 15) / 16;
          mbar_arrive_expect_tx(fb, C::kWeight + boxes * 16 * 128);
          const int k0 = kb * kSlabK, f0 = s.block * 128;
          if constexpr (kDA) {
            tma_load_3d_hint(sa, &tmap_w, f0, k0, s.e, fb, once);
            tma_load_3d_hint(sa + C::kWeight / 2, &tmap_w, f0 + 64, k0, s.e, fb, once);
          } else {
            tma_load_3d_hint(sa, &tmap_w, k0, f0, s.e, fb, once);
          }
          for (int i = 0; i < boxes; ++i)
            tma_load_2d_hint(sa + C::kWeight + i * 16 * 128, &tmap_t, k0, s.row0 + i * 16, fb,
                             keep);
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
        const uint32_t idesc =
            make_idesc_16bit(128, (s.rows + 15) & ~15, kFormat<T>, kDA, false);
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
          const uint64_t adesc = kDA ? make_sdesc_mn128(sa, C::kWeight / 2) : make_sdesc_k128(sa);
          const uint64_t bdesc = make_sdesc_k128(sa + C::kWeight);
#pragma unroll
          for (int k = 0; k < kSlabK / kMmaK; ++k)
            umma_bf16_1(d_tmem, adesc + (kDA ? 128ull : 2ull) * k, bdesc + 2ull * k, idesc,
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
    const int quarter = warp & 3;
    zero_unowned_rows(static_cast<T*>(args.out), args.ldo, args.feat, s_off[0],
                      s_off[args.experts], args.rows,
                      (long long)blockIdx.x * 128 + (threadIdx.x - 64), gridDim.x * 128ll);
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
      float acc[kTok];
      if (ok) {
        const uint32_t tbase = tmem_base + buf * kTok + ((uint32_t)(quarter * 32) << 16);
#pragma unroll
        for (int c = 0; c < kTok; c += 16) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(tbase + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 16; ++j) acc[c + j] = __uint_as_float(v[j]);
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(smem_u32(&bar_acc_empty[buf]));
      }
      stream_finish<kTok, T>(args, walk, s, quarter, quarter, 0, acc, ok != 0);
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
