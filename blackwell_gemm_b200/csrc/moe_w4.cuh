// Products with 4-bit weights and group scales, one matrix or a bank:
//
//   C[r, n] = sum_k A[r, k] (q[e, n, k] - z[e, n, k / G]) s[e, n, k / G]
//
// with q and z in 0 .. 15 (z = 8 where none are given) and G = 32, 64, 128.
//
// Few rows read every weight for a handful of products each, so the kernel
// is bound by the 4-bit stream from HBM and, close behind, by the integer
// work of unpacking it.  The tensor core takes the rest: warps unpack
// q - z -- small integers, exact in 16 bits -- into TMEM, where they are the
// MMA's A operand (128 weight rows), with the tokens as its N.  A group's
// product leaves the tensor core as fp32 and is multiplied by its scale
// there, in fp32, on the way into the running sum: no weight is ever rounded
// to 16 bits.
//
// Weights are laid out once (w4_pack_kernel) in records of 128 rows x 128 k,
// in the order a CTA walks them, so a record is one bulk copy and a CTA's
// whole share one sequential read:
//   8192 B  q: [4][128 rows][16 B], 32 k in 16 B; in a word the nibbles of
//           k = 0, 2, 4, 6 fill the low half and 1, 3, 5, 7 the high half,
//           so one shift and one mask give a pair in order
//   scales  [128 / G][128 rows], 16-bit
//   zeros   [128 / G][128 rows], 8-bit, when there are any
//
// Work is divided as in moe_stream.cuh (items are records).  Warps: 0 bulk
// and TMA copies, 1 MMA, 2-5 and 6-9 two sets of unpackers that take
// records in turn; a set unpacks record j + 1 while the MMA works on j.
#pragma once
#include "moe_stream.cuh"

namespace b200 {

constexpr int kW4Rows = 128, kW4K = 128, kW4Q = kW4Rows * kW4K / 2;

__host__ __device__ constexpr int w4_record_bytes(int group, bool zeros) {
  return kW4Q + kW4K / group * kW4Rows * (zeros ? 3 : 2);
}

template <int kTok, int kGroup>
struct W4Cfg {
  static constexpr int kSub = kW4K / kGroup;       // groups per record
  static_assert(kTok * kSub <= 128, "a set's products fill at most 128 TMEM columns");
  static constexpr int kTokens = 2 * kTok * 128;   // two 64-k slabs of the token operand
  static constexpr int kRecord = (w4_record_bytes(kGroup, true) + 1023) / 1024 * 1024;
  static constexpr int kStageBytes = kTokens + kRecord;
  static constexpr int kExchange = kTok * 128 * 4;
  static constexpr int kStages = (214 * 1024 - kExchange) / kStageBytes < 16
                                     ? (214 * 1024 - kExchange) / kStageBytes
                                     : 16;
  static constexpr int kThreads = 320;
  static constexpr int smem_bytes(int experts) {
    return kStages * kStageBytes + kExchange + group_table_bytes(experts) + 1024;
  }
};

// Pairs of 4-bit values (low and high half of `v`, already shifted) as 16-bit
// floats: the nibble set into the mantissa of 2^7 (bf16) or 2^10 (f16) gives
// that power plus q; both the sum and the difference taken from it are exact.
template <class T>
struct W4Magic;
template <>
struct W4Magic<__nv_bfloat16> {
  static constexpr uint32_t kBits = 0x43004300u;
  static __device__ __forceinline__ uint32_t bias(uint32_t z) { return (0x4300u + z) * 0x10001u; }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a),
                                     *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float wide(uint16_t s) {
    return __uint_as_float((uint32_t)s << 16);
  }
};
template <>
struct W4Magic<__half> {
  static constexpr uint32_t kBits = 0x64006400u;
  static __device__ __forceinline__ uint32_t bias(uint32_t z) { return (0x6400u + z) * 0x10001u; }
  static __device__ __forceinline__ uint32_t sub(uint32_t a, uint32_t b) {
    const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a),
                              *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&r);
  }
  static __device__ __forceinline__ float wide(uint16_t s) {
    return __half2float(*reinterpret_cast<const __half*>(&s));
  }
};

// tmap_t: the token operand (k, r), box 64 x 16.
template <int kTok, int kGroup, class T>
__global__ void __launch_bounds__(W4Cfg<kTok, kGroup>::kThreads, 1)
w4_stream_kernel(const __grid_constant__ CUtensorMap tmap_t, const StreamArgs args,
                 const bool has_zeros) {
  using C = W4Cfg<kTok, kGroup>;
  using M = W4Magic<T>;
  constexpr int kStages = C::kStages;
  constexpr int kSub = C::kSub;
  extern __shared__ uint8_t smem_raw[];
  __shared__ alignas(8) uint64_t bar_full[kStages];
  __shared__ alignas(8) uint64_t bar_empty[kStages];
  __shared__ alignas(8) uint64_t bar_a_full[2][2];  // [set][buffer]: unpacked weights in TMEM
  __shared__ alignas(8) uint64_t bar_d_full[2];     // [set]: products in TMEM
  __shared__ alignas(8) uint64_t bar_d_empty[2];
  __shared__ alignas(8) uint64_t bar_drain;
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_word;

  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);  // (warp-uniform)
  const int lane = threadIdx.x & 31;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t exchange = smem_base + kStages * C::kStageBytes;
  int* s_off = reinterpret_cast<int*>(smem_raw + (exchange + C::kExchange - smem_u32(smem_raw)));
  int* s_tiles = s_off + args.experts + 1;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 5);  // a set's four warps, and the MMA that read the tokens
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(smem_u32(&bar_a_full[s][0]), 4);
      mbar_init(smem_u32(&bar_a_full[s][1]), 4);
      mbar_init(smem_u32(&bar_d_full[s]), 1);
      mbar_init(smem_u32(&bar_d_empty[s]), 4);
    }
    mbar_init(smem_u32(&bar_drain), 1);
    abort_word = 0;
    fence_mbar_init_cluster();
    prefetch_tmap(&tmap_t);
  }
  if (warp == 1) {
    tmem_alloc_1(smem_u32(&tmem_slot), kTmemCols);
    tmem_relinquish_1();
  }
  if (warp == 2) stream_groups(args, kTok, s_off, s_tiles);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = tmem_slot;
  // TMEM columns: weights [set][buffer] 64 each, then products [set] 128 each
  const uint32_t tmem_d = tmem_base + 256;

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
      bool ok = true;
      while (ok && walk.next(&s)) {
        const uint8_t* records = args.packed + (long long)s.e * args.expert_bytes +
                                 (long long)s.block * args.red_blocks * args.record_bytes;
        const int boxes = (s.rows + 15) / 16;
        for (int kb = s.kb0; kb < s.kb1; ++kb) {
          if (!wait_bounded(smem_u32(&bar_empty[stage]), phase ^ 1u, wctx, kErrWaitEmpty)) {
            ok = false;
            break;
          }
          const uint32_t fb = smem_u32(&bar_full[stage]);
          const uint32_t sa = smem_base + stage * C::kStageBytes;
          mbar_arrive_expect_tx(fb, args.record_bytes + boxes * 2 * 16 * 128);
          bulk_load_hint(sa + C::kTokens, records + (long long)kb * args.record_bytes,
                         args.record_bytes, fb, once);
          for (int i = 0; i < boxes; ++i) {
            tma_load_2d_hint(sa + i * 16 * 128, &tmap_t, kb * kW4K, s.row0 + i * 16, fb, keep);
            tma_load_2d_hint(sa + (kTok + i * 16) * 128, &tmap_t, kb * kW4K + 64, s.row0 + i * 16,
                             fb, keep);
          }
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (elect_one()) {
      uint32_t stage = 0, phase = 0;
      uint32_t item = 0;
      bool ok = true;
      while (ok && walk.next(&s)) {
        const uint32_t idesc = make_idesc_16bit(128, (s.rows + 15) & ~15, kFormat<T>, false, false);
        for (int kb = s.kb0; kb < s.kb1; ++kb, ++item) {
          const uint32_t set = item & 1, j = item >> 1, buf = j & 1;
          if (!wait_bounded(smem_u32(&bar_full[stage]), phase, wctx, kErrWaitFull) ||
              !wait_bounded(smem_u32(&bar_a_full[set][buf]), (j >> 1) & 1, wctx, kErrWaitFull) ||
              !wait_bounded(smem_u32(&bar_d_empty[set]), (j & 1) ^ 1, wctx, kErrWaitAccEmpty)) {
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sx = smem_base + stage * C::kStageBytes;
          const uint32_t a = tmem_base + (set * 2 + buf) * 64;
          const uint32_t d = tmem_d + set * 128;
#pragma unroll
          for (int k = 0; k < kW4K / kMmaK; ++k) {
            const uint64_t bdesc = make_sdesc_k128(sx + (k >> 2) * kTok * 128) + 2ull * (k & 3);
            umma_tmem_a_1(d + k * kMmaK / kGroup * kTok, a + k * 8, bdesc, idesc,
                          k * kMmaK % kGroup != 0 ? 1u : 0u);
          }
          umma_commit_1(smem_u32(&bar_empty[stage]));
          umma_commit_1(smem_u32(&bar_d_full[set]));
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      umma_commit_1(smem_u32(&bar_drain));
      if (!mbar_try_wait(smem_u32(&bar_drain), 0))
        wait_slow(smem_u32(&bar_drain), 0, wctx, kErrWaitDrain, false);
    }
    __syncwarp();
  } else {
    const int set = (warp - 2) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    zero_unowned_rows(static_cast<T*>(args.out), args.ldo, args.feat, s_off[0],
                      s_off[args.experts], args.rows,
                      (long long)blockIdx.x * 256 + (threadIdx.x - 64), gridDim.x * 256ll);
    uint32_t item = 0;  // records this CTA has passed; this set takes every other one
    bool ok = true;
    auto wait_warp = [&](uint32_t bar, uint32_t parity, int code) {
      int got = 0;
      if (lane == 0) got = wait_bounded(bar, parity, wctx, code);
      got = __shfl_sync(0xffffffffu, got, 0);
      __syncwarp();
      return got != 0;
    };
    while (walk.next(&s)) {
      float acc[kTok];
#pragma unroll
      for (int c = 0; c < kTok; ++c) acc[c] = 0.0f;
      float scale[kSub];      // of the record whose products are still to be taken
      bool pending = false;
      uint32_t pending_j = 0;
      // Products of record j times their scales into the running sums.
      auto fold = [&]() {
        if (!wait_warp(smem_u32(&bar_d_full[set]), pending_j & 1, kErrWaitAccFull)) {
          ok = false;
          return;
        }
        tc_fence_after_sync();
#pragma unroll
        for (int g = 0; g < kSub; ++g) {
#pragma unroll
          for (int c = 0; c < kTok; c += 16) {
            if (c < s.rows) {
              uint32_t v[16];
              tmem_ld_32x32b_x16(tmem_d + set * 128 + g * kTok + c + lanes, v);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                acc[c + i] = fmaf(scale[g], __uint_as_float(v[i]), acc[c + i]);
            }
          }
        }
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(smem_u32(&bar_d_empty[set]));
      };
      for (int kb = s.kb0; kb < s.kb1; ++kb, ++item) {
        if ((int)(item & 1) != set || !ok) continue;
        const uint32_t stage = item % kStages, phase = (item / kStages) & 1;
        const uint32_t j = item >> 1, buf = j & 1;
        if (!wait_warp(smem_u32(&bar_full[stage]), phase, kErrWaitFull)) {
          ok = false;
          continue;
        }
        const uint32_t record = smem_base + stage * C::kStageBytes + C::kTokens;
        float next_scale[kSub];
        uint32_t bias[kSub];
#pragma unroll
        for (int g = 0; g < kSub; ++g) {
          next_scale[g] = M::wide(ld_shared_u16(record + kW4Q + (g * 128 + row) * 2));
          bias[g] = M::bias(
              has_zeros ? ld_shared_u8(record + kW4Q + kSub * 256 + g * 128 + row) : 8u);
        }
        // (this buffer's last MMA was record j - 2, whose products this warp
        // has already taken)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t r[32];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t w[4];
            ld_shared_v4_u32(record + (2 * h + c) * 2048 + row * 16, w);
            const uint32_t b = bias[(2 * h + c) * 32 / kGroup];
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
              for (int i = 0; i < 4; ++i)
                r[c * 16 + q * 4 + i] =
                    M::sub(((w[q] >> (4 * i)) & 0x000F000Fu) | M::kBits, b);
          }
          tmem_st_32x32b_x32(tmem_base + (set * 2 + buf) * 64 + h * 32 + lanes, r);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive_local(smem_u32(&bar_empty[stage]));
        tmem_wait_st();
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive_local(smem_u32(&bar_a_full[set][buf]));
        if (pending) fold();
#pragma unroll
        for (int g = 0; g < kSub; ++g) scale[g] = next_scale[g];
        pending = true;
        pending_j = j;
      }
      if (pending && ok) fold();
      // The second set hands its sums to the first, which finishes the tile.
      float* sums = reinterpret_cast<float*>(smem_raw + (exchange - smem_u32(smem_raw))) + row;
      if (set == 1) {
#pragma unroll
        for (int c = 0; c < kTok; ++c)
          if (c < s.rows) sums[c * 128] = acc[c];
        named_bar_sync(1 + quarter, 64);
        named_bar_sync(1 + quarter, 64);
      } else {
        named_bar_sync(1 + quarter, 64);
#pragma unroll
        for (int c = 0; c < kTok; ++c)
          if (c < s.rows) acc[c] += sums[c * 128];
        named_bar_sync(1 + quarter, 64);
        const bool valid =
            __all_sync(0xffffffffu, ok && ld_volatile_shared(wctx.abort_local) == 0);
        stream_finish<kTok, T>(args, walk, s, quarter, acc, valid);
      }
    }
    __syncwarp();
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_1(tmem_base, kTmemCols);
  }
}

// q: experts x N x K / 2 bytes, the low nibble the even k; scales, zeros:
// experts x N x K / group, 16-bit and 8-bit; all contiguous.  One block per
// record; rows and k past the matrix get scale 0 and q = 8.
__global__ void __launch_bounds__(256)
w4_pack_kernel(const uint8_t* __restrict__ q, const uint16_t* __restrict__ scales,
               const uint8_t* __restrict__ zeros, uint8_t* __restrict__ out, int N, int K, int group,
               int blocks, int red_blocks, int record_bytes) {
  const long long rec = blockIdx.x;
  const int kb = (int)(rec % red_blocks);
  const long long eb = rec / red_blocks;
  const int block = (int)(eb % blocks);
  const long long e = eb / blocks;
  uint8_t* dst = out + rec * record_bytes;
  // 128 rows x 16 words of 8 k; consecutive threads share a row's 64 bytes
  for (int i = threadIdx.x; i < kW4Rows * 16; i += blockDim.x) {
    const int row = i >> 4, word = i & 15;
    const int n = block * kW4Rows + row, k = kb * kW4K + word * 8;
    uint32_t v = 0x88888888u;
    if (n < N && k < K) {
      const uint8_t* p = q + ((e * N + n) * (long long)K + k) / 2;
      v = (uint32_t)p[0] | (uint32_t)p[1] << 8 | (uint32_t)p[2] << 16 | (uint32_t)p[3] << 24;
    }
    uint32_t w = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w |= (v >> (8 * j) & 15u) << (4 * j);
      w |= (v >> (8 * j + 4) & 15u) << (16 + 4 * j);
    }
    *reinterpret_cast<uint32_t*>(dst + (word >> 2) * 2048 + row * 16 + (word & 3) * 4) = w;
  }
  const int sub = kW4K / group, groups = K / group;
  for (int i = threadIdx.x; i < kW4Rows * sub; i += blockDim.x) {
    const int row = i / sub, g = i - row * sub;
    const int n = block * kW4Rows + row, kg = kb * sub + g;
    const bool in = n < N && kg < groups;
    const long long at = (e * N + n) * (long long)groups + kg;
    reinterpret_cast<uint16_t*>(dst + kW4Q)[g * 128 + row] = in ? scales[at] : (uint16_t)0;
    if (zeros != nullptr) dst[kW4Q + sub * 256 + g * 128 + row] = in ? zeros[at] & 15u : 8u;
  }
}

}  // namespace b200
